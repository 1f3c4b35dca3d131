// Kernels of the matrix operators (matrix_ops.cuh): orthogonalisation by
// Newton-Schulz products, and the Muon step around it.
//
//   k_matrix_norm   one pass over the matrices for their Frobenius norms; in a
//                   Muon step the same pass unscales and clips the gradient,
//                   updates the momentum and takes the step's decision.
//   k_matrix_split  X = G / (|G| + eps) as fp16 hi + lo, transposed where the
//                   matrix has more rows than columns.
//   k_ns            every product of every matrix in one persistent kernel.
//                   CTAs take tiles from one list in order; the list holds the
//                   products in an order in which every tile's inputs come
//                   before it, and a tile waits (bounded) until the tiles of
//                   its matrix that it reads are counted as done. So a CTA
//                   that waits, waits only for tiles that running CTAs hold,
//                   whatever else runs on the GPU.
//                   One warp loads operand tiles by TMA, one thread issues
//                   tcgen05.mma into one of two TMEM accumulators, four warps
//                   turn finished accumulators into the next operand: A, B =
//                   bA + cAA, X = aX + BX, or the result (for Muon: the
//                   weights' update). A and B are symmetric: only tiles on or
//                   above the diagonal are computed, and each is stored twice.
#include <algorithm>

#include "matrix_ops.cuh"
#include "pipeline.cuh"
#include "step.cuh"

namespace soarb {
namespace {

// ------------------------------------------------------------- elements -----

__device__ __forceinline__ void split_half(float v, __half& hi, __half& lo) {
    hi = __float2half_rn(v);
    lo = __float2half_rn(v - __half2float(hi));
}

// The matrix element a preparation pass works on: the source, or for Muon
// u = g + mu m (Nesterov) or m, from the updated momentum m.
template <int kSrc>
__device__ __forceinline__ float load_grad(const MatrixArgs& a, const NsStack& s, uint64_t at,
                                           const StepCoeffs& k) {
    const void* gp = a.grads[s.tensor];
    const float raw = kSrc == kSrcGradBf16
                          ? bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(gp) + at))
                          : __ldg(static_cast<const float*>(gp) + at);
    return __fmul_rn(__fmul_rn(raw, k.inv), k.coef);
}

__device__ __forceinline__ float direction(const MatrixArgs& a, float d, float mom) {
    return a.nesterov ? __fadd_rn(d, __fmul_rn(a.momentum, mom)) : mom;
}

template <int kSrc>
constexpr bool kIsMuon = kSrc == kSrcGradF32 || kSrc == kSrcGradBf16;

template <int kSrc>
__device__ __forceinline__ float load_src(const NsStack& s, uint64_t at) {
    if constexpr (kSrc == kSrcBf16)
        return bf16_bits_to_f32(__ldg(static_cast<const uint16_t*>(s.src) + at));
    else
        return __ldg(static_cast<const float*>(s.src) + at);
}

template <int kSrc>
__global__ void __launch_bounds__(kThreads)
k_matrix_norm(MatrixArgs a, Ctl* ctl, ApplyArgs step) {
    __shared__ double s_red[32];
    __shared__ StepDecision s_d;
    __shared__ int s_last;
    constexpr bool kMuon = kIsMuon<kSrc>;
    pdl_wait();
    pdl_trigger();
    // the product kernel of the run before is done: its counters start at 0 again
    for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < a.n_matrices; i += gridDim.x * kThreads)
        a.done[i] = 0u;
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.next = 0u;
    StepCoeffs k{1.0f, 1.0f, 0.0f, 1.0f, 1};
    if constexpr (kMuon) {
        if (threadIdx.x == 0) s_d = decide_step(step, ctl);
        __syncthreads();
        k = s_d.k;
    }
    if (!kMuon || !s_d.skip) {
        for (uint32_t q = blockIdx.x; q < a.n_prep; q += gridDim.x) {
            const PrepTile t = a.prep[q];
            const NsStack& s = a.stacks[t.stack];
            const uint32_t c = t.tc * kPrepTile + threadIdx.x % kPrepTile;
            const uint32_t r0 = t.tr * kPrepTile + threadIdx.x / kPrepTile;
            double acc = 0.0;
            if (c < s.cols) {
#pragma unroll 4
                for (uint32_t i = 0; i < kPrepTile; i += kThreads / kPrepTile) {
                    const uint32_t r = r0 + i;
                    if (r >= s.rows) break;
                    float u;
                    if constexpr (kMuon) {
                        const uint64_t at = (static_cast<uint64_t>(t.index) * s.rows + r) * s.cols + c;
                        const float d = load_grad<kSrc>(a, s, at, k);
                        const float m = __fadd_rn(__fmul_rn(a.momentum, s.mom[at]), d);
                        s.mom[at] = m;
                        u = direction(a, d, m);
                    } else {
                        u = load_src<kSrc>(s, t.index * s.src_mat + r * s.src_row + c);
                    }
                    // (the square of a float is exact in 64 bits)
                    acc = fma(static_cast<double>(u), static_cast<double>(u), acc);
                }
            }
            const double sum = block_sum(acc, s_red);
            const uint32_t matrix = s.first + t.index;
            if (threadIdx.x == 0) {
                a.partials[q] = sum;
                __threadfence();
                s_last = atomicAdd(a.tickets + matrix, 1u) == s.tiles - 1;
            }
            __syncthreads();
            if (s_last) {
                // the matrix's last tile: its sums in their order
                __threadfence();
                const double* p = a.partials + s.first_tile + static_cast<uint64_t>(t.index) * s.tiles;
                double v = 0.0;
                for (uint32_t i = threadIdx.x; i < s.tiles; i += kThreads) v += __ldcg(p + i);
                const double total = block_sum(v, s_red);
                if (threadIdx.x == 0) {
                    a.inv[matrix] = static_cast<float>(static_cast<double>(s.sx) / (sqrt(total) + a.eps));
                    a.tickets[matrix] = 0u;
                }
            }
        }
    }
    if constexpr (kMuon) {
        __syncthreads();
        if (threadIdx.x == 0) {
            // (the commit may change the loss scale: the next kernel takes this step's)
            if (blockIdx.x == 0) *a.step = MatrixStep{s_d.skip, k.inv, k.coef};
            commit_step(ctl, step, s_d);
        }
    }
}

template <int kSrc>
__global__ void __launch_bounds__(kThreads)
k_matrix_split(MatrixArgs a) {
    __shared__ float s_t[kPrepTile][kPrepTile + 1];
    constexpr bool kMuon = kIsMuon<kSrc>;
    pdl_wait();
    pdl_trigger();
    StepCoeffs k{1.0f, 1.0f, 0.0f, 1.0f, 1};
    if constexpr (kMuon) {
        const MatrixStep st = *a.step;
        if (st.skip) return;
        k.inv = st.inv;
        k.coef = st.coef;
    }
    for (uint32_t q = blockIdx.x; q < a.n_prep; q += gridDim.x) {
        const PrepTile t = a.prep[q];
        const NsStack& s = a.stacks[t.stack];
        const uint32_t lc = threadIdx.x % kPrepTile, lr = threadIdx.x / kPrepTile;
        const uint32_t c = t.tc * kPrepTile + lc;
        const float inv = a.inv[s.first + t.index];
        __half* xh = s.x[0] + static_cast<uint64_t>(t.index) * s.m * s.ldx;
        __half* xl = s.xl[0] + static_cast<uint64_t>(t.index) * s.m * s.ldx;
#pragma unroll 4
        for (uint32_t i = 0; i < kPrepTile; i += kThreads / kPrepTile) {
            const uint32_t r = t.tr * kPrepTile + lr + i;
            if (r >= s.rows || c >= s.cols) continue;
            float u;
            if constexpr (kMuon) {
                const uint64_t at = (static_cast<uint64_t>(t.index) * s.rows + r) * s.cols + c;
                const float m = s.mom[at];
                u = a.nesterov ? direction(a, load_grad<kSrc>(a, s, at, k), m) : m;
            } else {
                u = load_src<kSrc>(s, t.index * s.src_mat + r * s.src_row + c);
            }
            const float v = __fmul_rn(u, inv);
            if (s.transposed) {
                s_t[lr + i][lc] = v;
            } else {
                __half hi, lo;
                split_half(v, hi, lo);
                const uint64_t at = static_cast<uint64_t>(r) * s.ldx + c;
                xh[at] = hi;
                xl[at] = lo;
            }
        }
        if (s.transposed) {
            __syncthreads();
            const uint32_t r = t.tr * kPrepTile + lc;  // X's column
#pragma unroll 4
            for (uint32_t i = 0; i < kPrepTile; i += kThreads / kPrepTile) {
                const uint32_t xc = t.tc * kPrepTile + lr + i;  // X's row
                if (r >= s.rows || xc >= s.cols) continue;
                __half hi, lo;
                split_half(s_t[lc][lr + i], hi, lo);
                const uint64_t at = static_cast<uint64_t>(xc) * s.ldx + r;
                xh[at] = hi;
                xl[at] = lo;
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------ tcgen05 and TMA -----

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            uint32_t x, uint32_t y, uint32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle (64 fp16 wide rows of 128
// bytes, eight rows to a 1024-byte group). K-major: rows run along M or N,
// groups 1024 bytes apart. MN-major: rows run along K, groups 1024 bytes
// apart, and 64 elements further along M or N lie `lead` bytes away.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t lead) {
    return static_cast<uint64_t>((addr & 0x3FFFFu) >> 4) |
           (static_cast<uint64_t>((lead & 0x3FFFFu) >> 4) << 16) |
           (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// fp16 x fp16 -> fp32, M = 128, N = n; b_mn: the second operand is MN-major.
__device__ __forceinline__ uint32_t instr_desc(uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((kNsTileM >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc,
                                        bool accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     bar)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tc_fence_before() {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_async_proxy() { asm volatile("fence.proxy.async;" ::: "memory"); }
__device__ __forceinline__ uint32_t ld_acquire(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void red_release_add1(uint32_t* p) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}

// Bounded wait until *p >= need; gives up when the kernel's error word is set.
__device__ __forceinline__ bool wait_done(const uint32_t* p, uint32_t need, int* s_err,
                                          const int* err) {
    if (ld_acquire(p) >= need) return true;
    const uint64_t t0 = global_timer_ns();
    for (uint32_t i = 1;; ++i) {
        if (ld_acquire(p) >= need) return true;
        if ((i & 63u) == 0) {
            if (global_timer_ns() - t0 > kWaitLimitNs || *reinterpret_cast<const volatile int*>(err)) {
                atomicOr(s_err, 1);
                return false;
            }
            if (*reinterpret_cast<volatile int*>(s_err)) return false;
        }
    }
}

// 32 consecutive fp16 of one row (16-byte aligned) as floats; columns from
// `left` on are not read.
__device__ __forceinline__ void load_row32(const __half* p, uint32_t left, float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint4 q = make_uint4(0, 0, 0, 0);
        if (static_cast<uint32_t>(j * 8) < left) q = __ldcg(reinterpret_cast<const uint4*>(p) + j);
        const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = __half22float2(h[e]);
            v[j * 8 + 2 * e] = f.x;
            v[j * 8 + 2 * e + 1] = f.y;
        }
    }
}

// The row's 32 values as fp16 (hi, and lo where given), eight to a store. A
// store may run past `left` columns into the row's padding, never further.
template <bool kLo>
__device__ __forceinline__ void store_row32(__half* hp, __half* lp, uint32_t left, const float (&v)[32]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (static_cast<uint32_t>(j * 8) >= left) break;
        __half h[8], l[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) split_half(v[j * 8 + e], h[e], l[e]);
        reinterpret_cast<uint4*>(hp)[j] = *reinterpret_cast<uint4*>(h);
        if constexpr (kLo) reinterpret_cast<uint4*>(lp)[j] = *reinterpret_cast<uint4*>(l);
    }
}

// --------------------------------------------------------------- products ---

template <int kDst>
__global__ void __launch_bounds__(kNsThreads, 1)
k_ns(const __grid_constant__ MatrixArgs a, const __grid_constant__ ApplyArgs step) {
    // fp32 results take three products, bf16 results one
    constexpr bool kThree = kDst == kDstF32 || kDst == kDstParamF32;
    constexpr bool kMuon = kDst == kDstParamF32 || kDst == kDstParamMixed;
    constexpr uint32_t kPasses = kThree ? 3 : 1;
    constexpr int kRing = 4;  // tasks taken ahead
    constexpr uint32_t kEnd = 0xFFFFFFFFu;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kNsStages], empty_bar[kNsStages];
    __shared__ __align__(8) uint64_t acc_full[2], acc_empty[2], task_full[kRing], task_empty[kRing];
    __shared__ __align__(8) uint64_t drain_bar;
    __shared__ NsTask s_task[kRing];
    __shared__ uint32_t s_index[kRing];
    __shared__ uint32_t s_tmem;
    __shared__ int s_err, s_drain_err, s_cfail[2];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if constexpr (kMuon) {
        if (a.step->skip) return;
    }
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kNsStages; ++i) {
            mbar_init(smem_u32(&full_bar[i]), 1);
            mbar_init(smem_u32(&empty_bar[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 128);
        }
        for (int i = 0; i < kRing; ++i) {
            mbar_init(smem_u32(&task_full[i]), 1);
            mbar_init(smem_u32(&task_empty[i]), 2);
        }
        mbar_init(smem_u32(&drain_bar), 1);
        s_err = s_drain_err = s_cfail[0] = s_cfail[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(&s_tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp == 0) {
        // ---- takes tasks, waits for their inputs, loads operand tiles ----
        if (lane == 0) {
            fence_async_proxy();  // (X of the kernel before)
            uint32_t it = 0;      // stages issued
            uint32_t claim = atomicAdd(a.next, 1u);
            for (uint32_t q = 0;; ++q) {
                const uint32_t slot = q % kRing, idx = claim;
                if (q >= kRing && !mbar_wait(smem_u32(&task_empty[slot]), (q / kRing + 1) & 1, &s_err))
                    break;
                const bool end = idx >= a.n_tasks;
                NsTask t{};
                if (!end) {
                    t = a.tasks[idx];
                    s_task[slot] = t;
                }
                s_index[slot] = end ? kEnd : idx;
                mbar_arrive(smem_u32(&task_full[slot]));
                if (end) break;
                claim = atomicAdd(a.next, 1u);
                const NsStack& s = a.stacks[t.stack];
                const CUtensorMap* maps = a.maps + static_cast<uint64_t>(t.stack) * kMapsPerStack;
                if (t.need) {
                    if (!wait_done(a.done + s.first + t.index, t.need, &s_err, a.err)) break;
                    fence_async_proxy();  // written by other SMs' ordinary stores
                }
                const uint32_t row = t.row * kNsTileM, col = t.col * 16u;
                const int xmap = (t.step & 1) ? kMapX1 : kMapX0;
                const bool bx = t.kind >= kNsBX;
                const int ma = t.kind == kNsXXt ? xmap : t.kind == kNsAA ? kMapA : kMapB;
                const int mb = t.kind == kNsAA ? static_cast<int>(kMapA) : xmap;
                const uint32_t depth = t.kind == kNsXXt ? s.n : s.m;
                const uint32_t boxes_a = s.m - row > 64 ? 2 : 1, boxes_b = (t.width + 63u) / 64u;
                const uint32_t bytes = (boxes_a + boxes_b) * kNsBoxBytes;
                bool ok = true;
                for (uint32_t p = 0; p < kPasses && ok; ++p) {
                    // the small products first: lo hi, hi lo, hi hi
                    const CUtensorMap* mapa = maps + ma + (kThree && p == 0 ? kMapLo : 0);
                    const CUtensorMap* mapb = maps + mb + (kThree && p == 1 ? kMapLo : 0);
                    for (uint32_t k0 = 0; k0 < depth; k0 += kNsTileK, ++it) {
                        const uint32_t st = it % kNsStages;
                        if (it >= kNsStages &&
                            !mbar_wait(smem_u32(&empty_bar[st]), (it / kNsStages + 1) & 1, &s_err)) {
                            ok = false;
                            break;
                        }
                        const uint32_t bar = smem_u32(&full_bar[st]);
                        const uint32_t sa = smem + st * kNsStageBytes, sb = sa + 2 * kNsBoxBytes;
                        mbar_expect_tx(bar, bytes);
                        for (uint32_t i = 0; i < boxes_a; ++i)
                            tma_load_3d(sa + i * kNsBoxBytes, mapa, bar, k0, row + 64 * i, t.index);
                        for (uint32_t i = 0; i < boxes_b; ++i) {
                            if (bx)
                                tma_load_3d(sb + i * kNsBoxBytes, mapb, bar, col + 64 * i, k0, t.index);
                            else
                                tma_load_3d(sb + i * kNsBoxBytes, mapb, bar, k0, col + 64 * i, t.index);
                        }
                    }
                }
                if (!ok) break;
            }
            if (*reinterpret_cast<volatile int*>(&s_err)) {
                // copies in flight land before the CTA may end
                for (uint32_t j = it > kNsStages ? it - kNsStages : 0; j < it; ++j)
                    mbar_wait(smem_u32(&full_bar[j % kNsStages]), (j / kNsStages) & 1, &s_drain_err);
            }
        }
    } else if (warp == 1) {
        // ---- one thread issues the products ----
        if (lane == 0) {
            uint32_t it = 0;
            for (uint32_t q = 0;; ++q) {
                const uint32_t slot = q % kRing, buf = q & 1;
                if (!mbar_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err)) break;
                if (s_index[slot] == kEnd) break;
                const NsTask t = s_task[slot];
                mbar_arrive(smem_u32(&task_empty[slot]));
                if (q >= 2 && !mbar_wait(smem_u32(&acc_empty[buf]), (q / 2 + 1) & 1, &s_err)) break;
                tc_fence_after();
                const NsStack& s = a.stacks[t.stack];
                const bool bx = t.kind >= kNsBX;
                const uint32_t idesc = instr_desc((t.width + 15u) & ~15u, bx);
                const uint32_t depth = t.kind == kNsXXt ? s.n : s.m;
                const uint32_t d = tmem + buf * kNsTileN;
                bool ok = true;
                const uint32_t steps = kPasses * ((depth + kNsTileK - 1) / kNsTileK);
                for (uint32_t j = 0; j < steps; ++j, ++it) {
                    const uint32_t st = it % kNsStages;
                    if (!mbar_wait(smem_u32(&full_bar[st]), (it / kNsStages) & 1, &s_err)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem + st * kNsStageBytes, sb = sa + 2 * kNsBoxBytes;
#pragma unroll
                    for (uint32_t k = 0; k < kNsTileK / 16; ++k)
                        mma_f16(d, operand_desc(sa + k * 32, 16),
                                bx ? operand_desc(sb + k * 2048, kNsBoxBytes)
                                   : operand_desc(sb + k * 32, 16),
                                idesc, j + k > 0);
                    mma_commit(smem_u32(&empty_bar[st]));
                }
                if (!ok) break;
                mma_commit(smem_u32(&acc_full[buf]));
            }
            if (*reinterpret_cast<volatile int*>(&s_err)) {
                mma_commit(smem_u32(&drain_bar));
                mbar_wait(smem_u32(&drain_bar), 0, &s_drain_err);
            }
        }
    } else {
        // ---- four warps turn accumulators into operands or results ----
        const uint32_t quad = warp & 3;  // the TMEM lanes this warp may read
        const uint32_t tlane = quad * 32 + lane;
        for (uint32_t q = 0;; ++q) {
            const uint32_t slot = q % kRing, buf = q & 1;
            bool ok = mbar_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err);
            const bool end = ok && s_index[slot] == kEnd;
            if (ok && !end) ok = mbar_wait(smem_u32(&acc_full[buf]), (q / 2) & 1, &s_err);
            if (!ok) s_cfail[q & 1] = 1;
            consumers_sync<128>();
            if (s_cfail[q & 1] || end) break;
            const NsTask t = s_task[slot];
            consumers_sync<128>();
            if (threadIdx.x == 64) mbar_arrive(smem_u32(&task_empty[slot]));
            tc_fence_after();
            const NsStack& s = a.stacks[t.stack];
            const uint32_t r = t.row * kNsTileM + tlane;
            const uint32_t col0 = t.col * 16u;
            const bool sym = t.kind <= kNsAA;
            const uint32_t cols = sym ? s.m : s.n;
            const float ca = a.coef[t.step][0], cb = a.coef[t.step][1], cc = a.coef[t.step][2];
            const uint64_t abase = static_cast<uint64_t>(t.index) * s.m * s.lda;
            const uint64_t xbase = static_cast<uint64_t>(t.index) * s.m * s.ldx;
            for (uint32_t c = 0; c < t.width; c += 32) {
                float v[32];
                __syncwarp();
                tmem_ld32(tmem + buf * kNsTileN + ((quad * 32u) << 16) + c, v);
                const uint32_t col = col0 + c;
                if (r >= s.m || col >= cols) continue;
                const uint32_t left = cols - col;
                if (sym) {
                    __half* hp = t.kind == kNsXXt ? s.a : s.b;
                    __half* lp = t.kind == kNsXXt ? s.al : s.bl;
                    const uint64_t at = abase + static_cast<uint64_t>(r) * s.lda + col;
                    if (t.kind == kNsXXt) {
                        const float f = kNsScaleA / (s.sx * s.sx);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] *= f;
                    } else {
                        float x[32];
                        load_row32(s.a + at, left, x);
                        if constexpr (kThree) {
                            float y[32];
                            load_row32(s.al + at, left, y);
#pragma unroll
                            for (int j = 0; j < 32; ++j) x[j] += y[j];
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = cb * x[j] + (cc / kNsScaleA) * v[j];
                    }
                    store_row32<kThree>(hp + at, lp + at, left, v);
                    // the mirror image: right of the block on the diagonal
                    if (col >= (t.row + 1u) * kNsTileM) {
                        const uint64_t to = abase + static_cast<uint64_t>(col) * s.lda + r;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (static_cast<uint32_t>(j) >= left) break;
                            __half hi, lo;
                            split_half(v[j], hi, lo);
                            hp[to + static_cast<uint64_t>(j) * s.lda] = hi;
                            if constexpr (kThree) lp[to + static_cast<uint64_t>(j) * s.lda] = lo;
                        }
                    }
                } else {
                    const int in = t.step & 1;
                    const uint64_t at = xbase + static_cast<uint64_t>(r) * s.ldx + col;
                    {
                        float x[32], y[32];
                        load_row32(s.x[in] + at, left, x);
                        load_row32(s.xl[in] + at, left, y);
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            v[j] = ca * (x[j] + y[j]) + v[j] * (1.0f / kNsScaleA);
                    }
                    if (t.kind == kNsBX) {
                        store_row32<true>(s.x[in ^ 1] + at, s.xl[in ^ 1] + at, left, v);
                    } else {
                        const float f = 1.0f / s.sx;
                        const uint64_t mat = t.index;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (static_cast<uint32_t>(j) >= left) break;
                            const float o = v[j] * f;
                            const uint64_t orow = s.transposed ? col + j : r;
                            const uint64_t ocol = s.transposed ? r : col + j;
                            if constexpr (kDst == kDstF32) {
                                static_cast<float*>(s.dst)[mat * s.dst_mat + orow * s.dst_row + ocol] = o;
                            } else if constexpr (kDst == kDstBf16) {
                                static_cast<uint16_t*>(
                                    s.dst)[mat * s.dst_mat + orow * s.dst_row + ocol] = f32_to_bf16_rn(o);
                            } else {
                                const uint64_t e = (mat * s.rows + orow) * s.cols + ocol;
                                float w = s.master[e];
                                if (s.wd != 0.0f)
                                    w = __fsub_rn(w, __fmul_rn(__fmul_rn(step.lr, s.wd), w));
                                w = __fsub_rn(w, __fmul_rn(__fmul_rn(step.lr, s.factor), o));
                                s.master[e] = w;
                                if constexpr (kDst == kDstParamMixed)
                                    static_cast<uint16_t*>(s.param)[e] = f32_to_bf16_rn(w);
                                if (a.ema) {
                                    float* sh = s.mom + step.ema_delta;
                                    sh[e] = __fadd_rn(__fmul_rn(step.ema_decay, sh[e]),
                                                      __fmul_rn(step.ema_omd, w));
                                }
                            }
                        }
                    }
                }
            }
            tc_fence_before();
            mbar_arrive(smem_u32(&acc_empty[buf]));
            // this tile's stores, before it counts as done
            __threadfence();
            fence_async_proxy();
            consumers_sync<128>();
            if (threadIdx.x == 64) red_release_add1(a.done + s.first + t.index);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && (s_err | s_drain_err)) atomicOr(a.err, 1);
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int kSrc>
cudaError_t launch_prep(const MatrixArgs& a, Ctl* ctl, const ApplyArgs& step, int sms,
                        cudaStream_t stream) {
    const int grid = static_cast<int>(std::min<uint64_t>(std::max(1u, a.n_prep), 8ull * sms));
    cudaError_t e = launch_pdl(k_matrix_norm<kSrc>, dim3(grid), dim3(kThreads), 0, stream, a, ctl, step);
    if (e != cudaSuccess || a.n_prep == 0) return e;
    return launch_pdl(k_matrix_split<kSrc>, dim3(grid), dim3(kThreads), 0, stream, a);
}

template <int kDst>
cudaError_t launch_ns(const MatrixArgs& a, const ApplyArgs& step, int sms, cudaStream_t stream) {
    const int grid = static_cast<int>(std::min<uint64_t>(a.n_tasks, static_cast<uint64_t>(sms)));
    return launch_pdl(k_ns<kDst>, dim3(grid), dim3(kNsThreads), kNsSmemBytes, stream, a, step);
}

}  // namespace

cudaError_t prepare_matrix_kernels() {
    const void* fns[] = {reinterpret_cast<const void*>(k_ns<kDstF32>),
                         reinterpret_cast<const void*>(k_ns<kDstBf16>),
                         reinterpret_cast<const void*>(k_ns<kDstParamF32>),
                         reinterpret_cast<const void*>(k_ns<kDstParamMixed>)};
    for (const void* f : fns) {
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(kNsSmemBytes));
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

cudaError_t launch_matrix_ops(const MatrixArgs& a, int source, int dest, Ctl* ctl,
                              const ApplyArgs* step, int sms, cudaStream_t stream) {
    const ApplyArgs none{};
    const ApplyArgs& st = step ? *step : none;
    cudaError_t e;
    switch (source) {
        case kSrcF32: e = launch_prep<kSrcF32>(a, ctl, st, sms, stream); break;
        case kSrcBf16: e = launch_prep<kSrcBf16>(a, ctl, st, sms, stream); break;
        case kSrcGradF32: e = launch_prep<kSrcGradF32>(a, ctl, st, sms, stream); break;
        default: e = launch_prep<kSrcGradBf16>(a, ctl, st, sms, stream); break;
    }
    if (e != cudaSuccess || a.n_tasks == 0) return e;
    switch (dest) {
        case kDstF32: return launch_ns<kDstF32>(a, st, sms, stream);
        case kDstBf16: return launch_ns<kDstBf16>(a, st, sms, stream);
        case kDstParamF32: return launch_ns<kDstParamF32>(a, st, sms, stream);
        default: return launch_ns<kDstParamMixed>(a, st, sms, stream);
    }
}

}  // namespace soarb
