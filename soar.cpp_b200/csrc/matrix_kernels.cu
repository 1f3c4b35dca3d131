// Kernels of the matrix operators (matrix_ops.cuh): orthogonalisation by
// Newton-Schulz products, and the Muon step around it.
//
//   k_matrix_norm   one pass over the matrices for their Frobenius norms (64-bit
//                   sums, in a fixed order); in a Muon step the same pass
//                   unscales and clips the gradient, updates the momentum and
//                   takes the step's decision. Bound by memory: 200M mixed
//                   parameters, 10 bytes each, 338 to 347 us (5.9 TB/s).
//   k_matrix_split  X = G / (|G| + eps) as fp16 hi and lo, transposed where the
//                   matrix has more rows than columns. Bound by memory: the
//                   same parameters, 9 bytes each, 371 to 401 us (4.7 TB/s).
//   k_ns            every product of every matrix in one persistent kernel, a
//                   pair of CTAs to an SM pair. Pairs take tiles from one list
//                   in order; the list holds the products in an order in which
//                   every tile's inputs come before it, and a tile waits
//                   (bounded) until the tiles of its matrix that it reads are
//                   counted as done. So a pair that waits, waits only for
//                   tiles that running pairs hold, whatever else runs on the
//                   GPU. One warp loads operand tiles by TMA, one issues
//                   tcgen05.mma into one of two TMEM accumulators, one hands
//                   out tiles, one brings what the epilogue adds, two store,
//                   and eight turn finished accumulators into the next operand:
//                   A, B = aI + bA + cAA, X = BX, or the result (for Muon: the
//                   weights' update). A and B are symmetric: only tiles on or
//                   above the diagonal are computed, and each is stored twice.
//                   Large matrices are bound by the products (4096 x 4096 and
//                   2048 x 8192: 1.49 ms, 1.30 PFLOP/s with A and B
//                   counted by half, 0.79 of the library's rate for one
//                   large product), small ones by the epilogue (a 256 x 256 tile of
//                   depth 320 is multiplied in 1.4 us and passed on in about
//                   4) and by the wait from one product to the next, about 9 us.
//   k_panel         matrices of at most 256 rows (of X), whole, by a pair each.
//   k_few           matrices of at most 8 rows (of X), whole, by a CTA each.
#include <algorithm>

#include "matrix_ops.cuh"
#include "pipeline.cuh"
#include "step.cuh"

namespace soarb {
namespace {

// ------------------------------------------------------------- elements -----

template <int kSrc>
constexpr bool kIsMuon = kSrc == kSrcGradF32 || kSrc == kSrcGradBf16;
template <int kDst>  // (results in fp32 take three, all in k_ns)
constexpr bool kOneProduct = kDst == kDstBf16 || kDst == kDstParamMixed;
template <int kSrc>
constexpr bool kIsBf16 = kSrc == kSrcBf16 || kSrc == kSrcGradBf16;

// Up to four adjacent elements from `at` on, as floats (vec: all four, aligned).
template <bool kBf16>
__device__ __forceinline__ void read4(const void* p, uint64_t at, bool vec, uint32_t left, float (&v)[4]) {
    if constexpr (kBf16) {
        const uint16_t* q = static_cast<const uint16_t*>(p) + at;
        if (vec) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(q));
            v[0] = bf16_lo(w.x), v[1] = bf16_hi(w.x), v[2] = bf16_lo(w.y), v[3] = bf16_hi(w.y);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = e < left ? bf16_bits_to_f32(__ldg(q + e)) : 0.0f;
        }
    } else {
        const float* q = static_cast<const float*>(p) + at;
        if (vec) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(q));
            v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = e < left ? __ldg(q + e) : 0.0f;
        }
    }
}

// A preparation tile's 64 x 64 part: sixteen threads to a row, four elements
// each, sixteen rows at a time.
struct PrepPart {
    uint32_t row, col, left;  // this thread's first row and column, and its columns in the matrix
    const void* src;
    uint64_t at, pitch;       // of its first element, and from row to row
    bool vec;
};

template <int kSrc>
__device__ __forceinline__ PrepPart prep_part(const MatrixArgs& a, const NsStack& s, const PrepTile& t, uint32_t part) {
    const bool down = s.rows > s.cols;  // a tile's parts lie along the longer side
    PrepPart p;
    p.row = (t.tr + (down ? part : 0)) * kPrepTile + threadIdx.x / 16;
    p.col = (t.tc + (down ? 0 : part)) * kPrepTile + threadIdx.x % 16 * 4;
    p.left = p.col < s.cols ? s.cols - p.col : 0;
    if constexpr (kIsMuon<kSrc>) {
        p.src = a.grads[s.tensor];
        p.pitch = s.cols;
        p.at = static_cast<uint64_t>(t.index) * s.rows * s.cols;
    } else {
        p.src = s.src;
        p.pitch = s.src_row;
        p.at = t.index * s.src_mat;
    }
    const uintptr_t vector = kIsBf16<kSrc> ? 8 : 16;
    p.vec = p.left >= 4 && ((p.at | p.pitch) & 3u) == 0 && reinterpret_cast<uintptr_t>(p.src) % vector == 0 &&
            (!kIsMuon<kSrc> || reinterpret_cast<uintptr_t>(s.mom) % 16 == 0);
    p.at += p.row * p.pitch + p.col;
    return p;
}

// (Four 16-byte loads a thread leave the memory idle while the four are worked on; the next
// four asked for ahead: 46M-parameter Muon step 1612 -> 1580 us, 200M 5950 -> 5880.)
__device__ __forceinline__ void prefetch_l2(const void* p) {
    asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
}

// Unscaled and clipped.
__device__ __forceinline__ float clipped(float raw, const StepCoeffs& k) {
    return __fmul_rn(__fmul_rn(raw, k.inv), k.coef);
}

// 2^k, for -126 <= k <= 127.
__device__ __forceinline__ float pow2(int k) { return __uint_as_float(static_cast<uint32_t>(127 + k) << 23); }

// From a matrix's norm: what its X is held by before each step (powers of two), and what
// its elements are multiplied by at the start (by x, then by y: numbers at the end of fp32's
// range need more than one factor). `bound` is one of X's singular values, which
// a step multiplies by at most |a| + |b| bound^2 + |c| bound^4: they are held at 1/2 to 1 times
// sx, or, from a bound of 1/2 on, times sx itself.
__device__ __noinline__ float2 hold_lifted(const MatrixArgs& a, float sx, double norm, NsHold* hold) {
    constexpr int kMostLift = 100;
    const double full = norm + a.eps;
    // (NaN for zeros with an eps of 0 and of an inf or NaN: not lifted)
    float bound = static_cast<float>(norm / full);
    auto scale_of = [&]() {
        if (!(bound < 0.5f)) return sx;
        return sx * pow2(min(kMostLift, 126 - static_cast<int>(__float_as_uint(bound) >> 23)));
    };
    float scale = scale_of();
    float2 inv = make_float2(0.0f, 1.0f);  // (zeros with an eps of 0 stay zeros)
    if (full != 0.0) {
        const double q = static_cast<double>(scale) / full;
        if (q >= 0x1p64) inv = make_float2(static_cast<float>(q * 0x1p-64), 0x1p64f);
        else inv.x = static_cast<float>(q);
    }
    for (int i = 0; i < a.steps; ++i) {
        const float* c = a.coef[i];
        const float s2 = bound * bound, one_over = __fdiv_rn(1.0f, scale);
        bound *= fabsf(c[0]) + s2 * (fabsf(c[1]) + s2 * fabsf(c[2]));
        scale = scale_of();
        hold[i] = NsHold{one_over, scale * one_over};
    }
    return inv;
}
__device__ __forceinline__ float2 hold_x(const MatrixArgs& a, const NsStack& s, double norm, NsHold* hold) {
    const double q = static_cast<double>(s.sx) / (norm + a.eps);
    // (a bound of 1/2 or more stays one)
    if (!(norm >= a.eps && q < 0x1p64 && a.grows)) return hold_lifted(a, s.sx, norm, hold);
    for (int i = 0; i < a.steps; ++i) hold[i] = NsHold{s.one_over_sx, 1.0f};
    return make_float2(static_cast<float>(q), 1.0f);
}

template <int kSrc>
__global__ void __launch_bounds__(kThreads, 4)
k_matrix_norm(const __grid_constant__ MatrixArgs a, Ctl* ctl, ApplyArgs step) {
    __shared__ double s_red[32];
    __shared__ StepDecision s_d;
    __shared__ int s_last;
    constexpr bool kMuon = kIsMuon<kSrc>;
    pdl_wait();
    pdl_trigger();
    // the product kernels of the run before are done: their counters start at 0 again
    for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < a.n_matrices; i += gridDim.x * kThreads)
        a.done[i] = 0u;
    if (blockIdx.x == 0 && threadIdx.x < 2) a.next[threadIdx.x] = 0u;
    if (blockIdx.x == 0 && threadIdx.x == 2) *a.gave_up = 0u;
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
            double acc = 0.0;
            // (the square of a float is exact in 64 bits; what is not in the matrix is 0)
            auto square = [&](float x) { acc = fma(static_cast<double>(x), static_cast<double>(x), acc); };
            if constexpr (kMuon) {
                // A parameter's matrix is one run of elements, cut evenly whatever its columns: a tile
                // takes vectors of four from the run's first boundary of four on, tile 0 what is
                // before it, the last tile what is left over.
                const uint64_t numel = static_cast<uint64_t>(s.rows) * s.cols, base = t.index * numel;
                const uint32_t tile = q - s.first_tile - t.index * s.tiles;
                const uint64_t chunk = ((numel + s.tiles - 1) / s.tiles + 3) & ~3ull;
                const void* g = a.grads[s.tensor];
                float* mom = s.mom + base;
                const uint64_t lead = (16 - (reinterpret_cast<uintptr_t>(mom) & 15)) / 4 & 3;
                constexpr uint32_t kElem = kIsBf16<kSrc> ? 2 : 4;
                const bool vec = (reinterpret_cast<uintptr_t>(g) + (base + lead) * kElem) % (4 * kElem) == 0;
                const uint64_t from = tile * chunk + lead, end = from + chunk < numel ? from + chunk : numel;
                auto take = [&](float raw, float& m) {
                    const float d = clipped(raw, k);
                    m = __fadd_rn(__fmul_rn(a.momentum, m), d);
                    square(a.nesterov ? __fadd_rn(d, __fmul_rn(a.momentum, m)) : m);
                };
                auto alone = [&](uint64_t i) {
                    float one[4], m = mom[i];
                    read4<kIsBf16<kSrc>>(g, base + i, false, 1, one);
                    take(one[0], m);
                    mom[i] = m;
                };
                if (tile == 0 && threadIdx.x < lead && threadIdx.x < numel) alone(threadIdx.x);
                for (uint64_t i0 = from + 4 * threadIdx.x; i0 < end; i0 += 16 * kThreads) {
                    float u[4][4], m[4][4];
                    if ((threadIdx.x & 7) == 0) {
                        // the next ones' lines on their way to the L2 cache
#pragma unroll
                        for (uint32_t v = 4; v < 8; ++v) {
                            const uint64_t i = i0 + v * 4 * kThreads;
                            if (i >= end) continue;
                            prefetch_l2(static_cast<const char*>(g) + (base + i) * kElem);
                            prefetch_l2(mom + i);
                        }
                    }
#pragma unroll
                    for (uint32_t v = 0; v < 4; ++v) {
                        const uint64_t i = i0 + v * 4 * kThreads;
                        if (!vec || i + 4 > end) continue;
                        read4<kIsBf16<kSrc>>(g, base + i, true, 4, u[v]);
                        *reinterpret_cast<float4*>(m[v]) = *reinterpret_cast<const float4*>(mom + i);
                    }
#pragma unroll
                    for (uint32_t v = 0; v < 4; ++v) {
                        const uint64_t i = i0 + v * 4 * kThreads;
                        if (vec && i + 4 <= end) {
#pragma unroll
                            for (uint32_t e = 0; e < 4; ++e) take(u[v][e], m[v][e]);
                            *reinterpret_cast<float4*>(mom + i) = *reinterpret_cast<const float4*>(m[v]);
                        } else {
                            for (uint64_t e = i; e < end && e < i + 4; ++e) alone(e);
                        }
                    }
                }
            } else {
                const uint32_t rows = s.rows;
                for (uint32_t part = 0; part < t.parts; ++part) {
                    const PrepPart p = prep_part<kSrc>(a, s, t, part);
                    float u[4][4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const bool in = p.left && p.row + 16 * i < rows;
                        read4<kIsBf16<kSrc>>(p.src, p.at + 16 * i * p.pitch, p.vec && in, in ? p.left : 0, u[i]);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) square(u[i][e]);
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
                    a.inv[matrix] = hold_x(a, s, sqrt(total), a.hold + static_cast<uint64_t>(matrix) * a.steps);
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

// Two values as e5m2, the first in the low byte.
__device__ __forceinline__ uint32_t e5m2x2(float a, float b) {
    uint16_t d;
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(d) : "f"(b), "f"(a));
    return d;
}

// Four adjacent elements of X as hi and lo, lo in 16 or in 8 bits. `at` is a
// multiple of four, and a row of X goes on to one: the last ones may be padding,
// which then takes the zeros it has.
__device__ __forceinline__ void put_x4(const NsStack& s, uint64_t at, const float (&v)[4]) {
    __half hi[4];
    float lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = __float2half_rn(v[e]);
        lo[e] = v[e] - __half2float(hi[e]);
    }
    *reinterpret_cast<uint2*>(s.x[0] + at) = *reinterpret_cast<const uint2*>(hi);
    if (!s.three) {
        *reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(s.xl[0]) + at) =
            e5m2x2(lo[0] * kLoScale, lo[1] * kLoScale) |
            e5m2x2(lo[2] * kLoScale, lo[3] * kLoScale) << 16;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) hi[e] = __float2half_rn(lo[e]);
        *reinterpret_cast<uint2*>(s.xl[0] + at) = *reinterpret_cast<const uint2*>(hi);
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
    // In a Muon step the last tiles first: k_matrix_norm has left their momentum in the L2 cache,
    // and the products begin with what comes last here (46M parameters: 1614 -> 1606 us).
    for (uint32_t q = blockIdx.x; q < a.n_prep; q += gridDim.x) {
        const PrepTile t = a.prep[kMuon ? a.n_prep - 1 - q : q];
        const NsStack& s = a.stacks[t.stack];
        const float2 inv = a.inv[s.first + t.index];
        const uint32_t rows = s.rows, cols = s.cols, ldx = s.ldx;
        const bool transposed = s.transposed != 0;
        const uint64_t matrix = static_cast<uint64_t>(t.index) * s.m * ldx;
        for (uint32_t part = 0; part < t.parts; ++part) {
            const PrepPart p = prep_part<kSrc>(a, s, t, part);
            float u[4][4], m[4][4];
            if (part + 1 < t.parts && (threadIdx.x & 7) == 0) {
                // the next part's lines on their way to the L2 cache
                const uint64_t ahead = p.at + (transposed ? kPrepTile * p.pitch : kPrepTile);
                const uint32_t row = p.row + (transposed ? kPrepTile : 0), col = p.col + (transposed ? 0 : kPrepTile);
                constexpr uint32_t kElem = kIsBf16<kSrc> ? 2 : 4;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (row + 16 * i >= rows || col >= cols) continue;
                    if (!kMuon || a.nesterov)
                        prefetch_l2(static_cast<const char*>(p.src) + (ahead + 16 * i * p.pitch) * kElem);
                    if constexpr (kMuon) prefetch_l2(s.mom + ahead + 16 * i * p.pitch);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const bool in = p.left && p.row + 16 * i < rows;
                const uint64_t at = p.at + 16 * i * p.pitch;
                if (!kMuon || a.nesterov)
                    read4<kIsBf16<kSrc>>(p.src, at, p.vec && in, in ? p.left : 0, u[i]);
                if constexpr (kMuon) {
                    if (p.vec && in) {
                        *reinterpret_cast<float4*>(m[i]) = *reinterpret_cast<const float4*>(s.mom + at);
                    } else {
#pragma unroll
                        for (uint32_t e = 0; e < 4; ++e) m[i][e] = in && e < p.left ? s.mom[at + e] : 0.0f;
                    }
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint32_t r = p.row + 16 * i;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    if constexpr (kMuon)
                        u[i][e] = a.nesterov ? __fadd_rn(clipped(u[i][e], k), __fmul_rn(a.momentum, m[i][e])) : m[i][e];
                    u[i][e] = __fmul_rn(u[i][e], inv.x);
                    if (inv.y != 1.0f) u[i][e] = __fmul_rn(u[i][e], inv.y);
                }
                if (!transposed) {
                    if (p.left && r < rows) put_x4(s, matrix + static_cast<uint64_t>(r) * ldx + p.col, u[i]);
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) s_t[threadIdx.x / 16 + 16 * i][threadIdx.x % 16 * 4 + e] = u[i][e];
                }
            }
            if (transposed) {
                __syncthreads();
                // four source rows (X's columns) of one source column (X's row)
                const uint32_t r0 = (p.row - threadIdx.x / 16) + threadIdx.x % 16 * 4;
                const uint32_t c0 = p.col - threadIdx.x % 16 * 4;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const uint32_t c = threadIdx.x / 16 + 16 * i;
                    if (r0 >= rows || c0 + c >= cols) continue;
                    float v[4];
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) v[e] = s_t[threadIdx.x % 16 * 4 + e][c];
                    put_x4(s, matrix + static_cast<uint64_t>(c0 + c) * ldx + r0, v);
                }
                __syncthreads();
            }
        }
    }
}

// ------------------------------------------------------ tcgen05 and TMA -----

// The other CTA's (or this one's) copy of a shared-memory address.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// One lane of a converged warp, the same at every call. (Copies and products are
// issued from converged warps: their operands then stay in uniform registers.
// From a loop of one lane, each instruction cost 130 to 330 cycles, a stage of
// four copies more than 1000 where its products take 512.)
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xFFFFFFFF; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile(
        "barrier.cluster.arrive.release.aligned;\n"
        "barrier.cluster.wait.acquire.aligned;" ::
            : "memory");
}
// Arrives on a barrier of either CTA of the pair. What such a barrier orders is
// shared memory and TMEM that the pair's products read and write (through the
// async proxy, fenced for that), not global memory: a release at cluster scope
// would first wait for all of the thread's global accesses, about a microsecond.
// Without it nothing orders plain reads of shared memory before the arrival.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The same where it does order global memory, or plain reads of shared memory.
__device__ __forceinline__ void mbar_arrive_release(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_acquire(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; "
        "selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// Bounded waits, as pipeline.cuh's mbar_wait and wait_flags; the clock is first
// read after a thousand failed tries (%globaltimer is slow to read).
struct Patience {
    uint64_t t0 = 0;
    uint32_t tries = 0;
    // false: give up
    __device__ __forceinline__ bool more(int* s_err) {
        if ((++tries & 1023u) != 0) return true;
        if (*reinterpret_cast<volatile int*>(s_err)) return false;  // another thread gave up
        const uint64_t now = global_timer_ns();
        if (t0 == 0) t0 = now;
        if (now - t0 <= kWaitLimitNs) return true;
        atomicOr(s_err, 1);
        return false;
    }
};
// A converged warp's value, known to the compiler to be the same in all lanes.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_max_sync(0xFFFFFFFFu, x); }

// A converged warp's wait.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* s_err) {
    Patience p;
    while (!__all_sync(0xFFFFFFFFu, mbar_try(bar, parity)))
        if (!__all_sync(0xFFFFFFFFu, p.more(s_err))) return false;
    return true;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int* s_err) {
    Patience p;
    while (!mbar_try(bar, parity))
        if (!p.more(s_err)) return false;
    return true;
}
// The same for what mbar_arrive_release orders.
__device__ __forceinline__ bool warp_wait_acquire(uint32_t bar, uint32_t parity, int* s_err) {
    Patience p;
    while (!__all_sync(0xFFFFFFFFu, mbar_try_acquire(bar, parity)))
        if (!__all_sync(0xFFFFFFFFu, p.more(s_err))) return false;
    return true;
}
__device__ __forceinline__ bool bar_wait_acquire(uint32_t bar, uint32_t parity, int* s_err) {
    Patience p;
    while (!mbar_try_acquire(bar, parity))
        if (!p.more(s_err)) return false;
    return true;
}
// Sixteen bytes into the other CTA's shared memory, counted on a barrier there.
__device__ __forceinline__ void st_async_v4(uint32_t addr, const uint4& v, uint32_t bar) {
    asm volatile(
        "st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
        "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(bar)
        : "memory");
}

// Into this CTA's shared memory; the bytes count on `bar` of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                              uint32_t x, uint32_t y, uint32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                              uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, uint32_t bar, uint32_t x,
                                         uint32_t y, uint32_t z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, uint32_t x, uint32_t y,
                                          uint32_t z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(
                     map),
                 "r"(src), "r"(x), "r"(y), "r"(z)
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

// fp16 x fp16 -> fp32, M = 256 over the pair, N = n; b_mn: the second operand is MN-major.
__device__ __forceinline__ uint32_t instr_desc(uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((kNsTileM >> 4) << 24);
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc,
                                        bool accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// Arrives on `bar` of both CTAs when the products issued so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
          "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
          "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
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
__device__ __forceinline__ void fence_async_shared() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ uint32_t ld_acquire(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void red_release_add1(uint32_t* p) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(p) : "memory");
}

// Bounded wait until *p >= need; gives up when another CTA of this run has.
__device__ __forceinline__ bool wait_done(const uint32_t* p, uint32_t need, int* s_err,
                                          const uint32_t* gave_up) {
    Patience wait;
    while (ld_acquire(p) < need) {
        if (!wait.more(s_err)) return false;
        if ((wait.tries & 1023u) == 0 && *reinterpret_cast<const volatile uint32_t*>(gave_up)) {
            atomicOr(s_err, 1);
            return false;
        }
    }
    return true;
}

// ---------------------------------------------------------------- staging ---
// The epilogue's operands pass through shared memory in chunks of 64 columns
// of the CTA's 128 rows: a slot holds one fp16 chunk as TMA has it (rows of 128
// bytes, 128-byte swizzle).

// Byte offset of eight columns (group j of 8) of a row in a slot.
__device__ __forceinline__ uint32_t slot_at(uint32_t row, uint32_t j) {
    return row * 128u + ((j ^ (row & 7u)) << 4);
}
// Byte offset of (row, col) in a slot that holds the chunk's transpose: 64
// rows (its columns) of 128 (its rows), in two boxes of 64 x 64.
__device__ __forceinline__ uint32_t mirror_at(uint32_t row, uint32_t col) {
    return (row >> 6) * kNsBoxBytes + col * 128u + ((((row & 63u) >> 3) ^ (col & 7u)) << 4) + (row & 7u) * 2u;
}
// Word offset of (row, col) of a chunk of floats in two slots, 32 columns in
// each, a row where its fp16 are otherwise. Rows and columns are both read and
// written without bank conflicts.
__device__ __forceinline__ uint32_t block_at(uint32_t row, uint32_t col) {  // of a warp's 32 x 32
    return row * 32u + (((col >> 2) ^ (row & 7u)) << 2) + ((col + (row >> 3)) & 3u);
}
__device__ __forceinline__ uint32_t float_at(uint32_t row, uint32_t col) {
    return (col >> 5) * (kNsSlotBytes / 4) + (row & ~31u) * 32u + block_at(row & 31u, col & 31u);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr));
    return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
                 "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"(static_cast<uint16_t>(v)) : "memory");
}

// Byte offset of sixteen columns (group j of 4) of a row of a slot of 8-bit lo:
// rows of 64 bytes, 64-byte swizzle.
__device__ __forceinline__ uint32_t lo8_at(uint32_t row, uint32_t j) {
    return row * 64u + ((j ^ (row >> 1 & 3u)) << 4);
}
// v += f times the thread's row of a slot: 32 fp16.
__device__ __forceinline__ void add_half(uint32_t slot, uint32_t row, float f, float* v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint4 q = lds128(slot + lo8_at(row, j));
        const __half2* h = reinterpret_cast<const __half2*>(&q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 x = __half22float2(h[e]);
            v[j * 8 + 2 * e] = __fmaf_rn(f, x.x, v[j * 8 + 2 * e]);
            v[j * 8 + 2 * e + 1] = __fmaf_rn(f, x.y, v[j * 8 + 2 * e + 1]);
        }
    }
}
// v += f times sixteen lo (group j of the thread's row).
__device__ __forceinline__ void add_lo8(uint32_t slot, uint32_t row, uint32_t j, float f, float* v) {
    const uint4 p = lds128(slot + lo8_at(row, j));
    const uint32_t word[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        // (an e5m2 number is the upper byte of an fp16 one)
        const uint32_t lo01 = __byte_perm(word[e], 0, 0x1404), lo23 = __byte_perm(word[e], 0, 0x3424);
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&lo01));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&lo23));
        v[4 * e] = __fmaf_rn(f, x.x, v[4 * e]);
        v[4 * e + 1] = __fmaf_rn(f, x.y, v[4 * e + 1]);
        v[4 * e + 2] = __fmaf_rn(f, y.x, v[4 * e + 2]);
        v[4 * e + 3] = __fmaf_rn(f, y.y, v[4 * e + 3]);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Four values as packed fp16, and what is left of them in 8 bits.
__device__ __forceinline__ uint32_t split4(const float* v, uint32_t& h0, uint32_t& h1) {
    h0 = pack2(v[0], v[1]);
    h1 = pack2(v[2], v[3]);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h0));
    const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&h1));
    return e5m2x2((v[0] - x.x) * kLoScale, (v[1] - x.y) * kLoScale) |
           e5m2x2((v[2] - y.x) * kLoScale, (v[3] - y.y) * kLoScale) << 16;
}

// Two values as packed fp16 (hi), and what is left of them (lo).
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}

// --------------------------------------------------------------- products ---

// Where a stack's result goes, in registers.
struct Target {
    void* dst;          // the destination, or the parameters
    float* master;
    float* ema;
    uint64_t base, pitch;
    float lr_wd, lr_s;  // Muon: lr times the weight decay, and times the shape factor
    bool vec;           // in place for vectors of four
};

// A 32 x 32 block of the result, from floats in shared memory (`fs`, rows of 32,
// block_at), to the stack's destination or into Muon's update of the weights
// there. A lane has one column of it (`by_rows`) or one row, whose `count`
// elements lie `inc` apart from `to` on: either way a warp's accesses are
// consecutive. Sixteen weights at a time are read before the first is written,
// so that a block costs two round trips to memory.
template <int kDst>
__device__ __forceinline__ void put_block(const ApplyArgs& step, const Target& s, bool ema, const float* fs,
                                          bool by_rows, uint32_t lane, uint64_t to, uint64_t inc,
                                          uint32_t count) {
    auto value = [&](uint32_t i) { return by_rows ? fs[block_at(i, lane)] : fs[block_at(lane, i)]; };
    if constexpr (kDst == kDstF32 || kDst == kDstBf16) {
        if constexpr (kDst == kDstF32) {
            float* p = static_cast<float*>(s.dst) + to;
#pragma unroll 8
            for (uint32_t i = 0; i < count; ++i, p += inc) *p = value(i);
        } else {
            uint16_t* p = static_cast<uint16_t*>(s.dst) + to;
#pragma unroll 8
            for (uint32_t i = 0; i < count; ++i, p += inc) *p = f32_to_bf16_rn(value(i));
        }
    } else {
#pragma unroll 1
        for (uint32_t from = 0; from < count; from += 16, to += 16 * inc) {
            float w[16];
            const float* r = s.master + to;
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i, r += inc) w[i] = from + i < count ? *r : 0.0f;
            float* q = s.master + to;
            uint16_t* p = static_cast<uint16_t*>(s.dst) + to;
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i, q += inc, p += inc) {
                if (s.lr_wd != 0.0f) w[i] = __fsub_rn(w[i], __fmul_rn(s.lr_wd, w[i]));
                w[i] = __fsub_rn(w[i], __fmul_rn(s.lr_s, value(from + i)));
                if (from + i >= count) continue;
                *q = w[i];
                if constexpr (kDst == kDstParamMixed) *p = f32_to_bf16_rn(w[i]);
            }
            if (ema) {
                float* e = s.ema + to;
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i, e += inc)
                    if (from + i < count)
                        *e = __fadd_rn(__fmul_rn(step.ema_decay, *e), __fmul_rn(step.ema_omd, w[i]));
            }
        }
    }
}

// The same for a whole block in place for vectors (Target::vec): four lines of 32
// elements at a time, four elements to a lane. A line is a row of X, or a column
// where X is the transpose.
template <int kDst>
__device__ __forceinline__ void put_block4(const ApplyArgs& step, const Target& s, bool ema, const float* fs,
                                           bool by_rows, uint32_t lane, uint64_t to) {
    constexpr bool kMuon = kDst == kDstParamF32 || kDst == kDstParamMixed;
    constexpr bool kHalf = kDst == kDstBf16 || kDst == kDstParamMixed;  // writes bf16
    const uint32_t l = lane >> 3, k = 4 * (lane & 7);
    to += l * s.pitch + k;
    const uint64_t inc = 4 * s.pitch;
    float4 w[8];
    if constexpr (kMuon) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const float4*>(s.master + to + i * inc);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t line = 4 * i + l;
        float o[4];
        if (by_rows) {
            // the four lie in one 16-byte group, turned by line / 8 = i / 2
            const float4 q = *reinterpret_cast<const float4*>(fs + line * 32 + ((k >> 2 ^ (line & 7u)) << 2));
            const float t[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[e] = t[(e + i / 2) & 3];
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) o[e] = fs[block_at(k + e, line)];
        }
        if constexpr (kMuon) {
            float* v = &w[i].x;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                if (s.lr_wd != 0.0f) v[e] = __fsub_rn(v[e], __fmul_rn(s.lr_wd, v[e]));
                v[e] = __fsub_rn(v[e], __fmul_rn(s.lr_s, o[e]));
                o[e] = v[e];
            }
            *reinterpret_cast<float4*>(s.master + to + i * inc) = w[i];
        }
        if constexpr (kHalf)
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(s.dst) + to + i * inc) =
                make_uint2(pack_bf16x2_rn(o[0], o[1]), pack_bf16x2_rn(o[2], o[3]));
        else if constexpr (!kMuon)
            *reinterpret_cast<float4*>(static_cast<float*>(s.dst) + to + i * inc) = make_float4(o[0], o[1], o[2], o[3]);
    }
    if (kMuon && ema) {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            float4* p = reinterpret_cast<float4*>(s.ema + to + i * inc);
            float4 e = *p;
            e.x = __fadd_rn(__fmul_rn(step.ema_decay, e.x), __fmul_rn(step.ema_omd, w[i].x));
            e.y = __fadd_rn(__fmul_rn(step.ema_decay, e.y), __fmul_rn(step.ema_omd, w[i].y));
            e.z = __fadd_rn(__fmul_rn(step.ema_decay, e.z), __fmul_rn(step.ema_omd, w[i].z));
            e.w = __fadd_rn(__fmul_rn(step.ema_decay, e.w), __fmul_rn(step.ema_omd, w[i].w));
            *p = e;
        }
    }
}

// The block of X at (y, x), which is the caller's matrix or its transpose.
template <int kDst>
__device__ __forceinline__ void put_transposed_or_not(const ApplyArgs& step, const Target& s, bool ema,
                                                      const float* fs, bool transposed, uint32_t lane, uint32_t y,
                                                      uint32_t x, uint32_t m, uint32_t n) {
    if (s.vec && y + 32 <= m && x + 32 <= n) {
        put_block4<kDst>(step, s, ema, fs, !transposed, lane,
                         s.base + static_cast<uint64_t>(transposed ? x : y) * s.pitch + (transposed ? y : x));
        return;
    }
    const uint32_t mine = (transposed ? y : x) + lane, first = transposed ? x : y;
    if (mine >= (transposed ? m : n)) return;
    const uint32_t end = transposed ? n : m;
    const uint32_t count = first >= end ? 0 : end - first < 32 ? end - first : 32;
    put_block<kDst>(step, s, ema, fs, !transposed, lane, s.base + static_cast<uint64_t>(first) * s.pitch + mine,
                    s.pitch, count);
}

// Where a matrix of a stack goes.
template <int kDst>
__device__ __forceinline__ Target target_of(const NsStack& s, uint32_t index, const ApplyArgs& step, bool ema) {
    constexpr bool kMuon = kDst == kDstParamF32 || kDst == kDstParamMixed;
    constexpr bool kHalf = kDst == kDstBf16 || kDst == kDstParamMixed;
    Target t;
    t.dst = kMuon ? s.param : s.dst;
    t.master = s.master;
    t.ema = s.mom + step.ema_delta;
    t.base = kMuon ? static_cast<uint64_t>(index) * s.rows * s.cols : static_cast<uint64_t>(index) * s.dst_mat;
    t.pitch = kMuon ? s.cols : s.dst_row;
    t.lr_wd = __fmul_rn(step.lr, s.wd);
    t.lr_s = __fmul_rn(step.lr, s.factor);
    // four elements from a multiple of four on lie on a vector's boundary
    t.vec = ((t.base | t.pitch) & 3u) == 0 && (reinterpret_cast<uintptr_t>(t.dst) & (kHalf ? 7u : 15u)) == 0 &&
            (!kMuon || ((reinterpret_cast<uintptr_t>(t.master) |
                         (ema ? reinterpret_cast<uintptr_t>(t.ema) : 0)) & 15u) == 0);
    return t;
}

template <int kDst>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kNsThreads, 1)
k_ns(const __grid_constant__ MatrixArgs a, const __grid_constant__ ApplyArgs step) {
    constexpr bool kMuon = kDst == kDstParamF32 || kDst == kDstParamMixed;
    constexpr int kRing = 2;  // tasks handed out: one at work, one next
    constexpr int kMathWarp = 6;            // the first of them
    constexpr uint32_t kEnd = 0xFFFFFFFFu;  // stack of a task that ends the list
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kNsStages], empty_bar[kNsStages];
    __shared__ __align__(8) uint64_t acc_full[2], acc_empty[2], task_full[kRing], task_empty[kRing];
    __shared__ __align__(8) uint64_t in_full[2 * kNsGroups], in_empty[2 * kNsGroups];
    __shared__ __align__(8) uint64_t out_empty[kNsGroups];
    __shared__ __align__(8) uint64_t out_full[2][kNsGroups];  // of even and of odd tiles
    __shared__ __align__(8) uint64_t drain_bar;
    __shared__ __align__(16) NsTask s_task[kRing];
    __shared__ uint32_t s_tmem;
    __shared__ int s_err, s_drain_err;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if constexpr (kMuon) {
        if (a.step->skip) return;
    }
    const uint32_t rank = blockIdx.x & 1u;  // 0 leads the pair: hands out tasks, issues products
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t in_slots = smem + kNsStages * kNsStageBytes;
    const uint32_t out_slots = in_slots + 2 * kNsGroups * kLoBytes;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kNsStages; ++i) {
            mbar_init(smem_u32(&full_bar[i]), 1);
            mbar_init(smem_u32(&empty_bar[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&acc_full[i]), 1);
            mbar_init(smem_u32(&acc_empty[i]), 2 * kNsMathWarps);  // both CTAs' warps
        }
        for (int i = 0; i < kNsGroups; ++i) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_u32(&in_full[2 * i + b]), 1);
                mbar_init(smem_u32(&in_empty[2 * i + b]), kNsMathWarps / kNsGroups);
            }
            for (int odd = 0; odd < 2; ++odd) mbar_init(smem_u32(&out_full[odd][i]), kNsMathWarps / kNsGroups);
            mbar_init(smem_u32(&out_empty[i]), 1);
        }
        for (int i = 0; i < kRing; ++i) {
            mbar_init(smem_u32(&task_full[i]), 1);
            // the leader: five readers, the arithmetic and the other CTA's word that it is done too;
            // the other CTA: four readers and the arithmetic
            mbar_init(smem_u32(&task_empty[i]), (rank == 0 ? 6 : 4) + kNsMathWarps);
            if (rank == 1) mbar_expect_tx(smem_u32(&task_full[i]), sizeof(NsTask));
        }
        mbar_init(smem_u32(&drain_bar), 1);
        s_err = s_drain_err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(&s_tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    // A reader of the tasks is done with slot q (one lane).
    auto release_task = [&](uint32_t slot) { mbar_arrive(smem_u32(&task_empty[slot])); };

    // What the epilogue does with a tile: chunks of 64 columns, taken by the two groups of its
    // warps by turns, `ins` slots to add to each (in order) and `outs` buffers made of each.
    struct Tile {
        uint32_t row0, col0, chunks, ins, outs;
        bool sym, three, lo, some, mirror;
    };
    auto tile_of = [&](const NsTask& t) {
        Tile u;
        u.row0 = t.row() + rank * kNsRows;
        u.col0 = t.col();
        u.chunks = (t.width() + 63u) / 64u;
        u.sym = t.kind() <= kNsAA;
        u.three = t.three();
        u.lo = !u.sym || u.three;                   // made of hi and lo
        u.some = u.row0 < t.m;                      // this CTA has rows in the tile
        u.mirror = u.sym && u.col0 >= t.row() + kNsTileM;  // right of the diagonal's block
        // A in two halves (and its lo), or X's lo where the product takes hi alone
        u.ins = t.kind() == kNsXXt ? 0 : u.sym ? (u.three ? 4 : 2) : (u.three ? 0 : 1);
        u.outs = u.three && u.mirror ? 2 : 1;
        return u;
    };

    if (warp == 0) {
        // ---- loads operand tiles ----
        fence_async_proxy();  // (X of the kernel before)
        uint32_t st = 0, phase = 1;  // the next stage; its empty barrier's phase to wait for
        uint32_t issued = 0;
        const uint32_t lead_full = uniform(map_to(smem_u32(&full_bar[0]), 0));
        for (uint32_t q = 0;; ++q) {
            const uint32_t slot = q % kRing;
            bool ok = warp_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const uint32_t stack = uniform(s_task[slot].stack);
            if (stack == kEnd) break;
            const uint32_t index = uniform(s_task[slot].index), place = uniform(s_task[slot].place);
            const uint32_t shape = uniform(s_task[slot].shape);
            const uint32_t tm = uniform(s_task[slot].m), tn = uniform(s_task[slot].n);
            __syncwarp();
            if (lane == 0) {
                // (the record of the slot's next task counts on its barrier as it comes)
                if (rank == 1) mbar_expect_tx(smem_u32(&task_full[slot]), sizeof(NsTask));
                release_task(slot);
            }
            const uint32_t width = shape & 0xFFFFu, kind = shape >> 16 & 15u, three = shape >> 20 & 1u;
            const CUtensorMap* maps = a.maps + static_cast<uint64_t>(stack) * kMapsPerStack;
            const bool bx = kind >= kNsBX;
            const uint32_t xmap = shape >> 24 & 1u ? kMapX1 : kMapX0;
            // this CTA's 128 rows of the first operand, its half of the second one's columns
            const bool narrow = width <= kNsTileN / 2;
            const uint32_t n_half = narrow ? kNsTileN / 4 : kNsTileN / 2;
            const uint32_t row = (place & 0xFFFFu) * kNsTileM + rank * kNsRows;
            const uint32_t col = (place >> 16) * 32u + rank * n_half;
            const uint32_t ma = kind == kNsXXt ? xmap : kind == kNsAA ? kMapA : kMapB;
            const uint32_t mb = (kind == kNsAA ? static_cast<uint32_t>(kMapA) : xmap) + (bx ? kMapN : 0) +
                                (narrow ? kMap64 : 0);
            const uint32_t depth = kind == kNsXXt ? tn : tm;
            // both CTAs' bytes count on the leader's barrier (boxes past the edge come as zeros)
            const uint32_t bytes = 4 * kNsBoxBytes + (narrow ? 2 : 4) * kNsBoxBytes;
            // The block on A's or B's diagonal, the largest, comes last: each addition rounds a
            // sum towards zero by up to 2^-23 of it, and few follow then.
            uint32_t first_k = kind == kNsXXt ? 0 : (place & 0xFFFFu) * kNsTileM + kNsTileM;
            if (first_k >= depth) first_k = 0;
            for (uint32_t p = three ? 0 : 2; p < 3 && ok; ++p) {
                // three products: the small ones first, lo hi, hi lo, hi hi
                const CUtensorMap* mapa = maps + ma + (p == 0 ? kMapLo : 0);
                const CUtensorMap* mapb = maps + mb + (p == 1 ? kMapLo : 0);
                for (uint32_t j = 0, k0 = first_k; j < depth; j += kNsTileK) {
                    ok = warp_wait(smem_u32(&empty_bar[st]), phase, &s_err);
                    if (!ok) break;
                    if (elect_one()) {
                        const uint32_t bar = lead_full + st * 8;
                        const uint32_t sa = smem + st * kNsStageBytes, sb = sa + 2 * kNsBoxBytes;
                        if (rank == 0) mbar_expect_tx(smem_u32(&full_bar[st]), bytes);
                        tma_load_pair(sa, mapa, bar, k0, row, index);
                        if (bx)
                            tma_load_pair(sb, mapb, bar, 0, k0, col / 64, index);
                        else
                            tma_load_pair(sb, mapb, bar, k0, col, index);
                    }
                    ++issued;
                    k0 += kNsTileK;
                    if (k0 >= depth) k0 = 0;
                    if (++st == kNsStages) {
                        st = 0;
                        phase ^= 1;
                    }
                }
            }
            if (!ok) break;
        }
        if (*reinterpret_cast<volatile int*>(&s_err) && rank == 0 && lane == 0) {
            // copies in flight land before the CTA may end
            for (uint32_t j = issued > kNsStages ? issued - kNsStages : 0; j < issued; ++j)
                bar_wait(smem_u32(&full_bar[j % kNsStages]), (j / kNsStages) & 1, &s_drain_err);
        }
    } else if (warp == 1) {
        // ---- the leader's second warp issues the pair's products ----
        uint32_t st = 0, phase = 0;  // the next stage; its full barrier's phase to wait for
        for (uint32_t q = 0; rank == 0; ++q) {
            const uint32_t slot = q % kRing, buf = q & 1;
            bool ok = warp_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            if (uniform(s_task[slot].stack) == kEnd) break;
            const uint32_t shape = uniform(s_task[slot].shape);
            const uint32_t width = shape & 0xFFFFu, kind = shape >> 16 & 15u, three = shape >> 20 & 1u;
            const uint32_t depth = uniform(kind == kNsXXt ? s_task[slot].n : s_task[slot].m);
            __syncwarp();
            if (lane == 0) release_task(slot);
            const bool bx = kind >= kNsBX;
            const uint32_t idesc = instr_desc(width <= kNsTileN / 2 ? kNsTileN / 2 : kNsTileN, bx);
            const uint32_t d = uniform(tmem) + buf * kNsTileN;
            const uint32_t blocks = (depth + kNsTileK - 1) / kNsTileK;
            // three products: the last one's first half has an accumulator of its own
            const uint32_t from = three ? 2 * blocks : 0, to = from + (three ? blocks / 2 : 0);
            const uint32_t steps = three ? 3 * blocks : blocks;
            // K steps of 16 lie 32 bytes apart in K-major operands, sixteen rows of 128 in the other
            const uint64_t da0 = operand_desc(smem, 16);
            const uint64_t db0 = operand_desc(smem + 2 * kNsBoxBytes, bx ? kNsBoxBytes : 16);
            const uint32_t db_k = bx ? 2048 >> 4 : 32 >> 4;
            if (q >= 2) ok = warp_wait(smem_u32(&acc_empty[buf]), (q / 2 + 1) & 1, &s_err);
            if (!ok) break;
            tc_fence_after();
            for (uint32_t j = 0; j < steps; ++j) {
                ok = warp_wait(smem_u32(&full_bar[st]), phase, &s_err);
                if (!ok) break;
                tc_fence_after();
                const bool second = j >= from && j < to;
                const uint32_t dd = d + (second ? kNsTileN / 2 : 0);
                const bool fresh = j == 0 || (second && j == from);
                if (elect_one()) {
                    const uint64_t da = da0 + st * (kNsStageBytes >> 4), db = db0 + st * (kNsStageBytes >> 4);
                    mma_f16(dd, da, db, idesc, !fresh);
#pragma unroll
                    for (uint32_t k = 1; k < kNsTileK / 16; ++k)
                        mma_f16(dd, da + k * 2, db + k * db_k, idesc, true);
                    mma_commit(smem_u32(&empty_bar[st]));
                    if (j + 1 == steps) mma_commit(smem_u32(&acc_full[buf]));
                }
                if (++st == kNsStages) {
                    st = 0;
                    phase ^= 1;
                }
            }
            if (!ok) break;
        }
        if (*reinterpret_cast<volatile int*>(&s_err) && rank == 0) {
            if (elect_one()) mma_commit(smem_u32(&drain_bar));
            bar_wait(smem_u32(&drain_bar), 0, &s_drain_err);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---- the leader hands out tasks, to both CTAs, once their inputs are there ----
        if (rank == 0 && lane == 0) {
            // A tile is taken only when the arithmetic begins with the last but one: a pair that
            // holds more leaves others without, and the next product waits for it (2048 x 2048 in
            // fp32 with two more taken ahead: 890 instead of 610 us).
            for (uint32_t q = 0;; ++q) {
                const uint32_t slot = q % kRing;
                if (q >= kRing && !bar_wait_acquire(smem_u32(&task_empty[slot]), (q / kRing + 1) & 1, &s_err))
                    break;
                const uint32_t claim = atomicAdd(a.next, 1u);
                NsTask t{};
                if (claim < a.n_tasks) t = a.tasks[claim];
                else t.stack = kEnd;
                if (t.stack != kEnd) {
                    t.hold = a.hold[static_cast<uint64_t>(t.matrix) * a.steps + t.step()];
                    if (t.need) {
                        if (!wait_done(a.done + t.matrix, t.need, &s_err, a.gave_up)) break;
                        fence_async_proxy();  // (other SMs' stores, by TMA, before loads by TMA)
                    }
                }
                const uint32_t there = map_to(smem_u32(&s_task[slot]), 1);
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    st_async_v4(there + 16 * i, reinterpret_cast<const uint4*>(&t)[i],
                                map_to(smem_u32(&task_full[slot]), 1));
                s_task[slot] = t;
                mbar_arrive(smem_u32(&task_full[slot]));
                if (t.stack == kEnd) break;
            }
        } else if (rank == 1 && lane == 0) {
            // the other CTA's reads of a slot come before the leader's next write into it: its readers
            // count here, and one thread without global accesses of its own passes that on
            for (uint32_t q = 0;; ++q) {
                const uint32_t slot = q % kRing;
                if (!bar_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err)) break;
                if (s_task[slot].stack == kEnd) break;
                if (!bar_wait(smem_u32(&task_empty[slot]), (q / kRing) & 1, &s_err)) break;
                mbar_arrive_release(map_to(smem_u32(&task_empty[slot]), 0));
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        // ---- brings what the epilogue adds ----
        fence_async_proxy();  // (X of the kernel before)
        uint32_t chunk = 0, turns = 0, phases = ~0u;  // chunks so far; by group, its next slot; by slot, its phase
        for (uint32_t q = 0;; ++q) {
            const uint32_t slot = q % kRing;
            bool ok = warp_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const NsTask t = s_task[slot];
            if (t.stack == kEnd) break;
            __syncwarp();
            if (lane == 0) release_task(slot);
            const Tile u = tile_of(t);
            if (!u.some) continue;
            const CUtensorMap* src = a.maps + static_cast<uint64_t>(t.stack) * kMapsPerStack +
                                     (u.sym ? kMapA + kMap32 : kMapLo + (t.step() & 1 ? kMapX1 : kMapX0));
            for (uint32_t c = 0; c < u.chunks && ok; ++c) {
                const uint32_t g = (chunk + c) % kNsGroups;
                for (uint32_t i = 0; i < u.ins && ok; ++i) {
                    const uint32_t b = 2 * g + (turns >> g & 1u);
                    turns ^= 1u << g;
                    ok = warp_wait(smem_u32(&in_empty[b]), phases >> b & 1u, &s_err);
                    if (!ok) break;
                    phases ^= 1u << b;
                    if (elect_one()) {
                        const uint32_t bar = smem_u32(&in_full[b]);
                        mbar_expect_tx(bar, kLoBytes);
                        tma_load(in_slots + b * kLoBytes, src + (i >= 2 ? kMapLo : 0), bar, u.col0 + c * 64 + (i & 1) * 32,
                                 u.row0, t.index);
                    }
                    __syncwarp();
                }
            }
            if (!ok) break;
            chunk += u.chunks;
        }
        if (*reinterpret_cast<volatile int*>(&s_err))
            // copies in flight land before the CTA may end
            for (uint32_t b = 0; b < 2 * kNsGroups; ++b)
                bar_wait(smem_u32(&in_full[b]), phases >> b & 1u, &s_drain_err);
        __syncwarp();
    } else if (warp < kMathWarp) {
        // ---- two warps, by turns, store what a tile makes: one waits for its tile's stores to
        // land while the other issues the next one's ----
        const uint32_t odd = warp & 1u;
        uint32_t chunk = 0, phases = 0;  // chunks so far; by group: its full buffer's phase to wait for
        for (uint32_t q = 0;; ++q) {
            const uint32_t slot = q % kRing;
            bool ok = warp_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const NsTask t = s_task[slot];
            if (t.stack == kEnd) break;
            __syncwarp();
            if (lane == 0) release_task(slot);
            const Tile u = tile_of(t);
            if (!u.some) continue;
            if ((q & 1) != odd) {
                chunk += u.chunks;
                continue;
            }
            const bool last = t.kind() == kNsLast;
            const CUtensorMap* dst = a.maps + static_cast<uint64_t>(t.stack) * kMapsPerStack +
                                     (t.kind() == kNsXXt ? kMapA
                                      : u.sym            ? kMapB
                                      : t.step() & 1     ? kMapX0
                                                         : kMapX1);
            const uint32_t units = u.chunks * u.outs;
            for (uint32_t i = 0; i < units; ++i) {
                const uint32_t c = u.outs == 2 ? i >> 1 : i, g = (chunk + c) % kNsGroups;
                const uint32_t at = out_slots + g * 2 * kNsSlotBytes;
                ok = warp_wait(smem_u32(&out_full[odd][g]), phases >> g & 1u, &s_err);
                if (!ok) break;
                phases ^= 1u << g;
                if (elect_one()) {
                    if (last) {  // (the result has left with the arithmetic)
                        mbar_arrive(smem_u32(&out_empty[g]));
                    } else {
                        const uint32_t x = u.col0 + c * 64;
                        const bool image_only = u.outs == 2 && (i & 1);
                        if (!image_only) {
                            tma_store(dst, at, x, u.row0, t.index);
                            if (u.lo) tma_store(dst + kMapLo, at + kNsSlotBytes, x, u.row0, t.index);
                        }
                        if (u.mirror && (image_only || !u.three)) {
                            const uint32_t image = at + (image_only ? 0 : kNsSlotBytes);
                            for (uint32_t h = 0; h < 2 && u.row0 + h * 64 < t.m; ++h) {
                                tma_store(dst + kMap64, image + h * kNsBoxBytes, u.row0 + h * 64, x, t.index);
                                if (image_only)
                                    tma_store(dst + kMapLo + kMap64, at + kNsSlotBytes + h * kNsBoxBytes,
                                              u.row0 + h * 64, x, t.index);
                            }
                        }
                        bulk_commit();
                        // a buffer is free once its stores have read it: seen when the other group's
                        // are on their way, or now where it is the same group's turn again or nobody's
                        const bool at_once = u.outs == 2 || i + 1 == units;
                        if (i > 0 && u.outs == 1) {
                            if (at_once) bulk_wait_read<0>();
                            else bulk_wait_read<1>();
                            mbar_arrive(smem_u32(&out_empty[(g + 1) % kNsGroups]));
                        }
                        if (at_once) {
                            bulk_wait_read<0>();
                            mbar_arrive(smem_u32(&out_empty[g]));
                        }
                        if (i + 1 == units) {
                            bulk_wait_all();  // this tile's stores, before it counts as done
                            fence_async_proxy();
                            __threadfence();
                            red_release_add1(a.done + t.matrix);
                        }
                    }
                }
                __syncwarp();
            }
            if (!ok) break;
            chunk += u.chunks;
        }
        __syncwarp();
    } else {
        // ---- arithmetic: two groups of four warps; a warp has 32 rows of its group's chunks ----
        const uint32_t quad = warp & 3, group = (warp - kMathWarp) >> 2;
        const uint32_t trow = quad * 32 + lane;  // this thread's row (TMEM lane) of the CTA's 128
        const uint32_t at = out_slots + group * 2 * kNsSlotBytes;
        const uint32_t out_free = smem_u32(&out_empty[group]);
        uint32_t chunk = 0, turn = 0, in_phases = 0, out_phase = 1;  // turn: the group's next in slot
        for (uint32_t q = 0;; ++q) {
            const uint32_t slot = q % kRing, buf = q & 1;
            if (!warp_wait(smem_u32(&task_full[slot]), (q / kRing) & 1, &s_err)) break;
            const NsTask t = s_task[slot];
            if (t.stack == kEnd) break;
            __syncwarp();
            if (lane == 0) release_task(slot);
            const Tile u = tile_of(t);
            const bool last = t.kind() == kNsLast;
            const uint32_t out_bar = smem_u32(&out_full[q & 1][group]);
            Target target{};
            if (last) target = target_of<kDst>(a.stacks[t.stack], t.index, step, a.ema != 0);
            const float ca = a.coef[t.step()][0], cb = a.coef[t.step()][1], cc = a.coef[t.step()][2];
            const bool two = u.three && (t.kind() == kNsXXt ? t.n : t.m) > kNsTileK;  // two accumulators
            // v = fv accumulator + fx addend (+ ca on the diagonal)
            const float regrade = last ? 1.0f : t.hold.regrade;
            const float fx = u.sym ? cb : ca * regrade;
            const float fv = t.kind() == kNsXXt  ? kNsScaleA * t.hold.inv * t.hold.inv
                             : t.kind() == kNsAA ? cc / kNsScaleA
                                                 : regrade / kNsScaleA;
            if (!warp_wait(smem_u32(&acc_full[buf]), (q / 2) & 1, &s_err)) break;
            tc_fence_after();
            bool ok = true, held = true;
            for (uint32_t c = 0; c < u.chunks && ok; ++c) {
                if (((u.some ? chunk : 0) + c) % kNsGroups != group) continue;
                const uint32_t col = u.col0 + c * 64;
                float v[64];
                const uint32_t acc = tmem + buf * kNsTileN + ((quad * 32u) << 16) + c * 64;
                __syncwarp();
                tmem_ld32(acc, v);
                tmem_ld32(acc + 32, v + 32);
                if (two) {
                    float w[32];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        tmem_ld32(acc + kNsTileN / 2 + h * 32, w);
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[h * 32 + j] += w[j];
                    }
                }
                if (c + kNsGroups >= u.chunks) {  // the group's last of this tile
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(map_to(smem_u32(&acc_empty[buf]), 0));
                    held = false;
                }
                if (!u.some) continue;
#pragma unroll
                for (int j = 0; j < 64; ++j) v[j] *= fv;
                auto take = [&](auto&& add) {
                    const uint32_t b = 2 * group + turn;
                    ok = ok && warp_wait(smem_u32(&in_full[b]), in_phases >> turn & 1u, &s_err);
                    in_phases ^= 1u << turn;
                    turn ^= 1;
                    add(in_slots + b * kLoBytes);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&in_empty[b]));
                };
                if (u.ins == 1) {
                    take([&](uint32_t slot) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) add_lo8(slot, trow, j, fx / kLoScale, v + 16 * j);
                    });
                } else if (u.ins) {
                    for (uint32_t i = 0; i < u.ins; i += 2) {
                        take([&](uint32_t slot) { add_half(slot, trow, fx, v); });
                        take([&](uint32_t slot) { add_half(slot, trow, fx, v + 32); });
                    }
                }
                if (!ok) break;
                if (t.kind() == kNsAA) {
                    const uint32_t diag = u.row0 + trow - col;  // (no match: no column)
#pragma unroll
                    for (int j = 0; j < 64; ++j) v[j] += diag == static_cast<uint32_t>(j) ? ca * kNsScaleA : 0.0f;
                }
                ok = ok && warp_wait(out_free, out_phase, &s_err);
                if (!ok) break;
                out_phase ^= 1;
                if (last) {
                    // through shared memory as floats, the warp's own 32 rows, so that the result is
                    // written along the rows of the caller's matrix
                    const float f = t.hold.inv;
                    float* fs = reinterpret_cast<float*>(smem_raw + (at - smem_u32(smem_raw)));
#pragma unroll
                    for (int j = 0; j < 64; ++j) fs[float_at(trow, j)] = v[j] * f;
                    __syncwarp();
#pragma unroll 1
                    for (uint32_t k = 0; k < 2; ++k) {
                        const uint32_t y = u.row0 + quad * 32, x = col + k * 32;  // the block's first element
                        put_transposed_or_not<kDst>(step, target, a.ema != 0, fs + float_at(quad * 32, k * 32),
                                                    t.transposed(), lane, y, x, t.m, t.n);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(out_bar);
                    continue;
                }
                if (!u.sym && !u.three) {
                    // hi, and lo in 8 bits
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t h[8], l[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) l[e] = split4(v + 16 * j + 4 * e, h[2 * e], h[2 * e + 1]);
                        sts128(at + slot_at(trow, 2 * j), make_uint4(h[0], h[1], h[2], h[3]));
                        sts128(at + slot_at(trow, 2 * j + 1), make_uint4(h[4], h[5], h[6], h[7]));
                        sts128(at + kNsSlotBytes + lo8_at(trow, j), make_uint4(l[0], l[1], l[2], l[3]));
                    }
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(out_bar);
                    continue;
                }
                // hi and lo; the mirror image in the second slot, or (hi and lo) in the buffer after them
                uint32_t h[32], l[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) split2(v[2 * j], v[2 * j + 1], h[j], l[j]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t o = slot_at(trow, j);
                    sts128(at + o, make_uint4(h[4 * j], h[4 * j + 1], h[4 * j + 2], h[4 * j + 3]));
                    if (u.lo)
                        sts128(at + kNsSlotBytes + o, make_uint4(l[4 * j], l[4 * j + 1], l[4 * j + 2], l[4 * j + 3]));
                }
                if (u.mirror) {
                    uint32_t image = at + kNsSlotBytes;
                    if (u.outs == 2) {
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(out_bar);
                        ok = warp_wait(out_free, out_phase, &s_err);
                        if (!ok) break;
                        out_phase ^= 1;
                        image = at;
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const uint32_t m0 = mirror_at(trow, 2 * j), m1 = mirror_at(trow, 2 * j + 1);
                        sts16(image + m0, h[j] & 0xFFFFu);
                        sts16(image + m1, h[j] >> 16);
                        if (u.lo) {
                            sts16(image + kNsSlotBytes + m0, l[j] & 0xFFFFu);
                            sts16(image + kNsSlotBytes + m1, l[j] >> 16);
                        }
                    }
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(out_bar);
            }
            if (!ok) break;
            if (held) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(map_to(smem_u32(&acc_empty[buf]), 0));
            }
            if (u.some) chunk += u.chunks;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && (s_err | s_drain_err)) {
        atomicOr(a.err, 1);
        atomicOr(a.gave_up, 1u);
        // the other CTA's copies may still be landing here, or counting on barriers here
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {}
    }
    __syncthreads();
    cluster_sync();  // the other CTA may use this one's shared memory until it is done too
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ----------------------------------------------------- one pair, one matrix ---
// k_panel: the whole iteration of a matrix with at most 256 rows (of X) by one
// pair of CTAs, 128 rows each. B (fp16) stays in shared memory as the first
// operand of B X. X goes by in blocks of 128 columns, read once and written once
// per iteration through the L2 cache; the block's new hi part, in shared memory
// on its way out, is at once the operand of its share of the next A = X X^T,
// which adds up in TMEM. Between two passes over X, A passes through shared
// memory for A A. So a matrix waits for nobody, and its 15 products cost two
// exchanges with the L2 cache per iteration. (In k_ns, tiles of such matrices
// spent most of their time waiting for one another: 64 matrices of 256 x 1024
// took 276 us there, 141 here.) With 256 rows a block takes 2.1 us an iteration,
// 1.5 of them its two products at the measured rate of large ones; with 64 rows
// 1.7, the products being as wide.
//
// Shared memory per CTA: four slots of 128 rows x 64 fp16 for A, or for the hi
// parts of two blocks; four for B; two blocks of X (64 columns of all rows); four
// slots of lo. TMEM: two accumulators of 128 columns (A A: both), one of 256 (A).
template <int kDst>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPanelThreads, 1)
k_panel(const __grid_constant__ MatrixArgs a, const __grid_constant__ ApplyArgs step) {
    constexpr bool kMuon = kDst == kDstParamF32 || kDst == kDstParamMixed;
    constexpr int kMathWarp = 4, kMathWarps = 16;
    constexpr int kRing = 1;  // matrices handed out ahead (46M parameters in ragged matrices: with two, 1357 us, with one 1315)
    constexpr uint32_t kEnd = 0xFFFFFFFFu;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t mat_full[kRing], mat_empty[kRing], mat_done;
    __shared__ __align__(8) uint64_t g0_full[4], g0_empty[4];       // X's slots of the first A
    __shared__ __align__(8) uint64_t x_full[2], x_empty[2], x_done;  // blocks of X; X of an iteration written
    __shared__ __align__(8) uint64_t lo_full[4], lo_empty[4];
    __shared__ __align__(8) uint64_t hi_full[4], hi_out[4], hi_empty[4];  // for products, for stores; free
    __shared__ __align__(8) uint64_t d_full[2], d_empty[2], a_full, aa_full, a_ready, b_ready, drain_bar;
    __shared__ __align__(16) uint4 s_mat[kRing];  // stack, matrix of the stack, m, n
    __shared__ uint32_t s_tmem;
    __shared__ int s_err, s_drain_err;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if constexpr (kMuon) {
        if (a.step->skip) return;
    }
    const uint32_t rank = blockIdx.x & 1u;  // 0 leads the pair
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t a_slots = smem, b_slots = smem + 4 * kNsSlotBytes;
    const uint32_t x_blocks = b_slots + 4 * kNsSlotBytes, lo_slots = x_blocks + 2 * kPanelBlockBytes;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kRing; ++i) {
            mbar_init(smem_u32(&mat_full[i]), 1);
            // copies in, products, copies out, arithmetic and the other CTA's word here; copies and
            // arithmetic there
            mbar_init(smem_u32(&mat_empty[i]), (rank == 0 ? 4 : 2) + kMathWarps);
            if (rank == 1) mbar_expect_tx(smem_u32(&mat_full[i]), sizeof(uint4));
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&x_full[i]), 1);
            mbar_init(smem_u32(&x_empty[i]), 1);
            mbar_init(smem_u32(&d_full[i]), 1);
            mbar_init(smem_u32(&d_empty[i]), 2 * kMathWarps);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_u32(&g0_full[i]), 1);
            mbar_init(smem_u32(&g0_empty[i]), 1);
            mbar_init(smem_u32(&lo_full[i]), 1);
            mbar_init(smem_u32(&lo_empty[i]), 1);
            mbar_init(smem_u32(&hi_full[i]), kMathWarps);      // both CTAs' eight warps of a chunk
            mbar_init(smem_u32(&hi_out[i]), kMathWarps / 2);
            mbar_init(smem_u32(&hi_empty[i]), 2);              // its product, its store
        }
        mbar_init(smem_u32(&mat_done), kMathWarps);
        mbar_init(smem_u32(&x_done), 2);
        mbar_init(smem_u32(&a_full), 1);
        mbar_init(smem_u32(&aa_full), 1);
        mbar_init(smem_u32(&a_ready), 2 * kMathWarps);
        mbar_init(smem_u32(&b_ready), 2 * kMathWarps);
        mbar_init(smem_u32(&drain_bar), 1);
        s_err = s_drain_err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                         smem_u32(&s_tmem))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t steps = static_cast<uint32_t>(a.steps);
    auto release_mat = [&](uint32_t slot) { mbar_arrive(smem_u32(&mat_empty[slot])); };
    auto lead = [&](uint64_t* bar) { return map_to(smem_u32(bar), 0); };
    // Copies of this CTA's that landed or not when something failed are waited for by this barrier's
    // owner below; nothing else may touch shared memory after that.

    if (warp == 0) {
        // ---- copies in ----
        fence_async_proxy();  // (X of the kernel before)
        uint32_t g0_phase = 0xF, x_phase = 3, lo_phase = 0xF, done_phase = 0;
        const uint32_t lead_g0 = uniform(lead(&g0_full[0])), lead_x = uniform(lead(&x_full[0]));
        bool ok = true;
        for (uint32_t q = 0; ok; ++q) {
            const uint32_t slot = q % kRing;
            ok = warp_wait(smem_u32(&mat_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const uint32_t stack = uniform(s_mat[slot].x), index = uniform(s_mat[slot].y);
            const uint32_t m = uniform(s_mat[slot].z), n = uniform(s_mat[slot].w);
            __syncwarp();
            if (lane == 0) {
                if (rank == 1) mbar_expect_tx(smem_u32(&mat_full[slot]), sizeof(uint4));
                release_mat(slot);
            }
            if (stack == kEnd) break;
            const CUtensorMap* maps = a.maps + static_cast<uint64_t>(stack) * kMapsPerStack;
            const uint32_t kb = (m + 63) / 64, chunks = (n + 63) / 64, blocks = (chunks + 1) / 2;
            // the matrix before is done with the slots
            if (q > 0) ok = warp_wait(smem_u32(&mat_done), (q + 1) & 1, &s_err);
            for (uint32_t c = 0; c < chunks && ok; ++c) {
                const uint32_t b = c & 3;
                ok = warp_wait(smem_u32(&g0_empty[b]), g0_phase >> b & 1, &s_err);
                if (!ok) break;
                g0_phase ^= 1u << b;
                if (elect_one()) {
                    if (rank == 0) mbar_expect_tx(smem_u32(&g0_full[b]), 2 * kNsSlotBytes);
                    tma_load_pair(a_slots + b * kNsSlotBytes, maps + kMapX0, lead_g0 + b * 8, c * 64, rank * kNsRows, index);
                }
                __syncwarp();
            }
            for (uint32_t it = 0; it < steps && ok; ++it) {
                const CUtensorMap* x = maps + (it & 1 ? kMapX1 : kMapX0);
                if (it > 0) {
                    // both CTAs' stores of the iteration before have landed
                    ok = warp_wait_acquire(smem_u32(&x_done), done_phase, &s_err);
                    done_phase ^= 1;
                    fence_async_proxy();
                }
                for (uint32_t j = 0; j < blocks && ok; ++j) {
                    const uint32_t b = j & 1;
                    ok = warp_wait(smem_u32(&x_empty[b]), x_phase >> b & 1, &s_err);
                    if (!ok) break;
                    x_phase ^= 1u << b;
                    if (elect_one()) {
                        if (rank == 0) mbar_expect_tx(smem_u32(&x_full[b]), 2 * kb * kNsBoxBytes);
                        for (uint32_t k = 0; k < kb; ++k)
                            tma_load_pair(x_blocks + b * kPanelBlockBytes + k * kNsBoxBytes, x + kMapN + kMap64,
                                          lead_x + b * 8, 0, k * 64, 2 * j + rank, index);
                    }
                    __syncwarp();
                    for (uint32_t g = 0; g < 2 && 2 * j + g < chunks && ok; ++g) {
                        const uint32_t l = 2 * b + g;
                        ok = warp_wait(smem_u32(&lo_empty[l]), lo_phase >> l & 1, &s_err);
                        if (!ok) break;
                        lo_phase ^= 1u << l;
                        if (elect_one()) {
                            mbar_expect_tx(smem_u32(&lo_full[l]), kLoBytes);
                            tma_load(lo_slots + l * kLoBytes, x + kMapLo, smem_u32(&lo_full[l]), (2 * j + g) * 64,
                                     rank * kNsRows, index);
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (*reinterpret_cast<volatile int*>(&s_err)) {
            // copies in flight land before the CTA may end
            for (uint32_t i = 0; i < 4; ++i) {
                if (rank == 0) bar_wait(smem_u32(&g0_full[i]), g0_phase >> i & 1, &s_drain_err);
                bar_wait(smem_u32(&lo_full[i]), lo_phase >> i & 1, &s_drain_err);
            }
            for (uint32_t i = 0; i < 2 && rank == 0; ++i) bar_wait(smem_u32(&x_full[i]), x_phase >> i & 1, &s_drain_err);
        }
        __syncwarp();
    } else if (warp == 1) {
        // ---- products, issued by the leader ----
        uint32_t g0_phase = 0, x_phase = 0, d_phase = 3, hi_phase = 0, a_phase = 0;
        bool ok = true;
        const uint32_t acc = uniform(tmem), gram = acc + 256;
        // one product of 64 columns' depth
        auto product = [&](uint32_t d, uint32_t first, uint32_t second, bool mn, uint32_t n, bool fresh) {
            const uint64_t da = operand_desc(first, 16), db = operand_desc(second, mn ? kNsBoxBytes : 16);
            const uint32_t db_k = mn ? 2048 >> 4 : 32 >> 4;
            const uint32_t idesc = instr_desc(n, mn);
            mma_f16(d, da, db, idesc, !fresh);
#pragma unroll
            for (uint32_t k = 1; k < 4; ++k) mma_f16(d, da + k * 2, db + k * db_k, idesc, true);
        };
        for (uint32_t q = 0; rank == 0 && ok; ++q) {
            const uint32_t slot = q % kRing;
            ok = warp_wait(smem_u32(&mat_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const uint32_t stack = uniform(s_mat[slot].x), m = uniform(s_mat[slot].z), n = uniform(s_mat[slot].w);
            __syncwarp();
            if (lane == 0) release_mat(slot);
            if (stack == kEnd) break;
            const uint32_t kb = (m + 63) / 64, chunks = (n + 63) / 64, blocks = (chunks + 1) / 2;
            for (uint32_t c = 0; c < chunks && ok; ++c) {
                const uint32_t b = c & 3, s = a_slots + b * kNsSlotBytes;
                ok = warp_wait(smem_u32(&g0_full[b]), g0_phase >> b & 1, &s_err);
                if (!ok) break;
                g0_phase ^= 1u << b;
                tc_fence_after();
                if (elect_one()) {
                    product(gram, s, s, false, 256, c == 0);
                    mma_commit(smem_u32(&g0_empty[b]));
                    if (c + 1 == chunks) mma_commit(smem_u32(&a_full));
                }
                __syncwarp();
            }
            for (uint32_t it = 0; it < steps && ok; ++it) {
                ok = warp_wait(smem_u32(&a_ready), a_phase, &s_err);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    for (uint32_t k = 0; k < kb; ++k)
                        product(acc, a_slots + k * kNsSlotBytes, a_slots + k * kNsSlotBytes, false, 256, k == 0);
                    mma_commit(smem_u32(&aa_full));
                }
                __syncwarp();
                ok = warp_wait(smem_u32(&b_ready), a_phase, &s_err);
                if (!ok) break;
                a_phase ^= 1;
                // the next A takes block j - 1 while block j's product is under way
                for (uint32_t j = 0; j <= blocks && ok; ++j) {
                    const uint32_t b = j & 1;
                    if (j < blocks) {
                        ok = warp_wait(smem_u32(&x_full[b]), x_phase >> b & 1, &s_err) &&
                             warp_wait(smem_u32(&d_empty[b]), d_phase >> b & 1, &s_err);
                        if (!ok) break;
                        x_phase ^= 1u << b;
                        d_phase ^= 1u << b;
                        tc_fence_after();
                        if (elect_one()) {
                            for (uint32_t k = 0; k < kb; ++k)
                                product(acc + b * 128, b_slots + k * kNsSlotBytes,
                                        x_blocks + b * kPanelBlockBytes + k * kNsBoxBytes, true, 128, k == 0);
                            mma_commit(smem_u32(&x_empty[b]));
                            mma_commit(smem_u32(&d_full[b]));
                        }
                        __syncwarp();
                    }
                    if (j == 0 || it + 1 == steps) continue;
                    for (uint32_t g = 0; g < 2 && 2 * (j - 1) + g < chunks && ok; ++g) {
                        const uint32_t h = 2 * ((j - 1) & 1) + g, s = a_slots + h * kNsSlotBytes;
                        ok = warp_wait(smem_u32(&hi_full[h]), hi_phase >> h & 1, &s_err);
                        if (!ok) break;
                        hi_phase ^= 1u << h;
                        tc_fence_after();
                        if (elect_one()) {
                            product(gram, s, s, false, 256, j == 1 && g == 0);
                            mma_commit(smem_u32(&hi_empty[h]));
                            if (j == blocks && (g == 1 || 2 * (j - 1) + 1 == chunks)) mma_commit(smem_u32(&a_full));
                        }
                        __syncwarp();
                    }
                }
            }
        }
        if (*reinterpret_cast<volatile int*>(&s_err) && rank == 0) {
            if (elect_one()) mma_commit(smem_u32(&drain_bar));
            bar_wait(smem_u32(&drain_bar), 0, &s_drain_err);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---- the leader hands out matrices, to both CTAs ----
        if (rank == 0 && lane == 0) {
            for (uint32_t q = 0;; ++q) {
                const uint32_t slot = q % kRing;
                if (q >= kRing && !bar_wait_acquire(smem_u32(&mat_empty[slot]), (q / kRing + 1) & 1, &s_err)) break;
                const uint32_t claim = atomicAdd(a.next + 1, 1u);
                uint4 w = make_uint4(kEnd, 0, 0, 0);
                if (claim < a.n_panels) {
                    const uint2 p = a.panels[claim];
                    const NsStack& s = a.stacks[p.x];
                    w = make_uint4(p.x, p.y, s.m, s.n);
                }
                st_async_v4(map_to(smem_u32(&s_mat[slot]), 1), w, map_to(smem_u32(&mat_full[slot]), 1));
                s_mat[slot] = w;
                mbar_arrive(smem_u32(&mat_full[slot]));
                if (w.x == kEnd) break;
            }
        } else if (rank == 1 && lane == 0) {
            // (as in k_ns: this CTA's reads of a slot come before the leader's next write into it)
            for (uint32_t q = 0;; ++q) {
                const uint32_t slot = q % kRing;
                if (!bar_wait(smem_u32(&mat_full[slot]), (q / kRing) & 1, &s_err)) break;
                if (s_mat[slot].x == kEnd) break;
                if (!bar_wait(smem_u32(&mat_empty[slot]), (q / kRing) & 1, &s_err)) break;
                mbar_arrive_release(map_to(smem_u32(&mat_empty[slot]), 0));
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        // ---- copies out ----
        uint32_t out_phase = 0;
        bool ok = true;
        for (uint32_t q = 0; ok; ++q) {
            const uint32_t slot = q % kRing;
            ok = warp_wait(smem_u32(&mat_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const uint4 w = s_mat[slot];
            __syncwarp();
            if (lane == 0) release_mat(slot);
            if (w.x == kEnd) break;
            const CUtensorMap* maps = a.maps + static_cast<uint64_t>(w.x) * kMapsPerStack;
            const bool some = rank * kNsRows < w.z;  // this CTA has rows
            const uint32_t chunks = (w.w + 63) / 64;
            for (uint32_t it = 0; it < steps && ok; ++it) {
                const CUtensorMap* x = maps + (it & 1 ? kMapX0 : kMapX1);
                for (uint32_t c = 0; c < chunks; ++c) {
                    const uint32_t h = c & 3;
                    ok = warp_wait(smem_u32(&hi_out[h]), out_phase >> h & 1, &s_err);
                    if (!ok) break;
                    out_phase ^= 1u << h;
                    if (elect_one()) {
                        if (it + 1 == steps) {  // (the result has left with the arithmetic)
                            mbar_arrive(smem_u32(&lo_empty[h]));
                        } else {
                            if (some) {
                                tma_store(x, a_slots + h * kNsSlotBytes, c * 64, rank * kNsRows, w.y);
                                tma_store(x + kMapLo, lo_slots + h * kLoBytes, c * 64, rank * kNsRows, w.y);
                            }
                            bulk_commit();
                            // a slot is free once its store has read it: the one before's has when
                            // this one's is on its way
                            if (c > 0) {
                                bulk_wait_read<1>();
                                mbar_arrive(smem_u32(&hi_empty[(h + 3) & 3]));
                                mbar_arrive(smem_u32(&lo_empty[(h + 3) & 3]));
                            }
                            if (c + 1 == chunks) {
                                bulk_wait_read<0>();
                                mbar_arrive(smem_u32(&hi_empty[h]));
                                mbar_arrive(smem_u32(&lo_empty[h]));
                                bulk_wait_all();  // all of X has landed
                                fence_async_proxy();
                                mbar_arrive_release(map_to(smem_u32(&x_done), 0));
                                mbar_arrive_release(map_to(smem_u32(&x_done), 1));
                            }
                        }
                    }
                    __syncwarp();
                }
            }
        }
        __syncwarp();
    } else {
        // ---- arithmetic: two groups of eight warps, each with every other 64 columns; a warp
        // has 32 rows of 32 of them ----
        const uint32_t quad = warp & 3, group = (warp - kMathWarp) >> 2 & 1, part = (warp - kMathWarp) >> 3;
        const uint32_t trow = quad * 32 + lane, row = rank * kNsRows + trow;
        const uint32_t lanes = tmem + ((quad * 32u) << 16);
        uint32_t a_phase = 0, d_phase = 0, lo_phase = 0, hi_phase = 0, hi_used = 0;
        bool ok = true;
        for (uint32_t q = 0; ok; ++q) {
            const uint32_t slot = q % kRing;
            ok = warp_wait(smem_u32(&mat_full[slot]), (q / kRing) & 1, &s_err);
            if (!ok) break;
            const uint4 w = s_mat[slot];
            __syncwarp();
            if (lane == 0) release_mat(slot);
            if (w.x == kEnd) break;
            const NsStack& s = a.stacks[w.x];
            const uint32_t m = w.z, n = w.w, kb = (m + 63) / 64, chunks = (n + 63) / 64, blocks = (chunks + 1) / 2;
            const NsHold* hold = a.hold + static_cast<uint64_t>(s.first + w.y) * steps;
            const bool transposed = s.transposed != 0;
            const Target target = target_of<kDst>(s, w.y, step, a.ema != 0);
            for (uint32_t it = 0; it < steps && ok; ++it) {
                const bool last = it + 1 == steps;
                const NsHold held = hold[it];
                // (B and the addend carry the next iteration's scale)
                const float regrade = last ? 1.0f : held.regrade;
                const float ca = a.coef[it][0] * regrade, cb = a.coef[it][1] * regrade, cc = a.coef[it][2] * regrade;
                // A, from its accumulator to shared memory (the slots' last blocks have left them)
                ok = warp_wait(smem_u32(&a_full), a_phase, &s_err);
                for (uint32_t h = 0; h < 4 && ok; ++h)
                    if (hi_used >> h & 1) ok = warp_wait(smem_u32(&hi_empty[h]), (hi_phase >> h & 1) ^ 1, &s_err);
                if (!ok) break;
                tc_fence_after();
                for (uint32_t c = group; c < kb; c += 2) {
                    float v[32];
                    __syncwarp();
                    tmem_ld32(lanes + 256 + c * 64 + part * 32, v);
                    const float f = kNsScaleA * held.inv * held.inv;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) h[e] = pack2(v[8 * j + 2 * e] * f, v[8 * j + 2 * e + 1] * f);
                        sts128(a_slots + c * kNsSlotBytes + slot_at(trow, part * 4 + j), make_uint4(h[0], h[1], h[2], h[3]));
                    }
                }
                fence_async_shared();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(lead(&a_ready));
                // B = a I + b A + c A A
                ok = warp_wait(smem_u32(&aa_full), a_phase, &s_err);
                if (!ok) break;
                a_phase ^= 1;
                tc_fence_after();
                for (uint32_t c = group; c < kb; c += 2) {
                    float v[32];
                    __syncwarp();
                    tmem_ld32(lanes + c * 64 + part * 32, v);
                    const float f2 = cc / (kNsScaleA * kNsScaleA), f1 = cb / kNsScaleA;
                    const uint32_t diag = row - c * 64 - part * 32;  // (no match: no column)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 p = lds128(a_slots + c * kNsSlotBytes + slot_at(trow, part * 4 + j));
                        const __half2* ah = reinterpret_cast<const __half2*>(&p);
                        uint32_t h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float2 x = __half22float2(ah[e]);
                            const int i = 8 * j + 2 * e;
                            float y0 = __fmaf_rn(f1, x.x, f2 * v[i]), y1 = __fmaf_rn(f1, x.y, f2 * v[i + 1]);
                            y0 += diag == static_cast<uint32_t>(i) ? ca : 0.0f;
                            y1 += diag == static_cast<uint32_t>(i + 1) ? ca : 0.0f;
                            h[e] = pack2(y0, y1);
                        }
                        sts128(b_slots + c * kNsSlotBytes + slot_at(trow, part * 4 + j), make_uint4(h[0], h[1], h[2], h[3]));
                    }
                }
                fence_async_shared();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_pair(lead(&b_ready));
                // X = B X, block by block
                for (uint32_t j = 0; j < blocks && ok; ++j) {
                    const uint32_t b = j & 1, c = 2 * j + group, h = 2 * b + group;
                    ok = warp_wait(smem_u32(&d_full[b]), d_phase >> b & 1, &s_err);
                    if (!ok) break;
                    d_phase ^= 1u << b;
                    tc_fence_after();
                    float v[32];
                    if (c < chunks) {
                        __syncwarp();
                        tmem_ld32(lanes + b * 128 + group * 64 + part * 32, v);
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_pair(lead(&d_empty[b]));
                    if (c >= chunks) continue;
                    ok = warp_wait(smem_u32(&lo_full[h]), lo_phase >> h & 1, &s_err);
                    if (!ok) break;
                    lo_phase ^= 1u << h;
                    const uint32_t lo = lo_slots + h * kLoBytes;
#pragma unroll
                    for (int k = 0; k < 2; ++k) add_lo8(lo, trow, part * 2 + k, ca / kLoScale, v + 16 * k);
                    if (last) {
                        // through shared memory as floats, the warp's own 32 rows, so that the result
                        // is written along the rows of the caller's matrix (in the group's two slots,
                        // which nothing else uses by now)
                        const float f = held.inv;
                        float* fs = reinterpret_cast<float*>(
                            smem_raw + (a_slots - smem_u32(smem_raw) + group * 2 * kNsSlotBytes));
                        __syncwarp();
#pragma unroll
                        for (int k = 0; k < 32; ++k) fs[float_at(trow, part * 32 + k)] = v[k] * f;
                        __syncwarp();
                        put_transposed_or_not<kDst>(step, target, a.ema != 0, fs + float_at(quad * 32, part * 32),
                                                    transposed, lane, rank * kNsRows + quad * 32, c * 64 + part * 32,
                                                    m, n);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(smem_u32(&hi_out[h]));
                        continue;
                    }
                    // hi, for its store and for the next A; lo in place of the old one
                    if (hi_used >> h & 1) ok = warp_wait(smem_u32(&hi_empty[h]), (hi_phase >> h & 1) ^ 1, &s_err);
                    if (!ok) break;
                    hi_used |= 1u << h;
                    hi_phase ^= 1u << h;
                    uint32_t lo_word[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t hw[4];
                        lo_word[2 * k] = split4(v + 8 * k, hw[0], hw[1]);
                        lo_word[2 * k + 1] = split4(v + 8 * k + 4, hw[2], hw[3]);
                        sts128(a_slots + h * kNsSlotBytes + slot_at(trow, part * 4 + k), make_uint4(hw[0], hw[1], hw[2], hw[3]));
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        sts128(lo + lo8_at(trow, part * 2 + k), make_uint4(lo_word[4 * k], lo_word[4 * k + 1], lo_word[4 * k + 2],
                                                                lo_word[4 * k + 3]));
                    fence_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_pair(lead(&hi_full[h]));
                        mbar_arrive(smem_u32(&hi_out[h]));
                    }
                }
            }
            // the slots are the next matrix's
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&mat_done));
        }
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && (s_err | s_drain_err)) {
        atomicOr(a.err, 1);
        atomicOr(a.gave_up, 1u);
        // the other CTA's copies may still be landing here, or counting on barriers here
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 2000000ull) {}
    }
    __syncthreads();
    cluster_sync();  // the other CTA may use this one's shared memory until it is done too
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ------------------------------------------------------ matrices of few rows ---
// k_few: the whole iteration of a matrix with at most 8 rows (of X) by one CTA. Products of 11
// bits are off by up to 1 % there: the roundings of A's and B's few elements do not average out
// (2 x 3: 1.0 %, 4 x 4 0.6 %, 1 x 1 0.5 %). Every X of the iteration is a polynomial P of the
// first A times the first X, and neither P nor A has more than 8 x 8 elements. So one pass
// over the first X (22 bits, from the L2 cache) sums A, the steps are P <- B P and A <- B A B in
// shared memory, and a second pass writes P X. All of it in 64 bits. A <- B A B multiplies
// the roundings in small directions of A by up to a^2 a step: where they may have grown by more
// than 2^27, A is summed again from P X (with the usual coefficients after the eighth step). The
// call takes 28 us for 8 x 4096 and 94 us for 200 of those, 12 us for 8 x 8 (as tiles and pairs'
// matrices, in products of 11 bits, 153, 833 and 30).
constexpr int kFewMost = static_cast<int>(kFewRows);
constexpr double kFewGrowth = 0x1p27;
struct FewShared {
    double p[kFewMost][kFewMost], a[kFewMost][kFewMost], b[kFewMost][kFewMost], t[kFewMost][kFewMost];
    double part[kThreads / 32][kFewMost * (kFewMost + 1) / 2];
};

// One element of the result at `at`, or Muon's update of one weight.
template <int kDst>
__device__ __forceinline__ void put_one(const ApplyArgs& step, const Target& s, bool ema, uint64_t at, float o) {
    if constexpr (kDst == kDstBf16) {
        static_cast<uint16_t*>(s.dst)[at] = f32_to_bf16_rn(o);
    } else {
        static_assert(kDst == kDstParamMixed, "results that take one product");
        float w = s.master[at];
        if (s.lr_wd != 0.0f) w = __fsub_rn(w, __fmul_rn(s.lr_wd, w));
        w = __fsub_rn(w, __fmul_rn(s.lr_s, o));
        s.master[at] = w;
        static_cast<uint16_t*>(s.dst)[at] = f32_to_bf16_rn(w);
        if (ema) s.ema[at] = __fadd_rn(__fmul_rn(step.ema_decay, s.ema[at]), __fmul_rn(step.ema_omd, w));
    }
}

// (kRows: m, or the next power of two; rows that X does not have are zeros)
template <int kDst, int kRows>
__device__ __forceinline__ void few_rows(const MatrixArgs& a, const ApplyArgs& step, const NsStack& s, uint32_t index,
                                         FewShared& sh) {
    constexpr int kPairs = kRows * (kRows + 1) / 2;
    using Square = double[kFewMost][kFewMost];
    const uint32_t m = s.m, n = s.n, ldx = s.ldx;
    const uint64_t base = static_cast<uint64_t>(index) * m * ldx;
    const __half *hi = s.x[0] + base, *lo = s.xl[0] + base;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool mine = threadIdx.x < kRows * kRows;  // an element of P, A and B
    const int ti = threadIdx.x / kRows, tk = threadIdx.x % kRows;
    auto read = [&](uint32_t j, double (&x)[kRows]) {
#pragma unroll
        for (int k = 0; k < kRows; ++k) {
            const uint32_t at = k * ldx + j;
            x[k] = k < m ? static_cast<double>(__half2float(hi[at]) + __half2float(lo[at])) : 0.0;
        }
    };
    auto times_p = [&](const double (&x)[kRows], double (&y)[kRows]) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            y[i] = 0.0;
#pragma unroll
            for (int k = 0; k < kRows; ++k) y[i] = fma(sh.p[i][k], x[k], y[i]);
        }
    };
    // this thread's element of a product
    auto element = [&](const Square& p, const Square& q) {
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < kRows; ++k) v = fma(p[ti][k], q[k][tk], v);
        return v;
    };
    // A = f (P X)(P X)^T, or f X X^T, in a fixed order
    auto sum_a = [&](bool first, double f) {
        double sum[kPairs];
#pragma unroll
        for (int e = 0; e < kPairs; ++e) sum[e] = 0.0;
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
            double x[kRows];
            read(j, x);
            if (!first) {
                double y[kRows];
                times_p(x, y);
#pragma unroll
                for (int i = 0; i < kRows; ++i) x[i] = y[i];
            }
#pragma unroll
            for (int i = 0, e = 0; i < kRows; ++i)
#pragma unroll
                for (int k = 0; k <= i; ++k, ++e) sum[e] = fma(x[i], x[k], sum[e]);
        }
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
            sum[e] = warp_sum(sum[e]);
            if (lane == 0) sh.part[warp][e] = sum[e];
        }
        __syncthreads();
        if (mine) {
            const int i = ti > tk ? ti : tk, k = ti > tk ? tk : ti;
            double v = 0.0;
#pragma unroll
            for (int w = 0; w < kThreads / 32; ++w) v += sh.part[w][i * (i + 1) / 2 + k];
            sh.a[ti][tk] = f * v;
        }
    };
    const double one_over = a.hold[(static_cast<uint64_t>(s.first) + index) * a.steps].inv;
    if (mine) sh.p[ti][tk] = ti == tk ? one_over : 0.0;
    sum_a(true, one_over * one_over);
    __syncthreads();
    double growth = 1.0;
#pragma unroll 1
    for (int it = 0; it < a.steps; ++it) {
        const double ca = a.coef[it][0], cb = a.coef[it][1], cc = a.coef[it][2];
        if (mine) sh.b[ti][tk] = cb * sh.a[ti][tk] + cc * element(sh.a, sh.a) + (ti == tk ? ca : 0.0);
        __syncthreads();
        const double p = mine ? element(sh.b, sh.p) : 0.0;
        if (mine) sh.t[ti][tk] = element(sh.b, sh.a);
        __syncthreads();
        if (mine) sh.p[ti][tk] = p;
        growth *= ca * ca > 1.0 ? ca * ca : 1.0;
        if (growth <= kFewGrowth) {
            if (mine) sh.a[ti][tk] = element(sh.t, sh.b);
        } else if (it + 1 < a.steps) {
            __syncthreads();
            sum_a(false, 1.0);
            growth = 1.0;
        }
        __syncthreads();
    }
    const Target target = target_of<kDst>(s, index, step, a.ema != 0);
    const uint64_t across = s.transposed ? 1 : target.pitch, along = s.transposed ? target.pitch : 1;
#pragma unroll 1
    for (uint32_t j = threadIdx.x; j < n; j += kThreads) {
        double x[kRows], y[kRows];
        read(j, x);
        times_p(x, y);
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            if (i < m) put_one<kDst>(step, target, a.ema != 0, target.base + i * across + j * along, static_cast<float>(y[i]));
    }
    __syncthreads();  // (the next matrix writes P)
}

template <int kDst>
__global__ void __launch_bounds__(kThreads, 2)
k_few(const __grid_constant__ MatrixArgs a, const __grid_constant__ ApplyArgs step) {
    __shared__ FewShared sh;
    pdl_wait();
    pdl_trigger();
    if constexpr (kDst == kDstParamMixed) {
        if (a.step->skip) return;
    }
    for (uint32_t q = blockIdx.x; q < a.n_few; q += gridDim.x) {
        const uint2 f = a.few[q];
        const NsStack& s = a.stacks[f.x];
        if (s.m == 1) few_rows<kDst, 1>(a, step, s, f.y, sh);
        else if (s.m == 2) few_rows<kDst, 2>(a, step, s, f.y, sh);
        else if (s.m <= 4) few_rows<kDst, 4>(a, step, s, f.y, sh);
        else few_rows<kDst, 8>(a, step, s, f.y, sh);
    }
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
    const uint64_t pairs = static_cast<uint64_t>(sms / 2);
    cudaError_t e = cudaSuccess;
    if (a.n_tasks)
        e = launch_pdl(k_ns<kDst>, dim3(2 * static_cast<unsigned>(std::min<uint64_t>(a.n_tasks, pairs))),
                       dim3(kNsThreads), kNsSmemBytes, stream, a, step);
    if constexpr (kOneProduct<kDst>) {
        if (e == cudaSuccess && a.n_panels)
            e = launch_pdl(k_panel<kDst>, dim3(2 * static_cast<unsigned>(std::min<uint64_t>(a.n_panels, pairs))),
                           dim3(kPanelThreads), kPanelSmemBytes, stream, a, step);
        if (e == cudaSuccess && a.n_few)
            e = launch_pdl(k_few<kDst>, dim3(static_cast<unsigned>(std::min<uint64_t>(a.n_few, 2ull * sms))),
                           dim3(kThreads), 0, stream, a, step);
    }
    return e;
}

}  // namespace

cudaError_t prepare_matrix_kernels() {
    const std::pair<const void*, size_t> fns[] = {
        {reinterpret_cast<const void*>(k_ns<kDstF32>), kNsSmemBytes},
        {reinterpret_cast<const void*>(k_ns<kDstBf16>), kNsSmemBytes},
        {reinterpret_cast<const void*>(k_ns<kDstParamF32>), kNsSmemBytes},
        {reinterpret_cast<const void*>(k_ns<kDstParamMixed>), kNsSmemBytes},
        {reinterpret_cast<const void*>(k_panel<kDstBf16>), kPanelSmemBytes},
        {reinterpret_cast<const void*>(k_panel<kDstParamMixed>), kPanelSmemBytes}};
    for (const auto& f : fns) {
        const cudaError_t e = cudaFuncSetAttribute(f.first, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   static_cast<int>(f.second));
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
    if (e != cudaSuccess) return e;
    switch (dest) {
        case kDstF32: return launch_ns<kDstF32>(a, st, sms, stream);
        case kDstBf16: return launch_ns<kDstBf16>(a, st, sms, stream);
        case kDstParamF32: return launch_ns<kDstParamF32>(a, st, sms, stream);
        default: return launch_ns<kDstParamMixed>(a, st, sms, stream);
    }
}

}  // namespace soarb
