// Device helpers shared by every optimizer's kernels: the deterministic block
// sum, and the step's decision and commit on the control block.
#pragma once

#include <cstdint>

#include "optim_kernels.cuh"

namespace soarb {
namespace {

// -------------------------------------------------------------- reductions --

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// Deterministic block sum (fixed shuffle pattern, fixed warp order).
__device__ __forceinline__ double block_sum(double x, double* smem /* >= 32 */) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    x = warp_sum(x);
    if (lane == 0) smem[warp] = x;
    __syncthreads();
    double r = 0.0;
    if (warp == 0) {
        r = lane < (kThreads / 32) ? smem[lane] : 0.0;
        r = warp_sum(r);
    }
    __syncthreads();
    return r;  // valid in thread 0
}

// Per-step values derived on the device from the control block. The
// host-known coefficients stay in the launch arguments (kernel parameter
// space), which keeps them out of the register file of the streaming loop.
struct StepCoeffs {
    float inv;        // 1 / loss scale
    float coef;       // clip coefficient (1: no clip)
    float step_size;  // lr / bias_correction1 (AdamW)
    float sqrt_bc2;   // (AdamW)
    int has_buf;      // SGD: momentum buffers hold a previous step (sgd.cpp:75-80)
};

// The step's decision, taken by one thread of every CTA from the same bits:
// skip (a failed peer sync, or inf/NaN with the scaler on), the pre-clip norm
// from the rank-ordered fp64 partial sums, the clip coefficient and the bias
// corrections of the step count the step will have. Counters are only read
// here and only written by the last CTA (commit_step).
struct StepDecision {
    StepCoeffs k;
    uint64_t t;
    float norm;
    int skip;
    int found;
};

__device__ __forceinline__ StepDecision decide_step(const ApplyArgs& a, const Ctl* ctl) {
    StepDecision d;
    d.skip = 0;
    d.found = 0;
    d.norm = 0.0f;
    float coef = a.pending_coef;
    if (a.skip_if && *a.skip_if) {
        d.skip = 1;  // a peer failed to synchronise: no update (the error flag tells)
    } else if (a.n_parts > 0) {
        double s = 0.0;
        for (int p = 0; p < a.n_parts; ++p) s += a.parts[p];
        d.found = !isfinite(s);
        d.norm = __double2float_rn(__dsqrt_rn(s));  // adamw.cpp:42
        if (a.use_scaler && d.found) d.skip = 1;
        // adamw.cpp:43-44: no eps, no min(1, .)
        if (a.max_norm > 0.0f && d.norm > a.max_norm && d.norm > 1e-6f)
            coef = __fdiv_rn(a.max_norm, d.norm);
    }
    d.t = ctl->t + (d.skip ? 0u : 1u);
    const uint64_t ti = d.t < a.bc_len ? d.t : static_cast<uint64_t>(a.bc_len - 1);
    const float2 bc = a.bc[ti];
    d.k.inv = a.use_scaler ? __fdiv_rn(1.0f, ctl->scale) : 1.0f;
    d.k.coef = coef;
    d.k.step_size = __fdiv_rn(a.lr, bc.x);  // adamw.cpp:71
    d.k.sqrt_bc2 = bc.y;
    d.k.has_buf = ctl->t > 0;  // applied steps so far (skipped steps never fill buffers)
    return d;
}

// Called by thread 0 of every CTA once the CTA is done: the last CTA to
// arrive (every CTA has read the counters by then) commits the step count,
// the bookkeeping and the loss-scaler update, and resets the tickets.
__device__ __forceinline__ void commit_step(Ctl* ctl, const ApplyArgs& a, const StepDecision& d) {
    __threadfence();
    const unsigned prev = atomicAdd(&ctl->ticket_apply, 1u);
    if (prev != gridDim.x - 1) return;
    ctl->t = d.t;
    ctl->last_norm = d.norm;
    ctl->last_found_inf = d.found;
    ctl->last_clip_coef = d.skip ? 1.0f : d.k.coef;
    ctl->last_lr = a.lr;
    if (d.skip) ctl->skipped += 1u;
    if (a.use_scaler) {
        if (d.skip) {
            ctl->scale = __fmul_rn(ctl->scale, a.backoff);
            ctl->tracker = 0;
        } else {
            const int32_t tr = ctl->tracker + 1;
            if (tr == a.interval) {
                ctl->scale = __fmul_rn(ctl->scale, a.growth);
                ctl->tracker = 0;
            } else {
                ctl->tracker = tr;
            }
        }
    }
    ctl->grab = 0u;  // every CTA has stopped grabbing
    ctl->ticket_apply = 0u;
}

}  // namespace
}  // namespace soarb
