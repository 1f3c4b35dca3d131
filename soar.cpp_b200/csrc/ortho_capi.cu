// C-ABI of the plain orthogonalisation (include/soar_optim.h, soar_ortho_*).
#include <cstring>
#include <exception>
#include <memory>
#include <string>
#include <unordered_set>
#include <vector>

#include <cuda_runtime.h>

#include "../../include/soar_optim.h"
#include "matrix_ops.cuh"

namespace soarb {
void record_error(const std::string& msg);  // optim_capi.cu
}  // namespace soarb

static_assert(SOAR_NS_MAX_STEPS == soarb::kNsMaxSteps, "one limit");

namespace {

int fail(const std::string& msg) {
    soarb::record_error(msg);
    return SOAR_ERROR;
}

struct DeviceGuard {
    int prev = -1;
    bool ok = false;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        ok = (prev == dev) || (cudaSetDevice(dev) == cudaSuccess);
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

struct Ortho {
    int device = 0;
    soarb::MatrixPlan* plan = nullptr;
};

// Whether the strides stay below 2^44 elements in all (so that no offset wraps).
bool within(uint64_t count, uint64_t rows, uint64_t row, uint64_t mat) {
    constexpr uint64_t kMost = 1ull << 43;
    return (rows <= 1 || row <= kMost / (rows - 1)) && (count <= 1 || mat <= kMost / (count - 1));
}

// Whether `count` matrices of `rows` rows of `cols` elements do not overlap.
bool apart(uint64_t count, uint64_t rows, uint64_t cols, uint64_t row, uint64_t mat) {
    if (rows > 1 && row < cols) return false;
    if (count <= 1) return true;
    const uint64_t matrix = (rows - 1) * row + cols;  // elements one matrix spans
    if (mat >= matrix) return true;
    // rows of all the matrices side by side
    return mat >= cols && (rows == 1 || row >= (count - 1) * mat + cols);
}

int create(const soar_matrix_desc* mats, int n, const soar_ortho_opts* opts, void** out) {
    if (!opts || !out || n < 0 || (n > 0 && !mats)) return fail("null argument");
    *out = nullptr;
    for (int32_t t : {opts->src_type, opts->dst_type})
        if (t != SOAR_DTYPE_FP32 && t != SOAR_DTYPE_BF16) return fail("unknown type");
    if (opts->steps < 1 || opts->steps > SOAR_NS_MAX_STEPS)
        return fail("steps must be 1 .. " + std::to_string(SOAR_NS_MAX_STEPS));
    if (!(opts->eps >= 0.0f)) return fail("eps must be >= 0");
    std::string bad;
    if (!soarb::matrix_coef_ok(opts->coef, opts->steps, &bad)) return fail(bad);
    const uint64_t sb = opts->src_type == SOAR_DTYPE_BF16 ? 2 : 4;
    const uint64_t db = opts->dst_type == SOAR_DTYPE_BF16 ? 2 : 4;
    std::vector<soarb::MatrixSpec> specs;
    std::unordered_set<const void*> taken;
    std::vector<soarb::MatrixSpan> spans;
    for (int i = 0; i < n; ++i) {
        const soar_matrix_desc& d = mats[i];
        const std::string at = "stack " + std::to_string(i) + ": ";
        std::string why;
        if (!soarb::matrix_shape_ok(d.count, d.rows, d.cols, &why)) return fail(at + why);
        if (!d.count || !d.rows || !d.cols) continue;
        if (!d.src || !d.dst) return fail(at + "null matrix");
        if (reinterpret_cast<uintptr_t>(d.src) % sb || reinterpret_cast<uintptr_t>(d.dst) % db)
            return fail(at + "pointer not aligned to its element size");
        for (uint64_t s : {d.src_row, d.src_mat, d.dst_row, d.dst_mat})
            if (s > (1ull << 40)) return fail(at + "a stride of more than 2^40 elements");
        if (!within(d.count, d.rows, d.src_row, d.src_mat) || !within(d.count, d.rows, d.dst_row, d.dst_mat))
            return fail(at + "strides over more than 2^44 elements");
        if (d.rows > 1 && d.src_row < d.cols) return fail(at + "source rows overlap");
        if (!apart(d.count, d.rows, d.cols, d.dst_row, d.dst_mat))
            return fail(at + "destination rows or matrices overlap");
        if (d.src == d.dst &&
            (sb != db || (d.rows > 1 && d.src_row != d.dst_row) || (d.count > 1 && d.src_mat != d.dst_mat)))
            return fail(at + "in place needs the same type and strides");
        if (!taken.insert(d.dst).second) return fail(at + "another stack has the same destination");
        soarb::MatrixSpec q;
        q.src = d.src;
        q.dst = d.dst;
        q.count = d.count;
        q.rows = d.rows;
        q.cols = d.cols;
        q.src_row = d.src_row;
        q.src_mat = d.src_mat;
        q.dst_row = d.dst_row;
        q.dst_mat = d.dst_mat;
        specs.push_back(q);
        spans.push_back({reinterpret_cast<uintptr_t>(d.dst), d.count, d.rows, d.cols * db, d.dst_row * db,
                         d.dst_mat * db, i});
    }
    int one = 0, other = 0;
    if (!soarb::matrix_spans_apart(std::move(spans), &one, &other))
        return fail("stacks " + std::to_string(one) + " and " + std::to_string(other) +
                    ": their destinations overlap");
    DeviceGuard g(opts->device);
    if (!g.ok) return fail("cannot select device " + std::to_string(opts->device));
    soarb::MatrixPlanOpts mo;
    mo.steps = opts->steps;
    std::memcpy(mo.coef, opts->coef, sizeof mo.coef);
    mo.eps = opts->eps;
    mo.source = opts->src_type == SOAR_DTYPE_BF16 ? soarb::kSrcBf16 : soarb::kSrcF32;
    mo.dest = opts->dst_type == SOAR_DTYPE_BF16 ? soarb::kDstBf16 : soarb::kDstF32;
    std::string why;
    auto o = std::make_unique<Ortho>();
    o->device = opts->device;
    o->plan = soarb::matrix_plan_create(specs.data(), static_cast<int>(specs.size()), mo, &why);
    if (!o->plan) return fail(why);
    *out = o.release();
    return SOAR_OK;
}

}  // namespace

extern "C" {

SOAR_API void soar_ortho_default_opts(soar_ortho_opts* out) {
    if (!out) return;
    std::memset(out, 0, sizeof *out);
    out->steps = 5;
    soarb::matrix_default_coef(out->coef);
    out->eps = 1e-7f;
    out->src_type = SOAR_DTYPE_FP32;
    out->dst_type = SOAR_DTYPE_BF16;
}

SOAR_API int soar_ortho_create(const soar_matrix_desc* mats, int n_mats, const soar_ortho_opts* opts,
                               void** out_handle) {
    try {
        return create(mats, n_mats, opts, out_handle);
    } catch (const std::exception& ex) {
        return fail(ex.what());
    } catch (...) {
        return fail("unknown exception");
    }
}

SOAR_API int soar_ortho_run(void* handle, void* stream) {
    if (!handle) return fail("null handle");
    Ortho& o = *static_cast<Ortho*>(handle);
    DeviceGuard g(o.device);
    if (!g.ok) return fail("cannot select the plan's device");
    const cudaError_t e = soarb::matrix_plan_run(o.plan, static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return fail(std::string("launch: ") + cudaGetErrorString(e));
    return SOAR_OK;
}

SOAR_API int soar_ortho_error(void* handle, int* out_error) {
    if (!handle || !out_error) return fail("null argument");
    Ortho& o = *static_cast<Ortho*>(handle);
    DeviceGuard g(o.device);
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess)
        e = cudaMemcpy(out_error, soarb::matrix_plan_error_word(o.plan), sizeof(int),
                       cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) return fail(std::string("error word: ") + cudaGetErrorString(e));
    return SOAR_OK;
}

SOAR_API int soar_ortho_destroy(void* handle) {
    if (!handle) return fail("null handle");
    Ortho* o = static_cast<Ortho*>(handle);
    {
        DeviceGuard g(o->device);
        cudaDeviceSynchronize();
        soarb::matrix_plan_destroy(o->plan);
    }
    delete o;
    return SOAR_OK;
}

}  // extern "C"
