// The C++ classes over the matrix operators (include/soar_optim.hpp):
// Orthogonalizer and Muon against the definition in 64 bits on the host, a
// Muon optimizer that is moved between its steps, and a refusal as an exception.
// Exit code 0 = pass. No assert(): the checks stay on in release builds.
#include <cmath>
#include <cstdio>
#include <memory>
#include <stdexcept>
#include <string>
#include <vector>

#include <cuda_runtime.h>

#include "soar_optim.hpp"

namespace {

int g_failures = 0;
#define CHECK(cond, ...)                                      \
    do {                                                      \
        if (!(cond)) {                                        \
            std::printf("FAIL %s:%d: ", __FILE__, __LINE__);  \
            std::printf(__VA_ARGS__);                         \
            std::printf("\n");                                \
            ++g_failures;                                     \
        }                                                     \
    } while (0)

class DevTensor;
using TensorPtr = std::shared_ptr<DevTensor>;
class DevTensor {
public:
    explicit DevTensor(const std::vector<float>& v) : n_(v.size()) {
        cudaMalloc(&d_, n_ * sizeof(float));
        cudaMemcpy(d_, v.data(), n_ * sizeof(float), cudaMemcpyHostToDevice);
    }
    ~DevTensor() { cudaFree(d_); }
    DevTensor(const DevTensor&) = delete;
    DevTensor& operator=(const DevTensor&) = delete;
    size_t numel() const noexcept { return n_; }
    float* cuda_data() noexcept { return d_; }
    TensorPtr grad() const noexcept { return grad_; }
    void set_grad(TensorPtr g) { grad_ = std::move(g); }
    std::vector<float> host() const {
        std::vector<float> v(n_);
        cudaDeviceSynchronize();
        cudaMemcpy(v.data(), d_, n_ * sizeof(float), cudaMemcpyDeviceToHost);
        return v;
    }

private:
    float* d_{nullptr};
    size_t n_;
    TensorPtr grad_;
};

using Mat = std::vector<double>;

// rows <= cols
Mat newton_schulz(const Mat& g, int rows, int cols) {
    double sum = 0;
    for (double v : g) sum += v * v;
    Mat x(g);
    for (double& v : x) v /= std::sqrt(sum) + 1e-7;
    for (int it = 0; it < 5; ++it) {
        Mat a(rows * rows), b(rows * rows), y(rows * cols);
        for (int i = 0; i < rows; ++i)
            for (int j = 0; j < rows; ++j)
                for (int k = 0; k < cols; ++k) a[i * rows + j] += x[i * cols + k] * x[j * cols + k];
        for (int i = 0; i < rows; ++i)
            for (int j = 0; j < rows; ++j) {
                double t = 0;
                for (int k = 0; k < rows; ++k) t += a[i * rows + k] * a[k * rows + j];
                b[i * rows + j] = -4.7750 * a[i * rows + j] + 2.0315 * t + (i == j ? 3.4445 : 0.0);
            }
        for (int i = 0; i < rows; ++i)
            for (int k = 0; k < rows; ++k)
                for (int j = 0; j < cols; ++j) y[i * cols + j] += b[i * rows + k] * x[k * cols + j];
        x = y;
    }
    return x;
}

std::vector<float> noise(size_t n, uint32_t seed, float rms) {
    std::vector<float> v(n);
    for (float& x : v) {
        seed = seed * 1664525u + 1013904223u;
        x = rms * 3.4641f * (static_cast<float>(seed >> 8) / 16777216.0f - 0.5f);
    }
    return v;
}

double rel(const std::vector<float>& got, const Mat& want) {
    double d = 0, n = 0;
    for (size_t i = 0; i < got.size(); ++i) {
        d += (got[i] - want[i]) * (got[i] - want[i]);
        n += want[i] * want[i];
    }
    return std::sqrt(d / n);
}

// Operands of 22 bits and 32-bit arithmetic: five steps, of which each may add
// 44 roundings of 2^-24 and three of 2^-22 (the products' operands, times the
// terms' 14.6), and multiplies what it is given by at most 1.71: 19 times
// (44 x 2^-24 + 44 x 2^-22) < 2.6e-4.
constexpr double kTolerance = 2.6e-4;

constexpr int kRows = 48, kCols = 130;

void test_orthogonalizer() {
    const auto g = noise(kRows * kCols, 1, 0.01f);
    DevTensor src(g), dst(std::vector<float>(g.size()));
    soar_matrix_desc m{src.cuda_data(), dst.cuda_data(), 1, kRows, kCols, kCols, kRows * kCols, kCols, kRows * kCols};
    auto o = soar::optim::Orthogonalizer::default_options();
    o.dst_type = SOAR_DTYPE_FP32;
    soar::optim::Orthogonalizer first({m}, o);
    soar::optim::Orthogonalizer plan(std::move(first));
    plan.run();
    const double e = rel(dst.host(), newton_schulz(Mat(g.begin(), g.end()), kRows, kCols));
    std::printf("  orthogonalisation: off by %.3g\n", e);
    CHECK(e <= kTolerance, "orthogonalisation off by %.3g", e);
    CHECK(plan.error() == 0, "error word");
    bool thrown = false;
    try {
        m.src_row = kCols - 1;
        soar::optim::Orthogonalizer bad({m}, o);
    } catch (const std::runtime_error& x) {
        thrown = std::string(x.what()).find("overlap") != std::string::npos;
    }
    CHECK(thrown, "overlapping rows are refused");
}

void test_muon() {
    const auto w = noise(kRows * kCols, 2, 0.02f), g = noise(kRows * kCols, 3, 0.01f);
    auto p = std::make_shared<DevTensor>(w);
    p->set_grad(std::make_shared<DevTensor>(g));
    soar::optim::MuonOptions opt;
    opt.lr = 0.05f;
    opt.weight_decay = 0.1f;
    soar::optim::Muon muon(std::vector<TensorPtr>{p}, {{1, kRows, kCols}}, opt);
    muon.step();
    soar::optim::Muon moved(std::move(muon));
    moved.step();
    // two steps with one gradient: u is a multiple of it
    const Mat ns = newton_schulz(Mat(g.begin(), g.end()), kRows, kCols);
    const double lr = 0.05f, keep = 1.0 - lr * 0.1f;
    Mat want(w.begin(), w.end()), moves(w.size());
    for (int step = 0; step < 2; ++step)
        for (size_t i = 0; i < want.size(); ++i) want[i] = keep * want[i] - lr * ns[i];
    auto got = p->host();
    // compared as moves, so that the weights' own size does not hide an error; a
    // weight below 1/8 carries a rounding of at most 2^-28 a step
    for (size_t i = 0; i < want.size(); ++i) {
        moves[i] = want[i] - w[i];
        got[i] -= w[i];
    }
    const double e = rel(got, moves);
    std::printf("  Muon, two steps: moves off by %.3g\n", e);
    CHECK(e <= kTolerance, "moves off by %.3g", e);
    CHECK(moved.info().step == 2 && moved.info().error == 0, "bookkeeping");
    CHECK(moved.get_lr() == 0.05f, "lr");
    moved.zero_grad();
    for (float v : p->grad()->host()) CHECK(v == 0.0f, "zero_grad");
    bool thrown = false;
    try {
        soar::optim::Muon bad(std::vector<TensorPtr>{p}, {{1, kRows, kCols + 1}}, opt);
    } catch (const std::runtime_error&) {
        thrown = true;
    }
    CHECK(thrown, "a shape of another size is refused");
}

}  // namespace

int main() {
    test_orthogonalizer();
    test_muon();
    if (g_failures) {
        std::printf("%d FAILURES\n", g_failures);
        return 1;
    }
    std::printf("ALL MATRIX TESTS PASSED\n");
    return 0;
}
