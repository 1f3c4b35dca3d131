// Orthogonalisation of lists of matrices by Newton-Schulz products, and the
// Muon step built on it: structures shared by the kernels (matrix_kernels.cu)
// and the host code that plans them (matrix_plan.cu).
//
// For a matrix G with shorter side m and longer side n (transposed where it
// has more rows than columns, so that X is m x n):
//   X = G / (|G|_F + eps);  per iteration:  A = X X^T,  B = a I + b A + c A A,
//   X <- B X.
//
// Numbers: the products run on the tensor cores with fp16 operands and fp32
// sums. X is kept as hi + lo, hi an fp16 number of 11 bits, lo what is left of it
// in 3 more: with B = a I + b A + c A A, X becomes B hi + a lo, so that only
// products of small entries lose lo. A rounding of X's small singular directions would otherwise grow by
// a factor of a (3.4) per iteration: with X in hi alone, a matrix of a few
// strong directions over noise comes out 0.6 % to 7 % off (bf16 operands: 5 %
// to 60 %), with hi + lo 0.04 % to 0.25 %, about what the rounding of a bf16
// result costs (0.17 % rms); with fewer than 64 rows, whose roundings average out
// less, up to 0.5 %, and with at most 8 it would be up to 1 %: those are worked on in 64 bits. For fp32 results lo is an fp16 number too, of A and B as
// well, and every product is taken as hi hi + hi lo + lo hi (22 bits). The tensor
// cores round a sum towards zero at each addition, so there the large terms come
// last and half of them have an accumulator of their own (2048 x 2048: 4.6e-6 off
// instead of 1.1e-5).
//
// fp16's range is met by powers of two: X is held times sx = 2^floor(log2 sqrt(m n))
// (within 2^6 .. 2^12), which gives its elements an rms of about 1 at the start
// and of at most sqrt(m) at the end; A and B are held times 2^10, where their
// eigenvalues (at most about 1.5, and 4) stay below 2^12 and entries down to
// 2^-34 still count. Where eps is larger than |G|, X starts at |G| / (|G| + eps) and
// grows by a factor of a an iteration: it is then held by a larger power of two, before
// every iteration the one that a bound on its singular values allows
// (NsHold), so that its parts keep their bits (with sx alone, fp32 results for
// |G| = 1e-12 and eps = 1e-7 came out 0.35 % off, below 1e-16 as zeros).
#pragma once

#include <cstdint>
#include <string>
#include <vector>

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "optim_kernels.cuh"

namespace soarb {

constexpr int kNsMaxSteps = 16;
constexpr float kNsScaleA = 1024.0f;  // A and B are held times this

// Tile of a product: 256 rows by 256 or 128 columns (fewer at a matrix's edge), by a pair of CTAs (a
// cluster of two): each holds 128 rows of the first operand, half of the second
// one's columns and the accumulator of its 128 rows. A pair's tile needs two
// thirds of the operand traffic of two 128 x 256 tiles.
constexpr int kNsTileM = 256;
constexpr int kNsTileN = 256;
constexpr int kNsRows = 128;   // a CTA's share of the rows
constexpr int kNsTileK = 64;   // depth of one stage
constexpr int kNsStages = 4;
constexpr int kNsMathWarps = 8;  // two groups of four, each with every other chunk of 64 columns
// operand copies, products, hand-out, epilogue's copies in, and out (two), arithmetic
constexpr int kNsThreads = (6 + kNsMathWarps) * 32;
constexpr uint32_t kNsBoxBytes = 64 * 64 * 2;  // one TMA box: 64 rows of 64 fp16
constexpr uint32_t kNsStageBytes = 4 * kNsBoxBytes;
constexpr uint32_t kNsSlotBytes = 2 * kNsBoxBytes;  // epilogue: 128 rows of 64 fp16
constexpr uint32_t kLoBytes = 128 * 64;  // a slot of 128 rows of 64 bytes: of lo, or of 32 columns of A
constexpr int kNsGroups = 2;  // each with two such slots of what it adds, and two slots of what it makes
constexpr size_t kNsSmemBytes =
    static_cast<size_t>(kNsStages) * kNsStageBytes + kNsGroups * (2 * kLoBytes + 2 * kNsSlotBytes) + 1024;

// Where products take hi alone, X's lo is held in 8 bits (e5m2, times 2^8: 3 more
// bits of X). That leaves the errors stated above (16 bits: 0.03 % to 0.16 %), and
// lo is a quarter of what is read and written beside the products' operands.
constexpr float kLoScale = 256.0f;

// Matrices whose shorter side is at most this, and whose result takes one
// product, are worked on whole by one pair of CTAs (k_panel): A and B stay in
// shared memory, X streams through it once per iteration.
constexpr uint32_t kPanelSide = 256;
constexpr uint32_t kPanelAnyColumns = 1152;  // up to this longer side always, beyond it in long lists
constexpr int kPanelThreads = 640;  // copies in, products, hand-out, copies out, sixteen warps of arithmetic
constexpr uint32_t kPanelBlockBytes = 4 * 64 * 64 * 2;  // a CTA's 64 columns of X, 256 rows
constexpr size_t kPanelSmemBytes =
    8 * 2 * kNsBoxBytes + 2 * kPanelBlockBytes + 4 * kLoBytes + 1024;

// Matrices with at most this many rows (of X) whose result takes one product go to k_few, in
// 64 bits on the ordinary cores.
constexpr uint32_t kFewRows = 8;

// Tensor maps of a stack. Operand rows run along a product's depth ("K": boxes
// of 64 columns of 128 or 64 rows) except X in B X, whose columns are taken
// ("N": boxes of 64 rows of two or one groups of 64 columns). The lo parts'
// maps follow the hi parts'.
enum NsMap {
    kMapX0 = 0,        // {K128, K64, N128, N64} of the first X buffer, then of the second
    kMapX1 = 4,
    kMapA = 8,         // {K128, K64, 128 rows of 32 columns}
    kMapB = 11,        // {K128, K64}
    kMapLo = 13,
    kMapsPerStack = 26
};
constexpr int kMap32 = 2;  // from A's K128 map to its last
constexpr int kMap64 = 1;  // from a K128 (N128) map to its K64 (N64) one
constexpr int kMapN = 2;   // from X's K maps to its N maps

// One over the power of two that a matrix's X is held by before an iteration, and what it is
// held by after that over what it was held by before.
struct __align__(8) NsHold {
    float inv, regrade;
};

// One stack of equal matrices.
struct NsStack {
    __half* x[2];   // X hi, double-buffered across iterations: [count][m][ldx]
    __half* xl[2];  // X lo (three products; else 8-bit numbers, of the same pitch in elements)
    __half* a;      // [count][m][lda]
    __half* al;     // (three products only)
    __half* b;
    __half* bl;
    uint32_t m, n;        // shorter and longer side
    uint32_t ldx, lda;    // row pitches (ldx: whole groups of 64 columns)
    uint32_t rows, cols;  // as the caller has it
    uint32_t count;
    uint32_t first;       // index of its first matrix in the plan
    uint32_t transposed;  // rows > cols: X is the transpose
    uint32_t three;       // X in 22 bits (and products in three parts)
    uint32_t panel;       // worked on by k_panel
    uint32_t few;         // worked on by k_few
    uint32_t tiles;       // preparation tiles per matrix
    uint32_t first_tile;
    float sx, one_over_sx;  // power of two X is held by at least (NsHold)
    // input and output of a plain orthogonalisation; row and matrix strides in elements
    const void* src;
    void* dst;
    uint64_t src_row, src_mat, dst_row, dst_mat;
    // Muon: contiguous rows x cols matrices
    void* param;
    float* master;
    float* mom;
    float wd;
    float factor;         // the update's shape factor s
    uint32_t tensor;      // index of its tensor in the list (its gradient's place)
};

// Preparation tile: `parts` squares of 64 x 64 elements of one matrix, along
// its longer side.
constexpr int kPrepTile = 64;
struct PrepTile {
    uint32_t stack;
    uint32_t index;   // matrix of the stack
    uint16_t tr, tc;  // first square's row and column
    uint32_t parts;
};

// One output tile of one product of one matrix.
enum NsKind : uint32_t { kNsXXt = 0, kNsAA = 1, kNsBX = 2, kNsLast = 3 };
struct __align__(16) NsTask {
    uint32_t stack;
    uint32_t index;   // matrix of the stack
    uint32_t place;   // first row / 256 | first column / 32 << 16
    uint32_t shape;   // columns | kind << 16 | three products << 20 | transposed << 21 | step << 24
    // of the stack, so that a tile needs one read
    uint32_t m, n;
    uint32_t matrix;  // matrix of the plan
    uint32_t need;    // CTAs' tiles of this matrix that must be done before
    NsHold hold;      // the matrix's before the step, read as the task is handed out
    uint32_t pad[2];

    __host__ __device__ uint32_t row() const { return (place & 0xFFFFu) * kNsTileM; }
    __host__ __device__ uint32_t col() const { return (place >> 16) * 32u; }
    __host__ __device__ uint32_t width() const { return shape & 0xFFFFu; }
    __host__ __device__ uint32_t kind() const { return shape >> 16 & 15u; }
    __host__ __device__ bool three() const { return shape >> 20 & 1u; }
    __host__ __device__ bool transposed() const { return shape >> 21 & 1u; }
    __host__ __device__ uint32_t step() const { return shape >> 24; }
};
static_assert(sizeof(NsTask) == 48, "a task is three 16-byte loads");

// A Muon step's decision, from its first kernel for the others.
struct MatrixStep {
    int skip;    // nonzero: nothing is updated
    float inv;   // 1 / loss scale
    float coef;  // clip coefficient
};

// What a plan's kernels need, passed by value.
struct MatrixArgs {
    const NsStack* stacks;
    const CUtensorMap* maps;
    const NsTask* tasks;
    uint32_t n_tasks;
    const uint2* panels;   // k_panel's matrices: stack, matrix of the stack
    uint32_t n_panels;
    const uint2* few;      // k_few's
    uint32_t n_few;
    const PrepTile* prep;
    uint32_t n_prep;
    uint32_t n_matrices;
    double* partials;      // one per preparation tile
    uint32_t* tickets;     // per matrix: preparation tiles summed (0 between launches)
    float2* inv;           // per matrix: what X is held by at first / (norm + eps), in two factors
    NsHold* hold;          // per matrix, per step
    uint32_t* done;        // per matrix: product tiles done, counted by each CTA with rows in one
    uint32_t* next;        // tasks handed out, and k_panel's matrices
    int steps;
    MatrixStep* step;
    int* err;              // nonzero: a wait ran out in some run (stays)
    uint32_t* gave_up;     // nonzero: a wait ran out in this run (0 at its start): others need not wait
    float coef[kNsMaxSteps][3];
    int grows;             // every |a| is at least 1: a step does not shrink a bound on X's singular values
    double eps;
    const void* const* grads;  // Muon: gradient per tensor
    float momentum;
    int nesterov;
    int ema;
};

enum MatrixSource { kSrcF32 = 0, kSrcBf16 = 1, kSrcGradF32 = 2, kSrcGradBf16 = 3 };
enum MatrixDest { kDstF32 = 0, kDstBf16 = 1, kDstParamF32 = 2, kDstParamMixed = 3 };

cudaError_t prepare_matrix_kernels();
// Sum of squares per matrix (and the momentum update of a Muon step, which
// also takes and commits the step's decision), then the normalised hi + lo
// split, then all products and the output in one persistent kernel.
cudaError_t launch_matrix_ops(const MatrixArgs& args, int source, int dest, Ctl* ctl,
                              const ApplyArgs* step, int sms, cudaStream_t stream);

// ---- host: plans (matrix_plan.cu) ----
// Whether a stack's shape can be planned (a stack without elements can).
bool matrix_shape_ok(uint64_t count, uint64_t rows, uint64_t cols, std::string* why);
// Whether fp16 holds what these coefficients make of singular values of up to 1: X's below 7.99
// (A is held times 2^10), and B's eigenvalues up to 60 (likewise).
bool matrix_coef_ok(const float (*coef)[3], int steps, std::string* why);
// A stack that is written: `count` matrices of `rows` rows of `width` bytes, which do not
// overlap one another; strides in bytes.
struct MatrixSpan {
    uint64_t base;
    uint64_t count, rows, width, row, mat;
    int index;  // of the caller's list
};
// Whether no two of them share a byte; else the indices of two that do.
bool matrix_spans_apart(std::vector<MatrixSpan> spans, int* one, int* other);
// The quintic's usual coefficients, for every step.
void matrix_default_coef(float (*coef)[3]);
struct MatrixSpec {
    const void* src = nullptr;
    void* dst = nullptr;
    uint64_t rows = 0, cols = 0, count = 0;
    uint64_t src_row = 0, src_mat = 0, dst_row = 0, dst_mat = 0;
    void* param = nullptr;
    float* master = nullptr;
    float* mom = nullptr;
    float wd = 0.0f, factor = 1.0f;
    uint32_t tensor = 0;
};
struct MatrixPlanOpts {
    int steps = 5;
    float coef[kNsMaxSteps][3] = {};
    double eps = 1e-7;
    int source = kSrcF32, dest = kDstF32;
    int* err = nullptr;  // error word (nullptr: the plan's own)
};
struct MatrixPlan;
// nullptr on failure, with the reason in *why. The current device's.
MatrixPlan* matrix_plan_create(const MatrixSpec* specs, int n, const MatrixPlanOpts& opts,
                               std::string* why);
void matrix_plan_destroy(MatrixPlan* plan);
cudaError_t matrix_plan_run(MatrixPlan* plan, cudaStream_t stream);
// One Muon step (the decision from `step` and `ctl`).
cudaError_t matrix_plan_step(MatrixPlan* plan, Ctl* ctl, const ApplyArgs& step,
                             const void* const* grads, float momentum, bool nesterov, bool ema,
                             cudaStream_t stream);
int* matrix_plan_error_word(MatrixPlan* plan);

}  // namespace soarb
