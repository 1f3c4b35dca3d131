// Host side of the matrix operators: plans the preparation tiles, the product
// tiles and their order, and owns the workspace.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <memory>
#include <queue>
#include <vector>

#include <cudaTypedefs.h>

#include "matrix_ops.cuh"

namespace soarb {

struct MatrixPlan {
    int sms = 0;
    int source = 0, dest = 0;
    MatrixArgs args{};
    char* slab = nullptr;
};

namespace {

size_t up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// cuTensorMapEncodeTiled, from the driver through the runtime (the library
// does not link the driver's own library).
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) !=
            cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
        return nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
}

// A stack of `count` row-major fp16 matrices, in boxes of `height` rows of 64 (or 32) columns.
bool encode_rows(PFN_cuTensorMapEncodeTiled_v12000 f, CUtensorMap* map, void* base, uint32_t rows,
                 uint32_t cols, uint32_t ld, uint32_t count, uint32_t height, uint32_t width = 64) {
    const cuuint64_t dims[3] = {cols, rows, count};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2,
                                   static_cast<cuuint64_t>(ld) * rows * 2};
    const cuuint32_t box[3] = {width, height, 1}, es[3] = {1, 1, 1};
    return f(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE,
             width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// X's lo in 8 bits, in boxes of 128 rows of 64 columns (a row of `ld` bytes).
bool encode_lo8(PFN_cuTensorMapEncodeTiled_v12000 f, CUtensorMap* map, void* base, uint32_t rows,
                uint32_t cols, uint32_t ld, uint32_t count) {
    const cuuint64_t dims[3] = {cols, rows, count};
    const cuuint64_t strides[2] = {ld, static_cast<cuuint64_t>(ld) * rows};
    const cuuint32_t box[3] = {64, 128, 1}, es[3] = {1, 1, 1};
    return f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// The same as groups of 64 columns, in boxes of 64 rows of `groups` groups, a
// group after another. (Columns of the last group that are padding come with
// it; they are columns of a product that nobody stores.)
bool encode_groups(PFN_cuTensorMapEncodeTiled_v12000 f, CUtensorMap* map, void* base, uint32_t rows,
                   uint32_t ld, uint32_t count, uint32_t groups) {
    const cuuint64_t dims[4] = {64, rows, ld / 64, count};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(ld) * 2, 128,
                                   static_cast<cuuint64_t>(ld) * rows * 2};
    const cuuint32_t box[4] = {64, 64, groups, 1}, es[4] = {1, 1, 1, 1};
    return f(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box, es,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tiles of one product of one matrix: (first row / 256, first column / 32, width).
struct Tile {
    uint16_t row, col, width;
};
// A symmetric product: the blocks on the diagonal and what is right of them.
std::vector<Tile> symmetric_tiles(uint32_t m, uint32_t wide) {
    std::vector<Tile> out;
    for (uint32_t r = 0; r * kNsTileM < m; ++r)
        for (uint32_t c = r * kNsTileM; c < m; c += wide)
            out.push_back({static_cast<uint16_t>(r), static_cast<uint16_t>(c / 32),
                           static_cast<uint16_t>(std::min(wide, m - c))});
    return out;
}
std::vector<Tile> full_tiles(uint32_t m, uint32_t n, uint32_t wide) {
    std::vector<Tile> out;
    for (uint32_t c = 0; c < n; c += wide)
        for (uint32_t r = 0; r * kNsTileM < m; ++r)
            out.push_back({static_cast<uint16_t>(r), static_cast<uint16_t>(c / 32),
                           static_cast<uint16_t>(std::min(wide, n - c))});
    return out;
}
std::vector<Tile> product_tiles(const NsStack& s, uint32_t kind, uint32_t wide) {
    if (s.three) wide = std::min(wide, static_cast<uint32_t>(kNsTileN / 2));
    return kind == kNsBX ? full_tiles(s.m, s.n, wide) : symmetric_tiles(s.m, wide);
}

}  // namespace

bool matrix_shape_ok(uint64_t count, uint64_t rows, uint64_t cols, std::string* why) {
    constexpr uint64_t kMostSide = 1ull << 20, kMost = 1ull << 38;
    if (rows > kMostSide || cols > kMostSide) {
        *why = "a side of more than 1048576";
        return false;
    }
    if (rows && cols && count > kMost / (rows * cols)) {
        *why = "more than 2^38 elements";
        return false;
    }
    if (count > 0x7FFFFFFFull) {
        *why = "more than 2^31 - 1 matrices";
        return false;
    }
    return true;
}

bool matrix_coef_ok(const float (*coef)[3], int steps, std::string* why) {
    // X's singular values lie in [0, most], and |s p(s)| takes that to [0, its largest value there]
    constexpr int kPoints = 4096;
    double most = 1.0;
    for (int k = 0; k < steps; ++k) {
        double next = 0.0, b = 0.0;
        bool finite = true;
        for (int i = 0; i <= kPoints; ++i) {
            const double s = most * i / kPoints, q = s * s;
            const double p = std::fabs(coef[k][0] + q * (coef[k][1] + q * static_cast<double>(coef[k][2])));
            finite = finite && std::isfinite(p);
            b = std::max(b, p);
            next = std::max(next, s * p);
        }
        if (!finite || b > 60.0 || next >= 7.99) {
            *why = "coefficients of step " + std::to_string(k) + ": " +
                   (!finite   ? "not finite"
                    : b > 60.0 ? "|a + b s^2 + c s^4| above 60 at a singular value of X"
                               : "a singular value of X would reach 7.99");
            return false;
        }
        most = next;
    }
    return true;
}

namespace {
// A span's rows one after another, by their addresses.
struct SpanRows {
    const MatrixSpan* s;
    bool by_matrix;  // all of a matrix's rows come before the next matrix's
    uint64_t matrix = 0, row = 0;
    uint64_t begin() const { return s->base + matrix * s->mat + row * s->row; }
    bool next() {
        uint64_t& inner = by_matrix ? row : matrix;
        uint64_t& outer = by_matrix ? matrix : row;
        if (++inner < (by_matrix ? s->rows : s->count)) return true;
        inner = 0;
        return ++outer < (by_matrix ? s->count : s->rows);
    }
};
uint64_t span_end(const MatrixSpan& s) { return s.base + (s.count - 1) * s.mat + (s.rows - 1) * s.row + s.width; }
}  // namespace

bool matrix_spans_apart(std::vector<MatrixSpan> spans, int* one, int* other) {
    for (MatrixSpan& s : spans) {
        if (s.rows > 1 && s.row == s.width) s.width *= s.rows, s.rows = 1;
        if (s.rows == 1 && s.count > 1 && s.mat == s.width) s.width *= s.count, s.count = 1;
    }
    std::sort(spans.begin(), spans.end(), [](const MatrixSpan& x, const MatrixSpan& y) { return x.base < y.base; });
    // those that reach into one another, row by row
    for (size_t i = 0, j; i < spans.size(); i = j) {
        uint64_t end = span_end(spans[i]);
        for (j = i + 1; j < spans.size() && spans[j].base < end; ++j) end = std::max(end, span_end(spans[j]));
        if (j == i + 1) continue;
        auto later = [](const SpanRows& x, const SpanRows& y) { return x.begin() > y.begin(); };
        std::priority_queue<SpanRows, std::vector<SpanRows>, decltype(later)> rows(later);
        for (size_t k = i; k < j; ++k) {
            const MatrixSpan& s = spans[k];
            rows.push({&s, s.count == 1 || s.mat >= (s.rows - 1) * s.row + s.width});
        }
        uint64_t taken = 0;
        int by = -1;
        while (!rows.empty()) {
            SpanRows r = rows.top();
            rows.pop();
            if (r.begin() < taken) {
                *one = std::min(by, r.s->index);
                *other = std::max(by, r.s->index);
                return false;
            }
            taken = r.begin() + r.s->width;
            by = r.s->index;
            if (r.next()) rows.push(r);
        }
    }
    return true;
}

void matrix_default_coef(float (*coef)[3]) {
    for (int i = 0; i < kNsMaxSteps; ++i) {
        coef[i][0] = 3.4445f;
        coef[i][1] = -4.7750f;
        coef[i][2] = 2.0315f;
    }
}

void matrix_plan_destroy(MatrixPlan* p) {
    if (!p) return;
    cudaFree(p->slab);
    delete p;
}

MatrixPlan* matrix_plan_create(const MatrixSpec* specs, int n_specs, const MatrixPlanOpts& opts,
                               std::string* why) {
    auto plan = std::make_unique<MatrixPlan>();
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess)
        e = cudaDeviceGetAttribute(&plan->sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = prepare_matrix_kernels();
    if (e != cudaSuccess) {
        *why = std::string("kernel set-up: ") + cudaGetErrorString(e);
        return nullptr;
    }
    const auto encoder = encode_fn();
    if (!encoder) {
        *why = "the driver offers no cuTensorMapEncodeTiled";
        return nullptr;
    }
    plan->source = opts.source;
    plan->dest = opts.dest;
    const bool three = opts.dest == kDstF32 || opts.dest == kDstParamF32;

    // stacks, and their places in the workspace
    std::vector<NsStack> stacks;
    std::vector<PrepTile> prep;
    struct Place {
        size_t x[2], xl[2], a, al, b, bl;
    };
    std::vector<Place> places;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = up(off + bytes, 1024);
        return at;
    };
    uint64_t matrices = 0, prep_tiles = 0;
    // A tile is one square where there are few (every SM gets some), four where there are many
    // (a sum and a ticket for 16384 elements instead of 4096).
    uint64_t squares = 0;
    for (int i = 0; i < n_specs; ++i)
        squares += specs[i].count * ((specs[i].rows + kPrepTile - 1) / kPrepTile) *
                   ((specs[i].cols + kPrepTile - 1) / kPrepTile);
    // k_panel or k_ns for a matrix of at most 256 rows (of X). k_panel gives it to one pair of CTAs
    // for 30 us + 0.075 us a column, k_ns deals its tiles to all pairs but goes through 15 products
    // one after the other. One 256 x 1024 matrix takes 120 us in either, 256 x 512 79 in k_panel and
    // 109 in k_ns, 256 x 4096 376 and 171; 37 of 256 x 4096 (half the pairs) 546 and 516, 74 of them
    // 731 and 906. So long matrices go to k_panel where the list has enough columns for all pairs.
    uint64_t panel_columns = 0;
    for (int i = 0; i < n_specs; ++i)
        if (const uint64_t m = std::min(specs[i].rows, specs[i].cols); !three && m > kFewRows && m <= kPanelSide)
            panel_columns += specs[i].count * std::max(specs[i].rows, specs[i].cols);
    const uint64_t panel_most = std::max<uint64_t>(kPanelAnyColumns, 2 * panel_columns / std::max(1, plan->sms / 2));
    const uint32_t prep_parts = squares >= 16ull * static_cast<uint64_t>(plan->sms) ? 4 : 1;
    for (int i = 0; i < n_specs; ++i) {
        const MatrixSpec& q = specs[i];
        if (!q.rows || !q.cols || !q.count) continue;
        NsStack s{};
        s.rows = static_cast<uint32_t>(q.rows);
        s.cols = static_cast<uint32_t>(q.cols);
        s.count = static_cast<uint32_t>(q.count);
        s.transposed = s.rows > s.cols;
        s.m = std::min(s.rows, s.cols);
        s.n = std::max(s.rows, s.cols);
        s.few = !three && s.m <= kFewRows;
        s.three = three || s.few;
        s.panel = !s.three && s.m <= kPanelSide && s.n <= panel_most;
        s.ldx = static_cast<uint32_t>(up(s.n, 64));
        s.lda = static_cast<uint32_t>(up(s.m, 8));
        s.first = static_cast<uint32_t>(matrices);
        matrices += s.count;
        const int lg = static_cast<int>(
            std::floor(0.5 * std::log2(static_cast<double>(s.m) * static_cast<double>(s.n))));
        s.sx = std::ldexp(1.0f, std::min(12, std::max(6, lg)));
        s.one_over_sx = 1.0f / s.sx;
        s.src = q.src;
        s.dst = q.dst;
        s.src_row = q.src_row;
        s.src_mat = q.src_mat;
        s.dst_row = q.dst_row;
        s.dst_mat = q.dst_mat;
        s.param = q.param;
        s.master = q.master;
        s.mom = q.mom;
        s.wd = q.wd;
        s.factor = q.factor;
        s.tensor = q.tensor;
        // (tiles lie along the longer side)
        const uint32_t along = (s.n + kPrepTile - 1) / kPrepTile, across = (s.m + kPrepTile - 1) / kPrepTile;
        s.tiles = across * ((along + prep_parts - 1) / prep_parts);
        s.first_tile = static_cast<uint32_t>(prep_tiles);
        prep_tiles += static_cast<uint64_t>(s.count) * s.tiles;
        Place p{};
        const size_t xb = static_cast<size_t>(s.count) * s.m * s.ldx * 2;
        const size_t ab = static_cast<size_t>(s.count) * s.m * s.lda * 2;
        for (int k = 0; k < (s.few ? 1 : 2); ++k) {
            p.x[k] = take(xb);
            p.xl[k] = take(s.three ? xb : xb / 2);
        }
        if (!s.panel && !s.few) {
            p.a = take(ab);
            p.b = take(ab);
        }
        if (three) {
            p.al = take(ab);
            p.bl = take(ab);
        }
        stacks.push_back(s);
        places.push_back(p);
    }
    // refused before the host's tables are made, which grow with the list as the workspace does
    size_t free_bytes = 0, all_memory = 0;
    if ((e = cudaMemGetInfo(&free_bytes, &all_memory)) != cudaSuccess) {
        *why = std::string("device memory: ") + cudaGetErrorString(e);
        return nullptr;
    }
    if (off > all_memory) {
        *why = "matrix workspace (" + std::to_string(off) + " bytes): more than the device's memory";
        return nullptr;
    }
    if (prep_tiles > 0xFFFF0000ull || matrices > 0xFFFF0000ull) {
        *why = "too many matrices in one list";
        return nullptr;
    }
    for (uint32_t si = 0; si < stacks.size(); ++si) {
        const NsStack& s = stacks[si];
        const bool down = s.rows > s.cols;
        const uint32_t along = (s.n + kPrepTile - 1) / kPrepTile, across = (s.m + kPrepTile - 1) / kPrepTile;
        for (uint32_t c = 0; c < s.count; ++c)
            for (uint32_t y = 0; y < across; ++y)
                for (uint32_t x = 0; x < along; x += prep_parts)
                    prep.push_back({si, c, static_cast<uint16_t>(down ? x : y), static_cast<uint16_t>(down ? y : x),
                                    std::min(prep_parts, along - x)});
    }

    // The tasks, in an order in which every tile's inputs come before it: lists
    // ("waves") of matrices go through their products side by side, one list
    // after another, all about as long. A product's last tiles are waited for by
    // the first ones of its matrix's next product, for some 10 us, which the other
    // matrices of the list have to fill: with 32, 64 and 128 MB in a list 46M
    // parameters in matrices of many shapes take 1682, 1369 and 1313 us a step, with
    // more no less. Nor does the L2 cache ask for short ones. A list of few tiles is
    // drawn out until a product of it occupies every pair of CTAs three times: 200M
    // parameters in layers 1024 wide take 5.70, 5.67, 5.62 and 5.69 ms with 64, 128, 256
    // and 512 MB, all of them in one list 5.70, and with a product that occupies the pairs
    // once 6.15, 5.88, 5.75 and 5.67. (The 46M in lists of 64 MB lose 29 us by it.)
    constexpr uint64_t kWaveBytes = 256ull << 20;
    const uint64_t wave_tiles = 3 * static_cast<uint64_t>(plan->sms) / 2;
    std::vector<NsTask> tasks;
    struct Run {
        uint32_t stack, from, to;
    };
    std::vector<Run> wave;
    uint64_t wave_bytes = 0;
    auto flush = [&]() {
        std::vector<uint32_t> counted(wave.size(), 0);  // tiles of a matrix before this product
        for (int step = 0; step < opts.steps; ++step) {
            for (uint32_t kind = kNsXXt; kind <= kNsBX; ++kind) {
                // narrower tiles where whole ones would leave pairs of CTAs idle
                uint32_t wide = kNsTileN;
                for (; wide > kNsTileN / 2; wide /= 2) {
                    uint64_t all = 0;
                    for (const Run& r : wave)
                        all += product_tiles(stacks[r.stack], kind, wide).size() * (r.to - r.from);
                    if (all >= static_cast<uint64_t>(plan->sms / 2)) break;
                }
                for (size_t w = 0; w < wave.size(); ++w) {
                    const NsStack& s = stacks[wave[w].stack];
                    const std::vector<Tile> tiles = product_tiles(s, kind, wide);
                    for (uint32_t i = wave[w].from; i < wave[w].to; ++i)
                        for (const Tile& t : tiles) {
                            NsTask k{};
                            k.stack = wave[w].stack;
                            k.index = i;
                            k.place = t.row | static_cast<uint32_t>(t.col) << 16;
                            k.shape = t.width |
                                      (kind == kNsBX && step + 1 == opts.steps ? kNsLast : kind) << 16 |
                                      s.three << 20 | s.transposed << 21 | static_cast<uint32_t>(step) << 24;
                            k.m = s.m;
                            k.n = s.n;
                            k.matrix = s.first + i;
                            k.need = counted[w];
                            tasks.push_back(k);
                        }
                    // (a CTA without rows in a tile does not count it)
                    for (const Tile& t : tiles)
                        counted[w] += s.m - t.row * kNsTileM > kNsRows ? 2 : 1;
                }
            }
        }
        wave.clear();
        wave_bytes = 0;
    };
    auto bytes_of = [&](const NsStack& s) {
        return s.m * ((three ? 8ull : 6ull) * s.ldx + (three ? 8ull : 4ull) * s.lda);
    };
    uint64_t all_bytes = 0;
    for (const NsStack& s : stacks)
        if (!s.panel && !s.few) all_bytes += s.count * bytes_of(s);
    const uint64_t wave_most = all_bytes / std::max<uint64_t>(1, all_bytes / kWaveBytes) + 1;
    uint64_t tiles_in_wave = 0;
    for (uint32_t si = 0; si < stacks.size(); ++si) {
        const NsStack& s = stacks[si];
        if (s.panel || s.few) continue;
        const uint64_t each = bytes_of(s);
        const uint64_t tiles = product_tiles(s, kNsXXt, kNsTileN).size();
        for (uint32_t i = 0; i < s.count;) {
            // as many as the wave still takes: until it has both the bytes and the tiles
            uint64_t k = 1;
            if (wave_bytes < wave_most) k = std::max(k, (wave_most - wave_bytes) / each);
            if (tiles_in_wave < wave_tiles) k = std::max(k, (wave_tiles - tiles_in_wave) / tiles);
            k = std::min<uint64_t>(k, s.count - i);
            wave.push_back({si, i, i + static_cast<uint32_t>(k)});
            wave_bytes += each * k;
            tiles_in_wave += tiles * k;
            i += static_cast<uint32_t>(k);
            if (wave_bytes >= wave_most && tiles_in_wave >= wave_tiles) {
                flush();
                tiles_in_wave = 0;
            }
        }
    }
    flush();
    // k_panel's and k_few's matrices, the longest first
    std::vector<uint2> panels, few;
    {
        std::vector<uint32_t> by;
        for (uint32_t si = 0; si < stacks.size(); ++si)
            if (stacks[si].panel || stacks[si].few) by.push_back(si);
        std::stable_sort(by.begin(), by.end(), [&](uint32_t x, uint32_t y) { return stacks[x].n > stacks[y].n; });
        for (uint32_t si : by)
            for (uint32_t i = 0; i < stacks[si].count; ++i)
                (stacks[si].few ? few : panels).push_back(make_uint2(si, i));
    }
    if (tasks.size() > 0xFFFF0000ull) {
        *why = "too many matrices in one list";
        return nullptr;
    }

    // tables behind the operands
    const size_t operand_bytes = off;
    const size_t o_stacks = take(stacks.size() * sizeof(NsStack));
    const size_t o_maps = take(stacks.size() * kMapsPerStack * sizeof(CUtensorMap));
    const size_t o_tasks = take(tasks.size() * sizeof(NsTask));
    const size_t o_prep = take(prep.size() * sizeof(PrepTile));
    const size_t o_panels = take(panels.size() * sizeof(uint2));
    const size_t o_few = take(few.size() * sizeof(uint2));
    const size_t tables_end = off;
    const size_t o_partials = take(prep.size() * sizeof(double));
    const size_t o_inv = take(matrices * sizeof(float2));
    const size_t o_hold = take(matrices * opts.steps * sizeof(NsHold));
    const size_t zero_from = off;
    const size_t o_tickets = take(matrices * sizeof(uint32_t));
    const size_t o_done = take(matrices * sizeof(uint32_t));
    const size_t o_words = take(256);
    if ((e = cudaMalloc(&plan->slab, off)) != cudaSuccess) {
        plan->slab = nullptr;
        *why = "matrix workspace (" + std::to_string(off) + " bytes): " + cudaGetErrorString(e);
        cudaGetLastError();
        return nullptr;
    }
    auto at = [&](size_t o) { return plan->slab + o; };
    std::vector<char> host(tables_end - operand_bytes);
    std::vector<CUtensorMap> maps(stacks.size() * kMapsPerStack);
    bool ok = true;
    for (size_t i = 0; i < stacks.size(); ++i) {
        NsStack& s = stacks[i];
        const Place& p = places[i];
        for (int k = 0; k < 2; ++k) {
            s.x[k] = reinterpret_cast<__half*>(at(p.x[k]));
            s.xl[k] = reinterpret_cast<__half*>(at(p.xl[k]));
        }
        s.a = reinterpret_cast<__half*>(at(p.a));
        s.b = reinterpret_cast<__half*>(at(p.b));
        s.al = three ? reinterpret_cast<__half*>(at(p.al)) : s.a;
        s.bl = three ? reinterpret_cast<__half*>(at(p.bl)) : s.b;
        CUtensorMap* m = maps.data() + i * kMapsPerStack;
        for (int k = 0; s.panel && k < 2; ++k) {
            CUtensorMap* qx = m + (k ? kMapX1 : kMapX0);
            ok = ok && encode_rows(encoder, qx, s.x[k], s.m, s.n, s.ldx, s.count, 128) &&
                 encode_groups(encoder, qx + kMapN + kMap64, s.x[k], s.m, s.ldx, s.count, 1) &&
                 encode_lo8(encoder, qx + kMapLo, s.xl[k], s.m, s.n, s.ldx, s.count);
        }
        for (int lo = 0; !s.panel && !s.few && lo < 2; ++lo) {
            CUtensorMap* q = m + (lo ? kMapLo : 0);
            for (int k = 0; k < 2; ++k) {
                __half* x = lo ? s.xl[k] : s.x[k];
                CUtensorMap* qx = q + (k ? kMapX1 : kMapX0);
                if (lo && !three) {
                    ok = ok && encode_lo8(encoder, qx, x, s.m, s.n, s.ldx, s.count);
                    continue;
                }
                ok = ok && encode_rows(encoder, qx, x, s.m, s.n, s.ldx, s.count, 128) &&
                     encode_rows(encoder, qx + kMap64, x, s.m, s.n, s.ldx, s.count, 64) &&
                     encode_groups(encoder, qx + kMapN, x, s.m, s.ldx, s.count, 2) &&
                     encode_groups(encoder, qx + kMapN + kMap64, x, s.m, s.ldx, s.count, 1);
                __half* ab = k ? (lo ? s.bl : s.b) : (lo ? s.al : s.a);
                CUtensorMap* qa = q + (k ? kMapB : kMapA);
                ok = ok && encode_rows(encoder, qa, ab, s.m, s.m, s.lda, s.count, 128) &&
                     encode_rows(encoder, qa + kMap64, ab, s.m, s.m, s.lda, s.count, 64) &&
                     (k || encode_rows(encoder, qa + kMap32, ab, s.m, s.m, s.lda, s.count, 128, 32));
            }
        }
    }
    auto put = [&](size_t o, const void* from, size_t bytes) {
        if (bytes) std::memcpy(host.data() + (o - operand_bytes), from, bytes);
    };
    put(o_stacks, stacks.data(), stacks.size() * sizeof(NsStack));
    put(o_maps, maps.data(), maps.size() * sizeof(CUtensorMap));
    put(o_tasks, tasks.data(), tasks.size() * sizeof(NsTask));
    put(o_prep, prep.data(), prep.size() * sizeof(PrepTile));
    put(o_panels, panels.data(), panels.size() * sizeof(uint2));
    put(o_few, few.data(), few.size() * sizeof(uint2));
    if (ok) {
        e = cudaMemset(plan->slab, 0, operand_bytes);
        if (e == cudaSuccess) e = cudaMemcpy(at(operand_bytes), host.data(), host.size(), cudaMemcpyHostToDevice);
        if (e == cudaSuccess) e = cudaMemset(at(zero_from), 0, off - zero_from);
        if (e == cudaSuccess) e = cudaDeviceSynchronize();
    }
    if (!ok || e != cudaSuccess) {
        *why = ok ? std::string("plan upload: ") + cudaGetErrorString(e) : "cuTensorMapEncodeTiled failed";
        cudaFree(plan->slab);
        return nullptr;
    }
    MatrixArgs& a = plan->args;
    a.stacks = reinterpret_cast<const NsStack*>(at(o_stacks));
    a.maps = reinterpret_cast<const CUtensorMap*>(at(o_maps));
    a.tasks = reinterpret_cast<const NsTask*>(at(o_tasks));
    a.n_tasks = static_cast<uint32_t>(tasks.size());
    a.prep = reinterpret_cast<const PrepTile*>(at(o_prep));
    a.n_prep = static_cast<uint32_t>(prep.size());
    a.panels = reinterpret_cast<const uint2*>(at(o_panels));
    a.n_panels = static_cast<uint32_t>(panels.size());
    a.few = reinterpret_cast<const uint2*>(at(o_few));
    a.n_few = static_cast<uint32_t>(few.size());
    a.steps = opts.steps;
    a.n_matrices = static_cast<uint32_t>(matrices);
    a.partials = reinterpret_cast<double*>(at(o_partials));
    a.inv = reinterpret_cast<float2*>(at(o_inv));
    a.hold = reinterpret_cast<NsHold*>(at(o_hold));
    a.tickets = reinterpret_cast<uint32_t*>(at(o_tickets));
    a.done = reinterpret_cast<uint32_t*>(at(o_done));
    a.next = reinterpret_cast<uint32_t*>(at(o_words));
    a.gave_up = a.next + 2;
    a.step = reinterpret_cast<MatrixStep*>(at(o_words + 64));
    a.err = opts.err ? opts.err : reinterpret_cast<int*>(at(o_words + 128));
    std::memcpy(a.coef, opts.coef, sizeof a.coef);
    a.grows = 1;
    for (int i = 0; i < opts.steps; ++i)
        if (!(std::fabs(opts.coef[i][0]) >= 1.0f)) a.grows = 0;
    a.eps = opts.eps;
    return plan.release();
}

cudaError_t matrix_plan_run(MatrixPlan* p, cudaStream_t stream) {
    return launch_matrix_ops(p->args, p->source, p->dest, nullptr, nullptr, p->sms, stream);
}

cudaError_t matrix_plan_step(MatrixPlan* p, Ctl* ctl, const ApplyArgs& step, const void* const* grads,
                             float momentum, bool nesterov, bool ema, cudaStream_t stream) {
    MatrixArgs a = p->args;
    a.grads = grads;
    a.momentum = momentum;
    a.nesterov = nesterov ? 1 : 0;
    a.ema = ema ? 1 : 0;
    return launch_matrix_ops(a, p->source, p->dest, ctl, &step, p->sms, stream);
}

int* matrix_plan_error_word(MatrixPlan* p) { return p->args.err; }

}  // namespace soarb
