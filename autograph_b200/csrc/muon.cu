// Newton-Schulz orthogonalisation of gradient matrices, and Muon's parameter update around it.
//
// With x = u / norm(u), as n x m with n <= m (the transpose of a taller u), a step is
//   a = x x^T,  b = B a + C a a,  x <- A x + b x,   (A, B, C) = (3.4445, -4.7750, 2.0315),
// which maps every singular value s to A s + B s^3 + C s^5 and keeps the singular vectors.  muon_product.cuh has the steps; here
// are the passes before them for large lists (25088 x 512 with its momentum: 42 and 50 us, 128 MB each), the choices by
// size, and the entry points.
#include <algorithm>
#include <vector>

#include "muon.cuh"
#include "muon_product.cuh"

namespace ag {
namespace muon {

constexpr int64_t kMostShort = 16384, kMostLong = 1 << 20;
constexpr int kMostMatrices = 4096, kMostSteps = 20;
constexpr int64_t kMostRows = 4ll << 23;      // of the workspace of a launch with more than one matrix: 4 GiB
constexpr int kMostParts = 2048;              // partial sums of squares of a matrix
// Values of a launch up to which its one kernel makes the planes too (LeNet5's weights 127.9 us, apart 129.8, one launch for
// three).  Larger passes are bound by memory, which that kernel's eleven warps an SM do not keep busy.
constexpr int64_t kInside = 1 << 20;

// The CTA's matrix, of which it takes the `count(m)`-th piece.
template <class F>
__device__ __forceinline__ int find_matrix(const Group &g, int &piece, F count) {
    int i = 0;
    for (piece = blockIdx.x; i + 1 < g.n && piece >= count(g.m[i]); ++i) piece -= count(g.m[i]);
    return i;
}

template <class T>
__global__ void __launch_bounds__(256) momentum_kernel(const __grid_constant__ Group g, double *parts) {
    __shared__ double scratch[8];
    int part;
    const int i = find_matrix(g, part, [](const Matrix &m) { return m.parts; });
    momentum_part<T, 256>(g.m[i], g.rule, part, parts, scratch);
}

template <class T>
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ Group g, const double *parts, __half *planes) {
    __shared__ double scratch[8];
    __shared__ float tile[64][65];
    int block;
    const int i = find_matrix(g, block, [](const Matrix &m) { return m.x(0).plane / 64; });
    const double inv = inverse_norm(g.m[i], parts, scratch);
    split_tile<T, 256>(g.m[i], g.rule, block, inv, planes, tile);
}

// First step on x x^T alone (muon_product.cuh): the last two, for bf16 results the last three, but not the first two.  Counted in
// products of planes of an n x n matrix, for x of r times its size, five steps are 22.5 r + 7.5 on x throughout, 18 r + 12 with
// two on x x^T, 13.5 r + 16.5 with three.  us, f32, two and three: 25088 x 512 with three small ones 636 and 548, four of 1024 x 4096
// 1025 and 892, 509 x 1531 twice and 777 x 1009 392 and 364.
static int squares_from(const Matrix &m, int steps, bool bf16) {
    if (m.n() < 128 || m.wide() < 2 * m.n()) return steps;
    return std::min(steps, std::max(2, steps - (bf16 ? 3 : 2)));
}

template <class T, int BN>
static int launch(ag_device *dev, const CUtensorMap &map, __half *planes, double *norms, float4 *slices, const Group &g) {
    auto kernel = muon_kernel<T, BN>;
    static SmemAllowed allowed;
    AG_TRY(allow_smem<kSmem>(dev, kernel, allowed));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)dev->sm_count);
    cfg.blockDim = kThreads;
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = dev->stream;
    // the grid's barrier needs all CTAs at once
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeCooperative;
    attr.val.cooperative = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    AG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, map, planes, norms, slices, dev->tile_counters, dev->status_dev, g));
    AG_CHECK_LAUNCH();
    return AG_OK;
}

// One launch: its matrices, and what it takes of the workspace.
struct Launch {
    Group g;
    int64_t space;       // rows of planes
    int parts, blocks;   // CTAs of the passes before the steps
    bool narrow;
};

// The launches that a list takes.
static int make_launches(const std::vector<Matrix> &matrices, const Rule &rule, int steps, bool bf16, int sm_count,
                         std::vector<Launch> &launches) {
    for (size_t first = 0; first < matrices.size(); first += launches.back().g.n) {
        launches.push_back({});
        Launch &l = launches.back();
        Group &g = l.g;
        g.steps = steps;
        g.rule = rule;
        int64_t values = 0, tiles = 0;
        for (; g.n < kGroup && first + g.n < matrices.size(); ++g.n) {
            Matrix &m = g.m[g.n];
            m = matrices[first + g.n];
            const int64_t n = m.n(), wide = m.wide();
            m.squares = squares_from(m, steps, bf16);
            if (g.n > 0 && l.space + m.space(steps) > kMostRows) break;
            m.row = (int)std::min<int64_t>(l.space, INT32_MAX);
            l.space += m.space(steps);
            g.phases = std::max(g.phases, m.phases(steps));
            m.part0 = l.parts;
            m.parts = (int)std::min<int64_t>(ceil_div(n * wide, 8192), kMostParts);
            l.parts += m.parts;
            l.blocks += m.x(0).plane / 64;
            values += n * wide;
            tiles += ceil_div(n, 128) * ceil_div(wide, 128);
        }
        AG_REQUIRE(l.space < (1ll << 31), AG_ERR_LIMIT, "newton_schulz: the matrices' workspace is too large");
        g.inside = values <= kInside;
        // Tiles of 64 columns where wide ones would leave SMs idle: us, wide and narrow, f32 1024 x 1024 329 and 242, 512 x 512 230
        // and 165, 1536 x 1024 331 and 313; beyond a tile an SM wide ones win (two 1024 x 1024 and 700 x 700 405 and 451).
        l.narrow = tiles <= sm_count;
    }
    return AG_OK;
}

// The workspace of all launches of a call, one after the other.
struct Space {
    double *norms;
    float4 *slices;
    __half *planes;
    int64_t rows;   // of the planes
};
static int take_space(ag_device *dev, const std::vector<Launch> &launches, Space &s) {
    s.rows = 0;
    for (const Launch &l : launches) s.rows = std::max(s.rows, l.space);
    const size_t heads = (size_t)kGroup * kMostParts * sizeof(double), sums = (size_t)dev->sm_count * 128 * 128 * sizeof(float);
    void *ws;
    AG_TRY(engine_scratch(dev, heads + sums + (size_t)s.rows * 128, &ws));
    s.norms = (double *)ws;
    s.slices = (float4 *)((char *)ws + heads);
    s.planes = (__half *)((char *)ws + heads + sums);
    return AG_OK;
}

// Nothing is launched before the whole list has its workspace: a call that fails has changed nothing.
template <class T>
int run(ag_device *dev, const std::vector<Matrix> &matrices, const Rule &rule, int steps) {
    std::vector<Launch> launches;
    AG_TRY(make_launches(matrices, rule, steps, sizeof(T) == 2, dev->sm_count, launches));
    if (launches.empty()) return AG_OK;
    Space s;
    AG_TRY(take_space(dev, launches, s));
    CUtensorMap map;
    const uint64_t dims[2] = {64, (uint64_t)s.rows}, strides[1] = {64};
    const uint32_t box[2] = {64, 64};
    AG_TRY(make_tmap_bf16(&map, s.planes, 2, dims, strides, box));   // f16 has the same size
    for (const Launch &l : launches) {
        const Group &g = l.g;
        if (!g.inside) {
            momentum_kernel<T><<<l.parts, 256, 0, dev->stream>>>(g, s.norms);
            AG_CHECK_LAUNCH();
            split_kernel<T><<<l.blocks, 256, 0, dev->stream>>>(g, s.norms, s.planes);
            AG_CHECK_LAUNCH();
        }
        AG_TRY((l.narrow ? launch<T, 64>(dev, map, s.planes, s.norms, s.slices, g)
                         : launch<T, 128>(dev, map, s.planes, s.norms, s.slices, g)));
    }
    return AG_OK;
}

// What a call may not do, whatever the matrix.
static int check_call(ag_dtype dtype, int32_t n, const void *matrices, int32_t steps) {
    AG_REQUIRE(is_float_dtype(dtype), AG_ERR_DTYPE, "newton_schulz: dtype %d unimplemented", (int)dtype);
    AG_REQUIRE(n >= 0, AG_ERR_INVALID, "newton_schulz: negative number of matrices");
    AG_REQUIRE(n <= kMostMatrices, AG_ERR_LIMIT, "newton_schulz: %d matrices, at most %d", n, kMostMatrices);
    AG_REQUIRE(n == 0 || matrices != nullptr, AG_ERR_INVALID, "newton_schulz: null pointer");
    AG_REQUIRE(steps >= 1 && steps <= kMostSteps, AG_ERR_INVALID, "newton_schulz: steps must be in 1..%d", kMostSteps);
    return AG_OK;
}

static int check_size(int64_t rows, int64_t cols) {
    AG_REQUIRE(rows > 0 && cols > 0, AG_ERR_SHAPE, "newton_schulz: a matrix needs at least one value");
    AG_REQUIRE(std::min(rows, cols) <= kMostShort && std::max(rows, cols) <= kMostLong && rows * cols < (1ll << 31), AG_ERR_LIMIT,
               "newton_schulz: a matrix of %lld x %lld is beyond the limit", (long long)rows, (long long)cols);
    return AG_OK;
}

// A range of bytes that a call reads or writes; `matrix` so that a matrix may lie on its own source.
struct Range {
    uintptr_t begin, end;
    bool written;
    int matrix;
    bool may_alias;
};

// Refuses written ranges that share bytes with another range of the call: the matrices run side by side.
static int check_overlap(std::vector<Range> &ranges) {
    std::sort(ranges.begin(), ranges.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
    for (size_t i = 0; i < ranges.size(); ++i)
        for (size_t j = i + 1; j < ranges.size() && ranges[j].begin < ranges[i].end; ++j) {
            const Range &a = ranges[i], &b = ranges[j];
            if (!a.written && !b.written) continue;
            if (a.matrix == b.matrix && a.may_alias && b.may_alias && a.begin == b.begin) continue;
            return fail(AG_ERR_INVALID, "newton_schulz: a matrix that is written overlaps another one");
        }
    return AG_OK;
}

}  // namespace muon

int muon_prepare(ag_device *dev, ag_dtype dtype, const std::vector<ag_muon_matrix> &matrices, int steps) {
    AG_REQUIRE(matrices.size() <= (size_t)muon::kMostMatrices, AG_ERR_LIMIT, "muon: %zu matrices, at most %d", matrices.size(),
               muon::kMostMatrices);
    if (matrices.empty()) return AG_OK;
    AG_TRY(muon::check_call(dtype, (int32_t)matrices.size(), matrices.data(), steps));
    std::vector<muon::Matrix> list;
    for (const ag_muon_matrix &m : matrices) {
        AG_TRY(muon::check_size(m.rows, m.cols));
        list.push_back({m.g, m.w, m.v, m.rows, m.cols, m.scale, 0, 0, 0, 0});
    }
    std::vector<muon::Launch> launches;
    AG_TRY(muon::make_launches(list, {}, steps, dtype == AG_BF16, dev->sm_count, launches));
    muon::Space space;
    return muon::take_space(dev, launches, space);
}

}  // namespace ag

using namespace ag;

extern "C" {

int ag_newton_schulz(ag_device *dev, ag_dtype dtype, int32_t n, const ag_polar_matrix *matrices, int32_t steps) {
    AG_ENTER(dev);
    AG_TRY(muon::check_call(dtype, n, matrices, steps));
    try {
        std::vector<muon::Matrix> list;
        std::vector<muon::Range> ranges;
        for (int32_t i = 0; i < n; ++i) {
            const ag_polar_matrix &m = matrices[i];
            AG_TRY(muon::check_size(m.rows, m.cols));
            AG_REQUIRE(m.g && m.o, AG_ERR_INVALID, "newton_schulz: null pointer");
            const uintptr_t bytes = (uintptr_t)(m.rows * m.cols) * dtype_size(dtype);
            ranges.push_back({(uintptr_t)m.g, (uintptr_t)m.g + bytes, false, i, true});
            ranges.push_back({(uintptr_t)m.o, (uintptr_t)m.o + bytes, true, i, true});
            list.push_back({m.g, m.o, nullptr, m.rows, m.cols, 1.f, 0, 0, 0, 0});
        }
        AG_TRY(muon::check_overlap(ranges));
        const muon::Rule rule = {0.f, 0.f, 0.f, 0};
        return dtype == AG_F32 ? muon::run<float>(dev, list, rule, steps) : muon::run<__nv_bfloat16>(dev, list, rule, steps);
    } catch (const std::bad_alloc &) {
        return fail(AG_ERR_OOM, "newton_schulz: out of host memory");
    }
}

int ag_muon_update(ag_device *dev, ag_dtype dtype, int32_t n, const ag_muon_matrix *matrices, float lr, float momentum,
                   int nesterov, float weight_decay, int32_t steps) {
    AG_ENTER(dev);
    AG_TRY(muon::check_call(dtype, n, matrices, steps));
    AG_REQUIRE(momentum >= 0.f && momentum <= 3e38f, AG_ERR_INVALID, "muon_update: momentum must not be negative");
    try {
        std::vector<muon::Matrix> list;
        std::vector<muon::Range> ranges;
        for (int32_t i = 0; i < n; ++i) {
            const ag_muon_matrix &m = matrices[i];
            AG_TRY(muon::check_size(m.rows, m.cols));
            AG_REQUIRE(m.w && m.g && m.v, AG_ERR_INVALID, "muon_update: null pointer");
            const uintptr_t count = (uintptr_t)(m.rows * m.cols), bytes = count * dtype_size(dtype);
            ranges.push_back({(uintptr_t)m.g, (uintptr_t)m.g + bytes, false, i, false});
            ranges.push_back({(uintptr_t)m.w, (uintptr_t)m.w + bytes, true, i, false});
            ranges.push_back({(uintptr_t)m.v, (uintptr_t)m.v + count * 4, true, i, false});
            list.push_back({m.g, m.w, m.v, m.rows, m.cols, m.scale, 0, 0, 0, 0});
        }
        AG_TRY(muon::check_overlap(ranges));
        const muon::Rule rule = {lr, momentum, weight_decay, nesterov ? 1 : 0};
        return dtype == AG_F32 ? muon::run<float>(dev, list, rule, steps) : muon::run<__nv_bfloat16>(dev, list, rule, steps);
    } catch (const std::bad_alloc &) {
        return fail(AG_ERR_OOM, "muon_update: out of host memory");
    }
}

}  // extern "C"
