// Newton-Schulz orthogonalisation of gradient matrices, and Muon's parameter update around it.
//
// With x = u / norm(u), as n x m with n <= m (the transpose of a taller u), a step is
//   a = x x^T,  b = B a + C a a,  x <- A x + b x,   (A, B, C) = (3.4445, -4.7750, 2.0315),
// which maps every singular value s to A s + B s^3 + C s^5 and keeps the singular vectors.
#include "common.cuh"

#include <algorithm>
#include <vector>

namespace ag {
namespace muon {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int64_t kMostShort = 16384, kMostLong = 1 << 20;
constexpr int kMostMatrices = 4096, kMostSteps = 20;
constexpr int kNormParts = 64;   // partial sums of squares of a matrix

// One matrix of a call.
struct Matrix {
    const void *g;
    void *o;        // result, or the weight that it updates
    float *v;       // momentum, or null
    int64_t rows, cols;
    float scale;
};

// The update's scalars.
struct Rule {
    float lr, momentum, decay;
    int nesterov;
};

// u from the gradient and, for an update, the momentum after it.
template <class T>
__device__ __forceinline__ float direction(const Matrix &m, const Rule &r, int64_t i) {
    const float g = to_f32(reinterpret_cast<const T *>(m.g)[i]);
    if (m.v == nullptr) return g;
    const float v = m.v[i];
    return r.nesterov ? fmaf(r.momentum, v, g) : v;
}

// v = momentum * v + g, and partial sums of u^2 in f64 (u^2 itself can exceed f32's range).
template <class T>
__global__ void __launch_bounds__(256) momentum_kernel(const Matrix m, const Rule r, double *parts) {
    __shared__ double scratch[8];
    let_dependents_launch();
    dependency_wait();
    const int64_t n = m.rows * m.cols;
    double s = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        if (m.v != nullptr) m.v[i] = __fadd_rn(__fmul_rn(r.momentum, m.v[i]), to_f32(reinterpret_cast<const T *>(m.g)[i]));
        const double u = direction<T>(m, r, i);
        s += u * u;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) s += scratch[i];
        parts[blockIdx.x] = s;
    }
}

// x = u / norm(u), transposed where u is taller than wide.  A norm of zero gives zeros, one that is not finite NaN.
template <class T>
__global__ void __launch_bounds__(256) scale_kernel(const Matrix m, const Rule r, const double *parts, float *x) {
    let_dependents_launch();
    dependency_wait();
    double s = 0;
    for (int i = 0; i < kNormParts; ++i) s += parts[i];
    const double inv = s == 0 ? 0. : isfinite(s) ? 1. / sqrt(s) : (double)NAN;
    const bool flip = m.rows > m.cols;
    const int64_t n = m.rows * m.cols, wide = flip ? m.rows : m.cols;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / wide, col = i - row * wide;
        x[i] = (float)(direction<T>(m, r, flip ? col * m.cols + row : i) * inv);
    }
}

// c = p * (a . b) + q * e, row-major f32: a [M, K], b [K, N], or [N, K] when bt; 32 x 32 outputs a CTA.
__global__ void __launch_bounds__(256)
    product_kernel(const float *a, const float *b, bool bt, int M, int N, int K, float p, float q, const float *e, float *c) {
    __shared__ float sa[32][33], sb[32][33];
    let_dependents_launch();
    dependency_wait();
    const int m0 = blockIdx.y * 32, n0 = blockIdx.x * 32, tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int k0 = 0; k0 < K; k0 += 32) {
        for (int i = ty; i < 32; i += 8) {
            sa[i][tx] = m0 + i < M && k0 + tx < K ? a[(int64_t)(m0 + i) * K + k0 + tx] : 0.f;
            if (bt)
                sb[tx][i] = n0 + i < N && k0 + tx < K ? b[(int64_t)(n0 + i) * K + k0 + tx] : 0.f;
            else
                sb[i][tx] = n0 + tx < N && k0 + i < K ? b[(int64_t)(k0 + i) * N + n0 + tx] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 32; ++k)
            for (int j = 0; j < 4; ++j) acc[j] = fmaf(sa[ty + 8 * j][k], sb[k][tx], acc[j]);
        __syncthreads();
    }
    for (int j = 0; j < 4; ++j) {
        const int64_t i = (int64_t)(m0 + ty + 8 * j) * N + n0 + tx;
        if (m0 + ty + 8 * j < M && n0 + tx < N) c[i] = q != 0.f ? fmaf(p, acc[j], q * e[i]) : p * acc[j];
    }
}

// o = x, or w = (1 - lr * decay) * w - lr * scale * x.
template <class T>
__global__ void __launch_bounds__(256) store_kernel(const Matrix m, const Rule r, const float *x) {
    let_dependents_launch();
    dependency_wait();
    const bool flip = m.rows > m.cols;
    const int64_t n = m.rows * m.cols, wide = flip ? m.rows : m.cols;
    T *o = reinterpret_cast<T *>(m.o);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / m.cols, col = i - row * m.cols;
        const float v = flip ? x[col * wide + row] : x[i];
        o[i] = from_f32<T>(m.v == nullptr ? v : fmaf(-r.lr * m.scale, v, (1.f - r.lr * r.decay) * to_f32(o[i])));
    }
}

template <class T>
int run(ag_device *dev, const std::vector<Matrix> &matrices, const Rule &rule, int steps) {
    int64_t most = 0;
    for (const Matrix &m : matrices) {
        const int64_t n = std::min(m.rows, m.cols);
        most = std::max(most, 2 * m.rows * m.cols + 2 * n * n);
    }
    void *ws;
    AG_TRY(workspace(dev, kNormParts * sizeof(double) + (size_t)most * sizeof(float), &ws));
    double *parts = (double *)ws;
    for (const Matrix &mat : matrices) {
        const int64_t n = std::min(mat.rows, mat.cols), m = std::max(mat.rows, mat.cols);
        float *x = (float *)(parts + kNormParts), *y = x + n * m, *a = y + n * m, *b = a + n * n;
        const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(n * m, 256), 8 * dev->sm_count);
        AG_TRY(launch_dependent(dev, momentum_kernel<T>, dim3(kNormParts), 256, 0, mat, rule, parts));
        AG_TRY(launch_dependent(dev, scale_kernel<T>, dim3(grid), 256, 0, mat, rule, (const double *)parts, x));
        const dim3 square((unsigned)ceil_div(n, 32), (unsigned)ceil_div(n, 32)), wide((unsigned)ceil_div(m, 32), square.y);
        for (int s = 0; s < steps; ++s) {
            AG_TRY(launch_dependent(dev, product_kernel, square, 256, 0, (const float *)x, (const float *)x, true, (int)n, (int)n,
                                    (int)m, 1.f, 0.f, (const float *)nullptr, a));
            AG_TRY(launch_dependent(dev, product_kernel, square, 256, 0, (const float *)a, (const float *)a, false, (int)n, (int)n,
                                    (int)n, kC, kB, (const float *)a, b));
            AG_TRY(launch_dependent(dev, product_kernel, wide, 256, 0, (const float *)b, (const float *)x, false, (int)n, (int)m,
                                    (int)n, 1.f, kA, (const float *)x, y));
            std::swap(x, y);
        }
        AG_TRY(launch_dependent(dev, store_kernel<T>, dim3(grid), 256, 0, mat, rule, (const float *)x));
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
            list.push_back({m.g, m.o, nullptr, m.rows, m.cols, 1.f});
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
            list.push_back({m.g, m.w, m.v, m.rows, m.cols, m.scale});
        }
        AG_TRY(muon::check_overlap(ranges));
        const muon::Rule rule = {lr, momentum, weight_decay, nesterov ? 1 : 0};
        return dtype == AG_F32 ? muon::run<float>(dev, list, rule, steps) : muon::run<__nv_bfloat16>(dev, list, rule, steps);
    } catch (const std::bad_alloc &) {
        return fail(AG_ERR_OOM, "muon_update: out of host memory");
    }
}

}  // extern "C"
