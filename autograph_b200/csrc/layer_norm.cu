// Layer norm over the rows of a [rows, cols] matrix, forward and backward.
//
// Forward, per row:    mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps),
//                      y = (x - mean) * rstd * weight + bias.
// Backward, with hat = (x - mean) * rstd and d = dy * weight:
//                      dx = rstd * (d - sum d / n - hat * sum(d * hat) / n),
//                      dweight = sum over rows of dy * hat,  dbias = sum over rows of dy.
// Everything is computed in f32 and rounded once where it is stored; mean and rstd are f32 tensors.
#include "common.cuh"

namespace ag {
namespace norm {

// Sum over the CTA's threads, to all of them; the same order on every run.
__device__ __forceinline__ float cta_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int warp = threadIdx.x / 32, warps = blockDim.x / 32;
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[warp] = v;
    __syncthreads();
    float s = 0.f;
    for (int i = 0; i < warps; ++i) s += scratch[i];
    return s;
}

template <class T>
__global__ void __launch_bounds__(256)
    layer_norm_kernel(const T *x, const T *weight, const T *bias, int64_t rows, int64_t cols, float eps, T *y, float *mean_out,
                      float *rstd_out) {
    __shared__ float scratch[8];
    let_dependents_launch();
    dependency_wait();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols;
        float s = 0.f;
        for (int64_t i = threadIdx.x; i < cols; i += 256) s += to_f32(xr[i]);
        const float mean = cta_sum(s, scratch) / (float)cols;
        s = 0.f;
        for (int64_t i = threadIdx.x; i < cols; i += 256) {
            const float c = to_f32(xr[i]) - mean;
            s += c * c;
        }
        const float rstd = 1.f / sqrtf(cta_sum(s, scratch) / (float)cols + eps);
        for (int64_t i = threadIdx.x; i < cols; i += 256) {
            float v = (to_f32(xr[i]) - mean) * rstd;
            if (weight != nullptr) v *= to_f32(weight[i]);
            if (bias != nullptr) v += to_f32(bias[i]);
            y[row * cols + i] = from_f32<T>(v);
        }
        if (threadIdx.x == 0) {
            if (mean_out != nullptr) mean_out[row] = mean;
            if (rstd_out != nullptr) rstd_out[row] = rstd;
        }
    }
}

template <class T>
__global__ void __launch_bounds__(256)
    layer_norm_backward_kernel(const T *x, const T *weight, const float *mean, const float *rstd, const T *dy, int64_t rows,
                               int64_t cols, T *dx) {
    __shared__ float scratch[8];
    let_dependents_launch();
    dependency_wait();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols, *dr = dy + row * cols;
        const float m = mean[row], r = rstd[row];
        float along = 0.f, across = 0.f;
        for (int64_t i = threadIdx.x; i < cols; i += 256) {
            const float hat = (to_f32(xr[i]) - m) * r;
            float d = to_f32(dr[i]);
            if (weight != nullptr) d *= to_f32(weight[i]);
            along += d;
            across += d * hat;
        }
        along = cta_sum(along, scratch) / (float)cols;
        across = cta_sum(across, scratch) / (float)cols;
        for (int64_t i = threadIdx.x; i < cols; i += 256) {
            const float hat = (to_f32(xr[i]) - m) * r;
            float d = to_f32(dr[i]);
            if (weight != nullptr) d *= to_f32(weight[i]);
            dx[row * cols + i] = from_f32<T>(r * (d - along - hat * across));
        }
    }
}

// A column's sums over all rows: a CTA takes 32 columns, its warps every eighth row.
template <class T>
__global__ void __launch_bounds__(256)
    layer_norm_columns_kernel(const T *x, const float *mean, const float *rstd, const T *dy, int64_t rows, int64_t cols,
                              float beta, T *dweight, T *dbias) {
    __shared__ float sums[2][8][33];
    let_dependents_launch();
    dependency_wait();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < cols; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + lane;
        float w = 0.f, b = 0.f;
        if (c < cols)
            for (int64_t r = warp; r < rows; r += 8) {
                const float d = to_f32(dy[r * cols + c]);
                w += d * ((to_f32(x[r * cols + c]) - mean[r]) * rstd[r]);
                b += d;
            }
        sums[0][warp][lane] = w;
        sums[1][warp][lane] = b;
        __syncthreads();
        if (warp < 2 && c < cols) {
            T *out = warp == 0 ? dweight : dbias;
            float s = 0.f;
            for (int i = 0; i < 8; ++i) s += sums[warp][i][lane];
            if (out != nullptr) out[c] = from_f32<T>(beta != 0.f ? beta * to_f32(out[c]) + s : s);
        }
        __syncthreads();
    }
}

template <class T>
int forward(ag_device *dev, const T *x, const T *weight, const T *bias, int64_t rows, int64_t cols, float eps, T *y,
            float *mean, float *rstd) {
    if (rows == 0) return AG_OK;
    const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : 1 << 20);
    return launch_dependent(dev, layer_norm_kernel<T>, dim3(grid), 256, 0, x, weight, bias, rows, cols, eps, y, mean, rstd);
}

template <class T>
int backward(ag_device *dev, const T *x, const T *weight, const float *mean, const float *rstd, const T *dy, int64_t rows,
             int64_t cols, T *dx, float beta, T *dweight, T *dbias) {
    if (rows > 0 && dx != nullptr) {
        const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : 1 << 20);
        AG_TRY(launch_dependent(dev, layer_norm_backward_kernel<T>, dim3(grid), 256, 0, x, weight, mean, rstd, dy, rows, cols, dx));
    }
    if (dweight == nullptr && dbias == nullptr) return AG_OK;
    const int64_t blocks = ceil_div(cols, 32);
    return launch_dependent(dev, layer_norm_columns_kernel<T>, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), 256, 0,
                            x, mean, rstd, dy, rows, cols, beta, dweight, dbias);
}

static int check_sizes(ag_dtype dtype, int64_t rows, int64_t cols) {
    AG_REQUIRE(is_float_dtype(dtype), AG_ERR_DTYPE, "layer_norm: dtype %d unimplemented", (int)dtype);
    AG_REQUIRE(rows >= 0, AG_ERR_SHAPE, "layer_norm: negative number of rows");
    AG_REQUIRE(cols > 0, AG_ERR_SHAPE, "layer_norm: a row needs at least one value");
    AG_REQUIRE(rows == 0 || cols <= INT64_MAX / 8 / rows, AG_ERR_SHAPE, "layer_norm: size overflows");
    return AG_OK;
}

// Whether two ranges of `na` and `nb` bytes share a byte.
static bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t p = (uintptr_t)a, q = (uintptr_t)b;
    return a != nullptr && b != nullptr && p < q + (uintptr_t)nb && q < p + (uintptr_t)na;
}

}  // namespace norm
}  // namespace ag

using namespace ag;

extern "C" {

int ag_layer_norm_forward(ag_device *dev, ag_dtype dtype, const void *x, const void *weight, const void *bias, int64_t rows,
                          int64_t cols, float eps, void *y, float *mean, float *rstd) {
    AG_ENTER(dev);
    AG_TRY(norm::check_sizes(dtype, rows, cols));
    AG_REQUIRE(eps > 0.f && eps <= 3.4e38f, AG_ERR_INVALID, "layer_norm: eps must be positive and finite");
    AG_REQUIRE(rows == 0 || (x && y), AG_ERR_INVALID, "layer_norm: null pointer");
    const int64_t n = rows * cols * (int64_t)dtype_size(dtype);
    AG_REQUIRE(x == y || !norm::overlap(x, n, y, n), AG_ERR_INVALID, "layer_norm: y must be x or not overlap it");
    if (dtype == AG_F32)
        return norm::forward(dev, (const float *)x, (const float *)weight, (const float *)bias, rows, cols, eps, (float *)y, mean,
                             rstd);
    return norm::forward(dev, (const __nv_bfloat16 *)x, (const __nv_bfloat16 *)weight, (const __nv_bfloat16 *)bias, rows, cols, eps,
                         (__nv_bfloat16 *)y, mean, rstd);
}

int ag_layer_norm_backward(ag_device *dev, ag_dtype dtype, const void *x, const void *weight, const float *mean,
                           const float *rstd, const void *dy, int64_t rows, int64_t cols, void *dx, float beta, void *dweight,
                           void *dbias) {
    AG_ENTER(dev);
    AG_TRY(norm::check_sizes(dtype, rows, cols));
    AG_REQUIRE(rows == 0 || (x && mean && rstd && dy), AG_ERR_INVALID, "layer_norm: null pointer");
    const int64_t es = (int64_t)dtype_size(dtype), n = rows * cols * es;
    AG_REQUIRE(!norm::overlap(dx, n, x, n) && !norm::overlap(dx, n, dy, n), AG_ERR_INVALID,
               "layer_norm: dx must not overlap x or dy");
    if (dtype == AG_F32)
        return norm::backward(dev, (const float *)x, (const float *)weight, mean, rstd, (const float *)dy, rows, cols, (float *)dx,
                              beta, (float *)dweight, (float *)dbias);
    return norm::backward(dev, (const __nv_bfloat16 *)x, (const __nv_bfloat16 *)weight, mean, rstd, (const __nv_bfloat16 *)dy, rows,
                          cols, (__nv_bfloat16 *)dx, beta, (__nv_bfloat16 *)dweight, (__nv_bfloat16 *)dbias);
}

}  // extern "C"
