// Layer norm over the rows of a [rows, cols] matrix, forward and backward.
//
// Forward, per row:    mean = sum x / n,  var = sum (x - mean)^2 / n,  rstd = 1 / sqrt(var + eps),
//                      y = (x - mean) * rstd * weight + bias.
// Backward, with hat = (x - mean) * rstd and d = dy * weight:
//                      dx = rstd * (d - sum d / n - hat * sum(d * hat) / n),
//                      dweight = sum over rows of dy * hat,  dbias = sum over rows of dy.
// Everything is computed in f32 and rounded once where it is stored; mean and rstd are f32 tensors.
//
// Both directions are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx, once each.  A row
// is held in registers by a group of G threads (a warp, or a whole CTA), up to 64 values a thread, so that its statistics, and
// the differences from its mean that the variance is a sum of, cost no second read.  Rows that start on 16 bytes and are
// whole vectors move 16 bytes a load, others one value, neighbouring lanes on neighbouring values either way.
// A backward group takes every `groups`-th row and adds dy * hat and dy of its columns in registers as it goes; the CTAs'
// sums are added in the order of the CTAs, by the CTA that finishes last or, where there is more to add, by a second
// kernel.  Longer rows take two kernels that read them again.
// Of the measured copy bandwidth, 65536 x 1024: f32 forward 0.95 (87 us), backward 0.90 (137), bf16 0.79 (52) and 0.70 (88: a
// quarter of the warps, whose 128 registers hold row and sums); 256 x 25088 f32 forward 0.43 (18 us: one row an SM at a time).
//
// Products that feed a sum are written as __fmul_rn or fmaf: left to the compiler, it fuses them one way in the loop for calls
// that ask for the statistics, or for one gradient, and another way in the next, and the same values would give other bits.
#include "common.cuh"

namespace ag {
namespace norm {

// VEC neighbouring values of T as they lie in memory.
template <class T, int VEC>
struct Pack;
template <>
struct Pack<float, 4> {
    float4 v;
    __device__ __forceinline__ float get(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
    __device__ __forceinline__ void set(const float (&x)[4]) { v = make_float4(x[0], x[1], x[2], x[3]); }
};
template <>
struct Pack<__nv_bfloat16, 8> {
    uint4 v;
    __device__ __forceinline__ float get(int i) const {
        const uint32_t w = i / 2 == 0 ? v.x : i / 2 == 1 ? v.y : i / 2 == 2 ? v.z : v.w;
        return __uint_as_float(i % 2 ? w & 0xffff0000u : w << 16);
    }
    __device__ __forceinline__ void set(const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&p);
        }
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <class T>
struct Pack<T, 1> {
    T v;
    __device__ __forceinline__ float get(int) const { return to_f32(v); }
    __device__ __forceinline__ void set(const float (&x)[1]) { v = from_f32<T>(x[0]); }
};

// Sums over a group's threads, to all of them; the same order on every run.  A group is a warp or the CTA; the CTA's scratch
// holds N floats a warp.
template <int G, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr (G > 32) {
        const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
        __syncthreads();   // the sums before have been read
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) scratch[i * 32 + warp] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lane < G / 32 ? scratch[i * 32 + lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
}

template <int G>
constexpr int threads_of() { return G == 32 ? 256 : G; }

// From the sums of the differences from a first mean, and of their squares: the mean, put right by what the differences leave, and
// 1 / sqrt(variance + eps).  The first mean is off by the roundings of a sum of n values, 1e-5 of it for 25088 equal ones; what
// these differences leave is off by the same share of them, so that of equal values the mean is that value and y is the bias.
// us with and without: bf16 65536 x 1024 52 to 55 and 51.8, 2048 x 25088 55 and 51, f32 256 x 25088 18.1 and 17.1.
__device__ __forceinline__ float finish_statistics(const float (&e)[2], float n, float eps, float &mean) {
    const float left = __fdiv_rn(e[0], n), var = fmaf(-left, left, __fdiv_rn(e[1], n));
    mean += left;
    return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);   // NaN stays
}

// Rows in registers: NC packs of VEC values a thread.
template <class T, int VEC, int G, int NC>
__global__ void __launch_bounds__(threads_of<G>())
    layer_norm_kernel(const T *x, const T *weight, const T *bias, int64_t rows, int cols, float eps, T *y, float *mean_out,
                      float *rstd_out) {
    using P = Pack<T, VEC>;
    __shared__ float scratch[64];
    let_dependents_launch();
    dependency_wait();
    constexpr int GROUPS = threads_of<G>() / G;
    const int t = threadIdx.x % G;
    const float n = (float)cols;
    for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; row < rows; row += (int64_t)gridDim.x * GROUPS) {
        const T *xr = x + row * cols;
        P p[NC];
        float s[1] = {0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * G + t) * VEC;
            if (col < cols) p[c] = *reinterpret_cast<const P *>(xr + col);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if ((c * G + t) * VEC < cols)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[0] += p[c].get(i);
        group_sum<G>(s, scratch);
        float mean = __fdiv_rn(s[0], n);
        float e[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
            if ((c * G + t) * VEC < cols)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = p[c].get(i) - mean;
                    e[0] += d;
                    e[1] = fmaf(d, d, e[1]);
                }
        group_sum<G>(e, scratch);
        const float rstd = finish_statistics(e, n, eps, mean);
        T *yr = y + row * cols;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * G + t) * VEC;
            if (col < cols) {
                float o[VEC];
                P w, b;
                if (weight != nullptr) w = *reinterpret_cast<const P *>(weight + col);
                if (bias != nullptr) b = *reinterpret_cast<const P *>(bias + col);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    o[i] = fmaf(__fmul_rn(p[c].get(i) - mean, rstd), weight != nullptr ? w.get(i) : 1.f,
                                bias != nullptr ? b.get(i) : 0.f);
                }
                P q;
                q.set(o);
                *reinterpret_cast<P *>(yr + col) = q;
            }
        }
        if (t == 0) {
            if (mean_out != nullptr) mean_out[row] = mean;
            if (rstd_out != nullptr) rstd_out[row] = rstd;
        }
    }
}

// Rows that no registers hold: read three times.
template <class T>
__global__ void __launch_bounds__(1024)
    layer_norm_long_kernel(const T *x, const T *weight, const T *bias, int64_t rows, int64_t cols, float eps, T *y,
                           float *mean_out, float *rstd_out) {
    __shared__ float scratch[64];
    let_dependents_launch();
    dependency_wait();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols;
        float s[1] = {0.f};
#pragma unroll 8
        for (int64_t i = threadIdx.x; i < cols; i += 1024) s[0] += to_f32(xr[i]);
        group_sum<1024>(s, scratch);
        float mean = __fdiv_rn(s[0], (float)cols);
        float e[2] = {0.f, 0.f};
#pragma unroll 8
        for (int64_t i = threadIdx.x; i < cols; i += 1024) {
            const float d = to_f32(xr[i]) - mean;
            e[0] += d;
            e[1] = fmaf(d, d, e[1]);
        }
        group_sum<1024>(e, scratch);
        const float rstd = finish_statistics(e, (float)cols, eps, mean);
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < cols; i += 1024) {
            const float w = weight != nullptr ? to_f32(weight[i]) : 1.f, b = bias != nullptr ? to_f32(bias[i]) : 0.f;
            y[row * cols + i] = from_f32<T>(fmaf(__fmul_rn(to_f32(xr[i]) - mean, rstd), w, b));
        }
        if (threadIdx.x == 0) {
            if (mean_out != nullptr) mean_out[row] = mean;
            if (rstd_out != nullptr) rstd_out[row] = rstd;
        }
    }
}

// Where the CTAs' column sums go: partial [CTA][2][cols], added by the CTA that arrives last (arrivals: a zero, and zero
// again afterwards) or, where that is null, by columns_kernel.
template <class T>
struct Columns {
    float *partial;
    int *arrivals;
    float beta;
    T *dweight, *dbias;
};

template <class T>
__device__ __forceinline__ void store_column(const Columns<T> &c, int cols, int i, float s) {
    T *out = i < cols ? c.dweight : c.dbias;
    if (out == nullptr) return;
    out += i < cols ? i : i - cols;
    *out = from_f32<T>(c.beta != 0.f ? fmaf(c.beta, to_f32(*out), s) : s);
}

template <class T, int VEC, int G, int NC>
__global__ void __launch_bounds__(threads_of<G>())
    layer_norm_backward_kernel(const T *x, const T *weight, const float *mean, const float *rstd, const T *dy, int64_t rows,
                               int cols, T *dx, const Columns<T> out) {
    using P = Pack<T, VEC>;
    constexpr int THREADS = threads_of<G>(), GROUPS = THREADS / G;
    // the groups' sums of G == 32, one of the two gradients at a time
    __shared__ float scratch[G == 32 ? GROUPS * 32 * NC * VEC : 64];
    __shared__ int last;
    let_dependents_launch();
    dependency_wait();
    const int t = threadIdx.x % G;
    const float n = (float)cols;
    float dw[NC * VEC], db[NC * VEC];
#pragma unroll
    for (int i = 0; i < NC * VEC; ++i) dw[i] = db[i] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / G; row < rows; row += (int64_t)gridDim.x * GROUPS) {
        P px[NC], pd[NC];
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * G + t) * VEC;
            if (col < cols) {
                px[c] = *reinterpret_cast<const P *>(x + row * cols + col);
                pd[c] = *reinterpret_cast<const P *>(dy + row * cols + col);
            }
        }
        const float m = mean[row], r = rstd[row];
        float s[2] = {0.f, 0.f};   // of d, of d * hat
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * G + t) * VEC;
            if (col < cols) {
                P w;
                if (weight != nullptr) w = *reinterpret_cast<const P *>(weight + col);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float hat = __fmul_rn(px[c].get(i) - m, r);
                    float d = pd[c].get(i);
                    dw[c * VEC + i] = fmaf(d, hat, dw[c * VEC + i]);
                    db[c * VEC + i] += d;
                    if (weight != nullptr) d = __fmul_rn(d, w.get(i));
                    s[0] += d;
                    s[1] = fmaf(d, hat, s[1]);
                }
            }
        }
        if (dx == nullptr) continue;
        group_sum<G>(s, scratch);
        const float along = __fdiv_rn(s[0], n), across = __fdiv_rn(s[1], n);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int col = (c * G + t) * VEC;
            if (col < cols) {
                P w;
                if (weight != nullptr) w = *reinterpret_cast<const P *>(weight + col);
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float hat = __fmul_rn(px[c].get(i) - m, r);
                    float d = pd[c].get(i);
                    if (weight != nullptr) d = __fmul_rn(d, w.get(i));
                    o[i] = r * fmaf(-hat, across, d - along);
                }
                P q;
                q.set(o);
                *reinterpret_cast<P *>(dx + row * cols + col) = q;
            }
        }
    }
    if (out.partial == nullptr) return;
    float *mine = out.partial + (int64_t)blockIdx.x * 2 * cols;
    if constexpr (G == 32) {
        // the CTA's warps, in order
        const int warp = threadIdx.x / 32;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NC * VEC; ++i) scratch[(warp * NC * VEC + i) * 32 + t] = half == 0 ? dw[i] : db[i];
            __syncthreads();
            for (int k = threadIdx.x; k < NC * VEC * 32; k += THREADS) {
                const int i = k / 32, lane = k % 32, col = (i / VEC * 32 + lane) * VEC + i % VEC;
                float s = 0.f;
#pragma unroll
                for (int w = 0; w < GROUPS; ++w) s += scratch[w * NC * VEC * 32 + k];
                if (col < cols) __stcg(mine + half * cols + col, s);
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int col = (c * G + t) * VEC + i;
                if (col < cols) {
                    __stcg(mine + col, dw[c * VEC + i]);
                    __stcg(mine + cols + col, db[c * VEC + i]);
                }
            }
    }
    if (out.arrivals == nullptr) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        last = atomicAdd(out.arrivals, 1) == (int)gridDim.x - 1;
        if (last) *out.arrivals = 0;
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    for (int i = threadIdx.x; i < 2 * cols; i += THREADS) {
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < (int)gridDim.x; ++k) s += __ldcg(out.partial + (int64_t)k * 2 * cols + i);
        store_column(out, cols, i, s);
    }
}

// The sums of `parts` CTAs: a CTA takes 32 columns of [2][cols], a warp every eighth part; a part-less call writes beta times
// what there was.
template <class T>
__global__ void __launch_bounds__(256) columns_kernel(int parts, int cols, const Columns<T> out) {
    __shared__ float sums[8][33];
    let_dependents_launch();
    dependency_wait();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t i = (int64_t)blockIdx.x * 32 + lane;
    float s = 0.f;
    if (i < 2 * (int64_t)cols)
#pragma unroll 8
        for (int k = warp; k < parts; k += 8) s += out.partial[(int64_t)k * 2 * cols + i];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < 2 * (int64_t)cols) {
        s = 0.f;
        for (int w = 0; w < 8; ++w) s += sums[w][lane];
        store_column(out, cols, (int)i, s);
    }
}

// Rows that no registers hold, VEC values at a time.
template <class T, int VEC>
__global__ void __launch_bounds__(1024)
    layer_norm_long_backward_kernel(const T *x, const T *weight, const float *mean, const float *rstd, const T *dy, int64_t rows,
                                    int64_t cols, T *dx) {
    using P = Pack<T, VEC>;
    __shared__ float scratch[64];
    let_dependents_launch();
    dependency_wait();
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *xr = x + row * cols, *dr = dy + row * cols;
        const float m = mean[row], r = rstd[row];
        float s[2] = {0.f, 0.f};
#pragma unroll 2
        for (int64_t i = threadIdx.x * VEC; i < cols; i += 1024 * VEC) {
            const P px = *reinterpret_cast<const P *>(xr + i), pd = *reinterpret_cast<const P *>(dr + i);
            P w;
            if (weight != nullptr) w = *reinterpret_cast<const P *>(weight + i);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float d = pd.get(k);
                if (weight != nullptr) d = __fmul_rn(d, w.get(k));
                s[0] += d;
                s[1] = fmaf(d, __fmul_rn(px.get(k) - m, r), s[1]);
            }
        }
        group_sum<1024>(s, scratch);
        const float along = s[0] / (float)cols, across = s[1] / (float)cols;
#pragma unroll 2
        for (int64_t i = threadIdx.x * VEC; i < cols; i += 1024 * VEC) {
            const P px = *reinterpret_cast<const P *>(xr + i), pd = *reinterpret_cast<const P *>(dr + i);
            P w, q;
            if (weight != nullptr) w = *reinterpret_cast<const P *>(weight + i);
            float o[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                float d = pd.get(k);
                if (weight != nullptr) d = __fmul_rn(d, w.get(k));
                o[k] = r * fmaf(-__fmul_rn(px.get(k) - m, r), across, d - along);
            }
            q.set(o);
            *reinterpret_cast<P *>(dx + row * cols + i) = q;
        }
    }
}

// Column sums of long rows: a CTA takes 256 * VEC columns and one of gridDim.y slices of the rows.
template <class T, int VEC>
__global__ void __launch_bounds__(256)
    layer_norm_long_columns_kernel(const T *x, const float *mean, const float *rstd, const T *dy, int64_t rows, int64_t cols,
                                   float *partial) {
    using P = Pack<T, VEC>;
    let_dependents_launch();
    dependency_wait();
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
    if (c >= cols) return;
    float w[VEC], b[VEC];
#pragma unroll
    for (int k = 0; k < VEC; ++k) w[k] = b[k] = 0.f;
#pragma unroll 4
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const P px = *reinterpret_cast<const P *>(x + r * cols + c), pd = *reinterpret_cast<const P *>(dy + r * cols + c);
        const float m = mean[r], rs = rstd[r];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float d = pd.get(k);
            w[k] = fmaf(d, __fmul_rn(px.get(k) - m, rs), w[k]);
            b[k] += d;
        }
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k) {
        partial[(int64_t)blockIdx.y * 2 * cols + c + k] = w[k];
        partial[(int64_t)blockIdx.y * 2 * cols + cols + c + k] = b[k];
    }
}

// ---- host ------------------------------------------------------------------------------------------

template <class T>
struct Forward {
    ag_device *dev;
    const T *x, *weight, *bias;
    int64_t rows, cols;
    float eps;
    T *y;
    float *mean, *rstd;
    template <int VEC, int G, int NC>
    int run() const {
        constexpr int GROUPS = threads_of<G>() / G;
        const int64_t blocks = ceil_div(rows, GROUPS), most = (int64_t)dev->sm_count * (2048 / threads_of<G>());
        return launch_dependent(dev, layer_norm_kernel<T, VEC, G, NC>, dim3((unsigned)(blocks < most ? blocks : most)),
                                threads_of<G>(), 0, x, weight, bias, rows, (int)cols, eps, y, mean, rstd);
    }
};

template <class T>
struct Backward {
    ag_device *dev;
    const T *x, *weight;
    const float *mean, *rstd;
    const T *dy;
    int64_t rows, cols;
    T *dx;
    float beta;
    T *dweight, *dbias;
    bool sums() const { return dweight != nullptr || dbias != nullptr; }

    int add_columns(int parts, Columns<T> out) const {
        return launch_dependent(dev, columns_kernel<T>, dim3((unsigned)ceil_div(2 * cols, 32)), 256, 0, parts, (int)cols, out);
    }
    template <int VEC, int G, int NC>
    int run() const {
        constexpr int GROUPS = threads_of<G>() / G;
        auto kernel = layer_norm_backward_kernel<T, VEC, G, NC>;
        static std::atomic<int> resident{0};   // CTAs of an SM
        int per_sm = resident.load(std::memory_order_relaxed);
        if (per_sm == 0) {
            AG_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads_of<G>(), 0));
            if (per_sm < 1) per_sm = 1;
            resident.store(per_sm, std::memory_order_relaxed);
        }
        const int64_t most = (int64_t)dev->sm_count * per_sm, blocks = ceil_div(rows, GROUPS);
        const int grid = (int)(blocks < most ? blocks : most);
        Columns<T> out = {nullptr, nullptr, beta, dweight, dbias};
        if (sums()) {
            void *ws;
            AG_TRY(workspace(dev, (size_t)grid * 2 * cols * sizeof(float), &ws));
            out.partial = (float *)ws;
            if ((int64_t)grid * cols <= kLastAdds) out.arrivals = dev->tile_counters;
        }
        AG_TRY(launch_dependent(dev, kernel, dim3((unsigned)grid), threads_of<G>(), 0, x, weight, mean, rstd, dy, rows, (int)cols,
                                dx, out));
        return out.partial != nullptr && out.arrivals == nullptr ? add_columns(grid, out) : AG_OK;
    }
    static constexpr int64_t kLastAdds = 16384;   // partial sums of each gradient that the last CTA adds
};

// The kernel whose registers hold a row.  With vectors as few threads as can hold it: a row of a warp needs no barrier, and what a
// row of a CTA waits at its barriers other rows of the SM fill.  us, with 256 threads or more from 1024 columns on, and so: bf16
// forward 32768 x 2048 95.6 and 50.1, 16384 x 4096 67.2 and 50.6, 8192 x 8192 73.2 and 53.8, backward 162 and 115.  Single values
// would be many loads of few threads: f32 4093 x 2011 forward 17.8 with 256 threads, 24.1 with 128, backward 27.9 and 36.9.
// (Forward figures here and below are from before the sum of the differences, which adds up to a tenth to either side.)
template <int VEC, class F>
int forward_by_columns(const F &f) {
    const int64_t n = f.cols;
    if (VEC < 8 && n <= 32 * 4) return f.template run<VEC, 32, 4 / (VEC < 8 ? VEC : 1)>();
    if (n <= 32 * 8) return f.template run<VEC, 32, 8 / VEC>();
    if (n <= 32 * 16) return f.template run<VEC, 32, 16 / VEC>();
    if (n <= 32 * 32) return f.template run<VEC, 32, 32 / VEC>();
    if constexpr (VEC > 1) {
        if (n <= 32 * 64) return f.template run<VEC, 32, 64 / VEC>();
        if (n <= 128 * 32) return f.template run<VEC, 128, 32 / VEC>();
        if (n <= 256 * 32) return f.template run<VEC, 256, 32 / VEC>();
        if (n <= 512 * 32) return f.template run<VEC, 512, 32 / VEC>();
        // f32 256 x 25088 from memory 17.1 us with 1024 threads, 20.1 with 512; bf16 2048 x 25088 60 and 46
        return f.template run<VEC, VEC == 8 ? 512 : 1024, VEC == 8 ? 8 : 32 / VEC>();
    }
    if (n <= 256 * 8) return f.template run<VEC, 256, 8 / VEC>();
    if (n <= 256 * 16) return f.template run<VEC, 256, 16 / VEC>();
    if (n <= 512 * 16) return f.template run<VEC, 512, 16 / VEC>();
    if (n <= 1024 * 16) return f.template run<VEC, 1024, 16 / VEC>();
    return f.template run<VEC, 1024, 32 / VEC>();
}
// The sums of the columns take two more registers a value.
template <int VEC, class F>
int backward_by_columns(const F &f) {
    const int64_t n = f.cols;
    if (VEC < 8 && n <= 32 * 4) return f.template run<VEC, 32, 4 / (VEC < 8 ? VEC : 1)>();
    if (n <= 32 * 8) return f.template run<VEC, 32, 8 / VEC>();
    if (n <= 32 * 16) return f.template run<VEC, 32, 16 / VEC>();
    // f32, many rows: 128 registers a thread keep a third of the warps; us, 65536 x 1024 177 and 136, 1000 x 1024 9.1 and 15.9
    // (bf16 86 and 116)
    if (VEC == 4 && n > 512 && n <= 32 * 32 && f.rows >= 16384) return f.template run<VEC, 128, 8 / VEC>();
    if (n <= 32 * 32) return f.template run<VEC, 32, 32 / VEC>();
    if constexpr (VEC == 8) {
        if (n <= 128 * 16) return f.template run<VEC, 128, 16 / VEC>();
        if (n <= 128 * 32) return f.template run<VEC, 128, 32 / VEC>();
        return f.template run<VEC, 256, 32 / VEC>();
    }
    if (VEC > 1 && n <= 128 * 16) return f.template run<VEC, 128, 16 / VEC>();
    if (n <= 256 * 8) return f.template run<VEC, 256, 8 / VEC>();
    if (n <= 256 * 16) return f.template run<VEC, 256, 16 / VEC>();
    return f.template run<VEC, 512, 16 / VEC>();
}

template <class T>
bool vectors(int64_t cols, std::initializer_list<const void *> tensors) {
    if (cols * sizeof(T) % 16 != 0) return false;
    for (const void *p : tensors)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;   // null is
    return true;
}

template <class T>
int forward(ag_device *dev, const T *x, const T *weight, const T *bias, int64_t rows, int64_t cols, float eps, T *y,
            float *mean, float *rstd) {
    if (rows == 0) return AG_OK;
    if (cols > 32768) {
        const int64_t most = 2 * dev->sm_count;
        return launch_dependent(dev, layer_norm_long_kernel<T>, dim3((unsigned)(rows < most ? rows : most)), 1024, 0, x, weight, bias,
                                rows, cols, eps, y, mean, rstd);
    }
    const Forward<T> f = {dev, x, weight, bias, rows, cols, eps, y, mean, rstd};
    return vectors<T>(cols, {x, weight, bias, y}) ? forward_by_columns<16 / sizeof(T)>(f) : forward_by_columns<1>(f);
}

template <class T>
int backward(ag_device *dev, const T *x, const T *weight, const float *mean, const float *rstd, const T *dy, int64_t rows,
             int64_t cols, T *dx, float beta, T *dweight, T *dbias) {
    const Backward<T> f = {dev, x, weight, mean, rstd, dy, rows, cols, dx, beta, dweight, dbias};
    if (dx == nullptr && !f.sums()) return AG_OK;
    if (rows == 0) return f.sums() ? f.add_columns(0, {nullptr, nullptr, beta, dweight, dbias}) : AG_OK;
    if (cols <= 512 * 16)
        return vectors<T>(cols, {x, weight, dy, dx}) ? backward_by_columns<16 / sizeof(T)>(f) : backward_by_columns<1>(f);
    const bool vec = vectors<T>(cols, {x, weight, dy, dx});
    constexpr int V = 16 / sizeof(T);
    if (dx != nullptr) {
        const int64_t most = 2 * dev->sm_count;
        AG_TRY(launch_dependent(dev, vec ? layer_norm_long_backward_kernel<T, V> : layer_norm_long_backward_kernel<T, 1>,
                                dim3((unsigned)(rows < most ? rows : most)), 1024, 0, x, weight, mean, rstd, dy, rows, cols, dx));
    }
    if (!f.sums()) return AG_OK;
    const int64_t blocks = ceil_div(cols, 256 * (vec ? V : 1)), want = ceil_div((int64_t)8 * dev->sm_count, blocks);
    const int slices = (int)(want < rows ? want : rows);
    void *ws;
    AG_TRY(workspace(dev, (size_t)slices * 2 * cols * sizeof(float), &ws));
    AG_TRY(launch_dependent(dev, vec ? layer_norm_long_columns_kernel<T, V> : layer_norm_long_columns_kernel<T, 1>,
                            dim3((unsigned)blocks, (unsigned)slices), 256, 0, x, mean, rstd, dy, rows, cols, (float *)ws));
    return f.add_columns(slices, {(float *)ws, nullptr, beta, dweight, dbias});
}

static int check_sizes(ag_dtype dtype, int64_t rows, int64_t cols) {
    AG_REQUIRE(is_float_dtype(dtype), AG_ERR_DTYPE, "layer_norm: dtype %d unimplemented", (int)dtype);
    AG_REQUIRE(rows >= 0, AG_ERR_SHAPE, "layer_norm: negative number of rows");
    AG_REQUIRE(cols > 0, AG_ERR_SHAPE, "layer_norm: a row needs at least one value");
    AG_REQUIRE(rows == 0 || cols <= INT64_MAX / 8 / rows, AG_ERR_SHAPE, "layer_norm: size overflows");
    AG_REQUIRE(cols < (1 << 30), AG_ERR_LIMIT, "layer_norm: rows of %lld values are beyond the limit", (long long)cols);
    return AG_OK;
}

// An operand of a call: its bytes, none where it is null.
struct Range {
    const void *p;
    int64_t bytes;
};

// Refuses results that share a byte with another operand: rows are written while others' operands are still read.
static int check_overlap(std::initializer_list<Range> results, std::initializer_list<Range> inputs) {
    auto overlap = [](const Range &a, const Range &b) {
        const uintptr_t p = (uintptr_t)a.p, q = (uintptr_t)b.p;
        return a.p != nullptr && b.p != nullptr && a.bytes > 0 && b.bytes > 0 && p < q + (uintptr_t)b.bytes &&
               q < p + (uintptr_t)a.bytes;
    };
    for (auto r = results.begin(); r != results.end(); ++r) {
        for (const Range &i : inputs)
            AG_REQUIRE(!overlap(*r, i), AG_ERR_INVALID, "layer_norm: a result overlaps an operand");
        for (auto other = r + 1; other != results.end(); ++other)
            AG_REQUIRE(!overlap(*r, *other), AG_ERR_INVALID, "layer_norm: the results must not overlap");
    }
    return AG_OK;
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
    const int64_t es = (int64_t)dtype_size(dtype), n = rows * cols * es;
    // y may be x: a row is read before it is written
    AG_TRY(norm::check_overlap({{y, n}, {mean, rows * 4}, {rstd, rows * 4}},
                               {{x == y ? nullptr : x, n}, {weight, cols * es}, {bias, cols * es}}));
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
    AG_TRY(norm::check_overlap({{dx, n}, {dweight, cols * es}, {dbias, cols * es}},
                               {{x, n}, {dy, n}, {weight, cols * es}, {mean, rows * 4}, {rstd, rows * 4}}));
    if (dtype == AG_F32)
        return norm::backward(dev, (const float *)x, (const float *)weight, mean, rstd, (const float *)dy, rows, cols, (float *)dx,
                              beta, (float *)dweight, (float *)dbias);
    return norm::backward(dev, (const __nv_bfloat16 *)x, (const __nv_bfloat16 *)weight, mean, rstd, (const __nv_bfloat16 *)dy, rows,
                          cols, (__nv_bfloat16 *)dx, beta, (__nv_bfloat16 *)dweight, (__nv_bfloat16 *)dbias);
}

}  // extern "C"
