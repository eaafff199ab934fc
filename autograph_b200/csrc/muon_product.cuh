// The Newton-Schulz steps of a list of matrices as one kernel: a CTA per SM that goes through the steps' products phase by
// phase, D = c0 * (P . Q) + c1 * E on tcgen05, with a barrier of the whole grid between two phases.
//
// Matrices live in one workspace as f16 planes.  A value x is held as hi + lo, hi = f16(x * 2^k) and lo = f16 of what
// that leaves: 22 bits, of which a product takes hi.hi + hi.lo + lo.hi.  lo is at most 2^-11 of hi, so what is dropped is at
// most 2^-22 of a product, and lo's own rounding 2^-22 of a value.  bf16 results take the same products: a step's map of the
// singular values has slopes of A at zero, -1.6 at 0.87 and 4 at 1.21, so that what a step rounds off stays or grows.  hi.hi
// alone in three steps of five was 1.0e-3 of the result off beside its rounding of 1.7e-3, in all but three of twenty 1e-2.  The
// scales 2^k are fixed, because the values are bounded: the singular values of every x of the iteration stay below 1.21.
//
// A matrix of R x C is stored in panels of 64 columns, [C / 64][Rp][64] with Rp = R rounded up to 128 and zeros in the
// padding, so that a panel's rows are 128 bytes: the whole workspace is one matrix of 128-byte rows behind one tensor map,
// and a box of 64 rows is a tile of the operand, K-major where the product runs along the columns and MN-major where it
// runs along the rows.
//
// What bounds it.  Small matrices: latency, 7 to 8 us a phase of fifteen (the barrier about 3, the first products 1.7, their
// read-out and stores 1.5; LeNet5's five weights f32 120 us; a CTA a matrix without the barrier took 242).  Large ones: what a
// tile of 128 x 128 reads of L2, 64 KB for 768 cycles of products: 4096 x 4096 bf16 4.3 ms of 2.5 at the measured bf16 rate,
// 1024 x 1024 f32 227 us of 39.  One launch a product, dependent
// or not, cost 10 us each where a phase costs 8.
#pragma once

#include <cuda_fp16.h>

#include "tc_ptx.cuh"

namespace ag {
namespace muon {

// A stored matrix: its first row in the workspace, rows of a panel, rows of a plane.
struct Stored {
    int row, rp, plane;
};

// One matrix of a call.
struct Matrix {
    const void *g;
    void *o;        // result, or the weight that it updates
    float *v;       // momentum, or null
    int64_t rows, cols;
    float scale;
    int part0, parts;   // its partial sums of squares
    int row;            // its first row in the workspace
    int squares;        // first step that is taken on x x^T alone; the number of steps where none is

    __device__ __host__ __forceinline__ int n() const { return (int)(rows < cols ? rows : cols); }
    __device__ __host__ __forceinline__ int wide() const { return (int)(rows < cols ? cols : rows); }
    // x and its successor, n x wide, and the n x n matrices of the steps
    __device__ __host__ __forceinline__ Stored x(int i) const {
        const int rp = (n() + 127) / 128 * 128, plane = (wide() + 63) / 64 * rp;
        return {row + i * 2 * plane, rp, plane};
    }
    __device__ __host__ __forceinline__ Stored square(int i) const {
        const int rp = (n() + 127) / 128 * 128, plane = (n() + 63) / 64 * rp, after = (wide() + 63) / 64 * rp * 4;
        return {row + after + i * 2 * plane, rp, plane};
    }
    __device__ __host__ __forceinline__ int64_t space(int steps) const {   // rows
        const int64_t rp = (n() + 127) / 128 * 128;
        return 4 * rp * ((wide() + 63) / 64) + (squares < steps ? 12 : 4) * rp * ((n() + 63) / 64);
    }
    __device__ __host__ __forceinline__ int phases(int steps) const { return 3 * steps + (squares < steps); }
};

// The update's scalars.
struct Rule {
    float lr, momentum, decay;
    int nesterov;
};

constexpr int kGroup = 32;   // matrices of a launch: a lane each, and its parameters stay below 4 KB
struct Group {
    int n, steps, phases;
    int inside;              // the kernel makes the momenta, norms and planes too
    Rule rule;
    Matrix m[kGroup];
};

// One product.
struct Job {
    Stored p, q, e, d;
    int q_mn;          // q's rows run along the product's depth
    int M, N;          // of D
    int steps;         // 64-k steps
    int symmetric;     // D is: only tiles on and above the diagonal are computed
    int has_e, final;
    float c0, c1;
    float diagonal;    // added to D's
};

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
// Scales of the stored matrices.  |x| <= 1.21, |a| <= 1.46, |b| <= 2.81, |p| <= 3.45 and |p a| <= 1.2 by their norms, f16
// ends at 65504; a product of i + 1 factors p is below 3.45^(i + 1) and has the scale kScaleB / 4^i.
constexpr float kScaleX = 32768.f, kScaleA = 32768.f, kScaleB = 16384.f;

using namespace tc;

// ---- epilogue ------------------------------------------------------------------------------------

__device__ __forceinline__ int64_t at(const Stored &m, int row, int col) {
    return ((int64_t)m.row + (int64_t)(col / 64) * m.rp + row) * 64 + col % 64;
}

// Eight neighbouring values of one row as two f16 planes.
__device__ __forceinline__ void split8(const float (&v)[8], uint4 &hi, uint4 &lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 a = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        const float2 f = __half22float2(a);
        const __half2 b = __floats2half2_rn(v[2 * i] - f.x, v[2 * i + 1] - f.y);
        h[i] = *reinterpret_cast<const uint32_t *>(&a);
        l[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    hi = make_uint4(h[0], h[1], h[2], h[3]);
    lo = make_uint4(l[0], l[1], l[2], l[3]);
}
__device__ __forceinline__ void join8(const uint4 &hi, const uint4 &lo, float (&v)[8]) {
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
        const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&l[i]));
        v[2 * i] = a.x + b.x;
        v[2 * i + 1] = a.y + b.y;
    }
}

// COLS neighbouring values of a row of the result from x: o = x, or w = (1 - lr * decay) * w - lr * scale * x.  All of w is
// loaded before any of it is stored.
template <class T, int COLS>
__device__ __forceinline__ void store_final(const Matrix &m, const Rule &r, int M, int N, int row, int col, const float *x) {
    if (row >= M || col >= N) return;
    T *o = reinterpret_cast<T *>(m.o);
    const bool update = m.v != nullptr;
    const float keep = 1.f - r.lr * r.decay, step = -r.lr * m.scale;
    const bool flip = m.rows > m.cols;
    constexpr int V = 16 / (int)sizeof(T);
    T *p = flip ? o + (int64_t)col * m.cols + row : o + (int64_t)row * m.cols + col;
    if (!flip && col + COLS <= N && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        uint4 w[COLS / V];
#pragma unroll
        for (int b = 0; b < COLS / V; ++b) w[b] = update ? reinterpret_cast<const uint4 *>(p)[b] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int b = 0; b < COLS / V; ++b) {
            uint32_t u[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (V == 4) {
                    const float v = x[b * V + i];
                    u[i] = __float_as_uint(update ? fmaf(step, v, keep * __uint_as_float(u[i])) : v);
                } else {
                    float lo = x[b * V + 2 * i], hi = x[b * V + 2 * i + 1];
                    if (update) {
                        lo = fmaf(step, lo, keep * __uint_as_float(u[i] << 16));
                        hi = fmaf(step, hi, keep * __uint_as_float(u[i] & 0xffff0000u));
                    }
                    const __nv_bfloat162 both = __floats2bfloat162_rn(lo, hi);
                    u[i] = *reinterpret_cast<const uint32_t *>(&both);
                }
            }
            reinterpret_cast<uint4 *>(p)[b] = make_uint4(u[0], u[1], u[2], u[3]);
        }
        return;
    }
    const int64_t next = flip ? m.cols : 1;
    T w[COLS];
    if (update)
#pragma unroll
        for (int i = 0; i < COLS; ++i)
            if (col + i < N) w[i] = p[i * next];
#pragma unroll
    for (int i = 0; i < COLS; ++i)
        if (col + i < N) p[i * next] = from_f32<T>(update ? fmaf(step, x[i], keep * to_f32(w[i])) : x[i]);
}

// Columns col .. col + 31 (col a multiple of 32) of a row of D from their sums, by whole warps whose lanes have neighbouring
// rows.  `mirror`: also the transposed place.  The addend is loaded before the sums are there; what another SM has stored in
// this launch is read past the SM's own cache.
struct Addend {
    uint4 hi[4], lo[4];
};
__device__ __forceinline__ void load_addend(const Job &j, const __half *planes, int row, int col, Addend &a) {
    if (!j.has_e || row >= (j.M + 127) / 128 * 128 || col >= (j.N + 63) / 64 * 64) return;
    const uint4 *e = reinterpret_cast<const uint4 *>(planes + at(j.e, row, col));
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        a.hi[b] = __ldcg(e + b);
        a.lo[b] = __ldcg(e + b + (int64_t)j.e.plane * 8);
    }
}
template <class T>
__device__ __forceinline__ void finish32(const Job &j, const Matrix &m, const Rule &r, __half *planes, int row, int col,
                                         float *v, const Addend &a, bool mirror) {
    const bool in = row < (j.M + 127) / 128 * 128;
    const int cols = (j.N + 63) / 64 * 64;
    if (col >= cols) return;   // 64 columns are all in or all out
    if (j.has_e) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float e8[8];
            join8(a.hi[b], a.lo[b], e8);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[8 * b + i] = fmaf(j.c0, v[8 * b + i], j.c1 * e8[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] *= j.c0;
    }
    if (j.diagonal != 0.f) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (row == col + i && row < j.M) v[i] += j.diagonal;
    }
    if (j.final) {
#pragma unroll
        for (int b = 0; b < 32; b += 8) store_final<T, 8>(m, r, j.M, j.N, row, col + b, v + b);
        return;
    }
    const int64_t plane = (int64_t)j.d.plane * 64;
    __half *d = planes + at(j.d, row, col);
    const int lane = threadIdx.x % 32;
    // the transposed place of rows row, row + 1: an even lane stores their upper halves, an odd one their lower
    uint32_t *t = reinterpret_cast<uint32_t *>(planes + at(j.d, col, row & ~1) + (lane & 1 ? plane : 0));
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = v[8 * b + i];
        uint4 hi, lo;
        split8(x, hi, lo);
        if (in) {
            reinterpret_cast<uint4 *>(d)[b] = hi;
            reinterpret_cast<uint4 *>(d + plane)[b] = lo;
        }
        if (mirror) {
            const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t sel = i % 2 ? 0x7632 : 0x5410;
                const uint32_t both = __byte_perm(h[i / 2], l[i / 2], sel);   // hi | lo << 16
                const uint32_t other = __shfl_xor_sync(0xffffffffu, both, 1);
                const uint32_t pair = lane & 1 ? __byte_perm(other, both, 0x7632) : __byte_perm(both, other, 0x5410);
                if (in) t[(8 * b + i) * 32] = pair;
            }
        }
    }
}

// ---- before the steps ------------------------------------------------------------------------------

// u from the gradient and, for an update, the momentum after it.
template <class T>
__device__ __forceinline__ float direction(const Matrix &m, const Rule &r, int64_t i) {
    const float g = to_f32(reinterpret_cast<const T *>(m.g)[i]);
    if (m.v == nullptr) return g;
    const float v = __ldcg(m.v + i);
    return r.nesterov ? fmaf(r.momentum, v, g) : v;
}

// Sum over the CTA's threads, to all of them; the same order on every run.
__device__ __forceinline__ double cta_sum(double s, double *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = s;
    __syncthreads();
    s = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) s += scratch[i];
    return s;
}

// v = momentum * v + g over one part of a matrix, and the part's sum of u^2 in f64 (u^2 itself can exceed f32's range).
template <class T, int THREADS>
__device__ __forceinline__ void momentum_part(const Matrix &m, const Rule &r, int part, double *parts, double *scratch) {
    const int64_t n = m.rows * m.cols, per = (n + m.parts - 1) / m.parts, first = part * per, last = min(n, first + per);
    double s = 0;
    for (int64_t base = first + threadIdx.x; base < last; base += 8 * THREADS) {
        float u[8], v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t i = base + k * THREADS;
            u[k] = v[k] = 0.f;
            if (i < last) {
                u[k] = to_f32(reinterpret_cast<const T *>(m.g)[i]);
                if (m.v != nullptr) v[k] = m.v[i];
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int64_t i = base + k * THREADS;
            if (m.v != nullptr) {
                v[k] = __fadd_rn(__fmul_rn(r.momentum, v[k]), u[k]);
                if (i < last) m.v[i] = v[k];
                u[k] = r.nesterov ? fmaf(r.momentum, v[k], u[k]) : v[k];
            }
            s += (double)u[k] * (double)u[k];
        }
    }
    s = cta_sum(s, scratch);
    if (threadIdx.x == 0) parts[m.part0 + part] = s;
}

// kScaleX / norm(u).  A norm of zero gives zeros, one that is not finite NaN.
__device__ __forceinline__ double inverse_norm(const Matrix &m, const double *parts, double *scratch) {
    double s = 0;
    for (int i = threadIdx.x; i < m.parts; i += blockDim.x) s += __ldcg(parts + m.part0 + i);
    s = cta_sum(s, scratch);
    return s == 0 ? 0. : isfinite(s) ? (double)kScaleX / sqrt(s) : (double)NAN;
}

// 64 x 64 values of x = u / norm(u), transposed where u is taller than wide, as planes.
template <class T, int THREADS>
__device__ __forceinline__ void split_tile(const Matrix &m, const Rule &r, int block, double inv, __half *planes,
                                           float (*tile)[65]) {
    const bool flip = m.rows > m.cols;
    const int N = (int)(flip ? m.cols : m.rows), M = (int)(flip ? m.rows : m.cols), tiles = m.x(0).rp / 64;
    const int i0 = block % tiles * 64, j0 = block / tiles * 64;
    const Stored xs = m.x(0);
#pragma unroll 4
    for (int t = threadIdx.x; t < 64 * 64; t += THREADS) {
        const int inner = t % 64, outer = t / 64, i = i0 + (flip ? inner : outer), j = j0 + (flip ? outer : inner);
        float u = 0.f;
        if (i < N && j < M) u = direction<T>(m, r, flip ? (int64_t)j * m.cols + i : (int64_t)i * m.cols + j);
        tile[i - i0][j - j0] = (float)(u * inv);
    }
    __syncthreads();
    for (int t = threadIdx.x; t < 64 * 8; t += THREADS) {
        const int i = t / 8, c = t % 8 * 8;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = tile[i][c + k];
        uint4 hi, lo;
        split8(v, hi, lo);
        const int64_t to = at(xs, i0 + i, j0 + c);
        *reinterpret_cast<uint4 *>(planes + to) = hi;
        *reinterpret_cast<uint4 *>(planes + to + (int64_t)xs.plane * 64) = lo;
    }
    __syncthreads();
}

// ---- the steps --------------------------------------------------------------------------------------

// Warps of a CTA: one issues the loads, one the products, those of the epilogue have 32 rows and half of the columns of the
// tile each, and one plans the next phase.
constexpr int kEpilogue = 8, kPlanner = 2 + kEpilogue, kThreads = (kPlanner + 1) * 32;
constexpr int kBox = 64 * 64 * 2;          // bytes of a box of the tensor map
// A stage: both planes of 64 k of 128 rows of P and up to 128 of Q.
constexpr int kStage = 8 * kBox, kStages = 3;
constexpr int kSmem = kStages * kStage + 1024;

// The products of a matrix, phase by phase.  On x itself a step is
//   kGram a = x x^T, kPoly b = B a + C a a, kApply x = A x + b x.
// From step `squares` on the steps need n x n matrices alone: every p = A + B a + C a a is a polynomial of the same a, so that
// they commute, x stays where it is, and
//   kFactor p = A + B a + C a a, kHalf r = p a beside kGather q = p q, kNext a = p r, ..., at last kFinish x = q x:
// four symmetric products a step instead of the long ones.  What the rounding of a leaves of small singular values is relative
// to the square of the largest, and grows by A^2 a step, so that only the last steps are taken so.  500 x 1300 of rank 40
// rounded to bf16, five steps, f32: 9.3e-6 off with two of them, 5.2e-5 with three (f32 products 1.9e-5).  Rank 5, bf16: with three
// of them 1.007 times its rounding, with four 2.6 times.
enum Kind { kNone = -1, kGram, kPoly, kApply, kFactor, kHalf, kGather, kNext, kFinish };
struct Phase {
    int first, second;   // kinds
    int step;            // of `squares` on: counted from there
};
__device__ __forceinline__ Phase phase_of(const Matrix &m, int phase, int steps) {
    if (phase < 3 * m.squares) return {phase < 3 * steps ? phase % 3 : kNone, kNone, phase / 3};
    const int q = phase - 3 * m.squares, all = steps - m.squares, i = (q - 1) / 3;
    if (q == 0) return {all > 0 ? kGram : kNone, kNone, m.squares};
    if (i >= all) return {kNone, kNone, 0};
    const bool last = i + 1 == all;
    switch ((q - 1) % 3) {
        case 0: return {kFactor, kNone, i};
        case 1: return last ? Phase{i > 0 ? kGather : kNone, kNone, i} : Phase{kHalf, i > 0 ? kGather : kNone, i};
        default: return {last ? kFinish : kNext, kNone, i};
    }
}
__device__ __forceinline__ bool is_symmetric(int kind) { return kind != kApply && kind != kFinish; }

template <class T>
__device__ __forceinline__ Job make_job(const Matrix &m, int kind, int step, int steps) {
    const int n = m.n(), wide = m.wide();
    const int at_x = kind == kFinish ? m.squares % 2 : step % 2;   // x moves with every step on x itself
    const Stored x = m.x(at_x), a = m.square(0);
    // p and the product q of all p so far change places; the first q is the first p
    const Stored p = m.square(1 + step % 2), q_old = step < 2 ? m.square(1) : m.square(4 + step % 2);
    const Stored q_new = m.square(4 + (step + 1) % 2);
    const float scale_q = kScaleB * exp2f(-2.f * (float)step), scale_old = kScaleB * exp2f(-2.f * (float)(step - 1));
    Job j;
    j.final = 0;
    j.M = n;
    j.N = n;
    j.q_mn = 0;
    j.steps = ((kind == kGram ? wide : n) + 63) / 64;
    j.symmetric = is_symmetric(kind);
    j.has_e = 0;
    j.c1 = 0.f;
    j.diagonal = 0.f;
    switch (kind) {
        case kGram:
            j.p = j.q = j.e = x;
            j.d = a;
            j.c0 = kScaleA / (kScaleX * kScaleX);
            break;
        case kPoly:
        case kFactor:
            j.p = j.q = j.e = a;
            j.d = kind == kPoly ? m.square(1) : p;
            j.has_e = 1;
            j.c0 = kC * kScaleB / (kScaleA * kScaleA);
            j.c1 = kB * kScaleB / kScaleA;
            if (kind == kFactor) j.diagonal = kA * kScaleB;
            break;
        case kHalf:
            j.p = p;
            j.q = j.e = a;
            j.d = m.square(3);
            j.c0 = 1.f / kScaleB;
            break;
        case kNext:
            j.p = p;
            j.q = j.e = m.square(3);
            j.d = a;
            j.c0 = 1.f / kScaleB;
            break;
        case kGather:
            j.p = p;
            j.q = j.e = q_old;
            j.d = q_new;
            j.c0 = scale_q / (kScaleB * scale_old);
            break;
        case kFinish:
            j.p = step == 0 ? p : q_new;
            j.q = j.e = j.d = x;
            j.q_mn = 1;
            j.N = wide;
            j.final = 1;
            j.c0 = 1.f / (scale_q * kScaleX);
            break;
        default:   // kApply
            j.p = m.square(1);
            j.q = j.e = x;
            j.d = m.x(1 - at_x);
            j.q_mn = 1;
            j.N = wide;
            j.has_e = 1;
            j.final = step + 1 == steps;
            j.c0 = 1.f / (kScaleB * (j.final ? kScaleX : 1.f));
            j.c1 = j.final ? kA / kScaleX : kA;
    }
    return j;
}

// The work items of a phase: tiles of 128 rows and BN columns, of all matrices in a row, each cut in `splits` slices of its depth.
struct Plan {
    int items, splits;
    int first[kGroup + 1];   // of each matrix's tiles
    int pair[kGroup];        // half of them where there are two products, else none
    Job job[2][kGroup];
};

// Tiles of a symmetric product: those that touch the diagonal or lie above it.  With tiles narrower than high, a row of
// tiles starts at the first that reaches its rows.
__device__ __forceinline__ int tiles_of(int n, int wide, bool symmetric, int width) {
    const int tm = (n + 127) / 128, tn = (wide + width - 1) / width;
    return symmetric ? tm * tn - 128 / width * (tm * (tm - 1) / 2) : tm * tn;
}

// By one warp.
template <class T, int BN>
__device__ __forceinline__ void make_plan(const Group &g, int phase, Plan *plan) {
    const int lane = threadIdx.x % 32;
    int n = 0, wide = 0, copies = 0, steps = 0;
    bool symmetric = false;
    if (lane < g.n) {
        const Matrix &m = g.m[lane];
        const Phase ph = phase_of(m, phase, g.steps);
        n = m.n();
        symmetric = is_symmetric(ph.first);
        wide = symmetric ? n : m.wide();
        copies = ph.first == kNone ? 0 : ph.second == kNone ? 1 : 2;   // a pair is symmetric both
        if (copies > 0) plan->job[0][lane] = make_job<T>(m, ph.first, ph.step, g.steps);
        if (copies > 1) plan->job[1][lane] = make_job<T>(m, ph.second, ph.step, g.steps);
        steps = copies == 0 ? 0 : ((ph.first == kGram ? m.wide() : n) + 63) / 64;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) steps = max(steps, __shfl_xor_sync(0xffffffffu, steps, o));
    const int tiles = copies * tiles_of(n, wide, symmetric, BN);
    int sum = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    if (lane < g.n) {
        plan->first[lane] = sum - tiles;
        plan->pair[lane] = copies == 2 ? tiles / 2 : tiles;
    }
    if (lane == 31) {
        plan->items = sum;
        plan->first[g.n] = sum;
        // Slices while every slice finds an SM at once and has eight steps to take.
        plan->splits = sum == 0 ? 1 : max(1, min(min((int)gridDim.x / sum, steps / 8), 16));
    }
}

struct Item {
    int matrix, copy, m0, n0, k0, k1;
    bool mirror;
};

template <int BN>
__device__ __forceinline__ Item find_item(const Plan &plan, int w) {
    Item it;
    int item = w, slice = 0;
    if (plan.splits > 1) {
        item = w / plan.splits;
        slice = w - item * plan.splits;
    }
    int i = 0;
    while (plan.first[i + 1] <= item) ++i;
    int t = item - plan.first[i], bi, bj;
    it.matrix = i;
    it.copy = t >= plan.pair[i];
    if (it.copy) t -= plan.pair[i];
    const Job &j = plan.job[it.copy][i];
    if (j.symmetric) {
        bi = 0;
        for (int left = (j.N + BN - 1) / BN; t >= left; left -= 128 / BN) {
            t -= left;
            ++bi;
        }
        bj = bi * (128 / BN) + t;
        it.mirror = bj * BN >= (bi + 1) * 128;
    } else {
        const int tm = (j.M + 127) / 128;
        bj = t / tm;
        bi = t - bj * tm;
        it.mirror = false;
    }
    it.m0 = bi * 128;
    it.n0 = bj * BN;
    it.k0 = 0;
    it.k1 = j.steps;
    if (plan.splits > 1) {
        const int per = (j.steps + plan.splits - 1) / plan.splits;
        it.k0 = min(j.steps, slice * per);
        it.k1 = min(j.steps, it.k0 + per);
    }
    return it;
}

// Instruction descriptor: f16 operands, f32 sums.
__host__ __device__ constexpr uint32_t half_idesc(bool q_mn, int m, int n) {
    return make_idesc(false, q_mn, m, n) & ~((7u << 7) | (7u << 10));
}

// The barrier of the grid, by all threads.  What a CTA wrote before it, in generic accesses, any CTA may read after it, by TMA
// too.  Every wait is bounded; false once a wait has given up, here or in another CTA.
__device__ __forceinline__ bool grid_sync(int *arrived, int target, int *status, volatile int *abort_flag) {
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        asm volatile("red.release.gpu.global.add.s32 [%0], 1;" ::"l"(arrived) : "memory");
        uint64_t t0 = 0;
        for (uint32_t it = 0;; ++it) {
            int seen;
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(seen) : "l"(arrived) : "memory");
            if (seen >= target) break;
            if ((it & 255u) == 255u) {
                const uint64_t now = global_timer_ns();
                if (t0 == 0) t0 = now;
                if (*abort_flag || now - t0 > 2000000000ull || *reinterpret_cast<volatile int *>(status) != 0) {
                    atomicCAS(status, 0, 234);
                    *abort_flag = 1;
                    break;
                }
            }
        }
        asm volatile("fence.proxy.async;" ::: "memory");   // this thread issues the loads by TMA
    }
    __syncthreads();
    return *abort_flag == 0;
}

// What the roles of a CTA share.
struct Cta {
    const CUtensorMap *map;
    const Group *g;            // in shared memory
    __half *planes;
    float4 *sums;
    int *counters, *status;
    uint32_t stages, full, empty, acc_full, acc_empty;   // in shared memory
    uint32_t tmem;
    volatile int *abort_flag;
    int *last_slice;
    Plan *plans;               // of this phase and of the next, by parity
};

// Reads a tile's accumulators out, `reads` of them from the accs-th on, adds them and stores the result.
template <class T, int BN>
__device__ __forceinline__ void finish_tile(const Cta &t, const Item &it, const Job &j, int w, int splits, int accs, int reads) {
    constexpr int COLS = BN / 2;
    const Matrix &m = t.g->m[it.matrix];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int quarter = warp % 4, part = (warp - 2) / 4, row = quarter * 32 + lane;
    const int m0 = it.m0, col = it.n0 + part * COLS;
    Addend e;
    if (splits == 1) load_addend(j, t.planes, m0 + row, col, e);   // on its way while the products run
    float sum[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) sum[c] = 0.f;
    bool good = true;
    for (int c = 0; c < reads; ++c) {
        const int acc = accs + c;
        good = __all_sync(0xffffffffu, mbar_wait(t.acc_full + acc % 2 * 8, acc / 2 & 1, t.abort_flag));
        if (!good) {
            if (lane == 0) atomicCAS(t.status, 0, 233);
            break;
        }
        tc_fence_after();
        const uint32_t from = t.tmem + acc % 2 * 128 + part * COLS + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
        for (int b = 0; b < COLS; b += 32) {
            uint32_t v[32];
            tmem_ld_32x32(from + b, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) sum[b + i] += __uint_as_float(v[i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(t.acc_empty + acc % 2 * 8);
    }
    __syncwarp();
    if (splits > 1) {
        // The slice that is done last adds all of them, in their order, and goes on.  (The warps meet at barriers without a
        // limit: a CTA has one slice a phase, and all of them come here whether a wait has given up or not.)
        const int item = w / splits;
        float4 *mine = t.sums + ((int64_t)w * 32 + part * (COLS / 4)) * 128 + row;
#pragma unroll
        for (int c = 0; c < COLS / 4; ++c)
            __stcg(mine + c * 128, make_float4(sum[4 * c], sum[4 * c + 1], sum[4 * c + 2], sum[4 * c + 3]));
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(kEpilogue * 32) : "memory");
        if (threadIdx.x == 64) {
            const int n = atomicAdd(t.counters + 2 + item, 1);
            if (n == splits - 1) t.counters[2 + item] = 0;
            *t.last_slice = n == splits - 1;
            __threadfence();
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kEpilogue * 32) : "memory");
        if (!*t.last_slice) return;
        load_addend(j, t.planes, m0 + row, col, e);
#pragma unroll
        for (int c = 0; c < COLS; ++c) sum[c] = 0.f;
        for (int z = 0; z < splits; ++z) {
            const float4 *from = t.sums + (((int64_t)item * splits + z) * 32 + part * (COLS / 4)) * 128 + row;
#pragma unroll
            for (int b = 0; b < COLS / 4; b += 8) {
                float4 p4[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) p4[c] = __ldcg(from + (b + c) * 128);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    sum[4 * (b + c)] += p4[c].x;
                    sum[4 * (b + c) + 1] += p4[c].y;
                    sum[4 * (b + c) + 2] += p4[c].z;
                    sum[4 * (b + c) + 3] += p4[c].w;
                }
            }
        }
    }
    if (!good) return;
#pragma unroll
    for (int b = 0; b < COLS; b += 32) {
        if (b > 0) load_addend(j, t.planes, m0 + row, col + b, e);
        finish32<T>(j, m, t.g->rule, t.planes, m0 + row, col + b, sum + b, e, it.mirror);
        __syncwarp();   // rows beyond the matrix leave the last step's stores early, and what follows takes whole warps
    }
}

// One phase.  stages, accs: stages and accumulators taken so far, which give the place in the rings and
// the parity of their barriers.  barrier: the arrivals that open it, 0 for the first phase.
template <class T, int BN>
__device__ __forceinline__ bool run_phase(const Cta &t, int phase, int barrier, int &stages_taken, int &accs_taken) {
    // 64-k steps that one accumulator adds, twelve additions each: tcgen05 cuts its sums off rather than rounding them, by up to
    // 2^-23 of the sum so far an addition.  1000 x 2100 of rank 5, bf16, twenty steps, in roundings of the result: 1.081 with
    // sixteen, 1.005 with four, 1.001 with one; us, 4096 x 4096 4040, 4320 and 4550.
    constexpr int kAccStages = sizeof(T) == 2 ? 4 : 1;
    constexpr int HALF = (2 + BN / 64) * kBox;   // of a stage: 128 rows of P, BN of Q
    const Group &g = *t.g;
    const Plan *plan = t.plans + phase % 2;
    const int warp = threadIdx.x / 32;
    const int units = plan->items * plan->splits, splits = plan->splits;
    int stages = stages_taken, accs = accs_taken;
    // Where this CTA's first item lies does not depend on what the others still compute.
    Item first = {};
    if ((int)blockIdx.x < units) first = find_item<BN>(*plan, blockIdx.x);
    if (barrier > 0 && !grid_sync(t.counters, barrier, t.status, t.abort_flag)) return false;

    if (warp == kPlanner) {
        // What does not depend on what the others compute is ready before the next barrier.
        if (phase + 1 < g.phases) make_plan<T, BN>(g, phase + 1, t.plans + (phase + 1) % 2);
    } else if (warp == 0) {
        for (int w = blockIdx.x; w < units; w += gridDim.x) {
            const Item it = w == (int)blockIdx.x ? first : find_item<BN>(*plan, w);
            const Job &j = plan->job[it.copy][it.matrix];
            const bool q_mn = j.q_mn;
            const int count = it.k1 - it.k0;
            // rows of a step's boxes, and from one to the next
            const int p_base = j.p.row + it.m0, p_plane = j.p.plane, p_step = j.p.rp;
            const int q_base = j.q.row + (q_mn ? it.n0 / 64 * j.q.rp : it.n0), q_plane = j.q.plane, q_step = q_mn ? 64 : j.q.rp;
            const int q_box = q_mn ? j.q.rp : 64;
            if (elect_one()) {
                for (int c = 0; c < count; ++c) {
                    const int at_stage = (stages + c) % kStages, round = (stages + c) / kStages;
                    if (!mbar_wait(t.empty + at_stage * 8, (round & 1) ^ 1, t.abort_flag)) {
                        atomicCAS(t.status, 0, 230);
                        break;
                    }
                    const uint32_t bar = t.full + at_stage * 8, dst = t.stages + at_stage * kStage;
                    const int k = it.k0 + c;
                    mbar_arrive_expect_tx(bar, 2 * HALF);
                    for (int h = 0; h < 2; ++h) {
                        const int p_row = p_base + h * p_plane + k * p_step, q_row = q_base + h * q_plane + k * q_step;
                        const uint32_t to = dst + h * HALF;
                        tma_load_2d(to, t.map, bar, 0, p_row);
                        tma_load_2d(to + kBox, t.map, bar, 0, p_row + 64);
#pragma unroll
                        for (int b = 0; b < BN / 64; ++b) tma_load_2d(to + (2 + b) * kBox, t.map, bar, 0, q_row + b * q_box);
                    }
                }
            }
            __syncwarp();
            stages += count;
        }
    } else if (warp == 1) {
        for (int w = blockIdx.x; w < units; w += gridDim.x) {
            const Item it = w == (int)blockIdx.x ? first : find_item<BN>(*plan, w);
            const Job &j = plan->job[it.copy][it.matrix];
            const bool q_mn = j.q_mn;
            const int count = it.k1 - it.k0;
            if (elect_one()) {
                const uint32_t idesc = half_idesc(q_mn, 128, BN);
                const uint32_t q_step = q_mn ? 16 * 128 : 32, q_lbo = q_mn ? kBox : 0;
                for (int c = 0; c < count; ++c) {
                    const int acc = accs + c / kAccStages;
                    if (c % kAccStages == 0 && !mbar_wait(t.acc_empty + acc % 2 * 8, (acc / 2 & 1) ^ 1, t.abort_flag)) {
                        atomicCAS(t.status, 0, 231);
                        break;
                    }
                    const int at_stage = (stages + c) % kStages;
                    if (!mbar_wait(t.full + at_stage * 8, (stages + c) / kStages & 1, t.abort_flag)) {
                        atomicCAS(t.status, 0, 232);
                        break;
                    }
                    tc_fence_after();
                    const uint32_t d = t.tmem + acc % 2 * 128, base = t.stages + at_stage * kStage;
                    auto mma = [&](int hp, int hq, int i, bool add) {
                        umma_bf16(d, make_smem_desc(base + hp * HALF + i * 32, 0, 1024),
                                  make_smem_desc(base + hq * HALF + 2 * kBox + i * q_step, q_lbo, 1024), idesc, add ? 1u : 0u);
                    };
                    const bool more = c % kAccStages != 0;
                    // the small products first: what an addition cuts off is a part of the sum so far
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        mma(0, 1, i, more || i > 0);
                        mma(1, 0, i, true);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma(0, 0, i, true);
                    umma_commit(t.empty + at_stage * 8);
                    if ((c + 1) % kAccStages == 0 || c + 1 == count) umma_commit(t.acc_full + acc % 2 * 8);
                }
            }
            __syncwarp();
            stages += count;
            accs += (count + kAccStages - 1) / kAccStages;
        }
    } else {
        for (int w = blockIdx.x; w < units; w += gridDim.x) {
            const Item it = w == (int)blockIdx.x ? first : find_item<BN>(*plan, w);
            const Job &j = plan->job[it.copy][it.matrix];
            const int reads = (it.k1 - it.k0 + kAccStages - 1) / kAccStages;
            finish_tile<T, BN>(t, it, j, w, splits, accs, reads);
            accs += reads;
        }
    }
    stages_taken = stages;
    accs_taken = accs;
    return true;
}

// counters: [0] arrivals at the grid's barrier, [1] CTAs that have left, [2 ...] slices of a tile that are done; zero before
// and after.  sums: a tile's slices, [item][slice][four columns][row].
template <class T, int BN>
__global__ void __launch_bounds__(kThreads, 1)
    muon_kernel(const __grid_constant__ CUtensorMap map, __half *planes, double *parts, float4 *sums, int *counters, int *status,
                const __grid_constant__ Group group) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    __shared__ uint64_t bars[2 * kStages + 4];
    __shared__ uint32_t slot;
    __shared__ int flags[2];
    __shared__ Plan plans[2];
    __shared__ Group g;
    __shared__ double scratch[kThreads / 32];
    volatile int *abort_flag = flags;
    const int warp = threadIdx.x / 32;
    const uint32_t bar0 = smem_u32(bars);

    if (threadIdx.x == 0) {
        prefetch_tmap(&map);
        for (int s = 0; s < kStages; ++s) {
            mbar_init(bar0 + s * 8, 1);
            mbar_init(bar0 + (kStages + s) * 8, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar0 + (2 * kStages + s) * 8, 1);
            mbar_init(bar0 + (2 * kStages + 2 + s) * 8, kEpilogue);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    for (int i = threadIdx.x; i < (int)(sizeof(Group) / 4); i += kThreads)
        reinterpret_cast<uint32_t *>(&g)[i] = reinterpret_cast<const uint32_t *>(&group)[i];
    if (warp == 1) {
        tmem_alloc(smem_u32(&slot), 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const Cta c = {&map, &g, planes, sums, counters, status, smem_u32(smem), bar0, bar0 + kStages * 8, bar0 + 2 * kStages * 8,
                   bar0 + (2 * kStages + 2) * 8, slot, abort_flag, flags + 1, plans};
    int barriers = 0;
    bool ok = true;

    if (g.inside) {
        for (int w = blockIdx.x, i = 0, before = 0; i < g.n; before += g.m[i].parts, ++i)
            for (; w < before + g.m[i].parts; w += gridDim.x) momentum_part<T, kThreads>(g.m[i], g.rule, w - before, parts, scratch);
        ok = grid_sync(counters, ++barriers * gridDim.x, status, abort_flag);
        for (int w = blockIdx.x, i = 0, before = 0; ok && i < g.n; ++i) {
            const int blocks = g.m[i].x(0).plane / 64;
            if (w < before + blocks) {
                const double inv = inverse_norm(g.m[i], parts, scratch);
                for (; w < before + blocks; w += gridDim.x)
                    split_tile<T, kThreads>(g.m[i], g.rule, w - before, inv, planes, reinterpret_cast<float(*)[65]>(smem));
            }
            before += blocks;
        }
    }

    int stages = 0, accs = 0;
    if (warp == kPlanner) make_plan<T, BN>(g, 0, plans);
    __syncthreads();
    for (int phase = 0; ok && phase < g.phases; ++phase) {
        if (phase > 0 || g.inside) ++barriers;
        ok = run_phase<T, BN>(c, phase, barriers * (int)gridDim.x, stages, accs);
        __syncthreads();
    }

    tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(c.tmem, 256);
    }
    // The last CTA to leave, when all have passed the last barrier, clears the counts for the next launch.
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(counters + 1, 1) == (int)gridDim.x - 1) {
            counters[0] = 0;
            counters[1] = 0;
        }
    }
}

}  // namespace muon
}  // namespace ag
