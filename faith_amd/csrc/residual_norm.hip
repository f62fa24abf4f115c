// The residual connection and the normalisation behind it, of a network's concrete pass: h = x + residual, then along the
// row of n
//     c = h - mean(h)  (root mean square: c = h),   z = c / sqrt(mean(c^2) + eps)  (without the variance: z = c),   y = w z + b
// and the gradients.  Everything is bound by HBM: forward 4 n elements a row (x, residual in; h, y out), backward 4 n (dy, h,
// dsum in; dx out).  Measured: 16384 rows of 4096 bf16 forward 94 us, 5.7 TB/s.  A row is read once and stays in registers
// between the statistics and the result: a wavefront to a row up to 128 groups of 16 bytes, four or eight wavefronts beyond that;
// rows that do not fall into 16-byte groups, and rows wider than the registers hold, take a kernel that goes over the row again (it
// comes from the L2).
// Statistics are sums in 32 bits: over at most 32 values a lane where the row stays in registers, n / 256 values a lane in the
// kernel for any width, and a tree above; the variance is that of the centred values, so nothing cancels.
#include "common.h"

namespace {

using namespace faith;

typedef unsigned uintx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

template <class T> struct Group { static constexpr int N = 16 / (int)sizeof(T); };
template <class T> struct Packed;
template <> struct Packed<float> { typedef floatx4 type; };
template <> struct Packed<__bf16> { typedef bf16x8 type; };
template <> struct Packed<_Float16> { typedef halfx8 type; };

template <class T> __device__ __forceinline__ void unpack(const T *p, float *v) {
    const typename Packed<T>::type x = *reinterpret_cast<const typename Packed<T>::type *>(p);
#pragma unroll
    for (int e = 0; e < Group<T>::N; ++e) v[e] = (float)x[e];
}
template <class T> __device__ __forceinline__ void pack(T *p, const float *v) {
    typename Packed<T>::type x;
#pragma unroll
    for (int e = 0; e < Group<T>::N; ++e) x[e] = (T)v[e];
    *reinterpret_cast<typename Packed<T>::type *>(p) = x;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// The larger of two magnitudes, NaN above everything: the bits of numbers without a sign are in their order as integers
__device__ __forceinline__ float larger(float a, float b) {
    const unsigned x = __float_as_uint(a), y = __float_as_uint(b);
    return __uint_as_float(x > y ? x : y);
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = larger(v, __shfl_xor(v, d));
    return v;
}

// Sums (or the largest magnitude) of a row over the wavefronts that share it.  `slot` has to differ between two calls that no other
// barrier separates.
template <int WAVES, bool MAX> __device__ __forceinline__ float across(float v, float *slot, int wave) {
    v = MAX ? wave_max(v) : wave_sum(v);
    if constexpr (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) slot[wave] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v = MAX ? larger(v, slot[w]) : v + slot[w];
    return v;
}

constexpr int RMS = FAITH_NORM_RMS, STANDARD = FAITH_NORM_STANDARD, NO_VAR = FAITH_NORM_NO_VAR;

struct NormArgs {
    const void *x, *residual, *weight, *bias;
    void *y, *sum;
    float *stats, *scales;
    long long rows;
    int n, kind, bits;
    float eps;
};

// A row with a NaN has a scale of NaN, and every value divided by it is one; one with an infinity an infinite scale
__device__ __forceinline__ float divided(float y, float scale) { return scale > 0.f ? y / scale : (scale == 0.f ? 0.f : y * scale); }
__device__ __forceinline__ unsigned char to_int8(float t) {
    t = __builtin_rintf(t);
    t = t > 127.f ? 127.f : t < -127.f ? -127.f : t == t ? t : 0.f;        // no value for NaN: 0
    return (unsigned char)(signed char)(int)t;
}
__device__ __forceinline__ float in_e4m3(float t) { return t > 448.f ? 448.f : t < -448.f ? -448.f : t; }
__device__ __forceinline__ unsigned to_e4m3(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(in_e4m3(a), in_e4m3(b), 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(in_e4m3(c), in_e4m3(d), w, true);
}
__device__ __forceinline__ float steps_of(int bits) { return bits == FAITH_BITS_INT8 ? 127.f : 448.f; }

// WAVES wavefronts to a row (a workgroup of four such rows, where one is enough), CH groups of 16 bytes to a lane
constexpr int rows_of(int waves) { return waves == 1 ? 4 : 1; }
constexpr int threads_of(int waves) { return 64 * waves * rows_of(waves); }
template <class T, int WAVES, int CH>
__global__ void __launch_bounds__(threads_of(WAVES)) residual_norm(const NormArgs g) {
    constexpr int N = Group<T>::N, LANES = 64 * WAVES;
    __shared__ __align__(16) float slot[3][WAVES];
    const int wave = threadIdx.x >> 6, t = (int)threadIdx.x % LANES;
    const long long row = (long long)blockIdx.x * rows_of(WAVES) + wave / WAVES;
    if (WAVES < 4 && row >= g.rows) return;                   // a whole wavefront; no barrier follows in this shape
    const long long at = row * g.n;
    const T *x = reinterpret_cast<const T *>(g.x) + at, *res = g.residual ? reinterpret_cast<const T *>(g.residual) + at : nullptr;
    float h[CH][N];
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (c * LANES + t) * N;
        if (e0 < g.n) unpack(x + e0, h[c]);
        else
#pragma unroll
            for (int e = 0; e < N; ++e) h[c][e] = 0.f;
    }
    if (res) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (c * LANES + t) * N;
            float r[N];
            if (e0 >= g.n) continue;
            unpack(res + e0, r);
#pragma unroll
            for (int e = 0; e < N; ++e) h[c][e] += r[e];
        }
    }
    if (g.sum) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (c * LANES + t) * N;
            if (e0 < g.n) pack(reinterpret_cast<T *>(g.sum) + at + e0, h[c]);
        }
    }
    const float inv_n = 1.f / (float)g.n;
    float mean = 0.f, r = 1.f;
    if (g.kind != RMS) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < N; ++e) s += h[c][e];
        mean = across<WAVES, false>(s, slot[0], wave) * inv_n;
    }
    if (g.kind != NO_VAR) {
        float q = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if ((c * LANES + t) * N >= g.n) continue;
#pragma unroll
            for (int e = 0; e < N; ++e) q = fmaf(h[c][e] - mean, h[c][e] - mean, q);
        }
        r = 1.f / sqrtf(fmaf(across<WAVES, false>(q, slot[1], wave), inv_n, g.eps));
    }
    if (g.stats && t == 0) g.stats[row] = r;
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (c * LANES + t) * N;
        if (e0 >= g.n) continue;
        float w[N], b[N];
        if (g.weight) unpack(reinterpret_cast<const T *>(g.weight) + e0, w);
        if (g.bias) unpack(reinterpret_cast<const T *>(g.bias) + e0, b);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            float y = (h[c][e] - mean) * r;
            if (g.weight) y *= w[e];
            if (g.bias) y += b[e];
            h[c][e] = y;
            top = larger(top, __builtin_fabsf(y));
        }
        if (!g.bits) pack(reinterpret_cast<T *>(g.y) + at + e0, h[c]);
    }
    if (!g.bits) return;
    const float scale = across<WAVES, true>(top, slot[2], wave) / steps_of(g.bits);
    if (t == 0) g.scales[row] = scale;
    unsigned char *q = reinterpret_cast<unsigned char *>(g.y) + at;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (c * LANES + t) * N;
        if (e0 >= g.n) continue;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = divided(h[c][e + i], scale);
            unsigned w;
            if (g.bits == FAITH_BITS_INT8) w = to_int8(v[0]) | (unsigned)to_int8(v[1]) << 8 | (unsigned)to_int8(v[2]) << 16 | (unsigned)to_int8(v[3]) << 24;
            else w = to_e4m3(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<unsigned *>(q + e0 + e) = w;
        }
    }
}

// any width and alignment: a workgroup to a row, which it goes over again for each of its sums
template <class T> __global__ void __launch_bounds__(256) residual_norm_any(const NormArgs g) {
    __shared__ __align__(16) float slot[3][4];
    const int wave = threadIdx.x >> 6;
    const long long at = (long long)blockIdx.x * g.n;
    const T *x = reinterpret_cast<const T *>(g.x) + at, *res = g.residual ? reinterpret_cast<const T *>(g.residual) + at : nullptr;
    const T *w = reinterpret_cast<const T *>(g.weight), *b = reinterpret_cast<const T *>(g.bias);
    auto sum_at = [&](int e) { return (float)x[e] + (res ? (float)res[e] : 0.f); };
    const float inv_n = 1.f / (float)g.n;
    float mean = 0.f, r = 1.f;
    if (g.kind != RMS) {
        float s = 0.f;
        for (int e = threadIdx.x; e < g.n; e += 256) s += sum_at(e);
        mean = across<4, false>(s, slot[0], wave) * inv_n;
    }
    if (g.kind != NO_VAR) {
        float q = 0.f;
        for (int e = threadIdx.x; e < g.n; e += 256) {
            const float c = sum_at(e) - mean;
            q = fmaf(c, c, q);
        }
        r = 1.f / sqrtf(fmaf(across<4, false>(q, slot[1], wave), inv_n, g.eps));
    }
    if (g.stats && threadIdx.x == 0) g.stats[blockIdx.x] = r;
    auto y_at = [&](int e, float h) {
        float y = (h - mean) * r;
        if (w) y *= (float)w[e];
        if (b) y += (float)b[e];
        return y;
    };
    float scale = 0.f;
    if (g.bits) {
        float top = 0.f;
        for (int e = threadIdx.x; e < g.n; e += 256) top = larger(top, __builtin_fabsf(y_at(e, sum_at(e))));
        scale = across<4, true>(top, slot[2], wave) / steps_of(g.bits);
        if (threadIdx.x == 0) g.scales[blockIdx.x] = scale;
    }
    for (int e = threadIdx.x; e < g.n; e += 256) {
        const float h = sum_at(e), y = y_at(e, h);
        if (g.sum) reinterpret_cast<T *>(g.sum)[at + e] = (T)h;
        if (!g.bits) reinterpret_cast<T *>(g.y)[at + e] = (T)y;
        else if (g.bits == FAITH_BITS_INT8) reinterpret_cast<unsigned char *>(g.y)[at + e] = to_int8(divided(y, scale));
        else reinterpret_cast<unsigned char *>(g.y)[at + e] = (unsigned char)(to_e4m3(divided(y, scale), 0.f, 0.f, 0.f) & 255u);
    }
}

struct NormGradArgs {
    const void *dy, *dsum, *h, *weight;
    const float *stats;
    void *dx, *dweight, *dbias;
    float *partial;              // [blocks][2][n]: a workgroup's sums for the weight's and the bias's gradient
    float *means;                // [rows], for the kernels of any width
    long long rows;
    int n, kind, blocks;
};

// dh = r (g - z mean(g z) [with the variance] - mean(g) [with the mean]) + dsum, g = w dy.  z comes from h as it was stored,
// and so does the mean: against that of the unrounded sum a row of almost equal values would come out off by its rounding
// over its spread.  A workgroup goes over rows blockIdx.x, + gridDim.x, ...; its columns' sums of dy z and dy stay in registers
// until the end and go to a row of `partial` of its own, which a second launch adds up in a fixed order: no atomics, the same bits
// every time.
//
// The next row is on its way while this one is worked on: without that a row's loads wait for the sums of the row before
// (8191 rows of 5120 bf16: 114 -> 84 us, now 80, 4.2 TB/s; sixteen wavefronts to a row instead of four take 95).
template <class T, int WAVES, int CH, bool BIAS>
__global__ void __launch_bounds__(threads_of(WAVES)) residual_norm_grad(const NormGradArgs g) {
    constexpr int N = Group<T>::N, LANES = 64 * WAVES;
    typedef typename Packed<T>::type Raw;
    __shared__ __align__(16) float slot[2][2][WAVES], mean_slot[2][WAVES];
    const int wave = threadIdx.x >> 6, t = (int)threadIdx.x % LANES;
    const float inv_n = 1.f / (float)g.n;
    float dw[CH][N], db[BIAS ? CH : 1][N];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < N; ++e) { dw[c][e] = 0.f; if (BIAS) db[c][e] = 0.f; }
    Raw raw_d[CH], raw_h[CH], raw_s[CH];
    float raw_r = 1.f;
    auto fetch = [&](long long row) {
        const long long at = row * g.n;
        if (g.kind != NO_VAR) raw_r = g.stats[row];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (c * LANES + t) * N;
            if (e0 >= g.n) continue;
            raw_d[c] = *reinterpret_cast<const Raw *>(reinterpret_cast<const T *>(g.dy) + at + e0);
            raw_h[c] = *reinterpret_cast<const Raw *>(reinterpret_cast<const T *>(g.h) + at + e0);
            if (g.dsum) raw_s[c] = *reinterpret_cast<const Raw *>(reinterpret_cast<const T *>(g.dsum) + at + e0);
        }
    };
    int parity = 0;
    const long long step = (long long)gridDim.x * rows_of(WAVES);
    long long row = (long long)blockIdx.x * rows_of(WAVES) + wave / WAVES;
    if (row < g.rows) fetch(row);
    for (; row < g.rows; row += step, parity ^= 1) {
        const float r = raw_r;
        float z[CH][N], d[CH][N];
        Raw s[CH];
        float s0 = 0.f, s1 = 0.f, mean = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const bool in = (c * LANES + t) * N < g.n;
            s[c] = raw_s[c];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                d[c][e] = in ? (float)raw_d[c][e] : 0.f;
                z[c][e] = in ? (float)raw_h[c][e] : 0.f;
            }
        }
        if (row + step < g.rows) fetch(row + step);
        if (g.kind != RMS) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int e = 0; e < N; ++e) mean += z[c][e];
            mean = across<WAVES, false>(mean, mean_slot[parity], wave) * inv_n;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (c * LANES + t) * N;
            float w[N];
            if (g.weight && e0 < g.n) unpack(reinterpret_cast<const T *>(g.weight) + e0, w);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                z[c][e] = e0 < g.n ? (z[c][e] - mean) * r : 0.f;
                dw[c][e] = fmaf(d[c][e], z[c][e], dw[c][e]);
                if (BIAS) db[c][e] += d[c][e];
                if (g.weight && e0 < g.n) d[c][e] *= w[e];
                s0 += d[c][e];
                s1 = fmaf(d[c][e], z[c][e], s1);
            }
        }
        float m0 = 0.f, m1 = 0.f;
        s0 = wave_sum(s0);
        s1 = wave_sum(s1);
        if constexpr (WAVES == 1) {
            m0 = s0 * inv_n;
            m1 = s1 * inv_n;
        } else {
            if ((threadIdx.x & 63) == 0) { slot[parity][0][wave] = s0; slot[parity][1][wave] = s1; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) { m0 += slot[parity][0][w]; m1 += slot[parity][1][w]; }
            m0 *= inv_n;
            m1 *= inv_n;
        }
        if (g.kind == RMS) m0 = 0.f;
        if (g.kind == NO_VAR) m1 = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e0 = (c * LANES + t) * N;
            if (e0 >= g.n) continue;
            float v[N];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float dh = (d[c][e] - m0 - z[c][e] * m1) * r;
                v[e] = g.dsum ? (float)s[c][e] + dh : dh;
            }
            pack(reinterpret_cast<T *>(g.dx) + row * g.n + e0, v);
        }
    }
    if (!g.partial) return;
    // rows of `partial`: one to a wavefront group
    float *p = g.partial + ((long long)blockIdx.x * rows_of(WAVES) + wave / WAVES) * 2 * g.n;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e0 = (c * LANES + t) * N;
        if (e0 >= g.n) continue;
#pragma unroll
        for (int e = 0; e < N; e += 4) {
            if (g.dweight) *reinterpret_cast<floatx4 *>(p + e0 + e) = floatx4{dw[c][e], dw[c][e + 1], dw[c][e + 2], dw[c][e + 3]};
            if constexpr (BIAS) *reinterpret_cast<floatx4 *>(p + g.n + e0 + e) = floatx4{db[c][e], db[c][e + 1], db[c][e + 2], db[c][e + 3]};
        }
    }
}

// any width and alignment: dx, a workgroup to a row
template <class T> __global__ void __launch_bounds__(256) residual_norm_grad_any(const NormGradArgs g) {
    __shared__ __align__(16) float slot[3][4];
    const int wave = threadIdx.x >> 6;
    const long long row = blockIdx.x, at = row * g.n;
    const T *dy = reinterpret_cast<const T *>(g.dy) + at, *hh = reinterpret_cast<const T *>(g.h) + at, *w = reinterpret_cast<const T *>(g.weight);
    const float r = g.kind == NO_VAR ? 1.f : g.stats[row], inv_n = 1.f / (float)g.n;
    float mean = 0.f;
    if (g.kind != RMS) {
        for (int e = threadIdx.x; e < g.n; e += 256) mean += (float)hh[e];
        mean = across<4, false>(mean, slot[2], wave) * inv_n;
    }
    if (g.means && threadIdx.x == 0) g.means[row] = mean;
    float s0 = 0.f, s1 = 0.f;
    for (int e = threadIdx.x; e < g.n; e += 256) {
        const float d = (float)dy[e] * (w ? (float)w[e] : 1.f);
        s0 += d;
        s1 = fmaf(d, ((float)hh[e] - mean) * r, s1);
    }
    float m0 = across<4, false>(s0, slot[0], wave) * inv_n, m1 = across<4, false>(s1, slot[1], wave) * inv_n;
    if (g.kind == RMS) m0 = 0.f;
    if (g.kind == NO_VAR) m1 = 0.f;
    const T *ds = g.dsum ? reinterpret_cast<const T *>(g.dsum) + at : nullptr;
    for (int e = threadIdx.x; e < g.n; e += 256) {
        const float d = (float)dy[e] * (w ? (float)w[e] : 1.f), z = ((float)hh[e] - mean) * r;
        reinterpret_cast<T *>(g.dx)[at + e] = (T)((d - m0 - z * m1) * r + (ds ? (float)ds[e] : 0.f));
    }
}
// and the sums over rows: workgroup (columns, b) adds the rows of block b to row b of `partial`
template <class T> __global__ void __launch_bounds__(256) residual_norm_columns_any(const NormGradArgs g) {
    const int e = (int)(blockIdx.x * 256 + threadIdx.x);
    if (e >= g.n) return;
    float dw = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < g.rows; row += gridDim.y) {
        const float mean = g.means[row], r = g.kind == NO_VAR ? 1.f : g.stats[row];
        const float d = (float)reinterpret_cast<const T *>(g.dy)[row * g.n + e];
        dw = fmaf(d, ((float)reinterpret_cast<const T *>(g.h)[row * g.n + e] - mean) * r, dw);
        db += d;
    }
    float *p = g.partial + (long long)blockIdx.y * 2 * g.n;
    p[e] = dw;
    p[g.n + e] = db;
}

// columns of `partial` added up: 32 columns to a workgroup, 32 threads down each
template <class T> __global__ void __launch_bounds__(1024) residual_norm_columns(const NormGradArgs g) {
    __shared__ __align__(16) float part[32][33];
    const int c = threadIdx.x & 31, s = threadIdx.x >> 5, e = (int)blockIdx.x * 32 + c;
    const bool bias = blockIdx.y == (g.dweight ? 1 : 0);
    float v = 0.f;
    if (e < g.n)
        for (int b = s; b < g.blocks; b += 32) v += g.partial[(long long)b * 2 * g.n + (bias ? g.n : 0) + e];
    part[s][c] = v;
    __syncthreads();
    if (s > 0 || e >= g.n) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) v += part[i][c];
    reinterpret_cast<T *>(bias ? g.dbias : g.dweight)[e] = (T)v;
}

// wavefronts to a row and 16-byte groups to a lane; 0: the kernel for any width
struct Shape { int waves, groups; };
Shape shape_of(int n, int dtype, bool aligned16) {
    const int per = dtype == FAITH_F32 ? 4 : 8;
    if (!aligned16 || n % per) return {0, 0};
    const int groups = n / per;
    if (groups <= 64) return {1, 1};
    if (groups <= 128) return {1, 2};
    if (groups <= 256) return {4, 1};
    if (groups <= 512) return {4, 2};
    if (groups <= 768) return {4, 3};
    if (groups <= 1024) return {8, 2};
    if (groups <= 2048) return {8, 4};
    return {0, 0};
}

#define FAITH_LAUNCH_SHAPE(KERNEL, WAVES, CH, GRID, ARGS, ...) \
    hipLaunchKernelGGL((KERNEL<T, WAVES, CH __VA_ARGS__>), GRID, dim3(threads_of(WAVES)), 0, stream, ARGS)
#define FAITH_BY_SHAPE(KERNEL, GRID, ARGS, ...)                                                              \
    do {                                                                                                     \
        if (s.waves == 1 && s.groups == 1) FAITH_LAUNCH_SHAPE(KERNEL, 1, 1, GRID, ARGS, __VA_ARGS__);          \
        else if (s.waves == 1) FAITH_LAUNCH_SHAPE(KERNEL, 1, 2, GRID, ARGS, __VA_ARGS__);                      \
        else if (s.waves == 4 && s.groups == 1) FAITH_LAUNCH_SHAPE(KERNEL, 4, 1, GRID, ARGS, __VA_ARGS__);     \
        else if (s.waves == 4 && s.groups == 2) FAITH_LAUNCH_SHAPE(KERNEL, 4, 2, GRID, ARGS, __VA_ARGS__);     \
        else if (s.waves == 4) FAITH_LAUNCH_SHAPE(KERNEL, 4, 3, GRID, ARGS, __VA_ARGS__);                      \
        else if (s.groups == 2) FAITH_LAUNCH_SHAPE(KERNEL, 8, 2, GRID, ARGS, __VA_ARGS__);                     \
        else FAITH_LAUNCH_SHAPE(KERNEL, 8, 4, GRID, ARGS, __VA_ARGS__);                                        \
    } while (0)
#define FAITH_COMMA ,

template <class T> int launch_norm(const NormArgs &g, const Shape &s, hipStream_t stream) {
    if (s.waves == 0) hipLaunchKernelGGL((residual_norm_any<T>), dim3((unsigned)g.rows), dim3(256), 0, stream, g);
    else FAITH_BY_SHAPE(residual_norm, dim3((unsigned)((g.rows + rows_of(s.waves) - 1) / rows_of(s.waves))), g, );
    return check_launch("faith_residual_norm");
}

template <class T> int launch_grad(const NormGradArgs &g, const Shape &s, hipStream_t stream) {
    if (g.rows > 0) {
        if (s.waves == 0) {
            hipLaunchKernelGGL((residual_norm_grad_any<T>), dim3((unsigned)g.rows), dim3(256), 0, stream, g);
            if (g.partial) hipLaunchKernelGGL((residual_norm_columns_any<T>), dim3((unsigned)ceil_div(g.n, 256), (unsigned)g.blocks), dim3(256), 0, stream, g);
        } else {
            const dim3 grid((unsigned)(g.blocks / rows_of(s.waves)));
            if (g.dbias) FAITH_BY_SHAPE(residual_norm_grad, grid, g, FAITH_COMMA true);
            else FAITH_BY_SHAPE(residual_norm_grad, grid, g, FAITH_COMMA false);
        }
    }
    if (g.dweight || g.dbias)
        hipLaunchKernelGGL((residual_norm_columns<T>), dim3((unsigned)ceil_div(g.n, 32), g.dweight && g.dbias ? 2 : 1), dim3(1024), 0, stream, g);
    return check_launch("faith_residual_norm_backward");
}

int norm_shapes(const char *fn, long long rows, int n, int kind, int dtype) {
    // the kernels count along a row in 32 bits, a step of the workgroup past its end
    FAITH_REQUIRE(rows >= 0 && rows < (1LL << 31) && n > 0 && n <= (1 << 30), FAITH_ERR_SHAPE, "%s: %lld rows of %d", fn, rows, n);
    FAITH_REQUIRE(kind >= FAITH_NORM_RMS && kind <= FAITH_NORM_NO_VAR, FAITH_ERR_UNSUPPORTED, "%s: kind %d", fn, kind);
    FAITH_REQUIRE(dtype == FAITH_F32 || dtype == FAITH_BF16 || dtype == FAITH_F16, FAITH_ERR_UNSUPPORTED, "%s: element type %d", fn, dtype);
    return FAITH_OK;
}

// Fewer than 2^32 threads: 256 to a row, or to four of one wavefront each, 512 to a row of eight.  (Four rows to a workgroup would allow more
// than 2^24 rows; they are refused alike, so that the limit does not depend on the width.)
bool one_launch(long long rows, int waves) { return rows < (1LL << 24) && rows * (waves == 8 ? 512 : 256) < (1LL << 32); }

int grad_blocks(long long rows, int waves) {
    if (rows <= 0) return 0;
    const int per = waves == 1 ? 4 : 1;
    const long long groups = (rows + per - 1) / per, most = 2LL * compute_units();
    return (int)(groups < most ? groups : most) * per;
}

}  // namespace

extern "C" int faith_residual_norm(const void *x, const void *residual, const void *weight, const void *bias, void *y, void *sum,
                                   float *stats, float *scales, long long rows, int n, int kind, int dtype, int bits, float eps, void *stream) {
    const int rc = norm_shapes(__func__, rows, n, kind, dtype);
    if (rc != FAITH_OK) return rc;
    FAITH_REQUIRE(bits == 0 || bits == FAITH_BITS_INT8 || bits == FAITH_BITS_E4M3, FAITH_ERR_UNSUPPORTED, "%s: output %d", __func__, bits);
    FAITH_REQUIRE(eps >= 0.f && eps < 1e30f, FAITH_ERR_UNSUPPORTED, "%s: eps must be finite and not negative", __func__);
    if (rows == 0) return FAITH_OK;
    FAITH_NOT_NULL(x);
    FAITH_NOT_NULL(y);
    FAITH_REQUIRE(!bits || scales, FAITH_ERR_NULL, "%s: an output in 8 bits has a scale for each row", __func__);
    const NormArgs g = {x, residual, weight, bias, y, sum, stats, scales, rows, n, kind, bits, eps};
    const bool whole = aligned(x, 16) && aligned(residual, 16) && aligned(weight, 16) && aligned(bias, 16) && aligned(y, 16) && aligned(sum, 16);
    const Shape s = shape_of(n, dtype, whole);
    FAITH_REQUIRE(one_launch(rows, s.waves), FAITH_ERR_UNSUPPORTED, "%s: %lld rows of %d are more than one launch holds", __func__, rows, n);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == FAITH_F32) return launch_norm<float>(g, s, st);
    if (dtype == FAITH_BF16) return launch_norm<__bf16>(g, s, st);
    return launch_norm<_Float16>(g, s, st);
}

extern "C" int faith_residual_norm_blocks(long long rows, int n, int dtype) { return grad_blocks(rows, shape_of(n, dtype, true).waves); }

extern "C" int faith_residual_norm_backward(const void *dy, const void *dsum, const void *sum, const void *weight, const float *stats,
                                            void *dx, void *dweight, void *dbias, float *partial, long long rows, int n, int kind,
                                            int dtype, void *stream) {
    const int rc = norm_shapes(__func__, rows, n, kind, dtype);
    if (rc != FAITH_OK) return rc;
    FAITH_REQUIRE(!(dweight || dbias) || partial || rows == 0, FAITH_ERR_NULL, "%s: the parameters' gradients need scratch", __func__);
    FAITH_REQUIRE(rows < (1LL << 24), FAITH_ERR_UNSUPPORTED, "%s: %lld rows are more than one launch holds", __func__, rows);
    if (rows > 0) {
        FAITH_NOT_NULL(dy);
        FAITH_NOT_NULL(sum);
        FAITH_NOT_NULL(stats);
        FAITH_NOT_NULL(dx);
    }
    const bool whole = aligned(dy, 16) && aligned(dsum, 16) && aligned(sum, 16) && aligned(weight, 16) && aligned(dx, 16) && aligned(partial, 16);
    const Shape s = shape_of(n, dtype, whole);
    // rows of `partial` by the aligned rule, which is what the caller made room for; the kernel for any width writes as many
    const int blocks = grad_blocks(rows, shape_of(n, dtype, true).waves);
    if (!dweight && !dbias) partial = nullptr;
    const NormGradArgs g = {dy, dsum, sum, weight, stats, dx, dweight, dbias, partial, partial ? partial + 2LL * n * blocks : nullptr, rows, n, kind, blocks};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == FAITH_F32) return launch_grad<float>(g, s, st);
    if (dtype == FAITH_BF16) return launch_grad<__bf16>(g, s, st);
    return launch_grad<_Float16>(g, s, st);
}
