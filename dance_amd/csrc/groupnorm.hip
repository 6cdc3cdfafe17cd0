// groupnorm.hip -- GroupNorm with an activation on channels-last maps, and its backward pass.
//
//   x (b, hw, c) with the channels innermost, G groups of gc = c / G channels; over a group's gc * hw values
//     mu = mean x,  rstd = 1 / sqrt(mean (x - mu)^2 + eps),  xh = (x - mu) rstd
//     z = xh w + beta,  y = act(z),  act one of none, ReLU, SiLU
//   backward, dz = dy act'(z):
//     dbeta = sum dz,  dw = sum dz xh                                       (over images and pixels)
//     dx = rstd (w dz - m1 - xh m2),  m1 = mean_group(w dz),  m2 = mean_group(w dz xh)
//
// Memory bound (about 8 operations an element forward, 24 backward).  The map is read twice: a pass for the
// sums, a pass that applies them.  No atomics: workgroups store partial sums, folded in a fixed order, so
// two runs give the same bits.
//
// Thread mapping of every pass: a thread owns one 16-byte vector of channels for good and walks down the
// pixels, so per-channel constants stay in registers and a wave reads whole 1 KB rows.
#include "common.h"

namespace {

using dance::ceil_div;
using dance::launch_check;

template <typename T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };

// 16 bytes of channels at any element alignment (a map whose pixels are not 16-byte aligned, for instance a
// channel slice): the hardware takes unaligned 128-bit accesses
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Word { T v[16 / sizeof(T)]; };

// Reads and writes of maps larger than the 256 MB cache can serve twice bypass it (STREAM): what is read for the last
// time and what is written would only push out what is read again.  (8, 256, 200, 304) fp32, us: statistics 124 -> 86,
// because they no longer wait for the outputs of the call before to be written back, apply 176 -> 158.  Not where in-
// and output fit: there the next layer finds its input in the cache.
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ float load_any(const void *p, int dtype, long long i)
{
    if (dtype == DANCE_F32)
        return ((const float *)p)[i];
    return dtype == DANCE_F16 ? (float)((const _Float16 *)p)[i] : (float)((const __bf16 *)p)[i];
}

__device__ __forceinline__ float load_affine(const void *p, int dtype, int i, float otherwise)
{
    return p == nullptr ? otherwise : load_any(p, dtype, i);
}

__device__ __forceinline__ void store_affine(void *p, int dtype, int i, double v)
{
    if (dtype == DANCE_F32)
        ((float *)p)[i] = (float)v;
    else if (dtype == DANCE_F16)
        ((_Float16 *)p)[i] = (_Float16)(float)v;
    else
        ((__bf16 *)p)[i] = (__bf16)(float)v;
}

constexpr int MAX_THREADS = 512;        // of a workgroup: 256 registers a thread, no pass spills

// What a workgroup covers: a slab of whole groups' channels, a chunk of an image's pixels.
struct GnDims {
    long long hw, chunk;        // pixels of an image; pixels of a workgroup
    int c, groups, gc, nch;     // channels and groups of the map; channels of a group; workgroups along the pixels
    int cs, cv, rows;           // channels of a slab; its vectors; pixels a workgroup covers at once
};

// the channel of the slab that element j of vector v holds.  WHOLE (whole vectors): 16 consecutive bytes;
// otherwise element j of the whole row of vectors, so that a wave's scalar accesses are consecutive
template <typename T, bool WHOLE> __device__ __forceinline__ int channel_of(const GnDims &d, int v, int j)
{
    return WHOLE ? v * Vec<T>::N + j : v + j * d.cv;
}

// pixel: the slab's first channel
template <typename T, bool WHOLE, bool STREAM = false>
__device__ __forceinline__ Word<T> load_word(const T *pixel, const GnDims &d, int v)
{
    if (WHOLE && STREAM)
        return __builtin_bit_cast(
            Word<T>, __builtin_nontemporal_load(reinterpret_cast<const u32x4_any *>(pixel + v * Vec<T>::N)));
    if (WHOLE)
        return *reinterpret_cast<const Word<T> *>(pixel + v * Vec<T>::N);
    Word<T> w;
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) {
        const int ch = v + j * d.cv;
        w.v[j] = ch < d.cs ? pixel[ch] : (T)0.0f;
    }
    return w;
}

template <typename T, bool WHOLE, bool STREAM = false>
__device__ __forceinline__ void store_word(T *pixel, const Word<T> &w, const GnDims &d, int v)
{
    if (WHOLE && STREAM) {
        __builtin_nontemporal_store(__builtin_bit_cast(u32x4_any, w), reinterpret_cast<u32x4_any *>(pixel + v * Vec<T>::N));
        return;
    }
    if (WHOLE) {
        *reinterpret_cast<Word<T> *>(pixel + v * Vec<T>::N) = w;
        return;
    }
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) {
        const int ch = v + j * d.cv;
        if (ch < d.cs)
            pixel[ch] = w.v[j];
    }
}

// ------------------------------------------------------------------- sums inside a workgroup
// red [rows][units] pairs -> red [0][units], a fixed order: a unit is folded by `lanes` neighbouring threads
// (a power of two up to a wave), rows lane, lane + lanes, ... each, then a butterfly over them
template <typename A> __device__ __forceinline__ void fold_rows(A (*red)[2], int rows, int units)
{
    int lanes = 64;
    while (lanes > 1 && (lanes * units > (int)blockDim.x || lanes >= 2 * rows))
        lanes >>= 1;
    __syncthreads();
    if (rows == 1)
        return;
    const int lane = threadIdx.x & (lanes - 1), step = blockDim.x / lanes;
    for (int u0 = 0; u0 < units; u0 += step) {
        const int u = u0 + threadIdx.x / lanes;
        A s = 0, q = 0;
        if (u < units)
            for (int r = lane; r < rows; r += lanes) {
                s += red[r * units + u][0];
                q += red[r * units + u][1];
            }
        for (int m = lanes >> 1; m >= 1; m >>= 1) {
            s += __shfl_xor(s, m, 64);
            q += __shfl_xor(q, m, 64);
        }
        // row 0 of a unit is read by its own lanes alone, and they have read it
        if (u < units && lane == 0) {
            red[u][0] = s;
            red[u][1] = q;
        }
    }
    __syncthreads();
}

// f(group, sum of its `per` units' pairs) for every group of the slab, red [units]; f runs in one thread a group
template <typename A, typename F>
__device__ __forceinline__ void for_group_sums(const A (*red)[2], int groups, int per, F &&f)
{
    int lanes = 64;
    while (lanes > 1 && (lanes * groups > (int)blockDim.x || lanes >= 2 * per))
        lanes >>= 1;
    const int lane = threadIdx.x & (lanes - 1), step = blockDim.x / lanes;
    for (int g0 = 0; g0 < groups; g0 += step) {
        const int g = g0 + threadIdx.x / lanes;
        A s = 0, q = 0;
        if (g < groups)
            for (int k = lane; k < per; k += lanes) {
                s += red[g * per + k][0];
                q += red[g * per + k][1];
            }
        for (int m = lanes >> 1; m >= 1; m >>= 1) {
            s += __shfl_xor(s, m, 64);
            q += __shfl_xor(q, m, 64);
        }
        if (g < groups && lane == 0)
            f(g, s, q);
    }
}

// ------------------------------------------------------------------------------------- statistics
// A unit of a workgroup's sums is a channel, or a whole vector where no vector holds two groups (gc a multiple of it): an
// eighth or a quarter of the LDS and of the folding.
template <typename T, bool WHOLE> __device__ __forceinline__ bool vector_units(const GnDims &d)
{
    return WHOLE && d.gc % Vec<T>::N == 0;
}

// Sums in fp64 of d = x - pivot and d d, the pivot of a group being its first value (channel g gc of pixel 0) in every
// workgroup.  The variance is the difference of mean d d and (mean d)^2; the pivot is one of the n values, so
// (mean d)^2 <= n var, and the roundings cost the variance a few n 2^-53 of itself at most, whatever the mean.  (Sums of
// x and x x: mean 1e6 and spread 0.1 left rstd 1e-3 off.)  An fp64 subtraction or fma is as fast as an fp32 one here;
// the pass stays bound by its loads.
template <typename T>
__device__ __forceinline__ void add_word(double (&s)[Vec<T>::N], double (&q)[Vec<T>::N], const Word<T> &w,
                                         const double (&pivot)[Vec<T>::N])
{
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) {
        const double x = (double)(float)w.v[j] - pivot[j];
        s[j] += x;
        q[j] = fma(x, x, q[j]);
    }
}

// pixel0: the slab's first channel of pixel 0.  A load a channel, behind the batch of vectors that the sums start with;
// sharing the groups' pivots through LDS instead was no faster (statistics of (3, 96, 67, 101) fp16, groups of 3, 7.4
// against 8.0 us, of (1, 256, 200, 304) bf16 10.5 against 10.1; k_gn_one 7.0 against 6.8).
template <typename T, bool WHOLE>
__device__ __forceinline__ void load_pivots(double (&pivot)[Vec<T>::N], const T *pixel0, const GnDims &d, int v)
{
    const bool vu = vector_units<T, WHOLE>(d);
    int first = channel_of<T, WHOLE>(d, v, 0) / d.gc * d.gc;                   // of the group
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) {
        const int c = min(channel_of<T, WHOLE>(d, v, j), d.cs - 1);
        first = !WHOLE ? c / d.gc * d.gc : c == first + d.gc ? c : first;
        pivot[j] = vu && j > 0 ? pivot[0] : (double)(float)pixel0[first];
    }
}

// A thread's sums into red [rows][units].
template <typename T, bool WHOLE>
__device__ __forceinline__ void put_units(double (*red)[2], const double (&s)[Vec<T>::N], const double (&q)[Vec<T>::N],
                                          const GnDims &d, int row, int v)
{
    constexpr int N = Vec<T>::N;
    if (vector_units<T, WHOLE>(d)) {
        double ss = 0.0, qq = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            ss += s[j];
            qq += q[j];
        }
        red[row * d.cv + v][0] = ss;
        red[row * d.cv + v][1] = qq;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int u = row * d.cv * N + channel_of<T, WHOLE>(d, v, j);
            red[u][0] = s[j];
            red[u][1] = q[j];
        }
    }
}

__device__ __forceinline__ void finish_group(double pivot, double s, double q, double count, double eps, double &mean, double &rstd)
{
    s /= count;
    mean = pivot + s;
    double var = q / count - s * s;
    var = var < 0.0 ? 0.0 : var;                          // (a NaN stays one: infinities in the map give NaN, as in torch)
    rstd = 1.0 / sqrt(var + eps);
}

// Vectors of a thread that are loaded at once; a vector of scalar loads counts for several
template <bool WHOLE> constexpr int IN_FLIGHT = WHOLE ? 8 : 2;

// FL pixels of a thread from pixel p on, rows apart; those past the chunk are its last one again, so that
// every load is issued
template <typename T, bool WHOLE, bool STREAM, int FL>
__device__ __forceinline__ void load_batch(Word<T> (&w)[FL], const T *x, long long pixel_stride, long long p, long long p1,
                                           const GnDims &d, int v)
{
    if (p + (FL - 1) * d.rows < p1) {
        const T *xp = x + p * pixel_stride;
        const long long step = d.rows * pixel_stride;
#pragma unroll
        for (int u = 0; u < FL; ++u)
            w[u] = load_word<T, WHOLE, STREAM>(xp + u * step, d, v);
    } else {
#pragma unroll
        for (int u = 0; u < FL; ++u)
            w[u] = load_word<T, WHOLE, STREAM>(x + min(p + u * d.rows, p1 - 1) * pixel_stride, d, v);
    }
}

// f(u) for the pixels p + u rows of a batch that lie in the chunk
template <int FL, typename F> __device__ __forceinline__ void for_batch(long long p, long long p1, int rows, F &&f)
{
    if (p + (FL - 1) * rows < p1) {
#pragma unroll
        for (int u = 0; u < FL; ++u)
            f(u);
    } else {
#pragma unroll
        for (int u = 0; u < FL; ++u)
            if (p + u * rows < p1)
                f(u);
    }
}

// partial (b, nch, groups, 2): sums of a chunk of pixels.  grid: b * nch workgroups, slab = the whole map.  Bound by
// memory: (8, 256, 200, 304) fp32 86 us (5.8 TB/s), (1, 256, 200, 304) bf16 10.5 us (3.0 TB/s, start and reduction show).
template <typename T, bool WHOLE>
__global__ __launch_bounds__(MAX_THREADS) void k_gn_stats(const T *__restrict__ x, long long image_stride,
                                                   long long pixel_stride, double *__restrict__ partial, GnDims d)
{
    constexpr int N = Vec<T>::N, FL = IN_FLIGHT<WHOLE>;
    extern __shared__ __align__(16) double red[][2];
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
    if (row < d.rows) {
        double s[N] = {}, q[N] = {};
        const T *xp = x + b * image_stride;
        Word<T> w[FL], next[FL];
        long long p = p0 + row;
        load_batch<T, WHOLE, false>(w, xp, pixel_stride, p, p1, d, v);
        double pivot[N];
        load_pivots<T, WHOLE>(pivot, xp, d, v);
        for (; p < p1; p += FL * d.rows) {
            if (p + FL * d.rows < p1)
                load_batch<T, WHOLE, false>(next, xp, pixel_stride, p + FL * d.rows, p1, d, v);
            for_batch<FL>(p, p1, d.rows, [&](int u) { add_word<T>(s, q, w[u], pivot); });
#pragma unroll
            for (int u = 0; u < FL; ++u)
                w[u] = next[u];
        }
        put_units<T, WHOLE>(red, s, q, d, row, v);
    }
    const bool vu = vector_units<T, WHOLE>(d);
    fold_rows(red, d.rows, vu ? d.cv : d.cv * N);
    double *out = partial + (long long)blockIdx.x * d.groups * 2;
    for_group_sums(red, d.groups, vu ? d.gc / N : d.gc, [&](int g, double s, double q) {
        out[g * 2] = s;
        out[g * 2 + 1] = q;
    });
}

// ----------------------------------------------------------------------------- a channel's constants
// The mean as a sum of two floats: x - mu keeps its low bits when the mean is large against the spread.  With
// e = x - mu:  z = e (rstd w) + beta.  Written once an image and channel (by k_gn_finish or k_gn_one), read
// as one 16-byte word: gathering mean, rstd, weight and bias of each of its channels cost a thread of the
// apply pass two dozen dependent loads (17.5 against 15.0 us on a (1, 256, 200, 304) bf16 map).
struct alignas(16) Channel {
    float mhi, mlo, rw, beta;
};

// What the forward call leaves for the backward one, in this order: the groups' mean and rstd, the channels'
// constants, the weight as fp32.
struct Saved {
    double *stats;              // (b, groups, 2)
    Channel *channels;          // (b, c)
    float *weight;              // (c)
};

__host__ __device__ inline Saved saved_at(void *p, int b, int c, int groups)
{
    Saved s;
    s.stats = (double *)p;
    s.channels = (Channel *)(s.stats + (size_t)b * groups * 2);
    s.weight = (float *)(s.channels + (size_t)b * c);
    return s;
}

__device__ __forceinline__ Channel channel_constants(double mean, double rstd, float weight, float beta)
{
    Channel k;
    k.mhi = (float)mean;
    k.mlo = (float)(mean - (double)k.mhi);
    k.rw = (float)(rstd * (double)weight);
    k.beta = beta;
    return k;
}

__device__ __forceinline__ float centred(float x, const Channel &k) { return (x - k.mhi) - k.mlo; }

// partial (b, nch, groups, 2) -> the saved words of a group and its channels.  grid: (groups, b).  3 - 5 us: a launch,
// the reads of a group's partial sums, the affine parameters and the pivot beside them.
__global__ __launch_bounds__(256) void k_gn_finish(const double *__restrict__ partial, const void *__restrict__ x, int dtype,
                                                   long long image_stride, Saved out, const void *weight, const void *bias,
                                                   int affine_dtype, double count, double eps, GnDims d)
{
    __shared__ double red[4][2];
    const int g = blockIdx.x, b = blockIdx.y;
    double s = 0.0, q = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < d.nch; i += 256) {
        const double2 p = *reinterpret_cast<const double2 *>(partial + (((long long)b * d.nch + i) * d.groups + g) * 2);
        s += p.x;
        q += p.y;
    }
    // (the pivot and the affine parameters arrive meanwhile)
    const double pivot = (double)load_any(x, dtype, b * image_stride + g * d.gc);
    int cl = threadIdx.x;
    float w = 1.0f, beta = 0.0f;
    if (cl < d.gc) {
        w = load_affine(weight, affine_dtype, g * d.gc + cl, 1.0f);
        beta = load_affine(bias, affine_dtype, g * d.gc + cl, 0.0f);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        s += __shfl_xor(s, m, 64);
        q += __shfl_xor(q, m, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6][0] = s;
        red[threadIdx.x >> 6][1] = q;
    }
    __syncthreads();
    double mean, rstd;
    finish_group(pivot, red[0][0] + red[1][0] + red[2][0] + red[3][0], red[0][1] + red[1][1] + red[2][1] + red[3][1], count,
                 eps, mean, rstd);
    if (threadIdx.x == 0) {
        double *o = out.stats + ((long long)b * d.groups + g) * 2;
        o[0] = mean;
        o[1] = rstd;
    }
    while (cl < d.gc) {
        const int c = g * d.gc + cl;
        out.channels[(long long)b * d.c + c] = channel_constants(mean, rstd, w, beta);
        if (b == 0)
            out.weight[c] = w;
        cl += 256;
        if (cl < d.gc) {
            w = load_affine(weight, affine_dtype, g * d.gc + cl, 1.0f);
            beta = load_affine(bias, affine_dtype, g * d.gc + cl, 0.0f);
        }
    }
}

// ------------------------------------------------------------------------------------------ apply
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

__device__ __forceinline__ float activate(float z, int act)
{
    if (act == DANCE_ACT_RELU)
        return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (act == DANCE_ACT_SILU)
        return z * sigmoid(z);
    return z;
}

template <typename T> __device__ __forceinline__ Word<T> apply_word(const Word<T> &w, const Channel (&k)[Vec<T>::N], int act)
{
    Word<T> r;
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j)
        r.v[j] = (T)activate(fmaf(centred((float)w.v[j], k[j]), k[j].rw, k[j].beta), act);
    return r;
}

// grid: b * nch workgroups, slab = the whole map.  Bound by memory: (8, 256, 200, 304) fp32 158 us (6.3 TB/s),
// (1, 256, 200, 304) bf16 12.5 us (5.0 TB/s).
template <typename T, bool WHOLE, int ACT, bool STREAM>
__global__ __launch_bounds__(MAX_THREADS) void k_gn_apply(const T *__restrict__ x, long long image_stride,
                                                          long long pixel_stride, const Channel *__restrict__ channels,
                                                          T *__restrict__ y, GnDims d)
{
    constexpr int N = Vec<T>::N, FL = IN_FLIGHT<WHOLE>;
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    if (row >= d.rows)
        return;
    const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
    const T *xp = x + b * image_stride;
    T *yp = y + b * d.hw * d.c;
    Word<T> w[FL], next[FL];
    long long p = p0 + row;
    load_batch<T, WHOLE, STREAM>(w, xp, pixel_stride, p, p1, d, v);        // in flight while the constants arrive
    Channel k[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
        k[j] = channels[(long long)b * d.c + min(channel_of<T, WHOLE>(d, v, j), d.c - 1)];
    const long long step = (long long)d.rows * d.c;
    for (; p < p1; p += FL * d.rows) {
        if (p + FL * d.rows < p1)
            load_batch<T, WHOLE, STREAM>(next, xp, pixel_stride, p + FL * d.rows, p1, d, v);
        T *yq = yp + p * d.c;
        for_batch<FL>(p, p1, d.rows, [&](int u) { store_word<T, WHOLE, STREAM>(yq + u * step, apply_word<T>(w[u], k, ACT), d, v); });
#pragma unroll
        for (int u = 0; u < FL; ++u)
            w[u] = next[u];
    }
}

// Small maps: a workgroup owns a slab of whole groups of an image over all its pixels, at most U vectors a
// thread, and keeps them in registers: one read, one launch.  grid: b * slabs.  (1, 256, 25, 38) fp32: 6.8 us, the trips
// to memory and the two reductions one after the other.
template <typename T, bool WHOLE, int U>
__global__ __launch_bounds__(MAX_THREADS) void k_gn_one(const T *__restrict__ x, long long image_stride, long long pixel_stride,
                                                 const void *weight, const void *bias, int affine_dtype, double eps,
                                                 int act, T *__restrict__ y, Saved out, GnDims d)
{
    constexpr int N = Vec<T>::N;
    extern __shared__ __align__(16) double lds[][2];
    const int slabs = d.c / d.cs, b = blockIdx.x / slabs, c0 = (blockIdx.x - b * slabs) * d.cs;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    const bool live = row < d.rows;
    const int sg = d.cs / d.gc;
    float *pivots = reinterpret_cast<float *>(lds);               // of the slab's groups
    double (*red)[2] = lds + (sg + 3) / 4;
    const T *xp = x + b * image_stride + c0;
    Word<T> w[U];
    double s[N] = {}, q[N] = {};
    if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            w[u] = load_word<T, WHOLE>(xp + min((long long)(row + u * d.rows), d.hw - 1) * pixel_stride, d, v);
        double pivot[N];
        load_pivots<T, WHOLE>(pivot, xp, d, v);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * d.rows < d.hw)
                add_word<T>(s, q, w[u], pivot);
        put_units<T, WHOLE>(red, s, q, d, row, v);
    }
    for (int g = threadIdx.x; g < sg; g += blockDim.x)
        pivots[g] = (float)xp[g * d.gc];
    const bool vu = vector_units<T, WHOLE>(d);
    const int units = vu ? d.cv : d.cv * N;
    fold_rows(red, d.rows, units);
    const double (*sums)[2] = red;
    double (*done)[2] = red + units;                      // behind row 0, whose sums are still read
    Channel *constants = reinterpret_cast<Channel *>(done + sg);
    double *st = out.stats + ((long long)b * d.groups + c0 / d.gc) * 2;
    for_group_sums(sums, sg, vu ? d.gc / N : d.gc, [&](int g, double gs, double gq) {
        finish_group((double)pivots[g], gs, gq, (double)d.gc * (double)d.hw, eps, done[g][0], done[g][1]);
        st[g * 2] = done[g][0];
        st[g * 2 + 1] = done[g][1];
    });
    __syncthreads();
    for (int cl = threadIdx.x; cl < d.cs; cl += blockDim.x) {
        const float wt = load_affine(weight, affine_dtype, c0 + cl, 1.0f);
        const Channel k = channel_constants(done[cl / d.gc][0], done[cl / d.gc][1], wt,
                                            load_affine(bias, affine_dtype, c0 + cl, 0.0f));
        constants[cl] = k;
        out.channels[(long long)b * d.c + c0 + cl] = k;
        if (b == 0)
            out.weight[c0 + cl] = wt;
    }
    __syncthreads();
    if (!live)
        return;
    Channel k[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
        k[j] = constants[min(channel_of<T, WHOLE>(d, v, j), d.cs - 1)];
    T *yp = y + b * d.hw * d.c + c0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (row + u * d.rows < d.hw)
            store_word<T, WHOLE>(yp + (long long)(row + u * d.rows) * d.c, apply_word<T>(w[u], k, act), d, v);
}

// --------------------------------------------------------------------------------------- backward
// dz = dy act'(z) and e = x - mu of one element.  ReLU: which side of zero z lies on decides whole gradients,
// so a z within fp32 rounding of zero is evaluated again in fp64 (the rounding of z is a few 2^-24 of its two
// terms; 2^-20 of them covers it, one element in a million takes the branch).  st: the group's mean and rstd,
// weight: the channel's, read there only.
__device__ __forceinline__ float grad_z(float dy, float x, const Channel &k, const double *st, const float *weight, int act,
                                        float &e)
{
    e = centred(x, k);
    if (act == DANCE_ACT_NONE)
        return dy;
    const float t = e * k.rw, z = t + k.beta;
    if (act == DANCE_ACT_RELU) {
        bool on = z > 0.0f;
        if (fabsf(z) <= 9.5367431640625e-7f * (fabsf(t) + fabsf(k.beta)))
            on = ((double)x - st[0]) * st[1] * (double)*weight + (double)k.beta > 0.0;
        return on ? dy : (z != z ? z : 0.0f);
    }
    const float s = sigmoid(z);
    return dy * (s * (1.0f + z * (1.0f - s)));
}

// dx = rstd (w dz - m1 - xh m2) = dz (rstd w) - a1 - e a2,  a1 = rstd m1,  a2 = rstd^2 m2
__device__ __forceinline__ float grad_x(float dz, float e, const Channel &k, float2 a)
{
    return fmaf(dz, k.rw, -fmaf(e, a.y, a.x));
}

template <bool WHOLE> constexpr int GRAD_IN_FLIGHT = WHOLE ? 4 : 1;       // of each of the two maps

// Per-channel sums of dz and dz xh over a chunk of pixels: partial (b, nch, c, 2) fp32, a thread's own sums
// of at most chunk / rows terms.  grid: b * nch, slab = the whole map.  Bound by memory: (2, 256, 200, 304) fp32 45 us
// (5.5 TB/s).
template <typename T, bool WHOLE, int ACT>
__global__ __launch_bounds__(MAX_THREADS) void k_gn_grad_sums(const T *__restrict__ dy, long long dy_image,
                                                              long long dy_pixel, const T *__restrict__ x,
                                                              long long image_stride, long long pixel_stride, Saved saved,
                                                              float *__restrict__ partial, GnDims d)
{
    constexpr int N = Vec<T>::N, FL = GRAD_IN_FLIGHT<WHOLE>;
    extern __shared__ __align__(16) float redf[][2];
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    const int units = d.cv * N;
    const double *st = saved.stats + (long long)b * d.groups * 2;
    if (row < d.rows) {
        const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
        const T *xp = x + b * image_stride, *dp = dy + b * dy_image;
        Word<T> w[FL], g[FL];
        long long p = p0 + row;
        load_batch<T, WHOLE, false>(w, xp, pixel_stride, p, p1, d, v);
        load_batch<T, WHOLE, false>(g, dp, dy_pixel, p, p1, d, v);
        Channel k[N];
        float s[N], q[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            k[j] = saved.channels[(long long)b * d.c + min(channel_of<T, WHOLE>(d, v, j), d.c - 1)];
            s[j] = q[j] = 0.0f;
        }
        while (p < p1) {
            for_batch<FL>(p, p1, d.rows, [&](int u) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int c = min(channel_of<T, WHOLE>(d, v, j), d.c - 1);
                    float e;
                    const float dz = grad_z((float)g[u].v[j], (float)w[u].v[j], k[j], st + c / d.gc * 2, saved.weight + c,
                                            ACT, e);
                    s[j] += dz;
                    q[j] = fmaf(dz, e, q[j]);
                }
            });
            p += FL * d.rows;
            if (p < p1) {
                load_batch<T, WHOLE, false>(w, xp, pixel_stride, p, p1, d, v);
                load_batch<T, WHOLE, false>(g, dp, dy_pixel, p, p1, d, v);
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float *o = redf[row * units + channel_of<T, WHOLE>(d, v, j)];
            o[0] = s[j];
            o[1] = q[j];
        }
    }
    fold_rows(redf, d.rows, units);
    float *out = partial + (long long)blockIdx.x * d.c * 2;
    for (int c = threadIdx.x; c < d.c; c += blockDim.x)
        *reinterpret_cast<float2 *>(out + c * 2) = float2{redf[c][0], redf[c][1] * (float)st[c / d.gc * 2 + 1]};
}

// partial (b, nch, c, 2) -> sums (b, c, 2) in fp64 and a group's a1, a2 of grad_x.  grid: (groups, b).  Neighbouring
// threads read neighbouring channels of a chunk, the chunks are dealt to rows of threads.  (2, 256, 200, 304): 7.3 us.
__global__ __launch_bounds__(MAX_THREADS) void k_gn_grad_finish(const float *__restrict__ partial, Saved saved,
                                                                double *__restrict__ sums, float2 *__restrict__ means,
                                                                GnDims d)
{
    __shared__ __align__(16) double red[MAX_THREADS][2];
    const int g = blockIdx.x, b = blockIdx.y;
    double m1 = 0.0, m2 = 0.0;                            // thread 0's
    for (int c0 = 0; c0 < d.gc; c0 += MAX_THREADS) {
        const int width = min(d.gc - c0, MAX_THREADS), rows = MAX_THREADS / width;
        const int row = threadIdx.x / width, cl = threadIdx.x - row * width, c = g * d.gc + c0 + cl;
        __syncthreads();                                  // (the channels before have been read)
        if (row < rows) {
            double s = 0.0, q = 0.0;
#pragma unroll 8
            for (int i = row; i < d.nch; i += rows) {
                const float2 p = *reinterpret_cast<const float2 *>(partial + (((long long)b * d.nch + i) * d.c + c) * 2);
                s += (double)p.x;
                q += (double)p.y;
            }
            red[row * width + cl][0] = s;
            red[row * width + cl][1] = q;
        }
        fold_rows(red, rows, width);
        if (row == 0) {
            const double s = red[cl][0], q = red[cl][1], w = (double)saved.weight[c];
            sums[((long long)b * d.c + c) * 2] = s;
            sums[((long long)b * d.c + c) * 2 + 1] = q;
            red[cl][0] = w * s;
            red[cl][1] = w * q;
        }
        __syncthreads();
        const double (*weighted)[2] = red;
        for_group_sums(weighted, 1, width, [&](int, double s, double q) {
            m1 += s;
            m2 += q;
        });
    }
    if (threadIdx.x == 0) {
        const double count = (double)d.gc * (double)d.hw, rstd = saved.stats[((long long)b * d.groups + g) * 2 + 1];
        means[(long long)b * d.groups + g] = float2{(float)(rstd * m1 / count), (float)(rstd * rstd * m2 / count)};
    }
}

// dw, dbeta: the images' sums added in order.  One thread a channel.
__device__ __forceinline__ void affine_gradient(const double *sums, void *dweight, void *dbias, int affine_dtype, int b,
                                                int c, int ch)
{
    double s = 0.0, q = 0.0;
    for (int i = 0; i < b; ++i) {
        s += sums[((long long)i * c + ch) * 2];
        q += sums[((long long)i * c + ch) * 2 + 1];
    }
    if (dweight)
        store_affine(dweight, affine_dtype, ch, q);
    if (dbias)
        store_affine(dbias, affine_dtype, ch, s);
}

// The same for many images: 16 channels a workgroup, the images dealt to its 32 rows of threads, which are folded in
// order.  A thread a channel took 10 ms for (65535, 4) and 0.5 ms for 2048 images of 256 channels.
constexpr int AFFINE_CHANNELS = 16;
__global__ __launch_bounds__(MAX_THREADS) void k_gn_grad_affine(const double *__restrict__ sums, void *dweight, void *dbias,
                                                                int affine_dtype, int b, int c)
{
    __shared__ __align__(16) double red[MAX_THREADS][2];
    constexpr int ROWS = MAX_THREADS / AFFINE_CHANNELS;
    const int row = threadIdx.x / AFFINE_CHANNELS, cl = threadIdx.x % AFFINE_CHANNELS, ch = blockIdx.x * AFFINE_CHANNELS + cl;
    double s = 0.0, q = 0.0;
    if (ch < c)
#pragma unroll 8
        for (int i = row; i < b; i += ROWS) {
            const double2 p = *reinterpret_cast<const double2 *>(sums + ((long long)i * c + ch) * 2);
            s += p.x;
            q += p.y;
        }
    red[threadIdx.x][0] = s;
    red[threadIdx.x][1] = q;
    fold_rows(red, ROWS, AFFINE_CHANNELS);
    if (row == 0 && ch < c) {
        if (dweight)
            store_affine(dweight, affine_dtype, ch, red[cl][1]);
        if (dbias)
            store_affine(dbias, affine_dtype, ch, red[cl][0]);
    }
}

// grid: b * nch workgroups, slab = the whole map; dx may be NULL (only dw, dbeta wanted: one workgroup then).
// The last workgroups write dw and dbeta, too: no launch of their own.  Bound by memory: (2, 256, 200, 304) fp32 54 us
// (6.9 TB/s).
template <typename T, bool WHOLE, int ACT, bool STREAM>
__global__ __launch_bounds__(MAX_THREADS) void k_gn_grad_apply(const T *__restrict__ dy, long long dy_image,
                                                               long long dy_pixel, const T *__restrict__ x,
                                                               long long image_stride, long long pixel_stride, Saved saved,
                                                               const float2 *__restrict__ means,
                                                               const double *__restrict__ sums, T *__restrict__ dx,
                                                               void *dweight, void *dbias, int affine_dtype, int images,
                                                               GnDims d)
{
    constexpr int N = Vec<T>::N, FL = GRAD_IN_FLIGHT<WHOLE>;
    if (dweight != nullptr || dbias != nullptr)
        for (int c = (gridDim.x - 1 - blockIdx.x) * blockDim.x + threadIdx.x; c < d.c; c += gridDim.x * blockDim.x)
            affine_gradient(sums, dweight, dbias, affine_dtype, images, d.c, c);
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    if (row >= d.rows || dx == nullptr)
        return;
    const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
    const T *xp = x + b * image_stride, *dp = dy + b * dy_image;
    T *op = dx + b * d.hw * d.c;
    Word<T> w[FL], g[FL];
    long long p = p0 + row;
    load_batch<T, WHOLE, STREAM>(w, xp, pixel_stride, p, p1, d, v);
    load_batch<T, WHOLE, STREAM>(g, dp, dy_pixel, p, p1, d, v);
    const double *st = saved.stats + (long long)b * d.groups * 2;
    Channel k[N];
    float2 a[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int c = min(channel_of<T, WHOLE>(d, v, j), d.c - 1);
        k[j] = saved.channels[(long long)b * d.c + c];
        a[j] = means[(long long)b * d.groups + c / d.gc];
    }
    const long long step = (long long)d.rows * d.c;
    while (p < p1) {
        T *oq = op + p * d.c;
        for_batch<FL>(p, p1, d.rows, [&](int u) {
            Word<T> r;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int c = min(channel_of<T, WHOLE>(d, v, j), d.c - 1);
                float e;
                const float dz = grad_z((float)g[u].v[j], (float)w[u].v[j], k[j], st + c / d.gc * 2, saved.weight + c, ACT, e);
                r.v[j] = (T)grad_x(dz, e, k[j], a[j]);
            }
            store_word<T, WHOLE, STREAM>(oq + u * step, r, d, v);
        });
        p += FL * d.rows;
        if (p < p1) {
            load_batch<T, WHOLE, STREAM>(w, xp, pixel_stride, p, p1, d, v);
            load_batch<T, WHOLE, STREAM>(g, dp, dy_pixel, p, p1, d, v);
        }
    }
}

// The backward pass of small maps as k_gn_one is the forward's: x and dy of a slab in registers.  sums
// (b, c, 2) for k_gn_grad_affine, or, of a single image, dw and dbeta themselves.  grid: b * slabs.  (2, 256, 25, 38)
// bf16: 12 us.
template <typename T, bool WHOLE, int U>
__global__ __launch_bounds__(MAX_THREADS) void k_gn_grad_one(const T *__restrict__ dy, long long dy_image,
                                                             long long dy_pixel, const T *__restrict__ x,
                                                             long long image_stride, long long pixel_stride, Saved saved,
                                                             int act, T *__restrict__ dx, void *dweight, void *dbias,
                                                             int affine_dtype, double *__restrict__ sums, int images,
                                                             GnDims d)
{
    constexpr int N = Vec<T>::N;
    extern __shared__ __align__(16) float redf[][2];
    const int slabs = d.c / d.cs, b = blockIdx.x / slabs, c0 = (blockIdx.x - b * slabs) * d.cs;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    const bool live = row < d.rows;
    const int units = d.cv * N, sg = d.cs / d.gc;
    const T *xp = x + b * image_stride + c0, *dp = dy + b * dy_image + c0;
    const double *st = saved.stats + ((long long)b * d.groups + c0 / d.gc) * 2;
    const float *weight = saved.weight + c0;
    Word<T> w[U], g[U];
    Channel k[N];
    if (live) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long pp = min((long long)(row + u * d.rows), d.hw - 1);
            w[u] = load_word<T, WHOLE>(xp + pp * pixel_stride, d, v);
            g[u] = load_word<T, WHOLE>(dp + pp * dy_pixel, d, v);
        }
        float s[N], q[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            k[j] = saved.channels[(long long)b * d.c + c0 + min(channel_of<T, WHOLE>(d, v, j), d.cs - 1)];
            s[j] = q[j] = 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (row + u * d.rows < d.hw)
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int cl = min(channel_of<T, WHOLE>(d, v, j), d.cs - 1);
                    float e;
                    const float dz = grad_z((float)g[u].v[j], (float)w[u].v[j], k[j], st + cl / d.gc * 2, weight + cl, act, e);
                    s[j] += dz;
                    q[j] = fmaf(dz, e, q[j]);
                }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float *o = redf[row * units + channel_of<T, WHOLE>(d, v, j)];
            o[0] = s[j];
            o[1] = q[j];
        }
    }
    fold_rows(redf, d.rows, units);
    // a channel's sums go out, and times its weight back for its group's a1 and a2
    float (*weighted)[2] = redf + units;
    float2 *means = reinterpret_cast<float2 *>(weighted + units);
    for (int cl = threadIdx.x; cl < d.cs; cl += blockDim.x) {
        const float s = redf[cl][0], q = redf[cl][1] * (float)st[cl / d.gc * 2 + 1], wt = weight[cl];
        weighted[cl][0] = wt * s;
        weighted[cl][1] = wt * q;
        if (images > 1) {
            sums[((long long)b * d.c + c0 + cl) * 2] = s;
            sums[((long long)b * d.c + c0 + cl) * 2 + 1] = q;
        } else {
            if (dweight)
                store_affine(dweight, affine_dtype, c0 + cl, q);
            if (dbias)
                store_affine(dbias, affine_dtype, c0 + cl, s);
        }
    }
    if (dx == nullptr)
        return;
    __syncthreads();
    const float (*wsums)[2] = weighted;
    for_group_sums(wsums, sg, d.gc, [&](int i, float s, float q) {
        const double count = (double)d.gc * (double)d.hw, rstd = st[i * 2 + 1];
        means[i] = float2{(float)(rstd * (double)s / count), (float)(rstd * rstd * (double)q / count)};
    });
    __syncthreads();
    if (!live)
        return;
    T *op = dx + b * d.hw * d.c + c0;
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (row + u * d.rows < d.hw) {
            Word<T> r;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int cl = min(channel_of<T, WHOLE>(d, v, j), d.cs - 1);
                float e;
                const float dz = grad_z((float)g[u].v[j], (float)w[u].v[j], k[j], st + cl / d.gc * 2, weight + cl, act, e);
                r.v[j] = (T)grad_x(dz, e, k[j], means[cl / d.gc]);
            }
            store_word<T, WHOLE>(op + (long long)(row + u * d.rows) * d.c, r, d, v);
        }
}

// ------------------------------------------------------------------------------------------- host
constexpr int MAX_VECTORS = MAX_THREADS;        // vectors of a pixel: a thread each

int vector_of(int dtype) { return dtype == DANCE_F32 ? 4 : 8; }

int vectors_of(int c, int dtype) { return ceil_div(c, vector_of(dtype)); }

int threads_of(int cv) { return cv <= 256 ? 256 : MAX_THREADS; }

// The two-pass form.  A workgroup takes 16 pixels a thread, so that its reduction is paid by enough reading, where that
// still gives every compute unit a workgroup, else 8 or 4; no more than 2048 workgroups (eight a compute unit).  us of
// statistics and apply pass with 16 / 8 pixels: (1, 256, 200, 304) bf16 10.5 + 12.5 / 12.2 + 14.9; with 8 / 4:
// (3, 96, 67, 101) fp16 7.6 + 6.9 / 7.5 + 5.5.
GnDims dims_of(int b, int c, long long hw, int groups, int dtype)
{
    GnDims d;
    d.hw = hw;
    d.c = d.cs = c;
    d.cv = vectors_of(c, dtype);
    d.rows = threads_of(d.cv) / d.cv;
    d.groups = groups;
    d.gc = c / groups;
    int pixels = 16;
    auto most_of = [&] { return (hw + (long long)pixels * d.rows - 1) / ((long long)pixels * d.rows); };
    while (pixels > 4 && b * most_of() < 256)
        pixels /= 2;
    const long long most = most_of();
    long long nch = (2048 + b - 1) / b;
    nch = nch < 1 ? 1 : (nch > most ? most : nch);
    d.chunk = (hw + nch - 1) / nch;
    d.nch = (int)((hw + d.chunk - 1) / d.chunk);
    return d;
}

// LDS of the one-launch form.  Forward: the groups' pivots; the sums of the rows, or row 0 and, behind it, the groups'
// statistics and the channels' constants.  Backward: the sums of the rows; or row 0, the weighted sums and the groups' means.
constexpr size_t LDS_MOST = 160 * 1024;

size_t one_lds(const GnDims &d, int dtype, bool backward)
{
    const int n = vector_of(dtype);
    const size_t groups = d.cs / d.gc, channels = (size_t)d.cv * n;
    if (backward) {
        const size_t sums = d.rows * channels, after = 2 * channels + groups;
        return (sums > after ? sums : after) * 2 * sizeof(float);
    }
    const size_t units = d.c % n == 0 && d.gc % n == 0 ? d.cv : channels;         // vector_units
    const size_t sums = d.rows * units * 2 * sizeof(double);
    const size_t after = (units + groups) * 2 * sizeof(double) + d.cs * sizeof(Channel);
    return (groups + 3) / 4 * 16 + (sums > after ? sums : after);
}

// The one-launch form: MAX_THREADS a workgroup, at most `most` vectors a thread.  A slab is the fewest whole groups that
// make whole vectors and a wanted width: the widest of 1 KB ... 64 bytes a pixel that gives every compute unit a
// workgroup, else 64 bytes.  Narrower ones, 32 and 16 bytes, read parts of cache lines and are for maps that are in the
// caches anyway; larger maps that fit no other slab take the two-pass form.  us forward and backward, this rule / at most
// 64 bytes always: 2048 of (256, 3, 3) 47 / 299, 64 of (256, 25, 38) 118 / 124; this rule / narrow slabs for any size:
// 64 of (256, 50, 50) fp32 232 / 333, bf16 172 / 373, (256, 50, 50) 24.0 / 27.3; narrow slabs / this rule without them:
// (256, 25, 38) fp32 16.2 / 20.3, bf16 16.2 / 30.1.  false: the map is too large for any, or only a slab of thousands of
// groups has whole vectors (a group a channel, a prime number of them) and their constants do not fit LDS.
constexpr int ONE_MOST = 16, GRAD_ONE_MOST = 8;
constexpr double NARROW_MOST = 1.5e6;                     // bytes

bool one_launch(GnDims &d, int b, int dtype, bool backward)
{
    const int n = vector_of(dtype);
    const bool whole = d.c % n == 0;
    int most = backward ? GRAD_ONE_MOST : ONE_MOST;
    if (!whole)
        most = 4;                                         // a vector of scalar loads is n registers
    const bool narrow = (double)b * d.c * d.hw * (16 / n) <= NARROW_MOST;
    bool fits = false;
    for (int least = 64 * n; least >= (narrow ? n : 4 * n); least /= 2) {
        int k = 1;                                        // groups of a slab
        while (k < d.groups && (d.groups % k != 0 || k * d.gc < least || (whole && k * d.gc % n != 0)))
            ++k;
        const int cs = k * d.gc, cv = ceil_div(cs, n);
        const bool enough = (long long)b * (d.c / cs) >= 256;
        if (cv > MAX_THREADS || (least > 4 * n && !enough))
            continue;
        const int rows = MAX_THREADS / cv;
        if (d.hw > (long long)rows * most)
            continue;
        GnDims slab = d;
        slab.cs = cs;
        slab.cv = cv;
        slab.rows = rows < d.hw ? rows : (int)d.hw;
        if (one_lds(slab, dtype, backward) > LDS_MOST)
            continue;
        fits = true;
        d = slab;
        if (enough)
            break;
    }
    return fits;
}

int words_of(const GnDims &d) { return (int)((d.hw + d.rows - 1) / d.rows); }

template <typename F> int with_type(int dtype, bool whole, F &&f)
{
    if (dtype == DANCE_F32)
        return whole ? f((float)0, std::true_type{}) : f((float)0, std::false_type{});
    if (dtype == DANCE_F16)
        return whole ? f((_Float16)0, std::true_type{}) : f((_Float16)0, std::false_type{});
    return whole ? f((__bf16)0.0f, std::true_type{}) : f((__bf16)0.0f, std::false_type{});
}

// Does a map (in- and output) go past the cache?
bool streams(int b, int c, long long hw, int dtype) { return (double)b * c * hw * (dtype == DANCE_F32 ? 4 : 2) >= 64e6; }

// Up to so many images k_gn_grad_apply adds the parameters' gradients on the way, in one thread a channel; of more
// k_gn_grad_affine does.
constexpr int FEW_IMAGES = 16;

template <typename F> int with_flag(bool on, F &&f) { return on ? f(std::true_type{}) : f(std::false_type{}); }

template <typename F> int with_act(int act, F &&f)
{
    if (act == DANCE_ACT_RELU)
        return f(std::integral_constant<int, DANCE_ACT_RELU>{});
    if (act == DANCE_ACT_SILU)
        return f(std::integral_constant<int, DANCE_ACT_SILU>{});
    return f(std::integral_constant<int, DANCE_ACT_NONE>{});
}

size_t whole_16(size_t bytes) { return (bytes + 15) & ~(size_t)15; }

bool known_dtype(int t) { return t == DANCE_F32 || t == DANCE_F16 || t == DANCE_BF16; }

}  // namespace

extern "C" int64_t dance_group_norm_workspace_bytes(int b, int c, int64_t hw, int groups, int dtype, int backward)
{
    if (b <= 0 || c <= 0 || hw <= 0 || groups <= 0 || c % groups || !known_dtype(dtype) || vectors_of(c, dtype) > MAX_VECTORS)
        return 0;
    GnDims d = dims_of(b, c, hw, groups, dtype), one = d;
    if (!backward)
        return one_launch(one, b, dtype, false) ? 0 : (int64_t)b * d.nch * groups * 2 * sizeof(double);
    if (one_launch(one, b, dtype, true))
        return b == 1 ? 0 : (int64_t)b * c * 2 * sizeof(double);
    return (int64_t)(whole_16((size_t)b * d.nch * c * 2 * sizeof(float)) + (size_t)b * c * 2 * sizeof(double) +
                     (size_t)b * groups * sizeof(float2));
}

extern "C" int64_t dance_group_norm_saved_bytes(int b, int c, int groups)
{
    if (b <= 0 || c <= 0 || groups <= 0 || c % groups)
        return 0;
    return (int64_t)((size_t)b * groups * 2 * sizeof(double) + (size_t)b * c * sizeof(Channel) + (size_t)c * sizeof(float));
}

extern "C" int dance_group_norm_act(const void *x, int64_t image_stride, int64_t pixel_stride, int dtype,
                                    const void *weight, const void *bias, int affine_dtype, float eps, int act,
                                    int groups, void *y, void *saved, void *ws, int64_t ws_bytes, int b, int c,
                                    int64_t hw, void *stream)
{
    DANCE_REQUIRE(b >= 0 && c >= 1 && hw >= 0 && groups >= 1 && c % groups == 0);
    DANCE_REQUIRE(known_dtype(dtype) && known_dtype(affine_dtype) && eps >= 0.0f);
    DANCE_REQUIRE(act == DANCE_ACT_NONE || act == DANCE_ACT_RELU || act == DANCE_ACT_SILU);
    DANCE_REQUIRE(vectors_of(c, dtype) <= MAX_VECTORS);
    DANCE_REQUIRE(image_stride >= 0 && pixel_stride >= 0);
    if (b == 0 || hw == 0)
        return 0;
    DANCE_REQUIRE(x && y && saved && ((uintptr_t)saved & 15) == 0 && b <= 65535 && groups <= 65535);
    DANCE_REQUIRE(ws_bytes >= dance_group_norm_workspace_bytes(b, c, hw, groups, dtype, 0) && (ws || ws_bytes <= 0));
    DANCE_REQUIRE(((uintptr_t)ws & 15) == 0);
    GnDims d = dims_of(b, c, hw, groups, dtype);
    DANCE_REQUIRE((long long)b * d.nch < (1ll << 31));
    const int threads = threads_of(d.cv);
    const dim3 grid((unsigned)(b * d.nch));
    hipStream_t st = (hipStream_t)stream;
    const Saved out = saved_at(saved, b, c, groups);
    const char *fn = "dance_group_norm_act";
    return with_type(dtype, c % vector_of(dtype) == 0, [&](auto t, auto whole) {
        using T = decltype(t);
        constexpr bool W = decltype(whole)::value;
        if (one_launch(d, b, dtype, false)) {
            auto one = [&](auto u) {
                constexpr int U = decltype(u)::value;
                const size_t lds = one_lds(d, dtype, false);
                if (int rc = dance::allow_lds((const void *)k_gn_one<T, W, U>, lds, fn))
                    return rc;
                hipLaunchKernelGGL((k_gn_one<T, W, U>), dim3((unsigned)(b * (c / d.cs))), dim3(MAX_THREADS), lds, st,
                                   (const T *)x, (long long)image_stride, (long long)pixel_stride, weight, bias,
                                   affine_dtype, (double)eps, act, (T *)y, out, d);
                return launch_check(fn);
            };
            if constexpr (W)
                if (words_of(d) > 4)
                    return one(std::integral_constant<int, ONE_MOST>{});
            return one(std::integral_constant<int, 4>{});
        }
        double *partial = (double *)ws;
        const bool vu = W && d.gc % Vec<T>::N == 0;
        const size_t lds = (size_t)d.rows * d.cv * (vu ? 1 : Vec<T>::N) * 2 * sizeof(double);
        if (int rc = dance::allow_lds((const void *)k_gn_stats<T, W>, lds, fn))
            return rc;
        hipLaunchKernelGGL((k_gn_stats<T, W>), grid, dim3(threads), lds, st, (const T *)x, (long long)image_stride,
                           (long long)pixel_stride, partial, d);
        if (int rc = launch_check(fn))
            return rc;
        hipLaunchKernelGGL(k_gn_finish, dim3(groups, b), dim3(256), 0, st, (const double *)partial, x, dtype,
                           (long long)image_stride, out, weight, bias, affine_dtype, (double)d.gc * (double)d.hw, (double)eps, d);
        if (int rc = launch_check(fn))
            return rc;
        return with_act(act, [&](auto a) {
            return with_flag(W && streams(b, c, hw, dtype), [&](auto stream) {
                hipLaunchKernelGGL((k_gn_apply<T, W, decltype(a)::value, W && decltype(stream)::value>), grid, dim3(threads), 0,
                                   st, (const T *)x, (long long)image_stride, (long long)pixel_stride,
                                   (const Channel *)out.channels, (T *)y, d);
                return launch_check(fn);
            });
        });
    });
}

extern "C" int dance_group_norm_act_backward(const void *dy, int64_t dy_image_stride, int64_t dy_pixel_stride,
                                             const void *x, int64_t image_stride, int64_t pixel_stride, int dtype,
                                             int affine_dtype, int act, int groups, const void *saved, void *dx,
                                             void *dweight, void *dbias, void *ws, int64_t ws_bytes, int b, int c,
                                             int64_t hw, void *stream)
{
    DANCE_REQUIRE(b >= 1 && c >= 1 && hw >= 1 && groups >= 1 && c % groups == 0);
    DANCE_REQUIRE(known_dtype(dtype) && known_dtype(affine_dtype));
    DANCE_REQUIRE(act == DANCE_ACT_NONE || act == DANCE_ACT_RELU || act == DANCE_ACT_SILU);
    DANCE_REQUIRE(vectors_of(c, dtype) <= MAX_VECTORS);
    DANCE_REQUIRE(dy_image_stride >= 0 && dy_pixel_stride >= 0 && image_stride >= 0 && pixel_stride >= 0);
    DANCE_REQUIRE(dy && x && saved && ((uintptr_t)saved & 15) == 0 && b <= 65535 && groups <= 65535);
    DANCE_REQUIRE(ws_bytes >= dance_group_norm_workspace_bytes(b, c, hw, groups, dtype, 1) && (ws || ws_bytes <= 0));
    DANCE_REQUIRE(((uintptr_t)ws & 15) == 0);
    if (!dx && !dweight && !dbias)
        return 0;
    GnDims d = dims_of(b, c, hw, groups, dtype);
    DANCE_REQUIRE((long long)b * d.nch < (1ll << 31));
    const int threads = threads_of(d.cv);
    const dim3 grid((unsigned)(b * d.nch));
    hipStream_t st = (hipStream_t)stream;
    const Saved sv = saved_at(const_cast<void *>(saved), b, c, groups);        // read only
    const char *fn = "dance_group_norm_act_backward";
    auto affine = [&](const double *sums) {
        hipLaunchKernelGGL(k_gn_grad_affine, dim3(ceil_div(c, AFFINE_CHANNELS)), dim3(MAX_THREADS), 0, st, sums, dweight, dbias,
                           affine_dtype, b, c);
        return launch_check(fn);
    };
    return with_type(dtype, c % vector_of(dtype) == 0, [&](auto t, auto whole) {
        using T = decltype(t);
        constexpr bool W = decltype(whole)::value;
        if (one_launch(d, b, dtype, true)) {
            auto one = [&](auto u) {
                constexpr int U = decltype(u)::value;
                const size_t lds = one_lds(d, dtype, true);
                if (int rc = dance::allow_lds((const void *)k_gn_grad_one<T, W, U>, lds, fn))
                    return rc;
                hipLaunchKernelGGL((k_gn_grad_one<T, W, U>), dim3((unsigned)(b * (c / d.cs))), dim3(MAX_THREADS), lds, st,
                                   (const T *)dy, (long long)dy_image_stride, (long long)dy_pixel_stride, (const T *)x,
                                   (long long)image_stride, (long long)pixel_stride, sv, act, (T *)dx, dweight, dbias,
                                   affine_dtype, (double *)ws, b, d);
                return launch_check(fn);
            };
            // (four vectors of scalar loads are the most of the other kind)
            constexpr int MOST = W ? GRAD_ONE_MOST : 4;
            if (int rc = words_of(d) <= 2 ? one(std::integral_constant<int, 2>{}) : one(std::integral_constant<int, MOST>{}))
                return rc;
            if (b == 1 || (!dweight && !dbias))
                return 0;
            return affine((const double *)ws);
        }
        float *partial = (float *)ws;
        double *sums = (double *)((char *)ws + whole_16((size_t)b * d.nch * c * 2 * sizeof(float)));
        float2 *means = (float2 *)(sums + (size_t)b * c * 2);
        return with_act(act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            const size_t lds = (size_t)d.rows * d.cv * Vec<T>::N * 2 * sizeof(float);
            if (int rc = dance::allow_lds((const void *)k_gn_grad_sums<T, W, ACT>, lds, fn))
                return rc;
            hipLaunchKernelGGL((k_gn_grad_sums<T, W, ACT>), grid, dim3(threads), lds, st, (const T *)dy,
                               (long long)dy_image_stride, (long long)dy_pixel_stride, (const T *)x,
                               (long long)image_stride, (long long)pixel_stride, sv, partial, d);
            if (int rc = launch_check(fn))
                return rc;
            hipLaunchKernelGGL(k_gn_grad_finish, dim3(groups, b), dim3(MAX_THREADS), 0, st, (const float *)partial, sv, sums, means, d);
            if (int rc = launch_check(fn))
                return rc;
            const bool apart = b > FEW_IMAGES;
            if (apart && (dweight || dbias))
                if (int rc = affine(sums))
                    return rc;
            if (apart && !dx)
                return 0;
            return with_flag(W && streams(b, c, hw, dtype), [&](auto stream) {
                hipLaunchKernelGGL((k_gn_grad_apply<T, W, ACT, W && decltype(stream)::value>), dx ? grid : dim3(1),
                                   dim3(threads), 0, st, (const T *)dy, (long long)dy_image_stride,
                                   (long long)dy_pixel_stride, (const T *)x, (long long)image_stride,
                                   (long long)pixel_stride, sv, (const float2 *)means, (const double *)sums, (T *)dx,
                                   apart ? nullptr : dweight, apart ? nullptr : dbias, affine_dtype, b, d);
                return launch_check(fn);
            });
        });
    });
}
