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

__device__ __forceinline__ float load_affine(const void *p, int dtype, int i, float otherwise)
{
    if (p == nullptr)
        return otherwise;
    if (dtype == DANCE_F32)
        return ((const float *)p)[i];
    return dtype == DANCE_F16 ? (float)((const _Float16 *)p)[i] : (float)((const __bf16 *)p)[i];
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

struct GnDims {
    long long hw, chunk;        // pixels of an image; pixels of a workgroup
    int c, cv, rows;            // channels; vectors of a pixel; pixels a workgroup covers at once
    int groups, gc, nch;        // groups; channels of one; workgroups of an image
};

// the channel that element j of vector v holds.  WHOLE (c a multiple of the vector): 16 consecutive bytes;
// otherwise element j of the whole row of vectors, so that a wave's scalar accesses are consecutive
template <typename T, bool WHOLE> __device__ __forceinline__ int channel_of(const GnDims &d, int v, int j)
{
    return WHOLE ? v * Vec<T>::N + j : v + j * d.cv;
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void load_vec(float (&r)[Vec<T>::N], const T *pixel, const GnDims &d, int v)
{
    if (WHOLE) {
        const Word<T> w = *reinterpret_cast<const Word<T> *>(pixel + v * Vec<T>::N);
#pragma unroll
        for (int j = 0; j < Vec<T>::N; ++j)
            r[j] = (float)w.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < Vec<T>::N; ++j) {
            const int ch = v + j * d.cv;
            r[j] = ch < d.c ? (float)pixel[ch] : 0.0f;
        }
    }
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void store_vec(T *pixel, const float (&r)[Vec<T>::N], const GnDims &d, int v)
{
    if (WHOLE) {
        Word<T> w;
#pragma unroll
        for (int j = 0; j < Vec<T>::N; ++j)
            w.v[j] = (T)r[j];
        *reinterpret_cast<Word<T> *>(pixel + v * Vec<T>::N) = w;
    } else {
#pragma unroll
        for (int j = 0; j < Vec<T>::N; ++j) {
            const int ch = v + j * d.cv;
            if (ch < d.c)
                pixel[ch] = (T)r[j];
        }
    }
}

// ------------------------------------------------------------------------------------- statistics
// Sum and sum of squares of a chunk of pixels, per group, both in fp64: the difference that makes the
// variance then loses nothing at any mean / spread ratio fp32 inputs can hold.
// partial (b, nch, groups, 2).  grid: b * nch workgroups.
template <typename T, bool WHOLE>
__global__ __launch_bounds__(1024) void k_gn_stats(const T *__restrict__ x, long long image_stride,
                                                   long long pixel_stride, double *__restrict__ partial, GnDims d)
{
    constexpr int N = Vec<T>::N;
    extern __shared__ double red[];                       // [rows][cv * N][2]
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
    double s[N], q[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
        s[j] = q[j] = 0.0;
    if (row < d.rows) {
        const T *xp = x + b * image_stride;
#pragma unroll 4
        for (long long p = p0 + row; p < p1; p += d.rows) {
            float r[N];
            load_vec<T, WHOLE>(r, xp + p * pixel_stride, d, v);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                s[j] += (double)r[j];
                q[j] = fma((double)r[j], (double)r[j], q[j]);
            }
        }
    }
    const int width = d.cv * N;
    if (row < d.rows)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            double *e = red + ((long long)row * width + channel_of<T, WHOLE>(d, v, j)) * 2;
            e[0] = s[j];
            e[1] = q[j];
        }
    __syncthreads();
    for (int n = d.rows; n > 1;) {                        // fold the rows onto row 0
        const int h = (n + 1) / 2;
        for (int i = threadIdx.x; i < (n - h) * width * 2; i += blockDim.x)
            red[i] += red[i + h * width * 2];
        __syncthreads();
        n = h;
    }
    for (int g = threadIdx.x; g < d.groups; g += blockDim.x) {
        double sg = 0.0, qg = 0.0;
        for (int k = 0; k < d.gc; ++k) {
            sg += red[(g * d.gc + k) * 2];
            qg += red[(g * d.gc + k) * 2 + 1];
        }
        double *o = partial + ((long long)blockIdx.x * d.groups + g) * 2;
        o[0] = sg;
        o[1] = qg;
    }
}

// partial (b, nch, groups, 2) -> stats (b, groups, 2) = mean, rstd.  grid: (groups, b), one wave each.
__global__ __launch_bounds__(64) void k_gn_finish(const double *__restrict__ partial, double *__restrict__ stats,
                                                  int groups, int nch, double count, double eps)
{
    const int g = blockIdx.x, b = blockIdx.y;
    double s = 0.0, q = 0.0;
    for (int i = threadIdx.x; i < nch; i += 64) {
        const double *p = partial + (((long long)b * nch + i) * groups + g) * 2;
        s += p[0];
        q += p[1];
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        s += __shfl_xor(s, m, 64);
        q += __shfl_xor(q, m, 64);
    }
    if (threadIdx.x == 0) {
        const double mean = s / count;
        double var = q / count - mean * mean;
        var = var < 0.0 ? 0.0 : var;                      // (a NaN stays one: infinities in the map give NaN, as in torch)
        stats[((long long)b * groups + g) * 2] = mean;
        stats[((long long)b * groups + g) * 2 + 1] = 1.0 / sqrt(var + eps);
    }
}

// ------------------------------------------------------------------------------------------ apply
// A channel's constants.  The mean as a sum of two floats: x - mu keeps its low bits when the mean is large
// against the spread.
struct Channel {
    float mhi, mlo, rstd, w, beta;
};

__device__ __forceinline__ Channel channel_constants(const double *stats, const void *weight, const void *bias,
                                                     int affine_dtype, const GnDims &d, int b, int ch)
{
    Channel k = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (ch < d.c) {
        const double *st = stats + ((long long)b * d.groups + ch / d.gc) * 2;
        k.mhi = (float)st[0];
        k.mlo = (float)(st[0] - (double)k.mhi);
        k.rstd = (float)st[1];
        k.w = load_affine(weight, affine_dtype, ch, 1.0f);
        k.beta = load_affine(bias, affine_dtype, ch, 0.0f);
    }
    return k;
}

__device__ __forceinline__ float normalised(float x, const Channel &k) { return ((x - k.mhi) - k.mlo) * k.rstd; }

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }

template <int ACT> __device__ __forceinline__ float activate(float z)
{
    if (ACT == DANCE_ACT_RELU)
        return z > 0.0f ? z : (z != z ? z : 0.0f);
    if (ACT == DANCE_ACT_SILU)
        return z * sigmoid(z);
    return z;
}

// grid: b * nch workgroups
template <typename T, bool WHOLE, int ACT>
__global__ __launch_bounds__(1024) void k_gn_apply(const T *__restrict__ x, long long image_stride,
                                                   long long pixel_stride, const double *__restrict__ stats,
                                                   const void *weight, const void *bias, int affine_dtype,
                                                   T *__restrict__ y, GnDims d)
{
    constexpr int N = Vec<T>::N;
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    if (row >= d.rows)
        return;
    Channel k[N];
#pragma unroll
    for (int j = 0; j < N; ++j)
        k[j] = channel_constants(stats, weight, bias, affine_dtype, d, b, channel_of<T, WHOLE>(d, v, j));
    const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
    const T *xp = x + b * image_stride;
    T *yp = y + b * d.hw * d.c;
#pragma unroll 4
    for (long long p = p0 + row; p < p1; p += d.rows) {
        float r[N];
        load_vec<T, WHOLE>(r, xp + p * pixel_stride, d, v);
#pragma unroll
        for (int j = 0; j < N; ++j)
            r[j] = activate<ACT>(fmaf(normalised(r[j], k[j]), k[j].w, k[j].beta));
        store_vec<T, WHOLE>(yp + p * d.c, r, d, v);
    }
}

// --------------------------------------------------------------------------------------- backward
// dz = dy act'(z) and xh of one element.  ReLU: which side of zero z lies on decides whole gradients, so a
// z within fp32 rounding of zero is evaluated again in fp64 (the rounding of z is a few 2^-24 of its two
// terms; 2^-20 of them covers it, one element in a million takes the branch).
template <int ACT>
__device__ __forceinline__ float grad_z(float dy, float x, const Channel &k, const double *st, float &xh)
{
    xh = normalised(x, k);
    if (ACT == DANCE_ACT_NONE)
        return dy;
    const float t = xh * k.w, z = t + k.beta;
    if (ACT == DANCE_ACT_RELU) {
        bool on = z > 0.0f;
        if (fabsf(z) <= 9.5367431640625e-7f * (fabsf(t) + fabsf(k.beta)))
            on = ((double)x - st[0]) * st[1] * (double)k.w + (double)k.beta > 0.0;
        return on ? dy : (z != z ? z : 0.0f);
    }
    const float s = sigmoid(z);
    return dy * (s * (1.0f + z * (1.0f - s)));
}

// Per-channel sums of dz and dz xh over a chunk of pixels: partial (b, nch, c, 2) fp32.  grid: b * nch.
template <typename T, bool WHOLE, int ACT>
__global__ __launch_bounds__(1024) void k_gn_grad_sums(const T *__restrict__ dy, long long dy_image, long long dy_pixel,
                                                       const T *__restrict__ x, long long image_stride,
                                                       long long pixel_stride, const double *__restrict__ stats,
                                                       const void *weight, const void *bias, int affine_dtype,
                                                       float *__restrict__ partial, GnDims d)
{
    constexpr int N = Vec<T>::N;
    extern __shared__ float redf[];                       // [rows][cv * N][2]
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    const int width = d.cv * N;
    if (row < d.rows) {
        Channel k[N];
        const double *st[N];
        float s[N], q[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = channel_of<T, WHOLE>(d, v, j);
            k[j] = channel_constants(stats, weight, bias, affine_dtype, d, b, c);
            st[j] = stats + ((long long)b * d.groups + min(c, d.c - 1) / d.gc) * 2;
            s[j] = q[j] = 0.0f;
        }
        const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
        const T *xp = x + b * image_stride, *dp = dy + b * dy_image;
#pragma unroll 2
        for (long long p = p0 + row; p < p1; p += d.rows) {
            float r[N], g[N];
            load_vec<T, WHOLE>(r, xp + p * pixel_stride, d, v);
            load_vec<T, WHOLE>(g, dp + p * dy_pixel, d, v);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float xh;
                const float dz = grad_z<ACT>(g[j], r[j], k[j], st[j], xh);
                s[j] += dz;
                q[j] = fmaf(dz, xh, q[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float *e = redf + ((long long)row * width + channel_of<T, WHOLE>(d, v, j)) * 2;
            e[0] = s[j];
            e[1] = q[j];
        }
    }
    __syncthreads();
    for (int n = d.rows; n > 1;) {
        const int h = (n + 1) / 2;
        for (int i = threadIdx.x; i < (n - h) * width * 2; i += blockDim.x)
            redf[i] += redf[i + h * width * 2];
        __syncthreads();
        n = h;
    }
    for (int i = threadIdx.x; i < d.c * 2; i += blockDim.x)
        partial[(long long)blockIdx.x * d.c * 2 + i] = redf[i];
}

// partial (b, nch, c, 2) -> sums (b, c, 2) and means (b, groups, 2) = m1, m2, in fp64.  grid: (groups, b).
__global__ __launch_bounds__(256) void k_gn_grad_finish(const float *__restrict__ partial, const void *weight,
                                                        int affine_dtype, double *__restrict__ sums,
                                                        double *__restrict__ means, GnDims d)
{
    __shared__ double red[256 * 2];
    const int g = blockIdx.x, b = blockIdx.y;
    double m1 = 0.0, m2 = 0.0;
    // a channel is folded by `lanes` threads (a power of two), the block takes 256 / lanes channels at once
    int lanes = 64;
    while (lanes > 1 && lanes * d.gc > 256)
        lanes >>= 1;
    const int sub = threadIdx.x / lanes, lane = threadIdx.x - sub * lanes;
    for (int c0 = 0; c0 < d.gc; c0 += 256 / lanes) {
        const int cl = c0 + sub, c = g * d.gc + cl;
        double s = 0.0, q = 0.0;
        if (cl < d.gc)
            for (int i = lane; i < d.nch; i += lanes) {
                const float *p = partial + (((long long)b * d.nch + i) * d.c + c) * 2;
                s += (double)p[0];
                q += (double)p[1];
            }
        for (int m = lanes >> 1; m >= 1; m >>= 1) {
            s += __shfl_xor(s, m, 64);
            q += __shfl_xor(q, m, 64);
        }
        if (cl < d.gc && lane == 0) {
            sums[((long long)b * d.c + c) * 2] = s;
            sums[((long long)b * d.c + c) * 2 + 1] = q;
            const double w = (double)load_affine(weight, affine_dtype, c, 1.0f);
            m1 += w * s;
            m2 += w * q;
        }
    }
    red[threadIdx.x * 2] = m1;
    red[threadIdx.x * 2 + 1] = m2;
    __syncthreads();
    for (int h = 128; h >= 1; h >>= 1) {
        if ((int)threadIdx.x < h) {
            red[threadIdx.x * 2] += red[(threadIdx.x + h) * 2];
            red[threadIdx.x * 2 + 1] += red[(threadIdx.x + h) * 2 + 1];
        }
        __syncthreads();
    }
    if (threadIdx.x < 2)
        means[((long long)b * d.groups + g) * 2 + threadIdx.x] = red[threadIdx.x] / ((double)d.gc * (double)d.hw);
}

// dw, dbeta: the images' sums added in order.  grid: ceil(c / 64)
__global__ __launch_bounds__(64) void k_gn_grad_affine(const double *__restrict__ sums, void *dweight, void *dbias,
                                                       int affine_dtype, int b, int c)
{
    const int ch = blockIdx.x * 64 + threadIdx.x;
    if (ch >= c)
        return;
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

// grid: b * nch workgroups
template <typename T, bool WHOLE, int ACT>
__global__ __launch_bounds__(1024) void k_gn_grad_apply(const T *__restrict__ dy, long long dy_image, long long dy_pixel,
                                                        const T *__restrict__ x, long long image_stride,
                                                        long long pixel_stride, const double *__restrict__ stats,
                                                        const double *__restrict__ means, const void *weight,
                                                        const void *bias, int affine_dtype, T *__restrict__ dx, GnDims d)
{
    constexpr int N = Vec<T>::N;
    const int b = blockIdx.x / d.nch, ch = blockIdx.x - b * d.nch;
    const int row = threadIdx.x / d.cv, v = threadIdx.x - row * d.cv;
    if (row >= d.rows)
        return;
    Channel k[N];
    const double *st[N];
    float m1[N], m2[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int c = channel_of<T, WHOLE>(d, v, j);
        const long long g = (long long)b * d.groups + min(c, d.c - 1) / d.gc;
        k[j] = channel_constants(stats, weight, bias, affine_dtype, d, b, c);
        st[j] = stats + g * 2;
        m1[j] = (float)means[g * 2];
        m2[j] = (float)means[g * 2 + 1];
    }
    const long long p0 = ch * d.chunk, p1 = min(p0 + d.chunk, d.hw);
    const T *xp = x + b * image_stride, *dp = dy + b * dy_image;
    T *op = dx + b * d.hw * d.c;
#pragma unroll 2
    for (long long p = p0 + row; p < p1; p += d.rows) {
        float r[N], g[N];
        load_vec<T, WHOLE>(r, xp + p * pixel_stride, d, v);
        load_vec<T, WHOLE>(g, dp + p * dy_pixel, d, v);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float xh;
            const float dz = grad_z<ACT>(g[j], r[j], k[j], st[j], xh);
            r[j] = k[j].rstd * (dz * k[j].w - m1[j] - xh * m2[j]);
        }
        store_vec<T, WHOLE>(op + p * d.c, r, d, v);
    }
}

// ------------------------------------------------------------------------------------------- host
constexpr int MAX_VECTORS = 1024;       // vectors of a pixel a workgroup can own

int vectors_of(int c, int dtype) { return ceil_div(c, dtype == DANCE_F32 ? 4 : 8); }

int threads_of(int cv) { return cv <= 256 ? 256 : cv <= 512 ? 512 : 1024; }

// Workgroups of an image: about 2048 over the whole batch (eight a compute unit), each with 8 pixels a
// thread at least, so that a workgroup's reduction is paid by enough reading.
GnDims dims_of(int b, int c, long long hw, int groups, int dtype)
{
    GnDims d;
    d.hw = hw;
    d.c = c;
    d.cv = vectors_of(c, dtype);
    d.rows = threads_of(d.cv) / d.cv;
    d.groups = groups;
    d.gc = c / groups;
    const long long most = (hw + 8 * d.rows - 1) / (8 * d.rows);
    long long nch = (2048 + b - 1) / b;
    nch = nch < 1 ? 1 : (nch > most ? most : nch);
    d.chunk = (hw + nch - 1) / nch;
    d.nch = (int)((hw + d.chunk - 1) / d.chunk);
    return d;
}

template <typename F> int with_type(int dtype, bool whole, F &&f)
{
    if (dtype == DANCE_F32)
        return whole ? f((float)0, std::true_type{}) : f((float)0, std::false_type{});
    if (dtype == DANCE_F16)
        return whole ? f((_Float16)0, std::true_type{}) : f((_Float16)0, std::false_type{});
    return whole ? f((__bf16)0.0f, std::true_type{}) : f((__bf16)0.0f, std::false_type{});
}

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
    const GnDims d = dims_of(b, c, hw, groups, dtype);
    if (!backward)
        return (int64_t)b * d.nch * groups * 2 * sizeof(double);
    return (int64_t)(whole_16((size_t)b * d.nch * c * 2 * sizeof(float)) + (size_t)b * c * 2 * sizeof(double) +
                     (size_t)b * groups * 2 * sizeof(double));
}

extern "C" int dance_group_norm_act(const void *x, int64_t image_stride, int64_t pixel_stride, int dtype,
                                    const void *weight, const void *bias, int affine_dtype, float eps, int act,
                                    int groups, void *y, double *stats, void *ws, int64_t ws_bytes, int b, int c,
                                    int64_t hw, void *stream)
{
    DANCE_REQUIRE(b >= 0 && c >= 1 && hw >= 0 && groups >= 1 && c % groups == 0);
    DANCE_REQUIRE(known_dtype(dtype) && known_dtype(affine_dtype) && eps >= 0.0f);
    DANCE_REQUIRE(act == DANCE_ACT_NONE || act == DANCE_ACT_RELU || act == DANCE_ACT_SILU);
    DANCE_REQUIRE(vectors_of(c, dtype) <= MAX_VECTORS);
    DANCE_REQUIRE(image_stride >= 0 && pixel_stride >= 0);
    if (b == 0 || hw == 0)
        return 0;
    DANCE_REQUIRE(x && y && stats && ws && b <= 65535 && groups <= 65535);
    DANCE_REQUIRE(ws_bytes >= dance_group_norm_workspace_bytes(b, c, hw, groups, dtype, 0));
    const GnDims d = dims_of(b, c, hw, groups, dtype);
    DANCE_REQUIRE((long long)b * d.nch < (1ll << 31));
    const int threads = threads_of(d.cv);
    const dim3 grid((unsigned)(b * d.nch));
    hipStream_t st = (hipStream_t)stream;
    double *partial = (double *)ws;
    return with_type(dtype, c % (dtype == DANCE_F32 ? 4 : 8) == 0, [&](auto t, auto whole) {
        using T = decltype(t);
        constexpr bool W = decltype(whole)::value;
        const size_t lds = (size_t)d.rows * d.cv * Vec<T>::N * 2 * sizeof(double);
        if (int rc = dance::allow_lds((const void *)k_gn_stats<T, W>, lds, "dance_group_norm_act"))
            return rc;
        hipLaunchKernelGGL((k_gn_stats<T, W>), grid, dim3(threads), lds, st, (const T *)x, (long long)image_stride,
                           (long long)pixel_stride, partial, d);
        if (int rc = launch_check("dance_group_norm_act"))
            return rc;
        hipLaunchKernelGGL(k_gn_finish, dim3(groups, b), dim3(64), 0, st, (const double *)partial, stats, groups, d.nch,
                           (double)d.gc * (double)d.hw, (double)eps);
        if (int rc = launch_check("dance_group_norm_act"))
            return rc;
        return with_act(act, [&](auto a) {
            hipLaunchKernelGGL((k_gn_apply<T, W, decltype(a)::value>), grid, dim3(threads), 0, st, (const T *)x,
                               (long long)image_stride, (long long)pixel_stride, (const double *)stats, weight, bias,
                               affine_dtype, (T *)y, d);
            return launch_check("dance_group_norm_act");
        });
    });
}

extern "C" int dance_group_norm_act_backward(const void *dy, int64_t dy_image_stride, int64_t dy_pixel_stride,
                                             const void *x, int64_t image_stride, int64_t pixel_stride, int dtype,
                                             const void *weight, const void *bias, int affine_dtype, int act, int groups,
                                             const double *stats, void *dx, void *dweight, void *dbias, void *ws,
                                             int64_t ws_bytes, int b, int c, int64_t hw, void *stream)
{
    DANCE_REQUIRE(b >= 1 && c >= 1 && hw >= 1 && groups >= 1 && c % groups == 0);
    DANCE_REQUIRE(known_dtype(dtype) && known_dtype(affine_dtype));
    DANCE_REQUIRE(act == DANCE_ACT_NONE || act == DANCE_ACT_RELU || act == DANCE_ACT_SILU);
    DANCE_REQUIRE(vectors_of(c, dtype) <= MAX_VECTORS);
    DANCE_REQUIRE(dy_image_stride >= 0 && dy_pixel_stride >= 0 && image_stride >= 0 && pixel_stride >= 0);
    DANCE_REQUIRE(dy && x && stats && ws && b <= 65535 && groups <= 65535);
    DANCE_REQUIRE(ws_bytes >= dance_group_norm_workspace_bytes(b, c, hw, groups, dtype, 1));
    const GnDims d = dims_of(b, c, hw, groups, dtype);
    DANCE_REQUIRE((long long)b * d.nch < (1ll << 31));
    const int threads = threads_of(d.cv);
    const dim3 grid((unsigned)(b * d.nch));
    hipStream_t st = (hipStream_t)stream;
    float *partial = (float *)ws;
    double *sums = (double *)((char *)ws + whole_16((size_t)b * d.nch * c * 2 * sizeof(float)));
    double *means = sums + (size_t)b * c * 2;
    const char *fn = "dance_group_norm_act_backward";
    return with_type(dtype, c % (dtype == DANCE_F32 ? 4 : 8) == 0, [&](auto t, auto whole) {
        using T = decltype(t);
        constexpr bool W = decltype(whole)::value;
        return with_act(act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            const size_t lds = (size_t)d.rows * d.cv * Vec<T>::N * 2 * sizeof(float);
            if (int rc = dance::allow_lds((const void *)k_gn_grad_sums<T, W, ACT>, lds, fn))
                return rc;
            hipLaunchKernelGGL((k_gn_grad_sums<T, W, ACT>), grid, dim3(threads), lds, st, (const T *)dy,
                               (long long)dy_image_stride, (long long)dy_pixel_stride, (const T *)x,
                               (long long)image_stride, (long long)pixel_stride, stats, weight, bias, affine_dtype,
                               partial, d);
            if (int rc = launch_check(fn))
                return rc;
            hipLaunchKernelGGL(k_gn_grad_finish, dim3(groups, b), dim3(256), 0, st, (const float *)partial, weight,
                               affine_dtype, sums, means, d);
            if (int rc = launch_check(fn))
                return rc;
            if (dweight || dbias) {
                hipLaunchKernelGGL(k_gn_grad_affine, dim3(ceil_div(c, 64)), dim3(64), 0, st, (const double *)sums,
                                   dweight, dbias, affine_dtype, b, c);
                if (int rc = launch_check(fn))
                    return rc;
            }
            if (dx) {
                hipLaunchKernelGGL((k_gn_grad_apply<T, W, ACT>), grid, dim3(threads), 0, st, (const T *)dy,
                                   (long long)dy_image_stride, (long long)dy_pixel_stride, (const T *)x,
                                   (long long)image_stride, (long long)pixel_stride, stats, (const double *)means,
                                   weight, bias, affine_dtype, (T *)dx, d);
                return launch_check(fn);
            }
            return 0;
        });
    });
}
