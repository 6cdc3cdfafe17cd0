// newton_schulz.hip -- orthogonalised updates: X = M / max(|M|_F, eps), then `steps` times
//     A = X X',   Q = a I + b A + c A A,   X <- Q X
// on the smaller side of M (rows r <= columns k of X, M transposed where it is tall), and the Muon step
// around it: momentum and Nesterov's look-ahead on the way in, the parameter update on the way out.
//
// Arithmetic.  The chain multiplies an error of its first step by up to a^4 = 140, so operands of 8 or 11 bits
// are not enough.  Every matrix is carried as split halves hi + lo (p16.h, 22 bits) and every product is three
// f16 MFMAs summed in fp32: the chain's error is then the fp32 chain's (5 steps on 128 x 1152: 1.4e-6 norm-wise
// either way), at 16/3 of the fp32 MFMA rate.  (The same steps taken on A alone, with one product by X at the
// end, would be a third of the work for wide matrices, but small singular values then come out of A, where
// they are squared: 1e-4 .. 1e-2 off.)  Normalisation bounds every entry, so the power-of-two scales that keep
// lo halves normal numbers are constants.
//
// Layout.  A GEMM here is  C[i][j] = sum_k U[i][k] V[j][k].  An operand of `rows` rows is stored
// [plane hi / lo][k / 8][row][8]: the 8 consecutive k of one row an MFMA lane takes are one 16-byte word, the
// 16 rows of a fragment are 256 consecutive bytes, so fragments come straight from L2, without LDS or barriers.
// X is kept twice, with k along its columns (for X X') and along its rows (for Q X); A and Q are symmetric.
// Rows and columns are padded with zeros to whole tiles of 64.
//
// One launch covers matrices of any number of shapes (up to NS_ITEMS): their descriptions travel in the kernel
// arguments, a workgroup finds its matrix from the tile counts.
#include "common.h"
#include "p16.h"

#include <math.h>

namespace {

using dance::launch_check;

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int TILE = 64, LDT = TILE + 1;            // LDS row stride: odd, conflict-free both ways
constexpr int NS_ITEMS = 48;                        // 48 descriptions fit the 4 KB of kernel arguments
constexpr int NS_SLICES = 64;                       // workgroups that share a matrix's norm
constexpr int X_EXP = 14;                           // X and A are stored times 2^14: |X|_2 < 2 (1.21 with the usual
                                                    // coefficients) keeps |A| below 65504 / 2^14

struct NsItem {
    const void *src;            // M, or the gradient
    void *momentum;             // Muon: the momentum buffer
    void *dst;                  // the result, or the parameter
    char *ws;
    int m, n;
    float scale;                // Muon: lr sqrt(max(1, m / n))
    int pad;
};

struct NsTable {
    NsItem it[NS_ITEMS];
    int square[NS_ITEMS];       // workgroups up to and including item i: lower tiles of the r x r matrices
    int rect[NS_ITEMS];         // tiles of the r x k matrices
    int slices[NS_ITEMS];       // slices of the norm
    int count, dtype;
    long long row_stride, col_stride;                // of src, orthogonalize only
    int muon, nesterov;
    float momentum, fresh, keep;        // mu, 1 - mu, 1 - lr weight_decay
    float a, b, c, q_mul;       // Q is stored times q_mul, a power of two
    double eps;
};
static_assert(sizeof(NsTable) <= 3840, "kernel arguments");

// A matrix's own part of the workspace
struct NsDims {
    int r, k, rp, kp, tall;
};

__host__ __device__ inline NsDims ns_dims(int m, int n)
{
    NsDims d;
    d.tall = m > n;
    d.r = d.tall ? n : m;
    d.k = d.tall ? m : n;
    d.rp = (d.r + TILE - 1) / TILE * TILE;
    d.kp = (d.k + TILE - 1) / TILE * TILE;
    return d;
}

struct NsSpace {
    double *sums;               // NS_SLICES partial sums of squares
    _Float16 *a, *q;            // [2][rp / 8][rp][8]
    _Float16 *xk[2], *xr[2];    // [2][kp / 8][rp][8], [2][rp / 8][kp][8]: this step's and the next one's
};

__host__ __device__ inline size_t ns_space(char *ws, const NsDims &d, NsSpace &s)
{
    size_t at = 0;
    s.sums = (double *)(ws + at);
    at += NS_SLICES * sizeof(double);
    const size_t square = (size_t)d.rp * d.rp * 4, rect = (size_t)d.rp * d.kp * 4;
    s.a = (_Float16 *)(ws + at);
    at += square;
    s.q = (_Float16 *)(ws + at);
    at += square;
    for (int i = 0; i < 2; ++i) {
        s.xk[i] = (_Float16 *)(ws + at);
        at += rect;
        s.xr[i] = (_Float16 *)(ws + at);
        at += rect;
    }
    return at;
}

// ---------------------------------------------------------------------------------- which matrix
// The item that workgroup `bid` belongs to and its number there
__device__ __forceinline__ int find_item(const int *ends, int count, int bid, int &local)
{
    const int lane = threadIdx.x & 63;
    const unsigned long long behind = __ballot(lane < count && ends[lane < count ? lane : 0] <= bid);
    const int i = __builtin_amdgcn_readfirstlane(__popcll(behind));
    local = bid - (i ? ends[i - 1] : 0);
    return i;
}

// tile t of the lower triangle of a square of tiles, row by row -> (i, j), j <= i
__device__ __forceinline__ void lower_tile(int t, int &i, int &j)
{
    i = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while (i * (i + 1) / 2 > t)
        --i;
    while ((i + 1) * (i + 2) / 2 <= t)
        ++i;
    j = t - i * (i + 1) / 2;
}

// ------------------------------------------------------------------------------------- elements
__device__ __forceinline__ float load_as_float(const void *p, int dtype, long long i)
{
    if (dtype == DANCE_F32)
        return ((const float *)p)[i];
    return dtype == DANCE_F16 ? (float)((const _Float16 *)p)[i] : (float)((const __bf16 *)p)[i];
}

__device__ __forceinline__ void store_as(void *p, int dtype, long long i, float v)
{
    if (dtype == DANCE_F32)
        ((float *)p)[i] = v;
    else if (dtype == DANCE_F16)
        ((_Float16 *)p)[i] = (_Float16)v;
    else
        ((__bf16 *)p)[i] = (__bf16)v;
}

// Element (row, col) of what is orthogonalised.  Muon: m = mu m + (1 - mu) g (returned in `mom`), and the update
// u = mu m + (1 - mu) g with Nesterov, m without; both in fp32, the unrounded m in u.
__device__ __forceinline__ float element(const NsTable &t, const NsItem &it, int row, int col, float &mom)
{
    if (!t.muon)
        return load_as_float(it.src, t.dtype, row * t.row_stride + col * t.col_stride);
    const long long e = (long long)row * it.n + col;
    const float g = load_as_float(it.src, t.dtype, e) * t.fresh;
    mom = fmaf(load_as_float(it.momentum, t.dtype, e), t.momentum, g);
    return t.nesterov ? fmaf(mom, t.momentum, g) : mom;
}

// sums[slice] = sum of squares of a slice of the matrix, in fp64: no square over- or underflows
__global__ __launch_bounds__(256) void k_ns_norm(NsTable t)
{
    __shared__ double red[4];
    int slice;
    const int i = find_item(t.slices, t.count, blockIdx.x, slice);
    const NsItem it = t.it[i];
    NsSpace s;
    ns_space(it.ws, ns_dims(it.m, it.n), s);
    const unsigned total = (unsigned)it.m * (unsigned)it.n, slices = t.slices[i] - (i ? t.slices[i - 1] : 0);
    double acc = 0.0;
#pragma unroll 4
    for (unsigned e = slice * 256u + threadIdx.x; e < total; e += slices * 256u) {
        float mom;
        const float u = element(t, it, (int)(e / (unsigned)it.n), (int)(e % (unsigned)it.n), mom);
        acc = fma((double)u, (double)u, acc);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        acc += __shfl_xor(acc, m, 64);
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0)
        s.sums[slice] = red[0] + red[1] + red[2] + red[3];
}

// ------------------------------------------------------------------------------ tiles in LDS, split
// word: 8 consecutive k of one row, in both planes
__device__ __forceinline__ void put_word(_Float16 *p, size_t plane, const float (&x)[8])
{
    h8 hi, lo;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        _Float16 h, l;
        dance::split_half(x[i], h, l);
        hi[i] = h;
        lo[i] = l;
    }
    *reinterpret_cast<h8 *>(p) = hi;
    *reinterpret_cast<h8 *>(p + plane) = lo;
}

// tile [i][j] -> operand with rows i (from i0 of `rows`) and k along j (from j0)
__device__ __forceinline__ void put_rows(_Float16 *out, size_t plane, int rows, int i0, int j0, const float (*tile)[LDT])
{
    for (int w = threadIdx.x; w < TILE * TILE / 8; w += blockDim.x) {
        const int i = w & (TILE - 1), jb = w / TILE;
        float x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            x[q] = tile[i][jb * 8 + q];
        put_word(out + ((size_t)(j0 / 8 + jb) * rows + i0 + i) * 8, plane, x);
    }
}

// tile [i][j] -> operand with rows j (from j0 of `rows`) and k along i (from i0)
__device__ __forceinline__ void put_cols(_Float16 *out, size_t plane, int rows, int i0, int j0, const float (*tile)[LDT])
{
    for (int w = threadIdx.x; w < TILE * TILE / 8; w += blockDim.x) {
        const int j = w & (TILE - 1), ib = w / TILE;
        float x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            x[q] = tile[ib * 8 + q][j];
        put_word(out + ((size_t)(i0 / 8 + ib) * rows + j0 + j) * 8, plane, x);
    }
}

__device__ __forceinline__ double norm_of(const double *sums, int slices, double eps)
{
    const int lane = threadIdx.x & 63;
    double s = lane < slices ? sums[lane] : 0.0;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        s += __shfl_xor(s, m, 64);
    s = sqrt(s);
    return s < eps ? eps : s;                       // (a NaN stays one)
}

// M / norm -> the first X, a tile of 64 x 64 a workgroup; Muon: the momentum is stored on the way
__global__ __launch_bounds__(256) void k_ns_pack(NsTable t)
{
    __shared__ float tile[TILE][LDT];
    int local;
    const int n_item = find_item(t.rect, t.count, blockIdx.x, local);
    const NsItem it = t.it[n_item];
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, s);
    const int across = d.kp / TILE, i0 = local / across * TILE, j0 = local % across * TILE;
    const double inv = ldexp(1.0, X_EXP) / norm_of(s.sums, t.slices[n_item] - (n_item ? t.slices[n_item - 1] : 0), t.eps);
#pragma unroll 4
    for (int e = threadIdx.x; e < TILE * TILE; e += 256) {
        // neighbouring threads take neighbours of a row of M
        const int hi = e / TILE, lo = e & (TILE - 1), i = d.tall ? lo : hi, j = d.tall ? hi : lo;
        float x = 0.0f;
        if (i0 + i < d.r && j0 + j < d.k) {
            const int row = d.tall ? j0 + j : i0 + i, col = d.tall ? i0 + i : j0 + j;
            float mom;
            x = (float)((double)element(t, it, row, col, mom) * inv);
            if (t.muon)
                store_as(it.momentum, t.dtype, (long long)row * it.n + col, mom);
        }
        tile[i][j] = x;
    }
    __syncthreads();
    const size_t plane = (size_t)d.rp * d.kp;
    put_rows(s.xk[0], plane, d.rp, i0, j0, tile);
    put_cols(s.xr[0], plane, d.kp, i0, j0, tile);
}

// ------------------------------------------------------------------------------------------- GEMM
// acc += U[i..][k0 .. k0 + 32 steps) V[j..]': the wave's IT x JT fragments of 16 x 16.
// u, v: this lane's words of the first fragments at k0 ((lane >> 4) is the k block, (lane & 15) the row)
template <int IT, int JT>
__device__ __forceinline__ void wave_gemm(f32x4 (&acc)[IT][JT], const _Float16 *u, size_t u_plane, int u_rows,
                                          const _Float16 *v, size_t v_plane, int v_rows, int steps)
{
    h8 ah[IT], al[IT], bh[JT], bl[JT];
    auto load = [&](int s) {
        const _Float16 *us = u + (size_t)s * 4 * u_rows * 8, *vs = v + (size_t)s * 4 * v_rows * 8;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            ah[i] = *reinterpret_cast<const h8 *>(us + i * 128);
            al[i] = *reinterpret_cast<const h8 *>(us + u_plane + i * 128);
        }
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            bh[j] = *reinterpret_cast<const h8 *>(vs + j * 128);
            bl[j] = *reinterpret_cast<const h8 *>(vs + v_plane + j * 128);
        }
    };
    if (steps <= 0)
        return;
    load(0);
    for (int s = 0; s < steps; ++s) {
        h8 ch[IT], cl[IT], dh[JT], dl[JT];
#pragma unroll
        for (int i = 0; i < IT; ++i) {
            ch[i] = ah[i];
            cl[i] = al[i];
        }
#pragma unroll
        for (int j = 0; j < JT; ++j) {
            dh[j] = bh[j];
            dl[j] = bl[j];
        }
        if (s + 1 < steps)
            load(s + 1);
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(cl[i], dh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch[i], dl[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ch[i], dh[j], acc[i][j], 0, 0, 0);
            }
    }
}

// A 64 x 64 tile of U V' by WM x WN waves on its parts times WK waves on shares of k, summed into `tile`
// (one buffer of TILE x LDT floats a share of k; the sum ends up in the first)
template <int WM, int WN, int WK>
__device__ __forceinline__ void tile_gemm(float (*tile)[LDT], const _Float16 *u, size_t u_plane, int u_rows, int i0,
                                          const _Float16 *v, size_t v_plane, int v_rows, int j0, int k)
{
    constexpr int IT = TILE / 16 / WM, JT = TILE / 16 / WN;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wk = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
    const int steps = k / 32, s0 = steps * wk / WK, s1 = steps * (wk + 1) / WK;
    f32x4 acc[IT][JT];
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < JT; ++j)
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const size_t kb = (size_t)s0 * 4 + (lane >> 4);
    wave_gemm<IT, JT>(acc, u + (kb * u_rows + i0 + wm * IT * 16 + (lane & 15)) * 8, u_plane, u_rows,
                      v + (kb * v_rows + j0 + wn * JT * 16 + (lane & 15)) * 8, v_plane, v_rows, s1 - s0);
    // a lane holds 4 consecutive rows of one column of every fragment
    float (*mine)[LDT] = tile + wk * TILE;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
        for (int j = 0; j < JT; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                mine[(wm * IT + i) * 16 + (lane >> 4) * 4 + q][(wn * JT + j) * 16 + (lane & 15)] = acc[i][j][q];
    __syncthreads();
    if (WK > 1) {
        for (int e = threadIdx.x; e < TILE * TILE; e += blockDim.x) {
            const int i = e / TILE, j = e & (TILE - 1);
            float s = tile[i][j];
#pragma unroll
            for (int w = 1; w < WK; ++w)
                s += tile[w * TILE + i][j];
            tile[i][j] = s;
        }
        __syncthreads();
    }
}

template <typename F> __device__ __forceinline__ void each(float (*tile)[LDT], F &&f)
{
    for (int e = threadIdx.x; e < TILE * TILE; e += blockDim.x) {
        const int i = e / TILE, j = e & (TILE - 1);
        tile[i][j] = f(i, j, tile[i][j]);
    }
    __syncthreads();
}

// a symmetric matrix's tile at (i0, j0) and its mirror image
__device__ __forceinline__ void put_symmetric(_Float16 *out, int rp, int i0, int j0, const float (*tile)[LDT])
{
    const size_t plane = (size_t)rp * rp;
    put_rows(out, plane, rp, i0, j0, tile);
    if (i0 != j0)
        put_cols(out, plane, rp, i0, j0, tile);
}

constexpr int GRAM_WK = 8;

// A = X X', lower tiles
__global__ __launch_bounds__(64 * GRAM_WK) void k_ns_gram(NsTable t, int step)
{
    extern __shared__ __align__(16) float lds[];
    float (*tile)[LDT] = reinterpret_cast<float (*)[LDT]>(lds);
    int local, ti, tj;
    const NsItem it = t.it[find_item(t.square, t.count, blockIdx.x, local)];
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, s);
    lower_tile(local, ti, tj);
    const _Float16 *x = step & 1 ? s.xk[1] : s.xk[0];
    const size_t plane = (size_t)d.rp * d.kp;
    tile_gemm<1, 1, GRAM_WK>(tile, x, plane, d.rp, ti * TILE, x, plane, d.rp, tj * TILE, d.kp);
    const float mul = dance::pow2f(-X_EXP);
    each(tile, [&](int, int, float v) { return v * mul; });
    put_symmetric(s.a, d.rp, ti * TILE, tj * TILE, tile);
}

// Q = a I + b A + c A A, lower tiles
__global__ __launch_bounds__(512) void k_ns_poly(NsTable t)
{
    extern __shared__ __align__(16) float lds[];
    float (*tile)[LDT] = reinterpret_cast<float (*)[LDT]>(lds);
    int local, ti, tj;
    const NsItem it = t.it[find_item(t.square, t.count, blockIdx.x, local)];
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, s);
    lower_tile(local, ti, tj);
    const size_t plane = (size_t)d.rp * d.rp;
    const int i0 = ti * TILE, j0 = tj * TILE;
    tile_gemm<2, 2, 2>(tile, s.a, plane, d.rp, i0, s.a, plane, d.rp, j0, d.rp);
    const float ca = t.c * dance::pow2f(-2 * X_EXP), ba = t.b * dance::pow2f(-X_EXP);
    each(tile, [&](int i, int j, float v) {
        const _Float16 *p = s.a + ((size_t)((j0 + j) / 8) * d.rp + i0 + i) * 8 + (j & 7);
        const float aij = (float)p[0] + (float)p[plane];
        v = fmaf(ca, v, ba * aij);
        if (i0 + i == j0 + j && i0 + i < d.r)
            v += t.a;
        return v * t.q_mul;
    });
    put_symmetric(s.q, d.rp, i0, j0, tile);
}

// X <- Q X, a tile of 64 x 64 a workgroup; the last step writes the result
__global__ __launch_bounds__(256) void k_ns_apply(NsTable t, int step, int last)
{
    __shared__ __align__(16) float tile[TILE][LDT];
    int local;
    const NsItem it = t.it[find_item(t.rect, t.count, blockIdx.x, local)];
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, s);
    const int down = d.rp / TILE, i0 = local % down * TILE, j0 = local / down * TILE;
    const size_t square = (size_t)d.rp * d.rp, rect = (size_t)d.rp * d.kp;
    tile_gemm<2, 2, 1>(tile, s.q, square, d.rp, i0, step & 1 ? s.xr[1] : s.xr[0], rect, d.kp, j0, d.rp);
    const float mul = 1.0f / t.q_mul;
    if (!last) {
        each(tile, [&](int, int, float v) { return v * mul; });
        put_rows(step & 1 ? s.xk[0] : s.xk[1], rect, d.rp, i0, j0, tile);
        put_cols(step & 1 ? s.xr[0] : s.xr[1], rect, d.kp, i0, j0, tile);
        return;
    }
    const float out = mul * dance::pow2f(-X_EXP);
    for (int e = threadIdx.x; e < TILE * TILE; e += 256) {
        const int hi = e / TILE, lo = e & (TILE - 1), i = d.tall ? lo : hi, j = d.tall ? hi : lo;
        if (i0 + i >= d.r || j0 + j >= d.k)
            continue;
        const long long at = d.tall ? (long long)(j0 + j) * it.n + i0 + i : (long long)(i0 + i) * it.n + j0 + j;
        float v = tile[i][j] * out;
        if (t.muon)
            v = fmaf(-it.scale, v, load_as_float(it.dst, t.dtype, at) * t.keep);
        store_as(it.dst, t.dtype, at, v);
    }
}

// ------------------------------------------------------------------------------------------- host
bool known_dtype(int t) { return t == DANCE_F32 || t == DANCE_F16 || t == DANCE_BF16; }

int64_t space_of(int m, int n)
{
    NsSpace s;
    return (int64_t)ns_space(nullptr, ns_dims(m, n), s);
}

// the largest power of two that keeps Q's entries, |Q| <= |a| + 1.5 |b| + 2.25 |c|, within fp16
float q_scale(float a, float b, float c)
{
    const double most = fabs((double)a) + 1.5 * fabs((double)b) + 2.25 * fabs((double)c);
    return most > 0.0 ? (float)exp2(fmin(14.0, floor(log2(60000.0 / most)))) : 1.0f;
}

// the chain over the items of a table whose sizes, pointers and settings are set
int run_chain(NsTable &t, int steps, hipStream_t st, const char *fn)
{
    int square = 0, rect = 0, slices = 0;
    for (int i = 0; i < t.count; ++i) {
        const NsDims d = ns_dims(t.it[i].m, t.it[i].n);
        const int down = d.rp / TILE, across = d.kp / TILE;
        const long long total = (long long)t.it[i].m * t.it[i].n, want = (total + 4095) / 4096;
        if ((long long)rect + (long long)down * across >= (1ll << 31) || (long long)square + (long long)down * (down + 1) / 2 >= (1ll << 31))
            return dance::fail((int)hipErrorInvalidValue, fn, "too many tiles");
        square += down * (down + 1) / 2;
        rect += down * across;
        slices += (int)(want < NS_SLICES ? want : NS_SLICES);
        t.square[i] = square;
        t.rect[i] = rect;
        t.slices[i] = slices;
    }
    const size_t gram_lds = GRAM_WK * TILE * LDT * sizeof(float), poly_lds = 2 * TILE * LDT * sizeof(float);
    if (int rc = dance::allow_lds((const void *)k_ns_gram, gram_lds, fn))
        return rc;
    hipLaunchKernelGGL(k_ns_norm, dim3(slices), dim3(256), 0, st, t);
    if (int rc = launch_check(fn))
        return rc;
    hipLaunchKernelGGL(k_ns_pack, dim3(rect), dim3(256), 0, st, t);
    if (int rc = launch_check(fn))
        return rc;
    for (int s = 0; s < steps; ++s) {
        hipLaunchKernelGGL(k_ns_gram, dim3(square), dim3(64 * GRAM_WK), gram_lds, st, t, s);
        if (int rc = launch_check(fn))
            return rc;
        hipLaunchKernelGGL(k_ns_poly, dim3(square), dim3(512), poly_lds, st, t);
        if (int rc = launch_check(fn))
            return rc;
        hipLaunchKernelGGL(k_ns_apply, dim3(rect), dim3(256), 0, st, t, s, (int)(s + 1 == steps));
        if (int rc = launch_check(fn))
            return rc;
    }
    return 0;
}

bool usable(double a, double b, double c) { return isfinite(a) && isfinite(b) && isfinite(c); }

}  // namespace

extern "C" int64_t dance_orthogonalize_workspace_bytes(int batch, int m, int n)
{
    if (batch <= 0 || m <= 0 || n <= 0 || (long long)m * n >= (1ll << 31))
        return 0;
    return (batch < NS_ITEMS ? batch : NS_ITEMS) * space_of(m, n);
}

extern "C" int dance_orthogonalize(const void *x, int64_t batch_stride, int64_t row_stride, int64_t col_stride,
                                   int dtype, void *out, int batch, int m, int n, int steps, float a, float b, float c,
                                   float eps, void *ws, int64_t ws_bytes, void *stream)
{
    DANCE_REQUIRE(batch >= 0 && m >= 0 && n >= 0 && (long long)m * n < (1ll << 31));
    DANCE_REQUIRE(known_dtype(dtype) && steps >= 1 && steps <= 100 && usable(a, b, c) && eps > 0.0f);
    DANCE_REQUIRE(batch_stride >= 0 && row_stride >= 0 && col_stride >= 0);
    if (batch == 0 || m == 0 || n == 0)
        return 0;
    DANCE_REQUIRE(x && out && ws && ((uintptr_t)ws & 15) == 0);
    DANCE_REQUIRE(ws_bytes >= dance_orthogonalize_workspace_bytes(batch, m, n));
    const int64_t size = dtype == DANCE_F32 ? 4 : 2, space = space_of(m, n);
    for (int b0 = 0; b0 < batch; b0 += NS_ITEMS) {
        NsTable t;
        memset(&t, 0, sizeof t);
        t.count = batch - b0 < NS_ITEMS ? batch - b0 : NS_ITEMS;
        t.dtype = dtype;
        t.row_stride = row_stride;
        t.col_stride = col_stride;
        t.a = a; t.b = b; t.c = c;
        t.q_mul = q_scale(a, b, c);
        t.eps = (double)eps;
        for (int i = 0; i < t.count; ++i) {
            t.it[i].src = (const char *)x + (b0 + i) * batch_stride * size;
            t.it[i].dst = (char *)out + (int64_t)(b0 + i) * m * n * size;
            t.it[i].ws = (char *)ws + i * space;
            t.it[i].m = m;
            t.it[i].n = n;
        }
        if (int rc = run_chain(t, steps, (hipStream_t)stream, __func__))
            return rc;
    }
    return 0;
}

extern "C" int64_t dance_muon_workspace_bytes(const dance_muon_item *items_host, int count)
{
    if (count <= 0 || !items_host)
        return 0;
    int64_t most = 0;
    for (int b0 = 0; b0 < count; b0 += NS_ITEMS) {
        int64_t sum = 0;
        for (int i = b0; i < count && i < b0 + NS_ITEMS; ++i) {
            const int m = items_host[i].rows, n = items_host[i].cols;
            if (m <= 0 || n <= 0 || (long long)m * n >= (1ll << 31))
                return 0;
            sum += space_of(m, n);
        }
        most = sum > most ? sum : most;
    }
    return most;
}

extern "C" int dance_muon_step(const dance_muon_item *items_host, int count, int dtype, double lr, double momentum,
                               int nesterov, double weight_decay, int steps, float a, float b, float c, float eps, void *ws,
                               int64_t ws_bytes, void *stream)
{
    DANCE_REQUIRE(count >= 0 && known_dtype(dtype) && steps >= 1 && steps <= 100 && usable(a, b, c) && eps > 0.0f);
    DANCE_REQUIRE(usable(lr, momentum, weight_decay));
    if (count == 0)
        return 0;
    DANCE_REQUIRE(items_host && ws && ((uintptr_t)ws & 15) == 0);
    for (int i = 0; i < count; ++i) {
        DANCE_REQUIRE(items_host[i].param && items_host[i].grad && items_host[i].momentum);
        DANCE_REQUIRE(items_host[i].rows >= 1 && items_host[i].cols >= 1);
        DANCE_REQUIRE((long long)items_host[i].rows * items_host[i].cols < (1ll << 31));
    }
    DANCE_REQUIRE(ws_bytes >= dance_muon_workspace_bytes(items_host, count));
    for (int b0 = 0; b0 < count; b0 += NS_ITEMS) {
        NsTable t;
        memset(&t, 0, sizeof t);
        t.count = count - b0 < NS_ITEMS ? count - b0 : NS_ITEMS;
        t.dtype = dtype;
        t.muon = 1;
        t.nesterov = nesterov != 0;
        t.momentum = (float)momentum;
        t.fresh = (float)(1.0 - momentum);
        t.keep = (float)(1.0 - lr * weight_decay);
        t.a = a; t.b = b; t.c = c;
        t.q_mul = q_scale(a, b, c);
        t.eps = (double)eps;
        int64_t at = 0;
        for (int i = 0; i < t.count; ++i) {
            const dance_muon_item &h = items_host[b0 + i];
            t.it[i].src = h.grad;
            t.it[i].momentum = h.momentum;
            t.it[i].dst = h.param;
            t.it[i].ws = (char *)ws + at;
            t.it[i].m = h.rows;
            t.it[i].n = h.cols;
            const double shape = h.rows > h.cols ? sqrt((double)h.rows / (double)h.cols) : 1.0;
            t.it[i].scale = (float)(lr * shape);
            at += space_of(h.rows, h.cols);
        }
        if (int rc = run_chain(t, steps, (hipStream_t)stream, __func__))
            return rc;
    }
    return 0;
}
