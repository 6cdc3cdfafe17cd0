// newton_schulz.hip -- orthogonalised updates: X = M / max(|M|_F, eps), then `steps` times
//     A = X X',   Q = a I + b A + c A A,   X <- Q X
// on the smaller side of M (rows r <= columns k of X, M transposed where it is tall), and the Muon step
// around it: momentum and Nesterov's look-ahead on the way in, the parameter update on the way out.
//
// Arithmetic.  The chain multiplies an error of its first step by up to a^4 = 140, so operands of 8 or 11 bits
// are not enough.  Every matrix is carried as split halves hi + lo (p16.h, 22 bits) and every product is three
// f16 MFMAs summed in fp32: the chain's error is then the fp32 chain's (5 steps on 128 x 1152, norm-wise: 0.6e-6
// against 1.3e-6), at 7.5 / 3 of the fp32 rate (f16 and fp32 products of 8192 x 8192: 1153 and 154 TFLOP/s).  (The same steps taken on A alone, with one product by X at the
// end, would be a third of the work for wide matrices, but small singular values then come out of A, where
// they are squared: 1e-4 .. 1e-2 off.)  Normalisation bounds every entry, so the power-of-two scales that keep
// lo halves normal numbers are constants.
//
// Layout.  A GEMM here is  C[i][j] = sum_k U[i][k] V[j][k].  An operand of `rows` rows is stored
// [plane hi / lo][k / 8][row][8]: the 8 consecutive k of one row an MFMA lane takes are one 16-byte word, the
// 16 rows of a fragment are 256 consecutive bytes: memory and LDS hold the same words, a copy moves them as they
// lie and fragments are read without bank conflicts.  X is kept twice, with k along its columns (for X X') and
// along its rows (for Q X); A and Q are symmetric, their products are taken on and below the diagonal.  Rows and
// columns are padded with zeros to whole tiles of 128.
//
// Three kinds of matrices: those whose chain fits one compute unit's LDS (k_ns_small: the whole chain in one
// workgroup, a launch for all of them), those of up to 128 rows (k_ns_narrow: a launch a step and one that adds
// shares), and the others (k_ns_gram, k_ns_sum, k_ns_poly, k_ns_apply).  us, its kind / the next one: 64 x 256 25 / 85,
// 64 of 32 x 288 34 / 184; 128 x 256 87 / 94, 21 of 128 x 1152 105 / 144.
//
// One launch covers matrices of any number of shapes (up to NS_ITEMS): a workgroup finds its matrix from the tile
// counts in a table.  The first kernel gets the table as its arguments and leaves it in the workspace for the
// others: kernel arguments lie in host memory.
#include "common.h"
#include "p16.h"

#include <limits.h>
#include <math.h>

namespace {

using dance::launch_check;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int PAD = 128;                            // rows and columns are padded to whole tiles of the GEMM
constexpr long long MOST_ELEMENTS = INT_MAX - PAD;  // of a matrix: its padded sides fit an int
constexpr int PACK = 64;                            // side of the tiles M is packed by
constexpr int NS_ITEMS = 48;                        // 48 descriptions fit the 4 KB of kernel arguments
constexpr int NS_SLICES = 256;                      // most workgroups that share a matrix's norm
constexpr int X_EXP = 14;                           // X and A are stored times 2^14: |X|_2 < 2 (1.21 with the usual
                                                    // coefficients) keeps |A| below 65504 / 2^14

struct NsItem {
    const void *src;            // M, or the gradient
    void *momentum;             // Muon: the momentum buffer
    void *dst;                  // the result, or the parameter
    char *ws;
    int m, n;
    float scale;                // Muon: lr sqrt(max(1, m / n))
    int split;                  // workgroups that share a tile of A along k
};
static_assert(sizeof(NsItem) == 48, "three words of 16 bytes: find_item");

struct NsTable {
    NsItem it[NS_ITEMS];
    // workgroups up to and including item i, INT_MAX past the last: slices of the norm; shares of a narrow matrix; fours of
    // fragments of the sum; of matrices that are not narrow the pack tiles, lower tiles of A, times split, lower tiles of
    // Q, tiles of X
    int slices[NS_ITEMS], pack[NS_ITEMS], narrow[NS_ITEMS], gram[NS_ITEMS], sum[NS_ITEMS], poly[NS_ITEMS], rect[NS_ITEMS];
    int count, dtype;
    long long row_stride, col_stride;                // of src, orthogonalize only
    int muon, nesterov, steps, gram_side;            // gram_side: of the tiles of A
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
    d.rp = (d.r + PAD - 1) / PAD * PAD;
    d.kp = (d.k + PAD - 1) / PAD * PAD;
    return d;
}

// one tile of rows: k_ns_narrow's
__host__ __device__ inline bool narrow(const NsDims &d) { return d.rp == PAD; }

// tiles of side `side` on and below the diagonal
__host__ __device__ inline int lower_tiles(const NsDims &d, int side) { return d.rp / side * (d.rp / side + 1) / 2; }

struct NsSpace {
    double *sums;               // NS_SLICES partial sums of squares
    float *part;                // [split][lower tile][side * side]: a tile of A summed over a share of k
    _Float16 *a, *q;            // [2][rp / 8][rp][8]
    _Float16 *xk[2], *xr[2];    // [2][kp / 8][rp][8], [2][rp / 8][kp][8]: this step's and the next one's (narrow: xr[0] alone)
};

__host__ __device__ inline size_t ns_space(char *ws, const NsDims &d, int split, NsSpace &s)
{
    size_t at = 0;
    s.sums = (double *)(ws + at);
    at += NS_SLICES * sizeof(double);
    s.part = (float *)(ws + at);
    at += (size_t)split * lower_tiles(d, PAD) * PAD * PAD * sizeof(float);         // (smaller tiles are less)
    const size_t square = (size_t)d.rp * d.rp * 4, rect = (size_t)d.rp * d.kp * 4;
    s.a = (_Float16 *)(ws + at);
    at += square;
    s.q = (_Float16 *)(ws + at);
    at += narrow(d) ? 0 : square;
    for (int i = 0; i < (narrow(d) ? 1 : 2); ++i) {
        s.xk[i] = (_Float16 *)(ws + at);
        at += narrow(d) ? 0 : rect;
        s.xr[i] = (_Float16 *)(ws + at);
        at += rect;
    }
    return at;
}

// ---------------------------------------------------------------------------------- which matrix
// Workgroups are dealt to the chip's 8 dies in turn: number them so that a die's are neighbours, which share
// operands in its L2
__device__ __forceinline__ int die_order()
{
    const int n = gridDim.x, die = blockIdx.x & 7, q = n >> 3, rest = n & 7;
    return die * q + min(die, rest) + ((int)blockIdx.x >> 3);
}

// The item that workgroup `bid` belongs to, its index and the workgroup's number there.  ends: past the last item they
// hold INT_MAX.  A lane reads each item's end and description, the right one is broadcast: one round trip to memory.
__device__ __forceinline__ NsItem find_item(const NsTable &t, const int *ends, int bid, int &index, int &local)
{
    const int lane = min((int)(threadIdx.x & 63), NS_ITEMS - 1), end = ends[lane];
    const int4 *from = reinterpret_cast<const int4 *>(&t.it[lane]);
    const int4 w[3] = {from[0], from[1], from[2]};
    index = __builtin_amdgcn_readfirstlane(min(__popcll(__ballot(end <= bid)), NS_ITEMS - 1));
    local = bid - (index ? __builtin_amdgcn_readlane(end, index - 1) : 0);
    union {
        NsItem it;
        int v[12];
    } u;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        u.v[4 * i] = __builtin_amdgcn_readlane(w[i].x, index);
        u.v[4 * i + 1] = __builtin_amdgcn_readlane(w[i].y, index);
        u.v[4 * i + 2] = __builtin_amdgcn_readlane(w[i].z, index);
        u.v[4 * i + 3] = __builtin_amdgcn_readlane(w[i].w, index);
    }
    return u.it;
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
// Element (row, col) of what is orthogonalised.  Muon: m = mu m + (1 - mu) g (returned in `mom`), and the update
// u = mu m + (1 - mu) g with Nesterov, m without; both in fp32, the unrounded m in u.
template <typename T>
__device__ __forceinline__ float element(const NsTable &t, const NsItem &it, int row, int col, float &mom)
{
    const long long e = t.muon ? (long long)row * it.n + col : row * t.row_stride + col * t.col_stride;
    float g = (float)((const T *)it.src)[e];
    if (!t.muon)
        return g;
    g *= t.fresh;
    mom = fmaf((float)((const T *)it.momentum)[e], t.momentum, g);
    return t.nesterov ? fmaf(mom, t.momentum, g) : mom;
}

__device__ __forceinline__ double wave_sum(double x)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        x += __shfl_xor(x, m, 64);
    return x;
}

// N consecutive elements of a dense matrix, at any alignment
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Word { T v[16 / sizeof(T)]; };

// What `element` is, for a vector of a dense matrix: g, and in Muon m, which becomes the new momentum -> x
template <typename T>
__device__ __forceinline__ void elements(const NsTable &t, const Word<T> &g, Word<T> &m, float (&x)[16 / sizeof(T)])
{
#pragma unroll
    for (int q = 0; q < (int)(16 / sizeof(T)); ++q) {
        x[q] = (float)g.v[q];
        if (t.muon) {
            x[q] *= t.fresh;
            const float mm = fmaf((float)m.v[q], t.momentum, x[q]);
            m.v[q] = (T)mm;
            x[q] = t.nesterov ? fmaf(mm, t.momentum, x[q]) : mm;
        }
    }
}

// the vector of the gradient and of the momentum from element e on
template <typename T>
__device__ __forceinline__ void load_words(const NsTable &t, const NsItem &it, long long e, Word<T> &g, Word<T> &m)
{
    g = *reinterpret_cast<const Word<T> *>((const T *)it.src + e);
    if (t.muon)
        m = *reinterpret_cast<const Word<T> *>((const T *)it.momentum + e);
}

// sums[slice] = sum of squares of a slice of the matrix, in fp64: no square over- or underflows.  DENSE: whole
// vectors first, the rest one by one; otherwise any strides.  Bound by its start and its loads: 5.9 us for 12.4 MB.
template <typename T, bool DENSE> __global__ __launch_bounds__(256) void k_ns_norm(NsTable t, NsTable *kept)
{
    constexpr int N = 16 / sizeof(T);
    __shared__ double red[4];
    int i, slice;
    const NsItem it = find_item(t, t.slices, blockIdx.x, i, slice);
    NsSpace s;
    ns_space(it.ws, ns_dims(it.m, it.n), it.split, s);
    if (blockIdx.x == 0)
        for (int w = threadIdx.x; w < (int)(sizeof(NsTable) / 4); w += 256)
            ((int *)kept)[w] = ((const int *)&t)[w];
    const unsigned total = (unsigned)it.m * (unsigned)it.n, slices = t.slices[i] - (i ? t.slices[i - 1] : 0);
    const unsigned first = slice * 256u + threadIdx.x, step = slices * 256u, vectors = DENSE ? total / N : 0u;
    double acc = 0.0;
    if (DENSE)
#pragma unroll 4
        for (unsigned v = first; v < vectors; v += step) {
            float x[N];
            Word<T> g, m;
            load_words<T>(t, it, (long long)v * N, g, m);
            elements<T>(t, g, m, x);
#pragma unroll
            for (int q = 0; q < N; ++q)
                acc = fma((double)x[q], (double)x[q], acc);
        }
    for (unsigned e = vectors * N + first; e < total; e += step) {
        float mom;
        const float u = element<T>(t, it, (int)(e / (unsigned)it.n), (int)(e % (unsigned)it.n), mom);
        acc = fma((double)u, (double)u, acc);
    }
    acc = wave_sum(acc);
    if ((threadIdx.x & 63) == 0)
        red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0)
        s.sums[slice] = red[0] + red[1] + red[2] + red[3];
}

// ------------------------------------------------------------------------------ tiles in LDS, split
// What hi = fp16(x) leaves of x, exactly: one v_fma_mix_f32, which reads the half as it lies (with a constant factor
// the compiler makes a conversion and a subtraction of it).  With the two conversions of v_cvt_pk_f16_f32 a pair of
// values is split by four instructions; the epilogues of the products are bound by them.
__device__ __forceinline__ float rest_of(_Float16 hi, float x)
{
    float minus = -1.0f;
    asm("" : "+s"(minus));
    return fmaf((float)hi, minus, x);
}

__device__ __forceinline__ unsigned pack2(float a, float b) { return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{a, b}, h2)); }

// x as a value of its own: out of a product the compiler would else round hi in one go (v_fma_mixlo_f16), and for one of
// its two uses only
__device__ __forceinline__ float settled(float x)
{
    asm("" : "+v"(x));
    return x;
}

// hi in the low half, lo in the high one: dance::split_half as one word
__device__ __forceinline__ unsigned split_word(float value)
{
    const float x = settled(value);
    return pack2(x, rest_of((_Float16)x, x));
}

// four values' halves, two of one plane a word
struct Quad {
    unsigned hi[2], lo[2];
};

__device__ __forceinline__ Quad split4(const f32x4 &x)
{
    Quad r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float a = settled(x[2 * i]), b = settled(x[2 * i + 1]);
        const h2 h = __builtin_convertvector(f32x2{a, b}, h2);
        r.hi[i] = __builtin_bit_cast(unsigned, h);
        r.lo[i] = pack2(rest_of(h[0], a), rest_of(h[1], b));
    }
    return r;
}

// c v + b A of an entry, A from its halves
__device__ __forceinline__ float poly_of(float c, float v, float b, _Float16 hi, _Float16 lo)
{
    return fmaf((float)hi, b, fmaf((float)lo, b, c * v));
}

__device__ __forceinline__ unsigned hi_pair(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ unsigned lo_pair(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// 8 (4) consecutive k of one row into both planes
__device__ __forceinline__ void put8(_Float16 *p, size_t plane, const unsigned (&x)[8])
{
    *reinterpret_cast<uint4 *>(p) = uint4{hi_pair(x[0], x[1]), hi_pair(x[2], x[3]), hi_pair(x[4], x[5]), hi_pair(x[6], x[7])};
    *reinterpret_cast<uint4 *>(p + plane) = uint4{lo_pair(x[0], x[1]), lo_pair(x[2], x[3]), lo_pair(x[4], x[5]), lo_pair(x[6], x[7])};
}

__device__ __forceinline__ void put4(_Float16 *p, size_t plane, const Quad &x)
{
    *reinterpret_cast<uint2 *>(p) = uint2{x.hi[0], x.hi[1]};
    *reinterpret_cast<uint2 *>(p + plane) = uint2{x.lo[0], x.lo[1]};
}

// 4 x 4 halves over 4 neighbouring lanes transposed: lane l's half q becomes lane q's half l
__device__ __forceinline__ void transpose4(unsigned (&x)[2])
{
    const bool odd = threadIdx.x & 1, upper = threadIdx.x & 2;
    // the second word of a lane against the first of the one two further
    const unsigned got = (unsigned)__builtin_amdgcn_mov_dpp((int)(upper ? x[0] : x[1]), 0x4E, 0xf, 0xf, true);     // 2 3 0 1
    x[0] = upper ? got : x[0];
    x[1] = upper ? x[1] : got;
    // both words' low halves of an even lane and its neighbour, or their high ones
    const unsigned pick = odd ? 0x03020706u : 0x05040100u;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const unsigned other = (unsigned)__builtin_amdgcn_mov_dpp((int)x[i], 0xB1, 0xf, 0xf, true);                // 1 0 3 2
        x[i] = __builtin_amdgcn_perm(other, x[i], pick);
    }
}

__device__ __forceinline__ void transpose4(Quad &x)
{
    transpose4(x.hi);
    transpose4(x.lo);
}

// tile [I][J] of split words in LDS, row stride J + 1 (odd: conflict-free both ways) -> operand with rows i (from i0
// of `rows`) and k along j (from j0).  By T threads.
template <int I, int J, int T>
__device__ __forceinline__ void put_rows(_Float16 *out, size_t plane, int rows, int i0, int j0, const unsigned *tile,
                                         int thread = threadIdx.x)
{
    const int i = thread % I, jb0 = thread / I;
    const unsigned *from = tile + i * (J + 1) + jb0 * 8;
    _Float16 *to = out + ((size_t)(j0 / 8 + jb0) * rows + i0 + i) * 8;
    const size_t step = (size_t)(T / I) * rows * 8;
#pragma unroll 4
    for (int n = 0; n < I * J / 8 / T; ++n) {
        unsigned x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            x[q] = from[n * (T / I) * 8 + q];
        put8(to, plane, x);
        to += step;
    }
}

// the same tile -> operand with rows j (from j0 of `rows`) and k along i (from i0)
template <int I, int J, int T>
__device__ __forceinline__ void put_cols(_Float16 *out, size_t plane, int rows, int i0, int j0, const unsigned *tile,
                                         int thread = threadIdx.x)
{
    const int j = thread % J, ib0 = thread / J;
    const unsigned *from = tile + ib0 * 8 * (J + 1) + j;
    _Float16 *to = out + ((size_t)(i0 / 8 + ib0) * rows + j0 + j) * 8;
    const size_t step = (size_t)(T / J) * rows * 8;
#pragma unroll 4
    for (int n = 0; n < I * J / 8 / T; ++n) {
        unsigned x[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            x[q] = from[(n * (T / J) * 8 + q) * (J + 1)];
        put8(to, plane, x);
        to += step;
    }
}

// 1 / max(norm, eps) as a power of two and a factor within (1, 2]: the exponents of M need not fit those of fp32's
// reciprocals
struct Scale {
    int exp;
    float by;
    __device__ float operator()(float x) const { return ldexpf(x, exp) * by; }
};

// sum: of the squares
__device__ __forceinline__ Scale scale_of(double sum, double eps)
{
    double norm = sqrt(sum);
    norm = norm < eps ? eps : norm;                 // (a NaN stays one)
    int e;
    const double m = frexp(norm, &e);
    return Scale{X_EXP - e, 1.0f / (float)m};
}

// 1 / norm of an item, by all lanes of a wave
__device__ __forceinline__ Scale item_scale(const NsTable &t, const NsSpace &s, int n_item)
{
    const int slices = t.slices[n_item] - (n_item ? t.slices[n_item - 1] : 0);
    double sum = 0.0;
    for (int i = threadIdx.x & 63; i < slices; i += 64)
        sum += s.sums[i];
    return scale_of(wave_sum(sum), t.eps);
}

// A square tile of M / norm, rows i and columns j of X from (i0, j0) on, as split words in LDS, row stride SIDE + 1;
// Muon: the momentum is stored on the way.  N neighbours of a row of M at once: along j, or along i where M is tall.
template <typename T, bool DENSE, int SIDE, int THREADS>
__device__ __forceinline__ void first_tile(const NsTable &t, const NsItem &it, const NsDims &d, Scale scaled, int i0, int j0,
                                           unsigned *tile)
{
    constexpr int N = DENSE ? 16 / sizeof(T) : 1, ACROSS = SIDE / N, DOWN = THREADS / ACROSS, WORDS = SIDE / DOWN, LD = SIDE + 1;
    constexpr int FLY = DENSE ? WORDS : WORDS < 8 ? WORDS : 8;               // loads under way
    const int step_j = d.tall ? LD : 1, step_i = d.tall ? 1 : LD;           // of a row and a column of M in the tile
    const int rr = threadIdx.x / ACROSS, cc = threadIdx.x % ACROSS * N;
    const int row0 = (d.tall ? j0 : i0) + rr, col = (d.tall ? i0 : j0) + cc;
    unsigned *to = tile + rr * step_i + cc * step_j;
#pragma unroll 1
    for (int first = 0; first < WORDS; first += FLY) {
        float x[FLY][16 / sizeof(T)] = {};
        if constexpr (DENSE) {
            const long long e = (long long)row0 * it.n + col, down = (long long)DOWN * it.n;
            Word<T> g[FLY], m[FLY];
#pragma unroll
            for (int w = 0; w < FLY; ++w)
                if (row0 + w * DOWN < it.m && col + N <= it.n)
                    load_words<T>(t, it, e + w * down, g[w], m[w]);
#pragma unroll
            for (int w = 0; w < FLY; ++w) {
                if (row0 + w * DOWN < it.m && col + N <= it.n) {
                    elements<T>(t, g[w], m[w], x[w]);
                    if (t.muon)
                        *reinterpret_cast<Word<T> *>((T *)it.momentum + e + w * down) = m[w];
                } else if (row0 + w * DOWN < it.m && col < it.n) {           // a row's last ones
#pragma unroll
                    for (int q = 0; q < N - 1; ++q)
                        if (col + q < it.n) {
                            float mom;
                            x[w][q] = element<T>(t, it, row0 + w * DOWN, col + q, mom);
                            if (t.muon)
                                ((T *)it.momentum)[e + w * down + q] = (T)mom;
                        }
                }
            }
        } else {
#pragma unroll
            for (int w = 0; w < FLY; ++w) {                                  // (strides are orthogonalize's alone)
                float mom;
                const int row = row0 + (first + w) * DOWN;
                if (row < it.m && col < it.n)
                    x[w][0] = element<T>(t, it, row, col, mom);
            }
        }
#pragma unroll
        for (int w = 0; w < FLY; ++w)
#pragma unroll
            for (int q = 0; q < N; ++q)
                to[(first + w) * DOWN * step_i + q * step_j] = split_word(scaled(x[w][q]));
    }
    __syncthreads();
}

// M / norm -> the first X, a tile of 64 x 64 a workgroup.  Bound by memory: 2 x 1024 x 4096 bf16, 17 MB in and 67 MB
// out, 16.9 us (5.0 TB/s).
template <typename T, bool DENSE> __global__ __launch_bounds__(256) void k_ns_pack(const NsTable *__restrict__ tp)
{
    const NsTable &t = *tp;
    __shared__ unsigned tile[PACK * (PACK + 1)];
    int index, local;
    const NsItem it = find_item(t, t.pack, blockIdx.x, index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    const int across = d.kp / PACK, i0 = local / across * PACK, j0 = local % across * PACK;
    first_tile<T, DENSE, PACK, 256>(t, it, d, item_scale(t, s, index), i0, j0, tile);
    const size_t plane = (size_t)d.rp * d.kp;
    put_rows<PACK, PACK, 256>(s.xk[0], plane, d.rp, i0, j0, tile);
    put_cols<PACK, PACK, 256>(s.xr[0], plane, d.kp, i0, j0, tile);
}

// ------------------------------------------------------------------------------------------- GEMM
// A square tile of side S = 32 F by 4 waves of F x F fragments of 16 x 16, three products each, k in steps of 32.  A
// step's operands, S rows of each side, are copied from L2 to LDS without passing registers (global_load_lds_dwordx4),
// into DEPTH buffers, DEPTH - 1 steps ahead.
//   F = 4 (128): per step and wave 48 MFMAs (768 clocks) stand against 16 KB read from LDS (about 300 clocks for all four
//     waves, at the 210 bytes a clock measured); two buffers, so that two workgroups share a compute unit and one
//     multiplies while the other waits: 820 clocks a step.
//   F = 2 (64): 192 against 150 clocks, but twice the copies a product and four times the workgroups: for launches whose
//     128-tiles would not give every compute unit one, where a step of those lasts 1550 clocks.  Up to two workgroups a
//     compute unit have four buffers and cover the copies' latency themselves, more of them two buffers, so that five
//     share a compute unit.  us with four / two: 272 tiles of 32 steps 19.7 / 21.1, 450 of 9 8.5 / 8.8, 720 of 8 14.4 / 13.0.
constexpr int STEP = 32;
template <int F> struct Tile {
    static constexpr int SIDE = 32 * F, LD = SIDE + 1;
    static constexpr int SIDE_BYTES = 2 * (STEP / 8) * SIDE * 16;        // [plane][k block][row] words of 16 bytes
    static constexpr int BUFFER = 2 * SIDE_BYTES, COPIES = STEP / 8 * F / 2;      // COPIES: of a wave and step
};
// the buffers, then the tile in 32 bits
template <int F, int DEPTH>
constexpr int TILE_LDS = DEPTH * Tile<F>::BUFFER > Tile<F>::SIDE * Tile<F>::LD * 4 ? DEPTH * Tile<F>::BUFFER
                                                                                   : Tile<F>::SIDE * Tile<F>::LD * 4;
constexpr int GEMM_THREADS = 256;

struct Side {
    const _Float16 *p;          // the operand's first row of the tile at the first k
    size_t plane;
    int rows;
};

__device__ __forceinline__ Side side_of(const _Float16 *op, size_t plane, int rows, int row0, int k0)
{
    return Side{op + ((size_t)(k0 / 8) * rows + row0) * 8, plane, rows};
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 words of 16 bytes, a lane each, from memory to LDS at byte `lds` on.  Inline assembly so that the compiler does
// not wait for the copy at every LDS read; gemm_wait does before the barrier.  The copy reads M0 one wait state after
// it was written at the earliest, which nothing but the s_nop sees to inside the assembly.
__device__ __forceinline__ void copy_words(const _Float16 *from, unsigned lds)
{
    const unsigned l = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "s"(l) : "memory", "m0");
}
#pragma clang diagnostic pop

// one plane of one side of one step into LDS at byte `lds`
template <int F> __device__ __forceinline__ void stage_plane(const Side &s, int plane, int step, unsigned lds)
{
    const int lane = threadIdx.x & 63;
    const _Float16 *src = s.p + (plane ? s.plane : 0) + ((size_t)step * (STEP / 8) * s.rows + lane) * 8;
    lds += plane * (Tile<F>::SIDE_BYTES / 2);
#pragma unroll
    for (int kb = 0; kb < STEP / 8; ++kb)
#pragma unroll
        for (int part = 0; part < F / 2; ++part)
            copy_words(src + ((size_t)kb * s.rows + part * 64) * 8, lds + (kb * Tile<F>::SIDE + part * 64) * 16);
}

// until at most LEFT of this wave's copies are under way (they end in order); in all waves
template <int LEFT = 0> __device__ __forceinline__ void gemm_wait()
{
    static_assert(LEFT == 0 || LEFT == 8, "the waits that occur");
    if (LEFT == 8)
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

__device__ __forceinline__ unsigned lds_address(const void *p)
{
    return (unsigned)(size_t)(__attribute__((address_space(3))) const char *)p;
}

// acc = U V' over `steps` steps; same: both sides are the same rows, copied once.  lds: the kernel's dynamic LDS,
// TILE_LDS bytes; free again at return.  acc[i][j]: rows 16 i + 4 (lane / 16) .., column 16 j + lane % 16 of the
// wave's quarter (wave / 2, wave % 2).
template <int F, int DEPTH>
__device__ __forceinline__ void tile_gemm(f32x4 (&acc)[F][F], char *lds, const Side &u, const Side &v, bool same, int steps)
{
    constexpr int SIDE_BYTES = Tile<F>::SIDE_BYTES, SIDE = Tile<F>::SIDE;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned base = lds_address(lds);
    auto stage = [&](int step, int buffer) {
        const unsigned to = base + buffer * Tile<F>::BUFFER;
        if (wave < 2)
            stage_plane<F>(u, wave, step, to);
        else if (!same)
            stage_plane<F>(v, wave - 2, step, to + SIDE_BYTES);
    };
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int word = (lane >> 4) * SIDE + (lane & 15);
    const char *us = lds + ((wave >> 1) * 16 * F + word) * 16;
    const char *vs = lds + (same ? 0 : SIDE_BYTES) + ((wave & 1) * 16 * F + word) * 16;
    constexpr int AHEAD = DEPTH - 1;
#pragma unroll
    for (int b = 0; b < AHEAD; ++b)
        if (b < steps)
            stage(b, b);
    for (int s = 0; s < steps; ++s) {
        // step s has arrived; and what step s - 1 was read from is free, after the barrier, for step s + AHEAD
        if (s + AHEAD <= steps)
            gemm_wait<(AHEAD - 1) * Tile<F>::COPIES>();
        else
            gemm_wait();
        const int now = s % DEPTH * Tile<F>::BUFFER;
        if (s + AHEAD < steps)
            stage(s + AHEAD, (s + AHEAD) % DEPTH);
        h8 uh[F], ul[F], vh[F], vl[F];
        auto load_u = [&](int i) {
            uh[i] = *reinterpret_cast<const h8 *>(us + now + i * 256);
            ul[i] = *reinterpret_cast<const h8 *>(us + now + SIDE_BYTES / 2 + i * 256);
        };
        load_u(0);
#pragma unroll
        for (int j = 0; j < F; ++j) {
            vh[j] = *reinterpret_cast<const h8 *>(vs + now + j * 256);
            vl[j] = *reinterpret_cast<const h8 *>(vs + now + SIDE_BYTES / 2 + j * 256);
        }
#pragma unroll
        for (int i = 1; i < F; ++i)
            load_u(i);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < F; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ul[i], vh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[i], vl[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[i], vh[j], acc[i][j], 0, 0, 0);
            }
    }
    __syncthreads();
}

// this lane's first value of the tile: acc[i][j][q] lies 16 i + q rows and 16 j columns from it
template <int F> __device__ __forceinline__ int lane_row() { return (threadIdx.x >> 7) * 16 * F + 4 * ((threadIdx.x & 63) >> 4); }

template <int F> __device__ __forceinline__ int lane_col() { return (threadIdx.x >> 6 & 1) * 16 * F + (threadIdx.x & 15); }

// the workgroup's tile as W = f(i, j, 4 accumulated values) of every fragment, 4 words of 32 bits, in LDS
template <typename W, int F, typename V>
__device__ __forceinline__ const W *tile_to_lds(const f32x4 (&acc)[F][F], char *lds, V &&f)
{
    W *mine = reinterpret_cast<W *>(lds) + lane_row<F>() * Tile<F>::LD + lane_col<F>();
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const f32x4 v = f(i, j, acc[i][j]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if constexpr (std::is_same<W, unsigned>::value)
                    mine[(16 * i + q) * Tile<F>::LD + 16 * j] = split_word(v[q]);
                else
                    mine[(16 * i + q) * Tile<F>::LD + 16 * j] = v[q];
            }
        }
    __syncthreads();
    return reinterpret_cast<const W *>(lds);
}

// A = X X', lower tiles, each over a share of k: the accumulators as they lie, 16 bytes a lane.  2 x 1024 x 4096: 32 us,
// 900 TFLOP/s of f16 products where a library product of 8192 reaches 1153; two workgroups a compute unit, the first and
// the last steps of each are what is lost.
template <int F, int DEPTH>
__global__ __launch_bounds__(GEMM_THREADS, 2) void k_ns_gram(const NsTable *__restrict__ tp, int step)
{
    const NsTable &t = *tp;
    constexpr int SIDE = Tile<F>::SIDE;
    extern __shared__ __align__(16) char lds[];
    int index, local, ti, tj;
    const NsItem it = find_item(t, t.gram, die_order(), index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    const int tiles = lower_tiles(d, SIDE), share = local / tiles, all = d.kp / STEP;
    lower_tile(local - share * tiles, ti, tj);
    const int s0 = (int)((long long)all * share / it.split), s1 = (int)((long long)all * (share + 1) / it.split);
    const _Float16 *x = step & 1 ? s.xk[1] : s.xk[0];
    const size_t plane = (size_t)d.rp * d.kp;
    f32x4 acc[F][F];
    tile_gemm<F, DEPTH>(acc, lds, side_of(x, plane, d.rp, ti * SIDE, s0 * STEP), side_of(x, plane, d.rp, tj * SIDE, s0 * STEP),
                 ti == tj, s1 - s0);
    f32x4 *out = reinterpret_cast<f32x4 *>(s.part + (size_t)local * SIDE * SIDE) + (threadIdx.x >> 6) * F * F * 64 + (threadIdx.x & 63);
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
            out[(i * F + j) * 64] = acc[i][j];
}

// The shares added in order, split, mirrored: a fragment on or below the diagonal a wave, 16 bytes of a share a lane,
// eight shares at once.  What lies above the diagonal is the mirror image of what lies below it, so A is symmetric to the
// bit at either side of the tiles, and a matrix gets the same bits whatever the launch holds besides it.  7 shares of
// 2 x 1024 x 1024 (31 MB in, 17 MB out) 8.2 us, 9 shares of 21 x 128 x 128 4.2 us; through LDS, 64 x 64 a workgroup, 9.9
// and 4.7, and far more for long matrices (128 x 16384 in all 178 -> 150 us).
constexpr int SUM_THREADS = 256;
__global__ __launch_bounds__(SUM_THREADS) void k_ns_sum(const NsTable *__restrict__ tp)
{
    const NsTable &t = *tp;
    int index, local, fi, fj;
    const NsItem it = find_item(t, t.sum, die_order(), index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int fragment = local * (SUM_THREADS / 64) + wave;
    if (fragment >= lower_tiles(d, 16))
        return;
    lower_tile(fragment, fi, fj);
    fi = __builtin_amdgcn_readfirstlane(fi);
    fj = __builtin_amdgcn_readfirstlane(fj);
    // the fragment's tile, and its place there: quarter by quarter, as the waves of k_ns_gram have them
    const int side = narrow(d) ? PAD : t.gram_side, f = side / 32, ti = fi / (2 * f), tj = fj / (2 * f);
    const int i = fi % (2 * f), j = fj % (2 * f), place = ((i / f) * 2 + j / f) * f * f + i % f * f + j % f;
    const size_t share = (size_t)lower_tiles(d, side) * side * side / 4;
    const f32x4 *in = reinterpret_cast<const f32x4 *>(s.part + (size_t)(ti * (ti + 1) / 2 + tj) * side * side) + place * 64 + lane;
    f32x4 v = in[0];
    for (int k = 1; k < it.split; k += 8) {
        f32x4 w[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            w[u] = in[min(k + u, it.split - 1) * share];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (k + u < it.split)
                v += w[u];
    }
    Quad x = split4(v * dance::pow2f(-X_EXP));
    const size_t plane = (size_t)d.rp * d.rp;
    const int row = 16 * fi + 4 * (lane >> 4), col = 16 * fj + (lane & 15);
    put4(s.a + ((size_t)(row >> 3) * d.rp + col) * 8 + (row & 7), plane, x);
    if (fi != fj) {
        transpose4(x);                                            // 4 columns of row row + lane % 4
        put4(s.a + ((size_t)(col >> 3) * d.rp + row + (lane & 3)) * 8 + (col & 4), plane, x);
    }
}

// Q = a I + b A + c A A, lower tiles and their mirror images.  2 x 1024 x 1024, 272 tiles of 64: 19 us, 0.45 us a step of
// 32 k; more buffers, fragments read a step ahead or products in another order did not change that, and 128-tiles would
// be 72 workgroups for 256 compute units.
template <int F, int DEPTH>
__global__ __launch_bounds__(GEMM_THREADS, 2) void k_ns_poly(const NsTable *__restrict__ tp)
{
    const NsTable &t = *tp;
    constexpr int SIDE = Tile<F>::SIDE;
    extern __shared__ __align__(16) char lds[];
    int index, local, ti, tj;
    const NsItem it = find_item(t, t.poly, die_order(), index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    lower_tile(local, ti, tj);
    const size_t plane = (size_t)d.rp * d.rp;
    const int i0 = ti * SIDE, j0 = tj * SIDE;
    // A's own values, for the end: a lane's 4 rows of a column are, A being symmetric, 4 neighbours of that column's row
    const int row = i0 + lane_row<F>(), col = j0 + lane_col<F>();
    const _Float16 *p = s.a + ((size_t)(row / 8) * d.rp + col) * 8 + (row & 7);
    h4 hi[F][F], lo[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const _Float16 *pij = p + ((size_t)(2 * i) * d.rp + 16 * j) * 8;
            hi[i][j] = *reinterpret_cast<const h4 *>(pij);
            lo[i][j] = *reinterpret_cast<const h4 *>(pij + plane);
        }
    f32x4 acc[F][F];
    tile_gemm<F, DEPTH>(acc, lds, side_of(s.a, plane, d.rp, i0, 0), side_of(s.a, plane, d.rp, j0, 0), ti == tj, d.rp / STEP);
    const float ca = t.c * dance::pow2f(-2 * X_EXP) * t.q_mul, ba = t.b * dance::pow2f(-X_EXP) * t.q_mul, a = t.a * t.q_mul;
    const unsigned *tile = tile_to_lds<unsigned>(acc, lds, [&](int i, int j, f32x4 v) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
            v[q] = poly_of(ca, v[q], ba, hi[i][j][q], lo[i][j][q]);
        if (ti == tj && i == j) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[q] += row + 16 * i + q == col + 16 * j && col + 16 * j < d.r ? a : 0.0f;
        }
        return v;
    });
    if (F == 4 && ti == tj) {
        // the quarter above the diagonal from the one below it, as tiles of 64 have it
        unsigned *w = reinterpret_cast<unsigned *>(lds);
#pragma unroll 4
        for (int e = threadIdx.x; e < 64 * 64; e += GEMM_THREADS)
            w[(e & 63) * Tile<F>::LD + 64 + (e >> 6)] = w[(64 + (e >> 6)) * Tile<F>::LD + (e & 63)];
        __syncthreads();
    }
    put_rows<SIDE, SIDE, GEMM_THREADS>(s.q, plane, d.rp, i0, j0, tile);
    if (ti != tj)
        put_cols<SIDE, SIDE, GEMM_THREADS>(s.q, plane, d.rp, i0, j0, tile);
}

// a tile of the result, rows i and columns j of X from (i0, j0) on; Muon: the parameter's update
template <typename T, int SIDE, int THREADS>
__device__ __forceinline__ void put_result(const NsTable &t, const NsItem &it, const NsDims &d, int i0, int j0, const float *tile)
{
    const int row0 = d.tall ? j0 : i0, col = (d.tall ? i0 : j0) + (int)threadIdx.x % SIDE;
    const int step_row = d.tall ? 1 : (SIDE + 1);
    const float *from = tile + threadIdx.x % SIDE * (d.tall ? (SIDE + 1) : 1);
    if (col >= it.n)
        return;
#pragma unroll 1
    for (int r = threadIdx.x / SIDE; r < SIDE && row0 + r < it.m; r += 8 * (THREADS / SIDE)) {
        T *to = (T *)it.dst + (long long)(row0 + r) * it.n + col;
        T old[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int rr = r + u * (THREADS / SIDE);
            if (t.muon && row0 + rr < it.m)
                old[u] = to[(long long)u * (THREADS / SIDE) * it.n];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int rr = r + u * (THREADS / SIDE);
            const float v = from[rr * step_row];
            if (row0 + rr < it.m)
                to[(long long)u * (THREADS / SIDE) * it.n] = (T)(t.muon ? fmaf(-it.scale, v, (float)old[u] * t.keep) : v);
        }
    }
}

// X <- Q X; the last step writes the result.  2 x 1024 x 4096: 52 us, 983 TFLOP/s of f16 products: bound by the matrix
// cores.
template <int F, int DEPTH>
__global__ __launch_bounds__(GEMM_THREADS, 2) void k_ns_apply(const NsTable *__restrict__ tp, int step, int last)
{
    const NsTable &t = *tp;
    constexpr int SIDE = Tile<F>::SIDE;
    extern __shared__ __align__(16) char lds[];
    int index, local;
    const NsItem it = find_item(t, t.rect, die_order(), index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    const int down = d.rp / SIDE, i0 = local % down * SIDE, j0 = local / down * SIDE;
    const size_t square = (size_t)d.rp * d.rp, rect = (size_t)d.rp * d.kp;
    f32x4 acc[F][F];
    tile_gemm<F, DEPTH>(acc, lds, side_of(s.q, square, d.rp, i0, 0), side_of(step & 1 ? s.xr[1] : s.xr[0], rect, d.kp, j0, 0), false,
              d.rp / STEP);
    const float mul = 1.0f / t.q_mul;
    if (!last) {
        const unsigned *tile = tile_to_lds<unsigned>(acc, lds, [&](int, int, f32x4 v) { return v * mul; });
        put_rows<SIDE, SIDE, GEMM_THREADS>(step & 1 ? s.xk[0] : s.xk[1], rect, d.rp, i0, j0, tile);
        put_cols<SIDE, SIDE, GEMM_THREADS>(step & 1 ? s.xr[0] : s.xr[1], rect, d.kp, i0, j0, tile);
        return;
    }
    const float out = mul * dance::pow2f(-X_EXP);
    const float *tile = tile_to_lds<float>(acc, lds, [&](int, int, f32x4 v) { return v * out; });
    // neighbouring threads write neighbours of a row of M
    if (t.dtype == DANCE_F32)
        put_result<float, SIDE, GEMM_THREADS>(t, it, d, i0, j0, tile);
    else if (t.dtype == DANCE_F16)
        put_result<_Float16, SIDE, GEMM_THREADS>(t, it, d, i0, j0, tile);
    else
        put_result<__bf16, SIDE, GEMM_THREADS>(t, it, d, i0, j0, tile);
}

// ------------------------------------------------------------------------------ narrow matrices
// Up to 128 rows: a step is a launch of its own and one that adds the shares of A (k_ns_sum).  A workgroup owns columns of
// X, a tile of 128 at a time.  It takes A, computes Q (in every workgroup: cheaper than a launch), replaces its columns
// by Q X and sums their own share of the next A.  A, then Q, and the columns lie in LDS, 64 KB each; 8 waves, of 64 x 32
// in Q X.  21 x 128 x 1152, 189 workgroups: 14.2 us a step.  Of a workgroup's 20 thousand clocks 6.5 are the matrix
// instructions' own; copies in, three epilogues and the way out wait for each other, a second workgroup has no room.
constexpr int NARROW_THREADS = 512;
constexpr int REGION = 2 * (PAD / 8) * PAD * 16;             // [plane][k block][row] words of 16 bytes
constexpr int NARROW_LDS = 2 * REGION;

__device__ __forceinline__ void narrow_gemm(f32x4 (&acc)[4][2], const char *u, const char *v)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const char *us = u + ((lane >> 4) * PAD + (wave >> 2) * 64 + (lane & 15)) * 16;
    const char *vs = v + ((lane >> 4) * PAD + (wave & 3) * 32 + (lane & 15)) * 16;
#pragma unroll 1
    for (int s = 0; s < PAD / 32; ++s) {
        h8 uh[4], ul[4], vh[2], vl[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            vh[j] = *reinterpret_cast<const h8 *>(vs + j * 256);
            vl[j] = *reinterpret_cast<const h8 *>(vs + REGION / 2 + j * 256);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uh[i] = *reinterpret_cast<const h8 *>(us + i * 256);
            ul[i] = *reinterpret_cast<const h8 *>(us + REGION / 2 + i * 256);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ul[i], vh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[i], vl[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[i], vh[j], acc[i][j], 0, 0, 0);
            }
        us += 4 * PAD * 16;
        vs += 4 * PAD * 16;
    }
}

// f(i, j, row, col) for this lane's fragments: rows row .. row + 3 of column col
template <typename F> __device__ __forceinline__ void narrow_each(F &&f)
{
    const int row = (threadIdx.x >> 8) * 64 + 4 * ((threadIdx.x & 63) >> 4), col = (threadIdx.x >> 6 & 3) * 32 + (threadIdx.x & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            f(i, j, row + 16 * i, col + 16 * j);
}

__device__ __forceinline__ void zero(f32x4 (&acc)[4][2])
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// Symmetric products U U' of 128 rows: the 36 fragments on and below the diagonal, over 8 waves.  The quarter below the
// diagonal is four waves' (BLOCK, 2 x 2 fragments each), a quarter on the diagonal two waves': (3, 0) (3, 1) (3, 2)
// (3, 3) (0, 0) of its own rows (LAST_ROW) and (1, 0) (1, 1) (2, 0) (2, 1) (2, 2) (MIDDLE).  A fragment's rows are the
// same words as a left and as a right operand, so a wave reads four rows of fragments at most.  Each SIMD has a wave of
// four and one of five fragments: 1728 clocks of MFMAs where all 64 take 3072.
enum Triangle { BLOCK, LAST_ROW, MIDDLE };

struct Triangular {
    int kind, row[4];           // rows of fragments, in units of 16
};

__device__ __forceinline__ Triangular triangular()
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wave & 2;
    if (wave < 4)
        return {BLOCK, {4 + half, 5 + half, (wave & 1) * 2, (wave & 1) * 2 + 1}};
    const int q = half * 2;
    return {wave & 1 ? MIDDLE : LAST_ROW, {q, q + 1, q + 2, q + 3}};
}

// f(s, i, j) for the wave's fragments: s their place in a wave's five, (i, j) two of its four rows
template <int KIND, typename F> __device__ __forceinline__ void triangular_of(F &&f)
{
    if (KIND == BLOCK) {
        f(0, 0, 2);
        f(1, 0, 3);
        f(2, 1, 2);
        f(3, 1, 3);
    } else if (KIND == LAST_ROW) {
        f(0, 3, 0);
        f(1, 3, 1);
        f(2, 3, 2);
        f(3, 3, 3);
        f(4, 0, 0);
    } else {
        f(0, 1, 0);
        f(1, 1, 1);
        f(2, 2, 0);
        f(3, 2, 1);
        f(4, 2, 2);
    }
}

template <typename F> __device__ __forceinline__ void with_kind(const Triangular &t, F &&f)
{
    if (t.kind == BLOCK)
        f(std::integral_constant<int, BLOCK>{});
    else if (t.kind == LAST_ROW)
        f(std::integral_constant<int, LAST_ROW>{});
    else
        f(std::integral_constant<int, MIDDLE>{});
}

// acc += the wave's fragments of U U', 128 k
template <int KIND> __device__ __forceinline__ void triangular_gemm(f32x4 (&acc)[5], const Triangular &t, const char *u)
{
    const int lane = threadIdx.x & 63;
    const char *at = u + ((lane >> 4) * PAD + (lane & 15)) * 16;
#pragma unroll 1
    for (int s = 0; s < PAD / 32; ++s) {
        h8 h[4], l[4];
#pragma unroll
        for (int i = 0; i < (KIND == MIDDLE ? 3 : 4); ++i) {
            h[i] = *reinterpret_cast<const h8 *>(at + t.row[i] * 256);
            l[i] = *reinterpret_cast<const h8 *>(at + t.row[i] * 256 + REGION / 2);
        }
        triangular_of<KIND>([&](int f, int i, int j) { acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(l[i], h[j], acc[f], 0, 0, 0); });
        triangular_of<KIND>([&](int f, int i, int j) { acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[i], l[j], acc[f], 0, 0, 0); });
        triangular_of<KIND>([&](int f, int i, int j) { acc[f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(h[i], h[j], acc[f], 0, 0, 0); });
        at += 4 * PAD * 16;
    }
}

__device__ __forceinline__ void triangular_gemm(f32x4 (&acc)[5], const Triangular &t, const char *u)
{
    with_kind(t, [&](auto kind) { triangular_gemm<decltype(kind)::value>(acc, t, u); });
}

// a symmetric matrix into a region: each value at its mirror image, where a lane's 4 are neighbours, and in its place
template <int KIND> __device__ __forceinline__ void put_triangular(char *region, const Triangular &t, const f32x4 (&m)[5])
{
    const int row = 4 * ((threadIdx.x & 63) >> 4), col = threadIdx.x & 15;
    triangular_of<KIND>([&](int f, int i, int j) {
        const int i0 = 16 * t.row[i], j0 = 16 * t.row[j];
        Quad x = split4(m[f]);
        put4((_Float16 *)region + (((i0 + row) >> 3) * PAD + j0 + col) * 8 + (row & 7), REGION / 4, x);
        if (KIND == BLOCK || i != j) {
            transpose4(x);                                    // 4 columns of row row + lane % 4
            put4((_Float16 *)region + (((j0 + col) >> 3) * PAD + i0 + row + (threadIdx.x & 3)) * 8 + (col & 4), REGION / 4, x);
        }
    });
}

// an operand's 128 rows and 128 k into a region, 8 pieces a wave
__device__ __forceinline__ void narrow_stage(const _Float16 *p, size_t plane, int rows, const char *region)
{
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned to = lds_address(region) + wave * 4 * PAD * 16;
    const _Float16 *src = p + (wave >> 2) * plane + ((size_t)(wave & 3) * 4 * rows + lane) * 8;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        copy_words(src + ((size_t)(c >> 1) * rows + (c & 1) * 64) * 8, to + ((c >> 1) * PAD + (c & 1) * 64) * 16);
}

// a share of A, where k_ns_sum looks for it: quarter by quarter of the tile, 4 x 4 fragments each
__device__ __forceinline__ void put_share(float *part, const Triangular &t, const f32x4 (&v)[5])
{
    f32x4 *out = reinterpret_cast<f32x4 *>(part) + (threadIdx.x & 63);
    with_kind(t, [&](auto kind) {
        triangular_of<decltype(kind)::value>([&](int f, int i, int j) {
            const int fi = t.row[i], fj = t.row[j];
            out[(((fi >> 2) * 2 + (fj >> 2)) * 16 + (fi & 3) * 4 + (fj & 3)) * 64] = v[f];
        });
    });
}

__device__ __forceinline__ void zero(f32x4 (&acc)[5])
{
#pragma unroll
    for (int f = 0; f < 5; ++f)
        acc[f] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// M / norm -> the first X and the shares of its A: 12.7 us for 21 x 128 x 1152, where a launch that lays X out both ways
// and one that takes A were 10.5 + 7.4
constexpr int FIRST_TILE = PAD * (PAD + 1) * 4, FIRST_LDS = FIRST_TILE + REGION;
template <typename T, bool DENSE> __global__ __launch_bounds__(NARROW_THREADS) void k_ns_narrow_first(const NsTable *__restrict__ tp)
{
    const NsTable &t = *tp;
    extern __shared__ __align__(16) char lds[];
    unsigned *tile = reinterpret_cast<unsigned *>(lds);
    char *columns = lds + FIRST_TILE;
    int index, local;
    const NsItem it = find_item(t, t.narrow, die_order(), index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    const Scale scaled = item_scale(t, s, index);
    const Triangular mine = triangular();
    f32x4 next[5];
    zero(next);
#pragma unroll 1
    for (int c = local; c < d.kp / PAD; c += it.split) {
        first_tile<T, DENSE, PAD, NARROW_THREADS>(t, it, d, scaled, 0, c * PAD, tile);
        put_rows<PAD, PAD, NARROW_THREADS>((_Float16 *)columns, REGION / 4, PAD, 0, 0, tile);
        put_cols<PAD, PAD, NARROW_THREADS>(s.xr[0], (size_t)PAD * d.kp, d.kp, 0, c * PAD, tile);
        __syncthreads();
        triangular_gemm(next, mine, columns);
    }
    put_share(s.part + (size_t)local * PAD * PAD, mine, next);
}

// A step; the last one writes the result, and no A
template <typename T> __global__ __launch_bounds__(NARROW_THREADS) void k_ns_narrow(const NsTable *__restrict__ tp, int last)
{
    const NsTable &t = *tp;
    extern __shared__ __align__(16) char lds[];
    char *square = lds, *columns = lds + REGION;
    int index, local;
    const NsItem it = find_item(t, t.narrow, die_order(), index, local);
    const NsDims d = ns_dims(it.m, it.n);
    NsSpace s;
    ns_space(it.ws, d, it.split, s);
    const size_t rect = (size_t)PAD * d.kp, share = PAD * PAD;
    const int tiles = d.kp / PAD;
    const Triangular mine = triangular();
    f32x4 next[5], q[5], v[4][2];
    zero(next);
    zero(q);
    narrow_stage(s.a, share, PAD, square);
    narrow_stage(s.xr[0] + (size_t)local * PAD * 8, rect, d.kp, columns);
    gemm_wait<8>();                                       // A; the columns are on their way
    triangular_gemm(q, mine, square);
    const float ca = t.c * dance::pow2f(-2 * X_EXP) * t.q_mul, ba = t.b * dance::pow2f(-X_EXP) * t.q_mul, one = t.a * t.q_mul;
    with_kind(mine, [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        const int row = 4 * ((threadIdx.x & 63) >> 4), col = threadIdx.x & 15;
        triangular_of<KIND>([&](int f, int i, int j) {
            const int i0 = 16 * mine.row[i], j0 = 16 * mine.row[j];
            // A is symmetric: 4 rows of a column are 4 neighbours of that column's row
            const _Float16 *p = (const _Float16 *)square + (((i0 + row) >> 3) * PAD + j0 + col) * 8 + (row & 7);
            const h4 hi = *reinterpret_cast<const h4 *>(p), lo = *reinterpret_cast<const h4 *>(p + REGION / 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                q[f][e] = poly_of(ca, q[f][e], ba, hi[e], lo[e]);
                if (KIND != BLOCK && i == j)
                    q[f][e] += row + e == col && j0 + col < d.r ? one : 0.0f;
            }
        });
    });
    const float mul = 1.0f / t.q_mul;
#pragma unroll 1
    for (int c = local; c < tiles; c += it.split) {
        gemm_wait();                                      // A, and the columns before, have been read; the first are here
        if (c == local || last)
            with_kind(mine, [&](auto kind) { put_triangular<decltype(kind)::value>(square, mine, q); });
        __syncthreads();
        if (c != local) {
            narrow_stage(s.xr[0] + (size_t)c * PAD * 8, rect, d.kp, columns);
            gemm_wait();
        }
        zero(v);
        narrow_gemm(v, square, columns);
        __syncthreads();
        if (!last) {
            // in place, and with k along the columns for the share of A
            _Float16 *to = s.xr[0] + (size_t)c * PAD * 8;
            narrow_each([&](int i, int j, int row, int col) {
                Quad x = split4(v[i][j] * mul);
                put4(to + ((size_t)(row >> 3) * d.kp + col) * 8 + (row & 7), rect, x);
                transpose4(x);                            // 4 columns of row row + lane % 4
                put4((_Float16 *)columns + ((col >> 3) * PAD + row + (threadIdx.x & 3)) * 8 + (col & 4), REGION / 4, x);
            });
            __syncthreads();
            triangular_gemm(next, mine, columns);
        } else {
            // the tile in fp32 over both regions; Q is needed again if there are more columns
            float *tile = reinterpret_cast<float *>(lds);
            narrow_each([&](int i, int j, int row, int col) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    tile[(row + q) * (PAD + 1) + col] = v[i][j][q] * (mul * dance::pow2f(-X_EXP));
            });
            __syncthreads();
            put_result<T, PAD, NARROW_THREADS>(t, it, d, 0, c * PAD, tile);
        }
    }
    if (!last)
        put_share(s.part + local * share, mine, next);
}

// ------------------------------------------------------------------------------- small matrices
// The whole chain of a matrix in one workgroup, X, A and Q in LDS: [plane][k / 8][row][8] as above, padded to 32.
// 16 waves; a fragment of 16 x 16 of a product is one wave's.  64 x 256, 5 steps: 24 us, 11 thousand clocks until the
// first X stands and 8.5 a step: X X' 2.4, Q 1.6 and Q X 4.5, whose epilogue (split, transposed, written both ways) is
// bound by vector instructions.
constexpr int SMALL_THREADS = 1024, SMALL_WAVES = SMALL_THREADS / 64, SMALL_PAD = 32;
constexpr size_t SMALL_LDS = 160 * 1024;
constexpr size_t SMALL_MOST = SMALL_LDS - 1024;
static_assert(12 * 128 * 128 > SMALL_MOST, "12 rp^2 bytes at least: rp <= 96");

struct SmallDims {
    int r, k, rp, kp, tall;
    size_t bytes;
};

__host__ __device__ inline SmallDims small_dims(int m, int n)
{
    SmallDims d;
    d.tall = m > n;
    d.r = d.tall ? n : m;
    d.k = d.tall ? m : n;
    d.rp = (d.r + SMALL_PAD - 1) / SMALL_PAD * SMALL_PAD;
    d.kp = (d.k + SMALL_PAD - 1) / SMALL_PAD * SMALL_PAD;
    d.bytes = 8 * (size_t)d.rp * d.kp + 4 * (size_t)d.rp * d.rp;        // X both ways; A, which Q replaces
    return d;
}

// A fragment of U V': this lane's first words of U and V, `rows` words from one block of 8 k to the next, planes `plane`
// halves apart, over `steps` steps of 32 k.  A step's words are read while the one before is multiplied, into the other
// of two sets of registers (the compiler does not unroll the loop, matrix instructions are convergent).
__device__ __forceinline__ f32x4 small_gemm(const _Float16 *u, const _Float16 *v, int rows, int plane, int steps)
{
    // three sums, so that a product does not wait for the one before it
    f32x4 hh = {0.0f, 0.0f, 0.0f, 0.0f}, hl = hh, lh = hh;
    h8 uh[2], ul[2], vh[2], vl[2];
    auto load = [&](int set, int step) {
        const _Float16 *us = u + step * 32 * rows, *vs = v + step * 32 * rows;
        uh[set] = *reinterpret_cast<const h8 *>(us);
        ul[set] = *reinterpret_cast<const h8 *>(us + plane);
        vh[set] = *reinterpret_cast<const h8 *>(vs);
        vl[set] = *reinterpret_cast<const h8 *>(vs + plane);
    };
    auto multiply = [&](int set) {
        lh = __builtin_amdgcn_mfma_f32_16x16x32_f16(ul[set], vh[set], lh, 0, 0, 0);
        hl = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[set], vl[set], hl, 0, 0, 0);
        hh = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[set], vh[set], hh, 0, 0, 0);
    };
    load(0, 0);
#pragma unroll 1
    for (int s = 1; s < steps; s += 2) {
        load(1, s);
        multiply(0);
        load(0, min(s + 1, steps - 1));
        multiply(1);
    }
    if (steps & 1)
        multiply(0);
    return hh + (hl + lh);
}

// a / b of small numbers (a < 2^20) by the reciprocal 1 / b: a + 1/2 is at least 1/2 from a multiple of b, the error of
// the product at most 2^-23 (a + 1/2) / b
__device__ __forceinline__ int small_div(int a, float reciprocal) { return (int)(((float)a + 0.5f) * reciprocal); }

struct SmallSettings {
    float ca, ba, one, mul;
    int steps;
};

// The unscaled M in LDS as fp32 [i][j], behind xk -> the result, for rp = 32 R
template <int R, typename T>
__device__ __forceinline__ void small_steps(const NsTable &t, const NsItem &it, const SmallDims &d, const SmallSettings &c,
                                            Scale scaled, _Float16 *xk)
{
    constexpr int RP = 32 * R, FR = 2 * R, LOWER = FR * (FR + 1) / 2, MINE = (LOWER + SMALL_WAVES - 1) / SMALL_WAVES, SQUARE = RP * RP;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int rect = RP * d.kp, ld = d.kp + 1;
    _Float16 *xr = xk + 2 * rect, *a = xr + 2 * rect;
    const float *tile = reinterpret_cast<const float *>(xr);
    // X both ways.  The words that replace the tile wait in registers until everybody has read it.
    constexpr int HELD = (int)(SMALL_MOST / 64 / SMALL_THREADS) + 1;
    Quad held[HELD][2];
    const float per_k = 1.0f / (float)d.kp;
#pragma unroll
    for (int n = 0; n < HELD; ++n) {
        const int w = threadIdx.x + n * SMALL_THREADS, ib = small_div(w, per_k), j = w - ib * d.kp;
        if (w < rect / 8) {
            const float *from = tile + ib * 8 * ld + j;
#pragma unroll
            for (int h = 0; h < 2; ++h, from += 4 * ld)
                held[n][h] = split4(f32x4{scaled(from[0]), scaled(from[ld]), scaled(from[2 * ld]), scaled(from[3 * ld])});
        }
    }
#pragma unroll 1
    for (int w = threadIdx.x; w < rect / 8; w += SMALL_THREADS) {
        const float *from = tile + w % RP * ld + w / RP * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h, from += 4)
            put4(xk + w * 8 + 4 * h, rect, split4(f32x4{scaled(from[0]), scaled(from[1]), scaled(from[2]), scaled(from[3])}));
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < HELD; ++n) {
        const int w = threadIdx.x + n * SMALL_THREADS;
        if (w < rect / 8)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                put4(xr + w * 8 + 4 * h, rect, held[n][h]);
    }
    __syncthreads();

    const int i4 = 4 * (lane >> 4), j1 = lane & 15;               // a lane's rows and column in a fragment
    const int word = ((lane >> 4) * RP + j1) * 8;                 // its first word of a side, at row 0
    int i0[MINE], j0[MINE];                                       // the wave's fragments on and below the diagonal
#pragma unroll
    for (int n = 0; n < MINE; ++n) {
        lower_tile(wave + n * SMALL_WAVES, i0[n], j0[n]);
        i0[n] = __builtin_amdgcn_readfirstlane(i0[n]) * 16;
        j0[n] = __builtin_amdgcn_readfirstlane(j0[n]) * 16;
    }
    // a fragment of a symmetric matrix: its mirror image, where a lane's 4 values are neighbours, and itself
    auto put_square = [&](const f32x4 &v, int i0, int j0) {
        Quad x = split4(v);
        put4(a + (((i0 + i4) >> 3) * RP + j0 + j1) * 8 + (i4 & 7), SQUARE, x);
        if (i0 != j0) {
            transpose4(x);                                        // 4 columns of row i + lane % 4
            put4(a + (((j0 + j1) >> 3) * RP + i0 + i4 + (lane & 3)) * 8 + (j1 & 4), SQUARE, x);
        }
    };
#pragma unroll 1
    for (int step = 1;; ++step) {
#pragma unroll
        for (int n = 0; n < MINE; ++n)
            if (wave + n * SMALL_WAVES < LOWER)
                put_square(small_gemm(xk + word + i0[n] * 8, xk + word + j0[n] * 8, RP, rect, d.kp / 32) * dance::pow2f(-X_EXP), i0[n],
                           j0[n]);
        __syncthreads();
        f32x4 q[MINE];
#pragma unroll
        for (int n = 0; n < MINE; ++n) {
            if (wave + n * SMALL_WAVES >= LOWER)
                continue;
            q[n] = small_gemm(a + word + i0[n] * 8, a + word + j0[n] * 8, RP, SQUARE, R);
            const _Float16 *p = a + (((i0[n] + i4) >> 3) * RP + j0[n] + j1) * 8 + (i4 & 7);
            const h4 ah = *reinterpret_cast<const h4 *>(p), al = *reinterpret_cast<const h4 *>(p + SQUARE);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                q[n][e] = poly_of(c.ca, q[n][e], c.ba, ah[e], al[e]);
            if (i0[n] == j0[n]) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    q[n][e] += i4 + e == j1 && j0[n] + j1 < d.r ? c.one : 0.0f;
            }
        }
        __syncthreads();                                          // every wave has read A: Q takes its place
#pragma unroll
        for (int n = 0; n < MINE; ++n)
            if (wave + n * SMALL_WAVES < LOWER)
                put_square(q[n], i0[n], j0[n]);
        __syncthreads();
        // X <- Q X: a wave owns 16 columns of X at a time, holds them in registers and replaces them
        const bool last = step == c.steps;
#pragma unroll 1
        for (int f = wave; f < d.kp / 16; f += SMALL_WAVES) {
            const int j = f * 16 + j1;
            h8 vh[R], vl[R];
#pragma unroll
            for (int n = 0; n < R; ++n) {
                const _Float16 *p = xr + ((n * 4 + (lane >> 4)) * d.kp + j) * 8;
                vh[n] = *reinterpret_cast<const h8 *>(p);
                vl[n] = *reinterpret_cast<const h8 *>(p + rect);
            }
            // Q's rows of a fragment are read while the one before is multiplied and written
            h8 uh[2][R], ul[2][R];
            auto load = [&](int set, int i) {
#pragma unroll
                for (int n = 0; n < R; ++n) {
                    const _Float16 *p = a + word + (n * 4 * RP + i) * 8;
                    uh[set][n] = *reinterpret_cast<const h8 *>(p);
                    ul[set][n] = *reinterpret_cast<const h8 *>(p + SQUARE);
                }
            };
            auto fragment = [&](int set) {
                f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < R; ++n) {
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(ul[set][n], vh[n], x, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[set][n], vl[n], x, 0, 0, 0);
                }
#pragma unroll
                for (int n = 0; n < R; ++n)
                    x = __builtin_amdgcn_mfma_f32_16x16x32_f16(uh[set][n], vh[n], x, 0, 0, 0);
                return x * c.mul;
            };
            load(0, 0);
            if (!last) {
                _Float16 *to_r = xr + ((i4 >> 3) * d.kp + j) * 8 + (i4 & 7);
                _Float16 *to_k = xk + ((j >> 3) * RP + i4 + (lane & 3)) * 8 + (j & 4);
#pragma unroll
                for (int i = 0; i < FR; ++i) {
                    if (i + 1 < FR)
                        load((i + 1) & 1, 16 * (i + 1));
                    Quad x = split4(fragment(i & 1));
                    put4(to_r + 16 * i * d.kp, rect, x);
                    transpose4(x);
                    put4(to_k + 16 * i * 8, rect, x);
                }
            } else {
                const int step_i = d.tall ? 1 : it.n;
                const float out = dance::pow2f(-X_EXP);
#pragma unroll 1
                for (int i0 = 0; i0 < RP; i0 += 16) {
                    const int i = i0 + i4;
                    T *to = (T *)it.dst + (d.tall ? j * it.n + i : i * it.n + j);
                    float old[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        old[e] = t.muon && i + e < d.r && j < d.k ? (float)to[e * step_i] : 0.0f;
                    load(0, i0);
                    const f32x4 x = fragment(0) * out;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (i + e < d.r && j < d.k)
                            to[e * step_i] = (T)(t.muon ? fmaf(-it.scale, x[e], old[e] * t.keep) : x[e]);
                }
            }
        }
        if (last)
            return;
        __syncthreads();
    }
}

template <typename T, bool DENSE> __global__ __launch_bounds__(SMALL_THREADS) void k_ns_small(NsTable t)
{
    constexpr int N = 16 / sizeof(T), WORDS = (int)(SMALL_MOST / 8 / N / SMALL_THREADS) + 1;      // vectors of M a thread
    extern __shared__ __align__(16) char lds[];
    __shared__ double red[SMALL_WAVES];
    const NsItem it = t.it[blockIdx.x];
    const SmallDims d = small_dims(it.m, it.n);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int rect = d.rp * d.kp;
    const SmallSettings c = {t.c * dance::pow2f(-2 * X_EXP) * t.q_mul, t.b * dance::pow2f(-X_EXP) * t.q_mul, t.a * t.q_mul,
                             1.0f / t.q_mul, t.steps};
    // (here and not where they are used, each a trip to the kernel's arguments in host memory)
    asm volatile("" : : "v"(c.ca), "v"(c.ba), "v"(c.one), "v"(c.mul), "s"(c.steps));

    // M (Muon: the update) once from memory, its norm on the way, then unscaled into LDS, as fp32 [i][j] where X with k
    // along its rows and A will be
    float *tile = reinterpret_cast<float *>(lds) + rect;
    const int ld = d.kp + 1;                        // odd; rp (kp + 1) floats are inside xr and A
    const int total = it.m * it.n, step_col = d.tall ? ld : 1, step_row = d.tall ? 1 : ld;
    const float per_row = 1.0f / (float)it.n;
    double acc = 0.0;
    auto padding = [&] {                            // while the first loads are under way
        if (d.r < d.rp || d.k < d.kp) {
#pragma unroll 1
            for (int e = threadIdx.x; e < d.rp * ld; e += SMALL_THREADS)
                tile[e] = 0.0f;
            __syncthreads();
        }
    };
    const int vectors = DENSE ? total / N : 0;
    if (DENSE) {
        Word<T> g[WORDS], m[WORDS];
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {           // every load is issued before the first is waited for
            const int v = threadIdx.x + w * SMALL_THREADS;
            if (v < vectors)
                load_words<T>(t, it, (long long)v * N, g[w], m[w]);
        }
        padding();
#pragma unroll
        for (int w = 0; w < WORDS; ++w) {
            const int v = threadIdx.x + w * SMALL_THREADS;
            if (v < vectors) {
                float x[N];
                elements<T>(t, g[w], m[w], x);
                const int row = small_div(v * N, per_row);
                int col = v * N - row * it.n;
                float *to = tile + row * step_row + col * step_col;
#pragma unroll
                for (int q = 0; q < N; ++q) {
                    acc = fma((double)x[q], (double)x[q], acc);
                    *to = x[q];
                    const bool end = ++col == it.n;
                    to += end ? step_row - (it.n - 1) * step_col : step_col;
                    col = end ? 0 : col;
                }
                if (t.muon)
                    reinterpret_cast<Word<T> *>(it.momentum)[v] = m[w];
            }
        }
    } else
        padding();
#pragma unroll 1
    for (int e = vectors * N + threadIdx.x; e < total; e += SMALL_THREADS) {
        float mom;
        const int row = small_div(e, per_row), col = e - row * it.n;
        const float x = element<T>(t, it, row, col, mom);
        if (t.muon)
            ((T *)it.momentum)[e] = (T)mom;
        acc = fma((double)x, (double)x, acc);
        tile[row * step_row + col * step_col] = x;
    }
    acc = wave_sum(acc);
    if (lane == 0)
        red[wave] = acc;
    __syncthreads();
    double sum = red[0];
#pragma unroll
    for (int w = 1; w < SMALL_WAVES; ++w)
        sum += red[w];
    const Scale scaled = scale_of(sum, t.eps);
    if (d.rp == 32)
        small_steps<1, T>(t, it, d, c, scaled, (_Float16 *)lds);
    else if (d.rp == 64)
        small_steps<2, T>(t, it, d, c, scaled, (_Float16 *)lds);
    else
        small_steps<3, T>(t, it, d, c, scaled, (_Float16 *)lds);
}

// ------------------------------------------------------------------------------------------- host
bool known_dtype(int t) { return t == DANCE_F32 || t == DANCE_F16 || t == DANCE_BF16; }

bool is_small(int m, int n) { return small_dims(m, n).bytes <= SMALL_MOST; }

// Workgroups along k that a tile of A is shared by: about 256 a matrix, each with 8 steps of the GEMM at least; more
// shares are more partial sums to add.  By the matrix alone, so that one of a batch gives the bits it gives alone.
int split_of(const NsDims &d)
{
    if (narrow(d)) {
        // of the T column tiles: a share is about 350 clocks to add, a tile 32 times that.  128 x 65536 with two tiles a
        // workgroup 284 us, with four 268; 8 x 128 x 16384 with two 311, with one 376
        const int tiles = d.kp / PAD, each = (int)sqrt(tiles / 32.0);
        return each <= 1 ? tiles : (tiles + each - 1) / each;
    }
    const int want = 256 / lower_tiles(d, PAD), most = d.kp / STEP / 8, split = want < most ? want : most;
    return split < 1 ? 1 : split > 32 ? 32 : split;
}

// the tiles' side for a launch of `tiles` tiles of 128: those where every compute unit gets one of them
int side_for(long long tiles) { return tiles >= 256 ? 128 : 64; }

// Lays out the items' shares of the workspace -> its size.  t.it[].m, n set; ws may be NULL.
int64_t lay_out(NsTable &t, char *ws)
{
    bool small = true;
    for (int i = 0; i < t.count; ++i)
        small = small && is_small(t.it[i].m, t.it[i].n);
    if (small)
        return 0;
    int64_t at = (sizeof(NsTable) + 15) & ~(size_t)15;       // the table itself comes first
    for (int i = 0; i < t.count; ++i) {
        const NsDims d = ns_dims(t.it[i].m, t.it[i].n);
        NsSpace s;
        t.it[i].split = split_of(d);
        t.it[i].ws = ws + at;
        at += (int64_t)ns_space(nullptr, d, t.it[i].split, s);
    }
    return at;
}

// the largest power of two that keeps Q's entries, |Q| <= |a| + 1.5 |b| + 2.25 |c|, within fp16
float q_scale(float a, float b, float c)
{
    const double most = fabs((double)a) + 1.5 * fabs((double)b) + 2.25 * fabs((double)c);
    return most > 0.0 ? (float)exp2(fmin(14.0, floor(log2(60000.0 / most)))) : 1.0f;
}

// A chain over the items of a table whose sizes, pointers and settings are set, in pieces: prepare, then step(-1),
// step(0), ... step(t.steps - 1).  Matrices that all fit a compute unit's LDS are done in one launch, a workgroup each,
// by prepare.
struct Chain {
    NsTable t;
    NsTable *kept;
    hipStream_t st;
    const char *fn;
    bool dense, done;
    long long narrows, gram, sum, poly, rect;
    int poly_side, rect_side;

    template <typename F> int with_type(F &&f) const
    {
        if (t.dtype == DANCE_F32)
            return dense ? f((float)0, std::true_type{}) : f((float)0, std::false_type{});
        if (t.dtype == DANCE_F16)
            return dense ? f((_Float16)0, std::true_type{}) : f((_Float16)0, std::false_type{});
        return dense ? f((__bf16)0.0f, std::true_type{}) : f((__bf16)0.0f, std::false_type{});
    }

    int launched() const { return launch_check(fn); }

    int small() const
    {
        size_t lds = 0;
        for (int i = 0; i < t.count; ++i) {
            const size_t bytes = small_dims(t.it[i].m, t.it[i].n).bytes;
            lds = bytes > lds ? bytes : lds;
        }
        return with_type([&](auto type, auto is_dense) {
            using T = decltype(type);
            constexpr bool D = decltype(is_dense)::value;
            if (int rc = dance::allow_lds((const void *)k_ns_small<T, D>, lds, fn))
                return rc;
            hipLaunchKernelGGL((k_ns_small<T, D>), dim3(t.count), dim3(SMALL_THREADS), lds, st, t);
            return launched();
        });
    }

    int prepare(char *ws, hipStream_t stream, const char *name)
    {
        st = stream;
        fn = name;
        kept = (NsTable *)ws;
        dense = true;
        for (int i = 0; i < t.count; ++i)
            dense = dense && (t.muon || (t.col_stride == 1 && (t.row_stride == t.it[i].n || t.it[i].m == 1)));
        done = lay_out(t, ws) == 0;
        if (done)
            return t.count > 0 ? small() : 0;
        gram = poly = rect = 0;
        for (int i = 0; i < t.count; ++i) {
            const NsDims d = ns_dims(t.it[i].m, t.it[i].n);
            if (!narrow(d)) {
                gram += (long long)lower_tiles(d, PAD) * t.it[i].split;
                poly += lower_tiles(d, PAD);
                rect += (long long)(d.rp / PAD) * (d.kp / PAD);
            }
        }
        t.gram_side = side_for(gram);
        poly_side = side_for(poly);
        rect_side = side_for(rect);
        long long slices = 0, pack = 0;
        narrows = gram = sum = poly = rect = 0;
        for (int i = t.count; i < NS_ITEMS; ++i)
            t.slices[i] = t.pack[i] = t.narrow[i] = t.gram[i] = t.sum[i] = t.poly[i] = t.rect[i] = INT_MAX;
        for (int i = 0; i < t.count; ++i) {
            const NsDims d = ns_dims(t.it[i].m, t.it[i].n);
            const long long want = ((long long)t.it[i].m * t.it[i].n + 8191) / 8192;
            slices += want < NS_SLICES ? want : NS_SLICES;
            sum += (lower_tiles(d, 16) + SUM_THREADS / 64 - 1) / (SUM_THREADS / 64);
            if (narrow(d)) {
                narrows += t.it[i].split;
            } else {
                pack += (long long)(d.rp / PACK) * (d.kp / PACK);
                gram += (long long)lower_tiles(d, t.gram_side) * t.it[i].split;
                poly += lower_tiles(d, poly_side);
                rect += (long long)(d.rp / rect_side) * (d.kp / rect_side);
            }
            if (pack >= (1ll << 31) || gram >= (1ll << 31) || sum >= (1ll << 31) || rect >= (1ll << 31) || narrows >= (1ll << 31))
                return dance::fail((int)hipErrorInvalidValue, fn, "too many tiles");
            t.slices[i] = (int)slices;
            t.pack[i] = (int)pack;
            t.narrow[i] = (int)narrows;
            t.gram[i] = (int)gram;
            t.sum[i] = (int)sum;
            t.poly[i] = (int)poly;
            t.rect[i] = (int)rect;
        }
        return with_type([&](auto type, auto is_dense) {
            using T = decltype(type);
            constexpr bool D = decltype(is_dense)::value;
            hipLaunchKernelGGL((k_ns_norm<T, D>), dim3((unsigned)slices), dim3(256), 0, st, t, kept);
            if (int e = launched())
                return e;
            if (pack == 0)
                return 0;
            hipLaunchKernelGGL((k_ns_pack<T, D>), dim3((unsigned)pack), dim3(256), 0, st, (const NsTable *)kept);
            return launched();
        });
    }

    // kernel<F, DEPTH> on `tiles` tiles of side `side`, F = side / 32
    template <typename K, typename... Args> int tiled(int side, long long tiles, K &&kernel, Args... args) const
    {
        auto go = [&](auto f, auto depth) {
            constexpr int LDS = TILE_LDS<decltype(f)::value, decltype(depth)::value>;
            auto k = kernel(f, depth);
            if (int r = dance::allow_lds((const void *)k, LDS, fn))
                return r;
            hipLaunchKernelGGL(k, dim3((unsigned)tiles), dim3(GEMM_THREADS), LDS, st, (const NsTable *)kept, args...);
            return launched();
        };
        constexpr std::integral_constant<int, 2> two{};
        constexpr std::integral_constant<int, 4> four{};
        return side == 128 ? go(four, two) : tiles > 512 ? go(two, two) : go(two, four);
    }

    // step s of the X of all matrices, and the A of the next step; X itself is the -1st
    int step(int s) const
    {
        const int last = s + 1 == t.steps;
        int e = 0;
        if (done)
            return 0;
        if (narrows > 0) {
            e = with_type([&](auto type, auto is_dense) {
                using T = decltype(type);
                constexpr bool D = decltype(is_dense)::value;
                const dim3 grid((unsigned)narrows), block(NARROW_THREADS);
                const NsTable *table = kept;
                if (int r = s < 0 ? dance::allow_lds((const void *)k_ns_narrow_first<T, D>, FIRST_LDS, fn)
                                  : dance::allow_lds((const void *)k_ns_narrow<T>, NARROW_LDS, fn))
                    return r;
                if (s < 0)
                    hipLaunchKernelGGL((k_ns_narrow_first<T, D>), grid, block, FIRST_LDS, st, table);
                else
                    hipLaunchKernelGGL(k_ns_narrow<T>, grid, block, NARROW_LDS, st, table, last);
                return launched();
            });
        }
        if (e == 0 && rect > 0 && s >= 0)
            e = tiled(poly_side, poly, [](auto f, auto depth) { return k_ns_poly<decltype(f)::value, decltype(depth)::value>; });
        if (e == 0 && rect > 0 && s >= 0)
            e = tiled(rect_side, rect, [](auto f, auto depth) { return k_ns_apply<decltype(f)::value, decltype(depth)::value>; }, s, last);
        if (e == 0 && rect > 0 && !last)
            e = tiled(t.gram_side, gram, [](auto f, auto depth) { return k_ns_gram<decltype(f)::value, decltype(depth)::value>; }, s + 1);
        if (e == 0 && !last) {
            hipLaunchKernelGGL(k_ns_sum, dim3((unsigned)sum), dim3(SUM_THREADS), 0, st, (const NsTable *)kept);
            e = launched();
        }
        return e;
    }
};

bool usable(double a, double b, double c) { return isfinite(a) && isfinite(b) && isfinite(c); }

}  // namespace

extern "C" int64_t dance_orthogonalize_workspace_bytes(int batch, int m, int n)
{
    if (batch <= 0 || m <= 0 || n <= 0 || (long long)m * n > MOST_ELEMENTS)
        return 0;
    NsTable t;
    t.count = batch < NS_ITEMS ? batch : NS_ITEMS;
    for (int i = 0; i < t.count; ++i) {
        t.it[i].m = m;
        t.it[i].n = n;
    }
    return lay_out(t, nullptr);
}

extern "C" int dance_orthogonalize(const void *x, int64_t batch_stride, int64_t row_stride, int64_t col_stride,
                                   int dtype, void *out, int batch, int m, int n, int steps, float a, float b, float c,
                                   float eps, void *ws, int64_t ws_bytes, void *stream)
{
    DANCE_REQUIRE(batch >= 0 && m >= 0 && n >= 0 && (long long)m * n <= MOST_ELEMENTS);
    DANCE_REQUIRE(known_dtype(dtype) && steps >= 1 && steps <= 100 && usable(a, b, c) && eps > 0.0f);
    DANCE_REQUIRE(batch_stride >= 0 && row_stride >= 0 && col_stride >= 0);
    if (batch == 0 || m == 0 || n == 0)
        return 0;
    const int64_t need = dance_orthogonalize_workspace_bytes(batch, m, n);
    DANCE_REQUIRE(x && out && ((uintptr_t)ws & 15) == 0);
    DANCE_REQUIRE(ws_bytes >= need && (ws || need == 0));
    const int64_t size = dtype == DANCE_F32 ? 4 : 2;
    for (int b0 = 0; b0 < batch; b0 += NS_ITEMS) {
        Chain chain;
        NsTable &t = chain.t;
        memset(&t, 0, sizeof t);
        t.count = batch - b0 < NS_ITEMS ? batch - b0 : NS_ITEMS;
        t.dtype = dtype;
        t.row_stride = row_stride;
        t.col_stride = col_stride;
        t.steps = steps;
        t.a = a; t.b = b; t.c = c;
        t.q_mul = q_scale(a, b, c);
        t.eps = (double)eps;
        for (int i = 0; i < t.count; ++i) {
            t.it[i].src = (const char *)x + (b0 + i) * batch_stride * size;
            t.it[i].dst = (char *)out + (int64_t)(b0 + i) * m * n * size;
            t.it[i].m = m;
            t.it[i].n = n;
        }
        if (int rc = chain.prepare((char *)ws, (hipStream_t)stream, __func__))
            return rc;
        for (int s = -1; s < steps; ++s)
            if (int rc = chain.step(s))
                return rc;
    }
    return 0;
}

namespace {
// the next matrices of a kind, narrow or not, from items[at] on into a table -> where to go on
int take(const dance_muon_item *items, int count, bool wide, int at, NsTable &t)
{
    t.count = 0;
    for (; at < count && t.count < NS_ITEMS; ++at) {
        const dance_muon_item &h = items[at];
        if (narrow(ns_dims(h.rows, h.cols)) == wide)
            continue;
        NsItem &it = t.it[t.count++];
        it.src = h.grad;
        it.momentum = h.momentum;
        it.dst = h.param;
        it.m = h.rows;
        it.n = h.cols;
    }
    return at;
}

// The workspace of the narrow matrices' chains and of the others', the largest of either kind: the chains of a kind
// follow each other on one stream, those of the other kind run beside them on another -> both together
int64_t muon_space(const dance_muon_item *items, int count, int64_t (&most)[2])
{
    for (int wide = 0; wide < 2; ++wide) {
        most[wide] = 0;
        for (int at = 0; at < count;) {
            NsTable t;
            at = take(items, count, wide, at, t);
            const int64_t bytes = lay_out(t, nullptr);
            most[wide] = bytes > most[wide] ? bytes : most[wide];
        }
    }
    return most[0] + most[1];
}
}  // namespace

extern "C" int64_t dance_muon_workspace_bytes(const dance_muon_item *items_host, int count)
{
    if (count <= 0 || !items_host)
        return 0;
    for (int i = 0; i < count; ++i)
        if (items_host[i].rows <= 0 || items_host[i].cols <= 0 || (long long)items_host[i].rows * items_host[i].cols > MOST_ELEMENTS)
            return 0;
    int64_t most[2];
    return muon_space(items_host, count, most);
}

extern "C" int dance_muon_step(const dance_muon_item *items_host, int count, int dtype, double lr, double momentum,
                               int nesterov, double weight_decay, int steps, float a, float b, float c, float eps, void *ws,
                               int64_t ws_bytes, void *stream, void *side_stream)
{
    DANCE_REQUIRE(count >= 0 && known_dtype(dtype) && steps >= 1 && steps <= 100 && usable(a, b, c) && eps > 0.0f);
    DANCE_REQUIRE(usable(lr, momentum, weight_decay));
    if (count == 0)
        return 0;
    DANCE_REQUIRE(items_host && ((uintptr_t)ws & 15) == 0);
    for (int i = 0; i < count; ++i) {
        DANCE_REQUIRE(items_host[i].param && items_host[i].grad && items_host[i].momentum);
        DANCE_REQUIRE(items_host[i].rows >= 1 && items_host[i].cols >= 1);
        DANCE_REQUIRE((long long)items_host[i].rows * items_host[i].cols <= MOST_ELEMENTS);
    }
    int64_t most[2];
    const int64_t need = muon_space(items_host, count, most);
    DANCE_REQUIRE(ws_bytes >= need && (ws || need == 0));
    for (int at[2] = {0, 0}; at[0] < count || at[1] < count;) {
        // the narrow matrices and the others: two chains, launched in turn so that two streams run beside each other
        Chain chains[2];
        for (int wide = 1; wide >= 0; --wide) {
            NsTable &t = chains[wide].t;
            memset(&t, 0, sizeof t);
            at[wide] = take(items_host, count, wide, at[wide], t);
            t.dtype = dtype;
            t.muon = 1;
            t.nesterov = nesterov != 0;
            t.momentum = (float)momentum;
            t.fresh = (float)(1.0 - momentum);
            t.keep = (float)(1.0 - lr * weight_decay);
            t.steps = steps;
            t.a = a; t.b = b; t.c = c;
            t.q_mul = q_scale(a, b, c);
            t.eps = (double)eps;
            for (int i = 0; i < t.count; ++i) {
                const double m = t.it[i].m, n = t.it[i].n;
                t.it[i].scale = (float)(lr * (m > n ? sqrt(m / n) : 1.0));
            }
            if (int rc = chains[wide].prepare((char *)ws + (wide ? most[0] : 0),
                                              (hipStream_t)(wide && side_stream ? side_stream : stream), __func__))
                return rc;
        }
        for (int s = -1; s < steps; ++s)
            for (int wide = 1; wide >= 0; --wide)
                if (int rc = chains[wide].step(s))
                    return rc;
    }
    return 0;
}
