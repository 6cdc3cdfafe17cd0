// mfma16.h -- the pieces of the fast precision mode's GEMM loop that more than one translation
// unit uses (snake16.hip, tail16.hip): LDS chunk-image geometry, the 32x32x16 f16 MFMA core loop
// with its rotating weight / vertex-tile buffers, accumulator initialisation.  See snake16.hip's
// header comment for the operand layout.
#pragma once
#include "common.h"
#include "p16.h"

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int ring16(int vv, int off, int v)
{
    int t = vv + off;
    t = t < 0 ? t + v : t;
    t = t >= v ? t - v : t;
    t = t >= v ? t - v : t;
    return t;
}

// Geometry of one LDS chunk image: [plane 2][CBC channel blocks][VP words of 16 B].
template <int RT, int CBC>
struct Geo {
    static constexpr int VP = RT * 32 + 1;          // odd row stride: conflict-free b128 reads
    static constexpr int CPR = (RT + 1) / 2;        // 64-lane passes along a row
    static constexpr int PLANE = CBC * VP * 16;     // bytes
    static constexpr int BYTES = 2 * PLANE;
};

// acc[ot][rt] += W[o-tiles, chunk] * X[chunk, :] for one LDS-resident chunk of 2 * NST channel
// blocks.
//   xs + lds0   : the chunk image (Geo<RT, 2 * NST>)
//   wchunk      : uniform byte pointer to W[plane 0][tap 0][chunk's first block][wave's o-tile 0]
//   wlane       : this lane's constant byte offset ((h * cout + r) * 16)
//   wps_b / wts_b / wstep_b : byte strides of a plane / a tap / two channel blocks (one step)
//   hook(s)     : called once per step of tap 0, after the step's weight prefetch was issued
//                 (the place for staged activation loads)
// AD weight buffers rotate (prefetch distance AD - 1 steps); NB vertex-tile (B) buffers rotate
// over the flat tile sequence q = s * RT + rt (prefetch distance NB - 1 tiles).
template <int RT, int OTW, int NST, int AD, int NB, int TERMS, typename Hook>
__device__ __forceinline__ void mfma16_core(f32x16 (&acc)[OTW][RT], const char *xs, unsigned lds0, int v,
                                            const char *wchunk, unsigned wlane, long long wps_b,
                                            long long wts_b, long long wstep_b, int taps, int dilation,
                                            int r, int h, Hook hook)
{
    constexpr int NT = NST * RT, DB = NB - 1, D = AD - 1;
    static_assert(NST % AD == 0 && D <= NST, "weight buffer rotation must close over a tap");
    static_assert(NT % NB == 0 && DB <= NT - RT && DB >= 1, "tile buffer rotation must close over a tap");
    using G = Geo<RT, 2 * NST>;
    constexpr int SSTEP = 2 * G::VP * 16;
    const unsigned rowb = lds0 + h * G::VP * 16;
    const unsigned lim = rowb + v * 16, d16 = dilation * 16, v16 = v * 16;
    unsigned p[RT];                             // LDS byte address of this lane's word, per vertex tile
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
        p[rt] = rowb + ring16(rt * 32 + r, -(taps >> 1) * dilation, v) * 16;

    h8 ah[AD][OTW], al[AD][OTW];
#define DANCE_LOAD_A(SLOT, PTR)                                                                   \
    do {                                                                                          \
        const char *pa_ = (PTR);                                                                  \
        _Pragma("unroll") for (int ot_ = 0; ot_ < OTW; ++ot_) {                                   \
            ah[SLOT][ot_] = *reinterpret_cast<const h8 *>(pa_ + wlane + ot_ * 512);               \
            if constexpr (TERMS == 3)                                                             \
                al[SLOT][ot_] = *reinterpret_cast<const h8 *>(pa_ + wps_b + wlane + ot_ * 512);   \
        }                                                                                         \
    } while (0)
    // tile Q of the current tap (Q < NT) or of the next one (p[] of its vertex tile already
    // advanced); p[rt] advances right after its last use in a tap (the fetch of step NST - 1)
#define DANCE_LOAD_B(Q)                                                                           \
    do {                                                                                          \
        constexpr int q_ = (Q) % NT, s_ = q_ / RT, rt_ = q_ % RT;                                 \
        bh[(Q) % NB] = *reinterpret_cast<const h8 *>(xs + p[rt_] + s_ * SSTEP);                   \
        if constexpr (TERMS == 3)                                                                 \
            bl[(Q) % NB] = *reinterpret_cast<const h8 *>(xs + p[rt_] + s_ * SSTEP + G::PLANE);    \
        if (s_ == NST - 1) {                                                                      \
            const unsigned tpos_ = p[rt_] + d16;                                                  \
            p[rt_] = tpos_ >= lim ? tpos_ - v16 : tpos_;                                          \
        }                                                                                         \
    } while (0)
#pragma unroll
    for (int q = 0; q < D; ++q)
        DANCE_LOAD_A(q, wchunk + q * wstep_b);
    h8 bh[NB], bl[NB];
    dance::static_for<0, DB>([&](auto q) __attribute__((always_inline)) { DANCE_LOAD_B(decltype(q)::value); });

    const char *wtap = wchunk;
    for (int tap = 0; tap < taps; ++tap) {
        const bool more = tap + 1 < taps;
        dance::static_for<0, NT>([&](auto qq) __attribute__((always_inline)) {
            constexpr int q = decltype(qq)::value, s = q / RT, rt = q % RT;
            if constexpr (rt == 0) {
                if (s + D < NST)
                    DANCE_LOAD_A((s + D) % AD, wtap + (s + D) * wstep_b);
                else if (more)
                    DANCE_LOAD_A((s + D) % AD, wtap + wts_b + (s + D - NST) * wstep_b);
                if (tap == 0)
                    hook(s);
            }
            DANCE_LOAD_B(q + DB);
            // keep the prefetch ahead of this tile's MFMAs (the scheduler otherwise sinks it
            // below them and the rotation collapses into load -> wait -> use)
            __builtin_amdgcn_sched_barrier(0);
            // an accumulator tile's three products back to back (see mfma16_core_sw)
#pragma unroll
            for (int ot = 0; ot < OTW; ++ot) {
                if constexpr (TERMS == 3) {
                    acc[ot][rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(al[s % AD][ot], bh[q % NB], acc[ot][rt], 0, 0, 0);
                    acc[ot][rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[s % AD][ot], bl[q % NB], acc[ot][rt], 0, 0, 0);
                }
                acc[ot][rt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ah[s % AD][ot], bh[q % NB], acc[ot][rt], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        });
        wtap += wts_b;
    }
#undef DANCE_LOAD_A
#undef DANCE_LOAD_B
}

// The same contraction on v_mfma_f32_16x16x32_f16 (K = 32 channels = 4 channel blocks per
// MFMA, 16 x 16 output tiles): the chip holds a higher clock on this shape under load
// (MI355X_MICROARCH.md, DVFS give-back item 7).  A wave's 32 x (RT * 32) output is 2 row tiles
// x 2 RT column tiles of 4 accumulator registers.
//   lane = (q4 = lane >> 4, c16 = lane & 15):  A word W[o0 + 16 i + c16][block 4 s + q4],
//   B word X[block 4 s + q4][vertex 16 j + c16],  C/D: vertex 16 j + c16, channels 4 q4 .. + 3.
// NST = steps of 32 channels per chunk; wlane = (q4 * cout + c16) * 16; wstep_b = 4 blocks.
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A wave owns CTW of the ring's 16-wide vertex tiles, starting at tile j0 (rings above 128 vertices split
// their tiles over two groups of waves).  RTG sizes the LDS image (row stride 32 * RTG + 1 words).
template <int RTG, int CTW, int NST, int AD, int NB, int TERMS, typename Hook>
__device__ __forceinline__ void mfma16_core_sw(f32x4 (&acc)[2][CTW], const char *xs, unsigned lds0, int v,
                                               const char *wchunk, unsigned wlane, long long wps_b,
                                               long long wts_b, long long wstep_b, int taps, int dilation,
                                               int c16, int q4, int j0, Hook hook)
{
    constexpr int CT = CTW, NT = NST * CT, DB = NB - 1, D = AD - 1;
    static_assert(NST % AD == 0 && D <= NST && D >= 1, "weight buffer rotation must close over a tap");
    static_assert(NT % NB == 0 && DB <= NT - CT && DB >= 1, "tile buffer rotation must close over a tap");
    using G = Geo<RTG, 4 * NST>;
    constexpr int SSTEP = 4 * G::VP * 16;
    const unsigned rowb = lds0 + q4 * G::VP * 16;
    const unsigned lim = rowb + v * 16, d16 = dilation * 16, v16 = v * 16;
    unsigned p[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j)
        p[j] = rowb + ring16((j0 + j) * 16 + c16, -(taps >> 1) * dilation, v) * 16;

    h8 ah[AD][2], al[AD][2];
#define DANCE_LOAD_A(SLOT, PTR)                                                                   \
    do {                                                                                          \
        const char *pa_ = (PTR);                                                                  \
        _Pragma("unroll") for (int i_ = 0; i_ < 2; ++i_) {                                        \
            ah[SLOT][i_] = *reinterpret_cast<const h8 *>(pa_ + wlane + i_ * 256);                 \
            if constexpr (TERMS == 3)                                                             \
                al[SLOT][i_] = *reinterpret_cast<const h8 *>(pa_ + wps_b + wlane + i_ * 256);     \
        }                                                                                         \
    } while (0)
#define DANCE_LOAD_B(Q)                                                                           \
    do {                                                                                          \
        constexpr int q_ = (Q) % NT, s_ = q_ / CT, j_ = q_ % CT;                                  \
        bh[(Q) % NB] = *reinterpret_cast<const h8 *>(xs + p[j_] + s_ * SSTEP);                    \
        if constexpr (TERMS == 3)                                                                 \
            bl[(Q) % NB] = *reinterpret_cast<const h8 *>(xs + p[j_] + s_ * SSTEP + G::PLANE);     \
        if (s_ == NST - 1) {                                                                      \
            const unsigned tpos_ = p[j_] + d16;                                                   \
            p[j_] = tpos_ >= lim ? tpos_ - v16 : tpos_;                                           \
        }                                                                                         \
    } while (0)
#pragma unroll
    for (int q = 0; q < D; ++q)
        DANCE_LOAD_A(q, wchunk + q * wstep_b);
    h8 bh[NB], bl[NB];
    dance::static_for<0, DB>([&](auto q) __attribute__((always_inline)) { DANCE_LOAD_B(decltype(q)::value); });

    const char *wtap = wchunk;
    for (int tap = 0; tap < taps; ++tap) {
        const bool more = tap + 1 < taps;
        dance::static_for<0, NT>([&](auto qq) __attribute__((always_inline)) {
            constexpr int q = decltype(qq)::value, s = q / CT, j = q % CT;
            if constexpr (j == 0) {
                if (s + D < NST)
                    DANCE_LOAD_A((s + D) % AD, wtap + (s + D) * wstep_b);
                else if (more)
                    DANCE_LOAD_A((s + D) % AD, wtap + wts_b + (s + D - NST) * wstep_b);
                if (tap == 0)
                    hook(s);
            }
            DANCE_LOAD_B(q + DB);
            __builtin_amdgcn_sched_barrier(0);
            // the three products of an accumulator tile back to back, then the other row tile's: a dependent MFMA
            // takes its C operand from the one before it instead of the register file -- measured (same box,
            // bit-identical: the order per accumulator is unchanged) residual stack 0.890 -> 0.867 ms, head
            // 0.304 -> 0.300 ms against the row tiles alternating (LAB.md section 10)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if constexpr (TERMS == 3) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al[s % AD][i], bh[q % NB], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[s % AD][i], bl[q % NB], acc[i][j], 0, 0, 0);
                }
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah[s % AD][i], bh[q % NB], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        });
        wtap += wts_b;
    }
#undef DANCE_LOAD_A
#undef DANCE_LOAD_B
}

// Staging of the next chunk image: this wave's rows (wave, wave + NW, ...), lanes along the
// row; lanes past the ring length repeat the last vertex (same value to the same address),
// which keeps loads and stores branch-free and the staging array in registers.
template <int RT, int CBC, int NW>
struct StageGeo {
    using G = Geo<RT, CBC>;
    static constexpr int RPW = (2 * CBC) / NW;      // rows per wave
    static constexpr int N = RPW * G::CPR;          // 16-B loads per lane
    static_assert((2 * CBC) % NW == 0, "rows split evenly over the waves");
};

// src: uniform byte pointer to (plane 0, chunk's first block) of the P16 slot
// vs: vertices per row of the P16 slot in memory (the ring length); v: vertices staged (a part
// of the ring when the caller splits it, src then points at the part's first vertex)
template <int RT, int CBC, int NW>
__device__ __forceinline__ void stage_load(u32x4 (&reg)[(StageGeo<RT, CBC, NW>::N)], int jlo, int jhi,
                                           const char *src, int v, int wave, int lane, int vs)
{
    using S = StageGeo<RT, CBC, NW>;
#pragma unroll
    for (int j = 0; j < S::N; ++j)
        if (j >= jlo && j < jhi) {
            const int row = wave + NW * (j / S::G::CPR);
            const int plane = row >= CBC ? 1 : 0, cbl = row - plane * CBC;
            const unsigned col = min((j % S::G::CPR) * 64 + lane, v - 1);
            reg[j] = *reinterpret_cast<const u32x4 *>(src + (plane * 256ll + cbl * 16ll) * vs + col * 16u);
        }
}

template <int RT, int CBC, int NW>
__device__ __forceinline__ void stage_load(u32x4 (&reg)[(StageGeo<RT, CBC, NW>::N)], int jlo, int jhi,
                                           const char *src, int v, int wave, int lane)
{
    stage_load<RT, CBC, NW>(reg, jlo, jhi, src, v, wave, lane, v);
}

template <int RT, int CBC, int NW>
__device__ __forceinline__ void stage_commit(const u32x4 (&reg)[(StageGeo<RT, CBC, NW>::N)], char *xs,
                                             unsigned lds0, int v, int wave, int lane)
{
    using S = StageGeo<RT, CBC, NW>;
#pragma unroll
    for (int j = 0; j < S::N; ++j) {
        const int row = wave + NW * (j / S::G::CPR);
        const unsigned col = min((j % S::G::CPR) * 64 + lane, v - 1);
        *reinterpret_cast<u32x4 *>(xs + lds0 + (row * S::G::VP + col) * 16u) = reg[j];
    }
}

// The same staging without registers: global_load_lds_dwordx4 moves 16 B per lane straight into
// LDS (destination = M0 base + lane * 16: a wave-instruction fills 64 consecutive words of an
// image row).  Written as inline asm on purpose: through the builtin the compiler cannot tell the
// image being filled from the one being read and puts s_waitcnt vmcnt(0) in front of the MFMA
// loop's ds_reads, which also drains the weight prefetch (measured: slower than registers).  The
// asm is invisible to its counter bookkeeping -- its own waits for the weight loads stay correct
// (vmcnt retires in order, they only ever wait for more) -- so the CALLER must issue
// s_waitcnt vmcnt(0) before the barrier that publishes the image (stage_dma_wait).
//   lds_dst: byte offset of the image inside the workgroup's LDS (wave-uniform)
// (M0 is on the asm's clobber list so that the compiler never carries a value of its own in it across
// the statement; clang notes that M0 is a reserved register it will not save -- which is what is wanted.
// s_nop: the copy needs one wait state after the write of M0, and the compiler adds none inside the asm)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int RT, int CBC, int NW>
__device__ __forceinline__ void stage_dma(int jlo, int jhi, const char *src, unsigned lds_dst, int v, int wave,
                                          int lane, int vs)
{
    using S = StageGeo<RT, CBC, NW>;
#pragma unroll
    for (int j = 0; j < S::N; ++j)
        if (j >= jlo && j < jhi) {
            const int row = wave + NW * (j / S::G::CPR);
            const int plane = row >= CBC ? 1 : 0, cbl = row - plane * CBC;
            const int col0 = (j % S::G::CPR) * 64;
            const unsigned col = min(col0 + lane, v - 1);
            const char *g = src + (plane * 256ll + cbl * 16ll) * vs + col * 16u;
            const unsigned l = __builtin_amdgcn_readfirstlane(lds_dst + (unsigned)(row * S::G::VP + col0) * 16u);
            // an odd number of 32-wide tiles: the last pass covers half a row, the other lanes
            // would land in the next row
            if (RT % 2 == 0 || col0 + lane < RT * 32)
                // nt: the staged activations are read once; without the hint they displace the
                // weights every workgroup re-reads from L2 (fusion 0.464 -> 0.452 ms at 1536 contours)
                // (m0 is clobbered: the compiler must not keep a value of its own in it across the asm)
                asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" : : "v"(g), "s"(l) : "memory", "m0");
        }
}

#pragma clang diagnostic pop

__device__ __forceinline__ void stage_dma_wait()
{
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <int RT, int OTW>
__device__ __forceinline__ void init_acc16(f32x16 (&acc)[OTW][RT], const float *bias_s, int o0, int h, float mul)
{
#pragma unroll
    for (int ot = 0; ot < OTW; ++ot)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            float4 b = {0.f, 0.f, 0.f, 0.f};
            if (bias_s)
                b = *reinterpret_cast<const float4 *>(bias_s + o0 + ot * 32 + 8 * g + 4 * h);
            const float bb[4] = {b.x * mul, b.y * mul, b.z * mul, b.w * mul};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                    acc[ot][rt][4 * g + i] = bb[i];
        }
}

__device__ __forceinline__ float relu_nan(float x) { return x > 0.0f ? x : (x != x ? x : 0.0f); }

// acc = fma(a, b, acc) as ONE v_fmac_f32 the compiler cannot pair into v_pk_fma_f32.
// Measured on MI355X (round 2, tools/tail_probe.py): with the row-constant GEMV of k_tail16 compiled to
// v_pk_fma_f32 (accumulator pairs, the LDS-sourced factor broadcast through op_sel, younger
// global loads of the same wave still in flight), workgroups that start while other workgroups
// of the CU are in their MFMA phase get wrong LOW halves of the pairs in lanes 48..63 -- run to
// run different, ~1e-2 relative, every counter wait in the ISA in place.  The first resident
// batch of workgroups (all in the GEMV at the same time, no MFMA beside it) never shows it, nor
// does the same code with single v_fmac_f32.  Round 3 (tools/lerp_probe.sh) localised it to the
// op_sel bit that sends source 1's HIGH half to the LOW result, dropped in the last quarter-wave pass beside MFMA
// issue; the GEMV stays unpaired and the whole library is built without packed fp32 forms.
__device__ __forceinline__ void fma1(float &acc, float a, float b)
{
    asm("v_fmac_f32 %0, %1, %2" : "+v"(acc) : "v"(a), "v"(b));
}

}  // namespace
