// Device code of the attention kernels whose columns (tokens or rows, and the q heads of a KV head) share one
// cache's K and V (k2t_attn_shared.hip, k2t_attn_tokens.hip): tiles of 32 positions, the running softmax, queries, joins.
//
// Scores S^T = K Q^T by the int8 MFMA, whose sums are exact, and outputs O^T = V^T W^T by the f16 MFMA. V's codes are
// exact in f16; a weight times its V scale is split into two f16 pieces that hold it to 2^-23 (an fp32 product to 2^-24,
// at several times the MFMAs). f16's range decides what the running softmax refers to: not a column's largest score, but
// its largest product of weight and V scale, so that a large scale of small weight takes no bits from the others.
// References are raised lazily, sums and outputs are fp32 and joined in a fixed order.
#pragma once

#include <float.h>
#include <math.h>

#include <type_traits>

#include "k2t_device.h"
#include "k2t_kv_dev.h"

namespace k2t {

namespace {
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4, kTile = 32;  // waves of a workgroup (where none is given); positions of a wave's tile
// A column's reference m is a power of two such that its products 2^(s - m) * V scale * kLift have reached 2^8
// and stay below 2^15.8: pieces below f16's smallest step, 2^-24, are then 2^-32 of the largest product. It is
// raised (a rescaling of the outputs, which some column of a tile would nearly always ask for) only where a
// product would pass 2^15.5, and then to bring that one to 2^8 .. 2^9.  kLift makes s - m, which fp32 rounds by
// 2^-24 of itself, a small number for scales of the usual size (2^-8 .. 1).
// A wave looks at its references where a bound of some column's products passes kLimit, and raises those whose
// products pass kRaise: so much later that a column's own bound has passed then, however the two were rounded
// (by 2^-3 each below kFar), and another column's products change nothing in it.
constexpr float kTop = 9.0f, kLimit = 15.0f, kRaise = 15.5f, kLift = 256.0f, kLog2Lift = 8.0f;
// Scales below 2^-100 count as that much in the reference, so that a weight is at most 2^107 and a sum of
// 2^16 of them finite (from 2^120 on, half of the largest scale that a head has, kLift overflows); an NF4 head's second block has a reference of its own (its scales may be of another
// size), but a weight refers to the first, which therefore counts as 2^-60 of the second at least.
// Nor is that block's reference lower than 2^-119 of the first one's: up1, 2^(m - m1) times kLift, stays finite.
constexpr float kLeastScale = 7.888609052210118e-31f, kApart = 60.0f, kWidest = 119.0f;
// Scores so far from zero that fp32 hardly tells whole numbers apart, or not at all.  An exact product less the reference would
// be up to half a step of the score off then, which may be any power of two: in a column whose reference is so far, scores
// are rounded before the reference, the largest rounded one, is taken off.  What V scales ask for cannot be part of such a
// reference, whose steps may be larger than that, and whose rounding would put it a step above every score: it is a
// second number (State::beside), taken off after.  Waves and parts are joined by the first one alone, in sums of V
// that such columns' scales may take to 2^100.
constexpr float kFar = 0x1p22f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= kFar && m > -FLT_MAX; }
constexpr float kLog2e = 1.44269504088896340736f;

// What the kernels' argument structs share: the columns' queries and outputs.
struct ColumnArgs {
    const float *q;
    uint32_t q_stride;
    float per_group;  // 1 / group
    int nq, group;    // group: q heads per KV head
    float attn_scale;
    int parts;     // of the positions that a column's row has at most
    float *part;   // [row][head][parts][HD]
    float2 *stat;  // [row][head][parts]: reference (in powers of two), sum
    float *out;
};

// Row and head (counted from an item's) of column c: c / group by a product, exact for c below 2^22: c + 0.5
// is half a step at least from a multiple of the group, and the product off by 2^-23 of itself.
struct Column {
    uint32_t row, head;
};
__device__ __forceinline__ Column column(const ColumnArgs &A, int c) {
    const uint32_t row = (uint32_t)(((float)c + 0.5f) * A.per_group);
    return Column{row, (uint32_t)c - row * (uint32_t)A.group};
}

__device__ __forceinline__ int row_len(const k2t_kv_rows &kv, int row) {
    return kv.d_len ? max(0, min(kv.d_len[row], kv.len)) : kv.len;
}

// A wave's tile of 32 positions as its lanes load it (li = lane % 16, lg = lane / 16), in two halves
// that are dead at different times.  K: rows 16 j + li, the 16 (NF4: 8) bytes lg of every 64-block,
// and the scales of positions 16 j + 4 lg + i.  V: those positions, the HD / 16 bytes li of the row
// (NF4: two bytes of every block).
template <int HD, int BITS>
struct TileK {
    static constexpr int NB = HD / 64, KW = BITS == 8 ? 4 : 2, SN = BITS == 8 ? 1 : NB;
    uint32_t k[2][NB][KW];
    uint32_t ks[2][4], vs[2][4];  // float, or the slot's BF16 scales (block 0 low)

    static __device__ __forceinline__ float scale(uint32_t w, int n) {
        return __uint_as_float(BITS == 8 ? w : n ? w & 0xFFFF0000u : w << 16);
    }
};
template <int HD, int BITS>
struct TileV {
    uint32_t v[2][4][HD / 64];
};

// The tile whose first position has slot `slot`; n positions of it exist (rows behind them repeat the
// last).  Addresses are a wave-uniform pointer and a small offset per lane.
template <int HD, int BITS>
__device__ __forceinline__ void load_k(TileK<HD, BITS> &T, const k2t_kv_rows &kv, size_t slot, int n, uint32_t li,
                                       uint32_t lg) {
    constexpr int NB = HD / 64, RB = BITS == 8 ? HD : HD / 2;
    const auto at = [&](uint32_t p) { return min(p, (uint32_t)n - 1u); };
    const uint8_t *kq = (const uint8_t *)kv.kq + slot * RB;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint32_t row = at(16u * j + li) * RB;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if constexpr (BITS == 8) {
                const uint4 w = *reinterpret_cast<const uint4 *>(kq + (row + 64 * b + 16 * lg));
                T.k[j][b][0] = w.x;
                T.k[j][b][1] = w.y;
                T.k[j][b][2] = w.z;
                T.k[j][b][3] = w.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2 *>(kq + (row + 32 * b + 8 * lg));
                T.k[j][b][0] = w.x;
                T.k[j][b][1] = w.y;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t p = at(16u * j + 4u * lg + i);
            if constexpr (BITS == 8 || NB == 2) {
                T.ks[j][i] = ((const uint32_t *)kv.ks + slot)[p];
                T.vs[j][i] = ((const uint32_t *)kv.vs + slot)[p];
            } else {
                T.ks[j][i] = ((const uint16_t *)kv.ks + slot)[p];
                T.vs[j][i] = ((const uint16_t *)kv.vs + slot)[p];
            }
        }
    }
}
template <int HD, int BITS>
__device__ __forceinline__ void load_v(TileV<HD, BITS> &T, const k2t_kv_rows &kv, size_t slot, int n, uint32_t li,
                                       uint32_t lg) {
    constexpr int RB = BITS == 8 ? HD : HD / 2;
    const uint8_t *vq = (const uint8_t *)kv.vq + slot * RB;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t p = 16u * j + 4u * lg + i, row = min(p, (uint32_t)n - 1u) * RB;
            if constexpr (BITS == 8 && HD == 128) {
                const uint2 w = *reinterpret_cast<const uint2 *>(vq + (row + 8 * li));
                T.v[j][i][0] = w.x;
                T.v[j][i][1] = w.y;
            } else if constexpr (BITS == 8) {
                T.v[j][i][0] = *reinterpret_cast<const uint32_t *>(vq + (row + 4 * li));
            } else {
#pragma unroll
                for (int b = 0; b < HD / 64; b++)
                    T.v[j][i][b] = *reinterpret_cast<const uint16_t *>(vq + (row + 32 * b + 2 * li));
            }
        }
}

// The NF4 KV codebook's tables (nf4_xor_tables).
struct Nf4 {
    uint32_t t0, t1, u0, u1;
};

// A 64-block of a K row as the i8 MFMA's A operand: for NF4 the lane's eight bytes hold elements
// e .. e + 7 and e + 16 .. e + 23, e = 32 (lg / 2) + 8 (lg % 2); the q operand is read in that order.
template <int BITS>
__device__ __forceinline__ v4i k_operand(const uint32_t *w, const Nf4 &c) {
    if constexpr (BITS == 8) {
        return v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    } else {
        const auto lut = [&](uint32_t n) { return (int)nf4_xlut(n, c.t0, c.t1, c.u0, c.u1); };
        return v4i{lut(w[0] & 0x0F0F0F0Fu), lut(w[1] & 0x0F0F0F0Fu), lut((w[0] >> 4) & 0x0F0F0F0Fu),
                   lut((w[1] >> 4) & 0x0F0F0F0Fu)};
    }
}

// Four consecutive positions' words (one byte per output tile) as the f16 A operands' halves: out[c]
// holds byte c of the four words.  A byte v becomes 1024 + (v + 128) by placing it under 0x64, then
// 1152 is taken off: exact.
__device__ __forceinline__ void v_halves(const uint32_t w0, const uint32_t w1, const uint32_t w2, const uint32_t w3,
                                         uint32_t (&out)[4][2]) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const uint32_t pair[2][2] = {{w0, w1}, {w2, w3}};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint32_t a = pair[h][0] ^ 0x80808080u, b = pair[h][1] ^ 0x80808080u;
        const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u), hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
        const uint32_t m[4] = {__builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u),
                               __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const v2h f = __builtin_bit_cast(v2h, m[c]) - v2h{(_Float16)1152.0f, (_Float16)1152.0f};
            out[c][h] = __builtin_bit_cast(uint32_t, f);
        }
    }
}

// A position's four V values of one word: int8 as they are; NF4 from four nibbles, in the order 0, 2,
// 1, 3 of the byte pair.
template <int BITS>
__device__ __forceinline__ uint32_t v_word(uint32_t w, const Nf4 &c) {
    if constexpr (BITS == 8) return w;
    return nf4_xlut((w & 0x0F0Fu) | ((w & 0xF0F0u) << 12), c.t0, c.t1, c.u0, c.u1);
}

// Two floats as f16 pairs hi + lo, each rounded to nearest: x = hi + lo within 2^-23 |x| (what is left of x has 2^-11 of it at
// most, and a sign).  Cut off instead, pieces were off by up to 2^-21.4, always towards zero, which the sum that
// outputs are divided by is not.
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    const auto pack = [](float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2h)); };
    hi = pack(x0, x1);
    float r0, r1;  // x - hi, exact: one mixed-precision fma each (the compiler converts and subtracts)
#if defined(__HIP_DEVICE_COMPILE__)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(hi), "v"(x1));
#else
    r0 = x0;
    r1 = x1;
#endif
    lo = pack(r0, r1);
}

// The lane's column, counted anew: as a value kept over the loop it would cost a register where none is left.
__device__ __forceinline__ uint32_t own_column() {
    uint32_t all = ~0u;
    asm volatile("" : "+s"(all));
    return __builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u)) & 15u;
}

// What a wave carries from tile to tile for NQ tiles of 16 columns: lane li is a column.  SN: V scales of a
// slot (NF4 heads of two blocks have one each).
template <int HD, int NQ, int SN>
struct State {
    v4f o[NQ][HD / 16];  // output tile b of column li: sums of 2^(s - m) V, times kLift (block 1: and 2^(m - m1))
    float m[NQ], l[NQ];  // reference (a whole number; -FLT_MAX: no score yet); this lane's share of the sum of 2^(s - m)
    float m1[SN > 1 ? NQ : 1], up1[SN > 1 ? NQ : 1];  // block 1's own reference, and 2^(m - m1) kLift
    // Columns whose reference is far (is_far): it is m + beside, and block 1's m + m1 (up1: 2^(beside - m1) kLift).  In LDS, for
    // such columns alone; far: the wave has met one.
    float *beside;
    bool far;

    __device__ __forceinline__ void clear(float *lds) {
        beside = lds;
        far = false;
#pragma unroll
        for (int a = 0; a < NQ; a++) {
            m[a] = -FLT_MAX;
            l[a] = 0.0f;
            if constexpr (SN > 1) {
                m1[a] = -FLT_MAX;
                up1[a] = kLift;
            }
#pragma unroll
            for (int b = 0; b < HD / 16; b++) o[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    // The wave's lane's place of column tile a.
    __device__ __forceinline__ float &beside_of(int a) const { return beside[16 * a + own_column()]; }
    // What takes output tiles of 64-block b of column tile a back to sums of 2^(s - m) V; block 0's times kLift, its sum.
    __device__ __forceinline__ float back(int a, int b) const {
        if (SN > 1 && b) return __builtin_amdgcn_exp2f(far && is_far(m[a]) ? m1[SN > 1 ? a : 0] : m1[SN > 1 ? a : 0] - m[a]) * (1.0f / kLift);
        return far && is_far(m[a]) ? __builtin_amdgcn_exp2f(beside_of(a)) * (1.0f / kLift) : 1.0f / kLift;
    }
};

// Scores of 16 positions x 16 columns, 64-block b of NB: int8 sums the blocks' dots, which are exact,
// and scales them once; NF4 scales every block's.  s: lane (lg, li) positions 4 lg + i, column li.
template <int BITS, int NB, typename Scale>
__device__ __forceinline__ void scores(const v4i (&kf)[NB], const v4i (&qb)[NB], Scale ks, float (&s)[4]) {
    v4i d = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < NB; b++) {
        if (BITS == 4 && b) d = v4i{0, 0, 0, 0};
        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[b], qb[b], d, 0, 0, 0);
        if (BITS == 8 && b + 1 < NB) continue;
#pragma unroll
        for (int i = 0; i < 4; i++)
            s[i] = BITS == 4 && b ? fmaf((float)d[i], ks(i, b), s[i]) : (float)d[i] * ks(i, 0);
    }
}

// log2 of a positive float by its bits, plus `add`: they are its exponent and then its mantissa, at most 0.09
// below the logarithm, and a product so much past the limit is still below f16's largest.
__device__ __forceinline__ float log2_bits(uint32_t bits, float add) { return fmaf((float)bits, 0x1p-23f, add - 127.0f); }
__device__ __forceinline__ float column_max(float v) {  // over a column's four lanes
    v = fmaxf(v, xor_lane(v, 16));
    return fmaxf(v, xor_lane(v, 32));
}

// The largest of three: fmaxf's result, without the instructions that quiet each operand first.
__device__ __forceinline__ float max3(float a, float b, float c) {
#if defined(__HIP_DEVICE_COMPILE__)
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
#else
    return fmaxf(fmaxf(a, b), c);
#endif
}
__device__ __forceinline__ float max8(const float (&t)[2][4]) {
    return max3(max3(t[0][0], t[0][1], t[0][2]), max3(t[0][3], t[1][0], t[1][1]), fmaxf(t[1][2], t[1][3]));
}

// What weights() does to the references of column tile a where a column of the wave is far, in it or in another.  mn: the
// column's new reference but for that; u1: log2 of its block 1's largest product.
template <int HD, int NQ, int SN>
__device__ __forceinline__ void far_references(State<HD, NQ, SN> &S, int a, const float (&t)[2][4], float qas, const float (&vs)[2][4][SN],
                                               float top, float u1, float mn, float to_lift, float &down, float &down1) {
    const bool was = is_far(S.m[a]);
    const float best = column_max(top * qas);
    // (near kFar the scale may ask for a far reference where the score is none)
    const float at = fmaxf(S.m[a], fabsf(best) >= kFar ? best : copysignf(kFar, mn));
    const bool now = is_far(mn) && is_far(at);
    mn = now ? at : mn;
    float v[SN];
    // (as if not known: the scales' logarithms, kept from the caller's loop, would not fit the registers)
    uint32_t magnitude = 0x7FFFFFFFu;
    asm volatile("" : "+s"(magnitude));
#pragma unroll
    for (int k = 0; k < SN; k++) {
        v[k] = top * qas - mn + (kLog2Lift - 100.0f);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                v[k] = fmaxf(v[k], (t[j][i] * qas - mn) + log2_bits(__float_as_uint(vs[j][i][k]) & magnitude, to_lift));
    }
    if constexpr (SN > 1) v[0] = fmaxf(v[0], v[1] - kApart);
    // the blocks' references, counted from m: before, and after
    const float shift = S.m[a] - mn;
    const float at0 = (was ? S.beside_of(a) : 0.0f) + shift, most0 = column_max(v[0]);
    const float to0 = !now ? 0.0f : most0 > at0 + kRaise ? ceilf(most0) - kTop : at0;
    down = at0 == to0 ? 1.0f : __builtin_amdgcn_exp2f(at0 - to0);
    down1 = down;
    if constexpr (SN > 1) {
        const float at1 = (was ? S.m1[a] : S.m1[a] - S.m[a]) + shift, most1 = column_max(v[SN - 1]);
        float to1;
        if (now) {
            to1 = fmaxf(most1 > at1 + kRaise ? ceilf(most1) - kTop : at1, to0 - kWidest);
        } else {
            const float m1 = was ? S.m[a] + S.m1[a] : S.m1[a], most = column_max(u1);
            to1 = fmaxf(most > m1 + kRaise ? ceilf(most) - kTop : m1, mn - kWidest) - mn;
        }
        down1 = at1 == to1 ? 1.0f : __builtin_amdgcn_exp2f(at1 - to1);
        S.m1[a] = now ? to1 : mn + to1;
        S.up1[a] = __builtin_amdgcn_exp2f(to0 - to1) * kLift;
    }
    S.m[a] = mn;
    if (now) S.beside_of(a) = to0;
}

// Weights of a tile from its scores: t = dots * K scales of positions 16 j + 4 lg + i of the columns
// li, n of the tile's 32 exist; vs = V scales.  Leaves pairs of weights times V scale times kLift as hi and
// lo pieces.  References change in one place, off the usual path: where the largest score of a lane's eight
// positions with the largest of their scales would pass the limit.  LIFTED: vs are V scales times kLift already.
template <int HD, int NQ, int SN, bool LIFTED = false>
__device__ __forceinline__ void weights(State<HD, NQ, SN> &S, float (&t)[NQ][2][4], const float (&qas)[NQ], float (&vs)[2][4][SN],
                                        int n, uint32_t lg, uint32_t (&ph)[NQ][SN][4], uint32_t (&pl)[NQ][SN][4]) {
    constexpr float kLifted = LIFTED ? kLift : 1.0f, kToLift = LIFTED ? 0.0f : kLog2Lift;
    float lv[SN];
#pragma unroll
    for (int k = 0; k < SN; k++) {
        uint32_t vmax = 0;  // (a negative scale, which is none of the cache's, counts as a large one here)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) vmax = max(vmax, __float_as_uint(vs[j][i][k]));
        lv[k] = log2_bits(max(vmax, __float_as_uint(kLeastScale * kLifted)), kToLift - kLimit);
    }
    if constexpr (SN > 1) lv[0] = fmaxf(lv[0], lv[1] - kApart);
    float top[NQ];
    bool news = false;
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        top[a] = max8(t[a]);
        // (qas >= 0: the largest t is the largest score)
        news |= fmaf(top[a], qas[a], lv[0]) > S.m[a];
        if constexpr (SN > 1) news |= fmaf(top[a], qas[a], lv[1]) > S.m1[a];
    }
    if (S.far || __any(news)) {
#pragma unroll
        for (int a = 0; a < NQ; a++) {
            float u[SN];
#pragma unroll
            for (int k = 0; k < SN; k++) {
                u[k] = fmaf(top[a], qas[a], kLog2Lift - 100.0f);  // (kLeastScale)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        u[k] = fmaxf(u[k], fmaf(t[a][j][i], qas[a], log2_bits(__float_as_uint(vs[j][i][k]) & 0x7FFFFFFFu, kToLift)));
            }
            if constexpr (SN > 1) u[0] = fmaxf(u[0], u[1] - kApart);
            const float most = column_max(u[0]);
            float mn = most > S.m[a] + kRaise ? ceilf(most) - kTop : S.m[a];
            S.far |= __any(is_far(mn)) != 0;
            float down, down1;
            if (__builtin_expect(!S.far, 1)) {
                down = mn == S.m[a] ? 1.0f : __builtin_amdgcn_exp2f(S.m[a] - mn);
                down1 = down;
                if constexpr (SN > 1) {
                    const float most1 = column_max(u[SN - 1]);
                    const float m1 = fmaxf(most1 > S.m1[a] + kRaise ? ceilf(most1) - kTop : S.m1[a], mn - kWidest);
                    down1 = m1 == S.m1[a] ? 1.0f : __builtin_amdgcn_exp2f(S.m1[a] - m1);
                    S.m1[a] = m1;
                    S.up1[a] = __builtin_amdgcn_exp2f(mn - m1) * kLift;
                }
                S.m[a] = mn;
            } else {
                far_references(S, a, t[a], qas[a], vs, top[a], u[SN - 1], mn, kToLift, down, down1);
            }
            S.l[a] *= down;
#pragma unroll
            for (int b = 0; b < HD / 16; b++) S.o[a][b] = S.o[a][b] * (SN > 1 && b >= 4 ? down1 : down);
        }
    }
    float by[NQ], from[NQ];
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        by[a] = qas[a];
        from[a] = S.m[a];
    }
    if (__builtin_expect(S.far, 0)) {
#pragma unroll
        for (int a = 0; a < NQ; a++) {
            const bool far = is_far(S.m[a]);  // (the other columns: t * 1 - 0)
            const float by0 = far ? qas[a] : 1.0f, from0 = far ? S.m[a] : 0.0f, beside = far ? S.beside_of(a) : 0.0f;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) t[a][j][i] = (t[a][j][i] * by0 - from0) - beside;
            by[a] = far ? 1.0f : qas[a];
            from[a] = far ? 0.0f : S.m[a];
        }
    }
#pragma unroll
    for (int a = 0; a < NQ; a++) {
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) t[a][j][i] = __builtin_amdgcn_exp2f(fmaf(t[a][j][i], by[a], -from[a]));
    }
    if (n < kTile) {  // positions behind the last one repeat it: they weigh nothing
#pragma unroll
        for (int a = 0; a < NQ; a++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (16 * j + 4 * (int)lg + i >= n) t[a][j][i] = 0.0f;
    }
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        S.l[a] += ((t[a][0][0] + t[a][0][1]) + (t[a][0][2] + t[a][0][3])) + ((t[a][1][0] + t[a][1][1]) + (t[a][1][2] + t[a][1][3]));
#pragma unroll
        for (int k = 0; k < SN; k++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    float x[2];
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        if (SN > 1 && k) x[e] = (t[a][j][i + e] * vs[j][i + e][k]) * (S.up1[SN > 1 ? a : 0] * (1.0f / kLifted));
                        else x[e] = t[a][j][i + e] * (LIFTED ? vs[j][i + e][k] : vs[j][i + e][k] * kLift);
                    }
                    split2(x[0], x[1], ph[a][k][2 * j + i / 2], pl[a][k][2 * j + i / 2]);
                }
    }
}

// Takes out of a tile what its columns do not see: bit 4 j + i of counts(a), the lane's column of tile a, is set for what it
// sees.  A score of -inf weighs nothing (the columns' qas are positive).  What is not seen may have any V scale, and a
// weight of zero times NaN is NaN: a scale that is not finite, or would not be once times kLift, counts as zero, and the
// columns that do see its position get a NaN score, so that their outputs are NaN.
template <bool LIFTED, int NQ, int SN, typename Counts>
__device__ __forceinline__ void hide_tile(float (&t)[NQ][2][4], float (&vs)[2][4][SN], const Counts &counts) {
    bool bad[2][4];
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            bad[j][i] = false;
#pragma unroll
            for (int k = 0; k < SN; k++) {
                const bool b = !(fabsf(vs[j][i][k]) <= FLT_MAX / (LIFTED ? 1.0f : kLift));
                vs[j][i][k] = b ? 0.0f : vs[j][i][k];
                bad[j][i] |= b;
            }
        }
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        const uint32_t m = counts(a);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                t[a][j][i] = m >> (4 * j + i) & 1u ? (bad[j][i] ? NAN : t[a][j][i]) : -INFINITY;
    }
}

// o += V^T w^T over 32 positions for one tile of output and 16 columns.
__device__ __forceinline__ v4f add_tile(v8h va, const uint32_t (&w)[4], v4f o) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(va, __builtin_bit_cast(v8h, make_uint4(w[0], w[1], w[2], w[3])), o, 0, 0, 0);
}

// Dimension of row x (0 .. 15) of output tile b.
template <int HD, int BITS>
__device__ __forceinline__ int out_dim(int b, int x) {
    if constexpr (BITS == 8) return HD == 128 ? 8 * x + b : 4 * x + b;
    // block b / 4, byte y of its 32 (tiles 0, 2: low nibbles 0, 1: see nf4_xlut's order above)
    const int t = b & 3, y = 2 * x + (t & 1), hi = t >> 1;
    return 64 * (b >> 2) + 32 * (y >> 4) + 16 * hi + (y & 15);
}

// What an item works on: columns col0 .. col0 + n - 1, column x being head head0 + x % group of row
// row0 + x / group, over len[0] positions of one cache from slot[0] on, then len[1] of another.
struct Item {
    k2t_kv_rows kv[2];
    size_t slot[2];
    int len[2];
    int row0, head0, col0, n, part;
};

template <int HD, int COLS>
struct Queries {
    __align__(16) int8_t q[COLS][HD + 16];
    float qas[COLS];
};

// One 64-block of a query head by sixteen lanes (four elements each), rotated and quantized with one
// scale per head as k2t_kv_store's int8 heads; block b of NB, the blocks of a head in neighbouring
// groups of lanes.  All lanes take part.
struct Quant4 {
    uint32_t w;  // four codes
    float qas;   // scale of the head's scores, in powers of two
};
template <int NB>
__device__ __forceinline__ Quant4 quantize_block(float4 f, uint32_t sb, uint32_t li, float attn_scale) {
    float v[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = flip_sign(v[j], (sb >> j) & 1u) * 0.125f;
    butterflies_slice4(v, li);
    float mx = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    mx = fmaxf(mx, xchg1(mx));
    mx = fmaxf(mx, xchg2(mx));
    mx = fmaxf(mx, xchg4(mx));
    mx = fmaxf(mx, xchg8(mx));
    if (NB > 1) mx = fmaxf(mx, xor_lane(mx, 16));
    const bool tiny = mx <= FLT_EPSILON;
    const float inv = 127.0f / mx;
    Quant4 r{0u, tiny ? 0.0f : ((mx / 127.0f) * attn_scale) * kLog2e};
#pragma unroll
    for (int j = 0; j < 4; j++) r.w |= (tiny ? 0u : (uint32_t)(int)rintf(v[j] * inv) & 0xFFu) << (8 * j);
    return r;
}

// The item's queries (columns behind the last repeat it) into LDS.
template <int WAVES, int HD, int COLS>
__device__ __forceinline__ void quantize_queries(const ColumnArgs &A, const Item &I, Queries<HD, COLS> &Q) {
    constexpr int NB = HD / 64, kTurns = (COLS * NB + 4 * WAVES - 1) / (4 * WAVES);
    const uint32_t lane = threadIdx.x & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const float *q0 = A.q + (size_t)I.row0 * A.q_stride + (size_t)I.head0 * HD;
    float4 f[kTurns];  // every load in flight at once
#pragma unroll
    for (int k = 0; k < kTurns; k++) {
        const int u = 4 * (wave + WAVES * k) + (int)lg, c = I.col0 + min(u / NB, I.n - 1);
        const Column at = column(A, c);
        f[k] = *reinterpret_cast<const float4 *>(q0 + ((uint64_t)at.row * A.q_stride + at.head * HD + 64 * (u % NB) + 4 * li));
    }
#pragma unroll
    for (int k = 0; k < kTurns; k++) {
        const int u = 4 * (wave + WAVES * k) + (int)lg, x = u / NB, b = u % NB;
        const Quant4 r = quantize_block<NB>(f[k], head_signs4<NB>(b, li), li, A.attn_scale);
        if (x >= COLS) continue;
        *reinterpret_cast<uint32_t *>(&Q.q[x][64 * b + 4 * li]) = r.w;
        if (li == 0 && b == 0) Q.qas[x] = r.qas;
    }
    __syncthreads();
}

// The score MFMA's B operand of 16 columns, lane li's codes at r, in the K operand's element order.
template <int HD, int BITS>
__device__ __forceinline__ void query_operand(const int8_t *r, uint32_t lg, v4i (&qb)[HD / 64]) {
#pragma unroll
    for (int b = 0; b < HD / 64; b++) {
        if constexpr (BITS == 8) {
            const int4 w = *reinterpret_cast<const int4 *>(r + 64 * b + 16 * lg);
            qb[b] = v4i{w.x, w.y, w.z, w.w};
        } else {
            const int e = 64 * b + 32 * (int)(lg >> 1) + 8 * (int)(lg & 1u);
            const int2 u = *reinterpret_cast<const int2 *>(r + e), w = *reinterpret_cast<const int2 *>(r + e + 16);
            qb[b] = v4i{u.x, u.y, w.x, w.y};
        }
    }
}
// Scores that are all zero, by a scale above zero: what hide_tile needs.
template <int NB>
__device__ __forceinline__ void above_zero(float &qas, v4i (&qb)[NB]) {
    if (qas != 0.0f) return;
    qas = FLT_MIN;
#pragma unroll
    for (int b = 0; b < NB; b++) qb[b] = v4i{0, 0, 0, 0};
}

// The waves' results, added in wave order, 16 columns at a time: a part for the merge, or (WHOLE) the
// output itself.
template <int HD, int WAVES>
struct Join {
    float m[WAVES][16], l[WAVES][16];
    __align__(16) float o[WAVES][16][HD + 4];
};
// any(c): column c has a position at all (else its output is zeros).
template <int HD, int BITS, int NQ, bool WHOLE, int SN, int WAVES, typename Any>
__device__ __forceinline__ void join(const ColumnArgs &A, const Item &I, const State<HD, NQ, SN> &S, const Any &any, Join<HD, WAVES> &J) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        if (16 * a >= I.n) break;
        const float back[2] = {S.back(a, 0), S.back(a, SN - 1)};
        float l = S.l[a] * (back[0] * kLift);
        l += xor_lane(l, 16);
        l += xor_lane(l, 32);
        if (lg == 0) {
            J.m[wave][li] = S.m[a];
            J.l[wave][li] = l;
        }
#pragma unroll
        for (int b = 0; b < HD / 16; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) J.o[wave][li][out_dim<HD, BITS>(b, 4 * (int)lg + i)] = S.o[a][b][i] * back[b >= 4];
        __syncthreads();
        // column, sixteenth of a 64-block's dimensions, and the first such block (four waves take one at a time)
        const int x = (int)(tid >> 4 & 15u), sl = (int)(tid & 15u), d0 = 64 * (wave >> 2);
        if (16 * a + x < I.n && d0 < HD) {
            float M = -FLT_MAX, L = 0.0f, e[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; w++) M = fmaxf(M, J.m[w][x]);
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                e[w] = __builtin_amdgcn_exp2f(J.m[w][x] - M);
                L = fmaf(J.l[w][x], e[w], L);
            }
            const int c = I.col0 + 16 * a + x;
            const Column to = column(A, c);
            const size_t pair = (size_t)(I.row0 + to.row) * A.nq + I.head0 + to.head;
            const size_t at = WHOLE ? pair : pair * A.parts + I.part;
#pragma unroll
            for (int d = d0; d < HD; d += 16 * WAVES) {
                float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < WAVES; w++) {
                    const float4 v = *reinterpret_cast<const float4 *>(&J.o[w][x][d + 4 * sl]);
                    r.x = fmaf(v.x, e[w], r.x);
                    r.y = fmaf(v.y, e[w], r.y);
                    r.z = fmaf(v.z, e[w], r.z);
                    r.w = fmaf(v.w, e[w], r.w);
                }
                if constexpr (WHOLE) {
                    // ifwht64 with four elements on each of sixteen lanes (those of a column take part together)
                    const float inv = 1.0f / L;
                    float v[4] = {r.x * inv, r.y * inv, r.z * inv, r.w * inv};
                    if (!any(c)) v[0] = v[1] = v[2] = v[3] = 0.0f;
                    butterflies_slice4(v, (uint32_t)sl);
                    const uint32_t sb = head_signs4<HD / 64>(d / 64, (uint32_t)sl);
                    r = make_float4(flip_sign(v[0] * 0.125f, sb & 1u), flip_sign(v[1] * 0.125f, (sb >> 1) & 1u),
                                    flip_sign(v[2] * 0.125f, (sb >> 2) & 1u), flip_sign(v[3] * 0.125f, sb >> 3));
                }
                *reinterpret_cast<float4 *>((WHOLE ? A.out : A.part) + at * HD + d + 4 * sl) = r;
            }
            if (!WHOLE && sl == 0 && d0 == 0) A.stat[at] = make_float2(M, L);
        }
        __syncthreads();
    }
}

// An item's columns (16 NQ at most): each wave takes every WAVES-th tile of 32 positions.  The next tile's K is
// loaded as soon as this one's scores are taken, the next V once this one's products are under way.
template <int HD, int NQ, int WAVES = kWaves>
struct Shared {
    Queries<HD, 16 * NQ> q;
    Join<HD, WAVES> j;
    float beside[WAVES][16 * NQ];
};
// hide(i, t, vs): takes out of tile i what a column does not see (Hidden); NoMask: columns see all positions of the item.
struct NoMask {};
template <int HD, int BITS, int NQ, bool WHOLE, int WAVES, typename Hide, typename Any>
__device__ __forceinline__ void attend(const ColumnArgs &A, const Item &I, const Hide &hide, const Any &any, Shared<HD, NQ, WAVES> &sh) {
    constexpr int NB = HD / 64, DB = HD / 16, SN = TileK<HD, BITS>::SN;
    const uint32_t lane = threadIdx.x & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    Nf4 cb{};
    if constexpr (BITS == 4) nf4_xor_tables(kNf4Cb0, kNf4Cb1, kNf4Cb2, kNf4Cb3, cb.t0, cb.t1, cb.u0, cb.u1);
    TileK<HD, BITS> K;
    TileV<HD, BITS> V;
    const int first = (I.len[0] + kTile - 1) / kTile, tiles = first + (I.len[1] + kTile - 1) / kTile;
    // (loads behind the last tile repeat it: issued without a branch, so that a wait for the older ones
    // can leave the newer ones in flight)
    const auto place = [&](int i, const k2t_kv_rows *&kv, size_t &slot, int &n) {
        const int k = i < first ? 0 : 1, at = kTile * (k ? i - first : i);
        kv = &I.kv[k];
        slot = I.slot[k] + at;
        n = I.len[k] - at;
    };
    const auto next_k = [&](int i) {
        const k2t_kv_rows *kv;
        size_t slot;
        int n;
        place(min(i, tiles - 1), kv, slot, n);
        load_k(K, *kv, slot, n, li, lg);
    };
    const auto next_v = [&](int i) {
        const k2t_kv_rows *kv;
        size_t slot;
        int n;
        place(min(i, tiles - 1), kv, slot, n);
        load_v(V, *kv, slot, n, li, lg);
    };
    next_k(wave);
    next_v(wave);
    quantize_queries<WAVES>(A, I, sh.q);
    v4i qb[NQ][NB];
    float qas[NQ];
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        qas[a] = sh.q.qas[16 * a + li];
        query_operand<HD, BITS>(sh.q.q[16 * a + li], lg, qb[a]);
        if constexpr (!std::is_same<Hide, NoMask>::value) above_zero(qas[a], qb[a]);
    }
    State<HD, NQ, SN> S;
    S.clear(sh.beside[wave]);
    for (int i = wave; i < tiles; i += WAVES) {
        const int left = i < first ? I.len[0] - kTile * i : I.len[1] - kTile * (i - first);
        float s[NQ][2][4], vs[2][4][SN];
        v4i kf[2][NB];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int b = 0; b < NB; b++) kf[j][b] = k_operand<BITS>(K.k[j][b], cb);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int a = 0; a < NQ; a++)
                scores<BITS>(kf[j], qb[a], [&](int i, int n) { return K.scale(K.ks[j][i], n); }, s[a][j]);
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int n = 0; n < SN; n++) vs[j][i][n] = K.scale(K.vs[j][i], n);
        // (behind the last use, so that the same registers take the load: a copy of them would wait for it)
        __builtin_amdgcn_sched_barrier(0);
        next_k(i + WAVES);
        uint32_t ph[NQ][SN][4], pl[NQ][SN][4];
        if constexpr (std::is_same<Hide, NoMask>::value) {
            weights<HD, NQ, SN>(S, s, qas, vs, left, lg, ph, pl);
        } else {  // (which takes out the positions behind the last one as well)
            hide(i, s, vs);
            weights<HD, NQ, SN>(S, s, qas, vs, kTile, lg, ph, pl);
        }
        // four output tiles (one 4-byte word of V per position) at a time
#pragma unroll
        for (int g = 0; g < DB / 4; g++) {
            uint32_t h[2][4][2];
#pragma unroll
            for (int j = 0; j < 2; j++)
                v_halves(v_word<BITS>(V.v[j][0][g], cb), v_word<BITS>(V.v[j][1][g], cb), v_word<BITS>(V.v[j][2][g], cb),
                         v_word<BITS>(V.v[j][3][g], cb), h[j]);
            if (g + 1 == DB / 4) {
                __builtin_amdgcn_sched_barrier(0);
                next_v(i + WAVES);
            }
            // the small pieces of all four tiles, then the large ones: no product waits for the one before
            constexpr int kBlocks = SN - 1;  // (NF4 blocks have weights of their own)
            v8h va[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                va[u] = __builtin_bit_cast(v8h, make_uint4(h[0][u][0], h[0][u][1], h[1][u][0], h[1][u][1]));
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int a = 0; a < NQ; a++) S.o[a][4 * g + u] = add_tile(va[u], pl[a][g & kBlocks], S.o[a][4 * g + u]);
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int a = 0; a < NQ; a++) S.o[a][4 * g + u] = add_tile(va[u], ph[a][g & kBlocks], S.o[a][4 * g + u]);
        }
    }
    join<HD, BITS, NQ, WHOLE>(A, I, S, any, sh.j);
}

// Joins the parts of one column: out = ifwht64(sum_i e_i part_i / sum_i e_i l_i), e_i = 2^(m_i - max m). A chain of
// latencies (lengths, statistics, partials, the transform): 3 to 5 us where the parts are a few MB (16480 heads of 128, 42 MB: 12).
// One (head, row) per WAVES waves: its parts' maxima and sums one per lane, then the outputs of every
// WAVES-th part, eight or sixteen loads in flight, joined in wave order, and ifwht64.  Parts that hold no
// positions (not live_part) were not written and count nothing; any: there is one that does.
template <int HD, int WAVES, int AHEAD = (WAVES > 1 ? 8 : 16), typename LivePart>
__device__ __forceinline__ void merge_parts(const ColumnArgs &A, int pair, const LivePart &live_part, bool any,
                                            float (*sum)[HD]) {
    constexpr int E = HD / 64, kAhead = AHEAD;  // values per lane; loads in flight
    const uint32_t lane = threadIdx.x & 63u;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int w0 = WAVES == 1 ? 0 : wave, n = A.parts;
    const size_t at = (size_t)pair * n;
    float m = -INFINITY, l = 0.0f, o[E] = {};
    for (int i0 = 0; i0 < n; i0 += 64) {
        const int mine = i0 + (int)lane, cnt = min(64, n - i0);
        float v[kAhead][E];
        const auto load = [&](int j0) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const float *p = A.part + (at + i0 + min(j0 + u * WAVES, cnt - 1)) * HD + E * lane;
                if constexpr (E == 2) {
                    const float2 f = *reinterpret_cast<const float2 *>(p);
                    v[u][0] = f.x;
                    v[u][1] = f.y;
                } else {
                    v[u][0] = *p;
                }
            }
        };
        const float2 st = A.stat[at + min(mine, n - 1)];
        load(w0);
        __builtin_amdgcn_sched_barrier(0);  // (all of them in flight before the reductions)
        const bool live = mine < n && live_part(mine);
        const float mn = fmaxf(m, wave_max_f(live ? st.x : -INFINITY));
        // (-inf: no live one yet; -FLT_MAX in a part whose scores are NaN)
        const float e = live ? __builtin_amdgcn_exp2f(st.x - mn) : 0.0f;
        const float corr = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l = fmaf(l, corr, wave_sum_f(live ? st.y * e : 0.0f));
#pragma unroll
        for (int k = 0; k < E; k++) o[k] *= corr;
        m = mn;
        // (e is zero behind the last part; the first batch outside the loop, and no branch before it: its loads would sink there)
        const auto add = [&](int j0) {
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const float w = lane_val(e, j0 + u * WAVES);
#pragma unroll
                for (int k = 0; k < E; k++) o[k] = w != 0.0f ? fmaf(v[u][k], w, o[k]) : o[k];
            }
        };
        add(w0);
        for (int j0 = w0 + kAhead * WAVES; j0 < cnt; j0 += kAhead * WAVES) {
            load(j0);
            add(j0);
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int k = 0; k < E; k++) sum[wave][E * lane + k] = o[k];
        __syncthreads();
        if (wave >= E) return;
    }
    // one 64-block per wave or turn, one element per lane
    const float inv = any ? 1.0f / l : 0.0f;
    float *out = A.out + (size_t)pair * HD;
    if constexpr (WAVES > 1) {
        float r = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) r += sum[w][64 * wave + lane];
        out[64 * wave + lane] = flip_sign(wave_butterflies64(r * inv, lane) * 0.125f, head_sign<E>(wave, lane));
    } else {
        // (a lane's two neighbouring elements of HD = 128 to one element of each block)
#pragma unroll
        for (int b = 0; b < E; b++) {
            float r = o[0];
            if constexpr (E == 2) {
                const int from = 32 * b + (int)(lane >> 1);
                const float r0 = __shfl(o[0], from, kWave), r1 = __shfl(o[E - 1], from, kWave);
                r = (lane & 1u) ? r1 : r0;
            }
            out[64 * b + lane] = flip_sign(wave_butterflies64(r * inv, lane) * 0.125f, head_sign<E>(b, lane));
        }
    }
}

}  // namespace

}  // namespace k2t
