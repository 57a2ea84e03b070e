// Attention of one token of every row of a batch whose rows share their sequence's prefix cache and
// have a tail cache each (k2t_attn_shared): int8 or NF4 Hadamard caches, plain or grouped heads.
//
// For row r and q head h, over the positions t of its sequence's prefix and then of its tail:
//   s_t = scale_q scale_k[t] (codes_q . codes_k[t]) attn_scale,  w_t = exp(s_t - max s),
//   out = ifwht64( sum_t w_t scale_v[t] codes_v[t] / sum_t w_t ).
// The rows of a sequence and the q heads of a KV head are columns of one matrix against the same K and
// V, so both products are matrix products: scores S^T = K Q^T by the int8 MFMA, whose sums are exact,
// and outputs O^T = V^T W^T by the f16 MFMA. V's codes are exact in f16; a weight times its V scale is
// split into two f16 pieces that hold 21 bits of it (24 in an fp32 product, at several times the MFMAs).
// f16's range decides what the running softmax refers to: not a column's largest score, but its largest
// product of weight and V scale, so that a large scale of small weight takes no bits from the others.
// References are raised lazily, sums and outputs are fp32 and joined in a fixed order.
//
// Work is cut into (sequence, KV head, part of the positions, 16 or 32 columns), about two workgroups per
// CU; the parts' outputs are joined by a second kernel. The waves of a workgroup take tiles of 32
// positions in turn; K and V go from memory to registers in the operands' own layout, so a tile needs
// no LDS and no barrier.
//
// What bounds it: instructions, not bytes. A tile of 32 positions and 32 columns takes some 280 vector
// instructions (weights and their pieces, V's codes to f16, scales) next to 40 MFMAs, two waves to a
// SIMD; a part has few tiles, so its queries' transform and its join count too. Measured (passes in a row):
// 8 rows x 32 heads x 64, 1500 positions 9.5 us (0.9 TB/s of cache bytes); 64 rows x 32 / 4 heads x 128,
// 12000 + 333 positions 35.3 us (365 TFLOP/s); 3 sequences of 8 rows x 32 / 8 heads x 128, NF4, 4100 positions
// 19.0 us, a third of whose instructions look codes up; 4 rows x 9 / 3 heads x 64, 52 positions 5.2 us, a launch.
// References by products instead of scores cost NF4 heads of two blocks 2 to 3 % (a reference each: 19.9 and
// 20.3 us, 47.2 and 48.4 us with 64 rows), the others nothing where V scales are alike; with scales anywhere within
// 2^-2 .. 2^2 of each other references are raised more often (64 rows, int8: 35.4 and 36.5 us; 2^-8 .. 2^8: 38.6).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "k2t_branch.h"
#include "k2t_device.h"
#include "k2t_kv_dev.h"

namespace k2t {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4, kTile = 32;  // waves of a workgroup; positions of a wave's tile
// A column's reference m is a power of two such that its products 2^(s - m) * V scale * kLift have reached 2^8
// and stay below 2^15: pieces below f16's smallest step, 2^-24, are then 2^-32 of the largest product. It is
// raised (a rescaling of the outputs, which some column of a tile would nearly always ask for) only where a
// product would pass 2^15, and then to bring that one to 2^8 .. 2^9.  kLift makes s - m, which fp32 rounds by
// 2^-24 of itself, a small number for scales of the usual size (2^-8 .. 1).
constexpr float kTop = 9.0f, kLimit = 15.0f, kLift = 256.0f, kLog2Lift = 8.0f;
// Scales below 2^-100 count as that much in the reference, so that a weight is at most 2^107 and a sum of
// 2^16 of them finite (from 2^120 on, half of the largest scale that a head has, kLift overflows); an NF4 head's second block has a reference of its own (its scales may be of another
// size), but a weight refers to the first, which therefore counts as 2^-60 of the second at least.
constexpr float kLeastScale = 7.888609052210118e-31f, kApart = 60.0f;
// Scores so far from zero that fp32 does not tell whole numbers apart.  An exact product less the reference would
// be up to half a step of the score off then, which may be any power of two: in a column that has met one, scores
// are rounded before the reference, a rounded one itself, is taken off.
constexpr float kFar = 0x1p24f;
constexpr float kLog2e = 1.44269504088896340736f;

struct SharedArgs {
    const float *q;
    uint32_t q_stride;
    float per_group;  // 1 / group
    k2t_kv_rows pre, tail;
    int beams, nq, nkv, group;    // group: q heads per KV head
    int np, nt, plen, tlen;       // prefix and tail parts, and their positions
    int pgroups, tgroups, units;  // column groups of a prefix / tail item; prefix units (sequence, KV head, part)
    int pre_items;
    float attn_scale;
    float *part;   // [row][head][np + nt][HD]
    float2 *stat;  // [row][head][np + nt]: reference (in powers of two), sum
    float *out;
};

// Row and head (counted from an item's) of column c: c / group by a product, exact for c below 2^22: c + 0.5
// is half a step at least from a multiple of the group, and the product off by 2^-23 of itself.
struct Column {
    uint32_t row, head;
};
__device__ __forceinline__ Column column(const SharedArgs &A, int c) {
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

// Two floats as f16 pairs hi + lo: x = hi + lo within 2^-21 |x|.
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
    float r0, r1;  // x - hi, exact: one mixed-precision fma each (the compiler converts and subtracts)
#if defined(__HIP_DEVICE_COMPILE__)
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(hi), "v"(x0));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(hi), "v"(x1));
#else
    r0 = x0;
    r1 = x1;
#endif
    lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r0, r1));
}

// What a wave carries from tile to tile for NQ tiles of 16 columns: lane li is a column.  SN: V scales of a
// slot (NF4 heads of two blocks have one each).
template <int HD, int NQ, int SN>
struct State {
    v4f o[NQ][HD / 16];  // output tile b of column li: sums of 2^(s - m) V, times kLift (block 1: and 2^(m - m1))
    float m[NQ], l[NQ];  // reference (a whole number; -FLT_MAX: no score yet); this lane's share of the sum of 2^(s - m)
    float m1[SN > 1 ? NQ : 1], up1[SN > 1 ? NQ : 1];  // block 1's own reference, and 2^(m - m1) kLift
    bool far;            // some column of the wave has a reference beyond kFar

    __device__ __forceinline__ void clear() {
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
    // What takes output tile b of column tile a back to sums of 2^(s - m) V.
    __device__ __forceinline__ float back(int a, int b) const {
        if constexpr (SN > 1) {
            if (b >= 4) return __builtin_amdgcn_exp2f(m1[a] - m[a]) * (1.0f / kLift);
        }
        return 1.0f / kLift;
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

// Weights of a tile from its scores: t = dots * K scales of positions 16 j + 4 lg + i of the columns
// li, n of the tile's 32 exist; vs = V scales.  Leaves pairs of weights times V scale times kLift as hi and
// lo pieces.  References change in one place, off the usual path: where the largest score of a lane's eight
// positions with the largest of their scales would pass the limit.
template <int HD, int NQ, int SN>
__device__ __forceinline__ void weights(State<HD, NQ, SN> &S, float (&t)[NQ][2][4], const float (&qas)[NQ], float (&vs)[2][4][SN],
                                        int n, uint32_t lg, uint32_t (&ph)[NQ][SN][4], uint32_t (&pl)[NQ][SN][4]) {
    float lv[SN];
#pragma unroll
    for (int k = 0; k < SN; k++) {
        uint32_t vmax = 0;  // (a negative scale, which is none of the cache's, counts as a large one here)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) vmax = max(vmax, __float_as_uint(vs[j][i][k]));
        lv[k] = log2_bits(max(vmax, __float_as_uint(kLeastScale)), kLog2Lift - kLimit);
    }
    if constexpr (SN > 1) lv[0] = fmaxf(lv[0], lv[1] - kApart);
    float top[NQ];
    bool news = false;
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        top[a] = fmaxf(fmaxf(fmaxf(t[a][0][0], t[a][0][1]), fmaxf(t[a][0][2], t[a][0][3])),
                       fmaxf(fmaxf(t[a][1][0], t[a][1][1]), fmaxf(t[a][1][2], t[a][1][3])));
        // (qas >= 0: the largest t is the largest score)
        news |= fmaf(top[a], qas[a], lv[0]) > S.m[a];
        if constexpr (SN > 1) news |= fmaf(top[a], qas[a], lv[1]) > S.m1[a];
    }
    if (__any(news)) {
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
                        u[k] = fmaxf(u[k], fmaf(t[a][j][i], qas[a], log2_bits(__float_as_uint(vs[j][i][k]) & 0x7FFFFFFFu, kLog2Lift)));
            }
            if constexpr (SN > 1) u[0] = fmaxf(u[0], u[1] - kApart);
            const float most = column_max(u[0]);
            const float mn = most > S.m[a] + kLimit ? (fabsf(most) >= kFar ? most : ceilf(most) - kTop) : S.m[a];
            S.far |= __any(fabsf(mn) >= kFar && mn > -FLT_MAX) != 0;
            const float down = mn == S.m[a] ? 1.0f : __builtin_amdgcn_exp2f(S.m[a] - mn);
            float down1 = down;
            S.m[a] = mn;
            S.l[a] *= down;
            if constexpr (SN > 1) {
                // (no lower than 2^-120 of the first block's: 2^(m - m1) stays finite)
                const float most1 = column_max(u[SN - 1]);
                float m1 = fmaxf(most1 > S.m1[a] + kLimit ? ceilf(most1) - kTop : S.m1[a], mn - 120.0f);
                if (fabsf(mn) >= kFar) m1 = mn;
                down1 = m1 == S.m1[a] ? 1.0f : __builtin_amdgcn_exp2f(S.m1[a] - m1);
                S.m1[a] = m1;
                S.up1[a] = __builtin_amdgcn_exp2f(mn - m1) * kLift;
            }
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
    if (S.far) {
#pragma unroll
        for (int a = 0; a < NQ; a++) {
            const bool far = fabsf(S.m[a]) >= kFar;  // (the other columns: t * 1 - 0)
            const float by0 = far ? qas[a] : 1.0f, from0 = far ? S.m[a] : 0.0f;
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) t[a][j][i] = t[a][j][i] * by0 - from0;
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
                        if (SN > 1 && k) x[e] = (t[a][j][i + e] * vs[j][i + e][k]) * S.up1[SN > 1 ? a : 0];
                        else x[e] = t[a][j][i + e] * (vs[j][i + e][k] * kLift);
                    }
                    split2(x[0], x[1], ph[a][k][2 * j + i / 2], pl[a][k][2 * j + i / 2]);
                }
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
template <int HD, int COLS>
__device__ __forceinline__ void quantize_queries(const SharedArgs &A, const Item &I, Queries<HD, COLS> &Q) {
    constexpr int NB = HD / 64, kTurns = (COLS * NB + 4 * kWaves - 1) / (4 * kWaves);
    const uint32_t lane = threadIdx.x & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const float *q0 = A.q + (size_t)I.row0 * A.q_stride + (size_t)I.head0 * HD;
    float4 f[kTurns];  // every load in flight at once
#pragma unroll
    for (int k = 0; k < kTurns; k++) {
        const int u = 4 * (wave + kWaves * k) + (int)lg, c = I.col0 + min(u / NB, I.n - 1);
        const Column at = column(A, c);
        f[k] = *reinterpret_cast<const float4 *>(q0 + ((uint64_t)at.row * A.q_stride + at.head * HD + 64 * (u % NB) + 4 * li));
    }
#pragma unroll
    for (int k = 0; k < kTurns; k++) {
        const int u = 4 * (wave + kWaves * k) + (int)lg, x = u / NB, b = u % NB;
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
// The waves' results, added in wave order, 16 columns at a time: a part for the merge, or (WHOLE) the
// output itself.
template <int HD>
struct Join {
    float m[kWaves][16], l[kWaves][16];
    __align__(16) float o[kWaves][16][HD + 4];
};
template <int HD, int BITS, int NQ, bool WHOLE, int SN>
__device__ __forceinline__ void join(const SharedArgs &A, const Item &I, const State<HD, NQ, SN> &S, Join<HD> &J) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        if (16 * a >= I.n) break;
        float l = S.l[a];
        l += xor_lane(l, 16);
        l += xor_lane(l, 32);
        if (lg == 0) {
            J.m[wave][li] = S.m[a];
            J.l[wave][li] = l;
        }
#pragma unroll
        for (int b = 0; b < HD / 16; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) J.o[wave][li][out_dim<HD, BITS>(b, 4 * (int)lg + i)] = S.o[a][b][i] * S.back(a, b);
        __syncthreads();
        const int x = (int)(tid >> 4), sl = (int)(tid & 15u);  // column, sixteenth of its dimensions
        if (16 * a + x < I.n) {
            float M = -FLT_MAX, L = 0.0f, e[kWaves];
#pragma unroll
            for (int w = 0; w < kWaves; w++) M = fmaxf(M, J.m[w][x]);
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                e[w] = __builtin_amdgcn_exp2f(J.m[w][x] - M);
                L = fmaf(J.l[w][x], e[w], L);
            }
            const int c = I.col0 + 16 * a + x;
            const Column to = column(A, c);
            const size_t pair = (size_t)(I.row0 + to.row) * A.nq + I.head0 + to.head;
            const size_t at = WHOLE ? pair : pair * (A.np + A.nt) + I.part;
#pragma unroll
            for (int d = 0; d < HD; d += 64) {
                float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
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
                    butterflies_slice4(v, (uint32_t)sl);
                    const uint32_t sb = head_signs4<HD / 64>(d / 64, (uint32_t)sl);
                    r = make_float4(flip_sign(v[0] * 0.125f, sb & 1u), flip_sign(v[1] * 0.125f, (sb >> 1) & 1u),
                                    flip_sign(v[2] * 0.125f, (sb >> 2) & 1u), flip_sign(v[3] * 0.125f, sb >> 3));
                }
                *reinterpret_cast<float4 *>((WHOLE ? A.out : A.part) + at * HD + d + 4 * sl) = r;
            }
            if (!WHOLE && sl == 0) A.stat[at] = make_float2(M, L);
        }
        __syncthreads();
    }
}

// An item's columns (16 NQ at most): each wave takes every fourth tile of 32 positions.  The next tile's K is
// loaded as soon as this one's scores are taken, the next V once this one's products are under way.
template <int HD, int NQ>
struct Shared {
    Queries<HD, 16 * NQ> q;
    Join<HD> j;
};
template <int HD, int BITS, int NQ, bool WHOLE>
__device__ __forceinline__ void attend(const SharedArgs &A, const Item &I, Shared<HD, NQ> &sh) {
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
    quantize_queries(A, I, sh.q);
    v4i qb[NQ][NB];
    float qas[NQ];
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        qas[a] = sh.q.qas[16 * a + li];
        query_operand<HD, BITS>(sh.q.q[16 * a + li], lg, qb[a]);
    }
    State<HD, NQ, SN> S;
    S.clear();
    for (int i = wave; i < tiles; i += kWaves) {
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
        next_k(i + kWaves);
        uint32_t ph[NQ][SN][4], pl[NQ][SN][4];
        weights<HD, NQ, SN>(S, s, qas, vs, left, lg, ph, pl);
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
                next_v(i + kWaves);
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
    join<HD, BITS, NQ, WHOLE, SN>(A, I, S, sh.j);
}

template <int HD, int BITS, int NQ>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_part_kernel(SharedArgs A) {
    __shared__ union U {
        Shared<HD, NQ> prefix;
        Shared<HD, 1> tail;
        __device__ U() {}
    } sh;
    const int id = (int)blockIdx.x;
    Item I;
    if (id < A.pre_items) {
        // A unit's column groups read the same K / V: they get ids congruent mod 8, one XCD's.
        const int slot = id >> 3, unit = (id & 7) + 8 * (slot / A.pgroups), cg = slot % A.pgroups;
        if (unit >= A.units) return;
        const int sk = unit / A.np, head = sk % A.nkv, seq = sk / A.nkv;
        I.part = unit % A.np;
        const int t0 = I.part * A.plen;
        I.kv[0] = I.kv[1] = A.pre;
        I.slot[0] = I.slot[1] = ((size_t)seq * A.nkv + head) * A.pre.cap + t0;
        I.len[0] = min(row_len(A.pre, seq) - t0, A.plen);
        I.len[1] = 0;
        if (I.len[0] <= 0) return;
        I.row0 = seq * A.beams;
        I.head0 = head * A.group;
        I.col0 = 16 * NQ * cg;
        I.n = min(16 * NQ, A.beams * A.group - I.col0);
        attend<HD, BITS, NQ, false>(A, I, sh.prefix);
        return;
    }
    int t = id - A.pre_items;
    const int cg = t % A.tgroups;
    t /= A.tgroups;
    I.part = t % A.nt;
    t /= A.nt;
    const int head = t % A.nkv, row = t / A.nkv;
    const int t0 = I.part * A.tlen;
    I.kv[0] = I.kv[1] = A.tail;
    I.slot[0] = I.slot[1] = ((size_t)row * A.nkv + head) * A.tail.cap + t0;
    I.len[0] = min(row_len(A.tail, row) - t0, A.tlen);
    I.len[1] = 0;
    if (I.len[0] <= 0) return;
    I.part += A.np;
    I.row0 = row;
    I.head0 = head * A.group;
    I.col0 = 16 * cg;
    I.n = min(16, A.group - I.col0);
    attend<HD, BITS, 1, false>(A, I, sh.tail);
}

// Few positions: one workgroup per (row, KV head, 16 q heads) takes the prefix and the tail and writes
// the output; the prefix is read once per row, by so few bytes that a second launch costs more.
template <int HD, int BITS>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_whole_kernel(SharedArgs A) {
    __shared__ Shared<HD, 1> sh;
    int t = (int)blockIdx.x;
    const int cg = t % A.tgroups;
    t /= A.tgroups;
    const int head = t % A.nkv, row = t / A.nkv, seq = row / A.beams;
    Item I;
    I.kv[0] = A.pre;
    I.kv[1] = A.tail;
    I.slot[0] = ((size_t)seq * A.nkv + head) * A.pre.cap;
    I.slot[1] = ((size_t)row * A.nkv + head) * A.tail.cap;
    I.len[0] = A.pre.cap ? row_len(A.pre, seq) : 0;
    I.len[1] = A.tail.cap ? row_len(A.tail, row) : 0;
    I.row0 = row;
    I.head0 = head * A.group;
    I.col0 = 16 * cg;
    I.n = min(16, A.group - I.col0);
    I.part = 0;
    if (I.len[0] + I.len[1] == 0) {
        float *out = A.out + ((size_t)row * A.nq + I.head0 + I.col0) * HD;
        for (int i = (int)threadIdx.x; i < I.n * HD; i += 64 * kWaves) out[i] = 0.0f;
        return;
    }
    attend<HD, BITS, 1, true>(A, I, sh);
}

// Joins the parts: out = ifwht64(sum_i e_i part_i / sum_i e_i l_i), e_i = 2^(m_i - max m). A chain of
// latencies (lengths, statistics, partials, the transform): 3 to 5 us whatever the sizes here.
// One (head, row) per WAVES waves: its parts' maxima and sums one per lane, then the outputs of every
// WAVES-th part, eight or sixteen loads in flight, joined in wave order, and ifwht64.  Parts that hold no
// positions were not written and count nothing.
template <int HD, int WAVES>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs A, int pairs) {
    constexpr int E = HD / 64, kAhead = WAVES > 1 ? 8 : 16;  // values per lane; loads in flight
    __shared__ float sum[WAVES > 1 ? WAVES : 1][HD];
    const uint32_t lane = threadIdx.x & 63u;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int pair = WAVES == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x, w0 = WAVES == 1 ? 0 : wave;
    if (pair >= pairs) return;
    const int row = pair / A.nq, n = A.np + A.nt;
    const size_t at = (size_t)pair * n;
    const int np = A.np ? (row_len(A.pre, row / A.beams) + A.plen - 1) / A.plen : 0;
    const int nt = A.nt ? (row_len(A.tail, row) + A.tlen - 1) / A.tlen : 0;
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
        const bool live = mine < n && (mine < A.np ? mine < np : mine - A.np < nt);
        const float mn = fmaxf(m, wave_max_f(live ? st.x : -INFINITY));
        if (mn == -INFINITY) continue;  // (no live one: -FLT_MAX in a part whose scores are NaN)
        const float e = live ? __builtin_amdgcn_exp2f(st.x - mn) : 0.0f, corr = __builtin_amdgcn_exp2f(m - mn);
        l = fmaf(l, corr, wave_sum_f(live ? st.y * e : 0.0f));
#pragma unroll
        for (int k = 0; k < E; k++) o[k] *= corr;
        m = mn;
        for (int j0 = w0; j0 < cnt; j0 += kAhead * WAVES) {
            if (j0 > w0) load(j0);
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
                const int j = j0 + u * WAVES;
                const float w = j < cnt ? lane_val(e, j) : 0.0f;
#pragma unroll
                for (int k = 0; k < E; k++) o[k] = w != 0.0f ? fmaf(v[u][k], w, o[k]) : o[k];
            }
        }
    }
    if constexpr (WAVES > 1) {
#pragma unroll
        for (int k = 0; k < E; k++) sum[wave][E * lane + k] = o[k];
        __syncthreads();
        if (wave >= E) return;
    }
    // one 64-block per wave or turn, one element per lane
    const float inv = np + nt == 0 ? 0.0f : 1.0f / l;
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

// shared_whole_kernel up to this many positions, times its rounds of three workgroups per CU.  Measured
// on both sides (32 heads x 64, 8 rows: 320 positions 6.2 us and 8.4 in two launches, 720 8.4 and 8.6, 920 9.7
// and 8.6; 32 rows, two rounds, 320 positions 9.4 and 11.0, 520 11.8 and 11.3).
constexpr size_t kWholeMax = 720, kWholeRound = 3;
// Prefix items of two tiles of columns from this many (tile of columns, 32 positions) steps on: fewer
// instructions per step, but half the workgroups (32 / 4 heads x 128, 12000 positions: 32 rows, 24000
// steps, 28.4 us and 32.3 with one tile; 16 rows, 12000 steps, 22.9 and 21.2).
constexpr size_t kTwoTiles = 18000;

// How the work is cut.  nq: the prefix items' column tiles; parts so that there are about two
// workgroups for every CU, of a tile for every wave at least.
struct Plan {
    int nq, np, plen, pgroups, nt, tlen, tgroups;
    bool whole;  // shared_whole_kernel
};
Plan plan_of(const k2t_ctx *ctx, const SharedShape &s, int prefix_len, int tail_len) {
    const int group = s.nq / s.nkv, cols = s.beams * group, least = kTile * kWaves;
    Plan P{};
    P.tgroups = (group + 15) / 16;
    const size_t cus = (size_t)std::max(1, ctx->num_cus), wholes = (size_t)s.n_seq * s.beams * s.nkv * P.tgroups;
    P.whole = ((size_t)prefix_len + tail_len) * ((wholes + kWholeRound * cus - 1) / (kWholeRound * cus)) <= kWholeMax;
    if (P.whole) return P;
    const size_t steps = (size_t)s.n_seq * s.nkv * ((cols + 15) / 16) * (prefix_len / kTile);
    P.nq = steps >= kTwoTiles ? 2 : 1;
    P.pgroups = (cols + 16 * P.nq - 1) / (16 * P.nq);
    const auto cut = [&](int len, size_t items, int &n, int &each) {
        if (len == 0) return;
        const int want = (int)std::max<size_t>(1, 2 * cus / std::max<size_t>(1, items));
        each = ((len + want - 1) / want + least - 1) / least * least;
        n = (len + each - 1) / each;
    };
    cut(prefix_len, (size_t)s.n_seq * s.nkv * P.pgroups, P.np, P.plen);
    // The prefix items count among the tails': where they fill the card, a tail's further parts are only more
    // queries to transform and parts to join (64 rows x 32 / 4 heads x 128, 12000 + 333 positions: one part per
    // tail 41.3 us, two 45.1; 16 rows x 32 / 8, 4000 + 333: 16.5 and 18.0 with three).
    cut(tail_len, (size_t)s.n_seq * s.beams * s.nkv * P.tgroups + (size_t)s.n_seq * s.nkv * P.pgroups * P.np, P.nt, P.tlen);
    return P;
}
size_t part_slots(const SharedShape &s, int parts) { return (size_t)s.n_seq * s.beams * s.nq * parts; }
size_t ws_bytes_of(const SharedShape &s, int parts) {
    return std::max<size_t>(16, part_slots(s, parts) * (s.hd * sizeof(float) + sizeof(float2)));
}
// At least the parts (np + nt) of every plan of up to these lengths.  One plan's are not monotone: parts are
// whole tiles for every wave, so that a longer cache may be cut into fewer.  For every width of prefix items (two
// tiles of columns only where the longest has them) and np: as many tail parts as such a plan may want.
int most_parts(const k2t_ctx *ctx, const SharedShape &s, int prefix_len, int tail_len) {
    const Plan P = plan_of(ctx, s, prefix_len, tail_len);
    if (P.whole) return 0;  // (and so is every shorter one)
    const int least = kTile * kWaves, cols = s.beams * (s.nq / s.nkv);
    const size_t cus = (size_t)std::max(1, ctx->num_cus), heads = (size_t)s.n_seq * s.nkv;
    const auto cut = [&](int len, size_t items) {
        const size_t want = std::max<size_t>(1, 2 * cus / std::max<size_t>(1, items));
        return (int)std::min<size_t>(((size_t)len + least - 1) / least, want);
    };
    int most = 0;
    for (int nq = 1; nq <= P.nq; nq++) {
        const size_t pre = heads * ((cols + 16 * nq - 1) / (16 * nq));
        for (int np = 0; np <= cut(prefix_len, pre); np++)
            most = std::max(most, np + cut(tail_len, heads * s.beams * P.tgroups + pre * np));
    }
    return most;
}

template <int HD, int BITS>
void launch_parts(hipStream_t st, const SharedArgs &A, const Plan &P, size_t items) {
    const dim3 grid((unsigned)items), block(64 * kWaves);
    if (P.nq == 2) hipLaunchKernelGGL((shared_part_kernel<HD, BITS, 2>), grid, block, 0, st, A);
    else hipLaunchKernelGGL((shared_part_kernel<HD, BITS, 1>), grid, block, 0, st, A);
    hip_check(hipGetLastError(), "attn_shared launch");
}

template <int HD>
void launch_shared(hipStream_t st, int bits, const SharedArgs &A, const SharedShape &s, const Plan &P, size_t items) {
    const int pairs = s.n_seq * s.beams * s.nq;
    if (P.whole) {
        const dim3 grid((unsigned)((size_t)s.n_seq * s.beams * s.nkv * P.tgroups));
        if (bits == 8) hipLaunchKernelGGL((shared_whole_kernel<HD, 8>), grid, dim3(64 * kWaves), 0, st, A);
        else hipLaunchKernelGGL((shared_whole_kernel<HD, 4>), grid, dim3(64 * kWaves), 0, st, A);
        hip_check(hipGetLastError(), "attn_shared launch");
        return;
    }
    if (items && bits == 8) launch_parts<HD, 8>(st, A, P, items);
    if (items && bits == 4) launch_parts<HD, 4>(st, A, P, items);
    // Four waves share a head's parts where there are many, and so few heads (4 rows x 9 / 3 heads x 64,
    // 12000 positions, 95 parts: 10.4 us and 12.9 with one wave; 64 rows x 32 / 4 x 128, 9 parts: 39.9 and 37.3).
    if (A.np + A.nt > 16) hipLaunchKernelGGL((shared_merge_kernel<HD, 4>), dim3(pairs), dim3(256), 0, st, A, pairs);
    else hipLaunchKernelGGL((shared_merge_kernel<HD, 1>), dim3((pairs + 3) / 4), dim3(256), 0, st, A, pairs);
    hip_check(hipGetLastError(), "attn_shared merge launch");
}

}  // namespace

size_t attn_shared_ws_bytes(const k2t_ctx *ctx, const SharedShape &s, int prefix_len, int tail_len) {
    return ws_bytes_of(s, most_parts(ctx, s, prefix_len, tail_len));
}

void launch_attn_shared(k2t_ctx *ctx, hipStream_t st, int bits, const float *q, size_t q_stride, const SharedShape &s,
                        const k2t_kv_rows &prefix, const k2t_kv_rows &tail, float attn_scale, float *out, void *ws) {
    const Plan P = plan_of(ctx, s, prefix.cap ? prefix.len : 0, tail.cap ? tail.len : 0);
    SharedArgs A{};
    A.q = q;
    A.q_stride = (uint32_t)q_stride;
    A.per_group = (float)s.nkv / (float)s.nq;
    A.pre = prefix;
    A.tail = tail;
    A.beams = s.beams;
    A.nq = s.nq;
    A.nkv = s.nkv;
    A.group = s.nq / s.nkv;
    A.np = P.np;
    A.nt = P.nt;
    A.plen = P.plen;
    A.tlen = P.tlen;
    A.pgroups = P.pgroups;
    A.tgroups = P.tgroups;
    A.attn_scale = attn_scale;
    A.part = (float *)ws;
    A.stat = (float2 *)(A.part + part_slots(s, P.np + P.nt) * s.hd);
    A.out = out;
    const size_t units = (size_t)s.n_seq * s.nkv * P.np;
    const size_t pre = (units + 7) / 8 * 8 * P.pgroups, tails = (size_t)s.n_seq * s.beams * s.nkv * P.nt * P.tgroups;
    if (pre + tails > (size_t)1 << 23) throw Error(K2T_E_ARG, "too many rows, heads and positions in one call");
    A.units = (int)units;
    A.pre_items = P.np ? (int)pre : 0;
    if (s.hd == 128) launch_shared<128>(st, bits, A, s, P, A.pre_items + tails);
    else launch_shared<64>(st, bits, A, s, P, A.pre_items + tails);
}

}  // namespace k2t

using namespace k2t;

namespace {
SharedShape shared_shape(k2t_ctx *ctx, int n_seq, int beams, int nq, int nkv, int hd) {
    branch_arg(ctx != nullptr, "ctx is NULL");
    branch_arg(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    branch_arg(nq > 0 && nkv > 0 && nq % nkv == 0 && nq <= 1024, "n_heads must be a multiple of n_kv_heads, at most 1024");
    branch_arg(n_seq >= 0 && beams >= 1 && (size_t)n_seq * beams <= 65535, "n_seq * beams must be 0 .. 65535, beams >= 1");
    branch_arg((size_t)n_seq * beams * nq <= (size_t)1 << 22, "more than 2^22 query heads in one call");
    return SharedShape{n_seq, beams, nq, nkv, hd};
}
}  // namespace

extern "C" {

int32_t k2t_attn_shared_workspace(k2t_ctx *ctx, int32_t n_seq, int32_t beams, int32_t n_heads, int32_t n_kv_heads,
                                  int32_t head_dim, int32_t prefix_len, int32_t tail_len, size_t *bytes) {
    return branch_guard([&] {
        branch_arg(bytes != nullptr, "NULL argument");
        const SharedShape s = shared_shape(ctx, n_seq, beams, n_heads, n_kv_heads, head_dim);
        branch_arg(prefix_len >= 0 && prefix_len <= 1 << 24 && tail_len >= 0 && tail_len <= 1 << 24,
                   "prefix_len / tail_len out of range");
        *bytes = attn_shared_ws_bytes(ctx, s, prefix_len, tail_len);
    });
}

int32_t k2t_attn_shared(k2t_ctx *ctx, int32_t bits, const float *d_q, size_t q_stride, int32_t n_seq, int32_t beams,
                        int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, const k2t_kv_rows *prefix,
                        const k2t_kv_rows *tail, float attn_scale, float *d_out, void *d_ws, size_t ws_bytes) {
    return branch_guard([&] {
        const SharedShape s = shared_shape(ctx, n_seq, beams, n_heads, n_kv_heads, head_dim);
        branch_arg(prefix || tail, "neither a prefix nor a tail");
        // (the running maximum takes the largest dot product for the largest score)
        branch_arg(attn_scale >= 0.0f && attn_scale <= FLT_MAX, "attn_scale must be finite and not negative");
        for (const k2t_kv_rows *kv : {prefix, tail})
            if (kv) check_kv_rows(kv, bits, head_dim);
        if (n_seq == 0) return;
        branch_arg(d_q && d_out && d_ws, "NULL argument");
        const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
        branch_arg(q_stride >= (size_t)n_heads * head_dim && q_stride % 4 == 0 && q_stride < (size_t)1 << 31 &&
                       at(d_q) % 16 == 0,
                   "d_q must be 16-byte aligned, q_stride a multiple of 4, no smaller than a row, below 2^31");
        branch_arg((at(d_out) | at(d_ws)) % 16 == 0, "d_out and d_ws must be 16-byte aligned");
        const Plan P = plan_of(ctx, s, prefix ? prefix->len : 0, tail ? tail->len : 0);
        const size_t need = ws_bytes_of(s, P.np + P.nt);
        if (ws_bytes < need)
            throw Error(K2T_E_ARG, "the workspace holds " + std::to_string(ws_bytes) + " bytes, " +
                                       std::to_string(need) + " are needed");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        launch_attn_shared(ctx, ctx->stream, bits, d_q, q_stride, s, prefix ? *prefix : k2t_kv_rows{},
                           tail ? *tail : k2t_kv_rows{}, attn_scale, d_out, d_ws);
    });
}

}  // extern "C"
