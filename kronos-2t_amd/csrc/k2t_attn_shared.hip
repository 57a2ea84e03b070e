// Attention of one token of every row of a batch whose rows share their sequence's prefix cache and
// have a tail cache each (k2t_attn_shared): int8 or NF4 Hadamard caches, plain or grouped heads.
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
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kWaves = 4, kTile = 32;  // waves of a workgroup; positions of a wave's tile
constexpr float kLog2e = 1.44269504088896340736f;

struct SharedArgs {
    const float *q;
    size_t q_stride;
    k2t_kv_rows pre, tail;
    int beams, nq, nkv, group;    // group: q heads per KV head
    int np, nt, plen, tlen;       // prefix and tail parts, and their positions
    int pgroups, tgroups, units;  // column groups of a prefix / tail item; prefix units (sequence, KV head, part)
    int pre_items;
    float attn_scale;
    float *part;   // [row][head][np + nt][HD]
    float2 *stat;  // [row][head][np + nt]: maximum (in powers of two), sum
    float *out;
};

__device__ __forceinline__ int row_len(const k2t_kv_rows &kv, int row) {
    return kv.d_len ? max(0, min(kv.d_len[row], kv.len)) : kv.len;
}

// A wave's tile of 32 positions as its lanes load it (li = lane % 16, lg = lane / 16).
// K: rows 16 j + li, the 16 (NF4: 8) bytes lg of every 64-block.  V: positions 16 j + 4 lg + i, the
// HD / 16 bytes li of the row (NF4: two bytes of every block).  Scales: positions 16 j + 4 lg + i.
template <int HD, int BITS>
struct Tile {
    static constexpr int NB = HD / 64, KW = BITS == 8 ? 4 : 2, VW = BITS == 8 ? HD / 64 : NB;
    static constexpr int SN = BITS == 8 ? 1 : NB;  // scales per position
    uint32_t k[2][NB][KW];
    uint32_t v[2][4][VW];
    float ks[2][4][SN], vs[2][4][SN];
};

template <int HD, int BITS, bool PARTIAL>
__device__ __forceinline__ void load_tile(Tile<HD, BITS> &T, const k2t_kv_rows &kv, size_t base, int t0, int t1,
                                          uint32_t li, uint32_t lg) {
    constexpr int NB = HD / 64, RB = BITS == 8 ? HD : HD / 2;
    const auto clamp = [&](int t) { return PARTIAL ? min(t, t1 - 1) : t; };
    const uint8_t *kq = (const uint8_t *)kv.kq + base * RB, *vq = (const uint8_t *)kv.vq + base * RB;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint8_t *row = kq + (size_t)clamp(t0 + 16 * j + (int)li) * RB;
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if constexpr (BITS == 8) {
                const uint4 w = *reinterpret_cast<const uint4 *>(row + 64 * b + 16 * lg);
                T.k[j][b][0] = w.x;
                T.k[j][b][1] = w.y;
                T.k[j][b][2] = w.z;
                T.k[j][b][3] = w.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2 *>(row + 32 * b + 8 * lg);
                T.k[j][b][0] = w.x;
                T.k[j][b][1] = w.y;
            }
        }
        const int p0 = t0 + 16 * j + 4 * (int)lg;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint8_t *vr = vq + (size_t)clamp(p0 + i) * RB;
            if constexpr (BITS == 8) {
                if constexpr (HD == 128) {
                    const uint2 w = *reinterpret_cast<const uint2 *>(vr + 8 * li);
                    T.v[j][i][0] = w.x;
                    T.v[j][i][1] = w.y;
                } else {
                    T.v[j][i][0] = *reinterpret_cast<const uint32_t *>(vr + 4 * li);
                }
            } else {
#pragma unroll
                for (int b = 0; b < NB; b++) T.v[j][i][b] = *reinterpret_cast<const uint16_t *>(vr + 32 * b + 2 * li);
            }
        }
        if constexpr (BITS == 8) {
            const float *ks = (const float *)kv.ks + base, *vs = (const float *)kv.vs + base;
            if constexpr (PARTIAL) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    T.ks[j][i][0] = ks[clamp(p0 + i)];
                    T.vs[j][i][0] = vs[clamp(p0 + i)];
                }
            } else {
                const f4u a = *reinterpret_cast<const f4u *>(ks + p0), b = *reinterpret_cast<const f4u *>(vs + p0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    T.ks[j][i][0] = a[i];
                    T.vs[j][i][0] = b[i];
                }
            }
        } else {
            const uint16_t *ks = (const uint16_t *)kv.ks + base * NB, *vs = (const uint16_t *)kv.vs + base * NB;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const size_t at = (size_t)clamp(p0 + i) * NB + b;
                    T.ks[j][i][b] = __uint_as_float((uint32_t)ks[at] << 16);
                    T.vs[j][i][b] = __uint_as_float((uint32_t)vs[at] << 16);
                }
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

// Two floats as f16 pairs hi + lo: x = hi + lo within 2^-21 |x|.
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    typedef __fp16 v2hh __attribute__((ext_vector_type(2)));
    const v2hh h = __builtin_amdgcn_cvt_pkrtz(x0, x1);
    const v2hh l = __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], -1.0f, x0), fmaf((float)h[1], -1.0f, x1));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, l);
}

// What a wave carries from tile to tile for NQ tiles of 16 columns: lane li is a column.
template <int HD, int NQ>
struct State {
    v4f o[NQ][HD / 16];  // output tile b of column li, times 2^c
    float m[NQ], l[NQ];  // running maximum (powers of two); this lane's share of the sum
    uint32_t cexp;       // exponent of the V scales' common factor c (biased), 0: none yet
};

template <int HD, int BITS, int NQ, bool PARTIAL>
__device__ __forceinline__ void step(State<HD, NQ> &S, const Tile<HD, BITS> &T, const v4i (&qb)[NQ][HD / 64],
                                     const float (&qas)[NQ], const Nf4 &cb, int t0, int t1, uint32_t lg) {
    constexpr int NB = HD / 64, DB = HD / 16, SN = Tile<HD, BITS>::SN;
    // V scales times a power of two that brings the largest seen to 2^13 .. 2^14, so that the weights'
    // f16 pieces neither overflow nor lose bits; it changes when a larger one comes
    float vmax = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < SN; n++) vmax = fmaxf(vmax, fabsf(T.vs[j][i][n]));
    const uint32_t e_lane = __float_as_uint(vmax) >> 23;
    if (__any(e_lane > S.cexp)) {
        uint32_t e = e_lane;
        e = max(e, (uint32_t)xor_lane((int)e, 16));
        e = max(e, (uint32_t)xor_lane((int)e, 32));
        e = max(max(e, S.cexp), 27u);  // (scales below 2^-100 share its factor)
        if (S.cexp) {
            const float down = ldexpf(1.0f, (int)S.cexp - (int)e);
#pragma unroll
            for (int a = 0; a < NQ; a++)
#pragma unroll
                for (int b = 0; b < DB; b++) S.o[a][b] = S.o[a][b] * down;
        }
        S.cexp = e;
    }
    const float c = __uint_as_float((267u - S.cexp) << 23);
    uint32_t ph[NQ][SN][4], pl[NQ][SN][4];  // weights: pairs of positions, hi and lo pieces
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if constexpr (BITS == 8) {
                v4i d = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < NB; b++)
                    d = __builtin_amdgcn_mfma_i32_16x16x64_i8(k_operand<BITS>(T.k[j][b], cb), qb[a][b], d, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) s[j][i] = (float)d[i] * T.ks[j][i][0];
            } else {
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    const v4i z = {0, 0, 0, 0};
                    const v4i d = __builtin_amdgcn_mfma_i32_16x16x64_i8(k_operand<BITS>(T.k[j][b], cb), qb[a][b], z, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        s[j][i] = b == 0 ? (float)d[i] * T.ks[j][i][0] : fmaf((float)d[i], T.ks[j][i][b], s[j][i]);
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[j][i] = s[j][i] * qas[a];
                if (PARTIAL && t0 + 16 * j + 4 * (int)lg + i >= t1) s[j][i] = -INFINITY;
                top = fmaxf(top, s[j][i]);
            }
        if (__any(top > S.m[a])) {
            top = fmaxf(top, xor_lane(top, 16));
            top = fmaxf(top, xor_lane(top, 32));
            const float mn = fmaxf(S.m[a], top);
            const float corr = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(S.m[a] - mn);
            S.m[a] = mn;
            S.l[a] *= corr;
#pragma unroll
            for (int b = 0; b < DB; b++) S.o[a][b] = S.o[a][b] * corr;
        }
        const float m = S.m[a] == -INFINITY ? 0.0f : S.m[a];
        float p[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[j][i] = __builtin_amdgcn_exp2f(s[j][i] - m);
                S.l[a] += p[j][i];
            }
#pragma unroll
        for (int n = 0; n < SN; n++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i += 2)
                    split2(p[j][i] * (T.vs[j][i][n] * c), p[j][i + 1] * (T.vs[j][i + 1][n] * c), ph[a][n][2 * j + i / 2],
                           pl[a][n][2 * j + i / 2]);
    }
    // o^T += V^T w^T, four output tiles (one 4-byte word of V per position) at a time
#pragma unroll
    for (int g = 0; g < DB / 4; g++) {
        uint32_t h[2][4][2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[i] = T.v[j][i][g];
                if constexpr (BITS == 4)  // nibbles in the order 0, 2, 1, 3 of the byte pair
                    w[i] = nf4_xlut((w[i] & 0x0F0Fu) | ((w[i] & 0xF0F0u) << 12), cb.t0, cb.t1, cb.u0, cb.u1);
            }
            v_halves(w[0], w[1], w[2], w[3], h[j]);
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const v8h va = __builtin_bit_cast(v8h, make_uint4(h[0][t][0], h[0][t][1], h[1][t][0], h[1][t][1]));
#pragma unroll
            for (int a = 0; a < NQ; a++) {
                constexpr int last = SN - 1;
                const int n = g < last ? g : last;
                const v8h lo = __builtin_bit_cast(v8h, make_uint4(pl[a][n][0], pl[a][n][1], pl[a][n][2], pl[a][n][3]));
                const v8h hi = __builtin_bit_cast(v8h, make_uint4(ph[a][n][0], ph[a][n][1], ph[a][n][2], ph[a][n][3]));
                S.o[a][4 * g + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, lo, S.o[a][4 * g + t], 0, 0, 0);
                S.o[a][4 * g + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, hi, S.o[a][4 * g + t], 0, 0, 0);
            }
        }
    }
}

// Dimension of row x (0 .. 15) of output tile b.
template <int HD, int BITS>
__device__ __forceinline__ int out_dim(int b, int x) {
    if constexpr (BITS == 8) return HD == 128 ? 8 * x + b : 4 * x + b;
    // block b / 4, byte y of its 32 (tiles 0, 2: low nibbles 0, 1: see nf4_xlut's order above)
    const int t = b & 3, y = 2 * x + (t & 1), hi = t >> 1;
    return 64 * (b >> 2) + 32 * (y >> 4) + 16 * hi + (y & 15);
}

template <int HD>
struct Shared {
    __align__(16) int8_t qi[32][HD + 16];
    float qas[32];
    float wm[kWaves][16], wl[kWaves][16];
    __align__(16) float wo[kWaves][16][HD + 4];
};

// One item: `cols` columns (q heads of rows) from col0 on, 16 NQ at most, over positions [t0, t1) of
// one cache row.  Column x is head head0 + x % group of row row0 + x / group.
template <int HD, int BITS, int NQ>
__device__ __forceinline__ void item(const SharedArgs &A, Shared<HD> &sh, const k2t_kv_rows &kv, size_t base, int t0, int t1,
                                     int row0, int head0, int col0, int cols, int part) {
    constexpr int NB = HD / 64, DB = HD / 16;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const int n = min(16 * NQ, cols - col0);  // columns of this item
    // queries: sixteen lanes per 64-block, rotated and quantized with one scale per head
    uint64_t mask[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) mask[b] = __ballot(hadamard_sign_bit((uint64_t)b, lane) != 0u);
    for (int u = 4 * wave; u < 16 * NQ * NB; u += 4 * kWaves) {
        const int x = (u + (int)lg) / NB, b = (u + (int)lg) % NB;
        const int c = col0 + min(x, n - 1);
        const float *src = A.q + (size_t)(row0 + c / A.group) * A.q_stride + (size_t)(head0 + c % A.group) * HD;
        const float4 f = *reinterpret_cast<const float4 *>(src + 64 * b + 4 * li);
        float v[4] = {f.x, f.y, f.z, f.w};
        const uint32_t sb = (uint32_t)((NB > 1 && b ? mask[NB - 1] : mask[0]) >> (4u * li)) & 0xFu;
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
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w |= (tiny ? 0u : (uint32_t)(int)rintf(v[j] * inv) & 0xFFu) << (8 * j);
        *reinterpret_cast<uint32_t *>(&sh.qi[x][64 * b + 4 * li]) = w;
        if (li == 0 && b == 0) sh.qas[x] = tiny ? 0.0f : ((mx / 127.0f) * A.attn_scale) * kLog2e;
    }
    __syncthreads();
    v4i qb[NQ][NB];
    float qas[NQ];
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        const int8_t *r = sh.qi[16 * a + li];
        qas[a] = sh.qas[16 * a + li];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            if constexpr (BITS == 8) {
                const int4 w = *reinterpret_cast<const int4 *>(r + 64 * b + 16 * lg);
                qb[a][b] = v4i{w.x, w.y, w.z, w.w};
            } else {
                const int e = 64 * b + 32 * (int)(lg >> 1) + 8 * (int)(lg & 1u);
                const int2 x = *reinterpret_cast<const int2 *>(r + e), y = *reinterpret_cast<const int2 *>(r + e + 16);
                qb[a][b] = v4i{x.x, x.y, y.x, y.y};
            }
        }
    }
    Nf4 cb{};
    if constexpr (BITS == 4) nf4_xor_tables(kNf4Cb0, kNf4Cb1, kNf4Cb2, kNf4Cb3, cb.t0, cb.t1, cb.u0, cb.u1);
    State<HD, NQ> S;
    S.cexp = 0;
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        S.m[a] = -INFINITY;
        S.l[a] = 0.0f;
#pragma unroll
        for (int b = 0; b < DB; b++) S.o[a][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    for (int t = t0 + kTile * wave; t < t1; t += kTile * kWaves) {
        Tile<HD, BITS> T;
        if (t + kTile <= t1) {
            load_tile<HD, BITS, false>(T, kv, base, t, t1, li, lg);
            step<HD, BITS, NQ, false>(S, T, qb, qas, cb, t, t1, lg);
        } else {
            load_tile<HD, BITS, true>(T, kv, base, t, t1, li, lg);
            step<HD, BITS, NQ, true>(S, T, qb, qas, cb, t, t1, lg);
        }
    }
    // the waves' results joined in wave order, one tile of columns at a time
    const float back = S.cexp ? __uint_as_float((S.cexp - 13u) << 23) : 0.0f;  // 1 / c
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        if (16 * a >= n) break;
        float l = S.l[a];
        l += xor_lane(l, 16);
        l += xor_lane(l, 32);
        if (lg == 0) {
            sh.wm[wave][li] = S.m[a];
            sh.wl[wave][li] = l;
        }
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) sh.wo[wave][li][out_dim<HD, BITS>(b, 4 * (int)lg + i)] = S.o[a][b][i] * back;
        __syncthreads();
        const int x = (int)(tid >> 4), sl = (int)(tid & 15u);  // column, sixteenth of its dimensions
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; w++) M = fmaxf(M, sh.wm[w][x]);
        float e[kWaves], L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            e[w] = sh.wm[w][x] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sh.wm[w][x] - M);
            L = fmaf(sh.wl[w][x], e[w], L);
        }
        if (16 * a + x < n) {
            const int c = col0 + 16 * a + x;
            const size_t at = ((size_t)(row0 + c / A.group) * A.nq + head0 + c % A.group) * (A.np + A.nt) + part;
#pragma unroll
            for (int d = 0; d < HD; d += 64) {
                float4 r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWaves; w++) {
                    const float4 v = *reinterpret_cast<const float4 *>(&sh.wo[w][x][d + 4 * sl]);
                    r.x = fmaf(v.x, e[w], r.x);
                    r.y = fmaf(v.y, e[w], r.y);
                    r.z = fmaf(v.z, e[w], r.z);
                    r.w = fmaf(v.w, e[w], r.w);
                }
                *reinterpret_cast<float4 *>(A.part + at * HD + d + 4 * sl) = r;
            }
            if (sl == 0) A.stat[at] = make_float2(M, L);
        }
        __syncthreads();
    }
}

template <int HD, int BITS>
__global__ __launch_bounds__(64 * kWaves, 2) void shared_part_kernel(SharedArgs A) {
    __shared__ Shared<HD> sh;
    const int id = (int)blockIdx.x;
    if (id < A.pre_items) {
        // A unit's column groups read the same K / V: they get ids congruent mod 8, one XCD's.
        const int slot = id >> 3, unit = (id & 7) + 8 * (slot / A.pgroups), cg = slot % A.pgroups;
        if (unit >= A.units) return;
        const int part = unit % A.np, sk = unit / A.np, head = sk % A.nkv, seq = sk / A.nkv;
        const int t0 = part * A.plen, t1 = min(row_len(A.pre, seq), t0 + A.plen);
        if (t0 >= t1) return;
        item<HD, BITS, 2>(A, sh, A.pre, ((size_t)seq * A.nkv + head) * A.pre.cap, t0, t1, seq * A.beams, head * A.group,
                          32 * cg, A.beams * A.group, part);
        return;
    }
    int t = id - A.pre_items;
    const int cg = t % A.tgroups;
    t /= A.tgroups;
    const int part = t % A.nt;
    t /= A.nt;
    const int head = t % A.nkv, row = t / A.nkv;
    const int t0 = part * A.tlen, t1 = min(row_len(A.tail, row), t0 + A.tlen);
    if (t0 >= t1) return;
    item<HD, BITS, 1>(A, sh, A.tail, ((size_t)row * A.nkv + head) * A.tail.cap, t0, t1, row, head * A.group, 16 * cg, A.group,
                      A.np + part);
}

// One wave per (head, row): the parts that hold positions, in order, and ifwht64.
template <int HD>
__global__ __launch_bounds__(64) void shared_merge_kernel(SharedArgs A) {
    const uint32_t lane = threadIdx.x;
    const int head = blockIdx.x, row = blockIdx.y, n = A.np + A.nt;
    const int np = A.np ? (row_len(A.pre, row / A.beams) + A.plen - 1) / A.plen : 0;
    const int nt = A.nt ? (row_len(A.tail, row) + A.tlen - 1) / A.tlen : 0;
    const size_t at = ((size_t)row * A.nq + head) * n;
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int i = 0; i < np + nt; i++) {
        const size_t p = at + (i < np ? i : A.np + i - np);
        const float2 st = A.stat[p];
        const float mn = fmaxf(m, st.x), a = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float b = __builtin_amdgcn_exp2f(st.x - mn);
        l = fmaf(l, a, st.y * b);
        o0 = fmaf(o0, a, A.part[p * HD + lane] * b);
        if (HD > 64) o1 = fmaf(o1, a, A.part[p * HD + HD - 64 + lane] * b);
        m = mn;
    }
    const float inv = np + nt == 0 ? 0.0f : 1.0f / l;
    float *out = A.out + ((size_t)row * A.nq + head) * HD;
    out[lane] = ifwht_lane(o0 * inv, 0, lane);
    if (HD > 64) out[64 + lane] = ifwht_lane(o1 * inv, 1, lane);
}

// How the positions are cut into parts: enough workgroups for two on every CU, a tile per wave at
// least.
struct Plan {
    int np, plen, pgroups, nt, tlen, tgroups;
};
Plan plan_of(const k2t_ctx *ctx, const SharedShape &s, int prefix_len, int tail_len) {
    const int group = s.nq / s.nkv, least = kTile * kWaves;
    Plan P{};
    P.pgroups = (s.beams * group + 31) / 32;
    P.tgroups = (group + 15) / 16;
    const auto cut = [&](int len, int items, int &n, int &each) {
        if (len == 0) return;
        const int want = std::max(1, 2 * std::max(1, ctx->num_cus) / std::max(1, items));
        each = ((len + want - 1) / want + least - 1) / least * least;
        n = (len + each - 1) / each;
    };
    cut(prefix_len, s.n_seq * s.nkv * P.pgroups, P.np, P.plen);
    cut(tail_len, s.n_seq * s.beams * s.nkv * P.tgroups, P.nt, P.tlen);
    return P;
}
size_t part_slots(const SharedShape &s, const Plan &P) { return (size_t)s.n_seq * s.beams * s.nq * (P.np + P.nt); }

template <int HD>
void launch_shared(hipStream_t st, int bits, const SharedArgs &A, const SharedShape &s, size_t items) {
    const int rows = s.n_seq * s.beams;
    if (items) {
        if (bits == 8)
            hipLaunchKernelGGL((shared_part_kernel<HD, 8>), dim3((unsigned)items), dim3(64 * kWaves), 0, st, A);
        else
            hipLaunchKernelGGL((shared_part_kernel<HD, 4>), dim3((unsigned)items), dim3(64 * kWaves), 0, st, A);
        hip_check(hipGetLastError(), "attn_shared launch");
    }
    hipLaunchKernelGGL(shared_merge_kernel<HD>, dim3(s.nq, rows), dim3(64), 0, st, A);
    hip_check(hipGetLastError(), "attn_shared merge launch");
}

}  // namespace

size_t attn_shared_ws_bytes(const k2t_ctx *ctx, const SharedShape &s, int prefix_len, int tail_len) {
    const size_t slots = part_slots(s, plan_of(ctx, s, prefix_len, tail_len));
    return std::max<size_t>(16, slots * (s.hd * sizeof(float) + sizeof(float2)));
}

void launch_attn_shared(k2t_ctx *ctx, hipStream_t st, int bits, const float *q, size_t q_stride, const SharedShape &s,
                        const k2t_kv_rows &prefix, const k2t_kv_rows &tail, float attn_scale, float *out, void *ws) {
    const Plan P = plan_of(ctx, s, prefix.cap ? prefix.len : 0, tail.cap ? tail.len : 0);
    SharedArgs A{};
    A.q = q;
    A.q_stride = q_stride;
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
    A.stat = (float2 *)(A.part + part_slots(s, P) * s.hd);
    A.out = out;
    const size_t units = (size_t)s.n_seq * s.nkv * P.np;
    const size_t pre = (units + 7) / 8 * 8 * P.pgroups, tails = (size_t)s.n_seq * s.beams * s.nkv * P.nt * P.tgroups;
    if (pre + tails > (size_t)1 << 23) throw Error(K2T_E_ARG, "too many rows, heads and positions in one call");
    A.units = (int)units;
    A.pre_items = P.np ? (int)pre : 0;
    if (s.hd == 128) launch_shared<128>(st, bits, A, s, A.pre_items + tails);
    else launch_shared<64>(st, bits, A, s, A.pre_items + tails);
}

}  // namespace k2t

using namespace k2t;

namespace {
SharedShape shared_shape(k2t_ctx *ctx, int n_seq, int beams, int nq, int nkv, int hd) {
    branch_arg(ctx != nullptr, "ctx is NULL");
    branch_arg(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    branch_arg(nq > 0 && nkv > 0 && nq % nkv == 0 && nq <= 1024, "n_heads must be a multiple of n_kv_heads, at most 1024");
    branch_arg(n_seq >= 0 && beams >= 1 && (size_t)n_seq * beams <= 65535, "n_seq * beams must be 0 .. 65535, beams >= 1");
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
        for (const k2t_kv_rows *kv : {prefix, tail})
            if (kv) check_kv_rows(kv, bits, head_dim);
        if (n_seq == 0) return;
        branch_arg(d_q && d_out && d_ws, "NULL argument");
        const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
        branch_arg(q_stride >= (size_t)n_heads * head_dim && q_stride % 4 == 0 && at(d_q) % 16 == 0,
                   "d_q must be 16-byte aligned, q_stride a multiple of 4 and no smaller than a row");
        branch_arg((at(d_out) | at(d_ws)) % 16 == 0, "d_out and d_ws must be 16-byte aligned");
        const size_t need = attn_shared_ws_bytes(ctx, s, prefix ? prefix->len : 0, tail ? tail->len : 0);
        if (ws_bytes < need)
            throw Error(K2T_E_ARG, "the workspace holds " + std::to_string(ws_bytes) + " bytes, " +
                                       std::to_string(need) + " are needed");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        launch_attn_shared(ctx, ctx->stream, bits, d_q, q_stride, s, prefix ? *prefix : k2t_kv_rows{},
                           tail ? *tail : k2t_kv_rows{}, attn_scale, d_out, d_ws);
    });
}

}  // extern "C"
