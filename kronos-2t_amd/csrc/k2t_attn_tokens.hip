// Attention of a block of tokens of every row of a batch over the row's Hadamard cache (k2t_attn_tokens): prompts
// (causal) and trees of drafted tokens (a mask), int8 or NF4, plain or grouped heads.
//
// For token t and q head h, over the positions p that t sees:
//   s_p = scale_q scale_k[p] (codes_q . codes_k[p]) attn_scale,  w_p = exp(s_p - max s),
//   out = ifwht64( sum_p w_p scale_v[p] codes_v[p] / sum_p w_p ).
// A row's tokens and the q heads of a KV head are the columns of matrix products against the same K and V
// (k2t_attn_tile.h); column c is head c % group of token c / group.
//
// Few columns (short drafts, single tokens): the waves of a workgroup share 16 or 32 columns and take tiles of 32
// positions in turn, K and V from memory to registers (tokens_few_kernel).  Many: eight waves have 16 columns each, and
// a tile of positions is brought to LDS once for all of them, V as the f16 operand itself, so that its conversion is shared
// too (tokens_block_kernel).  Where that leaves CUs without a workgroup (tokens_block_kernel: without a second one),
// positions are cut into parts, which a second kernel joins.
//
// What bounds it (passes in a row, by events; kernels are longer under the profiler).
// 8192 tokens from the start, 32 / 4 heads x 128, int8: 780 to 865 us by the card, 0.55 TFLOP that count at 0.7 PFLOP/s.  The
// matrix cores and the power they draw (the core's clock is down at 2.0 GHz): outputs are done twice, for a weight's two
// pieces, and all products would take 555 us at the rate of a large one (1.24 PFLOP/s f16, int8 twice that).  68 us are the
// ends of items, queries and outputs (268 MB).  6 prompts of 389 to 777 tokens, 32 heads x 64: 38 to 41 us, the ends half of them;
// 6 of 777, 32 / 8 x 128, NF4: 96 to 102.  Chunks of a prompt behind a context: NF4's lookups, the ends, the join (515 tokens behind
// 4100, 32 / 8 x 128, NF4: 107 to 111 us; under the profiler 113 and 15 of join).  Drafts behind a context: latencies at two
// waves per SIMD, and what one CU loads at a time (64 tokens behind 12000, 32 / 4 x 128: 34 to 37 us, under the profiler 35
// and 5 of join; 8 x 13 behind 2100, 32 / 8 x 128, NF4: 24).  Short drafts: a launch, a few tiles and the transforms (10
// tokens behind 300, 9 / 3 x 64: 5.9 us).  Work is cut by the cache's len, not by what rows hold: with len 32768, 64 single tokens
// behind 2000 take 51 us for 45.5, the 8 x 13 39.5 for 24.5, prompts of 777 the same 84 to 88.
#include <float.h>
#include <math.h>

#include <algorithm>

#include "k2t_attn_tile.h"
#include "k2t_branch.h"

namespace k2t {

namespace {

constexpr int kMaxTree = 64;

struct TokensArgs : ColumnArgs {
    int ntok, nkv;
    const int *pos, *counts;
    const uint64_t *sees;
    k2t_kv_rows kv;
    int plen;          // positions of a part; of a tile of tokens_block_kernel's
    int cgs, units;    // column groups of a row; (row, KV head, part), of tokens_block_kernel (row, KV head)
    int tiles, chunk;  // tokens_block_kernel: tiles of an item's positions, and of a workgroup's (0: uncut)
};

// A row of the call: how many tokens it has, the position of its first, and how many positions its last one sees.
struct Row {
    int count, start, end;
};
__device__ __forceinline__ int clamp_pos(const TokensArgs &A, long long p) {
    return (int)max(0ll, min(p, (long long)A.kv.len));
}
__device__ __forceinline__ Row row_of(const TokensArgs &A, int row) {
    Row R;
    R.count = A.counts ? max(0, min(A.counts[row], A.ntok)) : A.ntok;
    R.start = A.pos[row];
    R.end = R.count ? clamp_pos(A, (long long)R.start + R.count) : 0;
    return R;
}
// What token t sees: positions below `limit` and, of the block's tokens j (at positions start + j), those of `bits`.
struct Sees {
    int limit;
    uint64_t bits;
};
__device__ __forceinline__ Sees sees_of(const TokensArgs &A, const Row &R, int row, int t) {
    if (!A.sees) return Sees{clamp_pos(A, (long long)R.start + t + 1), 0};
    // tokens that the row has, at positions of the cache
    const long long lo = max(0ll, -(long long)R.start), hi = min((long long)R.count, (long long)A.kv.len - R.start);
    uint64_t m = hi <= lo ? 0 : (hi >= 64 ? ~0ull : (1ull << hi) - 1) & ~(lo >= 64 ? ~0ull : (1ull << lo) - 1);
    return Sees{clamp_pos(A, R.start), A.sees[(size_t)row * A.ntok + t] & m};
}
// How many positions the tokens up to t (of a tree: any) see at most.
__device__ __forceinline__ int reach(const TokensArgs &A, const Row &R, int t) {
    return A.sees ? R.end : clamp_pos(A, (long long)R.start + t + 1);
}

// What NQ columns of a lane see of the 32 positions from p0 on.
template <int NQ>
struct Seen {
    int limit[NQ], least;  // least: of all of the wave's columns
    uint64_t bits[NQ];
    int start;
    int p0, lg;
    __device__ __forceinline__ bool whole() const { return p0 + kTile <= least; }
    __device__ __forceinline__ uint32_t counts(int a) const {
        // bits p - p0 of 32 positions: those below the limit, and the block's tokens from position start on
        const int under = limit[a] - p0, at = start - p0;
        uint32_t m = under <= 0 ? 0u : under >= 32 ? ~0u : (1u << under) - 1u;
        m |= at >= 32 || at <= -64 ? 0u : at >= 0 ? (uint32_t)bits[a] << at : (uint32_t)(bits[a] >> -at);
        m >>= 4 * lg;
        return (m & 0xFu) | (m >> 12 & 0xF0u);
    }
    // Columns c0 + 16 a + li of an item whose last column is c1 (those behind it repeat it).
    __device__ __forceinline__ void set(const TokensArgs &A, const Row &R, int row, int c0, int c1, uint32_t li) {
        start = R.start;
        least = 1 << 30;
#pragma unroll
        for (int a = 0; a < NQ; a++) {
            const Sees s = sees_of(A, R, row, (int)column(A, min(c0 + 16 * a + (int)li, c1)).row);
            limit[a] = s.limit;
            bits[a] = s.bits;
            least = min(least, s.limit);
        }
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) least = min(least, xor_lane(least, m));
        least = __builtin_amdgcn_readfirstlane(least);
    }
};

// Few columns: an item is (row, KV head, part, 16 NQ columns).  Launch bounds: three waves to a SIMD where one tile of columns of
// 128 or two of 64 leave the registers for it (by itself the compiler takes 2 to 10 more for some and leaves two).
template <int HD, int BITS, int NQ, bool WHOLE, int WAVES>
__global__ __launch_bounds__(64 * WAVES, HD * NQ <= 128 ? 3 : 2) void tokens_few_kernel(const TokensArgs A) {
    __shared__ Shared<HD, NQ, WAVES> sh;
    const uint32_t lane = threadIdx.x & 63u;
    const int unit = (int)blockIdx.x % A.units, cg = A.cgs - 1 - (int)blockIdx.x / A.units;
    const int rh = unit / A.parts, head = rh % A.nkv, row = rh / A.nkv;
    const Row R = row_of(A, row);
    Item I;
    I.part = unit % A.parts;
    I.col0 = 16 * NQ * cg;
    I.n = min(16 * NQ, R.count * A.group - I.col0);
    if (I.n <= 0) return;
    const int t0 = I.part * A.plen, last = I.col0 + I.n - 1;
    I.kv[0] = I.kv[1] = A.kv;
    I.slot[0] = I.slot[1] = ((size_t)row * A.nkv + head) * (size_t)A.kv.cap + t0;
    I.len[0] = min(reach(A, R, (int)column(A, last).row) - t0, A.plen);
    I.len[1] = 0;
    I.row0 = row * A.ntok;
    I.head0 = head * A.group;
    if (I.len[0] <= 0) {
        if constexpr (WHOLE) {  // nothing to see
            for (int i = (int)threadIdx.x; i < I.n * HD; i += 64 * WAVES) {
                const Column c = column(A, I.col0 + i / HD);
                A.out[((size_t)(I.row0 + c.row) * A.nq + I.head0 + c.head) * HD + i % HD] = 0.0f;
            }
        }
        return;
    }
    Seen<NQ> seen;
    seen.set(A, R, row, I.col0, last, lane & 15u);
    seen.lg = (int)(lane >> 4);
    const auto hide = [&](int i, auto &t, auto &vs) {
        seen.p0 = t0 + kTile * i;
        if (!seen.whole()) hide_tile<false>(t, vs, [&](int a) { return seen.counts(a); });
    };
    const auto any = [&](int c) {
        const Sees s = sees_of(A, R, row, (int)column(A, c).row);
        return s.limit > 0 || s.bits != 0;
    };
    attend<HD, BITS, NQ, WHOLE>(A, I, hide, any, sh);
}

// ---- many columns
// Eight waves of sixteen columns share a tile: four, and waves of 32 columns, are slower at every size (8192 tokens, 32 / 4 x
// 128: 905 and 802 us, 780 with eight), sixteen the same on long prompts and slower on others.
constexpr int kBlockWaves = 8;

template <int HD, int BITS>
struct BlockTile {
    static constexpr int P = 8192 / HD, S = P / kTile, DB = HD / 16, SN = TileK<HD, BITS>::SN;  // positions; subtiles of 32
    __align__(16) uint8_t k[P * HD];      // int8 rows of HD / 16 pieces, pieces permuted (k_at)
    uint4 v[S][DB][64];                   // the f16 operand of (32 positions, 16 dimensions), as lanes read it
    __align__(16) float ks[P][SN], vs[P][SN];  // vs: V scales times kLift

    // Piece c of row r: eight lanes that read the same piece of eight rows find them in different banks.
    static __device__ __forceinline__ int k_at(int r, int c) {
        return 16 * (r * (HD / 16) + (c ^ (HD == 128 ? r & 7 : r >> 1 & 3)));
    }
};

// A tile on its way from memory, in a portion for each of eight waves: 64 pieces of K; of V, of subtile s and its half j the
// words of four output tiles g, for positions 4 lg + i; one position's K or V scales.
template <int HD, int BITS>
struct BlockLoad {
    using T = BlockTile<HD, BITS>;
    static constexpr int RB = BITS == 8 ? HD : HD / 2, PC = HD / 16, KP = RB / PC;
    uint32_t k[KP / 4], v[4], scale;
    uint32_t tid;

    // Portion of V: subtile, tile group, half.
    static __device__ __forceinline__ void portion(int wave, int &s, int &g, int &j) {
        s = HD == 128 ? wave >> 2 : wave >> 1;
        g = HD == 128 ? wave >> 1 & 1 : 0;
        j = wave & 1;
    }
    // Positions p0 .. of a row's and head's slots from `base` on.  Past the cache's end the last of them, cap - 1, is repeated;
    // up to there, what lies behind the row's positions is loaded and hidden with all that a column does not see.
    __device__ __forceinline__ void load(const k2t_kv_rows &kv, size_t base, int p0) {
        const uint32_t li = tid & 15u, lg = tid >> 4 & 3u;
        const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
        p0 = min(p0, kv.cap - 1);
        const uint8_t *kq = (const uint8_t *)kv.kq + (base + p0) * RB, *vq = (const uint8_t *)kv.vq + (base + p0) * RB;
        // (a wave takes K scales or V scales, or none)
        const bool is_v = wave >= T::P / 64;
        constexpr int SB = BITS == 8 || HD == 128 ? 4 : 2;
        const uint8_t *sc = (const uint8_t *)(is_v ? kv.vs : kv.ks) + (base + p0) * SB;
        const uint32_t at = tid % T::P;
        const bool inside = p0 + T::P <= kv.cap;  // (one offset per lane and immediate ones from it)
        const uint32_t left = kv.cap - 1 - p0;
        const uint32_t off = inside ? tid * KP : min(tid / PC, left) * RB + KP * (tid % PC);
        if constexpr (BITS == 8) {
            const uint4 w = *reinterpret_cast<const uint4 *>(kq + off);
            k[0] = w.x, k[1] = w.y, k[2] = w.z, k[3] = w.w;
        } else {
            const uint2 w = *reinterpret_cast<const uint2 *>(kq + off);
            k[0] = w.x, k[1] = w.y;
        }
        const auto word = [&](const uint8_t *from, uint32_t off) -> uint32_t {
            if constexpr (BITS == 8) return *reinterpret_cast<const uint32_t *>(from + off);
            else return *reinterpret_cast<const uint16_t *>(from + off);
        };
        int s, g, j;
        portion(wave, s, g, j);
        const uint32_t col = BITS == 8 ? HD / 16 * li + 4 * g : 32 * g + 2 * li;
        if (inside) {
            const uint8_t *from = vq + (size_t)(32 * s + 16 * j) * RB;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = word(from + i * RB, 4 * lg * RB + col);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = word(vq, min(32 * s + 16 * j + 4 * lg + i, left) * RB + col);
        }
        if (wave < 2 * T::P / 64) {
            const uint32_t to = (inside ? at : min(at, left)) * SB;
            if constexpr (SB == 4) scale = *reinterpret_cast<const uint32_t *>(sc + to);
            else scale = *reinterpret_cast<const uint16_t *>(sc + to);
        }
    }
    __device__ __forceinline__ void store(T &tile, const Nf4 &cb) const {
        const int tid = (int)this->tid, lane = tid & 63;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        *reinterpret_cast<v4i *>(tile.k + T::k_at(tid / PC, tid % PC)) = k_operand<BITS>(k, cb);
        uint32_t h[4][2];
        int s, g, j;
        portion(wave, s, g, j);
        v_halves(v_word<BITS>(v[0], cb), v_word<BITS>(v[1], cb), v_word<BITS>(v[2], cb), v_word<BITS>(v[3], cb), h);
#pragma unroll
        for (int u = 0; u < 4; u++) reinterpret_cast<uint2 *>(&tile.v[s][4 * g + u][lane])[j] = make_uint2(h[u][0], h[u][1]);
        if (tid < 2 * T::P) {
            float *p = tid < T::P ? tile.ks[tid] : tile.vs[tid - T::P];
#pragma unroll
            for (int n = 0; n < T::SN; n++) p[n] = TileK<HD, BITS>::scale(scale, n) * (tid < T::P ? 1.0f : kLift);
        }
    }
};

template <int HD, int BITS>
struct BlockShared {
    union {
        BlockTile<HD, BITS> tile[2];
        Queries<HD, 16> q[kBlockWaves];
        float o[kBlockWaves][16][HD + 4];
    };
    float beside[kBlockWaves][16];
    __device__ BlockShared() {}
};

// The workgroup that has an item's first tile, where items are cut.
__device__ __forceinline__ int first_chunk(const TokensArgs &A, int item) { return item * A.tiles / A.chunk; }

// Positions t0 .. t1 - 1 of an item: (row, KV head, 16 columns for each of eight waves).  CUT: a part of it, for the merge.
template <int HD, int BITS, bool CUT>
__device__ __forceinline__ void block_item(const TokensArgs &A, int item, int part, int t0, int t1, uint32_t tid, BlockShared<HD, BITS> &sh) {
    using T = BlockTile<HD, BITS>;
    constexpr int NB = HD / 64, DB = HD / 16, SN = T::SN, NQ = 1, W = 16;
    const uint32_t lane = tid & 63u, li = lane & 15u, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
    // (the last columns first: theirs are the longest items of a prompt)
    const int rh = item % A.units, cg = A.cgs - 1 - item / A.units;
    const int head = rh % A.nkv, row = rh / A.nkv;
    const Row R = row_of(A, row);
    const int col0 = W * kBlockWaves * cg, cols = R.count * A.group, n_all = min(W * kBlockWaves, cols - col0);
    if (n_all <= 0) return;
    const int end = min(reach(A, R, (int)column(A, col0 + n_all - 1).row), t1);
    const bool none = end <= t0;
    if (none && CUT) return;
    // this wave's columns; a wave without any repeats the last one and writes nothing
    const int c0 = min(col0 + W * wave, cols - 1), n = max(0, min(W, cols - col0 - W * wave)), c1 = min(c0 + W, cols) - 1;
    const size_t base = ((size_t)row * A.nkv + head) * (size_t)A.kv.cap;
    const float *q0 = A.q + (size_t)row * A.ntok * A.q_stride + (size_t)head * A.group * HD;
    Nf4 cb{};
    if constexpr (BITS == 4) nf4_xor_tables(kNf4Cb0, kNf4Cb1, kNf4Cb2, kNf4Cb3, cb.t0, cb.t1, cb.u0, cb.u1);
    BlockLoad<HD, BITS> next;
    next.tid = tid;
    if (!none) next.load(A.kv, base, t0);
    // queries: four 64-blocks of columns at a time
    constexpr int kTurns = W * NB / 4, kBatch = kTurns < 8 ? kTurns : 8;
    for (int k0 = 0; k0 < kTurns; k0 += kBatch) {
        float4 f[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const int u = 4 * (k0 + k) + (int)lg;
            const Column at = column(A, min(c0 + u / NB, c1));
            f[k] = *reinterpret_cast<const float4 *>(q0 + ((uint64_t)at.row * A.q_stride + at.head * HD + 64 * (u % NB) + 4 * li));
        }
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const int u = 4 * (k0 + k) + (int)lg, x = u / NB, b = u % NB;
            const Quant4 r = quantize_block<NB>(f[k], head_signs4<NB>(b, li), li, A.attn_scale);
            *reinterpret_cast<uint32_t *>(&sh.q[wave].q[x][64 * b + 4 * li]) = r.w;
            if (li == 0 && b == 0) sh.q[wave].qas[x] = r.qas;
        }
    }
    Seen<NQ> seen;
    seen.set(A, R, row, c0, c1, li);
    seen.lg = (int)lg;
    const int far = min(end, reach(A, R, (int)column(A, c1).row));  // the wave's own last position
    __syncthreads();
    v4i qb[NQ][NB];
    float qas[NQ];
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        qas[a] = sh.q[wave].qas[16 * a + li];
        query_operand<HD, BITS>(sh.q[wave].q[16 * a + li], lg, qb[a]);
        above_zero(qas[a], qb[a]);
    }
    State<HD, NQ, SN> S;
    S.clear(sh.beside[wave]);
    __syncthreads();
    const int tiles = none ? 0 : (end - t0 + T::P - 1) / T::P;
    if (!none) {
        next.store(sh.tile[0], cb);
        next.load(A.kv, base, t0 + T::P);
    }
    __syncthreads();
    for (int i = 0; i < tiles; i++) {
        const T &tile = sh.tile[i & 1];
        // the next tile into the other half, which all waves have left, and the one behind it on its way
        if (i + 1 < tiles) next.store(sh.tile[(i + 1) & 1], cb);
        next.load(A.kv, base, t0 + T::P * (i + 2));
#pragma unroll 1
        for (int s = 0; s < T::S; s++) {
            seen.p0 = t0 + T::P * i + kTile * s;
            if (seen.p0 >= far || n == 0) break;
            float t[NQ][2][4], vs[2][4][SN];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int r = kTile * s + 16 * j;
                v4i kf[NB];
                float ks[4][SN];
#pragma unroll
                for (int b = 0; b < NB; b++)
                    kf[b] = *reinterpret_cast<const v4i *>(tile.k + T::k_at(r + (int)li, 4 * b + (int)lg));
#pragma unroll
                for (int x = 0; x < SN; x++) {
                    const float4 a = *reinterpret_cast<const float4 *>(&tile.ks[r + 4 * lg][0] + 4 * x);
                    const float4 b = *reinterpret_cast<const float4 *>(&tile.vs[r + 4 * lg][0] + 4 * x);
                    const float fa[4] = {a.x, a.y, a.z, a.w}, fb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        ks[(4 * x + e) / SN][(4 * x + e) % SN] = fa[e];
                        vs[j][(4 * x + e) / SN][(4 * x + e) % SN] = fb[e];
                    }
                }
#pragma unroll
                for (int a = 0; a < NQ; a++) scores<BITS>(kf, qb[a], [&](int e, int b) { return ks[e][SN > 1 ? b : 0]; }, t[a][j]);
            }
            uint32_t ph[NQ][SN][4], pl[NQ][SN][4];
            if (!seen.whole()) hide_tile<true>(t, vs, [&](int a) { return seen.counts(a); });
            weights<HD, NQ, SN, true>(S, t, qas, vs, kTile, lg, ph, pl);
#pragma unroll
            for (int g = 0; g < DB / 4; g++) {
                constexpr int kBlocks = SN - 1;  // (NF4 blocks have weights of their own)
                v8h va[4];
#pragma unroll
                for (int u = 0; u < 4; u++) va[u] = __builtin_bit_cast(v8h, tile.v[s][4 * g + u][lane]);
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
        __syncthreads();
    }
    // outputs: 16 columns of every wave at a time, four of them by sixteen lanes each
#pragma unroll
    for (int a = 0; a < NQ; a++) {
        const float back[2] = {S.back(a, 0), S.back(a, SN - 1)};
        float l = S.l[a] * (back[0] * kLift);
        l += xor_lane(l, 16);
        l += xor_lane(l, 32);
#pragma unroll
        for (int b = 0; b < DB; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) sh.o[wave][li][out_dim<HD, BITS>(b, 4 * (int)lg + i)] = S.o[a][b][i] * back[b >= 4];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int x = 4 * k + (int)lg;
            const float L = __shfl(l, x, kWave), M = __shfl(S.m[a], x, kWave);
            const int c = min(c0 + 16 * a + x, c1);
            const Column to = column(A, c);
            const size_t pair = (size_t)(row * A.ntok + (int)to.row) * A.nq + head * A.group + to.head;
            const bool mine = 16 * a + x < n;
            bool any = true;
            if constexpr (!CUT) {
                const Sees s = sees_of(A, R, row, (int)to.row);
                any = s.limit > 0 || s.bits != 0;
            } else if (mine && li == 0) {
                A.stat[pair * A.parts + part] = make_float2(M, L);
            }
            const float inv = 1.0f / L;
            float *out = CUT ? A.part + (pair * A.parts + part) * HD : A.out + pair * HD;
#pragma unroll
            for (int d = 0; d < HD; d += 64) {
                const float4 f = *reinterpret_cast<const float4 *>(&sh.o[wave][x][d + 4 * li]);
                float v[4] = {f.x, f.y, f.z, f.w};
                if constexpr (!CUT) {
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = any ? v[e] * inv : 0.0f;
                    butterflies_slice4(v, li);
                    const uint32_t sb = head_signs4<NB>(d / 64, li);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[e] = flip_sign(v[e] * 0.125f, sb >> e & 1u);
                }
                if (mine) *reinterpret_cast<float4 *>(out + d + 4 * li) = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
        __syncthreads();
    }
}

// CUT: workgroups take `chunk` tiles each of all items' positions one after another, from wherever an item has got to, so
// that a few long items fill the card evenly (515 tokens behind 4100, 32 / 8 heads x 128 NF4, 136 items for 512 workgroups:
// 119.5 us, 130 in three equal parts of every item); an item has a part for every workgroup that comes to it.  Else a
// workgroup has an item.
// (128-dimensional NF4 heads spill three registers, before the loop over tiles and behind it.)
template <int HD, int BITS, bool CUT>
__global__ __launch_bounds__(64 * kBlockWaves, 4) void tokens_block_kernel(const TokensArgs A) {
    constexpr int P = BlockTile<HD, BITS>::P;
    __shared__ BlockShared<HD, BITS> sh;
    if constexpr (!CUT) {
        block_item<HD, BITS, CUT>(A, (int)blockIdx.x, 0, 0, A.kv.len, threadIdx.x, sh);
        return;
    }
    int item = (int)blockIdx.x * A.chunk / A.tiles, first = (int)blockIdx.x * A.chunk - item * A.tiles;
    int left = min(A.chunk, A.units * A.cgs * A.tiles - (int)blockIdx.x * A.chunk);
#pragma unroll 1
    do {
        const int n = min(A.tiles - first, left);
        // (as if not known before: lanes' offsets kept from item to item would not fit the registers)
        uint32_t tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        block_item<HD, BITS, CUT>(A, item, (int)blockIdx.x - first_chunk(A, item), P * first, P * (first + n), tid, sh);
        item++;
        first = 0;
        left -= n;
    } while (left > 0);
}

// Joins the parts of every token that its row has (merge_parts).  item: columns of a workgroup that wrote them.
template <int HD, int WAVES, int AHEAD>
__global__ __launch_bounds__(256) void tokens_merge_kernel(const TokensArgs A, int pairs, int item) {
    __shared__ float sum[WAVES > 1 ? WAVES : 1][HD];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int pair = WAVES == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x;
    if (pair >= pairs) return;
    const int token = pair / A.nq, row = token / A.ntok, t = token - row * A.ntok;
    const Row R = row_of(A, row);
    if (t >= R.count) return;
    const Sees s = sees_of(A, R, row, t);
    // an item wrote the parts that its last column reaches
    const int c = t * A.group + pair % A.nq % A.group, last = min(c / item * item + item, R.count * A.group) - 1;
    const bool any = s.limit > 0 || s.bits != 0;  // (else parts may hold the NaN of a query without positions)
    const int end = any ? reach(A, R, last / A.group) : 0;
    int live = (end + A.plen - 1) / A.plen;
    if (A.chunk && end > 0) {
        const int at = (A.cgs - 1 - c / item) * A.units + row * A.nkv + pair % A.nq / A.group;
        live = (at * A.tiles + (end - 1) / A.plen) / A.chunk - first_chunk(A, at) + 1;
    }
    merge_parts<HD, WAVES, AHEAD>(A, pair, [=](int i) { return i < live; }, any, sum);
}

struct TokensShape {
    int batch, ntok, nq, nkv, hd;
};

// How the work is cut.  block: tokens_block_kernel; else tokens_few_kernel, nq column tiles per workgroup of `waves`.
struct Plan {
    bool block;
    int nq, waves, cgs, parts, plen;  // plen: see TokensArgs
    int tiles, chunk;                 // (tokens_block_kernel)
    int item() const { return 16 * (block ? kBlockWaves : nq); }
};
// Items of one tile of columns (16) up to so much work: more workgroups, and a shorter way through each.  Measured on both
// sides (us, one tile and two): 300 tokens, 32 heads x 64: 2.8 rounds, 7.0 and 8.5; 8 x 13 tokens behind 2100, 32 / 8 x 128: 16.5
// rounds, 20.1 and 23.0; 777 tokens, 32 heads x 64: 18 rounds, 17.9 and 15.8; 64 tokens behind 12000, 32 / 4 x 128: 47 rounds, 51.7 and
// 37.3.  tokens_block_kernel: from three workgroups for two CUs on (1024 tokens, 32 / 4 x 128, one for a CU: 32.0 and 42.2 with it;
// 2048, two: 83.9 and 80.0; 8192, eight: 923 and 770).  For NF4, whose lookups it shares, also behind long contexts (512 tokens,
// 32 / 8 x 128, behind 0, 2100, 4100 and 16000 positions: 22, 68, 107 and 357, and 33, 80, 108 and 287 with it; int8 behind 4100
// and 16000: 72 and 234, 90 and 233; 515 tokens, NF4, behind 4100: 152 and 120), if there is one for four CUs (2 x 40 tokens
// behind 6100, one for eight: 37 and 46; 8 x 40, one for two: 136 and 106).  Never where half of its columns would be idle (64
// rows x 4, 8 and 16 tokens behind 2000, 32 / 8 x 128: 48, 54 and 95, and 65, 75 and 86; 16 rows x 30 and 60, 32 x 64: 32 and
// 54, and 52 and 57).  Columns that fill one tile take one (64 rows x 1 token behind 2000, 32 / 8 x 128, one and two: 45 and 48,
// NF4 41 and 53).
constexpr double kLittleWork = 17.0;
constexpr int kLeastPart = 256, kLongContext = 4000, kBlockColumns = 64;

// The most parts that an item is cut into where a call has so many: a workgroup for every CU; two of tokens_block_kernel,
// and a part more where an item begins and ends within other items' workgroups.
int most_parts(const k2t_ctx *ctx, bool block, size_t items, int len) {
    const size_t slots = (block ? 2 : 1) * (size_t)std::max(1, ctx->num_cus), longest = ((size_t)len + kLeastPart - 1) / kLeastPart;
    if (!block) return (int)std::max<size_t>(1, std::min(slots / std::max<size_t>(1, items), longest));
    return items >= slots || longest <= 1 ? 1 : (int)std::min((slots + items - 1) / items, longest) + 1;
}
// What a call cut into n parts of `each` positions costs, in microseconds: rounds of items on the card, the transforms at
// an item's ends, and the joining (3 us and its bytes).
double plan_cost(const TokensShape &s, const Plan &P, int bits, size_t cus, size_t items, int n, int each) {
    const double position = (P.block ? 0.025 : P.nq == 2 ? 0.0095 : 0.007) * (s.hd / 128.0) * (bits == 4 ? 1.4 : 1.0), ends = 5.0;
    // (a workgroup of tokens_block_kernel by itself waits at its barriers)
    const double rounds = (double)((items + cus - 1) / cus) * (P.block && items <= cus ? 1.15 : 1.0);
    const double join = n == 1 ? 0.0 : 3.0 + (double)s.batch * s.ntok * s.nq * n * s.hd * 1.5e-6;
    return rounds * each * position + (items > 2 * cus || (P.block && n > 1) ? std::max(rounds / 2, 2.0) : 1) * ends + join;
}
Plan plan_of(const k2t_ctx *ctx, const TokensShape &s, int bits, bool tree, int len) {
    const int cols = s.ntok * (s.nq / s.nkv);
    const size_t cus = (size_t)std::max(1, ctx->num_cus), heads = (size_t)s.batch * s.nkv;
    Plan P{};
    const auto items = [&](int item) { return std::max<size_t>(1, heads * ((cols + item - 1) / item)); };
    // rounds of 128 positions that items of one tile of columns make on a CU
    const int mean = tree ? len : std::max(len - s.ntok / 2, 1);
    const double work = (double)items(16) * mean / 128 / cus;
    const size_t blocks = items(16 * kBlockWaves);
    P.block = cols >= kBlockColumns && (2 * blocks >= 3 * cus || (bits == 4 && mean >= kLongContext && 4 * blocks >= cus));
    P.nq = cols <= 16 || work <= kLittleWork ? 1 : 2;
    P.cgs = (cols + P.item() - 1) / P.item();
    const size_t each_part = items(P.item());
    const int most = most_parts(ctx, P.block, each_part, len);
    // tokens_few_kernel: eight waves where a CU has one workgroup at most, and there is more than a tile for each of four
    // (8 x 13 tokens behind 2100, 32 / 8 x 128 NF4, one workgroup on a CU: 26.0 us and 31.4 with four waves; 64 tokens behind
    // 2000, 32 heads x 64, one on two: 13.1 and 17.8, 14.2 in parts; 300 tokens, 32 heads x 64, two on a CU: 13.2 and 7.1).
    P.waves = P.block ? kBlockWaves : each_part <= cus && len > 4 * kTile ? 8 : 4;
    P.parts = 1;
    P.plen = std::max(len, 1);
    if (P.block) {
        P.plen = 8192 / s.hd;
        P.tiles = std::max(1, (len + P.plen - 1) / P.plen);
        if (most == 1) return P;
        const size_t slots = 2 * cus, total = each_part * P.tiles;
        const int chunk = (int)std::max((total + slots - 1) / slots, (size_t)kLeastPart / P.plen);
        const int parts = (P.tiles + chunk - 2) / chunk + 1;
        const double cut = plan_cost(s, P, bits, cus, (total + chunk - 1) / chunk, parts, chunk * P.plen);
        if (parts > 1 && cut < plan_cost(s, P, bits, cus, each_part, 1, len)) {
            P.parts = parts;
            P.chunk = chunk;
        }
        return P;
    }
    double least = plan_cost(s, P, bits, cus, each_part, 1, len);
    for (int n = 2; n <= most; n++) {
        const int each = ((len + n - 1) / n + 127) / 128 * 128;
        if ((len + each - 1) / each < n) continue;  // (as many parts as a smaller n's)
        const double cost = plan_cost(s, P, bits, cus, each_part * n, n, each);
        if (cost >= least) continue;
        least = cost;
        P.parts = n;
        P.plen = each;
    }
    return P;
}
size_t part_slots(const TokensShape &s, int parts) { return (size_t)s.batch * s.ntok * s.nq * parts; }
size_t slot_bytes(int hd) { return hd * sizeof(float) + sizeof(float2); }
size_t ws_bytes_of(const TokensShape &s, int parts) { return parts == 1 ? 16 : part_slots(s, parts) * slot_bytes(s.hd); }
// At least that of every plan of up to so many rows, tokens and positions: for every kind of item, number of rows and of column
// groups, as many columns as they have and as many parts as they may be cut into (fewer where there are more items).
size_t most_ws_bytes(const k2t_ctx *ctx, const TokensShape &s, int len) {
    size_t most = 16;
    if (s.batch == 0) return most;
    const int cols = s.ntok * (s.nq / s.nkv);
    for (int item : {16, 32, 16 * kBlockWaves}) {
        const auto parts = [&](size_t items) { return most_parts(ctx, item == 16 * kBlockWaves, items, len); };
        for (int rows = 1; rows <= s.batch; rows++) {
            const size_t heads = (size_t)rows * s.nkv;
            if (parts(heads) <= 1) break;
            for (int cgs = 1; (cgs - 1) * item < cols; cgs++) {
                const int n = parts(heads * cgs);
                if (n <= 1) break;
                most = std::max(most, heads * std::min(cols, cgs * item) * n * slot_bytes(s.hd));
            }
        }
    }
    return most;
}

template <int HD, int BITS>
void launch_parts(hipStream_t st, const TokensArgs &A, const Plan &P) {
    const size_t items = (size_t)A.units * A.cgs;
    const dim3 grid((unsigned)(A.chunk ? (items * A.tiles + A.chunk - 1) / A.chunk : items)), block(64 * P.waves);
    if (P.block && P.parts > 1) hipLaunchKernelGGL((tokens_block_kernel<HD, BITS, true>), grid, block, 0, st, A);
    else if (P.block) hipLaunchKernelGGL((tokens_block_kernel<HD, BITS, false>), grid, block, 0, st, A);
    else if (P.parts > 1 && P.nq == 2) hipLaunchKernelGGL((tokens_few_kernel<HD, BITS, 2, false, 8>), grid, block, 0, st, A);
    else if (P.parts > 1) hipLaunchKernelGGL((tokens_few_kernel<HD, BITS, 1, false, 8>), grid, block, 0, st, A);
    else if (P.waves == 8 && P.nq == 2) hipLaunchKernelGGL((tokens_few_kernel<HD, BITS, 2, true, 8>), grid, block, 0, st, A);
    else if (P.waves == 8) hipLaunchKernelGGL((tokens_few_kernel<HD, BITS, 1, true, 8>), grid, block, 0, st, A);
    else if (P.nq == 2) hipLaunchKernelGGL((tokens_few_kernel<HD, BITS, 2, true, 4>), grid, block, 0, st, A);
    else hipLaunchKernelGGL((tokens_few_kernel<HD, BITS, 1, true, 4>), grid, block, 0, st, A);
    hip_check(hipGetLastError(), "attn_tokens launch");
}

template <int HD>
void launch_tokens(hipStream_t st, int bits, const TokensArgs &A, const TokensShape &s, const Plan &P) {
    if (bits == 8) launch_parts<HD, 8>(st, A, P);
    else launch_parts<HD, 4>(st, A, P);
    if (P.parts == 1) return;
    const int pairs = s.batch * s.ntok * s.nq;
    // Loads ahead: as many as there are parts, or nearly (515 tokens, 32 heads x 128, three parts: 13.7 us with sixteen, 11.5 with
    // four).  Four waves for a head's parts where there are many, and so few heads.
    if (P.parts > 16) hipLaunchKernelGGL((tokens_merge_kernel<HD, 4, 8>), dim3(pairs), dim3(256), 0, st, A, pairs, P.item());
    else if (P.parts > 8) hipLaunchKernelGGL((tokens_merge_kernel<HD, 1, 16>), dim3((pairs + 3) / 4), dim3(256), 0, st, A, pairs, P.item());
    else hipLaunchKernelGGL((tokens_merge_kernel<HD, 1, 8>), dim3((pairs + 3) / 4), dim3(256), 0, st, A, pairs, P.item());
    hip_check(hipGetLastError(), "attn_tokens merge launch");
}

TokensShape tokens_shape(k2t_ctx *ctx, int batch, int ntok, int nq, int nkv, int hd) {
    branch_arg(ctx != nullptr, "ctx is NULL");
    branch_arg(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    branch_arg(nq > 0 && nkv > 0 && nq % nkv == 0 && nq <= 1024, "n_heads must be a multiple of n_kv_heads, at most 1024");
    branch_arg(batch >= 0 && batch <= 65535 && ntok >= 0, "batch must be 0 .. 65535, ntok >= 0");
    branch_arg((size_t)batch * ntok * nq <= (size_t)1 << 22, "more than 2^22 query heads in one call");
    return TokensShape{batch, ntok, nq, nkv, hd};
}

}  // namespace

}  // namespace k2t

using namespace k2t;

extern "C" {

int32_t k2t_attn_tokens_workspace(k2t_ctx *ctx, int32_t batch, int32_t ntok, int32_t n_heads, int32_t n_kv_heads,
                                  int32_t head_dim, int32_t len, size_t *bytes) {
    return branch_guard([&] {
        branch_arg(bytes != nullptr, "NULL argument");
        const TokensShape s = tokens_shape(ctx, batch, ntok, n_heads, n_kv_heads, head_dim);
        branch_arg(len >= 0 && len <= 1 << 24, "len out of range");
        *bytes = most_ws_bytes(ctx, s, len);
    });
}

int32_t k2t_attn_tokens(k2t_ctx *ctx, int32_t bits, const float *d_q, size_t q_stride, int32_t batch, int32_t ntok,
                        int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, const int32_t *d_pos,
                        const int32_t *d_counts, const uint64_t *d_sees, const k2t_kv_rows *kv, float attn_scale,
                        float *d_out, void *d_ws, size_t ws_bytes) {
    return branch_guard([&] {
        const TokensShape s = tokens_shape(ctx, batch, ntok, n_heads, n_kv_heads, head_dim);
        branch_arg(kv != nullptr, "NULL argument");
        check_kv_rows(kv, bits, head_dim);
        branch_arg(!d_sees || ntok <= kMaxTree, "a tree has at most 64 tokens");
        // (the running maximum takes the largest dot product for the largest score)
        branch_arg(attn_scale >= 0.0f && attn_scale <= FLT_MAX, "attn_scale must be finite and not negative");
        if (batch == 0 || ntok == 0) return;
        branch_arg(d_q && d_out && d_ws && d_pos, "NULL argument");
        const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
        branch_arg(q_stride >= (size_t)n_heads * head_dim && q_stride % 4 == 0 && q_stride < (size_t)1 << 31 &&
                       at(d_q) % 16 == 0,
                   "d_q must be 16-byte aligned, q_stride a multiple of 4, no smaller than a token's heads, below 2^31");
        branch_arg((at(d_out) | at(d_ws)) % 16 == 0, "d_out and d_ws must be 16-byte aligned");
        branch_arg(at(d_sees) % 8 == 0, "d_sees must be 8-byte aligned");
        const Plan P = plan_of(ctx, s, bits, d_sees != nullptr, kv->len);
        const size_t need = ws_bytes_of(s, P.parts);
        if (ws_bytes < need)
            throw Error(K2T_E_ARG, "the workspace holds " + std::to_string(ws_bytes) + " bytes, " +
                                       std::to_string(need) + " are needed");
        // (with cgs at most as many as there are columns, or two workgroups for every CU: grids are within 2^23)
        const size_t units = (size_t)batch * n_kv_heads * (P.block ? 1 : P.parts);
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        TokensArgs A{};
        A.q = d_q;
        A.q_stride = (uint32_t)q_stride;
        A.per_group = (float)n_kv_heads / (float)n_heads;
        A.nq = n_heads;
        A.group = n_heads / n_kv_heads;
        A.attn_scale = attn_scale;
        A.parts = P.parts;
        A.part = (float *)d_ws;
        A.stat = (float2 *)(A.part + part_slots(s, P.parts) * s.hd);
        A.out = d_out;
        A.ntok = ntok;
        A.nkv = n_kv_heads;
        A.pos = d_pos;
        A.counts = d_counts;
        A.sees = d_sees;
        A.kv = *kv;
        A.plen = P.plen;
        A.cgs = P.cgs;
        A.units = (int)units;
        A.tiles = P.tiles;
        A.chunk = P.chunk;
        if (head_dim == 128) launch_tokens<128>(ctx->stream, bits, A, s, P);
        else launch_tokens<64>(ctx->stream, bits, A, s, P);
    });
}

}  // extern "C"
