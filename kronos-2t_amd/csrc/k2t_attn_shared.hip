// Attention of one token of every row of a batch whose rows share their sequence's prefix cache and
// have a tail cache each (k2t_attn_shared): int8 or NF4 Hadamard caches, plain or grouped heads.
//
// For row r and q head h, over the positions t of its sequence's prefix and then of its tail:
//   s_t = scale_q scale_k[t] (codes_q . codes_k[t]) attn_scale,  w_t = exp(s_t - max s),
//   out = ifwht64( sum_t w_t scale_v[t] codes_v[t] / sum_t w_t ).
// The rows of a sequence and the q heads of a KV head are columns of one matrix against the same K and
// V, so both products are matrix products (k2t_attn_tile.h).
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
// 12000 + 333 positions 35.3 to 36.5 us by the card (365 TFLOP/s); 3 sequences of 8 rows x 32 / 8 heads x 128, NF4, 4100 positions
// 19.0 us, a third of whose instructions look codes up; 4 rows x 9 / 3 heads x 64, 52 positions 5.2 us, a launch.
// References by products instead of scores cost NF4 heads of two blocks 2 to 3 % (a reference each: 19.9 and
// 20.3 us, 47.2 and 48.4 us with 64 rows), the others nothing where V scales are alike; with scales anywhere within
// 2^-2 .. 2^2 of each other references are raised more often (64 rows, int8: 35.4 and 36.5 us; 2^-8 .. 2^8: 38.6).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "k2t_attn_tile.h"
#include "k2t_branch.h"

namespace k2t {

namespace {

struct SharedArgs : ColumnArgs {
    k2t_kv_rows pre, tail;
    int beams, nkv;
    int np, nt, plen, tlen;       // prefix and tail parts, and their positions
    int pgroups, tgroups, units;  // column groups of a prefix / tail item; prefix units (sequence, KV head, part)
    int pre_items;
};

template <int HD, int BITS, int NQ>
__global__ __launch_bounds__(64 * kWaves, HD * NQ <= 128 ? 3 : 2) void shared_part_kernel(SharedArgs A) {
    __shared__ union U {
        Shared<HD, NQ> prefix;
        Shared<HD, 1> tail;
        __device__ U() {}
    } sh;
    const auto all = [](int) { return true; };
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
        attend<HD, BITS, NQ, false>(A, I, NoMask{}, all, sh.prefix);
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
    attend<HD, BITS, 1, false>(A, I, NoMask{}, all, sh.tail);
}

// Few positions: one workgroup per (row, KV head, 16 q heads) takes the prefix and the tail and writes
// the output; the prefix is read once per row, by so few bytes that a second launch costs more.
template <int HD, int BITS>
__global__ __launch_bounds__(64 * kWaves, 3) void shared_whole_kernel(SharedArgs A) {
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
    attend<HD, BITS, 1, true>(A, I, NoMask{}, [](int) { return true; }, sh);
}

// Joins the parts (merge_parts).
template <int HD, int WAVES>
__global__ __launch_bounds__(256) void shared_merge_kernel(SharedArgs A, int pairs) {
    __shared__ float sum[WAVES > 1 ? WAVES : 1][HD];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int pair = WAVES == 1 ? (int)blockIdx.x * 4 + wave : (int)blockIdx.x;
    if (pair >= pairs) return;
    const int row = pair / A.nq;
    const int np = A.np ? (row_len(A.pre, row / A.beams) + A.plen - 1) / A.plen : 0;
    const int nt = A.nt ? (row_len(A.tail, row) + A.tlen - 1) / A.tlen : 0;
    const auto live = [&](int i) { return i < A.np ? i < np : i - A.np < nt; };
    merge_parts<HD, WAVES>(A, pair, live, np + nt != 0, sum);
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
    A.parts = P.np + P.nt;
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
