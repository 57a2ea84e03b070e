// The batched Hadamard KV cache of rows that continue one prompt: heads quantized into it at each
// row's position, read back, whole rows rearranged in place, and the positions that a row keeps moved together
// (include/k2t_hip.h, k2t_kv_rows).
//
// append: r = fwht64(signs x) / 8 per 64-block; int8: scale = max |r| / 127 over the head, code =
// round(r / scale); NF4: the block's codes c_i nearest to 127 r_i / max |r|, scale = bf16(sum r_i c_i /
// sum c_i^2), codes again with that scale. load: signs ifwht64(code scale). reorder: row r becomes row
// parent[r] below its length.
//
// What bounds them: 6 rows of 777 tokens, 4 heads x 128, int8 (24 MB each): append 7.8 us, load 6.4 us (3.1 and
// 3.7 TB/s); rows of 389 to 777 tokens, the two in a row, 36 MB in all: 12.8 us. Waves that start, load once,
// transform and end are the larger part; 515 tokens of 32 heads x 64, NF4: append 7.7 us (9.1 by the profiler's
// clock), its instructions (both roundings of every element, three quotients per block), load 4.1 us (4.5); 11.9 us
// in a row. One token of 4 rows: 2.2 us each, a launch. Sixteen lanes per block, four elements a lane, instead of a wave per head with one
// element a lane: 26.5 -> 15.2 us and, with the NF4 sums from LDS, 39.6 -> 12.7 us.
#include <float.h>
#include <math.h>

#include "k2t_branch.h"
#include "k2t_device.h"
#include "k2t_kv_dev.h"

namespace k2t {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct RowsArgs {
    const float *k, *v;
    float *ko, *vo;
    size_t row_stride;
    int ntok, nkv;
    const int *pos, *counts;
    k2t_kv_rows kv;
    uint32_t units;  // 64-blocks of a row's tokens: ntok * 2 * nkv * (hd / 64)
};

// The kernels below give every 64-block of a head to sixteen lanes, four consecutive elements each
// (butterflies_slice4: the bits of kv_store_kernel's one element per lane); the blocks of a head are
// neighbours.  Grid y: the row of the call.
//
// Block `u` of a row: token t, K or V, KV head; the head's place in the call and its cache slot.  False
// where the token does not exist or its position lies outside the cache.
struct BlockAt {
    size_t in, slot;
    int is_v, b;
};
template <int NB>
__device__ __forceinline__ bool block_at(const RowsArgs &A, uint32_t u, BlockAt &h) {
    const uint32_t heads = 2u * (uint32_t)A.nkv, hu = u / NB, t = hu / heads, hv = hu - t * heads;
    const int row = (int)blockIdx.y;
    h.b = (int)(u % NB);
    h.is_v = hv >= (uint32_t)A.nkv;
    const uint32_t head = h.is_v ? hv - A.nkv : hv;
    const long long p = (long long)A.pos[row] + t;
    h.in = ((size_t)row * A.ntok + t) * A.row_stride + (size_t)head * (64 * NB) + 64 * h.b;
    h.slot = ((size_t)row * A.nkv + head) * (size_t)A.kv.cap + (size_t)p;
    return u < A.units && (!A.counts || (int)t < A.counts[row]) && p >= 0 && p < A.kv.cap;
}

// Magnitude place p (0 .. 7) of the nearest codebook value, and nf4_nearest_idx from it (three levels of
// comparisons; a NaN takes the last place there as well).
__device__ __forceinline__ uint32_t nf4_place(float y) {
    const float a = fabsf(y);
    const bool c1 = !(a < 51.0f), c2 = !(a < (c1 ? 85.5f : 24.5f));
    const bool c3 = !(a < (c1 ? (c2 ? 111.5f : 66.5f) : (c2 ? 37.5f : 12.0f)));
    return (c1 ? 4u : 0u) + (c2 ? 2u : 0u) + (c3 ? 1u : 0u);
}
__device__ __forceinline__ uint32_t nf4_index(float y) {
    const uint32_t p = nf4_place(y);
    return y >= 0.0f ? 8u + p : 7u - p;
}
// The nearest codebook value itself.
__device__ __forceinline__ float nf4_nearest(float y) {
    const float m = (float)__builtin_amdgcn_perm(kNf4Cb3, kNf4Cb2, nf4_place(y) | 0x0C0C0C00u);
    return y >= 0.0f ? m : -m;
}

__device__ __forceinline__ float group_max(float v) {  // of sixteen lanes
    v = fmaxf(v, xchg1(v));
    v = fmaxf(v, xchg2(v));
    v = fmaxf(v, xchg4(v));
    return fmaxf(v, xchg8(v));
}

// Heads quantized into the cache: kv_store_kernel's arithmetic and bytes.
// NF4: the block's scale is num / den with num summed in element order, 64 dependent additions: a wave
// puts the terms of 4 TURNS blocks in LDS and as many lanes add one block each.
template <int NB, int BITS, int TURNS>
__global__ __launch_bounds__(256) void kv_append_kernel(RowsArgs A) {
    __shared__ __align__(16) float term[BITS == 4 ? 4 : 1][BITS == 4 ? 4 * TURNS : 1][68];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, sl = lane & 15u, lg = lane >> 4, wave = tid >> 6;
    BlockAt at[TURNS];
    bool live[TURNS];
    float v[TURNS][4];
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
        live[k] = block_at<NB>(A, (blockIdx.x * TURNS + k) * 16u + 4u * wave + lg, at[k]);
        const float4 f = live[k] ? *reinterpret_cast<const float4 *>((at[k].is_v ? A.v : A.k) + at[k].in + 4 * sl)
                                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        v[k][0] = f.x;
        v[k][1] = f.y;
        v[k][2] = f.z;
        v[k][3] = f.w;
    }
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
        const uint32_t sb = head_signs4<NB>(at[k].b, sl);
#pragma unroll
        for (int j = 0; j < 4; j++) v[k][j] = flip_sign(v[k][j], (sb >> j) & 1u) * 0.125f;
        butterflies_slice4(v[k], sl);
    }
    if constexpr (BITS == 8) {
#pragma unroll
        for (int k = 0; k < TURNS; k++) {
            float mx = group_max(fmaxf(fmaxf(fabsf(v[k][0]), fabsf(v[k][1])), fmaxf(fabsf(v[k][2]), fabsf(v[k][3]))));
            // (kv_store_head's maximum of a one-block head starts from zero: nothing but NaN is a head of zeros)
            mx = fmaxf(mx, NB > 1 ? xor_lane(mx, 16) : 0.0f);
            const bool tiny = mx <= FLT_EPSILON;
            const float inv = 127.0f / mx;
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) w |= (tiny ? 0u : (uint32_t)(int)rintf(v[k][j] * inv) & 0xFFu) << (8 * j);
            if (!live[k]) continue;
            int8_t *q = (int8_t *)(at[k].is_v ? A.kv.vq : A.kv.kq) + at[k].slot * (64 * NB) + 64 * at[k].b;
            *reinterpret_cast<uint32_t *>(q + 4 * sl) = w;
            if (sl == 0 && at[k].b == 0) ((float *)(at[k].is_v ? A.kv.vs : A.kv.ks))[at[k].slot] = tiny ? 0.0f : mx / 127.0f;
        }
    } else {
        float mx[TURNS], den[TURNS], num[TURNS];
#pragma unroll
        for (int k = 0; k < TURNS; k++) {
            mx[k] = group_max(fmaxf(fmaxf(fabsf(v[k][0]), fabsf(v[k][1])), fmaxf(fabsf(v[k][2]), fabsf(v[k][3]))));
            const float inv0 = 127.0f / mx[k];
            float4 t;
            float c[4], cc = 0.0f;  // (squares of codes: whole numbers below 2^24, any order)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                c[j] = nf4_nearest(v[k][j] * inv0);
                cc += c[j] * c[j];
            }
            t = make_float4(v[k][0] * c[0], v[k][1] * c[1], v[k][2] * c[2], v[k][3] * c[3]);
            *reinterpret_cast<float4 *>(&term[wave][4 * k + lg][4 * sl]) = t;
            cc += xchg1(cc);
            cc += xchg2(cc);
            cc += xchg4(cc);
            den[k] = cc + xchg8(cc);
        }
        __builtin_amdgcn_wave_barrier();
        float sum = 0.0f;
        const float *mine = term[wave][lane % (4 * TURNS)];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float4 t = *reinterpret_cast<const float4 *>(mine + 4 * i);
            sum += t.x;
            sum += t.y;
            sum += t.z;
            sum += t.w;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int k = 0; k < TURNS; k++) num[k] = __shfl(sum, 4 * k + (int)lg, kWave);
#pragma unroll
        for (int k = 0; k < TURNS; k++) {
            const float s_ref = (den[k] > 1e-12f && num[k] > 0.0f) ? num[k] / den[k] : mx[k] / 127.0f;
            const bool none = mx[k] < 1e-30f;
            const uint16_t sb = none ? 0 : f32_to_bf16_rne(s_ref);
            const float s_fin = __uint_as_float((uint32_t)sb << 16);
            const float inv = s_fin > 1e-30f ? 1.0f / s_fin : 0.0f;
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) w |= (none ? 8u : nf4_index(v[k][j] * inv)) << (8 * j);
            // byte h * 16 + i: element h * 32 + i low, h * 32 + 16 + i high, four slices further on
            const uint32_t hi = (uint32_t)xchg4((int)w);
            if (!live[k]) continue;
            uint8_t *q = (uint8_t *)(at[k].is_v ? A.kv.vq : A.kv.kq) + at[k].slot * (32 * NB) + 32 * at[k].b;
            if ((sl & 4u) == 0) *reinterpret_cast<uint32_t *>(q + 16 * (sl >> 3) + 4 * (sl & 3u)) = w | (hi << 4);
            if (sl == 0) ((uint16_t *)(at[k].is_v ? A.kv.vs : A.kv.ks))[at[k].slot * NB + at[k].b] = sb;
        }
    }
}

// The same positions read back: code * scale and ifwht64.  (Stored past L2, where heads of any number do not
// stay: 6 rows of 777 tokens, 4 heads x 128: 6.4 us and 7.6 with ordinary stores.)
template <int NB, int BITS, int TURNS>
__global__ __launch_bounds__(256) void kv_load_kernel(RowsArgs A) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, sl = lane & 15u, lg = lane >> 4, wave = tid >> 6;
    BlockAt at[TURNS];
    bool live[TURNS];
    uint32_t w[TURNS];
    float scale[TURNS];
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
        live[k] = block_at<NB>(A, (blockIdx.x * TURNS + k) * 16u + 4u * wave + lg, at[k]);
        w[k] = 0;
        scale[k] = 0.0f;
        if (!live[k]) continue;
        const void *q = at[k].is_v ? A.kv.vq : A.kv.kq, *s = at[k].is_v ? A.kv.vs : A.kv.ks;
        if constexpr (BITS == 8) {
            w[k] = *reinterpret_cast<const uint32_t *>((const int8_t *)q + at[k].slot * (64 * NB) + 64 * at[k].b + 4 * sl);
            scale[k] = ((const float *)s)[at[k].slot];
        } else {
            w[k] = *reinterpret_cast<const uint32_t *>((const uint8_t *)q + at[k].slot * (32 * NB) + 32 * at[k].b +
                                                       16 * (sl >> 3) + 4 * (sl & 3u));
            scale[k] = __uint_as_float((uint32_t)((const uint16_t *)s)[at[k].slot * NB + at[k].b] << 16);
        }
    }
    uint32_t t0, t1, u0, u1;
    nf4_xor_tables(kNf4Cb0, kNf4Cb1, kNf4Cb2, kNf4Cb3, t0, t1, u0, u1);
#pragma unroll
    for (int k = 0; k < TURNS; k++) {
        if constexpr (BITS == 4) w[k] = nf4_xlut(((sl & 4u) ? w[k] >> 4 : w[k]) & 0x0F0F0F0Fu, t0, t1, u0, u1);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = (float)(int8_t)((w[k] >> (8 * j)) & 0xFFu) * scale[k];
        butterflies_slice4(v, sl);
        const uint32_t sb = head_signs4<NB>(at[k].b, sl);
        if (!live[k]) continue;
        const f32x4 out = {flip_sign(v[0] * 0.125f, sb & 1u), flip_sign(v[1] * 0.125f, (sb >> 1) & 1u),
                           flip_sign(v[2] * 0.125f, (sb >> 2) & 1u), flip_sign(v[3] * 0.125f, sb >> 3)};
        __builtin_nontemporal_store(out, reinterpret_cast<f32x4 *>((at[k].is_v ? A.vo : A.ko) + at[k].in + 4 * sl));
    }
}

// A step's qkv rows of the engine's beam search: qkv_post_kernel with every row at position *pos_dev and
// K / V into the row's tail, at position *pos_dev - pos0.
__global__ __launch_bounds__(64) void beam_post_kernel(float *__restrict__ qkv, const float *__restrict__ bias,
                                                       const float *__restrict__ qn, const float *__restrict__ kn,
                                                       float eps, const float *__restrict__ rope,
                                                       const int *__restrict__ pos_dev, int pos0, int nq, int nkv, int hd,
                                                       int bits, k2t_kv_rows tail) {
    const uint32_t lane = threadIdx.x;
    const int head = blockIdx.x, row = blockIdx.y, nb = hd / 64, pos = pos_dev[0];
    float *h = qkv + ((size_t)row * (nq + 2 * nkv) + head) * hd;
    float v0, v1;
    head_post(h, head, nq, nkv, hd, bias, qn, kn, eps, rope, pos, lane, v0, v1);
    if (head < nq) {
        h[lane] = v0;
        if (nb > 1) h[64 + lane] = v1;
        return;
    }
    const bool is_k = head < nq + nkv;
    const int kvh = is_k ? head - nq : head - nq - nkv, t = pos - pos0;
    if (t < 0 || t >= tail.cap) return;
    const float r0 = fwht_lane(v0, 0, lane);
    const float r1 = nb > 1 ? fwht_lane(v1, 1, lane) : 0.0f;
    kv_store_head(r0, r1, nb, lane, bits, hd, ((size_t)row * nkv + kvh) * tail.cap + t,
                  (int8_t *)(is_k ? tail.kq : tail.vq), (float *)(is_k ? tail.ks : tail.vs));
}

// Rows of one (layer, sequence, KV head, K or V) rearranged in place.  A thread owns one column (the
// same T-sized piece of every row): it reads the column of every row that moves from its source row
// before it writes any, so no other thread or buffer is involved.
// Bound by bytes: 24 layers, 8 rows of 32 heads x 64, 200 positions, 256 MB read and written in 47 to 57 us
// (4.5 to 5.4 TB/s, which is the large copy's), 64 to 70 us with stores that go through L2, 114 us with
// 4-byte columns too. Up to 32 rows go through
// registers as 16-byte columns, 64 as 8-byte ones.
template <typename T, int NB>
__device__ __forceinline__ void move_column(T *col, size_t pitch, const int *par, int beams, const int *lens, int pos) {
    T v[NB];
    bool mv[NB];
#pragma unroll
    for (int r = 0; r < NB; r++) {
        const int p = r < beams ? par[r] : r;
        mv[r] = r < beams && p != r && p >= 0 && p < beams && pos < lens[p];
        if (mv[r]) v[r] = col[(size_t)p * pitch];
    }
#pragma unroll
    for (int r = 0; r < NB; r++)
        if (mv[r]) __builtin_nontemporal_store(v[r], col + (size_t)r * pitch);
}

struct ReorderArgs {
    k2t_kv_rows kv;
    const int *parents;
    int n_seq, beams, nkv, hd, bits;
    int code_bytes, scale_bytes;  // per slot
    int code_blocks;              // workgroups per (layer, sequence, head, K / V) on the codes
};

template <int NB, typename TC>
__global__ __launch_bounds__(256) void kv_reorder_kernel(ReorderArgs A) {
    __shared__ int par[kMaxBeams], lens[kMaxBeams];
    // grid x: ((layer * n_seq + seq) * nkv + head) * 2 + (K, V)
    const size_t g = blockIdx.x / 2;
    const int is_v = blockIdx.x & 1, head = (int)(g % A.nkv);
    const size_t ls = g / A.nkv;
    const int seq = (int)(ls % A.n_seq);
    if ((int)threadIdx.x < A.beams) {
        const int r = seq * A.beams + threadIdx.x;
        par[threadIdx.x] = A.parents[r] - seq * A.beams;
        lens[threadIdx.x] = A.kv.d_len ? min(A.kv.d_len[r], A.kv.len) : A.kv.len;
    }
    __syncthreads();
    const size_t slot0 = (ls * A.beams * A.nkv + head) * (size_t)A.kv.cap;  // row 0's slots of this head
    const size_t slots = (size_t)A.nkv * A.kv.cap;                          // from one row to the next
    if ((int)blockIdx.y < A.code_blocks) {
        const size_t c = (size_t)blockIdx.y * 256 + threadIdx.x, per = A.code_bytes / sizeof(TC);
        if (c >= per * A.kv.len) return;
        TC *q = (TC *)(is_v ? A.kv.vq : A.kv.kq) + slot0 * per;
        move_column<TC, NB>(q + c, slots * per, par, A.beams, lens, (int)(c / per));
        return;
    }
    const int pos = ((int)blockIdx.y - A.code_blocks) * 256 + (int)threadIdx.x;
    if (pos >= A.kv.len) return;
    void *s = is_v ? A.kv.vs : A.kv.ks;
    if (A.scale_bytes == 4)
        move_column<uint32_t, NB>((uint32_t *)s + slot0 + pos, slots, par, A.beams, lens, pos);
    else
        move_column<uint16_t, NB>((uint16_t *)s + slot0 + pos, slots, par, A.beams, lens, pos);
}

// Positions of one (layer, row, KV head, K or V) moved together: position p0 + j from p0 + keep[j], keep[j] >= j.
// Entries are taken in order, a chunk of them at a time: a chunk's sources are all read before its
// positions are written, and those that earlier chunks have written lie before every later source.
// What bounds it: bytes. 24 layers, 32 heads x 64, 3000 of 4000 positions (627 MB read and written): 105 to 124 us by where
// the buffers lie, 5 to 6 TB/s, partly from the Infinity Cache (143 with a chunk's stores before the next one's loads). Few
// heads: the chain of chunks (17 layers, 3 rows, 2 heads x 128, 6027 positions, 325 MB: 54 us; 124 in chunks of 128 one
// after another). 30 layers, 4 rows, 4 of 10 positions: 3.6 us, a launch.
constexpr int kKeepPieces = 4;  // of a thread and chunk

struct KeepArgs {
    k2t_kv_rows kv;
    const int *pos, *keep, *counts;
    size_t keep_stride;
    int n_keep, rows, nkv;
    int code_bytes, scale_bytes;  // per slot
};

// What a chunk moves: entries a .. of the list, kKeepPieces * THREADS / PER of them, each a slot of PER pieces of type T.
template <typename T, int PER, int THREADS>
struct KeepChunk {
    static constexpr int kEntries = kKeepPieces * THREADS / PER;
    T v[kKeepPieces];
    long long to[kKeepPieces];

    __device__ __forceinline__ void load(const T *base, const int *keep, long long p0, int cap, int a, int n) {
#pragma unroll
        for (int k = 0; k < kKeepPieces; k++) {
            const int g = (int)threadIdx.x + THREADS * k, j = a + g / PER;
            to[k] = -1;
            if (j >= n) continue;
            const int from = keep[j];
            const long long t = p0 + j, f = p0 + from;
            if (from <= j || t < 0 || f >= cap) continue;  // (from == j: it is there already)
            to[k] = t * PER + g % PER;
            v[k] = base[f * PER + g % PER];
        }
    }
    __device__ __forceinline__ void store(T *base) const {
#pragma unroll
        for (int k = 0; k < kKeepPieces; k++)
            if (to[k] >= 0) base[to[k]] = v[k];
    }
};

// A chunk is written once every wave has read it, and while the next one is read: that one's sources lie behind all
// that this one writes, and what it writes in turn is no source of this one any more.
template <typename T, int PER, int THREADS>
__device__ __forceinline__ void keep_slots(T *base, const int *keep, long long p0, int cap, int n) {
    using Chunk = KeepChunk<T, PER, THREADS>;
    Chunk now, next;
    now.load(base, keep, p0, cap, 0, n);
    for (int a = 0; a < n; a += Chunk::kEntries) {
        // (the loads themselves, not only their issue, come before any wave's stores)
#if defined(__HIP_DEVICE_COMPILE__)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#endif
        __syncthreads();
        next.load(base, keep, p0, cap, a + Chunk::kEntries, n);
        now.store(base);
        now = next;
    }
}

template <int CODE, int THREADS>  // bytes of a slot's codes
__global__ __launch_bounds__(THREADS) void kv_keep_kernel(const KeepArgs A) {
    // grid x: ((layer * rows + row) * nkv + head) * 2 + (K, V)
    const size_t g = blockIdx.x / 2;
    const int is_v = blockIdx.x & 1, row = (int)(g / A.nkv % A.rows);
    const int n = A.counts ? max(0, min(A.counts[row], A.n_keep)) : A.n_keep;
    const int *keep = A.keep + (size_t)row * A.keep_stride;
    const long long p0 = A.pos[row];
    const size_t slot = g * (size_t)A.kv.cap;
    if (blockIdx.y == 0) {
        keep_slots<u32x4, CODE / 16, THREADS>((u32x4 *)(is_v ? A.kv.vq : A.kv.kq) + slot * (CODE / 16), keep, p0, A.kv.cap, n);
        return;
    }
    void *s = is_v ? A.kv.vs : A.kv.ks;
    if (A.scale_bytes == 4) keep_slots<uint32_t, 1, THREADS>((uint32_t *)s + slot, keep, p0, A.kv.cap, n);
    else keep_slots<uint16_t, 1, THREADS>((uint16_t *)s + slot, keep, p0, A.kv.cap, n);
}

RowsArgs rows_args(const k2t_kv_rows &kv, size_t row_stride, int ntok, int nkv, int hd, const int *pos, const int *counts) {
    RowsArgs A{};
    A.row_stride = row_stride;
    A.ntok = ntok;
    A.nkv = nkv;
    A.pos = pos;
    A.counts = counts;
    A.kv = kv;
    A.units = (uint32_t)((size_t)ntok * 2 * nkv * (hd / 64));
    return A;
}

// Two blocks per sixteen lanes from this many on, where every SIMD has its waves anyway (8 x 1024
// tokens, 8 heads x 128, 262144 blocks: NF4 append 38.8 us and 42.8 with one, int8 load 18.9 and 20.2; 515
// tokens, 32 heads x 64, 32960 blocks: int8 append 4.6 and 4.3, NF4 append 7.8 and 7.7).
constexpr size_t kManyBlocks = 1 << 16;

template <int NB, int BITS, bool LOAD>
void launch_rows(hipStream_t st, const RowsArgs &A, int batch) {
    const bool many = (size_t)A.units * batch >= kManyBlocks;
    const dim3 grid((A.units + (many ? 31 : 15)) / (many ? 32 : 16), (unsigned)batch), block(256);
    if constexpr (LOAD) {
        if (many) hipLaunchKernelGGL((kv_load_kernel<NB, BITS, 2>), grid, block, 0, st, A);
        else hipLaunchKernelGGL((kv_load_kernel<NB, BITS, 1>), grid, block, 0, st, A);
    } else {
        if (many) hipLaunchKernelGGL((kv_append_kernel<NB, BITS, 2>), grid, block, 0, st, A);
        else hipLaunchKernelGGL((kv_append_kernel<NB, BITS, 1>), grid, block, 0, st, A);
    }
    hip_check(hipGetLastError(), LOAD ? "kv_load launch" : "kv_append launch");
}
template <bool LOAD>
void launch_rows_of(hipStream_t st, int bits, int hd, const RowsArgs &A, int batch) {
    if (bits == 8 && hd == 64) launch_rows<1, 8, LOAD>(st, A, batch);
    else if (bits == 8) launch_rows<2, 8, LOAD>(st, A, batch);
    else if (hd == 64) launch_rows<1, 4, LOAD>(st, A, batch);
    else launch_rows<2, 4, LOAD>(st, A, batch);
}

bool heads_aligned(const float *k, const float *v) {
    return (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0;
}

void check_heads_call(k2t_ctx *ctx, int bits, int batch, int ntok, int nkv, int hd, size_t row_stride,
                      const void *d_pos, const k2t_kv_rows *kv) {
    branch_arg(ctx != nullptr && kv != nullptr, "NULL argument");
    branch_arg(batch >= 0 && batch <= 65535 && ntok >= 0 && nkv > 0 && nkv <= 1024,
               "batch must be 0 .. 65535, ntok >= 0, n_kv_heads 1 .. 1024");
    check_kv_rows(kv, bits, hd);
    branch_arg((size_t)batch * ntok * nkv <= (size_t)1 << 24, "more than 2^24 heads in one call");
    branch_arg(row_stride >= (size_t)nkv * hd && row_stride % 4 == 0,
               "row_stride is smaller than a row's heads, or no multiple of 4");
    branch_arg(batch == 0 || ntok == 0 || d_pos != nullptr, "d_pos is NULL");
}

}  // namespace

void check_kv_rows(const k2t_kv_rows *kv, int bits, int hd) {
    branch_arg(bits == 4 || bits == 8, "KV bits must be 4 or 8");
    branch_arg(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    branch_arg(kv->kq && kv->ks && kv->vq && kv->vs, "a cache pointer is NULL");
    branch_arg(kv->cap >= 1 && kv->cap <= 1 << 24, "cap out of range");
    branch_arg(kv->len >= 0 && kv->len <= kv->cap, "len must be 0 .. cap");
    const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
    branch_arg((at(kv->kq) | at(kv->vq)) % 16 == 0, "kq and vq must be 16-byte aligned");
    const uintptr_t scale = bits == 8 ? 4 : hd / 32;
    branch_arg((at(kv->ks) | at(kv->vs)) % scale == 0, "ks and vs must be aligned to one slot's scales");
}

void launch_beam_post(hipStream_t st, float *qkv, const float *bias, const float *qn, const float *kn, float eps,
                      const float *rope, const int *pos_dev, int pos0, int nq, int nkv, int hd, int rows, int bits,
                      const k2t_kv_rows &tail) {
    hipLaunchKernelGGL(beam_post_kernel, dim3(nq + 2 * nkv, rows), dim3(64), 0, st, qkv, bias, qn, kn, eps, rope, pos_dev,
                       pos0, nq, nkv, hd, bits, tail);
    hip_check(hipGetLastError(), "beam_post launch");
}

void launch_kv_reorder(hipStream_t st, int bits, const k2t_kv_rows &kv, const int *parents, int n_layers, int n_seq,
                       int beams, int nkv, int hd) {
    ReorderArgs A{kv, parents, n_seq, beams, nkv, hd, bits, bits == 8 ? hd : hd / 2, bits == 8 ? 4 : hd / 32, 0};
    // pieces of 16 bytes up to 32 rows; 64 rows hold theirs in as many registers with 8 bytes
    const int piece = beams > 32 ? 8 : 16;
    A.code_blocks = (int)(((size_t)kv.len * (A.code_bytes / piece) + 255) / 256);
    const dim3 grid((unsigned)(2 * (size_t)n_layers * n_seq * nkv), (unsigned)(A.code_blocks + (kv.len + 255) / 256));
    if (beams <= 4) hipLaunchKernelGGL((kv_reorder_kernel<4, u32x4>), grid, dim3(256), 0, st, A);
    else if (beams <= 8) hipLaunchKernelGGL((kv_reorder_kernel<8, u32x4>), grid, dim3(256), 0, st, A);
    else if (beams <= 16) hipLaunchKernelGGL((kv_reorder_kernel<16, u32x4>), grid, dim3(256), 0, st, A);
    else if (beams <= 32) hipLaunchKernelGGL((kv_reorder_kernel<32, u32x4>), grid, dim3(256), 0, st, A);
    else hipLaunchKernelGGL((kv_reorder_kernel<64, u32x2>), grid, dim3(256), 0, st, A);
    hip_check(hipGetLastError(), "kv_reorder launch");
}

template <int THREADS>
static void launch_keep(dim3 grid, hipStream_t st, const KeepArgs &A) {
    if (A.code_bytes == 128) hipLaunchKernelGGL((kv_keep_kernel<128, THREADS>), grid, dim3(THREADS), 0, st, A);
    else if (A.code_bytes == 64) hipLaunchKernelGGL((kv_keep_kernel<64, THREADS>), grid, dim3(THREADS), 0, st, A);
    else hipLaunchKernelGGL((kv_keep_kernel<32, THREADS>), grid, dim3(THREADS), 0, st, A);
}

void launch_kv_keep(int cus, hipStream_t st, int bits, const k2t_kv_rows &kv, const int *pos, const int *keep, size_t keep_stride,
                    const int *counts, int n_keep, int n_layers, int rows, int nkv, int hd) {
    const KeepArgs A{kv, pos, keep, counts, keep_stride, n_keep, rows, nkv, bits == 8 ? hd : hd / 2, bits == 8 ? 4 : hd / 32};
    const dim3 grid((unsigned)(2 * (size_t)n_layers * rows * nkv), 2);
    // Sixteen waves, and chunks four times as long, where there are few workgroups or long lists (us, four waves and sixteen: 204
    // workgroups of heads x 128, 6027 entries 98 and 54; 384 of 3000 59 and 40; 768 of 3000 121 and 110; 1536 of heads x
    // 64 124 both; 256 of 150 to 400 the same; but 960 of 293 9.8 and 13.1, some 3000 of 400 46 and 52).  (A launch has fewer
    // than 2^32 threads in a direction: four million workgroups are of four waves.)
    if ((grid.x <= 2 * (unsigned)cus || n_keep >= 1024) && grid.x < 1u << 22) launch_keep<1024>(grid, st, A);
    else launch_keep<256>(grid, st, A);
    hip_check(hipGetLastError(), "kv_keep launch");
}

}  // namespace k2t

using namespace k2t;

extern "C" {

int32_t k2t_kv_append(k2t_ctx *ctx, int32_t bits, const float *d_k, const float *d_v, size_t row_stride,
                      int32_t batch, int32_t ntok, int32_t n_kv_heads, int32_t head_dim, const int32_t *d_pos,
                      const int32_t *d_counts, const k2t_kv_rows *kv) {
    return branch_guard([&] {
        check_heads_call(ctx, bits, batch, ntok, n_kv_heads, head_dim, row_stride, d_pos, kv);
        if (batch == 0 || ntok == 0) return;
        branch_arg(d_k && d_v, "NULL argument");
        branch_arg(heads_aligned(d_k, d_v), "d_k and d_v must be 16-byte aligned");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        RowsArgs A = rows_args(*kv, row_stride, ntok, n_kv_heads, head_dim, d_pos, d_counts);
        A.k = d_k;
        A.v = d_v;
        launch_rows_of<false>(ctx->stream, bits, head_dim, A, batch);
    });
}

int32_t k2t_kv_load(k2t_ctx *ctx, int32_t bits, const k2t_kv_rows *kv, int32_t batch, int32_t ntok,
                    int32_t n_kv_heads, int32_t head_dim, const int32_t *d_pos, const int32_t *d_counts, float *d_k,
                    float *d_v, size_t row_stride) {
    return branch_guard([&] {
        check_heads_call(ctx, bits, batch, ntok, n_kv_heads, head_dim, row_stride, d_pos, kv);
        if (batch == 0 || ntok == 0) return;
        branch_arg(d_k && d_v, "NULL argument");
        branch_arg(heads_aligned(d_k, d_v), "d_k and d_v must be 16-byte aligned");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        RowsArgs A = rows_args(*kv, row_stride, ntok, n_kv_heads, head_dim, d_pos, d_counts);
        A.ko = d_k;
        A.vo = d_v;
        launch_rows_of<true>(ctx->stream, bits, head_dim, A, batch);
    });
}

int32_t k2t_kv_reorder(k2t_ctx *ctx, int32_t bits, const k2t_kv_rows *kv, const int32_t *d_parents,
                       int32_t n_layers, int32_t n_seq, int32_t beams, int32_t n_kv_heads, int32_t head_dim) {
    return branch_guard([&] {
        branch_arg(ctx && kv && d_parents, "NULL argument");
        check_kv_rows(kv, bits, head_dim);
        branch_arg(n_layers >= 0 && n_seq >= 0 && n_kv_heads > 0 && n_kv_heads <= 1024,
                   "negative n_layers or n_seq, or n_kv_heads not 1 .. 1024");
        branch_arg(beams >= 1 && beams <= kMaxBeams, "beams must be 1 .. 64");
        branch_arg(n_seq <= 65535 && (size_t)n_layers * n_seq * n_kv_heads <= (size_t)1 << 22,
                   "too many layers, sequences and heads");
        branch_arg((size_t)kv->len * head_dim <= (size_t)1 << 26, "len too large");
        if (n_layers == 0 || n_seq == 0 || beams == 1 || kv->len == 0) return;
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        launch_kv_reorder(ctx->stream, bits, *kv, d_parents, n_layers, n_seq, beams, n_kv_heads, head_dim);
    });
}

int32_t k2t_kv_keep(k2t_ctx *ctx, int32_t bits, const k2t_kv_rows *kv, const int32_t *d_pos, const int32_t *d_keep,
                    size_t keep_stride, const int32_t *d_counts, int32_t n_keep, int32_t n_layers, int32_t rows,
                    int32_t n_kv_heads, int32_t head_dim) {
    return branch_guard([&] {
        branch_arg(ctx && kv, "NULL argument");
        check_kv_rows(kv, bits, head_dim);
        branch_arg(n_layers >= 0 && rows >= 0 && rows <= 65535 && n_kv_heads > 0 && n_kv_heads <= 1024,
                   "negative n_layers, rows not 0 .. 65535, or n_kv_heads not 1 .. 1024");
        branch_arg((size_t)n_layers * rows <= (size_t)1 << 22 && (size_t)n_layers * rows * n_kv_heads <= (size_t)1 << 22,
                   "too many layers, rows and heads");
        branch_arg(n_keep >= 0 && n_keep <= 1 << 24 && keep_stride >= (size_t)n_keep && keep_stride < (size_t)1 << 40,
                   "n_keep must be 0 .. 2^24, keep_stride no smaller");
        if (n_layers == 0 || rows == 0 || n_keep == 0) return;
        branch_arg(d_pos && d_keep, "NULL argument");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        launch_kv_keep(ctx->num_cus, ctx->stream, bits, *kv, d_pos, d_keep, keep_stride, d_counts, n_keep, n_layers, rows, n_kv_heads,
                       head_dim);
    });
}

}  // extern "C"
