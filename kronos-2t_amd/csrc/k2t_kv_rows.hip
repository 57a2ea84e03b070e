// The batched Hadamard KV cache of rows that continue one prompt: heads quantized into it at each
// row's position, read back, and whole rows rearranged in place (include/k2t_hip.h, k2t_kv_rows).
#include <float.h>
#include <math.h>

#include "k2t_branch.h"
#include "k2t_device.h"
#include "k2t_kv_dev.h"

namespace k2t {

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct RowsArgs {
    const float *k, *v;
    float *ko, *vo;
    size_t row_stride;
    int ntok, nkv, hd, bits;
    const int *pos, *counts;
    k2t_kv_rows kv;
    size_t row0;  // first cache row
    size_t units;  // heads of the call: batch * ntok * 2 * nkv
};

// Head `u` of a call: token (row, t), K or V, KV head; its cache slot, or false where the token does
// not exist or its position lies outside the cache.
struct HeadAt {
    size_t in, slot;
    int is_v;
};
__device__ __forceinline__ bool head_at(const RowsArgs &A, size_t u, HeadAt &h) {
    const int hv = (int)(u % (2u * A.nkv));
    const size_t tok = u / (2u * A.nkv);
    const int row = (int)(tok / A.ntok), t = (int)(tok % A.ntok);
    h.is_v = hv >= A.nkv;
    const int head = h.is_v ? hv - A.nkv : hv;
    if (A.counts && t >= A.counts[row]) return false;
    const long long p = (long long)A.pos[row] + t;
    if (p < 0 || p >= A.kv.cap) return false;
    h.in = tok * A.row_stride + (size_t)head * A.hd;
    h.slot = ((A.row0 + row) * A.nkv + head) * (size_t)A.kv.cap + (size_t)p;
    return true;
}

// One wave per head, one element (of each 64-block) per lane: kv_store_kernel's arithmetic.
__global__ __launch_bounds__(256) void kv_append_kernel(RowsArgs A) {
    const uint32_t lane = threadIdx.x & 63u;
    const size_t u = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    HeadAt h;
    if (u >= A.units || !head_at(A, u, h)) return;
    const float *x = (h.is_v ? A.v : A.k) + h.in;
    const int nb = A.hd / 64;
    const float r0 = fwht_lane(x[lane], 0, lane);
    const float r1 = nb > 1 ? fwht_lane(x[64 + lane], 1, lane) : 0.0f;
    kv_store_head(r0, r1, nb, lane, A.bits, A.hd, h.slot, (int8_t *)(h.is_v ? A.kv.vq : A.kv.kq),
                  (float *)(h.is_v ? A.kv.vs : A.kv.ks));
}

__global__ __launch_bounds__(256) void kv_load_kernel(RowsArgs A) {
    const uint32_t lane = threadIdx.x & 63u;
    const size_t u = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    HeadAt h;
    if (u >= A.units || !head_at(A, u, h)) return;
    float *y = (h.is_v ? A.vo : A.ko) + h.in;
    const void *q = h.is_v ? A.kv.vq : A.kv.kq, *s = h.is_v ? A.kv.vs : A.kv.ks;
    for (int b = 0; b < A.hd / 64; b++) {
        float v;
        if (A.bits == 8) {
            v = (float)((const int8_t *)q)[h.slot * A.hd + 64 * b + lane] * ((const float *)s)[h.slot];
        } else {
            // byte h * 16 + i: element h * 32 + i low, h * 32 + 16 + i high
            const uint8_t w = ((const uint8_t *)q)[h.slot * (A.hd / 2) + 32 * b + 16 * (lane >> 5) + (lane & 15u)];
            const uint16_t sb = ((const uint16_t *)s)[h.slot * (A.hd / 64) + b];
            v = (float)nf4_cb_value((lane & 16u) ? w >> 4 : w & 15) * __uint_as_float((uint32_t)sb << 16);
        }
        y[64 * b + lane] = ifwht_lane(v, b, lane);
    }
}

// Rows of one (layer, sequence, KV head, K or V) rearranged in place.  A thread owns one column (the
// same T-sized piece of every row): it reads the column of every row that moves from its source row
// before it writes any, so no other thread or buffer is involved.
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
        if (mv[r]) col[(size_t)r * pitch] = v[r];
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

RowsArgs rows_args(const k2t_kv_rows &kv, int bits, size_t row_stride, int batch, int ntok, int nkv, int hd,
                   const int *pos, const int *counts, int layer) {
    RowsArgs A{};
    A.row_stride = row_stride;
    A.ntok = ntok;
    A.nkv = nkv;
    A.hd = hd;
    A.bits = bits;
    A.pos = pos;
    A.counts = counts;
    A.kv = kv;
    A.row0 = (size_t)layer * batch;
    A.units = (size_t)batch * ntok * 2 * nkv;
    return A;
}

bool heads_aligned(const float *k, const float *v) {
    return (reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 == 0;
}

void check_heads_call(k2t_ctx *ctx, int bits, int batch, int ntok, int nkv, int hd, size_t row_stride,
                      const void *d_pos, const k2t_kv_rows *kv) {
    branch_arg(ctx != nullptr && kv != nullptr, "NULL argument");
    branch_arg(batch >= 0 && ntok >= 0 && nkv > 0, "negative batch or ntok, or no KV heads");
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

void launch_kv_append(hipStream_t st, int bits, const float *k, const float *v, size_t row_stride, int batch, int ntok,
                      int nkv, int hd, const int *pos, const int *counts, const k2t_kv_rows &kv, int layer) {
    RowsArgs A = rows_args(kv, bits, row_stride, batch, ntok, nkv, hd, pos, counts, layer);
    A.k = k;
    A.v = v;
    hipLaunchKernelGGL(kv_append_kernel, dim3((unsigned)((A.units + 3) / 4)), dim3(256), 0, st, A);
    hip_check(hipGetLastError(), "kv_append launch");
}

static void launch_kv_load(hipStream_t st, RowsArgs A, float *k, float *v) {
    A.ko = k;
    A.vo = v;
    hipLaunchKernelGGL(kv_load_kernel, dim3((unsigned)((A.units + 3) / 4)), dim3(256), 0, st, A);
    hip_check(hipGetLastError(), "kv_load launch");
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
        launch_kv_append(ctx->stream, bits, d_k, d_v, row_stride, batch, ntok, n_kv_heads, head_dim, d_pos, d_counts,
                         *kv, 0);
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
        launch_kv_load(ctx->stream,
                       rows_args(*kv, bits, row_stride, batch, ntok, n_kv_heads, head_dim, d_pos, d_counts, 0), d_k,
                       d_v);
    });
}

int32_t k2t_kv_reorder(k2t_ctx *ctx, int32_t bits, const k2t_kv_rows *kv, const int32_t *d_parents,
                       int32_t n_layers, int32_t n_seq, int32_t beams, int32_t n_kv_heads, int32_t head_dim) {
    return branch_guard([&] {
        branch_arg(ctx && kv && d_parents, "NULL argument");
        check_kv_rows(kv, bits, head_dim);
        branch_arg(n_layers >= 0 && n_seq >= 0 && n_kv_heads > 0, "negative n_layers or n_seq, or no KV heads");
        branch_arg(beams >= 1 && beams <= kMaxBeams, "beams must be 1 .. 64");
        branch_arg((size_t)n_layers * n_seq * n_kv_heads <= (size_t)1 << 22, "too many layers, sequences and heads");
        branch_arg((size_t)kv->len * head_dim <= (size_t)1 << 26, "len too large");
        if (n_layers == 0 || n_seq == 0 || beams == 1 || kv->len == 0) return;
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        launch_kv_reorder(ctx->stream, bits, *kv, d_parents, n_layers, n_seq, beams, n_kv_heads, head_dim);
    });
}

}  // extern "C"
