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

constexpr int kPart = 256;  // positions of one part

struct SharedArgs {
    const float *q;
    size_t q_stride;
    k2t_kv_rows pre, tail;
    int beams, nq, nkv, hd, bits;
    int np, nt;  // prefix and tail parts
    float attn_scale;
    float *part;  // [row][head][np + nt][2 + hd]
    float *out;
};

__device__ __forceinline__ int row_len(const k2t_kv_rows &kv, int row) {
    return kv.d_len ? max(0, min(kv.d_len[row], kv.len)) : kv.len;
}

// One workgroup per (part, head, row): part p < np of the prefix, else of the tail.
__global__ __launch_bounds__(kPart) void shared_part_kernel(SharedArgs A) {
    __shared__ __align__(16) int8_t qi[128];
    __shared__ float qas_s, sc[kPart], red[8];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
    const int p = blockIdx.x, head = blockIdx.y, row = blockIdx.z, nb = A.hd / 64;
    const bool is_tail = p >= A.np;
    const k2t_kv_rows &kv = is_tail ? A.tail : A.pre;
    const int krow = is_tail ? row : row / A.beams;
    const int t0 = (is_tail ? p - A.np : p) * kPart, t1 = min(row_len(kv, krow), t0 + kPart);
    if (t0 >= t1) return;
    const size_t base = ((size_t)krow * A.nkv + head / (A.nq / A.nkv)) * kv.cap;
    if (wv == 0) {
        const float *x = A.q + row * A.q_stride + (size_t)head * A.hd;
        const float r0 = fwht_lane(x[lane], 0, lane);
        const float r1 = nb > 1 ? fwht_lane(x[64 + lane], 1, lane) : 0.0f;
        const float mx = wave_max_f(fmaxf(fabsf(r0), fabsf(r1)));
        const float inv = mx <= FLT_EPSILON ? 0.0f : 127.0f / mx;
        qi[lane] = (int8_t)(int)rintf(r0 * inv);
        qi[64 + lane] = (int8_t)(int)rintf(r1 * inv);
        if (lane == 0) qas_s = (mx <= FLT_EPSILON ? 0.0f : mx / 127.0f) * A.attn_scale;
    }
    __syncthreads();
    const int t = t0 + (int)tid;
    const int8_t *k8 = (const int8_t *)kv.kq, *v8 = (const int8_t *)kv.vq;
    const uint16_t *ks16 = (const uint16_t *)kv.ks, *vs16 = (const uint16_t *)kv.vs;
    // element e of slot s of an NF4 cache: its codebook value
    auto nf4 = [&](const void *q, size_t s, int e) {
        const uint8_t w = ((const uint8_t *)q)[s * (A.hd / 2) + 32 * (e >> 6) + 16 * ((e >> 5) & 1) + (e & 15)];
        return nf4_cb_value((e & 16) ? w >> 4 : w & 15);
    };
    float s = -INFINITY;
    if (t < t1) {
        s = 0.0f;
        for (int b = 0; b < nb; b++) {
            int dot = 0;
            for (int e = 64 * b; e < 64 * b + 64; e++)
                dot += (int)qi[e] * (A.bits == 8 ? (int)k8[(base + t) * A.hd + e] : nf4(kv.kq, base + t, e));
            const float ks = A.bits == 8 ? ((const float *)kv.ks)[base + t]
                                         : __uint_as_float((uint32_t)ks16[(base + t) * nb + b] << 16);
            s += ((float)dot * ks) * qas_s;
        }
    }
    const float wm = wave_max_f(s);
    if (lane == 0) red[wv] = wm;
    __syncthreads();
    const float m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float pw = t < t1 ? expf(s - m) : 0.0f;
    sc[tid] = pw;
    const float ws = wave_sum_f(pw);
    if (lane == 0) red[4 + wv] = ws;
    __syncthreads();
    float *pp = A.part + (((size_t)row * A.nq + head) * (A.np + A.nt) + p) * (2 + A.hd);
    if (tid == 0) {
        pp[0] = m;
        pp[1] = (red[4] + red[5]) + (red[6] + red[7]);
    }
    if ((int)tid < A.hd) {
        float o = 0.0f;
        for (int i = 0; i < t1 - t0; i++) {
            const size_t sl = base + t0 + i;
            const float v = A.bits == 8 ? (float)v8[sl * A.hd + tid] * ((const float *)kv.vs)[sl]
                                        : (float)nf4(kv.vq, sl, (int)tid) *
                                              __uint_as_float((uint32_t)vs16[sl * nb + (tid >> 6)] << 16);
            o = fmaf(sc[i], v, o);
        }
        pp[2 + tid] = o;
    }
}

// One wave per (head, row): the parts that hold positions, in order, and ifwht64.
__global__ __launch_bounds__(64) void shared_merge_kernel(SharedArgs A) {
    const uint32_t lane = threadIdx.x;
    const int head = blockIdx.x, row = blockIdx.y, nb = A.hd / 64, n = A.np + A.nt;
    const int np = A.np ? (row_len(A.pre, row / A.beams) + kPart - 1) / kPart : 0;
    const int nt = A.nt ? (row_len(A.tail, row) + kPart - 1) / kPart : 0;
    const float *pp = A.part + ((size_t)row * A.nq + head) * n * (2 + A.hd);
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    for (int i = 0; i < np + nt; i++) {
        const float *ps = pp + (size_t)(i < np ? i : A.np + i - np) * (2 + A.hd);
        const float mn = fmaxf(m, ps[0]), a = m == -INFINITY ? 0.0f : expf(m - mn), b = expf(ps[0] - mn);
        l = fmaf(l, a, ps[1] * b);
        o0 = fmaf(o0, a, ps[2 + lane] * b);
        if (nb > 1) o1 = fmaf(o1, a, ps[2 + 64 + lane] * b);
        m = mn;
    }
    const float inv = np + nt == 0 ? 0.0f : 1.0f / l;
    float *out = A.out + ((size_t)row * A.nq + head) * A.hd;
    out[lane] = ifwht_lane(o0 * inv, 0, lane);
    if (nb > 1) out[64 + lane] = ifwht_lane(o1 * inv, 1, lane);
}

int parts_of(int len) { return (len + kPart - 1) / kPart; }

}  // namespace

size_t attn_shared_ws_bytes(const k2t_ctx *, const SharedShape &s, int prefix_len, int tail_len) {
    return std::max<size_t>(16, (size_t)s.n_seq * s.beams * s.nq * (parts_of(prefix_len) + parts_of(tail_len)) *
                                    (2 + s.hd) * sizeof(float));
}

void launch_attn_shared(k2t_ctx *, hipStream_t st, int bits, const float *q, size_t q_stride, const SharedShape &s,
                        const k2t_kv_rows &prefix, const k2t_kv_rows &tail, float attn_scale, float *out, void *ws) {
    SharedArgs A{q, q_stride, prefix, tail, s.beams, s.nq, s.nkv, s.hd, bits, 0, 0, attn_scale, (float *)ws, out};
    A.np = prefix.cap ? parts_of(prefix.len) : 0;
    A.nt = tail.cap ? parts_of(tail.len) : 0;
    const int rows = s.n_seq * s.beams;
    if (A.np + A.nt) {
        hipLaunchKernelGGL(shared_part_kernel, dim3(A.np + A.nt, s.nq, rows), dim3(kPart), 0, st, A);
        hip_check(hipGetLastError(), "attn_shared launch");
    }
    hipLaunchKernelGGL(shared_merge_kernel, dim3(s.nq, rows), dim3(64), 0, st, A);
    hip_check(hipGetLastError(), "attn_shared merge launch");
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
