// Attention of a block of tokens of every row of a batch over the row's Hadamard cache (k2t_attn_tokens).
#include <float.h>
#include <math.h>

#include <algorithm>

#include "k2t_branch.h"
#include "k2t_device.h"
#include "k2t_kv_dev.h"

namespace k2t {

namespace {

constexpr int kMaxTree = 64;

struct TokensArgs {
    const float *q;
    size_t q_stride;
    int ntok, nq, nkv;
    const int *pos, *counts;
    const uint64_t *sees;
    k2t_kv_rows kv;
    float attn_scale;
    float *out;
};

// One workgroup per (token, head, row): a position per thread, 256 at a time.
template <int HD, int BITS>
__global__ __launch_bounds__(256) void tokens_simple_kernel(const TokensArgs A) {
    constexpr int NB = HD / 64;
    __shared__ int8_t q[HD];
    __shared__ float w[256], red[4], qs, o[256];
    const int tid = (int)threadIdx.x, head = (int)blockIdx.y, t = (int)blockIdx.x, row = (int)blockIdx.z;
    const uint32_t lane = tid & 63u, wave = tid >> 6;
    const int count = A.counts ? min(A.counts[row], A.ntok) : A.ntok;
    if (t >= count) return;
    const size_t token = (size_t)row * A.ntok + t;
    const float *qh = A.q + token * A.q_stride + (size_t)head * HD;
    if (wave == 0) {
        const float r0 = fwht_lane(qh[lane], 0, lane), r1 = NB > 1 ? fwht_lane(qh[64 + lane], 1, lane) : 0.0f;
        const float mx = wave_max_f(fmaxf(fabsf(r0), fabsf(r1)));
        const bool tiny = mx <= FLT_EPSILON;
        q[lane] = tiny ? 0 : (int8_t)(int)rintf(r0 * (127.0f / mx));
        if (NB > 1) q[64 + lane] = tiny ? 0 : (int8_t)(int)rintf(r1 * (127.0f / mx));
        if (lane == 0) qs = tiny ? 0.0f : (mx / 127.0f) * A.attn_scale;
    }
    __syncthreads();
    const long long start = A.pos[row], end = min((long long)A.kv.len, start + count);
    const size_t slot = ((size_t)row * A.nkv + head / (A.nq / A.nkv)) * A.kv.cap;
    const auto code = [&](const void *base, size_t s, int e) {
        if (BITS == 8) return (int)((const int8_t *)base)[s * HD + e];
        const uint8_t b = ((const uint8_t *)base)[s * (HD / 2) + e / 32 * 16 + e % 16];
        return nf4_cb_value(e & 16 ? b >> 4 : b & 15);
    };
    const auto scale = [&](const void *base, size_t s, int b) {
        if (BITS == 8) return ((const float *)base)[s];
        return __uint_as_float((uint32_t)((const uint16_t *)base)[s * NB + b] << 16);
    };
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    const int d = tid % HD, part = tid / HD;
    for (long long p0 = 0; p0 < end; p0 += 256) {
        const long long p = p0 + tid, j = p - start;
        const bool live = p < end && (j < 0 || (A.sees ? (A.sees[token] >> j & 1) != 0 : j <= t));
        float s = -INFINITY;
        if (live) {
            s = 0.0f;
            for (int b = 0; b < NB; b++) {
                int dot = 0;
                for (int e = 64 * b; e < 64 * b + 64; e++) dot += q[e] * code(A.kv.kq, slot + p, e);
                s += (float)dot * scale(A.kv.ks, slot + p, b);
            }
            s *= qs;
        }
        float mx = wave_max_f(s);
        if (lane == 0) red[wave] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(m, mx);
        const float corr = mn == -INFINITY || m == mn ? 1.0f : expf(m - mn);
        w[tid] = live ? expf(s - mn) : 0.0f;
        m = mn;
        __syncthreads();
        l *= corr;
        acc *= corr;
        const int n = (int)min(256ll, end - p0);
        for (int i = 0; i < n; i++) l += w[i];
        for (int i = part; i < n; i += 256 / HD)
            if (w[i] != 0.0f) acc += w[i] * ((float)code(A.kv.vq, slot + p0 + i, d) * scale(A.kv.vs, slot + p0 + i, d / 64));
        __syncthreads();
    }
    o[tid] = acc;
    __syncthreads();
    if ((int)wave < NB) {
        float v = 0.0f;
        for (int k = 0; k < 256 / HD; k++) v += o[k * HD + tid];
        v = m == -INFINITY && l == 0.0f ? 0.0f : v / l;
        A.out[(token * A.nq + head) * HD + tid] = ifwht_lane(v, wave, lane);
    }
}

template <int HD>
void launch_tokens(hipStream_t st, int bits, const TokensArgs &A, int batch) {
    const dim3 grid((unsigned)A.ntok, (unsigned)A.nq, (unsigned)batch);
    if (bits == 8) hipLaunchKernelGGL((tokens_simple_kernel<HD, 8>), grid, dim3(256), 0, st, A);
    else hipLaunchKernelGGL((tokens_simple_kernel<HD, 4>), grid, dim3(256), 0, st, A);
    hip_check(hipGetLastError(), "attn_tokens launch");
}

void check_tokens_shape(k2t_ctx *ctx, int batch, int ntok, int nq, int nkv, int hd) {
    branch_arg(ctx != nullptr, "ctx is NULL");
    branch_arg(hd == 64 || hd == 128, "head_dim must be 64 or 128");
    branch_arg(nq > 0 && nkv > 0 && nq % nkv == 0 && nq <= 1024, "n_heads must be a multiple of n_kv_heads, at most 1024");
    branch_arg(batch >= 0 && batch <= 65535 && ntok >= 0, "batch must be 0 .. 65535, ntok >= 0");
    branch_arg((size_t)batch * ntok * nq <= (size_t)1 << 22, "more than 2^22 query heads in one call");
}

}  // namespace

}  // namespace k2t

using namespace k2t;

extern "C" {

int32_t k2t_attn_tokens_workspace(k2t_ctx *ctx, int32_t batch, int32_t ntok, int32_t n_heads, int32_t n_kv_heads,
                                  int32_t head_dim, int32_t len, size_t *bytes) {
    return branch_guard([&] {
        branch_arg(bytes != nullptr, "NULL argument");
        check_tokens_shape(ctx, batch, ntok, n_heads, n_kv_heads, head_dim);
        branch_arg(len >= 0 && len <= 1 << 24, "len out of range");
        *bytes = 16;
    });
}

int32_t k2t_attn_tokens(k2t_ctx *ctx, int32_t bits, const float *d_q, size_t q_stride, int32_t batch, int32_t ntok,
                        int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, const int32_t *d_pos,
                        const int32_t *d_counts, const uint64_t *d_sees, const k2t_kv_rows *kv, float attn_scale,
                        float *d_out, void *d_ws, size_t ws_bytes) {
    return branch_guard([&] {
        check_tokens_shape(ctx, batch, ntok, n_heads, n_kv_heads, head_dim);
        branch_arg(kv != nullptr, "NULL argument");
        check_kv_rows(kv, bits, head_dim);
        branch_arg(!d_sees || ntok <= kMaxTree, "a tree has at most 64 tokens");
        branch_arg(attn_scale >= 0.0f && attn_scale <= FLT_MAX, "attn_scale must be finite and not negative");
        if (batch == 0 || ntok == 0) return;
        branch_arg(d_q && d_out && d_ws && d_pos, "NULL argument");
        const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
        branch_arg(q_stride >= (size_t)n_heads * head_dim && q_stride % 4 == 0 && q_stride < (size_t)1 << 31 &&
                       at(d_q) % 16 == 0,
                   "d_q must be 16-byte aligned, q_stride a multiple of 4, no smaller than a token's heads, below 2^31");
        branch_arg((at(d_out) | at(d_ws)) % 16 == 0, "d_out and d_ws must be 16-byte aligned");
        branch_arg(at(d_sees) % 8 == 0, "d_sees must be 8-byte aligned");
        const size_t need = 16;
        if (ws_bytes < need)
            throw Error(K2T_E_ARG, "the workspace holds " + std::to_string(ws_bytes) + " bytes, " +
                                       std::to_string(need) + " are needed");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        TokensArgs A{d_q, q_stride, ntok, n_heads, n_kv_heads, d_pos, d_counts, d_sees, *kv, attn_scale, d_out};
        if (head_dim == 128) launch_tokens<128>(ctx->stream, bits, A, batch);
        else launch_tokens<64>(ctx->stream, bits, A, batch);
    });
}

}  // extern "C"
