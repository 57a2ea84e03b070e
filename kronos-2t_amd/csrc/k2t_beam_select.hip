// Beam search's choice over the rows of a sequence and the vocabulary (k2t_beam_select).
#include <float.h>
#include <math.h>

#include "k2t_branch.h"
#include "k2t_device.h"

namespace k2t {

namespace {

constexpr int kSelThreads = 256, kSelPer = 16;           // a slice: 4096 logits of one row
constexpr int kSlice = kSelThreads * kSelPer;

// A logit as a key that orders as it does, the lower token first among equals; 0: no candidate.
__device__ __forceinline__ unsigned long long logit_key(float x, uint32_t token) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 counts as 0)
    const uint32_t o = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((unsigned long long)o << 32) | (0xFFFFFFFFu - token);
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t key_token(unsigned long long k) { return 0xFFFFFFFFu - (uint32_t)k; }

struct SelArgs {
    const float *logits;
    size_t row_stride;
    int vocab, slices, beams, k, eos;
    const float *scores;
    const int *done;
    float2 *stat;              // [row][slice]: maximum, sum of exp(x - maximum)
    unsigned long long *keys;  // [row][slice][k], best first
    float *o_scores;
    int *o_tokens, *o_parents, *o_done;
};

// One slice of one row: its maximum, its sum of exponentials and its k best logits.
__global__ __launch_bounds__(kSelThreads) void select_slice_kernel(SelArgs A) {
    __shared__ float redf[8];
    __shared__ unsigned long long redk[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
    const int slice = blockIdx.x, row = blockIdx.y;
    const float *x = A.logits + (size_t)row * A.row_stride;
    float v[kSelPer];
    float mx = -INFINITY;
#pragma unroll
    for (int j = 0; j < kSelPer; j++) {
        const int i = slice * kSlice + j * kSelThreads + (int)tid;
        float f = i < A.vocab ? x[i] : -INFINITY;
        f = f != f ? -INFINITY : fminf(f, FLT_MAX);
        v[j] = f;
        mx = fmaxf(mx, f);
    }
    mx = wave_max_f(mx);
    if (lane == 0) redf[wv] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(redf[0], redf[1]), fmaxf(redf[2], redf[3]));
    float sum = 0.0f;
    unsigned long long key[kSelPer];
#pragma unroll
    for (int j = 0; j < kSelPer; j++) {
        const bool in = v[j] > -INFINITY;
        sum += in ? expf(v[j] - mx) : 0.0f;
        key[j] = in ? logit_key(v[j], (uint32_t)(slice * kSlice + j * kSelThreads) + tid) : 0;
    }
    sum = wave_sum_f(sum);
    if (lane == 0) redf[4 + wv] = sum;
    __syncthreads();
    const size_t at = (size_t)row * A.slices + slice;
    if (tid == 0) A.stat[at] = make_float2(mx, (redf[4] + redf[5]) + (redf[6] + redf[7]));
    for (int n = 0; n < A.k; n++) {
        unsigned long long best = 0;
#pragma unroll
        for (int j = 0; j < kSelPer; j++) best = key[j] > best ? key[j] : best;
        for (int m = 32; m >= 1; m >>= 1) {
            const unsigned long long o = __shfl_xor(best, m, kWave);
            best = o > best ? o : best;
        }
        if (lane == 0) redk[wv] = best;
        __syncthreads();
        for (int w = 0; w < 4; w++) best = redk[w] > best ? redk[w] : best;
        __syncthreads();
        if (tid == 0) A.keys[at * A.k + n] = best;
#pragma unroll
        for (int j = 0; j < kSelPer; j++)
            if (key[j] == best) key[j] = 0;
    }
}

struct Pick {
    double score;
    int row;
    unsigned long long key;
};
// Higher score, then the lower row, then the higher logit, then the lower token.
__device__ __forceinline__ bool better(const Pick &a, const Pick &b) {
    if (a.score != b.score) return a.score > b.score;
    if (a.row != b.row) return a.row < b.row;
    return a.key > b.key;
}

// One sequence: its rows' log sums, then the k best heads of its slices' lists, one after another.
__global__ __launch_bounds__(256) void select_merge_kernel(SelArgs A) {
    __shared__ double base[kMaxBeams];  // score - log sum
    __shared__ float top[kMaxBeams];
    __shared__ float score[kMaxBeams];
    __shared__ int ended[kMaxBeams];
    __shared__ Pick red[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
    const int seq = blockIdx.x, row0 = seq * A.beams;
    if ((int)tid < A.beams) {
        const int r = row0 + (int)tid;
        float m = -INFINITY;
        for (int s = 0; s < A.slices; s++) m = fmaxf(m, A.stat[(size_t)r * A.slices + s].x);
        double sum = 0.0;
        for (int s = 0; s < A.slices; s++) {
            const float2 st = A.stat[(size_t)r * A.slices + s];
            if (st.x > -INFINITY) sum += (double)st.y * exp((double)st.x - (double)m);
        }
        const float sc = A.scores[r];
        score[tid] = sc;
        ended[tid] = A.done && A.done[r] != 0;
        top[tid] = m;
        base[tid] = sum > 0.0 ? log(sum) : 0.0;
    }
    __syncthreads();
    const int lists = A.beams * A.slices;
    constexpr Pick none{-INFINITY, 0x7fffffff, 0ull};
    Pick last{INFINITY, -1, ~0ull};
    for (int n = 0; n < A.k; n++) {
        // the best candidate that comes after the last one
        Pick best = none;
        for (int l = (int)tid; l < lists; l += 256) {
            const int b = l / A.slices;
            if (!(score[b] > -INFINITY) || ended[b]) continue;
            const unsigned long long *list = A.keys + ((size_t)row0 * A.slices + l) * A.k;
            for (int j = 0; j < A.k; j++) {
                const unsigned long long key = list[j];
                if (!key) break;
                const Pick p{(double)score[b] + (((double)key_logit(key) - (double)top[b]) - base[b]), b, key};
                if (!better(last, p)) continue;
                if (p.score > -INFINITY && better(p, best)) best = p;
                break;
            }
        }
        if ((int)tid < A.beams && ended[tid] && score[tid] > -INFINITY) {
            const Pick p{(double)score[tid], (int)tid, logit_key(0.0f, (uint32_t)A.eos)};
            if (better(last, p) && better(p, best)) best = p;
        }
        for (int m = 32; m >= 1; m >>= 1) {
            const Pick o{__shfl_xor(best.score, m, kWave), __shfl_xor(best.row, m, kWave),
                         __shfl_xor(best.key, m, kWave)};
            if (better(o, best)) best = o;
        }
        if (lane == 0) red[wv] = best;
        __syncthreads();
        for (int w = 0; w < 4; w++)
            if (better(red[w], best)) best = red[w];
        __syncthreads();
        if (tid == 0) {
            const size_t at = (size_t)seq * A.k + n;
            const bool got = best.row != none.row;
            const int token = got ? (int)key_token(best.key) : max(A.eos, 0);
            A.o_scores[at] = got ? (float)best.score : -INFINITY;
            A.o_tokens[at] = token;
            A.o_parents[at] = row0 + (got ? best.row : 0);
            if (A.o_done) A.o_done[at] = !got || ended[best.row] || token == A.eos;
        }
        last = best;
        if (best.row == none.row) last = Pick{-INFINITY, 0x7fffffff, 0ull};
    }
}

int slices_of(int vocab) { return (vocab + kSlice - 1) / kSlice; }

void check_select(k2t_ctx *ctx, int n_seq, int beams, int vocab, int k) {
    branch_arg(ctx != nullptr, "ctx is NULL");
    branch_arg(beams >= 1 && beams <= kMaxBeams, "beams must be 1 .. 64");
    branch_arg(k >= 1 && k <= kMaxPicks, "k must be 1 .. 128");
    branch_arg(n_seq >= 0 && (size_t)n_seq * beams <= 65535, "n_seq * beams must be 0 .. 65535");
    branch_arg(vocab >= 1 && vocab <= 1 << 24, "vocab out of range");
}

}  // namespace

size_t beam_select_ws_bytes(int n_seq, int beams, int vocab, int k) {
    const size_t lists = (size_t)n_seq * beams * slices_of(vocab);
    return std::max<size_t>(16, lists * (sizeof(float2) + (size_t)k * sizeof(unsigned long long)));
}

void launch_beam_select(hipStream_t st, const float *logits, int vocab, size_t row_stride, const float *scores,
                        const int *done, int n_seq, int beams, int k, int eos, float *out_scores, int *out_tokens,
                        int *out_parents, int *out_done, void *ws) {
    SelArgs A{logits, row_stride, vocab, slices_of(vocab), beams, k, eos, scores, done, nullptr, nullptr,
              out_scores, out_tokens, out_parents, out_done};
    A.stat = (float2 *)ws;
    A.keys = (unsigned long long *)(A.stat + (size_t)n_seq * beams * A.slices);
    hipLaunchKernelGGL(select_slice_kernel, dim3(A.slices, n_seq * beams), dim3(kSelThreads), 0, st, A);
    hip_check(hipGetLastError(), "beam_select launch");
    hipLaunchKernelGGL(select_merge_kernel, dim3(n_seq), dim3(256), 0, st, A);
    hip_check(hipGetLastError(), "beam_select merge launch");
}

}  // namespace k2t

using namespace k2t;

extern "C" {

int32_t k2t_beam_select_workspace(k2t_ctx *ctx, int32_t n_seq, int32_t beams, int32_t vocab, int32_t k,
                                  size_t *bytes) {
    return branch_guard([&] {
        branch_arg(bytes != nullptr, "NULL argument");
        check_select(ctx, n_seq, beams, vocab, k);
        *bytes = beam_select_ws_bytes(n_seq, beams, vocab, k);
    });
}

int32_t k2t_beam_select(k2t_ctx *ctx, const float *d_logits, int32_t vocab, size_t row_stride, const float *d_scores,
                        const int32_t *d_done, int32_t n_seq, int32_t beams, int32_t k, int32_t eos,
                        float *d_out_scores, int32_t *d_out_tokens, int32_t *d_out_parents, int32_t *d_out_done,
                        void *d_ws, size_t ws_bytes) {
    return branch_guard([&] {
        check_select(ctx, n_seq, beams, vocab, k);
        branch_arg(eos >= -1 && eos < vocab, "eos must be -1 (none) or a token");
        branch_arg(d_done == nullptr || eos >= 0, "d_done needs an eos token");
        branch_arg(row_stride >= (size_t)vocab, "row_stride is smaller than the vocabulary");
        if (n_seq == 0) return;
        branch_arg(d_logits && d_scores && d_out_scores && d_out_tokens && d_out_parents && d_ws, "NULL argument");
        branch_arg(reinterpret_cast<uintptr_t>(d_ws) % 16 == 0, "d_ws must be 16-byte aligned");
        const size_t need = beam_select_ws_bytes(n_seq, beams, vocab, k);
        if (ws_bytes < need)
            throw Error(K2T_E_ARG, "the workspace holds " + std::to_string(ws_bytes) + " bytes, " +
                                       std::to_string(need) + " are needed");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        launch_beam_select(ctx->stream, d_logits, vocab, row_stride, d_scores, d_done, n_seq, beams, k, eos,
                           d_out_scores, d_out_tokens, d_out_parents, d_out_done, d_ws);
    });
}

}  // extern "C"
