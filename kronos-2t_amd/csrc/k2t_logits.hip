// What a choice of the next token is made from: penalties for repeated tokens, biases and grammar masks on rows
// of logits (k2t_logits_adjust).
//
// For a row and a token with logit x, s: the token stands in the history, c: how often behind the prompt,
//   y = s ? (x > 0 ? x / repeat : x repeat) : x,  y -= c > 0 ? presence + frequency c : 0,  y += its biases,
//   y = -inf where the mask does not allow it,
// in 64 bits for the few tokens that the lists name; the others are copied bit for bit.
//
// A workgroup takes a slice of a row's vocabulary: it counts the history's tokens that fall into the slice in LDS
// (integer atomics: any order gives the same counts), notes for every token the first entry of the bias list that names
// it, and the entries of the list that fall into the slice, and then passes over its logits once. A token's biases are
// added in the list's order by the thread that owns the token, so that the sum does not depend on scheduling.
//
// What bounds it: bytes, and every slice's pass over the row's lists. 64 rows of 151936, histories of 2000, 40 biases and a
// mask (78 MB read and written): 18.8 us, 4.2 TB/s; slices of 1024, 4096 and 8192 logits 22.8, 23.7 and 32 us (more passes
// over the lists; fewer loads in flight), one load of the history at a time and cached stores 26.8. 4 rows of 49152: 4.1 us, a launch
// and the lists. Rows that do not begin at multiples of 16 bytes, a logit at a time: 64 of 50257 (contiguous) 12.5 us, of 50260 9.7. Tokens that are named twice (4 rows of 10536, 213 biases: 8.1 us; 128 rows of 32000, 300: 14.8): 17.0 and
// 33.4 with a search through the row's whole list. (4000 biases in 5 slices, most named twice: 356 us, 1890.)
#include <math.h>

#include <algorithm>

#include "k2t_branch.h"
#include "k2t_device.h"

namespace k2t {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kLogitSlice = 2048, kGroups = kLogitSlice / 4 / kThreads;  // groups of four logits per thread
constexpr int kMaxHistory = 1 << 20, kMaxBias = 4096, kAhead = 8;
constexpr int kFewBiases = 64, kManyBiases = 2048, kTokenBits = 11;  // (see NAMED)
constexpr uint32_t kSeen = 1u << 31;    // over the count of a token behind the prompt
constexpr uint32_t kNone = 0xFFFFu, kAgain = 1u << 15;  // no bias; more entries than the first name the token

static_assert(kLogitSlice == 1 << kTokenBits && kMaxBias <= 1 << (32 - kTokenBits), "an entry of `named` holds both");

struct LogitsArgs {
    const float *x;
    float *out;
    size_t x_stride, out_stride;
    int vocab;
    k2t_logits_rules R;
};

// NAMED: biases that are noted, as index << kTokenBits | token: the row's whole list (kFewBiases; ~0: of another slice), or the
// slice's; 0: the row has neither history nor biases.  VEC: rows start at multiples of 16 bytes.
template <int NAMED, bool VEC>
__global__ __launch_bounds__(kThreads) void logits_kernel(const LogitsArgs A) {
    constexpr bool LISTS = NAMED > 0, WHOLE = NAMED == kFewBiases;
    __shared__ __align__(16) uint32_t count[LISTS ? kLogitSlice : 4], first[LISTS ? kLogitSlice : 4], named[LISTS ? NAMED : 4];
    __shared__ int before[kThreads / 64];
    const int row = (int)blockIdx.y, v0 = (int)blockIdx.x * kLogitSlice, tid = (int)threadIdx.x;
    const int n = min(kLogitSlice, A.vocab - v0);
    const float *x = A.x + (size_t)row * A.x_stride + v0;
    float *out = A.out + (size_t)row * A.out_stride + v0;
    const bool moved = A.out != A.x;
    const auto load = [&](int i) {
        f32x4 f;
        if (VEC && i + 4 <= n) return *reinterpret_cast<const f32x4 *>(x + i);
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = x[min(i + j, n - 1)];
        return f;
    };
    f32x4 f[kGroups];
    if (moved) {  // (in place most groups are never read)
#pragma unroll
        for (int g = 0; g < kGroups; g++) f[g] = load(4 * min(tid + kThreads * g, (n - 1) / 4));
    }
    const k2t_logits_rules &R = A.R;
    const uint32_t *mask = nullptr;
    if (R.d_mask) {
        const int m = R.d_mask_row ? R.d_mask_row[row] : row;
        if (m >= 0 && m < R.mask_rows) mask = R.d_mask + (size_t)m * R.mask_stride + v0 / 32;
    }
    int biases = 0, mine = 0;  // of the row; that name the slice's tokens
    if constexpr (LISTS) {
        for (int i = 4 * tid; i < kLogitSlice; i += 4 * kThreads) {
            *reinterpret_cast<uint4 *>(count + i) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4 *>(first + i) = make_uint4(kNone, kNone, kNone, kNone);
        }
        __syncthreads();
        if (R.d_history) {
            const int len = R.d_history_len ? max(0, min(R.d_history_len[row], R.history_len)) : R.history_len;
            const int prompt = R.d_prompt_len ? R.d_prompt_len[row] : 0;
            const int *h = R.d_history + (size_t)row * R.history_stride;
            // (several loads in flight: the list is the longest chain of a short row)
            for (int i0 = tid; i0 < len; i0 += kAhead * kThreads) {
                int token[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; k++) token[k] = h[min(i0 + k * kThreads, len - 1)];
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    const int i = i0 + k * kThreads;
                    const uint32_t t = (uint32_t)token[k] - (uint32_t)v0;
                    if (i >= len || t >= (uint32_t)n) continue;
                    atomicOr(&count[t], kSeen);
                    if (i >= prompt) atomicAdd(&count[t], 1u);
                }
            }
        }
        const int *names = R.d_bias_tokens + (size_t)row * R.bias_stride;
        if (R.d_bias_tokens) {
            biases = R.d_bias_len ? max(0, min(R.d_bias_len[row], R.bias_len)) : R.bias_len;
            for (int i = tid; i < biases; i += kThreads) {
                const uint32_t t = (uint32_t)names[i] - (uint32_t)v0;
                if (t < (uint32_t)n) atomicMin(&first[t], (uint32_t)i);
                if (WHOLE) named[i] = t < (uint32_t)n ? (uint32_t)i << kTokenBits | t : ~0u;
            }
        }
        __syncthreads();
        if constexpr (WHOLE) {
            mine = biases;
            for (int i = tid; i < biases; i += kThreads) {
                const uint32_t t = named[i] & (kLogitSlice - 1);
                if (named[i] != ~0u && (first[t] & (kAgain - 1)) != (uint32_t)i) atomicOr(&first[t], kAgain);
            }
            __syncthreads();
        } else if (biases) {  // the slice's entries, in order: a thread takes some that follow each other
            const int per = (biases + kThreads - 1) / kThreads, a = min(tid * per, biases), b = min(a + per, biases);
            int own = 0;
            for (int i = a; i < b; i++) own += (uint32_t)names[i] - (uint32_t)v0 < (uint32_t)n;
            int upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int v = __shfl_up(upto, d, 64);
                upto += (tid & 63) >= d ? v : 0;
            }
            if ((tid & 63) == 63) before[tid >> 6] = upto;
            __syncthreads();
            int at = upto - own;
#pragma unroll
            for (int w = 0; w < kThreads / 64; w++) {
                at += w < tid >> 6 ? before[w] : 0;
                mine += before[w];
            }
            for (int i = a; i < b; i++) {
                const uint32_t t = (uint32_t)names[i] - (uint32_t)v0;
                if (t >= (uint32_t)n) continue;
                if ((first[t] & (kAgain - 1)) != (uint32_t)i) atomicOr(&first[t], kAgain);
                if (at < NAMED) named[at] = (uint32_t)i << kTokenBits | t;
                at++;
            }
            __syncthreads();
        }
    }
    const double repeat = LISTS && R.d_repeat ? (double)R.d_repeat[row] : 1.0;
    const double presence = LISTS && R.d_presence ? (double)R.d_presence[row] : 0.0;
    const double frequency = LISTS && R.d_frequency ? (double)R.d_frequency[row] : 0.0;
    const auto adjust = [&](float v, int i, uint32_t c, uint32_t b) {
        double y = (double)v;
        if (c & kSeen) y = y > 0.0 ? y / repeat : y * repeat;
        const uint32_t fresh = c & ~kSeen;
        if (fresh) y -= presence + frequency * (double)fresh;
        if (b != kNone) {
            const float *value = R.d_bias + (size_t)row * R.bias_stride;
            const int *names = R.d_bias_tokens + (size_t)row * R.bias_stride;
            const int at = (int)(b & (kAgain - 1));
            y += (double)value[at];
            if (b & kAgain && mine <= NAMED) {
                for (int k = 0; k < mine; k++) {
                    const uint32_t e = named[k];
                    if (e != ~0u && (e & (kLogitSlice - 1)) == (uint32_t)i && (int)(e >> kTokenBits) > at) y += (double)value[e >> kTokenBits];
                }
            } else if (b & kAgain) {  // (more biases than tokens)
                for (int k = at + 1; k < biases; k++)
                    if (names[k] == v0 + i) y += (double)value[k];
            }
        }
        return (float)y;
    };
#pragma unroll
    for (int g = 0; g < kGroups; g++) {
        const int i = 4 * (tid + kThreads * g);
        if (i >= n) break;
        uint32_t allowed = 0xFu, c[4] = {}, b[4] = {kNone, kNone, kNone, kNone};
        if (mask) allowed = mask[i / 32] >> (i % 32) & 0xFu;
        bool listed = false;
        if constexpr (LISTS) {
            const uint4 cc = *reinterpret_cast<const uint4 *>(count + i), bb = *reinterpret_cast<const uint4 *>(first + i);
            c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
            b[0] = bb.x, b[1] = bb.y, b[2] = bb.z, b[3] = bb.w;
            listed = (cc.x | cc.y | cc.z | cc.w) != 0 || (bb.x & bb.y & bb.z & bb.w) != kNone;
        }
        if (!moved) {
            if (!listed && allowed == 0xFu) continue;
            f[g] = load(i);
        }
        if (listed) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if ((c[j] != 0 || b[j] != kNone) && i + j < n) f[g][j] = adjust(f[g][j], i + j, c[j], b[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) f[g][j] = allowed >> j & 1u ? f[g][j] : -INFINITY;
        if (VEC && i + 4 <= n) {
            __builtin_nontemporal_store(f[g], reinterpret_cast<f32x4 *>(out + i));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < n) out[i + j] = f[g][j];
        }
    }
}

template <int NAMED>
void launch_logits(bool vec, dim3 grid, hipStream_t st, const LogitsArgs &A) {
    if (vec) hipLaunchKernelGGL((logits_kernel<NAMED, true>), grid, dim3(kThreads), 0, st, A);
    else hipLaunchKernelGGL((logits_kernel<NAMED, false>), grid, dim3(kThreads), 0, st, A);
}

}  // namespace

}  // namespace k2t

using namespace k2t;

extern "C" {

int32_t k2t_logits_adjust(k2t_ctx *ctx, const float *d_logits, int32_t vocab, size_t row_stride, int32_t rows,
                          const k2t_logits_rules *rules, float *d_out, size_t out_stride) {
    return branch_guard([&] {
        branch_arg(ctx && rules, "NULL argument");
        const k2t_logits_rules &R = *rules;
        branch_arg(vocab >= 1 && vocab <= 1 << 24, "vocab must be 1 .. 2^24");
        branch_arg(rows >= 0 && rows <= 65535, "rows must be 0 .. 65535");
        branch_arg(row_stride >= (size_t)vocab && out_stride >= (size_t)vocab, "a stride is smaller than the vocabulary");
        branch_arg(row_stride < (size_t)1 << 40 && out_stride < (size_t)1 << 40, "a stride is out of range");
        if (R.d_history)
            branch_arg(R.history_len >= 0 && R.history_len <= kMaxHistory && R.history_stride >= (size_t)R.history_len &&
                           R.history_stride < (size_t)1 << 40,
                       "history_len must be 0 .. 2^20, history_stride no smaller");
        else  // (a list without entries has no address)
            branch_arg(R.history_len == 0 || (!R.d_repeat && !R.d_presence && !R.d_frequency), "penalties without a history");
        branch_arg((R.d_bias_tokens != nullptr) == (R.d_bias != nullptr), "biases need both their tokens and their values");
        if (R.d_bias)
            branch_arg(R.bias_len >= 0 && R.bias_len <= kMaxBias && R.bias_stride >= (size_t)R.bias_len &&
                           R.bias_stride < (size_t)1 << 40,
                       "bias_len must be 0 .. 4096, bias_stride no smaller");
        if (R.d_mask)
            branch_arg(R.mask_rows >= (R.d_mask_row ? 0 : rows) && R.mask_stride >= ((size_t)vocab + 31) / 32 &&
                           R.mask_stride < (size_t)1 << 40,
                       "mask_rows or mask_stride too small");
        else
            branch_arg(R.mask_rows == 0 || !R.d_mask_row, "mask rows without masks");
        if (rows == 0) return;
        branch_arg(d_logits && d_out, "NULL argument");
        const auto at = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
        branch_arg((at(d_logits) | at(d_out)) % 4 == 0, "d_logits and d_out must be aligned to floats");
        branch_arg(d_logits != d_out || row_stride == out_stride, "in place the strides must be the same");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        LogitsArgs A{d_logits, d_out, row_stride, out_stride, vocab, R};
        const bool vec = (at(d_logits) | at(d_out)) % 16 == 0 && row_stride % 4 == 0 && out_stride % 4 == 0;
        const bool lists = (R.d_history && R.history_len) || (R.d_bias && R.bias_len);
        const dim3 grid((unsigned)((vocab + kLogitSlice - 1) / kLogitSlice), (unsigned)rows);
        // (a short list needs no sorting out by slices, and less LDS: 64 rows of 151936, 40 biases, 19.2 and 22.9 us; but
        // 4 rows of 10536, 213 biases that name tokens twice, 15.9 and 8.1)
        if (!lists) launch_logits<0>(vec, grid, ctx->stream, A);
        else if (!R.d_bias || R.bias_len <= kFewBiases) launch_logits<kFewBiases>(vec, grid, ctx->stream, A);
        else launch_logits<kManyBiases>(vec, grid, ctx->stream, A);
        hip_check(hipGetLastError(), "logits_adjust launch");
    });
}

}  // extern "C"
