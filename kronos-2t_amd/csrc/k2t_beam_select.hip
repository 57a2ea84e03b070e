// Beam search's choice over the rows of a sequence and the vocabulary (k2t_beam_select), in two
// launches: every slice of 4096 logits leaves its maximum, its sum of exponentials and its k best,
// sorted; one workgroup per sequence adds a row's slices up, merges their lists, and merges the rows'.
//
// A slice is read once into registers.  Its k best are among the elements that reach a bound: each of
// the four waves finds the (k/4)-th largest of its 64 threads' maxima (bit by bit, counting lanes by
// ballot), and at least k elements reach the smallest of the four; in random logits few more do.  They
// are sorted by counting, for each, the larger ones.  Everything that orders is a unique key, so the
// result depends on no timing.
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
    unsigned long long *keys;  // [row][slice][k], best first, 0 behind the last
    unsigned long long *far;   // [row][k], and tokens: a row's picks behind those that LDS holds
    int *far_token;
    float *o_scores;
    int *o_tokens, *o_parents, *o_done;
};

// The r-th largest of a wave's keys (`ord` the logit's order, 0 for none, `token` unique), as the
// smallest key that reaches it; 0 where fewer than r lanes have one.
__device__ __forceinline__ unsigned long long wave_kth(uint32_t ord, uint32_t token, int r) {
    uint32_t t = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t c = t | (1u << bit);
        if (__popcll(__ballot(ord >= c)) >= r) t = c;
    }
    if (t == 0) return 0;
    // equal logits at the bound: only the lowest tokens of them are needed
    const int need = r - __popcll(__ballot(ord > t));
    uint32_t low = 0xFFFFFFFFu;
    if (__popcll(__ballot(ord == t)) > need) {
        low = 0;  // the largest token that `need` of them do not pass
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t c = low | (1u << bit);
            if (__popcll(__ballot(ord == t && token < c)) < need) low = c;
        }
    }
    return ((unsigned long long)t << 32) | (0xFFFFFFFFu - low);
}

// One slice of one row: its maximum, its sum of exponentials and its k best logits.
__global__ __launch_bounds__(kSelThreads) void select_slice_kernel(SelArgs A) {
    constexpr int kSelWaves = kSelThreads / 64;
    __shared__ unsigned long long list[kSlice];
    __shared__ unsigned long long bound[kSelWaves];
    __shared__ float redf[2 * kSelWaves];
    __shared__ int count;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
    const int slice = blockIdx.x, row = blockIdx.y;
    const float *x = A.logits + (size_t)row * A.row_stride;
    const uint32_t first = (uint32_t)slice * kSlice + tid;  // this thread's tokens: first + 256 j
    float v[kSelPer];
#pragma unroll
    for (int j = 0; j < kSelPer; j++) v[j] = x[min((int)first + j * kSelThreads, A.vocab - 1)];
    float mx = -INFINITY;
    uint32_t at = 0;
#pragma unroll
    for (int j = 0; j < kSelPer; j++) {
        const bool none = v[j] != v[j] || (int)first + j * kSelThreads >= A.vocab;
        v[j] = none ? -INFINITY : fminf(v[j], FLT_MAX);
        if (v[j] > mx) {  // (the lowest token of equal ones)
            mx = v[j];
            at = first + j * kSelThreads;
        }
    }
    const unsigned long long best = mx > -INFINITY ? logit_key(mx, at) : 0;
    const unsigned long long kth = wave_kth((uint32_t)(best >> 32), at, (A.k + kSelWaves - 1) / kSelWaves);
    mx = wave_max_f(mx);
    if (tid == 0) count = 0;
    if (lane == 0) {
        bound[wv] = kth;
        redf[wv] = mx;
    }
    __syncthreads();
    unsigned long long b = bound[0];
    mx = redf[0];
#pragma unroll
    for (int w = 1; w < kSelWaves; w++) {
        b = bound[w] < b ? bound[w] : b;
        mx = fmaxf(mx, redf[w]);
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kSelPer; j++) {
        if (v[j] == -INFINITY) continue;
        sum += expf(v[j] - mx);
        const unsigned long long key = logit_key(v[j], first + j * kSelThreads);
        if (key >= b) list[atomicAdd(&count, 1)] = key;  // (their order does not matter: sorted below)
    }
    sum = wave_sum_f(sum);
    if (lane == 0) redf[kSelWaves + wv] = sum;
    __syncthreads();
    const size_t out = (size_t)row * A.slices + slice;
    if (tid == 0) {
        sum = 0.0f;
        for (int w = 0; w < kSelWaves; w++) sum += redf[kSelWaves + w];
        A.stat[out] = make_float2(mx, sum);
    }
    const int n = count;
    for (int c = (int)tid; c < n; c += kSelThreads) {
        const unsigned long long mine = list[c];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < n; i++) rank += list[i] > mine ? 1 : 0;
        if (rank < A.k) A.keys[out * A.k + rank] = mine;
    }
    for (int c = n + (int)tid; c < A.k; c += kSelThreads) A.keys[out * A.k + c] = 0;
}

// Largest of a wave's values (DPP row shifts and broadcasts: no LDS round trip), in every lane.
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
    const auto up = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false));  // row_shr:1
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false));  // row_shr:2
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false));  // row_shr:4
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false));  // row_shr:8
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));  // row_bcast:15
    v = up(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));  // row_bcast:31
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// The lane with the largest key (the lowest of equal ones); -1 where every key is 0.
__device__ __forceinline__ int wave_best(unsigned long long key) {
    const uint32_t hi = (uint32_t)(key >> 32), top = wave_max_u(hi);
    unsigned long long who = __ballot(hi == top);
    if (__popcll(who) > 1) {
        const uint32_t lo = hi == top ? (uint32_t)key : 0u, most = wave_max_u(lo);
        if (top == 0 && most == 0) return -1;
        who = __ballot(hi == top && lo == most);
    }
    return __ffsll(who) - 1;
}
// A score as a key that orders as it does; 0 for none.
__device__ __forceinline__ unsigned long long score_key(double s) {
    const unsigned long long u = (unsigned long long)__double_as_longlong(s);
    return (u >> 63) ? ~u : u | 0x8000000000000000ull;
}

__device__ __forceinline__ double key_score(unsigned long long k) {
    return __longlong_as_double((long long)((k >> 63) ? k ^ 0x8000000000000000ull : ~k));
}

constexpr int kMergeWaves = 16;
constexpr int kHeads = 8;       // entries of each list read at once
constexpr int kListLds = 512;   // keys of a row that a wave can sort in LDS
constexpr int kPickLds = 2048;  // picks of a sequence's rows that LDS holds
constexpr int kPoolLds = 2048;  // picks that the last sort takes

// Depth and count for a bound over `lists` sorted lists: `count` lists whose entry at `depth` reaches
// the bound hold k entries that do.
struct Cut {
    int depth, count;
};
__device__ __forceinline__ Cut cut_of(int lists, int k) {
    const int deep = min(k, (2 * k + lists - 1) / lists);
    return Cut{deep - 1, (k + deep - 1) / deep};
}
// Position of this lane among the lanes that `yes`, and their number.
__device__ __forceinline__ int lane_rank(unsigned long long yes) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(yes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)yes, 0u));
}

// One sequence.  Waves merge rows' lists, a list per lane: the entries that reach a bound (cut_of) are
// sorted by counting the larger ones.  Other waves add up the rows' sums meanwhile.  Then the rows'
// picks are merged, a row per lane, the same way.  Where more reach a bound than LDS holds (the best
// logits all in a few slices) the lists are merged step by step: the lane with the largest head gives
// the next one and moves on.
// What bounds it is latency: a handful of dependent reads and counts, not bytes.
__global__ __launch_bounds__(64 * kMergeWaves) void select_merge_kernel(SelArgs A) {
    __shared__ union {
        unsigned long long list[kMergeWaves][kListLds];
        struct {
            unsigned long long key[kPoolLds];
            uint32_t from[kPoolLds];  // row of the sequence << 8 | place among its picks
        } pool;
    } sh;
    __shared__ unsigned long long pick[kPickLds];  // logit keys, then score keys
    __shared__ int pick_token[kPickLds];
    __shared__ double row_lse[kMaxBeams];
    __shared__ float row_top[kMaxBeams], row_score[kMaxBeams];
    __shared__ int picks[kMaxBeams], ended[kMaxBeams];
    __shared__ int pool_n;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const int seq = blockIdx.x, row0 = seq * A.beams, S = A.slices, k = A.k;
    const int depth = min(k, kPickLds / A.beams);
    const bool mine = (int)lane < S;
    for (int task = wave; task < 2 * A.beams; task += kMergeWaves) {
        const int b = task < A.beams ? task : task - A.beams, row = row0 + b;
        const size_t base = (size_t)row * S;
        if (task >= A.beams) {
            const float2 st = mine ? A.stat[base + lane] : make_float2(-INFINITY, 0.0f);
            const float score = A.scores[row];
            const float top = wave_max_f(st.x);
            // (in 64 bits: scores of different rows are told apart by the sum's last bits)
            double sum = st.x > -INFINITY ? (double)st.y * exp((double)st.x - (double)top) : 0.0;
            for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, kWave);
            if (lane == 0) {
                row_top[b] = top;
                row_lse[b] = log(sum);
                row_score[b] = score;
            }
            continue;
        }
        const unsigned long long *list = A.keys + (base + min((int)lane, S - 1)) * k;
        const Cut cut = cut_of(S, k);
        const float score = A.scores[row];
        const bool over = A.done && A.done[row] != 0;
        unsigned long long deep = list[cut.depth];
        unsigned long long head[kHeads];  // (nearly always all that reaches the bound)
#pragma unroll
        for (int j = 0; j < kHeads; j++) head[j] = list[min(j, k - 1)];
#pragma unroll
        for (int j = 0; j < kHeads; j++) head[j] = mine && j < k ? head[j] : 0;
        deep = mine ? deep : 0;
        const unsigned long long bound = wave_kth((uint32_t)(deep >> 32), key_token(deep), cut.count);
        int found = 0;
        const auto keep = [&](unsigned long long key) {
            const unsigned long long yes = __ballot(key != 0 && key >= bound);
            const int at = found + lane_rank(yes);
            if (((yes >> lane) & 1) && at < kListLds) sh.list[wave][at] = key;
            found += __popcll(yes);
            return yes != 0;
        };
#pragma unroll
        for (int j = 0; j < kHeads; j++) keep(head[j]);
        if (__ballot(head[kHeads - 1] != 0 && head[kHeads - 1] >= bound))
            for (int j = kHeads; j < k; j++)
                if (!keep(mine ? list[j] : 0)) break;
        const auto put = [&](int n, unsigned long long key) {
            if (n < depth) pick[b * depth + n] = key;
            else A.far[(size_t)row * k + n] = key;
        };
        int n = min(found, k);
        if (found <= kListLds) {
            for (int c = (int)lane; c < found; c += 64) {
                const unsigned long long key = sh.list[wave][c];
                int rank = 0;
#pragma unroll 8
                for (int i = 0; i < found; i++) rank += sh.list[wave][i] > key ? 1 : 0;
                if (rank < k) put(rank, key);
            }
        } else {
            int at = 0;
            unsigned long long cur = head[0];
            for (n = 0; n < k; n++) {
                const int who = wave_best(cur);
                if (who < 0) break;
                if ((int)lane == who) {
                    put(n, cur);
                    at++;
                    cur = at < k ? list[at] : 0;
                }
            }
        }
        if (!(score > -INFINITY)) n = 0;
        else if (over) n = 1;
        if (lane == 0) {
            picks[b] = n;
            ended[b] = over;
        }
    }
    __syncthreads();
    // logit keys to score keys (never 0) and tokens
    const auto scored = [&](int b, unsigned long long key) {
        if (ended[b]) return score_key((double)row_score[b]);
        return score_key((double)row_score[b] + (((double)key_logit(key) - (double)row_top[b]) - row_lse[b]));
    };
    for (int i = (int)tid; i < A.beams * k; i += 64 * kMergeWaves) {
        const int b = i / k, n = i % k;
        if (n >= picks[b]) continue;
        if (n < depth) {
            const unsigned long long key = pick[b * depth + n];
            pick[b * depth + n] = scored(b, key);
            pick_token[b * depth + n] = ended[b] ? A.eos : (int)key_token(key);
        } else {
            const size_t at = (size_t)(row0 + b) * k + n;
            const unsigned long long key = A.far[at];
            A.far[at] = scored(b, key);
            A.far_token[at] = (int)key_token(key);
        }
    }
    __syncthreads();
    const auto score_at = [&](int b, int i) {
        if (i < depth) return ld_lds(&pick[b * depth + i]);
        return ld_global(A.far + (size_t)(row0 + b) * k + i);
    };
    const auto give = [&](int n, unsigned long long key, int b, int i) {
        const int token = i < depth ? ld_lds(&pick_token[b * depth + i]) : ld_global(A.far_token + (size_t)(row0 + b) * k + i);
        const size_t out = (size_t)seq * k + n;
        A.o_scores[out] = (float)key_score(key);
        A.o_tokens[out] = token;
        A.o_parents[out] = row0 + b;
        if (A.o_done) A.o_done[out] = ended[b] || token == A.eos;
    };
    if (wave == 0) {
        const int held = (int)lane < A.beams ? picks[lane] : 0;
        const Cut cut = cut_of(A.beams, k);
        // (a bound on the upper half of the key: a few more pass)
        const uint32_t deep = cut.depth < held ? (uint32_t)(score_at((int)lane, cut.depth) >> 32) : 0u;
        const unsigned long long bound = wave_kth(deep, lane, cut.count) & 0xFFFFFFFF00000000ull;
        int found = 0;
        for (int j = 0; j < k; j++) {
            const unsigned long long key = j < held ? score_at((int)lane, j) : 0;
            const unsigned long long yes = __ballot(key != 0 && key >= bound);
            if (!yes) break;
            const int at = found + lane_rank(yes);
            if (((yes >> lane) & 1) && at < kPoolLds) {
                sh.pool.key[at] = key;
                sh.pool.from[at] = (lane << 8) | (uint32_t)j;
            }
            found += __popcll(yes);
        }
        if (lane == 0) pool_n = found;
        if (found > kPoolLds) {
            int at = 0;
            unsigned long long key = held > 0 ? score_at((int)lane, 0) : 0;
            for (int n = 0; n < k; n++) {
                const int who = wave_best(key);  // (equal scores: the lower lane, so the lower row)
                if (who < 0) break;
                if ((int)lane == who) {
                    give(n, key, who, at);
                    at++;
                    key = at < held ? score_at(who, at) : 0;
                }
            }
        }
    }
    __syncthreads();
    const int found = pool_n;
    if (found > kPoolLds) return;  // (more than k: no place was left over)
    for (int c = (int)tid; c < found; c += 64 * kMergeWaves) {
        const unsigned long long key = sh.pool.key[c];
        const uint32_t from = sh.pool.from[c];
        int rank = 0;
#pragma unroll 8
        for (int i = 0; i < found; i++)
            rank += sh.pool.key[i] > key || (sh.pool.key[i] == key && sh.pool.from[i] < from) ? 1 : 0;
        if (rank < k) give(rank, key, (int)(from >> 8), (int)(from & 255u));
    }
    for (int n = found + (int)tid; n < k; n += 64 * kMergeWaves) {
        const size_t out = (size_t)seq * k + n;
        A.o_scores[out] = -INFINITY;
        A.o_tokens[out] = max(A.eos, 0);
        A.o_parents[out] = row0;
        if (A.o_done) A.o_done[out] = 1;
    }
}

int slices_of(int vocab) { return (vocab + kSlice - 1) / kSlice; }

void check_select(k2t_ctx *ctx, int n_seq, int beams, int vocab, int k) {
    branch_arg(ctx != nullptr, "ctx is NULL");
    branch_arg(beams >= 1 && beams <= kMaxBeams, "beams must be 1 .. 64");
    branch_arg(k >= 1 && k <= kMaxPicks, "k must be 1 .. 128");
    branch_arg(n_seq >= 0 && (size_t)n_seq * beams <= 65535, "n_seq * beams must be 0 .. 65535");
    static_assert(kMaxSelectVocab == 64 * kSlice, "a lane per slice");
    branch_arg(vocab >= 1 && vocab <= kMaxSelectVocab, "vocab must be 1 .. 262144");
}

}  // namespace

size_t beam_select_ws_bytes(int n_seq, int beams, int vocab, int k) {
    const size_t lists = (size_t)n_seq * beams * slices_of(vocab);
    return lists * (sizeof(float2) + (size_t)k * sizeof(unsigned long long)) + (size_t)n_seq * beams * k * 12 + 16;
}

void launch_beam_select(hipStream_t st, const float *logits, int vocab, size_t row_stride, const float *scores,
                        const int *done, int n_seq, int beams, int k, int eos, float *out_scores, int *out_tokens,
                        int *out_parents, int *out_done, void *ws) {
    SelArgs A{logits, row_stride, vocab, slices_of(vocab), beams, k, eos, scores, done, nullptr, nullptr, nullptr, nullptr,
              out_scores, out_tokens, out_parents, out_done};
    const size_t lists = (size_t)n_seq * beams * A.slices;
    A.stat = (float2 *)ws;
    A.keys = (unsigned long long *)(A.stat + lists);
    A.far = A.keys + lists * k;
    A.far_token = (int *)(A.far + (size_t)n_seq * beams * k);
    hipLaunchKernelGGL(select_slice_kernel, dim3(A.slices, n_seq * beams), dim3(kSelThreads), 0, st, A);
    hip_check(hipGetLastError(), "beam_select launch");
    hipLaunchKernelGGL(select_merge_kernel, dim3(n_seq), dim3(64 * kMergeWaves), 0, st, A);
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
