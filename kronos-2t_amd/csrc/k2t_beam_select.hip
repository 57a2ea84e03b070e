// Beam search's choice over the rows of a sequence and the vocabulary (k2t_beam_select): the k largest of
// score[r] + (x[r][t] - max x[r]) - log sum_t exp(x[r][t] - max x[r]), in two launches.  Every slice of 4096
// logits leaves its maximum, its sum of exponentials and its k best, sorted; one workgroup per sequence
// adds a row's slices up, and chooses among the entries of all rows' lists.
//
// A slice is read once into registers.  Its k best are among the elements that reach a bound: each of
// the four waves finds a bound that k/4 of its 64 threads' maxima reach, and at least k elements reach
// the smallest of the four; in random logits few more do.  They are sorted by counting, for each, the
// larger ones.  Everything that orders is a unique key, so the result depends on no timing.
//
// What bounds it: the logits have to be read once (12.6 MB at 8 sequences of 8 rows of 49152: 2.4 us), but
// both kernels take longer than their bytes, the first for its instructions (some 30 vector ones per logit of a lane on 3
// waves per SIMD: 6.0 us there, 8.3 us before exp came down to one v_exp_f32 and keys were only made
// for what reaches the bound), the second for chains of dependent steps on one CU (6.6 us there; 9.0 us
// for 16 rows of 151936, k 32).  Both: 8.9 us for one sequence of 4 rows of 8192, 13.3 us and 15.4 us.
// With slices of 4096, 22 rows of 49152 give every CU a workgroup; larger ones would leave more CUs idle under
// fewer rows, and smaller ones repeat a slice's fixed part (bound, sums, sort: about half of it).
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
    unsigned long long *keys;  // [row][k][slice], best first, 0 behind the last
    float *o_scores;
    int *o_tokens, *o_parents, *o_done;
};

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
// Up to this many a bound is found maximum by maximum, beyond by bits (which took 9.4, 13.9 and 16.0 us where
// it is 8.8, 13.4 and 15.4 now, in the three cases above; up to 8: no difference from 3).
constexpr int kFewMaxima = 3;

// A bound that at least r of a wave's keys reach (`ord` the logit's order, 0 for none, `token` unique)
// and hardly any other; 0 where fewer than r lanes have one.
__device__ __forceinline__ unsigned long long wave_kth(uint32_t ord, uint32_t token, int r) {
    uint32_t t = 0;
    if (r <= kFewMaxima) {  // maximum by maximum
        while (true) {
            t = wave_max_u(ord);
            r -= __popcll(__ballot(ord == t));
            if (r <= 0 || t == 0) return (unsigned long long)t << 32;
            ord = ord == t ? 0 : ord;
        }
    }
#pragma unroll
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t c = t | (1u << bit);
        const int n = __popcll(__ballot(ord >= c));
        if (n >= r) t = c;
        if (n == r) return (unsigned long long)t << 32;  // (nearly always within a dozen bits)
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

// Position of this lane among the lanes that `yes`.
__device__ __forceinline__ int lane_rank(unsigned long long yes) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(yes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)yes, 0u));
}

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // (rows start at any float)

// One slice of one row: its maximum, its sum of exponentials and its k best logits.
__global__ __launch_bounds__(kSelThreads) void select_slice_kernel(SelArgs A) {
    constexpr int kSelWaves = kSelThreads / 64;
    __shared__ unsigned long long list[kSlice];
    __shared__ unsigned long long wave_top[kSelWaves];
    __shared__ uint32_t bound[kSelWaves];
    __shared__ float redf[2 * kSelWaves];
    __shared__ int count;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
    const int slice = blockIdx.x, row = blockIdx.y;
    const float *x = A.logits + (size_t)row * A.row_stride;
    // a thread's tokens: four in a row, 1024 apart; in a slice that the vocabulary ends in 256 apart, so
    // that what there is goes to all threads
    const bool whole = (slice + 1) * kSlice <= A.vocab;
    const int first = slice * kSlice + (whole ? 4 : 1) * (int)tid, step = whole ? 1 : kSelThreads;
    const auto token_of = [&](int i) { return first + i / 4 * (4 * kSelThreads) + i % 4 * step; };
    float v[kSelPer];
    if (whole) {
#pragma unroll
        for (int j = 0; j < kSelPer; j += 4) {
            const f32x4u w = *reinterpret_cast<const f32x4u *>(x + token_of(j));
            for (int e = 0; e < 4; e++) v[j + e] = w[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < kSelPer; i++) v[i] = x[min(token_of(i), A.vocab - 1)];
#pragma unroll
        for (int i = 0; i < kSelPer; i++) v[i] = token_of(i) < A.vocab ? v[i] : -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < kSelPer; i++) {
        v[i] = fminf(fmaxf(v[i], -INFINITY), FLT_MAX);  // (the larger of NaN and -inf is -inf)
        mx = fmaxf(mx, v[i]);
    }
    const uint32_t best = mx > -INFINITY ? (uint32_t)(logit_key(mx, 0) >> 32) : 0u;
    const uint32_t kth = (uint32_t)(wave_kth(best, tid, (A.k + kSelWaves - 1) / kSelWaves) >> 32);
    mx = wave_max_f(mx);
    if (tid == 0) count = 0;
    if (lane == 0) {
        bound[wv] = kth;
        redf[wv] = mx;
    }
    __syncthreads();
    uint32_t least = bound[0];
    mx = redf[0];
#pragma unroll
    for (int w = 1; w < kSelWaves; w++) {
        least = min(least, bound[w]);
        mx = fmaxf(mx, redf[w]);
    }
    // (a wave without enough maxima: every logit but -inf)
    const float pass = least ? key_logit((unsigned long long)least << 32) : -FLT_MAX;
    // A slice's sum is fp32 and off by less than 2^-18 of itself: v_exp_f32 by 2^-23; its argument's difference,
    // product and log2 e by 2.7 x 2^-24 of an exponent whose mean, by weight, is at most log 4096; 26 additions
    // on end.  From here on, over slices, rows and candidates, everything is 64 bits.
    const float from = mx > -INFINITY ? mx : 0.0f;
    float sum = 0.0f;
    unsigned long long yes[kSelPer];
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kSelPer; i++) {
        sum += __builtin_amdgcn_exp2f((v[i] - from) * 1.4426950408889634f);
        yes[i] = __ballot(v[i] >= pass);
        mine += __popcll(yes[i]);
    }
    int at = 0;
    if (lane == 0) at = atomicAdd(&count, mine);  // (their order does not matter: sorted below)
    at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
    for (int i = 0; i < kSelPer; i++) {
        if (yes[i] == 0) continue;
        if ((yes[i] >> lane) & 1) list[at + lane_rank(yes[i])] = logit_key(v[i], (uint32_t)token_of(i));
        at += __popcll(yes[i]);
    }
    sum = wave_sum_f(sum);
    if (lane == 0) redf[kSelWaves + wv] = sum;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0f;
        for (int w = 0; w < kSelWaves; w++) sum += redf[kSelWaves + w];
        A.stat[(size_t)row * A.slices + slice] = make_float2(mx, sum);
    }
    unsigned long long *keys = A.keys + (size_t)row * A.k * A.slices + slice;
    const int n = count;
    for (int c = n + (int)tid; c < A.k; c += kSelThreads) keys[(size_t)c * A.slices] = 0;
    if (n <= kSlice / 4) {
        for (int c = (int)tid; c < n; c += kSelThreads) {
            const unsigned long long key = list[c];
            int rank = 0;
#pragma unroll 8
            for (int i = 0; i < n; i++) rank += list[i] > key ? 1 : 0;
            if (rank < A.k) keys[(size_t)rank * A.slices] = key;
        }
        return;
    }
    // equal logits by the hundred: one by one
    unsigned long long last = ~0ull;
    for (int r = 0; r < A.k; r++) {
        unsigned long long top = 0;
        for (int c = (int)tid; c < n; c += kSelThreads) top = list[c] < last && list[c] > top ? list[c] : top;
        for (int m = 32; m >= 1; m >>= 1) {
            const unsigned long long other = __shfl_xor(top, m, kWave);
            top = other > top ? other : top;
        }
        if (lane == 0) wave_top[wv] = top;
        __syncthreads();
        last = wave_top[0];
        for (int w = 1; w < kSelWaves; w++) last = wave_top[w] > last ? wave_top[w] : last;
        if (tid == 0) keys[(size_t)r * A.slices] = last;
        __syncthreads();
    }
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
constexpr int kHeads = 8;      // entries of each list read at once
constexpr int kCands = 14336;  // candidates of a sequence that LDS holds
constexpr int kPool = 1024;    // candidates that the sort takes

// Depth and count for a bound over `lists` sorted lists: `count` lists whose entry at `depth` reaches
// the bound hold k entries that do.
struct Cut {
    int depth, count;
};
__device__ __forceinline__ Cut cut_of(int lists, int k) {
    const int deep = min(k, (3 * k + 2 * lists - 1) / (2 * lists));  // (half as many again pass in random logits)
    return Cut{deep - 1, (k + deep - 1) / deep};
}
// A candidate of row b of the sequence: among equal scores the larger of these goes first (the lower
// row, then the higher logit, then the lower token).
__device__ __forceinline__ unsigned long long cand_of(int b, unsigned long long key) {
    return ((unsigned long long)(kMaxBeams - 1 - b) << 50) | ((key >> 32) << 18) | (key & 0x3FFFFu);
}
__device__ __forceinline__ int cand_row(unsigned long long c) { return kMaxBeams - 1 - (int)(c >> 50); }
__device__ __forceinline__ int cand_token(unsigned long long c) { return 0x3FFFF - (int)(c & 0x3FFFFu); }
__device__ __forceinline__ float cand_logit(unsigned long long c) { return key_logit((c >> 18) << 32); }

// One sequence.  Waves go through rows' lists, a list per lane, for the entries that reach a bound
// (cut_of), while other waves add up the rows' sums.  All rows' entries are then candidates like a
// slice's elements: a bound from each wave's share of them, and those that reach the smallest are
// sorted by counting the better ones, the counting shared out over the waves.  Where more reach a
// row's bound than its share of LDS (the best logits all in a few slices) its k best are taken one by
// one, and likewise the sequence's where more reach the last bound than the sort takes.
// What bounds it is latency and the issue rate of one CU: no bytes to speak of.
__global__ __launch_bounds__(64 * kMergeWaves) void select_merge_kernel(SelArgs A) {
    __shared__ unsigned long long cand[kCands];
    __shared__ ulonglong2 pool[kPool];  // score key, candidate
    __shared__ int pool_rank[kPool];
    __shared__ double row_lse[kMaxBeams];
    __shared__ float row_top[kMaxBeams], row_score[kMaxBeams];
    __shared__ int ended[kMaxBeams];
    __shared__ uint32_t wave_bound[kMergeWaves];
    __shared__ ulonglong2 wave_top[kMergeWaves];
    __shared__ int cands, pool_n;
    static_assert(kCands / kMaxBeams >= kMaxPicks, "every row's share holds its k best");
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const int wave = __builtin_amdgcn_readfirstlane((int)(tid >> 6));
    const int seq = blockIdx.x, row0 = seq * A.beams, S = A.slices, k = A.k;
    const int share = kCands / A.beams;
    const bool mine = (int)lane < S;
    if (tid == 0) cands = pool_n = 0;
    __syncthreads();
    for (int task = wave; task < 2 * A.beams; task += kMergeWaves) {
        const int b = task < A.beams ? task : task - A.beams, row = row0 + b;
        const size_t base = (size_t)row * S;
        if (task >= A.beams) {
            const float2 st = mine ? A.stat[base + lane] : make_float2(-INFINITY, 0.0f);
            const float top = wave_max_f(st.x);
            // (in 64 bits: scores of different rows are told apart by the sum's last bits)
            double sum = st.x > -INFINITY ? (double)st.y * exp((double)st.x - (double)top) : 0.0;
            for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, kWave);
            if (lane == 0) {
                row_top[b] = top;
                row_lse[b] = log(sum);
            }
            continue;
        }
        const unsigned long long *list = A.keys + base * k + min((int)lane, S - 1);  // its entry j: list[j * S]
        const Cut cut = cut_of(S, k);
        const float score = A.scores[row];
        const bool over = A.done && A.done[row] != 0;
        unsigned long long deep = list[cut.depth * S];
        unsigned long long head[kHeads];  // (nearly always all that reaches the bound)
#pragma unroll
        for (int j = 0; j < kHeads; j++) head[j] = list[min(j, k - 1) * S];
#pragma unroll
        for (int j = 0; j < kHeads; j++) head[j] = mine && j < k ? head[j] : 0;
        deep = mine ? deep : 0;
        const unsigned long long bound = wave_kth((uint32_t)(deep >> 32), key_token(deep), cut.count);
        const auto reach = [&](unsigned long long key) { return __ballot(key != 0 && key >= bound); };
        int found = 0;
#pragma unroll
        for (int j = 0; j < kHeads; j++) found += __popcll(reach(head[j]));
        const bool longer = reach(head[kHeads - 1]) != 0;
        for (int j = kHeads; longer && j < k; j++) {
            const unsigned long long yes = reach(mine ? list[j * S] : 0);
            found += __popcll(yes);
            if (!yes) break;
        }
        int n = found <= share ? found : k;
        if (!(score > -INFINITY)) n = 0;
        else if (over) n = 1;
        int at = 0;
        if (lane == 0) {
            at = atomicAdd(&cands, n);  // (their order does not matter)
            row_score[b] = score;
            ended[b] = over;
        }
        at = __builtin_amdgcn_readfirstlane(at);
        if (n == 0) continue;
        if (over) {
            if (lane == 0) cand[at] = cand_of(b, logit_key(0.0f, (uint32_t)A.eos));
        } else if (n == found) {
            const auto keep = [&](unsigned long long key) {
                const unsigned long long yes = reach(key);
                if ((yes >> lane) & 1) cand[at + lane_rank(yes)] = cand_of(b, key);
                at += __popcll(yes);
                return yes != 0;
            };
#pragma unroll
            for (int j = 0; j < kHeads; j++) keep(head[j]);
            for (int j = kHeads; longer && j < k; j++)
                if (!keep(mine ? list[j * S] : 0)) break;
        } else {
            int next = 0;
            unsigned long long cur = head[0];
            for (int i = 0; i < k; i++) {
                if ((int)lane == wave_best(cur)) {
                    cand[at + i] = cand_of(b, cur);
                    next++;
                    cur = next < k ? list[next * S] : 0;
                }
            }
        }
    }
    __syncthreads();
    const int total = cands;
    const auto score_of = [&](unsigned long long c) {  // (never 0)
        const int b = cand_row(c);
        if (ended[b]) return score_key((double)row_score[b]);
        return score_key((double)row_score[b] + (((double)cand_logit(c) - (double)row_top[b]) - row_lse[b]));
    };
    const auto give = [&](int n, unsigned long long score, unsigned long long c) {
        const size_t out = (size_t)seq * k + n;
        const int b = cand_row(c), token = cand_token(c);
        A.o_scores[out] = (float)key_score(score);
        A.o_tokens[out] = token;
        A.o_parents[out] = row0 + b;
        if (A.o_done) A.o_done[out] = ended[b] || token == A.eos;
    };
    // Every wave's share has some of every row's; (rotated: not all lanes on one bank)
    const int first = (int)(lane * kMergeWaves + ((lane + (uint32_t)wave) & (kMergeWaves - 1)));
    unsigned long long c0 = 0, s0 = 0;
    if (first < total) {
        c0 = cand[first];
        s0 = score_of(c0);
    }
    uint32_t best = (uint32_t)(s0 >> 32);
    for (int i = first + 64 * kMergeWaves; i < total; i += 64 * kMergeWaves)
        best = max(best, (uint32_t)(score_of(cand[i]) >> 32));
    const unsigned long long reached = wave_kth(best, lane, (k + kMergeWaves - 1) / kMergeWaves);
    if (lane == 0) wave_bound[wave] = (uint32_t)(reached >> 32);
    __syncthreads();
    uint32_t bound = wave_bound[0];
#pragma unroll
    for (int w = 1; w < kMergeWaves; w++) bound = min(bound, wave_bound[w]);
    const auto enter = [&](unsigned long long score, unsigned long long c) {
        if ((uint32_t)(score >> 32) < bound) return;
        const int at = atomicAdd(&pool_n, 1);  // (their order does not matter: sorted below)
        if (at >= kPool) return;
        pool[at] = make_ulonglong2(score, c);
        pool_rank[at] = 0;
    };
    if (first < total) enter(s0, c0);
    for (int i = first + 64 * kMergeWaves; i < total; i += 64 * kMergeWaves) enter(score_of(cand[i]), cand[i]);
    __syncthreads();
    const int found = pool_n;
    const auto before = [](ulonglong2 x, ulonglong2 y) {
        return (int)(x.x > y.x) | ((int)(x.x == y.x) & (int)(x.y > y.y));
    };
    if (found > kPool) {
        ulonglong2 last = make_ulonglong2(~0ull, ~0ull);
        for (int n = 0; n < k; n++) {  // (k are there)
            ulonglong2 top = make_ulonglong2(0, 0);
            for (int i = (int)tid; i < total; i += 64 * kMergeWaves) {
                const ulonglong2 x = make_ulonglong2(score_of(cand[i]), cand[i]);
                if (before(last, x) && before(x, top)) top = x;
            }
            for (int m = 32; m >= 1; m >>= 1) {
                const ulonglong2 x = make_ulonglong2(__shfl_xor(top.x, m, kWave), __shfl_xor(top.y, m, kWave));
                if (before(x, top)) top = x;
            }
            if (lane == 0) wave_top[wave] = top;
            __syncthreads();
            last = wave_top[0];
            for (int w = 1; w < kMergeWaves; w++)
                if (before(wave_top[w], last)) last = wave_top[w];
            if (tid == 0) give(n, last.x, last.y);
            __syncthreads();
        }
        return;
    }
    // a lane per candidate, the others to compare with shared out over the waves
    const int part = (found + kMergeWaves - 1) / kMergeWaves, lo = wave * part, hi = min(lo + part, found);
    for (int c = (int)lane; c < found; c += 64) {
        const ulonglong2 me = pool[c];
        int rank = 0;
#pragma unroll 4
        for (int i = lo; i < hi; i++) rank += before(pool[i], me);
        if (rank) atomicAdd(&pool_rank[c], rank);
    }
    __syncthreads();
    for (int c = (int)tid; c < found; c += 64 * kMergeWaves)
        if (pool_rank[c] < k) give(pool_rank[c], pool[c].x, pool[c].y);
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
    return lists * (sizeof(float2) + (size_t)k * sizeof(unsigned long long)) + 16;
}

void launch_beam_select(hipStream_t st, const float *logits, int vocab, size_t row_stride, const float *scores,
                        const int *done, int n_seq, int beams, int k, int eos, float *out_scores, int *out_tokens,
                        int *out_parents, int *out_done, void *ws) {
    SelArgs A{logits, row_stride, vocab, slices_of(vocab), beams, k, eos, scores, done, nullptr, nullptr,
              out_scores, out_tokens, out_parents, out_done};
    const size_t lists = (size_t)n_seq * beams * A.slices;
    A.stat = (float2 *)ws;
    A.keys = (unsigned long long *)(A.stat + lists);
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
        branch_arg(k == beams || (d_out_scores != d_scores && (!d_done || d_out_done != d_done)),
                   "scores and done flags may be replaced in place only where k == beams");
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
