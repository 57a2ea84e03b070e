// Rotary positions of the heads of a block of tokens (k2t_rope), and the plans that hold their frequencies.
//
// For a token at position p, pair i of a head (x0, x1) becomes
//   (x0 c - x1 s, x1 c + x0 s),  c = scale cos(2 pi p turns[i]),  s = scale sin(2 pi p turns[i]).
// Fractions of a turn are what the sine needs, and p turns[i] leaves few bits of them in fp32 from some 10^4
// positions on: product, reduction to a quarter turn and series are 64-bit, and each value is rounded once.
//
// A workgroup takes a few tokens: its threads work out the tokens' angles once, into LDS, while their first loads are
// under way, then rotate eight elements (four pairs) at a time.
//
// What bounds it: bytes. 6 rows of 389 to 777 tokens, 36 heads x 128 (129 MB read and written): 21 to 23 us, 5.5 to 6 TB/s (the
// inputs partly from the Infinity Cache); 34.7 with one piece in flight per thread and cached stores. 6 rows of 777, 168 MB: 28.5 to
// 30.7, interleaved 28.9 to 31.8 (49.9 with a thread's two pieces side by side), rot_dim 98, halves, a pair at a time, 54 (4 bytes
// per lane and access, since the halves of such a head do not begin at the same alignment).
// One token of 4 rows, 12 heads x 64: 3.6 us, a launch and the chain from position to angle to output.
#include <math.h>

#include <algorithm>

#include "k2t_branch.h"
#include "k2t_device.h"

namespace k2t {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct RopeArgs {
    const float *x;
    float *out;
    size_t x_stride, out_stride;
    int ntok, tokens, per;  // tokens of a row, of the call, of a workgroup
    int units;              // units of VEC elements in a token's heads
    int hd_shift;           // log2(hd / VEC)
    int hd;
    const int *pos, *depth, *counts;
    k2t_rope_plan plan;
};

// cos and sin of `turn` turns, times scale: the fraction to the nearest quarter is at most 1/8 turn, where the series
// below are off by less than 2^-33.
__device__ __forceinline__ float2 turn_cos_sin(double turn, double scale) {
    const double quarters = turn * 4.0, n = rint(quarters);
    const double r = (quarters - n) * 1.5707963267948966, r2 = r * r;
    const double s = r * fma(r2, fma(r2, fma(r2, fma(r2, fma(r2, -1.0 / 39916800, 1.0 / 362880), -1.0 / 5040), 1.0 / 120), -1.0 / 6), 1.0);
    const double c = fma(r2, fma(r2, fma(r2, fma(r2, fma(r2, -1.0 / 3628800, 1.0 / 40320), -1.0 / 720), 1.0 / 24), -0.5), 1.0);
    const int k = (int)((long long)n & 3);
    const double a = k & 1 ? s : c, b = k & 1 ? c : s;
    return make_float2((float)((k == 1 || k == 2 ? -a : a) * scale), (float)((k >= 2 ? -b : b) * scale));
}

// Where unit u's two halves lie in a head: of VEC / 2 elements each, and such that neighbouring units' lie next to each other.
// K2T_ROPE_HALF: first and second members of the same pairs, then halves of what is behind rot_dim.  INTERLEAVED: whole
// pairs each, of all of the head.
template <int VEC>
__device__ __forceinline__ void unit_at(const k2t_rope_plan &P, int hd, int u, int &a, int &b) {
    constexpr int H = VEC / 2;
    if (P.layout == K2T_ROPE_INTERLEAVED) {
        a = H * u;
        b = a + hd / 2;
    } else if (VEC * u < P.rot_dim) {
        a = H * u;
        b = a + P.rot_dim / 2;
    } else {
        a = P.rot_dim + H * (u - P.rot_dim / VEC);
        b = a + (hd - P.rot_dim) / 2;
    }
}

constexpr int kMaxPer = 3, kFlight = 4;  // tokens of a workgroup, whose angles wait in LDS; units in flight per thread

// VEC 8: units of two 16-byte pieces; VEC 2: K2T_ROPE_HALF whose rot_dim is no multiple of 8, a pair at a time.
template <int VEC>
__global__ __launch_bounds__(256) void rope_kernel(const RopeArgs A) {
    constexpr int H = VEC / 2;
    __shared__ __align__(16) float cs[kMaxPer][2][64];
    const int tid = (int)threadIdx.x, first = (int)blockIdx.x * A.per, n = min(A.per, A.tokens - first);
    const int pairs = A.plan.rot_dim / 2, total = n * A.units;
    const bool moved = A.out != A.x;
    struct Piece {
        f32x4 a, b;
    };
    const auto live = [&](int token) {
        const int row = token / A.ntok;
        return !A.counts || token - row * A.ntok < A.counts[row];
    };
    // (a workgroup whose tokens its rows do not have; one of them is loaded even so where others are there)
    bool some = false;
    for (int t = 0; t < n; t++) some |= live(first + t);
    if (!some) return;
    const auto load = [&](int g, Piece &p) {
        const int t = g / A.units, u = g - t * A.units, head = u >> A.hd_shift, e = u & ((1 << A.hd_shift) - 1);
        int a, b;
        unit_at<VEC>(A.plan, A.hd, e, a, b);
        const float *x = A.x + (size_t)(first + t) * A.x_stride + (size_t)head * A.hd;
        if constexpr (VEC == 8) {
            p.a = *reinterpret_cast<const f32x4 *>(x + a);
            p.b = *reinterpret_cast<const f32x4 *>(x + b);
        } else {
            p.a[0] = x[a];
            p.b[0] = x[b];
        }
    };
    const auto rotate = [&](int g, const Piece &p) {
        const int t = g / A.units, u = g - t * A.units, head = u >> A.hd_shift, e = u & ((1 << A.hd_shift) - 1);
        int a, b;
        unit_at<VEC>(A.plan, A.hd, e, a, b);
        const bool turns = a < A.plan.rot_dim;
        if (!live(first + t) || (!turns && !moved)) return;
        float *o = A.out + (size_t)(first + t) * A.out_stride + (size_t)head * A.hd;
        float x[VEC], y[VEC];
#pragma unroll
        for (int j = 0; j < H; j++) {
            x[j] = p.a[j];
            x[H + j] = p.b[j];
            y[j] = x[j];
            y[H + j] = x[H + j];
        }
        if (VEC == 8 && A.plan.layout == K2T_ROPE_INTERLEAVED) {
#pragma unroll
            for (int j = 0; j < H; j++) {
                const int pair = (j < H / 2 ? a : b) / 2 + j % (H / 2);
                if (pair >= pairs) continue;
                const float c = cs[t][0][pair], s = cs[t][1][pair];
                y[2 * j] = x[2 * j] * c - x[2 * j + 1] * s;
                y[2 * j + 1] = x[2 * j + 1] * c + x[2 * j] * s;
            }
        } else if (turns) {
#pragma unroll
            for (int j = 0; j < H; j++) {
                const float c = cs[t][0][H * e + j], s = cs[t][1][H * e + j];
                y[j] = x[j] * c - x[H + j] * s;
                y[H + j] = x[H + j] * c + x[j] * s;
            }
        }
        if constexpr (VEC == 8) {
            __builtin_nontemporal_store((f32x4{y[0], y[1], y[2], y[3]}), reinterpret_cast<f32x4 *>(o + a));
            __builtin_nontemporal_store((f32x4{y[4], y[5], y[6], y[7]}), reinterpret_cast<f32x4 *>(o + b));
        } else {
            o[a] = y[0];
            o[b] = y[1];
        }
    };
    Piece p[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; k++) load(min(tid + 256 * k, total - 1), p[k]);
    for (int i = tid; i < n * pairs; i += 256) {
        const int t = i / pairs, j = i - t * pairs, token = first + t, row = token / A.ntok;
        const long long at = (long long)A.pos[row] + (A.depth ? A.depth[token] : token - row * A.ntok);
        const float2 v = turn_cos_sin((double)at * A.plan.turns[j], A.plan.scale);
        cs[t][0][j] = v.x;
        cs[t][1][j] = v.y;
    }
    __syncthreads();
    for (int g = tid; g < total; g += 256 * kFlight) {
        if (g > tid) {
#pragma unroll
            for (int k = 0; k < kFlight; k++) load(min(g + 256 * k, total - 1), p[k]);
        }
#pragma unroll
        for (int k = 0; k < kFlight; k++)
            if (g + 256 * k < total) rotate(g + 256 * k, p[k]);
    }
}

}  // namespace

}  // namespace k2t

using namespace k2t;

extern "C" {

int32_t k2t_rope_plan_make(const k2t_rope_config *cfg, k2t_rope_plan *out) {
    return branch_guard([&] {
        branch_arg(cfg && out, "NULL argument");
        const k2t_rope_config &c = *cfg;
        branch_arg(c.layout == K2T_ROPE_HALF || c.layout == K2T_ROPE_INTERLEAVED, "unknown layout");
        branch_arg(c.rot_dim >= 2 && c.rot_dim <= 128 && c.rot_dim % 2 == 0, "rot_dim must be even, 2 .. 128");
        branch_arg(c.scaling >= K2T_ROPE_PLAIN && c.scaling <= K2T_ROPE_WAVE, "unknown scaling");
        const bool ends = c.scaling == K2T_ROPE_RAMP || c.scaling == K2T_ROPE_WAVE;
        branch_arg(std::isfinite(c.theta) && c.theta >= 1.0 && (c.scaling != K2T_ROPE_RAMP || c.theta > 1.0),
                   "theta must be finite and at least 1 (above 1 for K2T_ROPE_RAMP)");
        branch_arg(c.scaling == K2T_ROPE_PLAIN || (std::isfinite(c.factor) && c.factor > 0.0), "factor must be positive");
        branch_arg(c.scaling != K2T_ROPE_BASE || c.rot_dim > 2, "K2T_ROPE_BASE needs rot_dim above 2");
        double low = c.low, high = c.high;
        if (low == 0.0 && high == 0.0) {
            low = 1.0;
            high = c.scaling == K2T_ROPE_RAMP ? 32.0 : 4.0;
        }
        branch_arg(!ends || (c.original > 0 && low > 0.0 && high > low && std::isfinite(high)),
                   "original must be positive, and 0 < low < high");
        const double two_pi = 6.283185307179586, d = c.rot_dim;
        const double theta = c.scaling == K2T_ROPE_BASE ? c.theta * std::pow(c.factor, d / (d - 2.0)) : c.theta;
        k2t_rope_plan P{};
        P.layout = c.layout;
        P.rot_dim = c.rot_dim;
        P.scale = c.scaling == K2T_ROPE_RAMP ? 0.1 * std::log(c.factor) + 1.0 : 1.0;
        for (int i = 0; i < c.rot_dim / 2; i++) {
            double f = std::pow(theta, -2.0 * i / d);
            // the share of the unstretched frequency
            double keep = c.scaling == K2T_ROPE_LINEAR ? 0.0 : 1.0;
            if (c.scaling == K2T_ROPE_RAMP) {
                // the pair (a fraction) that makes `turns` turns over the original positions
                const auto pair = [&](double turns) { return d * std::log(c.original / (turns * two_pi)) / (2.0 * std::log(theta)); };
                const double a = std::max(std::floor(pair(high)), 0.0), b = std::min(std::ceil(pair(low)), d - 1.0);
                keep = 1.0 - std::min(std::max((i - a) / std::max(b - a, 0.001), 0.0), 1.0);
            } else if (c.scaling == K2T_ROPE_WAVE) {
                keep = std::min(std::max((c.original * f / two_pi - low) / (high - low), 0.0), 1.0);
            }
            if (keep < 1.0) f = f / c.factor * (1.0 - keep) + f * keep;
            P.turns[i] = f / two_pi;
            branch_arg(std::isfinite(P.turns[i]) && P.turns[i] <= 1.0, "a pair turns more than once per position");
        }
        branch_arg(std::isfinite(P.scale), "factor out of range");
        *out = P;
    });
}

int32_t k2t_rope(k2t_ctx *ctx, const float *d_x, size_t x_stride, int32_t batch, int32_t ntok, int32_t n_heads,
                 int32_t head_dim, const int32_t *d_pos, const int32_t *d_depth, const int32_t *d_counts,
                 const k2t_rope_plan *plan, float *d_out, size_t out_stride) {
    return branch_guard([&] {
        branch_arg(ctx && plan, "NULL argument");
        branch_arg(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
        branch_arg(batch >= 0 && batch <= 65535 && ntok >= 0 && n_heads > 0 && n_heads <= 2048,
                   "batch must be 0 .. 65535, ntok >= 0, n_heads 1 .. 2048");
        branch_arg((size_t)batch * ntok * n_heads <= (size_t)1 << 24, "more than 2^24 heads in one call");
        branch_arg(plan->layout == K2T_ROPE_HALF || plan->layout == K2T_ROPE_INTERLEAVED, "unknown layout");
        branch_arg(plan->rot_dim >= 2 && plan->rot_dim <= head_dim && plan->rot_dim % 2 == 0,
                   "rot_dim must be even, 2 .. head_dim");
        branch_arg(std::isfinite(plan->scale), "the plan's scale is not finite");
        for (int i = 0; i < plan->rot_dim / 2; i++)
            branch_arg(std::fabs(plan->turns[i]) <= 1.0, "the plan's turns must be within +-1");
        const size_t width = (size_t)n_heads * head_dim;
        branch_arg(x_stride >= width && out_stride >= width && x_stride % 4 == 0 && out_stride % 4 == 0,
                   "a stride is smaller than the heads, or no multiple of 4");
        branch_arg(x_stride < (size_t)1 << 40 && out_stride < (size_t)1 << 40, "a stride is out of range");
        if (batch == 0 || ntok == 0) return;
        branch_arg(d_x && d_out && d_pos, "NULL argument");
        branch_arg((reinterpret_cast<uintptr_t>(d_x) | reinterpret_cast<uintptr_t>(d_out)) % 16 == 0,
                   "d_x and d_out must be 16-byte aligned");
        branch_arg(d_x != d_out || x_stride == out_stride, "in place the strides must be the same");
        hip_check(hipSetDevice(ctx->device), "hipSetDevice");
        const bool wide = plan->rot_dim % 8 == 0 || plan->layout == K2T_ROPE_INTERLEAVED;
        RopeArgs A{};
        A.x = d_x;
        A.out = d_out;
        A.x_stride = x_stride;
        A.out_stride = out_stride;
        A.ntok = ntok;
        A.tokens = batch * ntok;
        A.per = std::min(std::max(A.tokens / (4 * std::max(1, ctx->num_cus)), 1), kMaxPer);
        A.hd = head_dim;
        A.hd_shift = (head_dim == 128 ? 7 : 6) - (wide ? 3 : 1);
        A.units = n_heads << A.hd_shift;
        A.pos = d_pos;
        A.depth = d_depth;
        A.counts = d_counts;
        A.plan = *plan;
        const dim3 grid((unsigned)((A.tokens + A.per - 1) / A.per));
        if (wide) hipLaunchKernelGGL((rope_kernel<8>), grid, dim3(256), 0, ctx->stream, A);
        else hipLaunchKernelGGL((rope_kernel<2>), grid, dim3(256), 0, ctx->stream, A);
        hip_check(hipGetLastError(), "rope launch");
    });
}

}  // extern "C"
