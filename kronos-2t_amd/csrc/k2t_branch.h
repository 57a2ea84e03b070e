// Several continuations of one prompt (k2t_kv_append / load / reorder, k2t_attn_shared,
// k2t_beam_select): what their entry points and the engine's beam search share.
#pragma once

#include <string>

#include "k2t_internal.h"

namespace k2t {

constexpr int kMaxBeams = 64, kMaxPicks = 128, kMaxSelectVocab = 262144;

inline void branch_arg(bool ok, const char *msg) {
    if (!ok) throw Error(K2T_E_ARG, msg);
}

// An entry point's body: no exception crosses the C ABI.
template <typename F>
int32_t branch_guard(F &&fn) {
    try {
        fn();
        return K2T_OK;
    } catch (const Error &e) {
        set_last_error(e.what());
        return e.code;
    } catch (const std::exception &e) {
        set_last_error(e.what());
        return K2T_E_INTERNAL;
    } catch (...) {
        set_last_error("unknown error");
        return K2T_E_INTERNAL;
    }
}

// Checks of a batched cache (k2t_kv_rows) that is read or written with wide accesses.
void check_kv_rows(const k2t_kv_rows *kv, int bits, int hd);

void launch_kv_reorder(hipStream_t st, int bits, const k2t_kv_rows &kv, const int *parents, int n_layers, int n_seq,
                       int beams, int nkv, int hd);

struct SharedShape {
    int n_seq, beams, nq, nkv, hd;
};
// Workspace for caches of up to these lengths.
size_t attn_shared_ws_bytes(const k2t_ctx *ctx, const SharedShape &s, int prefix_len, int tail_len);
// prefix / tail: their row caches' descriptions (cap 0: none); the layer's block is the caller's
// pointer arithmetic (kv_rows_at).
void launch_attn_shared(k2t_ctx *ctx, hipStream_t st, int bits, const float *q, size_t q_stride, const SharedShape &s,
                        const k2t_kv_rows &prefix, const k2t_kv_rows &tail, float attn_scale, float *out, void *ws);
// The cache `slots` slots further on.
inline k2t_kv_rows kv_rows_at(const k2t_kv_rows &kv, int bits, int hd, size_t slots) {
    k2t_kv_rows r = kv;
    const size_t code = slots * (size_t)(bits == 8 ? hd : hd / 2), scale = slots * (size_t)(bits == 8 ? 4 : hd / 32);
    r.kq = static_cast<char *>(kv.kq) + code;
    r.vq = static_cast<char *>(kv.vq) + code;
    r.ks = static_cast<char *>(kv.ks) + scale;
    r.vs = static_cast<char *>(kv.vs) + scale;
    return r;
}

size_t beam_select_ws_bytes(int n_seq, int beams, int vocab, int k);
void launch_beam_select(hipStream_t st, const float *logits, int vocab, size_t row_stride, const float *scores,
                        const int *done, int n_seq, int beams, int k, int eos, float *out_scores, int *out_tokens,
                        int *out_parents, int *out_done, void *ws);

}  // namespace k2t
