// attention_api.hip -- the C boundary of the attention half of a layer: every argument is checked before anything is
// launched.
#include <math.h>

#include "attention_internal.h"
#include "iq4xs_internal.h"
#include "iq4xs_mi355x.h"
#include "linear_internal.h"

using namespace iq4xs;

namespace {

constexpr int64_t MAX_COUNT = (int64_t)1 << 31;

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool given(const void* p) { return p && aligned16(p); }
bool count(int64_t n) { return n > 0 && n < MAX_COUNT; }
bool plain_type(int t) { return t == IQ4XS_TYPE_F32 || t == IQ4XS_TYPE_F16 || t == IQ4XS_TYPE_BF16; }
bool served_head(int d) { return d == 64 || d == 128 || d == 256; }
// A token stride that keeps rows apart and their vectors aligned.
bool stride_of(int64_t s, int64_t heads, int64_t d) { return s >= heads * d && s % 8 == 0 && s < MAX_COUNT; }

int check_cache(const iq4xs_kv_cache* c) {
    if (!c || !given(c->k) || !given(c->v) || !count(c->pages) || c->heads <= 0 || c->head_dim <= 0)
        return hipErrorInvalidValue;
    if (c->page < 16 || (c->page & (c->page - 1)) != 0 || c->pages >= MAX_COUNT / c->page) return hipErrorInvalidValue;
    if (c->type == IQ4XS_TYPE_Q8) {
        if (!given(c->k_scales) || !given(c->v_scales)) return hipErrorInvalidValue;
    } else if (c->type != IQ4XS_TYPE_F16 && c->type != IQ4XS_TYPE_BF16) {
        return hipErrorInvalidValue;
    }
    return served_head(c->head_dim) ? hipSuccess : hipErrorNotSupported;
}

int check_qk(const iq4xs_qk_norm_rope_args* a) {
    if (!a || a->tokens < 0 || a->tokens >= MAX_COUNT || a->q_heads <= 0 || a->k_heads <= 0 || a->head_dim <= 0)
        return hipErrorInvalidValue;
    if (!plain_type(a->in_type) || !plain_type(a->out_type) || !(a->eps >= 0.0f)) return hipErrorInvalidValue;
    if (a->rope != IQ4XS_ROPE_HALF && a->rope != IQ4XS_ROPE_INTERLEAVED) return hipErrorInvalidValue;
    if (a->rot < 0 || a->rot > a->head_dim) return hipErrorInvalidValue;
    if (!aligned16(a->q_gamma) || !aligned16(a->k_gamma)) return hipErrorInvalidValue;
    if (!served_head(a->head_dim) || a->rot % 16 != 0) return hipErrorNotSupported;
    if (a->tokens == 0) return hipSuccess;
    if (!given(a->q) || !given(a->k) || !given(a->q_out) || (a->rot > 0 && (!given(a->freqs) || !a->pos)))
        return hipErrorInvalidValue;
    if (!stride_of(a->q_stride, a->q_heads, a->head_dim) || !stride_of(a->k_stride, a->k_heads, a->head_dim))
        return hipErrorInvalidValue;
    return hipSuccess;
}

int check_attention(const iq4xs_paged_attention_args* a) {
    if (!a) return hipErrorInvalidValue;
    const int err = check_cache(a->cache);
    if (err != hipSuccess) return err;
    const iq4xs_kv_cache& c = *a->cache;
    if (a->q_heads <= 0 || a->q_heads % c.heads != 0 || a->window < 0 || !(a->scale == a->scale))
        return hipErrorInvalidValue;
    if (!plain_type(a->out_type) || (a->type != IQ4XS_TYPE_F16 && a->type != IQ4XS_TYPE_BF16))
        return hipErrorInvalidValue;
    if (c.type != IQ4XS_TYPE_Q8 && c.type != a->type) return hipErrorInvalidValue;
    if (a->total < 0 || a->total >= MAX_COUNT || a->seqs < 0 || a->seqs >= MAX_COUNT - 64) return hipErrorInvalidValue;
    if (a->total == 0 || a->seqs == 0) return hipSuccess;
    if (!given(a->q) || !given(a->out) || !a->table || !a->starts || !a->kv_len) return hipErrorInvalidValue;
    if (!count(a->table_width) || !count(a->most_q) || !count(a->most_kv)) return hipErrorInvalidValue;
    if (!stride_of(a->q_stride, a->q_heads, c.head_dim)) return hipErrorInvalidValue;
    return hipSuccess;
}

int check_shared(const iq4xs_paged_attention_args* a, const iq4xs_shared_prefix* x) {
    const int err = check_attention(a);
    if (err != hipSuccess) return err;
    if (!x || x->groups <= 0 || x->groups >= MAX_COUNT - 64) return hipErrorInvalidValue;
    if (!x->first && x->groups != 1) return hipErrorInvalidValue;
    if (x->path != IQ4XS_SHARED_AUTO && x->path != IQ4XS_SHARED_ONCE && x->path != IQ4XS_SHARED_EACH)
        return hipErrorInvalidValue;
    if (a->window != 0) return hipErrorNotSupported;
    if (a->total == 0 || a->seqs == 0) return hipSuccess;
    return x->len && count(x->most_len) && count(x->most_rows) ? hipSuccess : hipErrorInvalidValue;
}

int check_linear(const iq4xs_linear_attention_args* a) {
    if (!a || a->heads <= 0 || a->qk_heads <= 0 || a->heads % a->qk_heads != 0 || a->dk <= 0 || a->dv <= 0)
        return hipErrorInvalidValue;
    if (!plain_type(a->in_type) || !plain_type(a->out_type) || !(a->scale == a->scale)) return hipErrorInvalidValue;
    if (!served_head(a->dk) || !served_head(a->dv)) return hipErrorNotSupported;
    if (a->total < 0 || a->total >= MAX_COUNT || a->seqs < 0 || a->seqs >= MAX_COUNT - 64) return hipErrorInvalidValue;
    if (a->total == 0 || a->seqs == 0) return hipSuccess;
    if (!given(a->q) || !given(a->k) || !given(a->v) || !given(a->out) || !a->decay || !a->starts)
        return hipErrorInvalidValue;
    // places within a chunk of tokens are counted in 32 bits
    constexpr int64_t MOST_STRIDE = (int64_t)1 << 23;
    if (!count(a->most_q) || (a->decay_stride != 0 && a->decay_stride < a->heads)) return hipErrorInvalidValue;
    if (a->q_stride >= MOST_STRIDE || a->k_stride >= MOST_STRIDE || a->v_stride >= MOST_STRIDE ||
        a->decay_stride >= MOST_STRIDE)
        return hipErrorInvalidValue;
    if (!stride_of(a->q_stride, a->qk_heads, a->dk) || !stride_of(a->k_stride, a->qk_heads, a->dk) ||
        !stride_of(a->v_stride, a->heads, a->dv))
        return hipErrorInvalidValue;
    if (a->from_slots || a->to_slots) {
        // a slot's place is counted in 64 bits
        if (!given(a->states) || a->slots < 0 || a->slots >= MAX_COUNT) return hipErrorInvalidValue;
    }
    return hipSuccess;
}

}  // namespace

extern "C" {

int iq4xs_qk_norm_rope(const struct iq4xs_qk_norm_rope_args* args, void* stream) {
    const int err = check_qk(args);
    if (err != hipSuccess || args->tokens == 0) return err;
    if (!given(args->k_out)) return hipErrorInvalidValue;
    return launch_qk_norm_rope(*args, nullptr, static_cast<hipStream_t>(stream));
}

int iq4xs_qk_norm_rope_append(const struct iq4xs_qk_norm_rope_args* args, const struct iq4xs_kv_cache* cache,
                              void* stream) {
    int err = check_qk(args);
    if (err != hipSuccess) return err;
    err = check_cache(cache);
    if (err != hipSuccess) return err;
    if (cache->heads != args->k_heads || cache->head_dim != args->head_dim) return hipErrorInvalidValue;
    if (args->tokens == 0) return hipSuccess;
    if (!given(args->v) || !args->slots || !stride_of(args->v_stride, args->k_heads, args->head_dim))
        return hipErrorInvalidValue;
    return launch_qk_norm_rope(*args, cache, static_cast<hipStream_t>(stream));
}

int iq4xs_kv_gather(const struct iq4xs_kv_cache* cache, const int32_t* table, int64_t table_width,
                    const int32_t* starts, int64_t seqs, void* k_out, void* v_out, int64_t total, int out_type,
                    void* stream) {
    const int err = check_cache(cache);
    if (err != hipSuccess) return err;
    if (!plain_type(out_type) || total < 0 || total >= MAX_COUNT || seqs < 0 || seqs >= MAX_COUNT - 64)
        return hipErrorInvalidValue;
    if (total == 0) return hipSuccess;
    if (!starts || !given(k_out) || !given(v_out) || (seqs > 0 && (!table || !count(table_width))))
        return hipErrorInvalidValue;
    return launch_kv_gather(*cache, table, table_width, starts, seqs, k_out, v_out, total, out_type,
                            static_cast<hipStream_t>(stream));
}

size_t iq4xs_paged_attention_workspace_bytes(const struct iq4xs_paged_attention_args* args) {
    if (check_attention(args) != hipSuccess || args->total == 0 || args->seqs == 0) return 0;
    size_t bytes = 0;
    return paged_attention_workspace(*args, &bytes) == hipSuccess ? bytes : 0;
}

int iq4xs_paged_attention(const struct iq4xs_paged_attention_args* args, void* ws, size_t ws_bytes, void* stream) {
    const int err = check_attention(args);
    if (err != hipSuccess || args->total == 0 || args->seqs == 0) return err;
    return launch_paged_attention(*args, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

int iq4xs_paged_attention_sinks(const struct iq4xs_paged_attention_args* args, int64_t sinks, void* ws, size_t ws_bytes,
                                void* stream) {
    const int err = check_attention(args);
    if (err != hipSuccess) return err;
    if (sinks < 0) return hipErrorInvalidValue;
    if (args->total == 0 || args->seqs == 0) return hipSuccess;
    return launch_sinks_attention(*args, sinks, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t iq4xs_shared_attention_workspace_bytes(const struct iq4xs_paged_attention_args* args,
                                              const struct iq4xs_shared_prefix* prefix) {
    if (check_shared(args, prefix) != hipSuccess || args->total == 0 || args->seqs == 0) return 0;
    size_t bytes = 0;
    return shared_attention_workspace(*args, *prefix, &bytes) == hipSuccess ? bytes : 0;
}

int iq4xs_shared_attention(const struct iq4xs_paged_attention_args* args, const struct iq4xs_shared_prefix* prefix,
                           void* ws, size_t ws_bytes, void* stream) {
    const int err = check_shared(args, prefix);
    if (err != hipSuccess || args->total == 0 || args->seqs == 0) return err;
    return launch_shared_attention(*args, *prefix, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

size_t iq4xs_linear_attention_workspace_bytes(const struct iq4xs_linear_attention_args* args) {
    if (check_linear(args) != hipSuccess || args->total == 0 || args->seqs == 0) return 0;
    size_t bytes = 0;
    return linear_attention_workspace(*args, &bytes) == hipSuccess ? bytes : 0;
}

int iq4xs_linear_attention(const struct iq4xs_linear_attention_args* args, void* ws, size_t ws_bytes, void* stream) {
    const int err = check_linear(args);
    if (err != hipSuccess || args->total == 0 || args->seqs == 0) return err;
    return launch_linear_attention(*args, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
