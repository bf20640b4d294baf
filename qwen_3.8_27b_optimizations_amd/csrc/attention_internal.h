// attention_internal.h -- launchers of the attention half of a layer; arguments are checked by the C ABI
// (attention_api.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "iq4xs_mi355x.h"

namespace iq4xs {

// cache null: dense outputs.
hipError_t launch_qk_norm_rope(const iq4xs_qk_norm_rope_args& args, const iq4xs_kv_cache* cache, hipStream_t stream);

hipError_t launch_kv_gather(const iq4xs_kv_cache& cache, const int32_t* table, int64_t width, const int32_t* starts,
                            int64_t seqs, void* k_out, void* v_out, int64_t total, int out_type, hipStream_t stream);

// Args: AttentionArgs or MoreArgs.
// Rows of few new tokens; `tiles` 16-row tiles for each workgroup (1 or 2).
template <typename Args>
void launch_stream_attention(const Args& a, int head_dim, int tiles, int type, int cache_type, int64_t grid,
                             hipStream_t stream);
// Rows of many, 128 for each workgroup.
template <typename Args>
void launch_tile_attention(const Args& a, int head_dim, int type, int cache_type, bool exact, int64_t grid,
                           hipStream_t stream);

// hipErrorInvalidConfiguration: a call whose launches would be too large.
hipError_t paged_attention_workspace(const iq4xs_paged_attention_args& args, size_t* bytes);
// The same, and hipErrorInvalidValue for a workspace that is too small or not aligned to 256 bytes.
hipError_t launch_paged_attention(const iq4xs_paged_attention_args& args, void* ws, size_t ws_bytes, hipStream_t stream);

// The same calls with first tokens beside a window (the workspace is that without them), and with shared prefixes.
hipError_t launch_sinks_attention(const iq4xs_paged_attention_args& args, int64_t sinks, void* ws, size_t ws_bytes,
                                  hipStream_t stream);
hipError_t shared_attention_workspace(const iq4xs_paged_attention_args& args, const iq4xs_shared_prefix& prefix,
                                      size_t* bytes);
hipError_t launch_shared_attention(const iq4xs_paged_attention_args& args, const iq4xs_shared_prefix& prefix, void* ws,
                                   size_t ws_bytes, hipStream_t stream);

}  // namespace iq4xs
