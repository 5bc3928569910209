#pragma once
// Drafted tokens over a paged cache, over libpa_decode.so: attention of several new
// tokens per sequence, accepted rows kept, rows read back (no counterparts in the
// reference). What a cache and a call's tokens are: pa_cached_tokens.

#include "new_tokens.hpp"

#include <cstddef>
#include <cstdint>

namespace decode {

// Types of read_cache's outputs.
enum class ValueType { FP16 = PA_VALUE_FP16, BF16 = PA_VALUE_BF16, FP32 = PA_VALUE_FP32 };

// Bytes of workspace that tree_attention needs for these sizes on the current device.
inline size_t tree_attention_workspace(KVDtype dtype, const pa_cached_tokens& c, int num_q_heads) {
    size_t n = 0;
    detail::check(pa_tree_attention_workspace(static_cast<int>(dtype), &c, num_q_heads, &n));
    return n;
}

// q's tokens over their sequences: each sees the places before its entry's first, and
// of the entry's own the bits of its row of tree (device, [tokens][tree_words]; null:
// itself and those before it).
inline void tree_attention(KVDtype dtype, const pa_cached_tokens& c, const HeadRows& q, const uint64_t* tree,
                           int tree_words, float sm_scale, void* workspace, size_t workspace_bytes,
                           hipStream_t stream = 0) {
    const pa_head_rows r = detail::abi(q);
    detail::check(pa_tree_attention(static_cast<int>(dtype), &c, &r, tree, tree_words, sm_scale, workspace,
                                    workspace_bytes, stream));
}

// Accepted tokens (device, kept [entries][width], counts [entries]) up to the places
// start_pos[e], start_pos[e] + 1, ... of their sequences.
inline void keep_rows(KVDtype dtype, const pa_cached_tokens& c, const int32_t* kept, int width, const int32_t* counts,
                      hipStream_t stream = 0) {
    detail::check(pa_keep_rows(static_cast<int>(dtype), &c, kept, width, counts, stream));
}

// Rows as numbers of a type, token t's to k_out + t * k_stride and v_out + t * v_stride
// (elements; either null).
inline void read_cache(KVDtype dtype, const pa_cached_tokens& c, ValueType type, void* k_out, int64_t k_stride,
                       void* v_out, int64_t v_stride, hipStream_t stream = 0) {
    detail::check(pa_read_cache(static_cast<int>(dtype), &c, static_cast<int>(type), k_out, k_stride, v_out, v_stride,
                                stream));
}

}  // namespace decode
