// engine_util.h - what the engine's calls share: validation of layers and buffer
// sizes.  Included by the sources that implement Context.
#pragma once
#include "runtime.h"

namespace pam {

inline int32_t elem_bytes(int32_t dtype) { return dtype == kF32 ? 4 : (dtype == kF16 ? 2 : 1); }
inline int32_t io_bytes(int32_t dtype) { return dtype == kF32 ? 4 : 2; }  // Q / O / new K,V element

inline void validate_layer(const pam_layer_spec &l) {
    if (l.head_dim <= 0) throw invalid_configuration("headDim must be positive.");
    if (l.num_heads <= 0) throw invalid_configuration("numHeads must be positive.");
    if (l.num_kv_heads <= 0) throw invalid_configuration("numKVHeads must be positive.");
    if (l.num_heads % l.num_kv_heads != 0)
        throw invalid_configuration("numHeads must be divisible by numKVHeads for GQA/MQA mapping.");
    if (l.block_size <= 0) throw invalid_configuration("blockSize must be positive.");
    if (l.data_type < 0 || l.data_type > 2) throw invalid_configuration("unknown dtype");
    if (l.window_size < 0) throw invalid_configuration("windowSize must be non-negative.");
    // kernel envelope: 4-element slices per lane, at most 64 lanes per token row
    if (l.head_dim % 4 != 0 || l.head_dim > 256)
        throw PamError("Unsupported paged attention path: headDim must be a multiple of 4 and at most 256.");
}

inline void require(size_t actual, const char *name, int64_t expected) {
    if (actual != 0 && (int64_t)actual < expected) throw buffer_too_small(name, expected, (int64_t)actual);
}

inline int64_t q_bytes_per_token(const pam_layer_spec &l) { return (int64_t)l.num_heads * l.head_dim * io_bytes(l.data_type); }
inline int64_t kv_bytes_per_token(const pam_layer_spec &l) {
    return (int64_t)l.num_kv_heads * l.head_dim * elem_bytes(l.data_type);
}
inline int64_t pool_bytes_for(int64_t blocks, const pam_layer_spec &l) { return blocks * l.block_size * kv_bytes_per_token(l); }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace pam
