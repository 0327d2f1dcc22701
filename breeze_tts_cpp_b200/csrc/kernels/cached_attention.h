// Launcher of the attention over the quantized key/value cache. Operands are checked by the caller (ops/attention.cpp).
#pragma once
#include "core/cache.h"
#include <cstdint>
#include <cuda_runtime_api.h>

namespace tts {
// Query heads that share a cached one, at most: a query row's token is found by an fp32 product, which from 2^23 of them on may be one off.
constexpr int kMostGroup = 1 << 20;
struct AttentionProblem {
    TensorView queries, output; // [rows, heads * head_dim]
    CacheView cache;
    const int *pages = nullptr; // [sequences, page_columns], rows page_stride apart
    int sequences = 0, page_columns = 0, page_stride = 0;
    const int *lengths = nullptr;
    const int *query_offsets = nullptr; // [sequences + 1]; null = one query row per sequence
    const int *prefix_pages = nullptr, *prefix_length = nullptr;
    int prefix_columns = 0;
    float scale = 0.f;
};
// Bytes of workspace behind the context's header that a launch uses.
size_t attention_workspace_bytes(int rows, int sequences, int heads, int kv_heads, int head_dim, bool prefix, int multiprocessors);
// `status` and `pass_word`: in the workspace's header (quant_linear_workspace.h).
void launch_cached_attention(const AttentionProblem &, void *workspace, size_t workspace_bytes, int *status, int *pass_word, int multiprocessors,
                             cudaStream_t stream);
// Part of quant_linear_initialize: the instances' dynamic shared memory, on the current device.
void raise_attention_limits();
} // namespace tts
