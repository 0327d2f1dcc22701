// Launchers of the rotary positions and of the quantized key/value cache's writing and reading. Operands are checked by the callers
// (ops/attention.cpp).
#pragma once
#include "core/cache.h"
#include <cuda_runtime_api.h>

namespace tts {
// output[r] = input[r] with its heads turned by positions[r]; the two may be the same rows.
void launch_rotary(TensorView input, TensorView output, const int *positions, RotaryView rotary, int head_dim, cudaStream_t stream);
// Row r of keys and values, normalised (key_norm) and turned (rotary, keys only), quantized into slot slots[r]; negative slots and
// those past the cache are left out. With `queries`, their heads are normalised and turned into query_output in the same launch.
void launch_cache_write(CacheView cache, TensorView keys, TensorView values, const int *slots, const int *positions, RotaryView rotary,
                        TensorView queries, TensorView query_output, TensorView query_norm, TensorView key_norm, float epsilon,
                        cudaStream_t stream);
// keys[r], values[r] = slot slots[r] as 16-bit rows, zeros for a slot outside of the cache. Either may be empty.
void launch_cache_read(CacheView cache, const int *slots, TensorView keys, TensorView values, cudaStream_t stream);
} // namespace tts
