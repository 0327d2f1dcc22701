// What lies between a decoder's QKV and O projections: rotary positions, the quantized key/value cache and the attention that reads
// it. The reference keeps these 16-bit (its attention path is outside of its quantization); here the cache is quantized by the rules
// of the row quantizer, and the operators take the same borrowed views on the bound device as those of ops.h.
#pragma once
#include "core/cache.h"

namespace tts::ops {
// How the turns per position are stretched for contexts longer than a model was trained on.
enum class RotaryScaling {
    None,
    Linear,    // all turns divided by the factor
    Base,      // the base grows, so that the slowest pair is stretched by the factor and the fastest not at all
    Yarn,      // pairs with few turns within the original length are stretched, those with many are not, a ramp between; scales cos and sin
    Wavelength // the same by wavelength, with the ramp over the number of turns
};
struct RotaryPlan {
    int dims = 0;
    double base = 10000.0, factor = 1.0;
    RotaryScaling scaling = RotaryScaling::None;
    int original_length = 0;     // Yarn, Wavelength
    double low = 1.0, high = 0.; // turns within the original length between which the ramp lies; high 0: 32 (Yarn), 4 (Wavelength)
};
// turns[dims / 2] (host memory) and the factor for cosine and sine. Host only.
float rotary_turns(const RotaryPlan &, double *turns);

// output = input [rows, heads * head_dim] with each head's pairs turned by positions[row]; in place if both are the same view.
void rotary(TensorView input, TensorView positions, RotaryView plan, int head_dim, TensorView output);
// Quantizes row r of keys and values [rows, kv_heads * head_dim] into slot slots[r]. keys are normalised (key_norm, RMSNorm over a
// head) and turned first; queries, if given, are too, into query_output (may be the same view).
void cache_write(const CacheView &cache, TensorView keys, TensorView values, TensorView slots, TensorView positions = {}, RotaryView plan = {},
                 TensorView queries = {}, TensorView query_output = {}, TensorView query_norm = {}, TensorView key_norm = {},
                 float epsilon = 1e-6f);
// keys[r], values[r] = what slot slots[r] holds, as 16-bit rows; either may be empty.
void cache_read(const CacheView &cache, TensorView slots, TensorView keys, TensorView values);

// What the operators above refuse, and cached_attention below; without a context, so callers may ask ahead of time.
void validate_rotary(TensorView input, TensorView positions, RotaryView plan, int head_dim, TensorView output);
void validate_cache_write(const CacheView &cache, TensorView keys, TensorView values, TensorView slots, TensorView positions, RotaryView plan,
                          TensorView queries, TensorView query_output, TensorView query_norm, TensorView key_norm, float epsilon);
void validate_cache_read(const CacheView &cache, TensorView slots, TensorView keys, TensorView values);

struct Attention {
    TensorView queries, output;   // [rows, heads * head_dim], F16 or BF16
    TensorView pages, lengths;    // I32 [sequences, columns], [1, sequences]
    TensorView query_offsets;     // I32 [1, sequences + 1], or empty: one row per sequence
    TensorView prefix_pages;      // I32 [1, columns], or empty
    TensorView prefix_length;     // I32 [1, 1]
    float scale = 0.f;            // 0: 1 / sqrt(head_dim)
};
void cached_attention(const CacheView &cache, const Attention &);
void validate_cached_attention(const CacheView &cache, const Attention &);
// Context workspace that cached_attention needs for these shapes. Host only.
size_t cached_attention_workspace(int rows, int sequences, int heads, int kv_heads, int head_dim, bool prefix, int multiprocessors);
} // namespace tts::ops
