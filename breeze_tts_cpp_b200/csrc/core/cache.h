// The quantized key/value cache between a decoder's QKV and O projections, and the plan of its rotary positions. Metadata only.
//
// Keys and values are one byte each, [pages, kv_heads, page_size, head_dim], INT8 or FP8 e4m3, with one fp32 scale per token and
// head, [pages, kv_heads, page_size]. The tokens of one head of a page lie one behind the other, so that a tile of the attention is
// one box of a tensor map, and its scales are one run. A slot is page * page_size + the token's place in the page.
#pragma once
#include "core/tensor.h"

namespace tts {
struct CacheView {
    void *keys = nullptr, *values = nullptr;
    float *key_scales = nullptr, *value_scales = nullptr;
    int pages = 0, kv_heads = 0, page_size = 0, head_dim = 0;
    Type type = Type::I8;
    int device = -1;

    size_t rows() const { return size_t(pages) * kv_heads * page_size; }
    size_t slots() const { return size_t(pages) * page_size; }
    void validate() const {
        if (type != Type::I8 && type != Type::FP8) throw std::invalid_argument("a cache holds INT8 or FP8 values");
        if (head_dim != 64 && head_dim != 128) throw std::invalid_argument("cache heads are 64 or 128 wide");
        if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
            throw std::invalid_argument("cache pages hold 16 to 1024 tokens, a power of two");
        if (pages < 1 || kv_heads < 1) throw std::invalid_argument("empty cache");
        // Rows are a tensor map's coordinate, slots an int32 index, and so are the columns of a 16-bit row of all heads. The product of all three
        // sizes may pass 64 bits.
        constexpr size_t most = size_t(std::numeric_limits<int>::max());
        if (size_t(pages) * kv_heads > most / page_size) throw std::invalid_argument("cache has more than 2^31 - 1 rows");
        if (size_t(kv_heads) > most / head_dim) throw std::invalid_argument("cache heads have more than 2^31 - 1 columns in all");
        const void *parts[] = {keys, values, key_scales, value_scales};
        const size_t sizes[] = {rows() * head_dim, rows() * head_dim, rows() * 4, rows() * 4};
        for (int i = 0; i < 4; ++i) {
            const auto a = reinterpret_cast<uintptr_t>(parts[i]);
            if (!a || a % 16) throw std::invalid_argument("cache storage must be 16-byte aligned");
            for (int j = 0; j < i; ++j) {
                const auto b = reinterpret_cast<uintptr_t>(parts[j]);
                if (a < b + sizes[j] && b < a + sizes[i]) throw std::invalid_argument("cache keys, values and scales overlap");
            }
        }
    }
    bool overlaps(const TensorView &v) const {
        if (!v.data) return false;
        const void *parts[] = {keys, values, key_scales, value_scales};
        for (int i = 0; i < 4; ++i) {
            const auto a = reinterpret_cast<uintptr_t>(parts[i]), b = reinterpret_cast<uintptr_t>(v.data);
            if (a < b + v.span_bytes() && b < a + rows() * (i < 2 ? size_t(head_dim) : 4)) return true;
        }
        return false;
    }
};

// Pair i of a head turns by turns[i] revolutions per position; cosine and sine are multiplied by `scale`. The first `dims` columns
// of a head take part: pairs (i, i + dims / 2), or (2i, 2i + 1) when interleaved.
struct RotaryView {
    const double *turns = nullptr; // device, [dims / 2]
    int dims = 0;
    bool interleaved = false;
    float scale = 1.f;
    int device = -1;
};
} // namespace tts
