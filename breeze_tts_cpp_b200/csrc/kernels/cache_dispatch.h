// What the host sides of the cache operators share: run-time types as compile-time ones, alignment, powers of two.
#pragma once
#include "core/tensor.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace tts {
// Calls f(element, format, head width) with the run-time types as compile-time ones.
template <class Call> void by_type(Type element, Type format, int head_dim, Call &&call) {
    auto width = [&](auto t, auto f) {
        if (head_dim == 64) call(t, f, std::integral_constant<int, 64>{});
        else call(t, f, std::integral_constant<int, 128>{});
    };
    auto storage = [&](auto t) {
        if (format == Type::I8) width(t, std::integral_constant<Type, Type::I8>{});
        else width(t, std::integral_constant<Type, Type::FP8>{});
    };
    if (element == Type::F16) storage(__half{});
    else storage(__nv_bfloat16{});
}
// Whether every row of 16-bit elements starts on a multiple of `size` bytes; an absent operand has none that does not.
inline bool rows_start_on(size_t size, const TensorView &v) {
    return !v.data || (reinterpret_cast<uintptr_t>(v.data) % size == 0 && (v.rows <= 1 || size_t(v.ld()) * 2 % size == 0));
}
inline int shift_of(int power) {
    int s = 0;
    while ((1 << s) < power) ++s;
    return s;
}
} // namespace tts
