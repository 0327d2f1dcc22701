// Host side of the cache operators: argument checks, then the launch.
#include "ops/attention.h"
#include "kernels/cached_attention.h"
#include "kernels/quant_linear_workspace.h"
#include "kernels/rotary_cache.h"
#include "ops/context.h"
#include <cmath>

namespace tts::ops {
namespace {
[[noreturn]] void refuse(const char *what) { throw std::invalid_argument(what); }
bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
bool dense16(const TensorView &v) { return v.data && (v.type == Type::F16 || v.type == Type::BF16) && aligned(v.data, 2); }
// Positions are ints, and so is the end of the tile of 128 keys that the last one lies in.
bool too_long(int page_columns, int page_size) { return size_t(page_columns) * page_size > size_t(std::numeric_limits<int>::max()) - 127; }
void check_index(const TensorView &v, size_t count, const char *what) {
    if (!v.data || v.type != Type::I32 || v.rows != 1 || size_t(v.cols) != count || !aligned(v.data, 4)) refuse(what);
}
// Column slices of one buffer (a packed QKV row) interleave: their spans overlap, their elements need not.
bool collide(const TensorView &a, const TensorView &b) {
    if (!a.overlaps(b)) return false;
    if (bytes(a.type) != bytes(b.type) || a.ld() != b.ld()) return true;
    const int64_t pitch = int64_t(a.ld()) * int64_t(bytes(a.type));
    const int64_t apart = reinterpret_cast<intptr_t>(b.data) - reinterpret_cast<intptr_t>(a.data), offset = (apart % pitch + pitch) % pitch;
    return offset < int64_t(a.cols) * int64_t(bytes(a.type)) || offset + int64_t(b.cols) * int64_t(bytes(b.type)) > pitch;
}
bool same_rows(const TensorView &a, const TensorView &b) {
    return a.data == b.data && a.rows == b.rows && a.cols == b.cols && (a.rows <= 1 || a.ld() == b.ld());
}
void check_plan(const RotaryView &plan, int head_dim, int device) {
    if (!plan.turns || !aligned(plan.turns, 8) || plan.device != device) refuse("rotary plan is missing, misaligned or on another device");
    if (plan.dims < 16 || plan.dims > head_dim || plan.dims % 16) refuse("rotary columns must be a multiple of 16 within the head");
    if (!std::isfinite(plan.scale)) refuse("rotary scale is not finite");
}
TensorView turns_of(const RotaryView &plan) {
    return plan.turns ? TensorView(const_cast<double *>(plan.turns), 1, plan.dims / 2, Type::F64, 0, plan.device) : TensorView();
}
void check_devices(int device, std::initializer_list<TensorView> operands) {
    for (const TensorView &v : operands)
        if (v.data && v.device != device) refuse("operands are on different devices");
}
void check_cache(const CacheView &cache, std::initializer_list<TensorView> operands) {
    cache.validate();
    check_devices(cache.device, operands);
}
} // namespace

float rotary_turns(const RotaryPlan &plan, double *turns) {
    if (!turns || plan.dims < 2 || plan.dims % 2) refuse("rotary columns must be even");
    if (!(plan.base > 1.0) || !std::isfinite(plan.base) || !(plan.factor >= 1.0) || !std::isfinite(plan.factor))
        refuse("rotary base must exceed 1 and the factor must be at least 1");
    const bool ramped = plan.scaling == RotaryScaling::Yarn || plan.scaling == RotaryScaling::Wavelength;
    const double low = plan.low, high = plan.high != 0. ? plan.high : plan.scaling == RotaryScaling::Yarn ? 32. : 4.;
    if (ramped && (plan.original_length < 1 || !(low > 0.) || !(high > low) || !std::isfinite(high)))
        refuse("rotary scaling needs the original length and 0 < low < high");
    if (plan.scaling == RotaryScaling::Base && plan.dims == 2) refuse("a single pair has no base to stretch");
    const double tau = 6.283185307179586476925286766559, dims = plan.dims;
    const double base = plan.scaling == RotaryScaling::Base ? plan.base * std::pow(plan.factor, dims / (dims - 2)) : plan.base;
    // Yarn's ramp runs over the pair's index, between the pairs that make `high` and `low` turns within the original length.
    auto index_of = [&](double count) { return dims * std::log(plan.original_length / (count * tau)) / (2 * std::log(base)); };
    double first = 0, last = 0;
    if (plan.scaling == RotaryScaling::Yarn) {
        first = std::max(std::floor(index_of(high)), 0.);
        last = std::max(std::min(std::ceil(index_of(low)), dims - 1), first + 1e-3);
    }
    for (int i = 0; i < plan.dims / 2; ++i) {
        const double rate = std::pow(base, -2. * i / dims) / tau;
        double kept = 1.; // share of the pair that keeps its turns
        if (plan.scaling == RotaryScaling::Linear) kept = 0.;
        else if (plan.scaling == RotaryScaling::Yarn) kept = 1. - std::min(std::max((i - first) / (last - first), 0.), 1.);
        else if (plan.scaling == RotaryScaling::Wavelength)
            kept = std::min(std::max((plan.original_length * rate - low) / (high - low), 0.), 1.);
        turns[i] = rate * kept + rate / plan.factor * (1. - kept);
    }
    return plan.scaling == RotaryScaling::Yarn ? float(0.1 * std::log(plan.factor) + 1.) : 1.f;
}

void validate_rotary(TensorView input, TensorView positions, RotaryView plan, int head_dim, TensorView output) {
    if (!dense16(input) || !dense16(output) || input.type != output.type || input.rows != output.rows || input.cols != output.cols)
        refuse("rotary input/output shape/type mismatch");
    if (head_dim < 16 || head_dim > 512 || head_dim % 16 || !input.cols || input.cols % head_dim)
        refuse("rotary heads must be a multiple of 16 up to 512 wide and fill the row");
    check_index(positions, size_t(input.rows), "rotary positions must be int32, one per row");
    check_devices(input.device, {output, positions});
    check_plan(plan, head_dim, input.device);
    if (!same_rows(input, output) && collide(output, input)) refuse("rotary output overlaps its input");
    if (output.overlaps(positions)) refuse("rotary output overlaps its positions");
    if (output.overlaps(turns_of(plan))) refuse("rotary output overlaps its plan");
}
void rotary(TensorView input, TensorView positions, RotaryView plan, int head_dim, TensorView output) {
    validate_rotary(input, positions, plan, head_dim, output);
    auto &gpu = execution_context(input);
    launch_rotary(input, output, positions.ptr<int>(), plan, head_dim, gpu.stream);
}

void validate_cache_write(const CacheView &cache, TensorView keys, TensorView values, TensorView slots, TensorView positions, RotaryView plan,
                          TensorView queries, TensorView query_output, TensorView query_norm, TensorView key_norm, float epsilon) {
    check_cache(cache, {keys, values, slots, positions, queries, query_output, query_norm, key_norm});
    const int width = cache.kv_heads * cache.head_dim;
    if (!dense16(keys) || !dense16(values) || keys.type != values.type || keys.rows != values.rows || keys.cols != width || values.cols != width)
        refuse("cache keys/values shape/type mismatch");
    check_index(slots, size_t(keys.rows), "cache slots must be int32, one per row");
    if (plan.turns) {
        check_plan(plan, cache.head_dim, cache.device);
        check_index(positions, size_t(keys.rows), "rotary positions must be int32, one per row");
    } else if (positions.data) {
        refuse("positions without a rotary plan");
    }
    for (const TensorView *norm : {&query_norm, &key_norm})
        if (norm->data && (norm->type != keys.type || norm->numel() != size_t(cache.head_dim) || norm->rows != 1 || !aligned(norm->data, 2))) refuse("head norm weight shape/type mismatch");
    if ((query_norm.data || key_norm.data) && !(epsilon >= 0.f && std::isfinite(epsilon))) refuse("invalid norm epsilon");
    const TensorView turns = turns_of(plan);
    if (queries.data || query_output.data) {
        if (!dense16(queries) || !dense16(query_output) || queries.type != keys.type || query_output.type != keys.type ||
            queries.rows != keys.rows || query_output.rows != keys.rows || queries.cols != query_output.cols || !queries.cols ||
            queries.cols % cache.head_dim)
            refuse("query input/output shape/type mismatch");
        if (!same_rows(queries, query_output) && collide(query_output, queries)) refuse("query output overlaps its input");
        for (const TensorView &source : {keys, values, slots, positions, turns, query_norm, key_norm})
            if (collide(query_output, source)) refuse("query output overlaps another operand");
    } else if (query_norm.data) {
        refuse("a query norm without queries");
    }
    for (const TensorView &v : {keys, values, slots, positions, turns, queries, query_output, query_norm, key_norm})
        if (cache.overlaps(v)) refuse("an operand overlaps the cache");
}
void cache_write(const CacheView &cache, TensorView keys, TensorView values, TensorView slots, TensorView positions, RotaryView plan,
                 TensorView queries, TensorView query_output, TensorView query_norm, TensorView key_norm, float epsilon) {
    validate_cache_write(cache, keys, values, slots, positions, plan, queries, query_output, query_norm, key_norm, epsilon);
    auto &gpu = execution_context(keys);
    launch_cache_write(cache, keys, values, slots.ptr<int>(), positions.ptr<int>(), plan, queries, query_output, query_norm, key_norm, epsilon,
                       gpu.stream);
}

void validate_cache_read(const CacheView &cache, TensorView slots, TensorView keys, TensorView values) {
    check_cache(cache, {slots, keys, values});
    const int width = cache.kv_heads * cache.head_dim;
    const TensorView &any = keys.data ? keys : values;
    for (const TensorView *v : {&keys, &values})
        if (v->data && (!dense16(*v) || v->type != any.type || v->rows != any.rows || v->cols != width)) refuse("cache output shape/type mismatch");
    if (!any.data) refuse("cache read has no output");
    check_index(slots, size_t(any.rows), "cache slots must be int32, one per row");
    if (collide(keys, values)) refuse("cache outputs overlap");
    for (const TensorView *v : {&keys, &values})
        if (cache.overlaps(*v) || v->overlaps(slots)) refuse("a cache output overlaps another operand");
}
void cache_read(const CacheView &cache, TensorView slots, TensorView keys, TensorView values) {
    validate_cache_read(cache, slots, keys, values);
    auto &gpu = execution_context(slots);
    launch_cache_read(cache, slots.ptr<int>(), keys, values, gpu.stream);
}

size_t cached_attention_workspace(int rows, int sequences, int heads, int kv_heads, int head_dim, bool prefix, int multiprocessors) {
    if (rows < 0 || sequences < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || (head_dim != 64 && head_dim != 128) || multiprocessors < 1)
        refuse("invalid attention shape");
    return quant_linear_header_bytes() + attention_workspace_bytes(rows, sequences, heads, kv_heads, head_dim, prefix, multiprocessors);
}

void validate_cached_attention(const CacheView &cache, const Attention &a) {
    check_cache(cache, {a.queries, a.output, a.pages, a.lengths, a.query_offsets, a.prefix_pages, a.prefix_length});
    if (!dense16(a.queries) || !dense16(a.output) || a.queries.type != a.output.type || a.queries.rows != a.output.rows ||
        a.queries.cols != a.output.cols)
        refuse("attention queries/output shape/type mismatch");
    const int heads = a.queries.cols / cache.head_dim;
    if (!heads || a.queries.cols % cache.head_dim || heads % cache.kv_heads) refuse("query heads must be a multiple of the cache's heads");
    if (heads / cache.kv_heads > kMostGroup) refuse("more than 2^20 query heads to a cached one");
    if (size_t(a.queries.rows) * heads > size_t(std::numeric_limits<int>::max())) refuse("too many query rows");
    if (!a.pages.data || a.pages.type != Type::I32 || a.pages.rows < 1 || a.pages.cols < 1 || !aligned(a.pages.data, 4) ||
        too_long(a.pages.cols, cache.page_size))
        refuse("attention pages must be int32 [sequences, pages]");
    check_index(a.lengths, size_t(a.pages.rows), "attention lengths must be int32, one per sequence");
    if (a.query_offsets.data) check_index(a.query_offsets, size_t(a.pages.rows) + 1, "query offsets must be int32, one more than sequences");
    else if (a.queries.rows != a.pages.rows) refuse("without query offsets there is one query row per sequence");
    if (!a.prefix_pages.data != !a.prefix_length.data) refuse("a prefix needs its pages and its length");
    if (a.prefix_pages.data) {
        check_index(a.prefix_pages, size_t(a.prefix_pages.cols), "prefix pages must be int32 [1, pages]");
        if (a.prefix_pages.cols < 1 || too_long(a.prefix_pages.cols, cache.page_size))
            refuse("prefix pages must be int32 [1, pages]");
        check_index(a.prefix_length, 1, "the prefix length is one int32");
    }
    // The device counts tiles of 128 keys, per sequence, cached head and tile of at least eight query rows, in 32 bits.
    const int64_t group = heads / cache.kv_heads, segments = (int64_t(a.queries.rows) * group / 8 + a.pages.rows) * cache.kv_heads;
    const int64_t longest = (int64_t(std::max(a.pages.cols, a.prefix_pages.cols)) * cache.page_size + 127) / 128;
    if (double(segments) * double(longest) > double(1 << 27)) refuse("too many query rows for tables of this size");
    if (!std::isfinite(a.scale)) refuse("attention scale is not finite");
    if (cache.overlaps(a.output)) refuse("attention output overlaps the cache");
    for (const TensorView &v : {a.queries, a.pages, a.lengths, a.query_offsets, a.prefix_pages, a.prefix_length})
        if (collide(a.output, v)) refuse("attention output overlaps an operand");
}
void cached_attention(const CacheView &cache, const Attention &a) {
    validate_cached_attention(cache, a);
    auto &gpu = execution_context(a.queries);
    const int heads = a.queries.cols / cache.head_dim;
    const bool prefix = a.prefix_pages.data != nullptr;
    const size_t needed = cached_attention_workspace(a.queries.rows, a.pages.rows, heads, cache.kv_heads, cache.head_dim, prefix, gpu.multiprocessors);
    if (!gpu.gemm_workspace.data() || gpu.gemm_workspace.size() < needed)
        throw std::invalid_argument("attention needs a context workspace of " + std::to_string(needed) + " bytes");
    if (!aligned(gpu.gemm_workspace.data(), 32)) throw std::invalid_argument("attention needs a context workspace on a 32-byte boundary");
    AttentionProblem p;
    p.queries = a.queries, p.output = a.output, p.cache = cache;
    p.pages = a.pages.ptr<int>(), p.sequences = a.pages.rows, p.page_columns = a.pages.cols, p.page_stride = a.pages.ld();
    p.lengths = a.lengths.ptr<int>(), p.query_offsets = a.query_offsets.ptr<int>();
    p.prefix_pages = a.prefix_pages.ptr<int>(), p.prefix_length = a.prefix_length.ptr<int>(), p.prefix_columns = a.prefix_pages.cols;
    p.scale = a.scale != 0.f ? a.scale : 1.f / std::sqrt(float(cache.head_dim));
    launch_cached_attention(p, static_cast<char *>(gpu.gemm_workspace.data()) + quant_linear_header_bytes(),
                            gpu.gemm_workspace.size() - quant_linear_header_bytes(), quant_linear_status_word(gpu.gemm_workspace.data()),
                            attention_pass_word(gpu.gemm_workspace.data()), gpu.multiprocessors, gpu.stream);
}
} // namespace tts::ops
