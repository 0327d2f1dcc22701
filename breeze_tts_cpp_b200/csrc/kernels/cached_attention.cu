// Host side of the attention over the quantized cache: workspace, tensor maps, choice of the instance.
#include "kernels/cached_attention.h"
#include "kernels/cache_dispatch.h"
#include "kernels/cached_attention_tiles_sm100.cuh"
#include "kernels/tensor_map.h"
#include <algorithm>
#include <climits>

namespace tts {
namespace {
using namespace b200;

CUtensorMap cache_map(const void *base, const CacheView &cache, int box_rows) {
    CUtensorMap map;
    cuuint64_t dims[2] = {cuuint64_t(cache.head_dim), cuuint64_t(cache.rows())};
    cuuint64_t strides[1] = {cuuint64_t(cache.head_dim)};
    cuuint32_t box[2] = {cuuint32_t(cache.head_dim), cuuint32_t(box_rows)};
    cuuint32_t element_strides[2] = {1, 1};
    CUresult status = encode_tiled()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, element_strides,
                                     CU_TENSOR_MAP_INTERLEAVE_NONE, cache.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (status != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled (cache) failed with code " + std::to_string(int(status)));
    return map;
}

// Query rows of a cached head up to which segments of at most sixteen are used, several to a sequence, each of which reads the cache again. From
// 17 to 32 rows that takes 19.7 us against 21.6 with a segment of 128 (four sequences of up to 8000, up to six tokens, groups of eight), for a prefix's 24 rows
// 27.3 against 28.2; with more it falls behind (16 sequences of up to 2000, 40 rows on the average: 55 against 36).
// The offsets are on the device, so the batch's average decides for all of its sequences, and these figures are of batches whose sequences are alike. Decode rows
// beside a chunk of a prompt are served badly either way: 64 sequences of one token (200 to 2000 long) and a chunk of 700 take 145 us in one call, 79 in
// two; 60 and two chunks of 1024 145 and 110; 64 and a chunk of 200 82 and 68 (16 heads over 8, 128 wide, INT8). Callers are told to make two calls.
constexpr int kFewRows = 32;
constexpr size_t kPiece = 256; // parts of the workspace start on multiples of this
size_t padded(size_t bytes) { return (bytes + kPiece - 1) / kPiece * kPiece; }

// How one pass over a set of page tables is done.
struct PassPlan {
    bool many, narrow; // 128 query rows per segment on the tensor cores' own memory; else eight, or sixteen
    int part_columns;
};
PassPlan plan_pass(int rows, int sequences, int group, bool prefix) {
    // Query rows of a cached head, on the average: all of them share a prefix.
    const int64_t all = int64_t(rows) * group, each = prefix ? all : all / std::max(sequences, 1);
    PassPlan plan{each > kFewRows, each <= 8, 16};
    if (plan.many) plan.part_columns = int(std::min<int64_t>(kManyRows, all));
    return plan;
}
// A pass's workspace: the closed segments and the partial sums; with a shared prefix also the table of all rows and those done in one part.
struct Carve {
    size_t closed, table, partials, complete, bytes;
    Carve(int rows, int heads, int head_dim, bool prefix, int part_columns, int ctas) {
        const size_t row = size_t(head_dim + kPartialExtra) * 4;
        closed = 0;
        table = padded(size_t(ctas) * sizeof(ClosedSegment));
        partials = table + (prefix ? padded(size_t(rows) * heads * sizeof(int4)) : 0);
        complete = partials + padded(size_t(ctas) * 2 * part_columns * row);
        bytes = complete + (prefix ? padded(size_t(rows) * heads * row) : 0);
    }
};

template <class T, Type F, int HeadDim> void launch_many(const AttentionArgs &args, int ctas, cudaStream_t stream) {
    launch_pdl("cached attention", cached_attention_many<T, F, HeadDim>, dim3(unsigned(ctas)), dim3(kManyThreads), ManyShape<HeadDim>::smem, stream, args);
}
template <class T, Type F, int HeadDim, int Tiles>
void launch_pass(AttentionArgs args, int most_columns, const CUtensorMap &keys, const CUtensorMap &values, int ctas, cudaStream_t stream) {
    using Shape = AttentionShape<HeadDim, Tiles>;
    // What the workers leave for the mergers, several times where that is small, and as many stages as the rest of the shared memory holds.
    args.merge_columns = std::min(Shape::columns, most_columns);
    args.merge_buffers = args.merge_columns <= 2 ? kMergeBuffers : args.merge_columns <= 4 ? 2 : 1;
    const size_t merge = size_t(args.merge_buffers) * Shape::merge(args.merge_columns);
    args.stages = int(std::min<size_t>(kMaxRing, (kAttentionSmem - 1024 - merge) / Shape::stage));
    launch_pdl("cached attention", cached_attention<T, F, HeadDim, Tiles>, dim3(unsigned(ctas)), dim3(kAttentionThreads),
               1024 + args.stages * size_t(Shape::stage) + merge, stream, keys, values, args);
}
template <class T, Type F, int HeadDim>
void launch_pass(bool narrow, int most_columns, const AttentionArgs &args, const CUtensorMap &keys, const CUtensorMap &values, int ctas, cudaStream_t stream) {
    if (narrow) launch_pass<T, F, HeadDim, 1>(args, most_columns, keys, values, ctas, stream);
    else launch_pass<T, F, HeadDim, 2>(args, most_columns, keys, values, ctas, stream);
}
template <class T, Type F, int HeadDim> void raise_limit() {
    auto raise = [](auto *kernel, size_t bytes) {
        const cudaError_t status = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
        if (status != cudaSuccess) throw std::runtime_error(std::string("cudaFuncSetAttribute(attention): ") + cudaGetErrorString(status));
    };
    raise(cached_attention<T, F, HeadDim, 1>, kAttentionSmem);
    raise(cached_attention<T, F, HeadDim, 2>, kAttentionSmem);
    raise(cached_attention_many<T, F, HeadDim>, ManyShape<HeadDim>::smem);
}
} // namespace

void raise_attention_limits() {
    for (Type element : {Type::F16, Type::BF16})
        for (Type format : {Type::I8, Type::FP8})
            for (int head_dim : {64, 128})
                by_type(element, format, head_dim, [](auto t, auto f, auto width) { raise_limit<decltype(t), decltype(f)::value, decltype(width)::value>(); });
}

size_t attention_workspace_bytes(int rows, int sequences, int heads, int kv_heads, int head_dim, bool prefix, int multiprocessors) {
    size_t bytes = 0;
    for (int pass = 0; pass < (prefix ? 2 : 1); ++pass)
        bytes += Carve(rows, heads, head_dim, prefix, plan_pass(rows, sequences, heads / kv_heads, pass).part_columns, multiprocessors).bytes;
    return bytes;
}

void launch_cached_attention(const AttentionProblem &p, void *workspace, size_t workspace_bytes, int *status, int *pass_word,
                             int multiprocessors, cudaStream_t stream) {
    const int rows = p.queries.rows, head_dim = p.cache.head_dim, heads = p.queries.cols / head_dim, ctas = multiprocessors;
    const bool prefix = p.prefix_pages != nullptr;
    if (!rows) return;
    if (workspace_bytes < attention_workspace_bytes(rows, p.sequences, heads, p.cache.kv_heads, head_dim, prefix, ctas))
        throw std::invalid_argument("attention workspace is too small");

    AttentionArgs args{};
    args.queries = p.queries.data, args.output = p.output.data;
    args.query_stride = p.queries.ld(), args.output_stride = p.output.ld();
    args.rows = rows, args.heads = heads, args.kv_heads = p.cache.kv_heads, args.group = heads / p.cache.kv_heads;
    args.group_inverse = 1.f / float(args.group);
    args.aligned = rows_start_on(16, p.queries) && rows_start_on(16, p.output);
    args.sectors = args.aligned && rows_start_on(32, p.output);
    args.pages = p.pages, args.lengths = p.lengths, args.query_offsets = p.query_offsets;
    args.sequences = p.sequences, args.page_columns = p.page_columns, args.page_stride = p.page_stride;
    args.page_shift = shift_of(p.cache.page_size), args.total_pages = p.cache.pages, args.offset_count = p.sequences;
    args.box_shift = std::min(args.page_shift, shift_of(kTileKeys));
    args.cached_keys = p.cache.keys, args.cached_values = p.cache.values;
    args.key_scales = p.cache.key_scales, args.value_scales = p.cache.value_scales;
    const float format = p.cache.type == Type::FP8 ? 256.f : 1.f; // e4m3 values enter the second product times 2^-8
    args.score_scale = p.scale * 1.4426950408889634f;
    args.output_scale = format;
    args.status = status;
    args.pass_word = prefix ? pass_word : nullptr;

    CombineArgs combine{};
    combine.rows = rows, combine.heads = heads, combine.group = args.group, combine.output_stride = p.output.ld();
    combine.row_count = p.query_offsets ? p.query_offsets + p.sequences : nullptr;
    combine.output = p.output.data, combine.output_scale = format, combine.pass_word = args.pass_word;
    CUtensorMap keys{}, values{}; // of the kernel for few rows
    if (!plan_pass(rows, p.sequences, args.group, false).many || (prefix && !plan_pass(rows, p.sequences, args.group, true).many)) {
        keys = cache_map(p.cache.keys, p.cache, 1 << args.box_shift);
        values = cache_map(p.cache.values, p.cache, 1 << args.box_shift);
    }
    by_type(p.queries.type, p.cache.type, head_dim, [&](auto element, auto format, auto width) {
        using T = decltype(element);
        char *base = static_cast<char *>(workspace);
        int columns = 0; // rows of a split segment at most
        for (int pass = 0; pass < (prefix ? 2 : 1); ++pass) {
            const PassPlan plan = plan_pass(rows, p.sequences, args.group, pass);
            const Carve carve(rows, heads, head_dim, prefix, plan.part_columns, ctas);
            args.part_columns = plan.part_columns;
            args.closed = reinterpret_cast<ClosedSegment *>(base + carve.closed);
            args.table = prefix ? reinterpret_cast<int4 *>(base + carve.table) : nullptr;
            args.partials = reinterpret_cast<float *>(base + carve.partials);
            args.complete = prefix ? reinterpret_cast<float *>(base + carve.complete) : nullptr;
            base += carve.bytes;
            if (pass) {
                args.prefix = args.follows = true;
                args.pages = p.prefix_pages, args.lengths = p.prefix_length, args.sequences = 1;
                args.page_columns = args.page_stride = p.prefix_columns;
            }
            // Query rows of one segment at most: where each sequence has one row, those of a cached head.
            const int most = !pass && !p.query_offsets ? args.group : INT_MAX;
            if (plan.many) launch_many<T, decltype(format)::value, decltype(width)::value>(args, ctas, stream);
            else launch_pass<T, decltype(format)::value, decltype(width)::value>(plan.narrow, most, args, keys, values, ctas, stream);
            combine.source[pass] = {args.partials, args.complete, args.closed, args.table, ctas, plan.part_columns};
            columns = std::min(most, plan.part_columns);
        }
        constexpr int kWarps = kCombineThreads / 32;
        if (prefix)
            launch_pdl("attention combine", combine_prefixed<T, decltype(width)::value>, dim3(unsigned(((long long)rows * heads + kWarps - 1) / kWarps)),
                       dim3(kCombineThreads), 0, stream, combine);
        else // two rows a warp where there are many: most CTAs find no segment, the others have little to read
            launch_pdl("attention combine", combine_attention<T, decltype(width)::value>,
                       dim3(unsigned(ctas), unsigned(columns > 16 ? (columns + 2 * kWarps - 1) / (2 * kWarps) : (columns + kWarps - 1) / kWarps)), dim3(kCombineThreads),
                       0, stream, combine);
    });
}
} // namespace tts
