// Attention of a few query rows per sequence over the quantized, paged cache: decode, and drafts of some tokens.
//
// Mathematics. Keys and values are bytes with one fp32 scale per token, so s_j = (q . kq_j) ks_j times the softmax scale, and the output is
// sum p_j vs_j vq_j / sum p_j. The products run on the tensor cores in fp16 with fp32 sums: an INT8 byte is exact in fp16, and so is an
// e4m3 byte times 2^-8 (its bits shifted into place; the factor goes into the score's and the output's scale). Queries are exact too: each
// row is divided by the power of two of its largest element. What is rounded is p_j vs_j, to fp16. To keep that product in fp16's
// range whatever the scales are, the running maximum is taken over log2 p_j vs_j, so the product is at most one; the sum of p_j
// alone uses the same reference and is fp32.
//
// Layout. S is computed transposed: 16 keys are the rows of an m16n8k16 product and 8 query rows its columns, so a decode step with two
// query rows per cached head wastes 6 columns of 8, not 14 of 16. The order of the contraction over head_dim is free, so a thread's
// share of a key row is 32 consecutive bytes: operands come straight from the copied tile, with 16-byte shared loads and byte permutations. The
// transposed weights take one 8 x 8 transposition in registers to become the second product's operand; its rows are head_dim and a
// thread owns 16 consecutive columns of the output.
//
// Bound. A cached byte takes part in 2 x query rows multiply-adds and costs about 1.3 instructions of conversion; at two to eight rows per head memory is
// the floor. One CTA per multiprocessor streams 128-token tiles (box copies by the tensor map, 128-byte swizzle, so that no shared load has
// a bank conflict) through a ring; eight warps take 16 keys of a tile each and keep their own softmax state and output, which meet once per
// segment. Work is divided evenly over the CTAs in tiles, whatever the lengths are: a CTA's share is a run of consecutive tiles, a segment (sequence, cached
// head, query tile) that runs over a share's end leaves partial sums that a second launch adds in a fixed order.
#pragma once
#include "kernels/launch.cuh"
#include "kernels/sm100_ptx.cuh"
#include "core/tensor.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace tts::b200 {
constexpr int kTileKeys = 128, kAttentionWarps = 8, kAttentionThreads = 32 * (kAttentionWarps + 1);
constexpr int kPartialExtra = 4; // maximum and sum behind a partial row, padded to 16 bytes
constexpr size_t kAttentionSmem = 224 * 1024;

// One pass over one set of page tables: the sequences' own, or the shared prefix as one sequence of all query rows.
struct AttentionArgs {
    const void *queries;
    void *output;
    int query_stride, output_stride, rows, heads, group, kv_heads;
    bool aligned;
    const int *pages, *lengths, *query_offsets;
    int sequences, page_columns, page_stride, page_shift, total_pages, box_shift;
    int offset_count; // entries of query_offsets behind the first; the last one counts the rows
    bool prefix;
    const float *key_scales, *value_scales;
    float score_scale; // softmax scale, log2 e and the key format's factor
    float output_scale;
    float *partials; // [ctas][2][columns][head_dim + kPartialExtra]
    int4 *table;     // [rows * heads]: first CTA, parts, slot of the first part, column; parts == 0: complete
    float *complete; // [rows * heads][head_dim + kPartialExtra], or null: complete segments go to the output
    int *status;
};

__device__ __forceinline__ int load_index(const int *p) {
    int v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float log2_approx(float x) {
    float r;
    asm("lg2.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Untiled copy of a run of bytes (both ends and the size multiples of 16).
__device__ __forceinline__ void copy_run(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}
// The four bytes of x as fp16: lo = (byte 0, byte 1), hi = (byte 2, byte 3). INT8 exactly (x carries an offset of 128, see biased), e4m3
// times 2^-8 (whatever the bits: a NaN code reads as 480, so that masked garbage stays finite; the writer marks NaN in the scale).
template <Type F> __device__ __forceinline__ void widen(uint32_t x, uint32_t &lo, uint32_t &hi) {
    if constexpr (F == Type::I8) {
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342); // 1024 + byte
        const uint32_t offset = 0x64806480u;                                                              // 1152
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(offset));
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(offset));
    } else {
        const uint32_t a = __byte_perm(x, 0u, 0x1404), b = __byte_perm(x, 0u, 0x3424);
        lo = (a & 0x80008000u) | ((a >> 1) & 0x3f803f80u);
        hi = (b & 0x80008000u) | ((b >> 1) & 0x3f803f80u);
    }
}
template <Type F> __device__ __forceinline__ uint32_t biased(uint32_t x) { return F == Type::I8 ? x ^ 0x80808080u : x; }

// Where a row's 16-byte piece lies in a tile as the tensor map's swizzle lays it down.
template <int HeadDim> __device__ __forceinline__ uint32_t piece(int row, int chunk) {
    return HeadDim == 128 ? uint32_t(row * 128 + ((chunk ^ (row & 7)) << 4)) : uint32_t(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}

template <int HeadDim, int Tiles> struct AttentionShape {
    static constexpr int columns = 8 * Tiles; // query rows of a segment
    static constexpr int row = HeadDim + kPartialExtra;
    static constexpr uint32_t values = kTileKeys * HeadDim, scales = 2 * kTileKeys * HeadDim; // offsets in a stage
    static constexpr uint32_t stage = scales + 2 * kTileKeys * 4;
    static constexpr uint32_t merge = kAttentionWarps * columns * row * 4;
    static constexpr uint32_t stage_aligned = (stage + 1023) / 1024 * 1024;
    static constexpr int stages = int((kAttentionSmem - 2048 - merge) / stage_aligned) > 12 ? 12 : int((kAttentionSmem - 2048 - merge) / stage_aligned);
    static constexpr size_t smem = 1024 + size_t(stages) * stage_aligned + merge;
};

// What the producer tells the consumers about a tile.
struct TileNote {
    int key, head, row, count, flat, limit, flags, first_cta, first_slot, slot, pad[6];
};
constexpr int kNoteFirst = 1, kNoteLast = 2, kNoteSplit = 4;

// A sequence as the tables give it, made safe: rows and positions stay inside of what the caller passed.
struct SequenceShape {
    int length, count, row;
};
__device__ __forceinline__ SequenceShape sequence_of(const AttentionArgs &a, int b) {
    SequenceShape s;
    if (a.prefix) {
        s.row = 0;
        s.count = a.query_offsets ? load_index(a.query_offsets + a.offset_count) : a.rows;
    } else if (a.query_offsets) {
        s.row = load_index(a.query_offsets + b);
        s.count = load_index(a.query_offsets + b + 1) - s.row;
    } else {
        s.row = b;
        s.count = 1;
    }
    s.row = max(s.row, 0);
    s.count = max(0, min(s.count, a.rows - s.row));
    s.length = max(0, min(load_index(a.lengths + b), a.page_columns << a.page_shift));
    return s;
}
// Tiles of keys that query tile `qt` of a sequence sees; at least one, so that rows that see nothing are written too.
template <int Columns> __device__ __forceinline__ int tiles_of(const AttentionArgs &a, const SequenceShape &s, int qt) {
    int end = s.length;
    if (!a.prefix) end += min(s.count - 1, (qt * Columns + Columns - 1) / a.group) + 1 - s.count;
    return max(1, (end + kTileKeys - 1) / kTileKeys);
}
template <int Columns> __device__ __forceinline__ int query_tiles(const AttentionArgs &a, const SequenceShape &s) {
    return (s.count * a.group + Columns - 1) / Columns;
}
template <int Columns> __device__ __forceinline__ long long work_of(const AttentionArgs &a, const SequenceShape &s) {
    const int tiles = query_tiles<Columns>(a, s);
    if (a.prefix) return (long long)tiles * a.kv_heads * tiles_of<Columns>(a, s, 0);
    long long sum = 0;
    for (int qt = 0; qt < tiles; ++qt) sum += tiles_of<Columns>(a, s, qt);
    return sum * a.kv_heads;
}

// One query row's result: the output row, or what is kept of it for the second launch.
template <class T, int HeadDim>
__device__ __forceinline__ void store_row4(const AttentionArgs &a, T *to, float4 v, float factor) {
    union {
        uint2 word;
        T e[4];
    } out;
    out.e[0] = T(v.x * factor), out.e[1] = T(v.y * factor), out.e[2] = T(v.z * factor), out.e[3] = T(v.w * factor);
    if (a.aligned) {
        *reinterpret_cast<uint2 *>(to) = out.word;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) to[i] = out.e[i];
    }
}

template <class T, Type F, int HeadDim, int Tiles>
__global__ void __launch_bounds__(kAttentionThreads, 1)
    cached_attention(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, const AttentionArgs args) {
    using Shape = AttentionShape<HeadDim, Tiles>;
    constexpr int kColumns = Shape::columns, kStages = Shape::stages, kSteps = HeadDim / 16, kThreads = kAttentionThreads;
    extern __shared__ uint8_t raw_smem[];
    __shared__ uint64_t full[kStages], empty[kStages], meet[2];
    __shared__ TileNote notes[kStages];
    __shared__ long long sums[kAttentionWarps + 1];
    __shared__ long long found[2]; // sequence of this CTA's first tile, tiles of it that others take
    __shared__ int abort_flag;
    const uint32_t ring = (ptx::smem_u32(raw_smem) + 1023u) & ~1023u;
    float *merge = reinterpret_cast<float *>(raw_smem + (ring - ptx::smem_u32(raw_smem)) + kStages * Shape::stage_aligned);
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;

    if (!threadIdx.x) {
        for (int s = 0; s < kStages; ++s) {
            ptx::mbar_init(ptx::smem_u32(&full[s]), 1);
            ptx::mbar_init(ptx::smem_u32(&empty[s]), kAttentionWarps);
        }
        ptx::mbar_init(ptx::smem_u32(&meet[0]), kAttentionWarps);
        ptx::mbar_init(ptx::smem_u32(&meet[1]), kAttentionWarps);
        abort_flag = 0;
        found[0] = found[1] = 0;
        ptx::fence_barrier_init();
        ptx::prefetch_tensormap(&key_map);
        ptx::prefetch_tensormap(&value_map);
    }
    pdl_launch_dependents();
    pdl_wait_upstream();

    // Every CTA adds up all sequences' tiles: a thread takes a run of sequences, then a scan over the threads.
    const int run = (args.sequences + kThreads - 1) / kThreads;
    const int from = min(args.sequences, int(threadIdx.x) * run), to = min(args.sequences, from + run);
    long long own = 0;
    for (int b = from; b < to; ++b) own += work_of<kColumns>(args, sequence_of(args, b));
    long long before = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, before, d);
        if (lane >= d) before += other;
    }
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w <= kAttentionWarps; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    before -= own;
    // At least a tile for every CTA that takes part.
    const long long ctas = total < gridDim.x ? total : gridDim.x;
    if (blockIdx.x >= ctas) return;
    const long long begin = total * blockIdx.x / ctas, end = total * (blockIdx.x + 1) / ctas;
    if (before <= begin && begin < before + own) {
        long long at = before;
        for (int b = from; b < to; ++b) {
            const long long work = work_of<kColumns>(args, sequence_of(args, b));
            if (begin < at + work) {
                found[0] = b;
                found[1] = begin - at;
                break;
            }
            at += work;
        }
    }
    __syncthreads();
    const int count = int(end - begin);
    // Every wait is bounded, and a warp whose wait gave up leaves as one; the others follow when theirs do.
    auto wait = [&](uint64_t &bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar), parity, &abort_flag))) return true;
        if (!lane) *args.status = 1;
        return false;
    };

    if (warp == kAttentionWarps) { // ------------------------------------------------------------ producer
        int b = int(found[0]), skip = int(found[1]), h = 0, qt = 0, tile = 0;
        SequenceShape s = sequence_of(args, b);
        int qts = query_tiles<kColumns>(args, s), tiles = tiles_of<kColumns>(args, s, 0);
        auto next_segment = [&] { // heads outermost: their query tiles read the same keys, near one another in time
            if (++qt == qts) {
                qt = 0;
                if (++h == args.kv_heads) {
                    h = 0;
                    do {
                        if (++b >= args.sequences) return;
                        s = sequence_of(args, b);
                        qts = query_tiles<kColumns>(args, s);
                    } while (!qts);
                }
            }
            tiles = tiles_of<kColumns>(args, s, qt);
        };
        while (skip >= tiles) {
            skip -= tiles;
            next_segment();
        }
        tile = skip;
        const int box = 1 << args.box_shift, boxes = kTileKeys >> args.box_shift;
        const uint32_t box_bytes = uint32_t(box) * (2 * HeadDim + 8);
        int stage = 0, issued = 0;
        uint32_t phase = 0;
        for (; issued < count; ++issued) {
            if (issued >= kStages && !wait(empty[stage], phase ^ 1)) break;
            const int key = tile * kTileKeys, mine = lane >> 2, kind = lane & 3;
            const uint32_t at = ring + stage * Shape::stage_aligned, bar = ptx::smem_u32(&full[stage]);
            // Lane 4i + k copies part k (keys, values, their scales) of box i.
            const int position = key + (mine << args.box_shift);
            const bool wanted = mine < boxes && position < s.length;
            int page = -1;
            if (wanted) page = load_index(args.pages + size_t(b) * args.page_stride + (position >> args.page_shift));
            const bool good = wanted && unsigned(page) < unsigned(args.total_pages);
            // Positions on a page that the cache does not have read as NaN.
            if (wanted && !good && kind >= 2) {
                float *scales = reinterpret_cast<float *>(raw_smem + (at - ptx::smem_u32(raw_smem)) + Shape::scales) + (kind - 2) * kTileKeys;
                for (int i = 0; i < box; ++i) scales[(mine << args.box_shift) + i] = __int_as_float(0x7fffffff);
            }
            __syncwarp();
            const uint32_t copied = __popc(__ballot_sync(0xffffffffu, good)) / 4;
            if (!lane) {
                const long long at_tile = begin + issued, segment = at_tile - tile; // the segment's first tile
                TileNote &n = notes[stage];
                n.key = key, n.head = h, n.row = s.row, n.count = s.count, n.flat = qt * kColumns;
                n.limit = args.prefix ? s.length - 1 : s.length - s.count;
                const bool last = tile + 1 == tiles, starts_here = segment >= begin;
                const bool split = !starts_here || segment + tiles > end;
                n.flags = (tile == 0 || !issued ? kNoteFirst : 0) | (last || issued + 1 == count ? kNoteLast : 0) | (split ? kNoteSplit : 0);
                n.slot = segment > begin ? 1 : 0;
                n.first_cta = -1;
                if (last && split) { // this CTA closes the segment: it says where its parts lie
                    int cta = int(segment * ctas / total);
                    while (total * (cta + 1) / ctas <= segment) ++cta;
                    n.first_cta = cta;
                    n.first_slot = total * cta / ctas < segment ? 1 : 0;
                }
                ptx::mbar_arrive_expect_tx(bar, copied * box_bytes);
            }
            __syncwarp();
            if (good) {
                const int row = (((page * args.kv_heads) + h) << args.page_shift) + (position & ((1 << args.page_shift) - 1));
                const uint32_t offset = uint32_t(mine << args.box_shift);
                if (kind == 0) ptx::tma_load_2d(at + offset * HeadDim, &key_map, bar, 0, row);
                else if (kind == 1) ptx::tma_load_2d(at + Shape::values + offset * HeadDim, &value_map, bar, 0, row);
                else copy_run(at + Shape::scales + (kind - 2) * kTileKeys * 4 + offset * 4, (kind == 2 ? args.key_scales : args.value_scales) + row, uint32_t(box) * 4, bar);
            }
            if (++tile == tiles && issued + 1 < count) {
                tile = 0;
                next_segment();
            }
            if (++stage == kStages) stage = 0, phase ^= 1;
        }
        // No copy may be in flight when the CTA leaves, whatever the consumers did.
        int ignored = 0;
        for (int i = max(0, issued - kStages); i < issued; ++i)
            ptx::mbar_wait(ptx::smem_u32(&full[i % kStages]), uint32_t(i / kStages) & 1, &ignored);
        return;
    }

    // ------------------------------------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    uint32_t q[Tiles][kSteps][2];
    float out[Tiles][kSteps][4], most[Tiles][2], sum[Tiles][2], factor[Tiles][2];
    int limit[Tiles][2], least = 0;
    int stage = 0, segments = 0;
    uint32_t phase = 0;
    for (int i = 0; i < count; ++i) {
        if (!wait(full[stage], phase)) return;
        const TileNote &note = notes[stage];
        const uint32_t at = ring + stage * Shape::stage_aligned;
        const float *scales = reinterpret_cast<const float *>(raw_smem + (at - ptx::smem_u32(raw_smem)) + Shape::scales);
        const int flags = note.flags;
        if (flags & kNoteFirst) {
            const int columns = note.count * args.group - note.flat;
            least = INT_MAX;
#pragma unroll
            for (int n = 0; n < Tiles; ++n) {
                // This lane's share of query row 8n + g: columns [HeadDim / 4 * t, HeadDim / 4 * (t + 1)).
                constexpr int kShare = HeadDim / 4;
                const int column = 8 * n + g, flat = note.flat + column;
                const bool live = column < columns;
                const T *row = static_cast<const T *>(args.queries) + size_t(note.row + flat / args.group) * args.query_stride +
                               (note.head * args.group + flat % args.group) * HeadDim + kShare * t;
                alignas(16) T share[kShare];
                if (live && args.aligned) {
#pragma unroll
                    for (int c = 0; c < kShare / 8; ++c) {
                        uint4 v;
                        asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(row + 8 * c) : "memory");
                        *reinterpret_cast<uint4 *>(share + 8 * c) = v;
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < kShare; ++c) {
                        uint16_t v = 0;
                        if (live) asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(row + c) : "memory");
                        reinterpret_cast<uint16_t *>(share)[c] = v;
                    }
                }
                unsigned largest = 0;
#pragma unroll
                for (int c = 0; c < kShare; ++c) largest = max(largest, __float_as_uint(float(share[c])) & 0x7fffffffu);
                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                const int exponent = largest && largest < 0x7f800000u ? max(int(largest >> 23), 1) - 127 : 0;
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const __half2 v = __floats2half2_rn(ldexpf(float(share[4 * k + 2 * c]), -exponent), ldexpf(float(share[4 * k + 2 * c + 1]), -exponent));
                        q[n][k][c] = *reinterpret_cast<const uint32_t *>(&v);
                    }
                // The scores of this lane belong to columns 2t and 2t + 1, whose rows lanes 8t and 8t + 4 hold.
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int of = __shfl_sync(0xffffffffu, exponent, 8 * t + 4 * c), seen = 8 * n + 2 * t + c;
                    factor[n][c] = ldexpf(args.score_scale, of);
                    limit[n][c] = seen < columns ? (args.prefix ? note.limit : note.limit + (note.flat + seen) / args.group) : -1;
                    if (seen < columns) least = min(least, limit[n][c]);
                    most[n][c] = -INFINITY;
                    sum[n][c] = 0.f;
                }
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) out[n][k][c] = 0.f;
            }
            least = __reduce_min_sync(0xffffffffu, least);
        }

        // Scores of this warp's 16 keys.
        const int row = 16 * warp;
        uint32_t keys[2][HeadDim / 16];
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < HeadDim / 64; ++c)
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(keys[r][4 * c]), "=r"(keys[r][4 * c + 1]), "=r"(keys[r][4 * c + 2]), "=r"(keys[r][4 * c + 3])
                             : "r"(at + piece<HeadDim>(row + g + 8 * r, HeadDim / 64 * t + c)));
        float scores[Tiles][2][4] = {};
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            uint32_t a[4];
            widen<F>(biased<F>(keys[0][k]), a[0], a[2]);
            widen<F>(biased<F>(keys[1][k]), a[1], a[3]);
#pragma unroll
            for (int n = 0; n < Tiles; ++n) mma_f16(scores[n][k & 1], a[0], a[1], a[2], a[3], q[n][k][0], q[n][k][1]);
        }
        // Values of keys 2t, 2t + 1, 2t + 8, 2t + 9: this thread's 16 (8) columns.
        uint32_t values[4][HeadDim / 32];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int key = row + 2 * t + (r & 1) + 8 * (r >> 1);
            if constexpr (HeadDim == 128)
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(values[r][0]), "=r"(values[r][1]), "=r"(values[r][2]), "=r"(values[r][3])
                             : "r"(at + Shape::values + piece<HeadDim>(key, g)));
            else
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                             : "=r"(values[r][0]), "=r"(values[r][1])
                             : "r"(at + Shape::values + piece<HeadDim>(key, g >> 1) + 8 * (g & 1)));
        }
        const float key_scale[2] = {scales[row + g], scales[row + g + 8]};
        float value_scale[2] = {scales[kTileKeys + row + g], scales[kTileKeys + row + g + 8]};
        const int position = note.key + row + g;
        const bool masked = note.key + kTileKeys - 1 > least;
        uint32_t weights[Tiles][2];
#pragma unroll
        for (int n = 0; n < Tiles; ++n) {
            float x[2][2], highest[2] = {-INFINITY, -INFINITY};
            bool seen[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float shift = fmaxf(log2_approx(fabsf(value_scale[r])), -126.f);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    seen[r][c] = !masked || position + 8 * r <= limit[n][c];
                    x[r][c] = (scores[n][0][2 * r + c] + scores[n][1][2 * r + c]) * (key_scale[r] * factor[n][c]);
                    if (!seen[r][c]) x[r][c] = -INFINITY;
                    else highest[c] = fmaxf(highest[c], x[r][c] + shift);
                }
            }
            float raised[2];
            bool changed = false;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) highest[c] = fmaxf(highest[c], __shfl_xor_sync(0xffffffffu, highest[c], d));
                raised[c] = fmaxf(most[n][c], highest[c]);
                changed |= raised[c] > most[n][c];
            }
            if (__any_sync(0xffffffffu, changed)) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float shrink = raised[c] == -INFINITY ? 1.f : exp2_approx(most[n][c] - raised[c]);
                    sum[n][c] *= shrink;
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) out[n][k][c] *= shrink, out[n][k][2 + c] *= shrink;
                    most[n][c] = raised[c];
                }
            }
            float w[2][2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float reference = most[n][c] == -INFINITY ? 0.f : most[n][c];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float p = exp2_approx(x[r][c] - reference);
                    sum[n][c] += p;
                    w[r][c] = seen[r][c] ? p * value_scale[r] : 0.f; // a hidden row's scale may be anything
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const __half2 both = __floats2half2_rn(w[r][0], w[r][1]);
                weights[n][r] = transpose8x8(*reinterpret_cast<const uint32_t *>(&both));
            }
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const uint32_t order = k & 1 ? 0x7362u : 0x5140u; // bytes 2 (k & 1) and the next of two keys, side by side
            uint32_t a[4];
            widen<F>(biased<F>(__byte_perm(values[0][k >> 1], values[1][k >> 1], order)), a[0], a[1]);
            widen<F>(biased<F>(__byte_perm(values[2][k >> 1], values[3][k >> 1], order)), a[2], a[3]);
#pragma unroll
            for (int n = 0; n < Tiles; ++n) mma_f16(out[n][k], a[0], a[1], a[2], a[3], weights[n][0], weights[n][1]);
        }

        if (flags & kNoteLast) { // the eight warps' shares of the segment meet
            const int columns = min(kColumns, note.count * args.group - note.flat);
            if (segments && !wait(meet[1], uint32_t(segments - 1) & 1)) return;
#pragma unroll
            for (int n = 0; n < Tiles; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float l = sum[n][c];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                    const int column = 8 * n + 2 * t + c;
                    if (column >= columns) continue;
                    float *to = merge + (warp * kColumns + column) * Shape::row;
#pragma unroll
                    for (int k = 0; k < kSteps; k += 2)
                        *reinterpret_cast<float4 *>(to + g * kSteps * 2 + 2 * k) =
                            make_float4(out[n][k][c], out[n][k][2 + c], out[n][k + 1][c], out[n][k + 1][2 + c]);
                    if (!g) to[HeadDim] = most[n][c], to[HeadDim + 1] = l;
                }
            __syncwarp();
            if (!lane) ptx::mbar_arrive(ptx::smem_u32(&meet[0]));
            if (!wait(meet[0], uint32_t(segments) & 1)) return;
            for (int item = threadIdx.x; item < columns * (HeadDim / 4); item += 32 * kAttentionWarps) {
                const int column = item / (HeadDim / 4), d = 4 * (item % (HeadDim / 4));
                float highest = -INFINITY;
#pragma unroll
                for (int w = 0; w < kAttentionWarps; ++w) highest = fmaxf(highest, merge[(w * kColumns + column) * Shape::row + HeadDim]);
                const float reference = highest == -INFINITY ? 0.f : highest;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float l = 0.f;
#pragma unroll
                for (int w = 0; w < kAttentionWarps; ++w) {
                    const float *from = merge + (w * kColumns + column) * Shape::row;
                    const float f = exp2_approx(from[HeadDim] - reference);
                    const float4 x = *reinterpret_cast<const float4 *>(from + d);
                    v.x += f * x.x, v.y += f * x.y, v.z += f * x.z, v.w += f * x.w;
                    l += f * from[HeadDim + 1];
                }
                const int flat = note.flat + column, head = note.head * args.group + flat % args.group;
                const size_t at_row = size_t(note.row + flat / args.group), index = at_row * args.heads + head;
                float *kept = flags & kNoteSplit ? args.partials + (size_t(blockIdx.x * 2 + note.slot) * kColumns + column) * Shape::row
                              : args.complete    ? args.complete + index * Shape::row
                                                 : nullptr;
                if (kept) {
                    *reinterpret_cast<float4 *>(kept + d) = v;
                    if (!d) kept[HeadDim] = highest, kept[HeadDim + 1] = l;
                } else {
                    store_row4<T, HeadDim>(args, static_cast<T *>(args.output) + at_row * args.output_stride + head * HeadDim + d, v,
                                           l == 0.f ? 0.f : args.output_scale / l);
                }
                if (!d) {
                    if (!(flags & kNoteSplit)) args.table[index] = make_int4(0, 0, 0, 0);
                    else if (note.first_cta >= 0) args.table[index] = make_int4(note.first_cta, int(blockIdx.x) - note.first_cta + 1, note.first_slot, column);
                }
            }
            __syncwarp();
            if (!lane) ptx::mbar_arrive(ptx::smem_u32(&meet[1]));
            ++segments;
        }
        __syncwarp();
        if (!lane) ptx::mbar_arrive(ptx::smem_u32(&empty[stage]));
        if (++stage == kStages) stage = 0, phase ^= 1;
    }
}

// Second launch: a warp per query row and head adds up what the first left in parts (own, and the shared prefix's), in the order of the
// CTAs. Rows that are complete already cost it one read.
struct CombineSource {
    const float *partials, *complete; // complete == null: segments in one part are written already
    const int4 *table;
    int ctas, columns;
};
struct CombineArgs {
    CombineSource source[2];
    int sources, rows, heads, output_stride;
    bool aligned;
    const int *row_count; // last of the query offsets, or null
    void *output;
    float output_scale;
};
template <class T, int HeadDim> __global__ void __launch_bounds__(256) combine_attention(const CombineArgs args) {
    constexpr int kRow = HeadDim + kPartialExtra, kShare = HeadDim / 32;
    pdl_launch_dependents();
    pdl_wait_upstream();
    const int lane = threadIdx.x & 31;
    const long long index = (long long)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int rows = args.row_count ? min(args.rows, load_index(args.row_count)) : args.rows;
    if (index >= (long long)rows * args.heads) return;
    float highest = -INFINITY, l = 0.f, v[kShare] = {};
    bool written = args.sources == 1;
    for (int i = 0; i < args.sources; ++i) {
        const CombineSource &s = args.source[i];
        int4 entry;
        asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(entry.x), "=r"(entry.y), "=r"(entry.z), "=r"(entry.w) : "l"(s.table + index) : "memory");
        const bool whole = entry.y <= 0;
        if (whole && !s.complete) continue;
        // Rows that no sequence covers have no entry: whatever stands there stays inside the workspace.
        if (!whole && (entry.x < 0 || entry.y > s.ctas - entry.x || unsigned(entry.z) > 1u || unsigned(entry.w) >= unsigned(s.columns))) continue;
        written = false;
        const int parts = whole ? 1 : entry.y;
        for (int part = 0; part < parts; ++part) {
            const float *from = whole ? s.complete + size_t(index) * kRow
                                      : s.partials + (size_t((entry.x + part) * 2 + (part ? 0 : entry.z)) * s.columns + entry.w) * kRow;
            const float other = from[HeadDim], raised = fmaxf(highest, other), reference = raised == -INFINITY ? 0.f : raised;
            const float a = exp2_approx(highest - reference), b = exp2_approx(other - reference);
#pragma unroll
            for (int c = 0; c < kShare; ++c) v[c] = v[c] * a + from[kShare * lane + c] * b;
            l = l * a + from[HeadDim + 1] * b;
            highest = raised;
        }
    }
    if (written) return;
    const float factor = l == 0.f ? 0.f : args.output_scale / l;
    T *to = static_cast<T *>(args.output) + size_t(index / args.heads) * args.output_stride + size_t(index % args.heads) * HeadDim + kShare * lane;
#pragma unroll
    for (int c = 0; c < kShare; ++c) to[c] = T(v[c] * factor);
}
} // namespace tts::b200
