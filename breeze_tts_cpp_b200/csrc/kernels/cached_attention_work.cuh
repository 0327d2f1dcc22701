// What the attention kernels share: their arguments, and the division of the work over the CTAs.
//
// A segment is a sequence, a cached head and a tile of query rows; a tile is 128 keys of a segment. All CTAs get an equal run of the same list
// of tiles, whatever the lengths are, a segment's fixed cost counted as parts of a tile; a segment that runs over a share's end leaves partial
// sums, which a last launch adds in a fixed order. Lengths are on the device only, so every CTA adds the list up for itself.
#pragma once
#include "core/tensor.h"
#include "kernels/launch.cuh"
#include "kernels/quant_codec.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <climits>
#include <type_traits>

namespace tts::b200 {
constexpr int kTileKeys = 128;
constexpr int kPartialExtra = 8; // maximum and sum behind a partial row, padded to a sector of 32 bytes
constexpr int kScanAlone = 256;  // up to here a warp adds the sequences' work up by itself
constexpr size_t kAttentionSmem = 224 * 1024;

// The split segment that a CTA closes: where its parts lie, and whose rows they are. count == 0: none.
struct ClosedSegment {
    int first_cta, count, first_slot, row, flat, head, columns, unused;
};

// One pass over one set of page tables: the sequences' own, or the shared prefix as one sequence of all query rows.
struct AttentionArgs {
    const void *queries;
    void *output;
    int query_stride, output_stride, rows, heads, group, kv_heads;
    bool aligned, sectors; // rows of 16-bit elements start on 16 bytes; output rows on 32
    const int *pages, *lengths, *query_offsets;
    int sequences, page_columns, page_stride, page_shift, total_pages, box_shift;
    int offset_count; // entries of query_offsets behind the first; the last one counts the rows
    bool prefix;
    const void *cached_keys, *cached_values;
    const float *key_scales, *value_scales;
    float group_inverse;
    float score_scale; // softmax scale, log2 e and the key format's factor
    float output_scale;
    int stages, merge_columns, merge_buffers;
    int part_columns; // query rows that a partial sum has room for
    float *partials; // [ctas][2][part_columns][head_dim + kPartialExtra]
    ClosedSegment *closed; // [ctas]
    // With a shared prefix, whose rows take both passes' results: where each row's is, and the complete ones.
    int4 *table;     // [rows * heads]: first CTA, parts, slot of the first part, column; parts == 0: complete
    float *complete; // [rows * heads][head_dim + kPartialExtra]
    // The second pass of a call reads nothing that the first writes, so it does not wait for it (which has waited for what both read) before its end.
    bool follows;
    int *pass_word; // with a second pass: where the first says that it has waited; null otherwise
    int *status;
};

// The start of a pass, by all threads of a CTA; a barrier of the CTA among it. Dependents may start once what this pass reads is there.
__device__ __forceinline__ void begin_pass(const AttentionArgs &a) {
    if (a.follows) {
        // What came before the call was over (and its writes there for every proxy) when a thread of the first pass came out of its wait, released the word
        // and let this pass start. All CTAs of the first have to let it, so the word is there. A wait for all of the first pass instead takes 24 sequences
        // behind 509 tokens from 14.8 to 20.9 us and 128 behind 16384 from 85.3 to 92.0; the word itself costs 0.1 us at most.
        int word = 0;
        if (threadIdx.x == blockDim.x - 32) // the others set the CTA up meanwhile
            asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(word) : "l"(a.pass_word) : "memory");
        if (!__syncthreads_or(word == 1)) pdl_wait_upstream();
    } else {
        pdl_wait_upstream();
        if (a.pass_word && !blockIdx.x) { // one thread: no other of this CTA lets dependents start in front of the word
            if (threadIdx.x == blockDim.x - 32) {
                asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(a.pass_word), "r"(1) : "memory");
                pdl_launch_dependents();
            }
            __syncthreads();
            return;
        }
        __syncthreads();
    }
    pdl_launch_dependents();
}
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
    // A step of one token is spared the division, which several of its warps would wait for (one sequence of 777: 8.5 -> 8.2 us).
    if (!a.prefix && (Columns > 16 || s.count > 1)) end += min(s.count - 1, (qt * Columns + Columns - 1) / a.group) + 1 - s.count;
    return max(1, (end + kTileKeys - 1) / kTileKeys);
}
template <int Columns> __device__ __forceinline__ int query_tiles(const AttentionArgs &a, const SequenceShape &s) {
    return (s.count * a.group + Columns - 1) / Columns;
}
// Tiles of one head of a sequence, over its query tiles.
template <int Columns> __device__ __forceinline__ int head_tiles(const AttentionArgs &a, const SequenceShape &s, int count) {
    if (a.prefix || count <= 1) return count * tiles_of<Columns>(a, s, 0);
    int tiles = 0;
    for (int qt = 0; qt < count; ++qt) tiles += tiles_of<Columns>(a, s, qt);
    return tiles;
}
// Work of a run of sequences. The host refuses problems of more than kMostTiles, so all of it, in units, fits an int.
constexpr long long kMostTiles = 1ll << 27;
struct Work {
    int tiles = 0, segments = 0;
};
template <int Columns> __device__ __forceinline__ Work work_of(const AttentionArgs &a, int b) {
    const SequenceShape s = sequence_of(a, b);
    const int count = query_tiles<Columns>(a, s);
    return {a.kv_heads * head_tiles<Columns>(a, s, count), a.kv_heads * count};
}
__device__ __forceinline__ int scan_warp(int v, int lane) { // inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += other;
    }
    return v;
}
// Shares are counted in units: kTileUnits for a tile, `segment_units` more for a segment. A tile belongs to the CTA whose share holds its first unit.
constexpr int kTileUnits = 4;
struct Division {
    int each, rest, ctas, extra; // units per share, shares that have one more, shares, units of a segment

    // Where there is a CTA for every tile, each gets one. A share is never smaller than a tile, so that every CTA between a segment's first and
    // its last has a part of it.
    static __device__ Division of(const Work &all, int segment_units) {
        Division d{};
        d.ctas = min(all.tiles, int(gridDim.x));
        if (!d.ctas) return d;
        d.extra = all.tiles > int(gridDim.x) ? segment_units : 0;
        const unsigned total = d.units(all);
        d.each = int(total / unsigned(d.ctas)), d.rest = int(total) - d.each * d.ctas;
        return d;
    }
    __device__ int units(const Work &work) const { return kTileUnits * work.tiles + extra * work.segments; }
    __device__ int share_of(int cta) const { return each * min(cta, ctas) + min(min(cta, ctas), rest); } // its first unit
    __device__ int cta_of(int unit) const {
        const int larger = rest * (each + 1);
        return unit < larger ? int(unsigned(unit) / unsigned(each + 1)) : rest + int(unsigned(unit - larger) / unsigned(each));
    }
};
// Where a CTA's share begins: the sequence, and that sequence's first unit.
struct Start {
    Division division;
    int unit, sequence;
};
template <int Columns> __device__ __forceinline__ Work work_of_run(const AttentionArgs &a, int threads, int thread) {
    const int run = (a.sequences + threads - 1) / threads, from = min(a.sequences, thread * run), to = min(a.sequences, from + run);
    Work own;
    for (int b = from; b < to; ++b) {
        const Work w = work_of<Columns>(a, b);
        own.tiles += w.tiles, own.segments += w.segments;
    }
    return own;
}
// Whether this thread's run of sequences, `own` with `base` in front of it, holds the start of the CTA's share.
template <int Columns>
__device__ __forceinline__ bool holds_start(const AttentionArgs &a, int threads, int thread, const Work &base, const Work &own, Start &start) {
    const Division &d = start.division;
    const int begin = d.share_of(blockIdx.x);
    if (int(blockIdx.x) >= d.ctas || d.units(base) > begin || begin >= d.units(base) + d.units(own)) return false;
    const int run = (a.sequences + threads - 1) / threads, to = min(a.sequences, thread * run + run);
    start.unit = d.units(base);
    for (start.sequence = thread * run; start.sequence + 1 < to; ++start.sequence) {
        const int part = d.units(work_of<Columns>(a, start.sequence));
        if (begin < start.unit + part) break;
        start.unit += part;
    }
    return true;
}
// By one warp, for a batch of up to kScanAlone sequences.
template <int Columns> __device__ __forceinline__ Start start_alone(const AttentionArgs &a, int segment_units) {
    const int lane = threadIdx.x & 31;
    const Work own = work_of_run<Columns>(a, 32, lane);
    const Work through{scan_warp(own.tiles, lane), scan_warp(own.segments, lane)};
    Start start{};
    start.division = Division::of({__shfl_sync(0xffffffffu, through.tiles, 31), __shfl_sync(0xffffffffu, through.segments, 31)}, segment_units);
    const bool here = holds_start<Columns>(a, 32, lane, {through.tiles - own.tiles, through.segments - own.segments}, own, start);
    if (const unsigned who = __ballot_sync(0xffffffffu, here)) {
        start.sequence = __shfl_sync(0xffffffffu, start.sequence, __ffs(who) - 1);
        start.unit = __shfl_sync(0xffffffffu, start.unit, __ffs(who) - 1);
    }
    return start;
}
// By all threads of the CTA; `found` is for everyone behind the last barrier.
template <int Columns, int Warps> __device__ __forceinline__ void start_together(const AttentionArgs &a, int segment_units, Work *sums, Start *found) {
    const int warp = int(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const Work own = work_of_run<Columns>(a, 32 * Warps, int(threadIdx.x));
    Work before{scan_warp(own.tiles, lane), scan_warp(own.segments, lane)};
    Start start{};
    Work all;
    if (lane == 31) sums[warp] = before;
    __syncthreads();
    for (int w = 0; w < Warps; ++w) {
        if (w < warp) before.tiles += sums[w].tiles, before.segments += sums[w].segments;
        all.tiles += sums[w].tiles, all.segments += sums[w].segments;
    }
    before.tiles -= own.tiles, before.segments -= own.segments;
    start.division = Division::of(all, segment_units);
    if (!threadIdx.x) *found = start; // shares that hold nothing keep this
    __syncthreads();
    if (holds_start<Columns>(a, 32 * Warps, int(threadIdx.x), before, own, start)) *found = start;
    __syncthreads();
}

// The part of a segment that a CTA's share holds: tiles [low, high) of `tiles`.
struct SegmentPart {
    SequenceShape s;
    int sequence, head, query_tile, columns, tiles, low, high, ordinal;
    int first_cta, first_slot; // of all parts, for the CTA that closes a split segment; -1 elsewhere
    int slot;                  // where a partial sum goes: 0 for a share's first part, 1 for a later one
    bool split, final;
};
// What a CTA says about the segment that it closes, for the launch that adds up the parts; `part` null: that it closes none.
__device__ __forceinline__ void note_closed(const AttentionArgs &a, const SegmentPart *part, int columns_per_tile) {
    ClosedSegment c{};
    if (part)
        c = {part->first_cta, int(blockIdx.x) - part->first_cta + 1, part->first_slot, part->s.row, part->query_tile * columns_per_tile, part->head, part->columns, 0};
    a.closed[blockIdx.x] = c;
}
// Calls `each` for every part of this CTA's share, in order, until it returns false. Returns the number of parts.
template <int Columns, class Each>
__device__ __forceinline__ int walk_share(const AttentionArgs &a, const Start &start, Each &&each) {
    const Division &d = start.division;
    const int begin = d.share_of(blockIdx.x), end = d.share_of(int(blockIdx.x) + 1);
    int at = start.unit;
    SegmentPart p;
    p.ordinal = 0;
    for (p.sequence = start.sequence; begin < end && p.sequence < a.sequences && at < end; ++p.sequence) {
        p.s = sequence_of(a, p.sequence);
        const int count = query_tiles<Columns>(a, p.s);
        int segment = 0;
        if (begin > at) { // whole heads in front of the share
            const int head_units = kTileUnits * head_tiles<Columns>(a, p.s, count) + d.extra * count;
            const int heads = head_units ? min(int(unsigned(begin - at) / unsigned(head_units)), a.kv_heads) : 0;
            segment = heads * count, at += heads * head_units;
        }
        // Heads outermost: their query tiles read the same keys, near one another in time.
        for (; segment < count * a.kv_heads && at < end; ++segment) {
            p.head = count == 1 ? segment : segment / count, p.query_tile = segment - p.head * count, p.tiles = tiles_of<Columns>(a, p.s, p.query_tile);
            const int first_unit = at + d.extra;
            at = first_unit + kTileUnits * p.tiles;
            const auto tile_from = [&](int unit) { // first tile that starts at or behind a unit
                return unit <= first_unit ? 0 : unit >= at ? p.tiles : (unit - first_unit + kTileUnits - 1) / kTileUnits;
            };
            p.low = tile_from(begin), p.high = tile_from(end);
            if (p.low == p.high) continue;
            p.split = p.low || p.high < p.tiles;
            p.first_cta = -1, p.first_slot = 0;
            if (p.split && p.high == p.tiles) { // this CTA closes the segment: it says where its parts lie
                p.first_cta = d.cta_of(first_unit);
                p.first_slot = d.share_of(p.first_cta) < first_unit - d.extra ? 1 : 0;
            }
            p.slot = first_unit - d.extra > begin ? 1 : 0;
            p.columns = min(Columns, p.s.count * a.group - p.query_tile * Columns);
            p.final = p.high < p.tiles || at + d.extra >= end;
            if (!each(p)) return p.ordinal;
            ++p.ordinal;
        }
    }
    return p.ordinal;
}

// One query row's result: the output row, or what is kept of it for the second launch.
template <class T>
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

} // namespace tts::b200
