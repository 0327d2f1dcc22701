// Attention of a few query rows per sequence over the quantized, paged cache: decode, and drafts of some tokens.
//
// Mathematics. Keys and values are bytes with one fp32 scale per token, so s_j = (q . kq_j) ks_j times the softmax scale, and the output is
// sum p_j vs_j vq_j / sum p_j. The products run on the tensor cores in fp16 with fp32 sums: an INT8 byte is exact in fp16, and so is an
// e4m3 byte times 2^-8 (its bits shifted into place; the factor goes into the score's and the output's scale). Two things are rounded.
// BF16 queries (F16 ones enter as they are): a row is divided by the power of two of its largest element, which leaves elements down to 2^-17 of that
// power exact and rounds those below to within 2^-25 of it; a product in bf16 would keep them, but four bytes take eight instructions to become that, not five. And
// p_j vs_j, to fp16: to keep that product in fp16's range whatever the scales are, the running maximum is taken over log2 p_j vs_j, so it is at most
// one; the sum of p_j alone uses the same reference and is fp32.
//
// Layout. S is computed transposed: 16 keys are the rows of an m16n8k16 product and 8 query rows its columns, so a decode step with two
// query rows per cached head wastes 6 columns of 8, not 14 of 16. The order of the contraction over head_dim is free, so a thread's
// share of a key row is 32 consecutive bytes: operands come straight from the copied tile, with 16-byte shared loads and byte permutations. The
// transposed weights take one 8 x 8 transposition in registers to become the second product's operand; its rows are head_dim and a
// thread owns 16 consecutive columns of the output.
//
// Bound. A cached byte takes part in 2 x query rows multiply-adds and costs about 1.4 instructions of conversion; at two to eight rows per
// head memory is the floor. One CTA per multiprocessor streams 128-token tiles (box copies by the tensor map, 128-byte swizzle, so that no
// shared load has a bank conflict; the segment's query rows come with its first tiles) through a ring. Groups of four warps take the
// tiles in turn, 32 keys a warp, so that a warp has two independent chains and its scheduler other warps; each warp keeps its own softmax state and output.
// At a segment's end the warps leave theirs in shared memory and go on; two further warps add them up and store.
//
// Measured on the device (16 heads over 8, 128 wide, INT8, pages of 64). 64 sequences of up to 4096 tokens: 58.3 us for 275 MB, 4.7 TB/s, 73 % of what a copy
// reaches; 13 of up to 16001 with 32 heads, e4m3, pages of 16: 43.0 us, 4.35 TB/s. A warp's step of 32 keys takes about 1800 cycles, a segment's
// queries 1000 and its way out 800. One sequence of 777 tokens: 8.1 us for two launches, nearly all of it instructions met for the first time,
// the lengths, the pages and the copies, one behind the other.
//
// Division. A segment is a sequence, a cached head and a tile of query rows. All CTAs get an equal run of the same list of tiles, whatever
// the lengths are, a segment's fixed cost counted as a part of a tile; a segment that runs over a share's end leaves partial sums, which a second launch adds in
// a fixed order.
#pragma once
#include "kernels/cached_attention_work.cuh"
#include "kernels/sm100_ptx.cuh"

namespace tts::b200 {
constexpr int kTeam = 4, kTeams = 2, kWorkers = kTeam * kTeams, kProducers = 2, kMergers = 2, kMaxRing = 12, kMergeBuffers = 4;
constexpr int kAttentionWarps = kWorkers + kProducers + kMergers, kAttentionThreads = 32 * kAttentionWarps; // three per scheduler: 168 registers a thread
constexpr int kFewSegmentUnits = 6; // a segment's queries, flush and merge next to a tile's kTileUnits (64 sequences of up to 4096: 2 units 65.2 us, 4 60.9, 6 59.9)

// log2 of the least value scale that the reference follows. Behind smaller ones, zero among them, p_j grows to 2^96, of which fp32 holds a sum of 2^23
// (with many rows' slack); what their values add lies below 2^-96 of the format's range.
constexpr float kLeastScale = -96.f;
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
__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// The same for key bytes, e4m3 without a factor: a key that is not a number makes a score that is none, and hidden scores are replaced.
template <Type F> __device__ __forceinline__ void widen_key(uint32_t x, uint32_t &lo, uint32_t &hi) {
    if constexpr (F == Type::I8) widen<F>(x ^ 0x80808080u, lo, hi);
    else
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(x));
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
    static constexpr uint32_t queries = scales + 2 * kTileKeys * 4, query_row = HeadDim * 2 + 16; // the pad spreads rows over banks
    static constexpr uint32_t stage = (queries + columns * query_row + 1023) / 1024 * 1024;
    static __host__ __device__ constexpr uint32_t merge(int merge_columns) { return kWorkers * merge_columns * row * 4; }
};

// What the producer tells the workers about a tile, and they the mergers about a segment's part.
struct TileNote {
    int key, head, row, count, flat, limit, flags, ordinal, first_cta, first_slot, slot, parts, first_team, pad[3];
};
constexpr int kNoteFirst = 1, kNoteFlush = 2, kNoteEnd = 4, kNoteFinal = 16, kNoteSplit = 32, kNoteQuit = 64;


template <class T, Type F, int HeadDim, int Tiles>
__global__ void __launch_bounds__(kAttentionThreads, 1)
    cached_attention(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, const AttentionArgs args) {
    using Shape = AttentionShape<HeadDim, Tiles>;
    constexpr int kColumns = Shape::columns, kSteps = HeadDim / 16, kProducer = kWorkers, kMerger = kProducer + kProducers;
    extern __shared__ uint8_t raw_smem[];
    __shared__ uint64_t full[kTeams][kMaxRing], empty[kMaxRing], merge_full[kMergeBuffers]; // full: of each team
    __shared__ TileNote notes[kMaxRing], merge_notes[kMergeBuffers];
    __shared__ Work sums[kAttentionWarps];
    __shared__ Start found;
    __shared__ int abort_flag;
    __shared__ int merged[kMergers]; // parts that each merger is done with, written by that one only
    const uint32_t ring = (ptx::smem_u32(raw_smem) + 1023u) & ~1023u;
    uint8_t *const ring_bytes = raw_smem + (ring - ptx::smem_u32(raw_smem));
    const int stages = args.stages, merge_floats = int(Shape::merge(args.merge_columns) / 4);
    float *const merge = reinterpret_cast<float *>(ring_bytes + stages * Shape::stage);
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;

    if (!threadIdx.x) {
        for (int s = 0; s < stages; ++s) {
            for (int team = 0; team < kTeams; ++team) ptx::mbar_init(ptx::smem_u32(&full[team][s]), 33); // the leading producer's, and a lane's scales each
            ptx::mbar_init(ptx::smem_u32(&empty[s]), kTeam);
        }
        for (int b = 0; b < kMergeBuffers; ++b) ptx::mbar_init(ptx::smem_u32(&merge_full[b]), kWorkers);
        abort_flag = 0;
        for (int m = 0; m < kMergers; ++m) merged[m] = 0;
        ptx::fence_barrier_init();
        ptx::prefetch_tensormap(&key_map);
        ptx::prefetch_tensormap(&value_map);
    }
    begin_pass(args);

    // Only the producers need to know where the CTA's share lies; for a long batch all threads find out.
    if (args.sequences > kScanAlone) {
        start_together<kColumns, kAttentionWarps>(args, kFewSegmentUnits, sums, &found);
    }
    // Every wait is bounded, and a warp whose wait gave up leaves as one; the others follow when theirs do.
    auto wait = [&](uint64_t &bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar), parity, &abort_flag))) return true;
        if (!lane) *args.status = 1;
        return false;
    };

    // Until every merger is done with that many parts. A sum of theirs would not do: the one with less to do (with none at all, at one column of 128)
    // runs ahead by as many parts as there are buffers, and would stand in for the other.
    auto wait_merged = [&](int parts) {
        auto least = [&] {
            int done = INT_MAX;
#pragma unroll
            for (int m = 0; m < kMergers; ++m) done = min(done, const_cast<volatile int *>(merged)[m]);
            return done;
        };
        bool reached = false;
        const long long start = clock64();
        while (!(reached = least() >= parts) && !*const_cast<volatile int *>(&abort_flag))
            if (clock64() - start > ptx::kWaitLimitCycles) abort_flag = 1;
        reached = __all_sync(0xffffffffu, reached);
        __threadfence_block();
        if (!reached && !lane) *args.status = 1;
        return reached;
    };

    // Tile i of the share goes to team i % kTeams and stage i % stages. A stage may serve the teams in turn, so each team has its own barriers: waiting
    // on a common one, a team could be two phases off. A team comes back to a stage after `period` of its tiles.
    const int period = stages % kTeams ? stages : stages / kTeams;

    if (warp >= kProducer && warp < kMerger) { // --------------------------------------------------- producers
        // Two warps walk the same list: one copies keys and queries and writes the notes, the other copies values and scales. A tensor copy costs its
        // issuer 50 to 100 cycles and a tile of 16-token pages takes sixteen of them, so one warp would be what the ring waits for.
        const bool leads = warp == kProducer;
        int stage = 0, issued = 0, team = 0;
        uint32_t phase = 0;
        const Start start = args.sequences > kScanAlone ? found : start_alone<kColumns>(args, kFewSegmentUnits);
        const int box = 1 << args.box_shift, boxes = kTileKeys >> args.box_shift;
        const uint32_t box_bytes = uint32_t(box) * 2 * HeadDim;
        bool open = true;
        if (leads && !lane) note_closed(args, nullptr, kColumns);
        const int parts = walk_share<kColumns>(args, start, [&](const SegmentPart &part) {
            const SequenceShape &s = part.s;
            const int low = part.low, high = part.high, head = part.head, columns = part.columns;
            if (leads && !lane && part.first_cta >= 0) note_closed(args, &part, kColumns);
            const int *pages = args.pages + size_t(part.sequence) * args.page_stride;
            // Lane i's page of a tile: its box i. Always a load, of the last page where there is none, so that nothing waits for it here.
            auto page_at = [&](int tile) {
                return load_index(pages + (max(0, min(tile * kTileKeys + (min(lane, boxes - 1) << args.box_shift), s.length - 1)) >> args.page_shift));
            };
            int next = page_at(low);
            for (int tile = low; tile < high; ++tile) {
                const int page = next;
                if (tile + 1 < high) next = page_at(tile + 1); // on its way while this tile's stage is waited for
                if (issued >= stages && !wait(empty[stage], phase ^ 1)) return open = false;
                const uint32_t to = ring + stage * Shape::stage, bar = ptx::smem_u32(&full[team][stage]);
                uint8_t *const bytes = ring_bytes + stage * Shape::stage;
                const int key = tile * kTileKeys, position = key + (lane << args.box_shift);
                const bool good = lane < boxes && position < s.length && unsigned(page) < unsigned(args.total_pages);
                const uint32_t held = __ballot_sync(0xffffffffu, good);
                const int row = (((page * args.kv_heads) + head) << args.page_shift) + (position & ((1 << args.page_shift) - 1));
                if (leads) {
                    // Each team's first tile of the part brings the query rows.
                    const bool first = tile - low < kTeams, flush = tile + kTeams >= high;
                    const T *query = nullptr;
                    uint32_t query_bytes = 0;
                    if (first) {
                        const int flat = part.query_tile * kColumns + lane;
                        query = static_cast<const T *>(args.queries) + size_t(s.row + flat / args.group) * args.query_stride +
                                (head * args.group + flat % args.group) * HeadDim;
                        if (args.aligned) query_bytes = uint32_t(columns) * HeadDim * 2;
                        else if (lane < columns)
                            for (int d = 0; d < HeadDim; ++d) {
                                uint16_t v;
                                asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(query + d) : "memory");
                                *reinterpret_cast<uint16_t *>(bytes + Shape::queries + lane * Shape::query_row + 2 * d) = v;
                            }
                        __syncwarp();
                    }
                    if (!lane) {
                        TileNote &n = notes[stage];
                        n.key = key;
                        n.flags = (first ? kNoteFirst : 0) | (flush ? kNoteFlush : 0) | (tile + 1 == high ? kNoteEnd : 0) |
                                  (part.final ? kNoteFinal : 0) | (part.split ? kNoteSplit : 0);
                        if (first || flush) { // what the workers read at a part's ends only
                            n.head = head, n.row = s.row, n.count = s.count, n.flat = part.query_tile * kColumns;
                            n.limit = args.prefix ? s.length - 1 : s.length - s.count;
                            n.ordinal = part.ordinal, n.first_cta = part.first_cta, n.first_slot = part.first_slot;
                            n.slot = part.slot;
                            n.parts = min(kTeams, high - low), n.first_team = (issued - (tile - low)) % kTeams;
                        }
                        ptx::mbar_arrive_expect_tx(bar, __popc(held) * box_bytes + query_bytes);
                    }
                    __syncwarp();
                    if (query_bytes && lane < columns) copy_run(to + Shape::queries + lane * Shape::query_row, query, HeadDim * 2, bar);
                } else {
                    // Scales: a lane copies four of the keys' and four of the values'. Positions on a page that the cache does not have read as NaN.
                    const int owner = (4 * lane) >> args.box_shift;
                    const int its_row = __shfl_sync(0xffffffffu, row, owner) + ((4 * lane) & (box - 1));
                    if (held >> owner & 1) {
                        const uint32_t scales = to + Shape::scales + 16 * lane;
                        copy_async16(scales, args.key_scales + its_row);
                        copy_async16(scales + kTileKeys * 4, args.value_scales + its_row);
                        ptx::copy_async_arrive(bar);
                    } else {
                        const float nan = __int_as_float(0x7fffffff);
                        *reinterpret_cast<float4 *>(bytes + Shape::scales + 16 * lane) = make_float4(nan, nan, nan, nan);
                        *reinterpret_cast<float4 *>(bytes + Shape::scales + kTileKeys * 4 + 16 * lane) = make_float4(nan, nan, nan, nan);
                        ptx::mbar_arrive(bar);
                    }
                }
                // One thread issues the boxes, from rows gathered beforehand.
                int from_row[kTileKeys / 16];
#pragma unroll
                for (int i = 0; i < kTileKeys / 16; ++i) from_row[i] = __shfl_sync(0xffffffffu, row, i);
                if (ptx::elect_one()) {
                    const CUtensorMap *map = leads ? &key_map : &value_map;
                    const uint32_t into = to + (leads ? 0u : Shape::values), box_size = uint32_t(box) * HeadDim;
#pragma unroll
                    for (int i = 0; i < kTileKeys / 16; ++i)
                        if (held >> i & 1) ptx::tma_load_2d(into + i * box_size, map, bar, 0, from_row[i]);
                }
                __syncwarp();
                ++issued;
                if (++stage == stages) stage = 0, phase ^= 1;
                if (++team == kTeams) team = 0;
            }
            return true;
        });
        for (int i = 0; i < kTeams && open; ++i) { // an empty stage ends each team
            if (issued >= stages && !wait(empty[stage], phase ^ 1)) break;
            if (leads && !lane) notes[stage].flags = kNoteQuit;
            if (!leads || !lane) ptx::mbar_arrive(ptx::smem_u32(&full[team][stage]));
            ++issued;
            if (++stage == stages) stage = 0, phase ^= 1;
            if (++team == kTeams) team = 0;
        }
        if (!parts && leads && !lane) { // a share that holds no tile's first unit
            merge_notes[0].flags = kNoteQuit;
            for (int w = 0; w < kWorkers; ++w) ptx::mbar_arrive(ptx::smem_u32(&merge_full[0]));
        }
        // No copy may be in flight when the CTA leaves, whatever the workers did.
        int ignored = 0;
        for (int i = max(0, issued - stages); i < issued; ++i) ptx::mbar_wait(ptx::smem_u32(&full[i % kTeams][i % stages]), uint32_t((i / kTeams) / period) & 1, &ignored);
        if (args.follows) pdl_wait_upstream();
        return;
    }

    if (warp >= kMerger) { // ---------------------------------------------------------------------- mergers
        for (int ordinal = 0;; ++ordinal) {
            const int buffer = ordinal % args.merge_buffers;
            if (!wait(merge_full[buffer], uint32_t(ordinal / args.merge_buffers) & 1)) return;
            const TileNote &note = merge_notes[buffer];
            if (note.flags & kNoteQuit) return;
            const float *shares = merge + buffer * merge_floats;
            const int columns = min(kColumns, note.count * args.group - note.flat), flags = note.flags;
            const int count = kTeam * note.parts; // shares
            for (int item = int(threadIdx.x) - 32 * kMerger; item < columns * (HeadDim / 4); item += 32 * kMergers) {
                const int column = item / (HeadDim / 4), d = 4 * (item % (HeadDim / 4));
                float highest = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWorkers; ++w)
                    if (w < count) highest = fmaxf(highest, shares[(w * args.merge_columns + column) * Shape::row + HeadDim]);
                const float reference = highest == -INFINITY ? 0.f : highest;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                float l = 0.f;
#pragma unroll
                for (int w = 0; w < kWorkers; ++w) {
                    if (w >= count) break;
                    const float *from = shares + (w * args.merge_columns + column) * Shape::row;
                    const float f = exp2_approx(from[HeadDim] - reference);
                    const float4 x = *reinterpret_cast<const float4 *>(from + d);
                    v.x += f * x.x, v.y += f * x.y, v.z += f * x.z, v.w += f * x.w;
                    l += f * from[HeadDim + 1];
                }
                const int flat = note.flat + column, head = note.head * args.group + flat % args.group;
                const size_t at_row = size_t(note.row + flat / args.group), index = at_row * args.heads + head;
                float *kept = flags & kNoteSplit ? args.partials + (size_t(blockIdx.x * 2 + note.slot) * args.part_columns + column) * Shape::row
                              : args.complete    ? args.complete + index * Shape::row
                                                 : nullptr;
                if (kept) {
                    *reinterpret_cast<float4 *>(kept + d) = v;
                    if (!d) kept[HeadDim] = highest, kept[HeadDim + 1] = l;
                } else {
                    store_row4<T>(args, static_cast<T *>(args.output) + at_row * args.output_stride + head * HeadDim + d, v,
                                           l == 0.f ? 0.f : args.output_scale / l);
                }
                if (!d && args.table) {
                    if (!(flags & kNoteSplit)) args.table[index] = make_int4(0, 0, 0, 0);
                    else if (note.first_cta >= 0) args.table[index] = make_int4(note.first_cta, int(blockIdx.x) - note.first_cta + 1, note.first_slot, column);
                }
            }
            __syncwarp();
            if (!lane) {
                __threadfence_block();
                const_cast<volatile int *>(merged)[warp - kMerger] = ordinal + 1;
            }
            if (flags & kNoteFinal) return;
        }
    }

    // --------------------------------------------------------------------------------------------- workers
    const int g = lane >> 2, t = lane & 3, team = warp / kTeam, row = 32 * (warp % kTeam);
    uint32_t q[Tiles][kSteps][2];
    float out[Tiles][kSteps][4], most[Tiles][2], sum[Tiles][2], factor[Tiles][2];
    int limit[Tiles][2], least = 0;
    int stage = team, seen_stages = 0;
    uint32_t phase = 0;
    for (;;) {
        if (!wait(full[team][stage], phase)) return;
        const TileNote &note = notes[stage];
        const uint32_t at = ring + stage * Shape::stage;
        const uint8_t *bytes = ring_bytes + stage * Shape::stage;
        const float *scales = reinterpret_cast<const float *>(bytes + Shape::scales);
        const int flags = note.flags;
        if (flags & kNoteQuit) return;
        if (flags & kNoteFirst) {
            const int columns = note.count * args.group - note.flat;
            least = INT_MAX;
#pragma unroll
            for (int n = 0; n < Tiles; ++n) {
                // This lane's share of query row 8n + g: columns [HeadDim / 4 * t, HeadDim / 4 * (t + 1)).
                constexpr int kShare = HeadDim / 4;
                const bool live = 8 * n + g < columns;
                alignas(16) T share[kShare];
#pragma unroll
                for (int c = 0; c < kShare / 8; ++c) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(bytes + Shape::queries + (8 * n + g) * Shape::query_row + (kShare * t + 8 * c) * 2);
                    *reinterpret_cast<uint4 *>(share + 8 * c) = live ? v : make_uint4(0, 0, 0, 0);
                }
                const uint32_t *words = reinterpret_cast<const uint32_t *>(share);
                int exponent = 0; // BF16 rows are divided by the power of two of their largest element; FP16 ones are in range as they are
                if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    unsigned largest = 0;
#pragma unroll
                    for (int c = 0; c < kShare / 2; ++c) largest = max(largest, max(words[c] << 16 & 0x7fffffffu, words[c] & 0x7fff0000u));
                    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                    exponent = largest && largest < 0x7f800000u ? max(int(largest >> 23), 1) - 127 : 0;
                }
                const float down = __int_as_float(exponent < 127 ? (127 - exponent) << 23 : 0x00400000); // 2^-exponent
#pragma unroll
                for (int k = 0; k < kSteps; ++k)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t w = words[2 * k + c];
                        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                            const __half2 v = __floats2half2_rn(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down);
                            q[n][k][c] = *reinterpret_cast<const uint32_t *>(&v);
                        } else {
                            q[n][k][c] = w;
                        }
                    }
                // The scores of this lane belong to columns 2t and 2t + 1, whose rows lanes 8t and 8t + 4 hold.
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int of = __shfl_sync(0xffffffffu, exponent, 8 * t + 4 * c), seen = 8 * n + 2 * t + c;
                    factor[n][c] = args.score_scale * __int_as_float((127 + of) << 23);
                    limit[n][c] = seen >= columns ? -1 : args.prefix || note.count == 1 ? note.limit : note.limit + (note.flat + seen) / args.group;
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

        // This warp's 32 keys, two blocks of 16: all of its bytes into registers, so that the stage can be filled again while the warp computes
        // (the ring, not the arithmetic, is what bounds a long context). Not with 16 query rows, whose state needs the registers.
        constexpr bool kEarly = Tiles == 1;
        uint32_t keys[2][2][HeadDim / 16], values[2][4][HeadDim / 32];
        float key_scale[2][2], value_scale[2][2], shift[2][2];
        auto load_keys = [&](int m) {
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int c = 0; c < HeadDim / 64; ++c)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(keys[m][r][4 * c]), "=r"(keys[m][r][4 * c + 1]), "=r"(keys[m][r][4 * c + 2]), "=r"(keys[m][r][4 * c + 3])
                                 : "r"(at + piece<HeadDim>(row + 16 * m + g + 8 * r, HeadDim / 64 * t + c)));
        };
        // Values of keys 2t, 2t + 1, 2t + 8, 2t + 9 of the block: this thread's 16 (8) columns.
        auto load_values = [&](int m) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = row + 16 * m + 2 * t + (r & 1) + 8 * (r >> 1);
                if constexpr (HeadDim == 128)
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(values[m][r][0]), "=r"(values[m][r][1]), "=r"(values[m][r][2]), "=r"(values[m][r][3])
                                 : "r"(at + Shape::values + piece<HeadDim>(key, g)));
                else
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                                 : "=r"(values[m][r][0]), "=r"(values[m][r][1])
                                 : "r"(at + Shape::values + piece<HeadDim>(key, g >> 1) + 8 * (g & 1)));
            }
        };
        const int first_key = note.key;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (kEarly) load_keys(m);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                key_scale[m][r] = scales[row + 16 * m + g + 8 * r];
                value_scale[m][r] = scales[kTileKeys + row + 16 * m + g + 8 * r];
            }
        }
        if (kEarly) {
            load_values(0);
            load_values(1);
            if (!(flags & kNoteFlush)) { // a flush still needs the note
                __syncwarp();
                if (!lane) ptx::mbar_arrive(ptx::smem_u32(&empty[stage]));
            }
        }
        float scores[Tiles][2][4] = {};
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (!kEarly) load_keys(m);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                uint32_t a[4];
                widen_key<F>(keys[m][0][k], a[0], a[2]);
                widen_key<F>(keys[m][1][k], a[1], a[3]);
#pragma unroll
                for (int n = 0; n < Tiles; ++n) mma_f16(scores[n][m], a[0], a[1], a[2], a[3], q[n][k][0], q[n][k][1]);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) shift[m][r] = fmaxf(log2_approx(fabsf(value_scale[m][r])), kLeastScale);
        }
        const int position = first_key + row + g;
        const bool masked = first_key + kTileKeys - 1 > least;
        uint32_t weights[Tiles][2][2];
#pragma unroll
        for (int n = 0; n < Tiles; ++n) {
            float highest[2] = {-INFINITY, -INFINITY};
            unsigned hidden = 0;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float &x = scores[n][m][2 * r + c];
                        x *= key_scale[m][r] * factor[n][c];
                        if (masked && position + 16 * m + 8 * r > limit[n][c]) {
                            hidden |= 1u << (4 * m + 2 * r + c);
                            x = -INFINITY;
                        }
                        highest[c] = fmaxf(highest[c], hidden & (1u << (4 * m + 2 * r + c)) ? -INFINITY : x + shift[m][r]);
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
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float w[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float p = exp2_approx(scores[n][m][2 * r + c] - (most[n][c] == -INFINITY ? 0.f : most[n][c]));
                        sum[n][c] += p;
                        w[c] = hidden & (1u << (4 * m + 2 * r + c)) ? 0.f : p * value_scale[m][r]; // a hidden row's scale may be anything
                    }
                    const __half2 both = __floats2half2_rn(w[0], w[1]);
                    weights[n][m][r] = transpose8x8(*reinterpret_cast<const uint32_t *>(&both));
                }
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (!kEarly) load_values(m);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                const uint32_t order = k & 1 ? 0x7362u : 0x5140u; // bytes 2 (k & 1) and the next of two keys, side by side
                uint32_t a[4];
                widen<F>(biased<F>(__byte_perm(values[m][0][k >> 1], values[m][1][k >> 1], order)), a[0], a[1]);
                widen<F>(biased<F>(__byte_perm(values[m][2][k >> 1], values[m][3][k >> 1], order)), a[2], a[3]);
#pragma unroll
                for (int n = 0; n < Tiles; ++n) mma_f16(out[n][k], a[0], a[1], a[2], a[3], weights[n][m][0], weights[n][m][1]);
            }
        }

        if (flags & kNoteFlush) { // this warp's share of the segment's part; the mergers add the shares up
            const int ordinal = note.ordinal, buffer = ordinal % args.merge_buffers;
            const int columns = min(kColumns, note.count * args.group - note.flat);
            // Counts and not a barrier's phase: a group has no tile in some parts, and could be two phases off.
            if (ordinal >= args.merge_buffers && !wait_merged(ordinal - args.merge_buffers + 1)) return;
            const int share = (team - note.first_team + kTeams) % kTeams * kTeam + warp % kTeam;
            float *const shares = merge + buffer * merge_floats + share * args.merge_columns * Shape::row;
#pragma unroll
            for (int n = 0; n < Tiles; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float l = sum[n][c];
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                    const int column = 8 * n + 2 * t + c;
                    if (column >= columns) continue;
                    float *to = shares + column * Shape::row;
#pragma unroll
                    for (int k = 0; k < kSteps; k += 2)
                        *reinterpret_cast<float4 *>(to + g * kSteps * 2 + 2 * k) =
                            make_float4(out[n][k][c], out[n][k][2 + c], out[n][k + 1][c], out[n][k + 1][2 + c]);
                    if (!g) to[HeadDim] = most[n][c], to[HeadDim + 1] = l;
                }
            if ((flags & kNoteEnd) && !(warp % kTeam) && !lane) merge_notes[buffer] = note;
            __syncwarp();
            if (!lane) { // the team of the last tile also arrives for those that have none of this part
                ptx::mbar_arrive(ptx::smem_u32(&merge_full[buffer]));
                if (flags & kNoteEnd)
                    for (int i = note.parts; i < kTeams; ++i) ptx::mbar_arrive(ptx::smem_u32(&merge_full[buffer]));
            }
        }
        if (!kEarly || (flags & kNoteFlush)) {
            __syncwarp();
            if (!lane) ptx::mbar_arrive(ptx::smem_u32(&empty[stage]));
        }
        stage += kTeams;
        if (stage >= stages) stage -= stages;
        if (++seen_stages == period) seen_stages = 0, phase ^= 1;
    }
}

// Last launch: a warp per query row and head adds up what was left in parts, in the order of the CTAs.
constexpr int kCombineThreads = 128;
struct CombineSource {
    const float *partials, *complete;
    const ClosedSegment *closed;
    const int4 *table;
    int ctas, columns;
};
struct CombineArgs {
    CombineSource source[2];
    int rows, heads, group, output_stride;
    const int *row_count; // last of the query offsets, or null
    int *pass_word;
    void *output;
    float output_scale;
};
template <int HeadDim> struct RowSum {
    static constexpr int kRow = HeadDim + kPartialExtra, kShare = HeadDim / 32;
    float highest = -INFINITY, l = 0.f, v[kShare] = {};

    static __device__ __forceinline__ void read(const float *from, float (&x)[kShare]) {
        if constexpr (kShare == 4) {
            const float4 w = *reinterpret_cast<const float4 *>(from);
            x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
        } else {
            const float2 w = *reinterpret_cast<const float2 *>(from);
            x[0] = w.x, x[1] = w.y;
        }
    }
    // 32 parts at a time: a lane reads the maximum and the sum of one, and the first parts' rows are on their way meanwhile.
    template <class PartOf> __device__ __forceinline__ void add(int parts, PartOf &&part_of) {
        constexpr int kAhead = 8;
        const int lane = threadIdx.x & 31;
        for (int first = 0; first < parts; first += 32) {
            const int count = min(32, parts - first);
            float most = -INFINITY, sum = 0.f, ahead[kAhead][kShare];
            if (lane < count) {
                const float2 stats = *reinterpret_cast<const float2 *>(part_of(first + lane) + HeadDim);
                most = stats.x, sum = stats.y;
            }
#pragma unroll
            for (int part = 0; part < kAhead; ++part)
                if (part < count) read(part_of(first + part) + kShare * lane, ahead[part]);
            float raised = most;
#pragma unroll
            for (int d = 16; d; d >>= 1) raised = fmaxf(raised, __shfl_xor_sync(0xffffffffu, raised, d));
            raised = fmaxf(raised, highest);
            const float reference = raised == -INFINITY ? 0.f : raised, shrink = exp2_approx(highest - reference);
            const float factor = exp2_approx(most - reference);
            sum *= factor;
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            l = l * shrink + sum; // the same in all lanes
#pragma unroll
            for (int c = 0; c < kShare; ++c) v[c] *= shrink;
            highest = raised;
#pragma unroll
            for (int part = 0; part < kAhead; ++part) {
                if (part >= count) break;
                const float f = __shfl_sync(0xffffffffu, factor, part);
#pragma unroll
                for (int c = 0; c < kShare; ++c) v[c] += ahead[part][c] * f;
            }
#pragma unroll 8
            for (int part = kAhead; part < count; ++part) {
                const float f = __shfl_sync(0xffffffffu, factor, part);
                float x[kShare];
                read(part_of(first + part) + kShare * lane, x);
#pragma unroll
                for (int c = 0; c < kShare; ++c) v[c] += x[c] * f;
            }
        }
    }
    template <class T> __device__ __forceinline__ void store(const CombineArgs &a, int row, int head) const {
        const float factor = l == 0.f ? 0.f : a.output_scale / l;
        T *to = static_cast<T *>(a.output) + size_t(row) * a.output_stride + size_t(head) * HeadDim + kShare * int(threadIdx.x & 31);
#pragma unroll
        for (int c = 0; c < kShare; ++c) to[c] = T(v[c] * factor);
    }
};
// Without a prefix: only split segments are left to do, at most one for each CTA of the pass. A warp takes a few of a segment's rows.
template <class T, int HeadDim> __global__ void __launch_bounds__(kCombineThreads) combine_attention(const CombineArgs args) {
    pdl_launch_dependents();
    pdl_wait_upstream();
    const CombineSource &s = args.source[0];
    const int *entry = reinterpret_cast<const int *>(s.closed + blockIdx.x);
    int4 where, whose;
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(where.x), "=r"(where.y), "=r"(where.z), "=r"(where.w) : "l"(entry) : "memory");
    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(whose.x), "=r"(whose.y), "=r"(whose.z), "=r"(whose.w) : "l"(entry + 4) : "memory");
    // Offsets that fall can make the counts run over: what is read stays inside the workspace.
    if (where.y <= 0 || where.x < 0 || where.y > s.ctas - where.x) return;
    for (int column = int(blockIdx.y) * (kCombineThreads / 32) + int(threadIdx.x >> 5); column < whose.z; column += int(gridDim.y) * (kCombineThreads / 32)) {
        RowSum<HeadDim> sum;
        sum.add(where.y, [&](int part) {
            return s.partials + (size_t((where.x + part) * 2 + (part ? 0 : where.z)) * s.columns + column) * RowSum<HeadDim>::kRow;
        });
        const int flat = whose.x + column, token = flat / args.group;
        sum.template store<T>(args, where.w + token, whose.y * args.group + flat - token * args.group);
    }
}
// With a prefix: every row has a result of both passes, in one part or several.
template <class T, int HeadDim> __global__ void __launch_bounds__(kCombineThreads) combine_prefixed(const CombineArgs args) {
    pdl_launch_dependents();
    pdl_wait_upstream();
    if (!blockIdx.x && !threadIdx.x) *args.pass_word = 0; // both passes are over
    const long long index = (long long)blockIdx.x * (kCombineThreads / 32) + (threadIdx.x >> 5);
    const int rows = args.row_count ? min(args.rows, load_index(args.row_count)) : args.rows;
    if (index >= (long long)rows * args.heads) return;
    int4 entries[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(entries[i].x), "=r"(entries[i].y), "=r"(entries[i].z), "=r"(entries[i].w)
                     : "l"(args.source[i].table + index)
                     : "memory");
    RowSum<HeadDim> sum;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const CombineSource &s = args.source[i];
        const int4 entry = entries[i];
        const bool whole = entry.y <= 0;
        // Rows that no sequence covers have no entry: whatever stands there stays inside the workspace.
        if (!whole && (entry.x < 0 || entry.y > s.ctas - entry.x || unsigned(entry.z) > 1u || unsigned(entry.w) >= unsigned(s.columns))) continue;
        sum.add(whole ? 1 : entry.y, [&](int part) {
            return whole ? s.complete + size_t(index) * RowSum<HeadDim>::kRow
                         : s.partials + (size_t((entry.x + part) * 2 + (part ? 0 : entry.z)) * s.columns + entry.w) * RowSum<HeadDim>::kRow;
        });
    }
    sum.template store<T>(args, int(index / args.heads), int(index % args.heads));
}
} // namespace tts::b200
