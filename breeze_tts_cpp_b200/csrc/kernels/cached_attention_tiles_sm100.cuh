// Attention of many query rows over the quantized, paged cache: chunks of prompts, and a prefix that a whole batch shares.
//
// Mathematics: as for few query rows (cached_attention_sm100.cuh). Scores and outputs are fp16 products with fp32 sums on the tensor cores, and
// bytes enter them exactly. Rounded are BF16 queries more than 2^17 below their row's largest, to within 2^-25 of its power of two, and p_j vs_j, to
// fp16, against a running reference that keeps it at most 256. The reference moves only when a tile's maximum passes it by 2^8, so that the
// accumulated output is rescaled hardly ever.
//
// Layout. A segment is 128 query rows of one cached head (tokens times the group's heads; of a prefix: of all sequences), a tile 128 keys. Per tile
// a CTA does S = Q K^T and O += P V as tcgen05.mma, with S, P and O in tensor memory; P overwrites S, two halves to a column. Two teams of eight
// softmax warps, 16 rows a warp, take one half of a tile's keys each, and each team has a softmax state, an output and an issuing warp of its own;
// they meet once per segment. A team has the scores of two tiles, so that the products of one run while it works on the other. Eight warps turn
// bytes into fp16 operands: keys as they are, values transposed, so that both are K-major with the 128-byte swizzle. Tables of a tile's scales go
// to the softmax warps through shared memory.
//
// Bound. A 128 x 128 x 128 tile costs the tensor pipe about 1300 cycles, its exponentials the special-function units 1024, and its conversions and
// softmax 2500 issue slots of every scheduler, so all of them have to overlap; a tile takes about 4400 cycles in all, most of that the chain from
// bytes to products to weights to products with its barriers: without any arithmetic at all it would take 2700. Sixteen softmax warps rather than
// eight, whose tiles of 16 rows are half as long, take three chunks of 700 tokens (up to 2500 long, 16 heads over 8, e4m3) from 46.9 to 42.3 us.
// With a power of two for each BF16 row that is 42.2 us, 180 TFLOP/s of what the mask leaves. The first tile of a CTA takes 20000 cycles to come
// out, the schedule, the queries and the code itself being fetched one behind the other.
#pragma once
#include "kernels/cached_attention_sm100.cuh"

namespace tts::b200 {
constexpr int kManyRows = 128;
// Filling and draining the pipeline, the meeting of the teams and the store, next to a tile's kTileUnits (three chunks of 700: 6 units 45.8 us, 12 42.4,
// 20 44.1; 512 query rows 4000 long 28.9, 26.9, 28.6).
constexpr int kManySegmentUnits = 12;
constexpr int kSoftmaxWarps = 16, kConverters = 8, kManyWarps = kSoftmaxWarps + kConverters + 3, kManyThreads = 32 * kManyWarps; // 72 registers a thread
constexpr int kPartsAhead = 4;
constexpr float kReferenceSlack = 8.f; // powers of two that a weight may exceed one by

template <int HeadDim> struct ManyShape {
    static constexpr uint32_t operand = kManyRows * HeadDim * 2; // Q, one K, one V
    static constexpr uint32_t raw = kTileKeys * HeadDim + 2 * kTileKeys * 4;
    static constexpr int slots = HeadDim == 128 ? 3 : 6;
    static constexpr uint32_t keys = operand, values = 3 * operand, ring = 5 * operand;
    static constexpr size_t smem = 1024 + ring + slots * size_t(raw);
};

namespace many {
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24); }
__device__ __forceinline__ void mma_smem(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
                 "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(ptx::kDescHiK128)
                 : "memory");
}
__device__ __forceinline__ void mma_tmem(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 db, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(ptx::kDescHiK128)
                 : "memory");
}
// The fragment of tmem_load_rows16<32> back to where it came from.
__device__ __forceinline__ void tmem_store_scores16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// 16 lanes x 16 columns from a matrix fragment: lane l holds rows l / 4 (r[2j]) and l / 4 + 8 (r[2j + 1]), column 4j + l % 4.
__device__ __forceinline__ void tmem_store_rows16(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return ptx::pack2(__uint_as_float(lo), __uint_as_float(hi)); }
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16-byte chunk `chunk` of row `row` in a K-major operand panel (rows of 64 halves, 128-byte swizzle).
__device__ __forceinline__ uint32_t panel_at(int row, int chunk) { return uint32_t(row * 128 + ((chunk ^ (row & 7)) << 4)); }
template <class T> __device__ __forceinline__ void store_row16(const AttentionArgs &a, T *to, const float (&v)[16], float factor) {
    union {
        float words[8];
        uint4 fours[2];
        T e[16];
    } out;
#pragma unroll
    for (int i = 0; i < 16; ++i) out.e[i] = T(v[i] * factor);
    if (a.sectors) {
        ptx::store_sector(to, out.words);
    } else if (a.aligned) {
        reinterpret_cast<uint4 *>(to)[0] = out.fours[0];
        reinterpret_cast<uint4 *>(to)[1] = out.fours[1];
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) to[i] = out.e[i];
    }
}
} // namespace many

template <class T, Type F, int HeadDim>
__global__ void __launch_bounds__(kManyThreads, 1) cached_attention_many(const AttentionArgs args) {
    using namespace many;
    using Shape = ManyShape<HeadDim>;
    constexpr int kRows = kManyRows, kSlots = Shape::slots, kConverter = kSoftmaxWarps, kProducer = kConverter + kConverters, kIssuer = kProducer + 1; // an issuer per team
    constexpr uint32_t kOut = 2 * kTileKeys; // tensor memory: two teams' scores, then their outputs
    extern __shared__ uint8_t raw_smem[];
    // Tile i of the share has buffers and barriers i % 2, and these their use i / 2. Of each team: scored: S is done (of both: the keys' buffer is
    // free); softmaxed: P is ready; weighted: O has it (of both: the values' buffer is free). keys/values: operands are ready. tables_ready
    // has a use for every fourth tile: its tables are not written again before the teams are done with them.
    __shared__ uint64_t raw_full[kSlots], raw_free[kSlots], keys_ready[2], values_ready[2], scored[2][2], softmaxed[2][2], weighted[2][2], tables_ready[4];
    __shared__ uint64_t queries_ready, meet, outputs_free, drained[2]; // once per segment part, the last once
    __shared__ __align__(16) float table_key[4][kTileKeys], table_shift[4][kTileKeys], table_value[4][kTileKeys]; // of tile i: i % 4
    __shared__ float2 stats[2][kRows];
    // What a BF16 row's scores are multiplied by, by the part's ordinal: three parts on, the softmax warps have begun the first one's tiles.
    __shared__ float row_scale[4][kRows];
    constexpr bool kScaledRows = std::is_same<T, __nv_bfloat16>::value;
    __shared__ Work sums[kManyWarps];
    __shared__ Start found;
    __shared__ SegmentPart parts[kPartsAhead];
    __shared__ uint64_t part_full[kPartsAhead], part_free[kPartsAhead];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const uint32_t base = (ptx::smem_u32(raw_smem) + 1023u) & ~1023u;
    uint8_t *const base_bytes = raw_smem + (base - ptx::smem_u32(raw_smem));
    const int warp = ptx::warp_index(), lane = threadIdx.x & 31;

    if (!threadIdx.x) {
        for (int s = 0; s < kSlots; ++s) {
            ptx::mbar_init(ptx::smem_u32(&raw_full[s]), 33); // the copies, and a lane's scales each
            ptx::mbar_init(ptx::smem_u32(&raw_free[s]), kConverters);
        }
        for (int t = 0; t < 2; ++t) {
            ptx::mbar_init(ptx::smem_u32(&keys_ready[t]), kConverters);
            ptx::mbar_init(ptx::smem_u32(&values_ready[t]), kConverters);
            for (int h = 0; h < 2; ++h) {
                ptx::mbar_init(ptx::smem_u32(&scored[t][h]), 1);
                ptx::mbar_init(ptx::smem_u32(&softmaxed[t][h]), kSoftmaxWarps / 2);
                ptx::mbar_init(ptx::smem_u32(&weighted[t][h]), 1);
            }
            ptx::mbar_init(ptx::smem_u32(&drained[t]), 1);
            ptx::mbar_init(ptx::smem_u32(&tables_ready[2 * t]), kConverters);
            ptx::mbar_init(ptx::smem_u32(&tables_ready[2 * t + 1]), kConverters);
        }
        ptx::mbar_init(ptx::smem_u32(&queries_ready), kConverters);
        ptx::mbar_init(ptx::smem_u32(&outputs_free), kSoftmaxWarps);
        ptx::mbar_init(ptx::smem_u32(&meet), kSoftmaxWarps);
        for (int p = 0; p < kPartsAhead; ++p) {
            ptx::mbar_init(ptx::smem_u32(&part_full[p]), 1);
            ptx::mbar_init(ptx::smem_u32(&part_free[p]), kSoftmaxWarps + kConverters + 2);
        }
        abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == kIssuer) ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
    ptx::tcgen05_fence_before();
    begin_pass(args);
    ptx::tcgen05_fence_after();
    const uint32_t tmem = ptx::warp_uniform(tmem_slot);
    if (args.sequences > kScanAlone) start_together<kRows, kManyWarps>(args, kManySegmentUnits, sums, &found);

    // Every wait is bounded. A warp whose wait gave up goes to the end, where all meet; the others follow when theirs do.
    auto wait = [&](uint64_t &bar, int use) {
        if (__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bar), uint32_t(use) & 1, &abort_flag))) return true;
        if (!lane) *args.status = 1;
        return false;
    };
    auto arrive = [&](uint64_t &bar) {
        __syncwarp();
        if (!lane) ptx::mbar_arrive(ptx::smem_u32(&bar));
    };
    // The producer walks the share and hands its parts to the others. Calls `each` for every part until it returns false.
    auto for_parts = [&](auto &&each) {
        for (int ordinal = 0;; ++ordinal) {
            const int at = ordinal % kPartsAhead;
            if (!wait(part_full[at], ordinal / kPartsAhead)) return;
            const SegmentPart &part = parts[at];
            if (part.low == part.high || !each(part)) return;
            arrive(part_free[at]);
        }
    };
    int first_tile = 0; // of the part, in the share

    if (warp == kProducer) { // ------------------------------------------------------------------ bytes and scales
        const int box = 1 << args.box_shift, boxes = kTileKeys >> args.box_shift;
        int slot = 0, item = 0, reuse = -1; // reuse: the slot's use before this one
        auto publish = [&](const SegmentPart &part) {
            const int at = part.ordinal % kPartsAhead;
            if (part.ordinal >= kPartsAhead && !wait(part_free[at], part.ordinal / kPartsAhead - 1)) return false;
            if (!lane) {
                parts[at] = part;
                ptx::mbar_arrive(ptx::smem_u32(&part_full[at]));
            }
            __syncwarp();
            return true;
        };
        const Start start = args.sequences > kScanAlone ? found : start_alone<kRows>(args, kManySegmentUnits);
        bool open = true;
        SegmentPart nothing{};
        if (!lane) note_closed(args, nullptr, kRows);
        nothing.ordinal = walk_share<kRows>(args, start, [&](const SegmentPart &part) {
            if (!publish(part)) return open = false;
            if (!lane && part.first_cta >= 0) note_closed(args, &part, kRows);
            const int *pages = args.pages + size_t(part.sequence) * args.page_stride;
            // Lane i's box of a tile: whether the cache has its page, and its first row there.
            auto find = [&](int tile, bool &good, int &row) {
                const int position = tile * kTileKeys + (lane << args.box_shift);
                const bool wanted = lane < boxes && position < part.s.length;
                const int page = wanted ? load_index(pages + (position >> args.page_shift)) : -1;
                good = unsigned(page) < unsigned(args.total_pages);
                row = (((page * args.kv_heads) + part.head) << args.page_shift) + (position & ((1 << args.page_shift) - 1));
            };
            auto fetch = [&](bool values, bool good, int row) {
                if (reuse >= 0 && !wait(raw_free[slot], reuse)) return open = false;
                const uint32_t to = base + Shape::ring + slot * Shape::raw, bar = ptx::smem_u32(&raw_full[slot]), held = __ballot_sync(0xffffffffu, good);
                if (!lane) ptx::mbar_arrive_expect_tx(bar, __popc(held) * box * HeadDim);
                __syncwarp();
                if (good)
                    copy_run(to + uint32_t(lane << args.box_shift) * HeadDim,
                             static_cast<const uint8_t *>(values ? args.cached_values : args.cached_keys) + size_t(row) * HeadDim, uint32_t(box) * HeadDim, bar);
                // With the keys, a lane copies the scales of four keys and four values. Positions on a page that the cache does not have read as NaN.
                const int owner = (4 * lane) >> args.box_shift, its_row = __shfl_sync(0xffffffffu, row, owner) + ((4 * lane) & (box - 1));
                const uint32_t scales = to + kTileKeys * HeadDim + 16 * lane;
                if (values) {
                    ptx::mbar_arrive(bar);
                } else if (held >> owner & 1) {
                    copy_async16(scales, args.key_scales + its_row);
                    copy_async16(scales + kTileKeys * 4, args.value_scales + its_row);
                    ptx::copy_async_arrive(bar);
                } else {
                    st_shared16(scales, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu);
                    st_shared16(scales + kTileKeys * 4, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu);
                    ptx::mbar_arrive(bar);
                }
                ++item;
                if (++slot == kSlots) slot = 0, ++reuse;
                return true;
            };
            // A tile's keys come before the values of the tile in front of it: these wait for that team's product, those need not.
            bool good, next_good = false;
            int row, next_row = 0;
            find(part.low, good, row);
            if (!fetch(false, good, row)) return false;
            for (int tile = part.low; tile < part.high; ++tile) {
                if (tile + 1 < part.high) {
                    find(tile + 1, next_good, next_row);
                    if (!fetch(false, next_good, next_row)) return false;
                }
                if (!fetch(true, good, row)) return false;
                good = next_good, row = next_row;
            }
            return true;
        });
        if (open) publish(nothing);
        // No copy may be in flight when the CTA leaves, whatever the others did.
        int ignored = 0;
        for (int i = max(0, item - kSlots); i < item; ++i) ptx::mbar_wait(ptx::smem_u32(&raw_full[i % kSlots]), uint32_t(i / kSlots) & 1, &ignored);
    } else if (warp == kIssuer || warp == kIssuer + 1) { // -------------------------------------------------------------- products
        constexpr uint32_t kScoreIdesc = idesc_f16(kRows, kTileKeys / 2), kOutIdesc = idesc_f16(kRows, HeadDim);
        const int team = warp - kIssuer;
        constexpr int kHalf = kTileKeys / 2;
        auto score = [&](int i) { // S of the team's half of a tile, where the weights of the tile before the last stood
            const int buffer = i & 1;
            if (!wait(keys_ready[buffer], i >> 1) || (i >= 2 && !wait(weighted[team][buffer], (i >> 1) - 1))) return false;
            ptx::tcgen05_fence_after();
            if (ptx::elect_one()) {
                const uint32_t q = ptx::smem_desc_lo_k128(base), k = ptx::smem_desc_lo_k128(base + Shape::keys + buffer * Shape::operand + team * (kHalf * 128));
#pragma unroll
                for (int s = 0; s < HeadDim / 16; ++s) {
                    const uint32_t at = uint32_t(s >> 2) * (kRows * 128 >> 4) + uint32_t(s & 3) * 2;
                    mma_smem(tmem + team * kTileKeys + buffer * kHalf, q + at, k + at, kScoreIdesc, s > 0);
                }
                ptx::tcgen05_commit(ptx::smem_u32(&scored[team][buffer]));
            }
            __syncwarp();
            return true;
        };
        for_parts([&](const SegmentPart &part) {
            const int first = first_tile, end = first + part.high - part.low;
            if (!wait(queries_ready, part.ordinal)) return false;
            if (!score(first) || (first + 1 < end && !score(first + 1))) return false;
            if (part.ordinal && !wait(outputs_free, part.ordinal - 1)) return false;
#pragma unroll 1
            for (int i = first; i < end; ++i) {
                const int buffer = i & 1;
                if (!wait(values_ready[buffer], i >> 1) || !wait(softmaxed[team][buffer], i >> 1)) return false;
                ptx::tcgen05_fence_after();
                if (ptx::elect_one()) {
                    const uint32_t v = ptx::smem_desc_lo_k128(base + Shape::values + buffer * Shape::operand + team * (HeadDim * 128));
#pragma unroll
                    for (int s = 0; s < kHalf / 16; ++s)
                        mma_tmem(tmem + kOut + team * HeadDim, tmem + team * kTileKeys + buffer * kHalf + 8 * s, v + uint32_t(s) * 2, kOutIdesc, s > 0 || i > first);
                    ptx::tcgen05_commit(ptx::smem_u32(&weighted[team][buffer]));
                }
                __syncwarp();
                if (i + 2 < end && !score(i + 2)) return false;
            }
            first_tile = end;
            return true;
        });
        // No product may be in flight when the tensor memory is given back, whatever the others did.
        if (ptx::elect_one()) ptx::tcgen05_commit(ptx::smem_u32(&drained[team]));
        __syncwarp();
        int ignored = 0;
        ptx::mbar_wait(ptx::smem_u32(&drained[team]), 0, &ignored);
    } else if (warp >= kConverter && warp < kProducer) { // ----------------------------------------------------------- bytes to operands
        const int mine = warp - kConverter, thread = 32 * mine + lane;
        int slot = 0, use = 0;
        auto next_slot = [&] {
            if (++slot == kSlots) slot = 0, ++use;
        };
        for_parts([&](const SegmentPart &part) {
            // Queries, once the products of the part before have read theirs. Rows past the segment are zero. A BF16 row is divided by the power of two
            // of its largest element, which brings it into fp16's range whatever the rows beside it hold.
            for (int i = max(0, first_tile - 2); i < first_tile; ++i)
                if (!wait(scored[0][i & 1], i >> 1) || !wait(scored[1][i & 1], i >> 1)) return false;
            constexpr int kChunks = HeadDim / 8, kTurns = kRows * kChunks / (32 * kConverters); // kChunks: threads to a row
            const int flat = part.query_tile * kRows, chunk = thread % kChunks, whole = flat / args.group, over = flat - whole * args.group;
            const auto place = [&](int i) { // where this thread's piece of turn i goes; rows of a turn are a multiple of eight apart
                return base + uint32_t(chunk >> 3) * (kRows * 128) + panel_at(thread / kChunks, chunk & 7) + uint32_t(i) * (32 * kConverters / kChunks * 128);
            };
            static_assert(32 * kConverters / kChunks % 8 == 0);
#pragma unroll 1
            for (int i = 0; i < kTurns; ++i) { // all rows in flight at once, as they are
                const int row = thread / kChunks + 32 * kConverters / kChunks * i;
                const int tokens = int((float(over + row) + .5f) * args.group_inverse); // exact up to kMostGroup: the half is far more than the product is off by
                const T *at = static_cast<const T *>(args.queries) + size_t(part.s.row + whole + tokens) * args.query_stride +
                              (part.head * args.group + over + row - tokens * args.group) * HeadDim + 8 * chunk;
                if (row >= part.columns) {
                    st_shared16(place(i), 0, 0, 0, 0);
                } else if (args.aligned) {
                    copy_async16(place(i), at);
                } else {
                    uint16_t v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) asm volatile("ld.global.b16 %0, [%1];" : "=h"(v[e]) : "l"(at + e) : "memory");
                    st_shared16(place(i), v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
                }
            }
            auto convert_keys = [&](int i) {
                const int buffer = i & 1, before = (i >> 1) - 1;
                if (!wait(raw_full[slot], use) || (before >= 0 && (!wait(scored[0][buffer], before) || !wait(scored[1][buffer], before)))) return false;
                {
                    const uint32_t from = base + Shape::ring + slot * Shape::raw, to = base + Shape::keys + buffer * Shape::operand;
                    constexpr int kPieces = HeadDim / 16, kTurns = kTileKeys * kPieces / (32 * kConverters); // kPieces: lanes to a key row
                    uint32_t w[kTurns][4];
#pragma unroll
                    for (int u = 0; u < kTurns; ++u) // row HeadDim bytes long, so thread t's pieces lie 16 t bytes in and one turn apart
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(w[u][0]), "=r"(w[u][1]), "=r"(w[u][2]), "=r"(w[u][3])
                                     : "r"(from + 16 * (thread + 32 * kConverters * u)));
                    const int c = thread % kPieces, row = thread / kPieces;
                    // The second panel's lanes store their chunks in the other order: eight lanes then meet eight banks. Rows of a turn are a
                    // multiple of eight apart, so the swizzle is the same in all of them.
                    static_assert(32 * kConverters / kPieces % 8 == 0);
                    const int odd = (c >> 2) & 1;
                    const uint32_t panel = to + uint32_t(c >> 2) * (kTileKeys * 128), near = panel + panel_at(row, 2 * (c & 3) + odd),
                                   far = panel + panel_at(row, 2 * (c & 3) + 1 - odd);
#pragma unroll
                    for (int u = 0; u < kTurns; ++u) {
                        uint32_t h[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) widen_key<F>(odd ? w[u][e ^ 2] : w[u][e], h[2 * e], h[2 * e + 1]);
                        constexpr uint32_t kApart = 32 * kConverters / kPieces * 128;
                        st_shared16(near + u * kApart, h[0], h[1], h[2], h[3]);
                        st_shared16(far + u * kApart, h[4], h[5], h[6], h[7]);
                    }
                }
                ptx::fence_proxy_async_smem();
                arrive(keys_ready[buffer]);
                return true;
            };
            auto note_scales = [&](int i) { // of the keys that were converted last, and of their values
                if (thread < kTileKeys) {
                    const float *scales = reinterpret_cast<const float *>(base_bytes + Shape::ring + slot * Shape::raw + kTileKeys * HeadDim);
                    const float key_scale = scales[thread], value_scale = scales[kTileKeys + thread];
                    table_key[i & 3][thread] = key_scale * args.score_scale;
                    table_value[i & 3][thread] = value_scale;
                    table_shift[i & 3][thread] = fmaxf(log2_approx(fabsf(value_scale)), kLeastScale);
                }
                arrive(tables_ready[i & 3]);
                arrive(raw_free[slot]);
                next_slot();
            };
            // The first tile's keys while the queries are on their way.
            if (!convert_keys(first_tile)) return false;
            ptx::copy_async_wait_all();
            if constexpr (kScaledRows) {
#pragma unroll 4
                for (int i = 0; i < kTurns; ++i) { // kChunks lanes hold a row
                    uint32_t w[4];
                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(place(i)) : "memory");
                    unsigned most = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = max(most, max(w[e] << 16 & 0x7fffffffu, w[e] & 0x7fff0000u));
#pragma unroll
                    for (int d = 1; d < kChunks; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
                    const int exponent = most && most < 0x7f800000u ? max(int(most >> 23), 1) - 127 : 0;
                    const float down = __int_as_float(exponent < 127 ? (127 - exponent) << 23 : 0x00400000); // 2^-exponent
                    if (!chunk) row_scale[part.ordinal & 3][thread / kChunks + 32 * kConverters / kChunks * i] = __int_as_float(exponent > -127 ? (127 + exponent) << 23 : 0x00400000);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __half2 v = __floats2half2_rn(__uint_as_float(w[e] << 16) * down, __uint_as_float(w[e] & 0xffff0000u) * down);
                        w[e] = *reinterpret_cast<const uint32_t *>(&v);
                    }
                    st_shared16(place(i), w[0], w[1], w[2], w[3]);
                }
            }
            ptx::fence_proxy_async_smem();
            arrive(queries_ready);

            note_scales(first_tile);
            auto convert_values = [&](int i) {
                const int buffer = i & 1, before = (i >> 1) - 1;
                if (!wait(raw_full[slot], use) || (before >= 0 && (!wait(weighted[0][buffer], before) || !wait(weighted[1][buffer], before)))) return false;
                {
                    const uint32_t from = base + Shape::ring + slot * Shape::raw, to = base + Shape::values + buffer * Shape::operand;
                    // A lane takes four columns (a word) of eight keys, and stores eight keys of each column. Pairs of lanes take other groups of keys, so that
                    // eight lanes meet eight banks when they store.
                    constexpr int kWords = HeadDim / 4, kSets = 32 * kConverters / kWords, kTurns = kTileKeys / 8 / kSets; // kSets: threads that share a word
                    const int word = thread % kWords, set = thread / kWords;
                    const int first = (set & ~7) | ((((word >> 1) & 3) + set) & 7); // group of keys, kSets apart from turn to turn
                    static_assert(kSets % 8 == 0);
                    uint32_t w[kTurns][8];
#pragma unroll
                    for (int u = 0; u < kTurns; ++u)
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[u][k]) : "r"(from + (8 * (kSets * u + first) + k) * HeadDim + 4 * word));
                    arrive(raw_free[slot]);
#pragma unroll
                    for (int u = 0; u < kTurns; ++u) {
                        const int group = kSets * u + first;
                        uint32_t h[4][4]; // [column][pair of keys]
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                widen<F>(biased<F>(__byte_perm(w[u][2 * k], w[u][2 * k + 1], c ? 0x7362u : 0x5140u)), h[2 * c][k], h[2 * c + 1][k]);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            st_shared16(to + uint32_t(group >> 3) * (HeadDim * 128) + panel_at(4 * word + c, group & 7), h[c][0], h[c][1], h[c][2], h[c][3]);
                    }
                }
                ptx::fence_proxy_async_smem();
                arrive(values_ready[buffer]);
                next_slot();
                return true;
            };
            const int end = first_tile + part.high - part.low;
            for (; first_tile < end; ++first_tile) {
                if (first_tile + 1 < end) {
                    if (!convert_keys(first_tile + 1)) return false;
                    note_scales(first_tile + 1);
                }
                if (!convert_values(first_tile)) return false;
            }
            return true;
        });
    } else if (warp < kSoftmaxWarps) { // --------------------------------------------------------- softmax
        // Scores are read as matrix fragments: lane l has rows l / 4 and l / 4 + 8 of the warp's 16 and of each eight columns the two at 2 (l % 4), so that a
        // thread needs a quarter of the columns' scales. With a row per thread every scale went to every thread, and the shared memory's bandwidth, which
        // the products' operands need, was what a tile waited for.
        const int team = warp >> 3, block = warp >> 2 & 1, row = 32 * (warp & 3) + lane, g = lane >> 2, t = lane & 3;
        const int first_row = 32 * (warp & 3) + 16 * block + g; // this lane's rows: this one, and eight further on
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16, block_lanes = lanes + (uint32_t(block) << 20), at_out = tmem + lanes + kOut;
        const uint32_t at_scores = tmem + block_lanes + team * kTileKeys, own_out = tmem + block_lanes + kOut + team * HeadDim;
        for_parts([&](const SegmentPart &part) {
            const int count = part.high - part.low, end = first_tile + count, flat = part.query_tile * kRows + row;
            const bool live = row < part.columns;
            int limit[2], least = INT_MAX; // the last position that a row sees
            float most[2], sum[2];
            uint64_t up[2] = {};
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int its_row = first_row + 8 * r, token = (part.query_tile * kRows + its_row) / args.group;
                limit[r] = its_row >= part.columns ? -1 : args.prefix ? part.s.length - 1 : part.s.length - part.s.count + token;
                if (its_row < part.columns) least = min(least, limit[r]);
                most[r] = -INFINITY, sum[r] = 0.f;
            }
            least = __reduce_min_sync(0xffffffffu, least);
#pragma unroll 1
            for (int i = first_tile; i < end; ++i) {
                constexpr int kHalf = kTileKeys / 2;
                const int buffer = i & 1, key = (part.low + i - first_tile) * kTileKeys + team * kHalf + 2 * t;
                const uint32_t at = at_scores + buffer * kHalf;
                const float *const of_key = table_key[i & 3] + team * kHalf + 2 * t, *const of_shift = table_shift[i & 3] + team * kHalf + 2 * t,
                                  *const of_value = table_value[i & 3] + team * kHalf + 2 * t;
                const bool masked = key - 2 * t + kHalf - 1 > least;
                if (!wait(scored[team][buffer], i >> 1) || !wait(tables_ready[i & 3], i >> 2)) return false;
                ptx::tcgen05_fence_after();
                // 32 columns at a time, the next ones on their way while these are worked on.
                if (kScaledRows && i == first_tile) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) up[r] = ptx::pack2(row_scale[part.ordinal & 3][first_row + 8 * r], row_scale[part.ordinal & 3][first_row + 8 * r]);
                }
                float highest[2] = {-INFINITY, -INFINITY};
                auto find_highest = [&](auto masked_tile) {
                    constexpr bool kMasked = decltype(masked_tile)::value;
                    uint32_t s[2][16];
                    ptx::tmem_load_rows16<32>(at, s[0]);
#pragma unroll
                    for (int unit = 0; unit < kHalf / 32; ++unit) {
                        const int c = unit * 32;
                        ptx::tmem_load_wait();
                        if (unit + 1 < kHalf / 32) ptx::tmem_load_rows16<32>(at + c + 32, s[(unit + 1) & 1]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint64_t k = *reinterpret_cast<const uint64_t *>(of_key + c + 8 * j), shift = *reinterpret_cast<const uint64_t *>(of_shift + c + 8 * j);
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                float x, y;
                                ptx::unpack2(ptx::fma2(pair(s[unit & 1][4 * j + 2 * r], s[unit & 1][4 * j + 2 * r + 1]), kScaledRows ? ptx::mul2(k, up[r]) : k, shift), x, y);
                                if (kMasked && key + c + 8 * j > limit[r]) x = -INFINITY;
                                if (kMasked && key + c + 8 * j + 1 > limit[r]) y = -INFINITY;
                                highest[r] = fmaxf(highest[r], fmaxf(x, y));
                            }
                        }
                    }
                };
                if (masked) find_highest(std::true_type{});
                else find_highest(std::false_type{});
                // The reference rises where a row's maximum passes it, and from none at all.
                if (__any_sync(0xffffffffu, highest[0] > most[0] + kReferenceSlack || highest[1] > most[1] + kReferenceSlack)) {
                    float shrink[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        highest[r] = fmaxf(highest[r], __shfl_xor_sync(0xffffffffu, highest[r], 1)); // over the row's four lanes
                        highest[r] = fmaxf(highest[r], __shfl_xor_sync(0xffffffffu, highest[r], 2));
                        const bool its = highest[r] > most[r] + kReferenceSlack;
                        shrink[r] = its ? exp2_approx(most[r] - highest[r]) : 1.f;
                        if (its) most[r] = highest[r];
                        sum[r] *= shrink[r];
                    }
                    if (i > first_tile) { // this team's output so far, once the product before this one is in it
                        if (!wait(weighted[team][buffer ^ 1], (i - 1) >> 1)) return false;
                        ptx::tcgen05_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HeadDim; c += 32) {
                            uint32_t o[16];
                            ptx::tmem_load_rows16<32>(own_out + c, o);
                            ptx::tmem_load_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink[j >> 1 & 1]);
                            tmem_store_scores16(own_out + c, o);
                        }
                    }
                }
                uint64_t minus[2], total[2] = {};
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float reference = most[r] == -INFINITY ? 0.f : most[r];
                    minus[r] = ptx::pack2(-reference, -reference);
                }
                auto weigh = [&](auto masked_tile) {
                    constexpr bool kMasked = decltype(masked_tile)::value;
                    uint32_t s[2][16];
                    ptx::tmem_load_rows16<32>(at, s[0]);
#pragma unroll
                    for (int unit = 0; unit < kHalf / 32; ++unit) {
                        const int c = unit * 32;
                        ptx::tmem_load_wait();
                        if (unit + 1 < kHalf / 32) ptx::tmem_load_rows16<32>(at + c + 32, s[(unit + 1) & 1]);
                        uint32_t p[8];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint64_t k = *reinterpret_cast<const uint64_t *>(of_key + c + 8 * j), v = *reinterpret_cast<const uint64_t *>(of_value + c + 8 * j);
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                float x, y;
                                ptx::unpack2(ptx::fma2(pair(s[unit & 1][4 * j + 2 * r], s[unit & 1][4 * j + 2 * r + 1]), kScaledRows ? ptx::mul2(k, up[r]) : k, minus[r]), x, y);
                                const bool hide_x = kMasked && key + c + 8 * j > limit[r], hide_y = kMasked && key + c + 8 * j + 1 > limit[r];
                                const uint64_t both = ptx::pack2(exp2_approx(hide_x ? -INFINITY : x), exp2_approx(hide_y ? -INFINITY : y));
                                total[r] = ptx::add2(total[r], both);
                                ptx::unpack2(ptx::mul2(both, v), x, y);
                                if (hide_x) x = 0.f; // a hidden row's scale may be anything
                                if (hide_y) y = 0.f;
                                const __half2 w = __floats2half2_rn(x, y);
                                p[2 * j + r] = *reinterpret_cast<const uint32_t *>(&w);
                            }
                        }
                        tmem_store_rows16(at + c / 2, p); // over scores that have been read: those still to come lie behind these columns
                    }
                };
                if (masked) weigh(std::true_type{});
                else weigh(std::false_type{});
                tmem_store_wait();
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float x, y;
                    ptx::unpack2(total[r], x, y);
                    sum[r] += x + y; // of this lane's columns
                }
                ptx::tcgen05_fence_before();
                arrive(softmaxed[team][buffer]);
            }
            const int head = part.head * args.group + flat - flat / args.group * args.group;
            const size_t at_row = size_t(part.s.row) + flat / args.group, index = at_row * args.heads + head;
            float *kept = part.split      ? args.partials + (size_t(blockIdx.x * 2 + part.slot) * args.part_columns + row) * (HeadDim + kPartialExtra)
                          : args.complete ? args.complete + index * (HeadDim + kPartialExtra)
                                          : nullptr;
            if (!wait(weighted[team][(end - 1) & 1], (end - 1) >> 1)) return false;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
                sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
                if (!t) stats[team][first_row + 8 * r] = make_float2(most[r], sum[r]);
            }
            arrive(meet);
            if (!wait(meet, part.ordinal)) return false;
            ptx::tcgen05_fence_after();
            // Both teams' outputs, a thread to a row now; the four warps of its rows store a quarter of the columns each.
            const float2 mine[2] = {stats[0][row], stats[1][row]};
            const float highest = fmaxf(mine[0].x, mine[1].x), reference = highest == -INFINITY ? 0.f : highest;
            const float factor[2] = {exp2_approx(mine[0].x - reference), exp2_approx(mine[1].x - reference)}, l = factor[0] * mine[0].y + factor[1] * mine[1].y;
            const float scale = l == 0.f ? 0.f : args.output_scale / l;
#pragma unroll 1
            for (int c = (warp >> 2) * (HeadDim / 4); c < ((warp >> 2) + 1) * (HeadDim / 4); c += 16) {
                uint32_t o[2][16];
                ptx::tmem_load16(at_out + c, o[0]);
                ptx::tmem_load16(at_out + HeadDim + c, o[1]);
                ptx::tmem_load_wait();
                if (!live) continue;
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = factor[0] * __uint_as_float(o[0][e]) + factor[1] * __uint_as_float(o[1][e]);
                if (kept) {
#pragma unroll
                    for (int e = 0; e < 16; e += 8) ptx::store_sector(kept + c + e, *reinterpret_cast<const float(*)[8]>(v + e));
                } else {
                    store_row16(args, static_cast<T *>(args.output) + at_row * args.output_stride + size_t(head) * HeadDim + c, v, scale);
                }
            }
            if (live && warp < 4) {
                if (kept) kept[HeadDim] = highest, kept[HeadDim + 1] = l;
                if (!args.table) {
                } else if (!part.split) args.table[index] = make_int4(0, 0, 0, 0);
                else if (part.first_cta >= 0) args.table[index] = make_int4(part.first_cta, int(blockIdx.x) - part.first_cta + 1, part.first_slot, row);
            }
            ptx::tcgen05_fence_before();
            arrive(outputs_free);
            first_tile = end;
            return true;
        });
    }
    ptx::tcgen05_fence_before();
    __syncthreads();
    ptx::tcgen05_fence_after();
    if (warp == kIssuer) ptx::tmem_dealloc(tmem, 512);
    if (args.follows) pdl_wait_upstream();
}
} // namespace tts::b200
