// Attention of many query rows over the quantized, paged cache: chunks of prompts, and a prefix that a whole batch shares.
//
// Mathematics: as for few query rows (cached_attention_sm100.cuh). Scores and outputs are fp16 products with fp32 sums on the tensor cores,
// bytes enter them exactly, and what is rounded is p_j vs_j, to fp16, against a running reference that keeps it at most 256. The reference moves only
// when a tile's maximum passes it by 2^8, so that the accumulated output is rescaled hardly ever.
//
// Layout. A segment is 128 query rows of one cached head (tokens times the group's heads; of a prefix: of all sequences), a tile 128 keys. Per tile
// a CTA does S = Q K^T and O += P V as tcgen05.mma of 128 x 128 (x 64 or 128), with S, P and O in tensor memory; P overwrites S, two halves to a column. Tiles
// alternate between two teams of four softmax warps, a thread per query row, and each team has a softmax state and an output of its own: one team's
// exponentials run under the other's products, and the two meet once per segment. Four warps turn bytes into fp16 operands: keys as they are, values
// transposed, so that both are K-major with the 128-byte swizzle. Tables of a tile's scales go to the softmax warps through shared memory.
//
// Bound. A 128 x 128 x 128 tile costs the tensor pipe 1024 cycles, its exponentials the special-function units 1024, the conversions about
// 450 issue cycles, so all three have to overlap; what the two teams leave open is the latency from a product to its softmax and back.
#pragma once
#include "kernels/cached_attention_sm100.cuh"

namespace tts::b200 {
constexpr int kManyRows = 128;
constexpr int kManySegmentUnits = 6; // a segment's queries, the meeting of the teams and the store next to a tile's kTileUnits
constexpr int kSoftmaxWarps = 8, kConverters = 4, kManyWarps = kSoftmaxWarps + kConverters + 2, kManyThreads = 32 * kManyWarps;
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
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void st_shared16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 16-byte chunk `chunk` of row `row` in a K-major operand panel (rows of 64 halves, 128-byte swizzle).
__device__ __forceinline__ uint32_t panel_at(int row, int chunk) { return uint32_t(row * 128 + ((chunk ^ (row & 7)) << 4)); }
} // namespace many

template <class T, Type F, int HeadDim>
__global__ void __launch_bounds__(kManyThreads, 1) cached_attention_many(const AttentionArgs args) {
    using namespace many;
    using Shape = ManyShape<HeadDim>;
    constexpr int kRows = kManyRows, kSlots = Shape::slots, kConverter = kSoftmaxWarps, kProducer = kConverter + kConverters, kIssuer = kProducer + 1;
    constexpr uint32_t kOut = 2 * kTileKeys; // tensor memory: two teams' scores, then their outputs
    extern __shared__ uint8_t raw_smem[];
    // Tile i of the share is team i % 2's, and its barriers' use i / 2. scored: S is done (and the keys' buffer free); weighted: O is (and the
    // values' buffer, the tables and P's place are free); keys/values: operands are ready; softmaxed: P is.
    __shared__ uint64_t raw_full[kSlots], raw_free[kSlots], keys_ready[2], values_ready[2], scored[2], softmaxed[2], weighted[2];
    __shared__ uint64_t queries_ready, largest_known, meet, outputs_free, drained; // once per segment part, the last once
    __shared__ __align__(16) float table_key[2][kTileKeys], table_shift[2][kTileKeys], table_value[2][kTileKeys];
    __shared__ float2 stats[2][kRows];
    __shared__ unsigned largest[2]; // of a part's queries, by the part's parity
    __shared__ long long sums[kManyWarps];
    __shared__ Start found;
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
            ptx::mbar_init(ptx::smem_u32(&scored[t]), 1);
            ptx::mbar_init(ptx::smem_u32(&softmaxed[t]), kSoftmaxWarps / 2);
            ptx::mbar_init(ptx::smem_u32(&weighted[t]), 1);
            largest[t] = 0;
        }
        ptx::mbar_init(ptx::smem_u32(&queries_ready), kConverters);
        ptx::mbar_init(ptx::smem_u32(&largest_known), kConverters);
        ptx::mbar_init(ptx::smem_u32(&meet), kSoftmaxWarps);
        ptx::mbar_init(ptx::smem_u32(&outputs_free), kSoftmaxWarps);
        ptx::mbar_init(ptx::smem_u32(&drained), 1);
        abort_flag = 0;
        ptx::fence_barrier_init();
    }
    if (warp == kIssuer) ptx::tmem_alloc(ptx::smem_u32(&tmem_slot), 512);
    ptx::tcgen05_fence_before();
    pdl_launch_dependents();
    __syncthreads();
    ptx::tcgen05_fence_after();
    const uint32_t tmem = ptx::warp_uniform(tmem_slot);
    pdl_wait_upstream();
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
    // Every role walks the share for itself.
    const Start start = args.sequences > kScanAlone ? found : start_alone<kRows>(args, kManySegmentUnits);
    int first_tile = 0; // of the part, in the share

    if (warp == kProducer) { // ------------------------------------------------------------------ bytes and scales
        const int box = 1 << args.box_shift, boxes = kTileKeys >> args.box_shift;
        int slot = 0, item = 0, reuse = -1; // reuse: the slot's use before this one
        auto raw_tiles = [&](const SegmentPart &part) {
            const int *pages = args.pages + size_t(part.sequence) * args.page_stride;
            for (int tile = part.low; tile < part.high; ++tile) {
                const int key = tile * kTileKeys, position = key + (lane << args.box_shift);
                const bool wanted = lane < boxes && position < part.s.length;
                const int page = wanted ? load_index(pages + (position >> args.page_shift)) : -1;
                const bool good = unsigned(page) < unsigned(args.total_pages);
                const uint32_t held = __ballot_sync(0xffffffffu, good);
                const int row = (((page * args.kv_heads) + part.head) << args.page_shift) + (position & ((1 << args.page_shift) - 1));
                for (int values = 0; values < 2; ++values, ++item) {
                    if (reuse >= 0 && !wait(raw_free[slot], reuse)) return false;
                    const uint32_t to = base + Shape::ring + slot * Shape::raw, bar = ptx::smem_u32(&raw_full[slot]);
                    if (!lane) ptx::mbar_arrive_expect_tx(bar, __popc(held) * box * HeadDim);
                    __syncwarp();
                    if (good)
                        copy_run(to + uint32_t(lane << args.box_shift) * HeadDim,
                                 static_cast<const uint8_t *>(values ? args.cached_values : args.cached_keys) + size_t(row) * HeadDim, uint32_t(box) * HeadDim, bar);
                    // A lane copies the scales of four keys and four values. Positions on a page that the cache does not have read as NaN.
                    const int owner = (4 * lane) >> args.box_shift, its_row = __shfl_sync(0xffffffffu, row, owner) + ((4 * lane) & (box - 1));
                    const uint32_t scales = to + kTileKeys * HeadDim + 16 * lane;
                    if (!values) {
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
                    if (++slot == kSlots) slot = 0, ++reuse;
                }
            }
            return true;
        };
        walk_share<kRows>(args, kManySegmentUnits, start, raw_tiles);
        // No copy may be in flight when the CTA leaves, whatever the others did.
        int ignored = 0;
        for (int i = max(0, item - kSlots); i < item; ++i) ptx::mbar_wait(ptx::smem_u32(&raw_full[i % kSlots]), uint32_t(i / kSlots) & 1, &ignored);
    } else if (warp == kIssuer) { // -------------------------------------------------------------- products
        constexpr uint32_t kScoreIdesc = idesc_f16(kRows, kTileKeys), kOutIdesc = idesc_f16(kRows, HeadDim);
        auto score = [&](int i) { // S of tile i
            const int team = i & 1;
            if (!wait(keys_ready[team], i >> 1) || (i >= 2 && !wait(weighted[team], (i >> 1) - 1))) return false;
            ptx::tcgen05_fence_after();
            if (ptx::elect_one()) {
                const uint32_t q = ptx::smem_desc_lo_k128(base), k = ptx::smem_desc_lo_k128(base + Shape::keys + team * Shape::operand);
#pragma unroll
                for (int s = 0; s < HeadDim / 16; ++s) {
                    const uint32_t at = uint32_t(s >> 2) * (kRows * 128 >> 4) + uint32_t(s & 3) * 2;
                    mma_smem(tmem + team * kTileKeys, q + at, k + at, kScoreIdesc, s > 0);
                }
                ptx::tcgen05_commit(ptx::smem_u32(&scored[team]));
            }
            __syncwarp();
            return true;
        };
        walk_share<kRows>(args, kManySegmentUnits, start, [&](const SegmentPart &part) {
            const int count = part.high - part.low, end = first_tile + count;
            if (!wait(queries_ready, part.ordinal) || !score(first_tile)) return false;
            for (int i = first_tile; i < end; ++i) {
                const int team = i & 1;
                if (i + 1 < end && !score(i + 1)) return false;
                if (i == first_tile && part.ordinal && !wait(outputs_free, part.ordinal - 1)) return false;
                if (!wait(values_ready[team], i >> 1) || !wait(softmaxed[team], i >> 1)) return false;
                ptx::tcgen05_fence_after();
                if (ptx::elect_one()) {
                    const uint32_t v = ptx::smem_desc_lo_k128(base + Shape::values + team * Shape::operand);
#pragma unroll
                    for (int s = 0; s < kTileKeys / 16; ++s)
                        mma_tmem(tmem + kOut + team * HeadDim, tmem + team * kTileKeys + 8 * s,
                                 v + uint32_t(s >> 2) * (HeadDim * 128 >> 4) + uint32_t(s & 3) * 2, kOutIdesc, s > 0 || i >= first_tile + 2);
                    ptx::tcgen05_commit(ptx::smem_u32(&weighted[team]));
                }
                __syncwarp();
            }
            first_tile = end;
            return true;
        });
        // No product may be in flight when the tensor memory is given back, whatever the others did.
        if (ptx::elect_one()) ptx::tcgen05_commit(ptx::smem_u32(&drained));
        __syncwarp();
        int ignored = 0;
        ptx::mbar_wait(ptx::smem_u32(&drained), 0, &ignored);
    } else if (warp >= kConverter) { // ----------------------------------------------------------- bytes to operands
        const int mine = warp - kConverter, thread = 32 * mine + lane;
        int slot = 0, use = 0;
        auto next_slot = [&] {
            if (++slot == kSlots) slot = 0, ++use;
        };
        walk_share<kRows>(args, kManySegmentUnits, start, [&](const SegmentPart &part) {
            // Queries, once the products of the part before have read theirs. Rows past the segment are zero. BF16 rows are divided by the power of
            // two of their largest element of all, which brings them into fp16's range; what that costs the small ones is small next to the others.
            for (int i = max(0, first_tile - 2); i < first_tile; ++i)
                if (!wait(scored[i & 1], i >> 1)) return false;
            constexpr int kChunks = HeadDim / 8, kTurns = kRows * kChunks / (32 * kConverters);
            float scale_up = 1.f;
            uint4 chunk[kTurns];
            unsigned most = 0;
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int piece = thread + 32 * kConverters * i, row = piece / kChunks, c = piece % kChunks;
                const int flat = part.query_tile * kRows + row;
                chunk[i] = make_uint4(0, 0, 0, 0);
                if (row >= part.columns) continue;
                const T *from = static_cast<const T *>(args.queries) + size_t(part.s.row + flat / args.group) * args.query_stride +
                                (part.head * args.group + flat % args.group) * HeadDim + 8 * c;
                if (args.aligned) {
                    asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(chunk[i].x), "=r"(chunk[i].y), "=r"(chunk[i].z), "=r"(chunk[i].w)
                                 : "l"(from)
                                 : "memory");
                } else {
                    uint16_t v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) asm volatile("ld.global.b16 %0, [%1];" : "=h"(v[e]) : "l"(from + e) : "memory");
                    chunk[i] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
                }
            }
            if (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
                for (int i = 0; i < kTurns; ++i)
                    for (const uint32_t w : {chunk[i].x, chunk[i].y, chunk[i].z, chunk[i].w}) most = max(most, max(w << 16 & 0x7fffffffu, w & 0x7fff0000u));
                most = __reduce_max_sync(0xffffffffu, most);
                if (!lane) atomicMax(&largest[part.ordinal & 1], most);
                arrive(largest_known);
                if (!wait(largest_known, part.ordinal)) return false;
                most = *const_cast<volatile unsigned *>(&largest[part.ordinal & 1]);
                const int exponent = most && most < 0x7f800000u ? max(int(most >> 23), 1) - 127 : 0;
                const float down = __int_as_float(exponent < 127 ? (127 - exponent) << 23 : 0x00400000); // 2^-exponent
                scale_up = __int_as_float(exponent > -127 ? (127 + exponent) << 23 : 0x00400000);
#pragma unroll
                for (int i = 0; i < kTurns; ++i) {
                    uint32_t *w = &chunk[i].x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const __half2 v = __floats2half2_rn(__uint_as_float(w[e] << 16) * down, __uint_as_float(w[e] & 0xffff0000u) * down);
                        w[e] = *reinterpret_cast<const uint32_t *>(&v);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kTurns; ++i) {
                const int piece = thread + 32 * kConverters * i, row = piece / kChunks, c = piece % kChunks;
                st_shared16(base + uint32_t(c >> 3) * (kRows * 128) + panel_at(row, c & 7), chunk[i].x, chunk[i].y, chunk[i].z, chunk[i].w);
            }
            ptx::fence_proxy_async_smem();
            arrive(queries_ready);
            if (thread == 0) largest[~part.ordinal & 1] = 0; // everyone has read the part before's

            const float score_scale = args.score_scale * scale_up;
            for (int tile = part.low; tile < part.high; ++tile, ++first_tile) {
                const int team = first_tile & 1, before = (first_tile >> 1) - 1;
                if (!wait(raw_full[slot], use) || (before >= 0 && !wait(scored[team], before))) return false;
                {
                    const uint32_t from = base + Shape::ring + slot * Shape::raw, to = base + Shape::keys + team * Shape::operand;
                    constexpr int kPieces = HeadDim / 16; // lanes to a key row
#pragma unroll 4
                    for (int i = 0; i < kTileKeys * kPieces / (32 * kConverters); ++i) {
                        const int piece = thread + 32 * kConverters * i, row = piece / kPieces, c = piece % kPieces;
                        uint32_t w[4], h[8];
                        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(from + row * HeadDim + 16 * c));
#pragma unroll
                        for (int e = 0; e < 4; ++e) widen_key<F>(w[e], h[2 * e], h[2 * e + 1]);
                        const uint32_t panel = to + uint32_t(c >> 2) * (kTileKeys * 128);
                        // The second panel's lanes store their chunks in the other order: eight lanes then meet eight banks.
                        const int odd = (c >> 2) & 1;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const bool upper = e ^ odd;
                            st_shared16(panel + panel_at(row, 2 * (c & 3) + upper), upper ? h[4] : h[0], upper ? h[5] : h[1], upper ? h[6] : h[2], upper ? h[7] : h[3]);
                        }
                    }
                }
                ptx::fence_proxy_async_smem();
                arrive(raw_free[slot]);
                if (!lane) ptx::mbar_arrive(ptx::smem_u32(&keys_ready[team]));
                next_slot();
                if (!wait(raw_full[slot], use) || (before >= 0 && !wait(weighted[team], before))) return false;
                {
                    const uint32_t from = base + Shape::ring + slot * Shape::raw, to = base + Shape::values + team * Shape::operand;
                    const float *scales = reinterpret_cast<const float *>(base_bytes + Shape::ring + slot * Shape::raw + kTileKeys * HeadDim);
                    const float key_scale = scales[thread], value_scale = scales[kTileKeys + thread];
                    table_key[team][thread] = key_scale * score_scale;
                    table_value[team][thread] = value_scale;
                    table_shift[team][thread] = fmaxf(log2_approx(fabsf(value_scale)), -126.f);
                    // A lane takes four columns (a word) of eight keys, and stores eight keys of each column. Pairs of lanes take other groups of keys, so that
                    // eight lanes meet eight banks when they store.
                    constexpr int kWords = HeadDim / 4, kGroups = kTileKeys / 8, kSets = 32 * kConverters / kWords; // kSets: threads that share a word
                    const int word = thread % kWords, set = thread / kWords;
#pragma unroll 2
                    for (int i = 0; i < kGroups / kSets; ++i) {
                        const int group = kSets == 4 ? 4 * i + (((word >> 1) + set) & 3) : 8 * i + ((((word >> 1) & 3) + set) & 7);
                        uint32_t w[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[k]) : "r"(from + (8 * group + k) * HeadDim + 4 * word));
                        uint32_t h[4][4]; // [column][pair of keys]
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                widen<F>(biased<F>(__byte_perm(w[2 * k], w[2 * k + 1], c ? 0x7362u : 0x5140u)), h[2 * c][k], h[2 * c + 1][k]);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            st_shared16(to + uint32_t(group >> 3) * (HeadDim * 128) + panel_at(4 * word + c, group & 7), h[c][0], h[c][1], h[c][2], h[c][3]);
                    }
                }
                ptx::fence_proxy_async_smem();
                arrive(raw_free[slot]);
                if (!lane) ptx::mbar_arrive(ptx::smem_u32(&values_ready[team]));
                next_slot();
            }
            return true;
        });
    } else { // ----------------------------------------------------------------------------------- softmax
        const int team = warp >> 2, row = 32 * (warp & 3) + lane;
        const uint32_t lanes = uint32_t(32 * (warp & 3)) << 16, at_scores = tmem + lanes + team * kTileKeys, at_out = tmem + lanes + kOut;
        walk_share<kRows>(args, kManySegmentUnits, start, [&](const SegmentPart &part) {
            const int count = part.high - part.low, end = first_tile + count, flat = part.query_tile * kRows + row;
            const bool live = row < part.columns;
            const int limit = !live ? -1 : args.prefix ? part.s.length - 1 : part.s.length - part.s.count + flat / args.group;
            const int least = __reduce_min_sync(0xffffffffu, live ? limit : INT_MAX);
            float most = -INFINITY, sum = 0.f;
            int last = -1;
            for (int i = first_tile + ((first_tile ^ team) & 1); i < end; i += 2) {
                const int key = (part.low + i - first_tile) * kTileKeys;
                const bool masked = key + kTileKeys - 1 > least;
                if (!wait(scored[team], i >> 1) || !wait(values_ready[team], i >> 1)) return false; // the tables come with the values
                ptx::tcgen05_fence_after();
                float highest = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < kTileKeys; c += 32) {
                    uint32_t s[32];
                    ptx::tmem_load32(at_scores + c, s);
                    ptx::tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 k = *reinterpret_cast<const float4 *>(&table_key[team][c + j]), shift = *reinterpret_cast<const float4 *>(&table_shift[team][c + j]);
                        float t[4];
                        ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), ptx::pack2(k.x, k.y), ptx::pack2(shift.x, shift.y)), t[0], t[1]);
                        ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), ptx::pack2(k.z, k.w), ptx::pack2(shift.z, shift.w)), t[2], t[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (!masked || key + c + j + e <= limit) highest = fmaxf(highest, t[e]);
                    }
                }
                const bool raise = highest > most + kReferenceSlack; // also from no reference at all
                if (__any_sync(0xffffffffu, raise)) {
                    const float shrink = raise ? exp2_approx(most - highest) : 1.f;
                    if (raise) most = highest;
                    sum *= shrink;
                    if (last >= 0) // this team's output so far; the product that made it is done, or this tile's scores would not be
#pragma unroll 1
                        for (int c = 0; c < HeadDim; c += 16) {
                            uint32_t o[16];
                            ptx::tmem_load16(at_out + team * HeadDim + c, o);
                            ptx::tmem_load_wait();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                            tmem_store16(at_out + team * HeadDim + c, o);
                        }
                }
                const float reference = most == -INFINITY ? 0.f : most;
                const uint64_t minus = ptx::pack2(-reference, -reference);
                uint64_t total = 0;
#pragma unroll 1
                for (int c = 0; c < kTileKeys; c += 32) {
                    uint32_t s[32], p[16];
                    ptx::tmem_load32(at_scores + c, s);
                    ptx::tmem_load_wait();
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 k = *reinterpret_cast<const float4 *>(&table_key[team][c + j]), v = *reinterpret_cast<const float4 *>(&table_value[team][c + j]);
                        float x[4], w[4];
                        ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), ptx::pack2(k.x, k.y), minus), x[0], x[1]);
                        ptx::unpack2(ptx::fma2(ptx::pack2(__uint_as_float(s[j + 2]), __uint_as_float(s[j + 3])), ptx::pack2(k.z, k.w), minus), x[2], x[3]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = masked && key + c + j + e > limit ? 0.f : exp2_approx(x[e]);
                        const uint64_t low = ptx::pack2(x[0], x[1]), high = ptx::pack2(x[2], x[3]);
                        total = ptx::add2(total, ptx::add2(low, high));
                        ptx::unpack2(ptx::mul2(low, ptx::pack2(v.x, v.y)), w[0], w[1]);
                        ptx::unpack2(ptx::mul2(high, ptx::pack2(v.z, v.w)), w[2], w[3]);
                        if (masked) // a hidden row's scale may be anything
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = key + c + j + e > limit ? 0.f : w[e];
                        const __half2 a = __floats2half2_rn(w[0], w[1]), b = __floats2half2_rn(w[2], w[3]);
                        p[j / 2] = *reinterpret_cast<const uint32_t *>(&a), p[j / 2 + 1] = *reinterpret_cast<const uint32_t *>(&b);
                    }
                    tmem_store16(at_scores + c / 2, p); // over scores that have been read
                }
                tmem_store_wait();
                float a, b;
                ptx::unpack2(total, a, b);
                sum += a + b;
                ptx::tcgen05_fence_before();
                arrive(softmaxed[team]);
                last = i;
            }
            if (last >= 0) {
                if (!wait(weighted[team], last >> 1)) return false;
                stats[team][row] = make_float2(most, sum);
            }
            arrive(meet);
            if (!wait(meet, part.ordinal)) return false;
            ptx::tcgen05_fence_after();
            // Both teams' outputs; each team stores one half of the columns. A part of one tile has one team's only.
            const bool has[2] = {count > 1 || !(first_tile & 1), count > 1 || (first_tile & 1)};
            float highest = -INFINITY, l = 0.f, factor[2] = {0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (has[t]) highest = fmaxf(highest, stats[t][row].x);
            const float reference = highest == -INFINITY ? 0.f : highest;
#pragma unroll
            for (int t = 0; t < 2; ++t)
                if (has[t]) {
                    factor[t] = exp2_approx(stats[t][row].x - reference);
                    l += factor[t] * stats[t][row].y;
                }
            const int head = part.head * args.group + flat % args.group;
            const size_t at_row = size_t(part.s.row) + flat / args.group, index = at_row * args.heads + head;
            float *kept = part.split      ? args.partials + (size_t(blockIdx.x * 2 + part.slot) * args.part_columns + row) * (HeadDim + kPartialExtra)
                          : args.complete ? args.complete + index * (HeadDim + kPartialExtra)
                                          : nullptr;
            const float scale = l == 0.f ? 0.f : args.output_scale / l;
#pragma unroll 1
            for (int c = team * (HeadDim / 2); c < (team + 1) * (HeadDim / 2); c += 16) {
                uint32_t o[2][16];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    if (has[t]) ptx::tmem_load16(at_out + t * HeadDim + c, o[t]);
                    else
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[t][j] = 0;
                }
                ptx::tmem_load_wait();
                if (!live) continue;
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    float v[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = factor[0] * __uint_as_float(o[0][j + e]) + factor[1] * __uint_as_float(o[1][j + e]);
                    const float4 four = make_float4(v[0], v[1], v[2], v[3]);
                    if (kept) *reinterpret_cast<float4 *>(kept + c + j) = four;
                    else store_row4<T>(args, static_cast<T *>(args.output) + at_row * args.output_stride + size_t(head) * HeadDim + c + j, four, scale);
                }
            }
            if (live && !team) {
                if (kept) kept[HeadDim] = highest, kept[HeadDim + 1] = l;
                if (!part.split) args.table[index] = make_int4(0, 0, 0, 0);
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
}
} // namespace tts::b200
