// Rotary positions, and the quantized key/value cache: written from 16-bit rows, read back into them.
//
// Mathematics. Pair i of a head at position p turns by the angle 2 pi a, a = p * turns[i]: (x, y) -> (x c - y n, y c + x n) with
// c = s cos 2 pi a, n = s sin 2 pi a. Positions reach 10^5 and more, where an fp32 product has lost every digit behind the point, so
// p * turns[i] is taken in 64 bits and reduced to [-1/2, 1/2] there; sincospi works on the fp32 remainder. A stored row (one token,
// one head) has one scale: amax / range, as for any row of this library (quant_codec.cuh). Everything between the load and the store
// is fp32: a 16-bit rounding between the rotation and the quantizer would only add an error that nobody needs.
//
// All of it is bound by latency: where rows are few by loads one behind another, where they are many by how little is in flight, one row's loads a warp or
// CTA (3.7 to 4.3 TB/s). The angles of a row are the same for all heads, so they are computed once a row, while its loads are in flight. A thread takes 16
// columns of a head, two blocks of eight that hold both partners of its pairs, so no pair crosses lanes; a head's scale and norm reduce over the 4 or 8
// lanes that share it.
#include "kernels/rotary_cache.h"
#include "kernels/cache_dispatch.h"
#include "kernels/launch.cuh"
#include "kernels/quant_codec.cuh"
#include "kernels/sm100_ptx.cuh"
#include <algorithm>

namespace tts {
namespace {
using namespace b200;

template <class T> __device__ __forceinline__ void store8(T *p, bool aligned, const float (&v)[8]) {
    union {
        uint4 word;
        T e[8];
    } out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.e[i] = T(v[i]);
    if (aligned) {
        *reinterpret_cast<uint4 *>(p) = out.word;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = out.e[i];
    }
}

struct Turning {
    const double *turns;
    int half; // pairs; 0 = nothing turns
    float scale;
};
__device__ __forceinline__ float2 angle_of(const Turning &t, int position, int pair) {
    const double a = double(position) * t.turns[pair];
    float s, c;
    sincospif(2.f * float(a - rint(a)), &s, &c);
    return make_float2(t.scale * c, t.scale * s);
}
// The two blocks of eight columns that lane j of a head takes.
template <bool Interleaved> __device__ __forceinline__ int2 blocks_of(int j, int half) {
    if (!Interleaved && 8 * j < half) return make_int2(j, j + half / 8);
    return make_int2(2 * j, 2 * j + 1); // half layout: what lies behind the turning columns
}
// The cosines and sines that lane j of a head needs: for all of its pairs, or of either block where that turns.
template <bool Interleaved> __device__ __forceinline__ void angles_of(int j, int2 block, int half, const float2 *angles, float2 (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int pair = Interleaved ? 4 * (i < 4 ? block.x : block.y) + (i & 3) : 8 * j + i;
        w[i] = pair < half ? angles[pair] : make_float2(1.f, 0.f);
    }
}
template <bool Interleaved> __device__ __forceinline__ void turn(float (&a)[8], float (&b)[8], int j, int2 block, int half, const float2 (&w)[8]) {
    auto pair = [](float &x, float &y, float2 by) {
        const float from = x;
        x = from * by.x - y * by.y;
        y = y * by.x + from * by.y;
    };
    if (Interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { // columns behind the turning ones pass through as they are, NaN and zeros' signs among them
            if (4 * block.x < half) pair(a[2 * i], a[2 * i + 1], w[i]);
            if (4 * block.y < half) pair(b[2 * i], b[2 * i + 1], w[4 + i]);
        }
    } else if (8 * j < half) {
#pragma unroll
        for (int i = 0; i < 8; ++i) pair(a[i], b[i], w[i]);
    }
}

template <class T> struct RotaryArgs {
    const T *input;
    T *output;
    int rows, input_stride, output_stride, lanes, tasks; // lanes per head, lanes per row
    bool aligned;
    const int *positions;
    Turning turning;
};

// Eight 16-bit elements as they are, so that a thread can have many in flight.
template <class T> __device__ __forceinline__ uint4 fetch8(const T *p, bool aligned) {
    if (aligned) return load_upstream16(p);
    union {
        uint4 words;
        T e[8];
    } v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.e[i] = load_upstream(p + i);
    return v.words;
}
// A warp takes a row: its loads, four tasks a lane, are in flight while the lanes compute the row's angles, and no barrier of the CTA comes
// between. 8191 x 2048 columns: 15.6 us, against 17.9 with a CTA a row and 22 with a CTA for four.
constexpr int kRotaryWarps = 4, kRotaryAhead = 4;
template <class T, bool Interleaved> __global__ void __launch_bounds__(32 * kRotaryWarps) rotary_rows(const RotaryArgs<T> args) {
    __shared__ float2 all_angles[kRotaryWarps][256];
    pdl_launch_dependents();
    pdl_wait_upstream();
    const int lane = threadIdx.x & 31, half = args.turning.half;
    const long long row = (long long)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    if (row >= args.rows) return;
    float2 *const angles = all_angles[threadIdx.x >> 5];
    const T *input = args.input + size_t(row) * args.input_stride;
    T *output = args.output + size_t(row) * args.output_stride;
    for (int first = 0; first < args.tasks; first += 32 * kRotaryAhead) {
        uint4 raw[kRotaryAhead][2];
#pragma unroll
        for (int i = 0; i < kRotaryAhead; ++i) {
            const int task = first + 32 * i + lane;
            if (task >= args.tasks) break;
            const int head = task / args.lanes, j = task - head * args.lanes;
            const int2 block = blocks_of<Interleaved>(j, half);
            raw[i][0] = fetch8(input + head * args.lanes * 16 + 8 * block.x, args.aligned);
            raw[i][1] = fetch8(input + head * args.lanes * 16 + 8 * block.y, args.aligned);
        }
        if (!first) {
            const int position = load_index(args.positions + row);
            for (int i = lane; i < half; i += 32) angles[i] = angle_of(args.turning, position, i);
            __syncwarp();
        }
        float2 w[8]; // the same for all tasks of a lane where a head's lanes divide the warp
        const bool same = 32 % args.lanes == 0;
#pragma unroll
        for (int i = 0; i < kRotaryAhead; ++i) {
            const int task = first + 32 * i + lane;
            if (task >= args.tasks) break;
            const int head = task / args.lanes, j = task - head * args.lanes;
            const int2 block = blocks_of<Interleaved>(j, half);
            float a[8], b[8];
            unpack8<T>(raw[i][0], a);
            unpack8<T>(raw[i][1], b);
            if (!i || !same) angles_of<Interleaved>(j, block, half, angles, w);
            turn<Interleaved>(a, b, j, block, half, w);
            store8(output + head * args.lanes * 16 + 8 * block.x, args.aligned, a);
            store8(output + head * args.lanes * 16 + 8 * block.y, args.aligned, b);
        }
    }
}

template <class T> struct WriteArgs {
    const T *queries, *keys, *values, *query_norm, *key_norm;
    T *query_output;
    int query_stride, key_stride, value_stride, output_stride;
    bool aligned;
    int query_heads, kv_heads, page_shift;
    unsigned slots;
    unsigned char *cached_keys, *cached_values;
    float *key_scales, *value_scales;
    const int *slot_of, *positions;
    Turning turning;
    float epsilon;
};

// Lanes of one warp hold whole heads (4 or 8 lanes each). Key, value and query heads are told apart by their number only. A CTA takes a row, its
// angles shared in shared memory: a decoding step has few rows, and its latency is what counts (64 rows of 16 + 2 x 8 heads 128 wide with both
// norms: 3.1 us on the device, a few hundred KB; 1021 rows without, e4m3: 7.8 us for 15 MB).
template <class T, Type F, int HeadDim, bool Interleaved> __global__ void __launch_bounds__(256) write_rows(const WriteArgs<T> args) {
    constexpr int kLanes = HeadDim / 16;
    __shared__ float2 angles[HeadDim / 2];
    pdl_launch_dependents();
    pdl_wait_upstream();
    const int row = blockIdx.x, kv = args.kv_heads;
    const int slot = load_index(args.slot_of + row);
    const bool kept = unsigned(slot) < args.slots; // negative ones are past any cache, read as unsigned
    const int tasks = (args.query_heads + 2 * kv) * kLanes, j = threadIdx.x % kLanes;
    const int2 block = blocks_of<Interleaved>(j, args.turning.half);
    for (int task = threadIdx.x, first = 1; first || task - int(threadIdx.x & 31u) < tasks; task += blockDim.x, first = 0) {
        const bool live = task < tasks;
        const int number = task / kLanes; // keys first, then values, then queries
        const int head = number < 2 * kv ? (number < kv ? number : number - kv) : number - 2 * kv;
        const bool is_query = number >= 2 * kv, is_value = !is_query && number >= kv;
        const T *source = is_query ? args.queries + size_t(row) * args.query_stride
                          : is_value ? args.values + size_t(row) * args.value_stride
                                     : args.keys + size_t(row) * args.key_stride;
        source += head * HeadDim;
        float a[8] = {}, b[8] = {};
        if (live) {
            load8(source + 8 * block.x, 8, args.aligned, a);
            load8(source + 8 * block.y, 8, args.aligned, b);
        }
        if (first) {
            for (int i = threadIdx.x; i < args.turning.half; i += blockDim.x) angles[i] = angle_of(args.turning, load_index(args.positions + row), i);
            __syncthreads();
        }
        const T *norm = is_value ? nullptr : is_query ? args.query_norm : args.key_norm;
        float squares = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) squares += a[i] * a[i] + b[i] * b[i];
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) squares += __shfl_xor_sync(0xffffffffu, squares, d);
        if (norm && live) {
            const float r = 1.f / sqrtf(squares * (1.f / HeadDim) + args.epsilon);
            float w[8];
            load8(norm + 8 * block.x, 8, args.aligned, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = a[i] * r * w[i];
            load8(norm + 8 * block.y, 8, args.aligned, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = b[i] * r * w[i];
        }
        if (!is_value && args.turning.half) {
            float2 w[8];
            angles_of<Interleaved>(j, block, args.turning.half, angles, w);
            turn<Interleaved>(a, b, j, block, args.turning.half, w);
        }
        // Magnitudes order like their bits, and infinities and NaN lie above every finite one.
        unsigned most = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            most = max(most, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
        if (!live) continue;
        if (is_query) {
            T *output = args.query_output + size_t(row) * args.output_stride + head * HeadDim;
            store8(output + 8 * block.x, args.aligned, a);
            store8(output + 8 * block.y, args.aligned, b);
        } else if (kept) {
            const bool finite = most < 0x7f800000u;
            const float scale = finite ? quant_scale<F>(__uint_as_float(most)) : __int_as_float(0x7fffffff);
            const float inverse = finite ? __fdiv_rn(1.f, scale) : 0.f;
            const size_t at = ((size_t(slot >> args.page_shift) * kv + head) << args.page_shift) + (slot & ((1 << args.page_shift) - 1));
            unsigned char *to = (is_value ? args.cached_values : args.cached_keys) + at * HeadDim;
            if (!finite) { // the scale says NaN; the bytes stay numbers
#pragma unroll
                for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.f;
            }
            b200::store8<F>(to + 8 * block.x, 8, true, a, inverse);
            b200::store8<F>(to + 8 * block.y, 8, true, b, inverse);
            if (!j) (is_value ? args.value_scales : args.key_scales)[at] = scale;
        }
    }
}

template <class T> struct ReadArgs {
    const unsigned char *cached_keys, *cached_values;
    const float *key_scales, *value_scales;
    T *keys, *values;
    int key_stride, value_stride, rows, kv_heads, page_shift, per_row, rows_per_cta; // per_row: threads that share a row
    bool aligned, sectors; // rows start on 16 bytes; on 32
    unsigned slots;
    const int *slot_of;
};

template <Type F> __device__ __forceinline__ void decode16(uint4 raw, float scale, float (&a)[8], float (&b)[8]) {
    const unsigned words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        float v[4];
        if (F == Type::I8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = float(int(static_cast<signed char>(words[w] >> (8 * i))));
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const __half2_raw pair = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(words[w] >> (16 * i)), __NV_E4M3);
                const float2 f = __half22float2(__half2(pair));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) (w < 2 ? a : b)[4 * (w & 1) + i] = v[i] * scale;
    }
}

// Sixteen decoded values as one 32-byte store where the rows allow it: lanes then write whole sectors.
template <class T> __device__ __forceinline__ void store16(T *p, bool sectors, bool aligned, const float (&a)[8], const float (&b)[8]) {
    if (!sectors) {
        store8(p, aligned, a);
        store8(p + 8, aligned, b);
        return;
    }
    union {
        uint32_t words[8];
        T e[16];
    } out;
#pragma unroll
    for (int i = 0; i < 8; ++i) out.e[i] = T(a[i]), out.e[8 + i] = T(b[i]);
    ptx::store_sector(p, out.words);
}
// A thread takes 16 columns of a head, of keys and values: both 16-byte loads are in flight together. 1021 rows written and 8190 read back
// (8 heads 128 wide, e4m3): 18.0 us for 66 MB in two launches, 3.7 TB/s, of which the reading takes 10.9 alone; two rows a thread took 21.5, 16-byte
// stores 20.9.
template <class T, Type F, int HeadDim> __global__ void __launch_bounds__(256) read_rows(const ReadArgs<T> args) {
    constexpr int kLanes = HeadDim / 16;
    pdl_launch_dependents();
    pdl_wait_upstream();
    const int in_cta = int(threadIdx.x) / args.per_row, rest = int(threadIdx.x) - in_cta * args.per_row;
    const long long row = (long long)blockIdx.x * args.rows_per_cta + in_cta;
    if (in_cta >= args.rows_per_cta || row >= args.rows) return;
    const int slot = load_index(args.slot_of + row);
    const bool held = unsigned(slot) < args.slots;
    for (int task = rest; task < args.kv_heads * kLanes; task += args.per_row) {
        const int head = task / kLanes, j = task % kLanes;
        const size_t at =
            held ? ((size_t(slot >> args.page_shift) * args.kv_heads + head) << args.page_shift) + (slot & ((1 << args.page_shift) - 1)) : 0;
        uint4 k{}, v{};
        float ks = 0.f, vs = 0.f;
        if (held && args.keys) {
            k = load_upstream16(args.cached_keys + at * HeadDim + 16 * j);
            ks = __int_as_float(load_index(reinterpret_cast<const int *>(args.key_scales + at)));
        }
        if (held && args.values) {
            v = load_upstream16(args.cached_values + at * HeadDim + 16 * j);
            vs = __int_as_float(load_index(reinterpret_cast<const int *>(args.value_scales + at)));
        }
        float a[8], b[8];
        if (args.keys) {
            decode16<F>(k, ks, a, b);
            store16(args.keys + size_t(row) * args.key_stride + head * HeadDim + 16 * j, args.sectors, args.aligned, a, b);
        }
        if (args.values) {
            decode16<F>(v, vs, a, b);
            store16(args.values + size_t(row) * args.value_stride + head * HeadDim + 16 * j, args.sectors, args.aligned, a, b);
        }
    }
}

Turning turning_of(const RotaryView &r) { return {r.turns, r.turns ? r.dims / 2 : 0, r.scale}; }

template <class T>
void rotate(TensorView input, TensorView output, const int *positions, RotaryView rotary, int head_dim, cudaStream_t stream) {
    RotaryArgs<T> args{input.ptr<T>(), output.ptr<T>(), input.rows, input.ld(), output.ld(), head_dim / 16, input.cols / 16,
                       rows_start_on(16, input) && rows_start_on(16, output), positions, turning_of(rotary)};
    const int warps = std::clamp(input.rows / 128, 1, kRotaryWarps); // few rows spread over the multiprocessors
    launch_pdl("rotary", rotary.interleaved ? rotary_rows<T, true> : rotary_rows<T, false>, dim3(unsigned((input.rows + warps - 1) / warps)),
               dim3(unsigned(32 * warps)), 0, stream, args);
}
template <class T, Type F, int HeadDim> void write(const WriteArgs<T> &args, bool interleaved, int rows, cudaStream_t stream) {
    const int tasks = (args.query_heads + 2 * args.kv_heads) * (HeadDim / 16);
    launch_pdl("cache write", interleaved ? write_rows<T, F, HeadDim, true> : write_rows<T, F, HeadDim, false>, dim3(unsigned(rows)),
               dim3(unsigned(std::min(256, (tasks + 31) / 32 * 32))), 0, stream, args);
}
template <class T, Type F, int HeadDim> void read(const ReadArgs<T> &args, cudaStream_t stream) {
    const unsigned ctas = unsigned((args.rows + args.rows_per_cta - 1) / args.rows_per_cta);
    launch_pdl("cache read", read_rows<T, F, HeadDim>, dim3(ctas), dim3(256), 0, stream, args);
}
} // namespace

void launch_rotary(TensorView input, TensorView output, const int *positions, RotaryView rotary, int head_dim, cudaStream_t stream) {
    if (!input.rows || !input.cols) return;
    if (input.type == Type::F16) rotate<__half>(input, output, positions, rotary, head_dim, stream);
    else rotate<__nv_bfloat16>(input, output, positions, rotary, head_dim, stream);
}

void launch_cache_write(CacheView cache, TensorView keys, TensorView values, const int *slots, const int *positions, RotaryView rotary,
                        TensorView queries, TensorView query_output, TensorView query_norm, TensorView key_norm, float epsilon,
                        cudaStream_t stream) {
    if (!keys.rows) return;
    by_type(keys.type, cache.type, cache.head_dim, [&](auto element, auto format, auto width) {
        using T = decltype(element);
        WriteArgs<T> args{};
        args.queries = queries.ptr<T>(), args.keys = keys.ptr<T>(), args.values = values.ptr<T>();
        args.query_norm = query_norm.ptr<T>(), args.key_norm = key_norm.ptr<T>(), args.query_output = query_output.ptr<T>();
        args.query_stride = queries.ld(), args.key_stride = keys.ld(), args.value_stride = values.ld();
        args.output_stride = query_output.ld();
        args.aligned = rows_start_on(16, queries) && rows_start_on(16, keys) && rows_start_on(16, values) && rows_start_on(16, query_norm) && rows_start_on(16, key_norm) &&
                       rows_start_on(16, query_output);
        args.query_heads = queries.data ? queries.cols / cache.head_dim : 0;
        args.kv_heads = cache.kv_heads, args.page_shift = shift_of(cache.page_size), args.slots = unsigned(cache.slots());
        args.cached_keys = static_cast<unsigned char *>(cache.keys), args.cached_values = static_cast<unsigned char *>(cache.values);
        args.key_scales = cache.key_scales, args.value_scales = cache.value_scales;
        args.slot_of = slots, args.positions = positions, args.turning = turning_of(rotary), args.epsilon = epsilon;
        write<T, decltype(format)::value, decltype(width)::value>(args, rotary.interleaved, keys.rows, stream);
    });
}

void launch_cache_read(CacheView cache, const int *slots, TensorView keys, TensorView values, cudaStream_t stream) {
    const TensorView &any = keys.data ? keys : values;
    if (!any.rows) return;
    by_type(any.type, cache.type, cache.head_dim, [&](auto element, auto format, auto width) {
        using T = decltype(element);
        ReadArgs<T> args{};
        args.cached_keys = static_cast<unsigned char *>(cache.keys), args.cached_values = static_cast<unsigned char *>(cache.values);
        args.key_scales = cache.key_scales, args.value_scales = cache.value_scales;
        args.keys = keys.ptr<T>(), args.values = values.ptr<T>(), args.key_stride = keys.ld(), args.value_stride = values.ld();
        args.rows = any.rows, args.kv_heads = cache.kv_heads, args.page_shift = shift_of(cache.page_size);
        args.per_row = std::min(256, cache.kv_heads * cache.head_dim / 16), args.rows_per_cta = 256 / args.per_row;
        args.aligned = rows_start_on(16, keys) && rows_start_on(16, values);
        args.sectors = rows_start_on(32, keys) && rows_start_on(32, values), args.slots = unsigned(cache.slots()), args.slot_of = slots;
        read<T, decltype(format)::value, decltype(width)::value>(args, stream);
    });
}
} // namespace tts
