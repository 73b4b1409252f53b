// Device building blocks of the attention kernels: types and matrix instructions, tiles in LDS, the walk over a request's
// keys, and the bias by distance.
#pragma once

#include "attend.hpp"

namespace vk::attend {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Bf16 {
    using T = __bf16;
    typedef __bf16 x8 __attribute__((ext_vector_type(8)));
    static __device__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
};
struct F16 {
    using T = _Float16;
    typedef _Float16 x8 __attribute__((ext_vector_type(8)));
    static __device__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(x8, a), __builtin_bit_cast(x8, b), c, 0, 0, 0);
    }
};

// A 32x32 result of a matrix instruction: a lane holds column lane % 32 and the rows mfma_row(r, lane / 32), r = 0..15.
__device__ __forceinline__ constexpr int mfma_row(int r, int hi) { return 8 * (r / 4) + 4 * hi + r % 4; }
// Products over a tile's rows take them in an order of their own: row tile_row(r, hi) of the tile stands where the matrix
// instruction has row mfma_row(r, hi). Four results that a lane holds next to each other are then four rows apart.
__device__ __forceinline__ constexpr int tile_row(int r, int hi) { return 16 * (r / 8) + 4 * (r % 4) + 2 * (r / 4 % 2) + hi; }
// The tile's row where the matrix instruction has row m, and back.
__device__ __forceinline__ constexpr int row_at(int m) { return m / 16 * 16 + 4 * (m % 4) + 2 * (m / 8 % 2) + m / 4 % 2; }
__device__ __forceinline__ constexpr int place_of(int row) { return row / 16 * 16 + row % 16 / 4 + 8 * (row / 2 % 2) + 4 * (row % 2); }

// Eight of a lane's results, rounded, as the other operand of the next product over the tile's rows. transposed() gives the
// first operand the same order of rows, so no lane exchanges data.
template <class E>
__device__ __forceinline__ s16x8 rounded(const f32x16& x, int half) {
    typename E::x8 y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (typename E::T)x[8 * half + j];
    return __builtin_bit_cast(s16x8, y);
}

__device__ __forceinline__ float both_max(float x) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float both_sum(float x) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i);
    return x;
}

// Tiles in LDS: rows of DP 16-bit elements, 16 bytes apart. A ds_read_b128 of 16 consecutive lanes takes 16 bytes of 16 rows,
// the transposing read of 32 lanes 64 bytes of rows that are four apart: either covers the 64 banks of 4 bytes once. Every
// place of a tile is one lane's address plus a constant, so the reads take two address registers in all.
template <int DP>
constexpr int kPitch = DP * 2 + 16;
template <int DP, int ROWS>
constexpr int kTileBytes = ROWS * kPitch<DP>;

// Copies ROWS rows of a tensor into such a tile through registers; rows past `valid` and elements past d become zero (the
// buffer descriptor's range check), so nothing of what lies there, infinities and NaN included, reaches a product.
template <int DP, int ROWS, int THREADS>
struct Copier {
    static constexpr int kChunks = DP / 8, kEach = ROWS * kChunks / THREADS, kRows = THREADS / kChunks;
    static_assert(ROWS * kChunks % THREADS == 0 && THREADS % kChunks == 0, "every thread copies the same chunk of some rows");
    static constexpr int kOut = int(0x80000000u);  // past every descriptor's range
    int row, offset, step, to;
    u32x4 held[kEach];

    __device__ void init(int thread, int64_t stride, int d) {
        row = thread / kChunks;
        const int chunk = thread % kChunks;
        offset = chunk * 8 < d ? static_cast<int>(row * stride * 2) + chunk * 16 : kOut;
        step = static_cast<int>(kRows * stride * 2);
        to = row * kPitch<DP> + chunk * 16;
    }
    __device__ void load(const void* base, int valid) {
        auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            held[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, row + kRows * i < valid ? offset + step * i : kOut, 0, 0);
    }
    __device__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) *reinterpret_cast<u32x4*>(tile + to + kRows * i * kPitch<DP>) = held[i];
    }
};

// First operand, rows as they lie: 32 rows from `base` on, contracted elements 16 * step + 8 * hi ...
template <int DP>
__device__ __forceinline__ s16x8 straight(const char* tile, int base, int step, int lane) {
    return *reinterpret_cast<const s16x8*>(tile + row_at(lane % 32) * kPitch<DP> + lane / 32 * 16 + base * kPitch<DP> + step * 32);
}
// First operand, transposed: lane row = element 32 * part + lane % 32, contracted over the 16 rows from `base` on.
template <int DP>
__device__ __forceinline__ s16x8 transposed(const char* tile, int base, int part, int lane) {
    typedef __attribute__((address_space(3))) s16x4 L;
    const char* at = tile + (4 * (lane % 16 / 4) + lane / 32) * kPitch<DP> + lane % 32 / 16 * 32 + lane % 4 * 8;
    s16x8 y;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)(at + (base + 2 * half) * kPitch<DP> + part * 64));
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * half + j] = x[j];
    }
    return y;
}
// Second operand from global memory: column lane % 32 is the row `offset` elements into the tensor (used = false: zeros),
// elements 16 * step + 8 * hi ... What is not there is read at the tensor's start instead, so that no load waits for a branch.
__device__ __forceinline__ s16x8 column(const AttendView& v, int64_t offset, bool used, int step, int hi, int d) {
    const int at = 16 * step + 8 * hi;
    const bool there = used && at < d;
    const s16x8 x = *reinterpret_cast<const s16x8*>(static_cast<const char*>(v.p) + (there ? (offset + at) * 2 : 0));
    const s16x8 zero = {};
    return there ? x : zero;
}

// What lanes of a wave wrote to LDS before is there for its other lanes after.
__device__ __forceinline__ void between_lanes() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// How much a running maximum may be below the true one (attend_forward.inl).
constexpr float kSlack = 5.f;

// log(total) + top in two parts, so that nothing of log(total) is lost where every key of a row has a bias of the type's
// lowest value.
__device__ __forceinline__ float2 logarithm(float top, float total) {
    if (total == 0.f) return make_float2(-INFINITY, 0.f);
    const float b = logf(total), sum = top + b, over = sum - top;
    return make_float2(sum, isfinite(sum) ? (top - (sum - over)) + (b - over) : 0.f);
}

// One scalar-register value from a load whose address is the same in all lanes.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The bank row of passage r of request b, or -1 where there is none; rows outside the bank count as none.
__device__ __forceinline__ int64_t bank_row(const AttendArgs& a, int b, int r) {
    if (!a.rows) return static_cast<int64_t>(b) * a.passages + r;
    const int id = uniform(a.rows[b * a.rows_outer + r * a.rows_step]);
    return id >= 0 && id < a.bank ? id : -1;
}
__device__ __forceinline__ int row_length(const AttendArgs& a, int64_t row) {
    if (row < 0) return 0;
    if (!a.lengths) return a.length;
    return min(max(uniform(a.lengths[row]), 0), a.length);
}

// Walks the tiles of KEYS keys that have at least one (of `row`, from `first` on; the row holds `count`), of the places
// [begin, end) of passages x tiles.
template <int KEYS>
struct KeyWalk {
    int b, r, per_row, end, first, count;
    int64_t row;

    __device__ void begin(const AttendArgs& a, int batch, int place, int last) {
        b = batch;
        per_row = (a.length + KEYS - 1) / KEYS;
        end = min(last, per_row * a.passages);
        r = place / max(per_row, 1);
        first = (place - r * per_row) * KEYS;
        if (place < end) {
            row = bank_row(a, b, r);
            count = row_length(a, row);
            settle(a);
        } else {
            r = a.passages;
        }
    }
    __device__ bool valid() const { return r * per_row + first / KEYS < end; }
    __device__ void next(const AttendArgs& a) {
        first += KEYS;
        settle(a);
    }
    __device__ void settle(const AttendArgs& a) {
        while (first >= count) {
            ++r;
            first = 0;
            if (r * per_row >= end) return;
            row = bank_row(a, b, r);
            count = row_length(a, row);
        }
    }
};

// Blocks that read the same keys follow each other in the order of `place`; the hardware deals block ids over the 8 XCDs in
// turn, so each XCD is given one run of places and its L2 sees the same keys again.
__device__ __forceinline__ int xcd_place(int id, int total) {
    const int q = total / 8, extra = total % 8, x = id % 8, i = id / 8;
    return x * q + min(x, extra) + i;
}

// The bias by distance in LDS: held[i] = table[bucket(i - far - kPad)][head], i in [0, 2 * far + 2 * kPad]. Every distance from
// `far` on shares the last bucket of its side, so an index may be clamped; the pad at either end lets 16 neighbouring distances
// be clamped as one.
__device__ __forceinline__ int bias_places(int far) { return 2 * far + 2 * kPad + 1; }
__device__ __forceinline__ int bias_index(int far, int x) { return min(max(x + far + kPad, 0), 2 * far + kPad); }
__device__ __forceinline__ int bucket_of(const AttendBias& s, int x) {
    const int a = s.two_sided ? abs(x) : max(-x, 0), exact = s.side / 2;
    int beyond = exact;
    for (int i = 0; i < s.edges; i += 16) {  // the edges come through scalar registers; those past the last are out of reach
#pragma unroll
        for (int j = 0; j < 16; ++j) beyond += s.edge[i + j] <= a;
    }
    const int bucket = a < exact ? a : beyond;
    return bucket + (s.two_sided && x > 0 ? s.side : 0);
}
template <class E>
__device__ __forceinline__ float bias_at(const AttendBias& s, int head, int place) {
    const auto* t = static_cast<const typename E::T*>(s.table);
    return static_cast<float>(t[bucket_of(s, place - s.far - kPad) * s.bucket_stride + head * s.head_stride]);
}
template <class E>
__device__ __forceinline__ void fill_bias(const AttendBias& s, int head, float factor, float* held, int thread, int threads) {
    for (int i = thread; i < bias_places(s.far); i += threads) held[i] = bias_at<E>(s, head, i) * factor;
}
// Where a logit is scale * product + bias, the product's sum can begin with bias / scale, so that adding the bias costs no
// instruction. That is not so where a bias is so large that it swallows what is added to it (a type's lowest value, say, for
// "almost never"), or the scale so small that the quotient overflows: then the bias is added to each scaled product, as the
// definition does. The same for all threads of the block.
__device__ __forceinline__ bool is_large(float bias) { return fabsf(bias) > 1e4f && !isinf(bias); }
template <class E>
__device__ __forceinline__ bool large_bias(const AttendBias& s, int head, int heads, float scale, int thread, int threads) {
    const auto* t = static_cast<const typename E::T*>(s.table);
    bool large = scale < 1e-20f;
    for (int i = thread; i < s.buckets * heads; i += threads)
        large = large || is_large(static_cast<float>(t[i / heads * s.bucket_stride + (head + i % heads) * s.head_stride]));
    return __syncthreads_or(large);
}
// Both at once for `heads` heads, one behind the other: biases divided by the scale, or, where true is returned, as they are.
template <class E>
__device__ __forceinline__ bool fill_biases(const AttendBias& s, int head, int heads, float scale, float* held, int thread, int threads) {
    const int places = bias_places(s.far);
    bool large = scale < 1e-20f;
    for (int h = 0; h < heads; ++h)
        for (int i = thread; i < places; i += threads) {
            const float x = bias_at<E>(s, head + h, i);
            large = large || is_large(x);
            held[h * places + i] = x;
        }
    large = __syncthreads_or(large);
    if (!large)
        for (int h = 0; h < heads; ++h)
            for (int i = thread; i < places; i += threads) held[h * places + i] *= 1.f / scale;  // a thread's own
    return large;
}
// Whether all distances in [least, most] share one bucket of the far ends (one-sided: all that are not negative do too).
__device__ __forceinline__ bool far_apart(const AttendBias& s, int least, int most) {
    return most <= -s.far || least >= (s.two_sided ? s.far : 0);
}

// The biases of a 32 x 32 tile. x0: the distance at tile_row(0, hi) of the lane; STEP: how it changes from row to row.
template <int STEP, class F>
__device__ __forceinline__ void each_bias(const float* held, int far, int x0, F&& use) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int x = x0 + STEP * 16 * part;
        const float* at = held + bias_index(far, STEP > 0 ? x : x - 14);
#pragma unroll
        for (int r = 0; r < 8; ++r) use(8 * part + r, at[STEP > 0 ? tile_row(r, 0) : 14 - tile_row(r, 0)]);
    }
}

// Instruction order of a run of `n` products of the matrix cores whose first operands come from LDS, `reads` reads each: the
// reads are kept `ahead` products in front, as a read takes about as long as three to four products, and `others` vector
// instructions of another part of the tile, that runs beside it, follow each product.
template <int n, int reads, int ahead, int others = 0>
__device__ __forceinline__ void feed() {
    __builtin_amdgcn_sched_group_barrier(0x100, reads * ahead, 0);
#pragma unroll
    for (int i = 0; i < n; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i < n - ahead) __builtin_amdgcn_sched_group_barrier(0x100, reads, 0);
        if (others) __builtin_amdgcn_sched_group_barrier(0x002, others, 0);
    }
}
// Where one run ends and the next begins.
__device__ __forceinline__ void between_runs() { __builtin_amdgcn_sched_barrier(0); }

}  // namespace vk::attend
