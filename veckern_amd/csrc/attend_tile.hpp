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

// In the 32x32 result of a matrix instruction a lane holds column lane % 32 and the rows row_of(r, lane / 32), r = 0..15.
__device__ __forceinline__ constexpr int row_of(int r, int hi) { return 8 * (r / 4) + 4 * hi + r % 4; }

// Eight of a lane's results, rounded, as the other operand of the next product. Its 16 contracted indices are then in the
// order (hi, j) -> 8 * (j / 4) + 4 * hi + j % 4, which transposed() gives the first operand too, so no lane exchanges data.
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

// Tiles in LDS: rows of DP 16-bit elements, in 16-byte chunks; chunk c of a row lies at place c ^ spread(row). A
// ds_read_b128 of 16 consecutive lanes takes one chunk of 16 rows, and the transposing read of 32 lanes four chunks of four
// consecutive rows: with this order either covers the 64 banks of 4 bytes once.
template <int DP>
__device__ __forceinline__ constexpr int spread(int row) {
    return DP == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// Copies ROWS rows of a tensor into such a tile through registers; rows past `valid` and elements past d become zero (the
// buffer descriptor's range check), so nothing of what lies there, infinities and NaN included, reaches a product.
template <int DP, int ROWS, int THREADS>
struct Copier {
    static constexpr int kChunks = DP / 8, kEach = ROWS * kChunks / THREADS;
    static_assert(ROWS * kChunks % THREADS == 0, "every thread copies the same number of chunks");
    static constexpr int kOut = int(0x80000000u);  // past every descriptor's range
    int offset[kEach];
    u32x4 held[kEach];

    __device__ void init(int thread, int64_t stride, int d) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int p = thread + THREADS * i, row = p / kChunks, chunk = (p % kChunks) ^ spread<DP>(row);
            offset[i] = chunk * 8 < d ? static_cast<int>(row * stride * 2) + chunk * 16 : kOut;
        }
    }
    __device__ void load(int thread, const void* base, int valid) {
        auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int row = (thread + THREADS * i) / kChunks;
            held[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, row < valid ? offset[i] : kOut, 0, 0);
        }
    }
    __device__ void store(int thread, void* tile) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) static_cast<u32x4*>(tile)[thread + THREADS * i] = held[i];
    }
};

// First operand, rows as they lie: lane row = base + lane % 32, contracted elements 16 * step + 8 * hi ...
template <int DP>
__device__ __forceinline__ s16x8 straight(const void* tile, int base, int step, int lane) {
    const int row = base + lane % 32;
    return static_cast<const s16x8*>(tile)[row * (DP / 8) + ((2 * step + lane / 32) ^ spread<DP>(row))];
}
// First operand, transposed: lane row = element 32 * part + lane % 32, contracted over the tile's rows base + (hi, j).
template <int DP>
__device__ __forceinline__ s16x8 transposed(const void* tile, int base, int part, int lane) {
    typedef __attribute__((address_space(3))) s16x4 L;
    s16x8 y;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int row = base + 8 * half + 4 * (lane / 32) + lane % 16 / 4;
        const int chunk = 4 * part + lane % 32 / 16 * 2 + lane % 4 / 2;
        const char* at = static_cast<const char*>(tile) + (row * (DP / 8) + (chunk ^ spread<DP>(row))) * 16 + lane % 2 * 8;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L*)at);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[4 * half + j] = x[j];
    }
    return y;
}
// Second operand from global memory: column lane % 32 is the row at `p` (nullptr: zeros), elements 16 * step + 8 * hi ...
__device__ __forceinline__ s16x8 column(const void* p, int step, int hi, int d) {
    const int at = 16 * step + 8 * hi;
    s16x8 zero = {};
    return p && at < d ? *reinterpret_cast<const s16x8*>(static_cast<const char*>(p) + at * 2) : zero;
}

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

// Walks the key tiles (row, first, valid) with at least one key, of the places [begin, end) of passages x tiles.
struct KeyWalk {
    int b, r, per_row, end, first, count;
    int64_t row;

    __device__ void begin(const AttendArgs& a, int batch, int place, int last) {
        b = batch;
        per_row = (a.length + kKeyTile - 1) / kKeyTile;
        end = min(last, per_row * a.passages);
        r = place / max(per_row, 1);
        first = (place - r * per_row) * kKeyTile;
        if (place < end) {
            row = bank_row(a, b, r);
            count = row_length(a, row);
            settle(a);
        } else {
            r = a.passages;
        }
    }
    __device__ bool valid() const { return r * per_row + first / kKeyTile < end; }
    __device__ void next(const AttendArgs& a) {
        first += kKeyTile;
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

// The bias by distance in LDS: held[i] = table[bucket(i - far - 3)][head], i in [0, 2 * far + 7). Every distance
// from `far` on shares the last bucket of its side, so an index may be clamped; the three more at either end let four
// neighbouring distances be clamped as one.
__device__ __forceinline__ int bias_places(int far) { return 2 * far + 7; }
__device__ __forceinline__ int bias_index(int far, int x) { return min(max(x + far + 3, 0), 2 * far + 3); }
__device__ __forceinline__ int bucket_of(const AttendBias& s, int x) {
    const int a = s.two_sided ? abs(x) : max(-x, 0), exact = s.side / 2;
    int bucket = a;
    if (a >= exact) {
        int lo = 0, hi = s.edges;  // the number of edges <= a
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (s.edge[mid] <= a) lo = mid + 1;
            else hi = mid;
        }
        bucket = exact + lo;
    }
    return bucket + (s.two_sided && x > 0 ? s.side : 0);
}
template <class E>
__device__ __forceinline__ void fill_bias(const AttendBias& s, int head, float* held, int thread, int threads) {
    for (int i = thread; i < bias_places(s.far); i += threads) {
        const auto* t = static_cast<const typename E::T*>(s.table);
        held[i] = static_cast<float>(t[bucket_of(s, i - s.far - 3) * s.bucket_stride + head * s.head_stride]);
    }
}
// Whether all distances in [least, most] share one bucket of the far ends (one-sided: all that are not negative do too).
__device__ __forceinline__ bool far_apart(const AttendBias& s, int least, int most) {
    return most <= -s.far || least >= (s.two_sided ? s.far : 0);
}

// A bias beyond this swallows what is added to it in part or whole: it is added to each product first, as the definition
// does, also where a tile's keys share one.
constexpr float kLargeBias = 1e4f;

// The logits of a 32 x 32 tile, scores * scale + bias, in natural units (a type's lowest value, as a bias that almost never
// lets a key through, would overflow in log2 units). x0: the distance at the lane's row_of(0), step: the
// distance's change from row to row.
template <int STEP>
__device__ __forceinline__ void add_bias(f32x16& s, float scale, const float* held, int far, int x0) {
#pragma unroll
    for (int quad = 0; quad < 4; ++quad) {
        const int x = x0 + STEP * 8 * quad;
        const float* at = held + bias_index(far, STEP > 0 ? x : x - 3);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * quad + j] = __builtin_fmaf(s[4 * quad + j], scale, at[STEP > 0 ? j : 3 - j]);
    }
}

}  // namespace vk::attend
