// Device building blocks of the attention kernels: types and matrix instructions, tiles in LDS, the walk over a request's
// keys, and the bias by distance.
#pragma once

#include <type_traits>
#include <utility>

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

// A lane's and all lower lanes' sum.
template <class T>
__device__ __forceinline__ T wave_sums(T x) {
    auto moved = [&](auto way, auto rows) {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(way)::value,
                                                                 decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    const integral_constant<int, 0xf> all;
    x += moved(integral_constant<int, 0x111>(), all);  // one, two, four, eight lanes up within 16
    x += moved(integral_constant<int, 0x112>(), all);
    x += moved(integral_constant<int, 0x114>(), all);
    x += moved(integral_constant<int, 0x118>(), all);
    x += moved(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());  // lane 15 of the first and third 16 to the next
    x += moved(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());  // lane 31 to the upper half
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wave_sums(x)), 63));
}

// Tiles in LDS: rows of DP 16-bit elements, 16 bytes apart. A ds_read_b128 of 16 consecutive lanes takes 16 bytes of 16 rows,
// the transposing read of 32 lanes 64 bytes of rows that are four apart: either covers the 64 banks of 4 bytes once. Every
// place of a tile is one lane's address plus a constant, so the reads take two address registers in all.
template <int DP>
constexpr int kPitch = DP * 2 + 16;
template <int DP, int ROWS>
constexpr int kTileBytes = ROWS * kPitch<DP>;

// A tile's rows come in slots of 16: `left` positions from `first` on of a bank row, so that short passages share a tile.
struct Slot {
    int row, first, left;
};
__device__ __forceinline__ int slot_row(int r, int hi) { return tile_row(r % 8, hi); }  // of the slot that result r belongs to

// Copies ROWS rows of a tensor into such a tile through registers; rows past a slot's and elements past d become zero (the
// buffer descriptor's range check), so nothing of what lies there, infinities and NaN included, reaches a product. The rows that
// a wave copies in one step are of one slot.
template <int DP, int ROWS, int THREADS>
struct Copier {
    // threads to a row: as many as it has chunks, or, for 96 elements, four that only keep the rows apart
    static constexpr int kChunks = DP == 96 ? 16 : DP / 8;
    static constexpr int kEach = ROWS * kChunks / THREADS, kRows = THREADS / kChunks, kWaveRows = 64 / kChunks;
    static_assert(ROWS * kChunks % THREADS == 0 && THREADS % kChunks == 0, "every thread copies the same chunk of some rows");
    static_assert(kSlot % kWaveRows == 0 && (kRows % kSlot == 0 || kSlot % kRows == 0), "a wave's rows of a step are of one slot");
    static constexpr int kOut = int(0x80000000u);  // past every descriptor's range
    int row, offset, step, to, wave_row;
    bool mine;
    u32x4 held[kEach];

    __device__ void init(int thread, int64_t stride, int d) {
        const int chunk = thread % kChunks;
        mine = chunk < DP / 8;
        row = thread / kChunks % kSlot;
        wave_row = __builtin_amdgcn_readfirstlane(thread / 64) * kWaveRows;
        offset = chunk * 8 < d ? static_cast<int>(row * stride * 2) + chunk * 16 : kOut;
        step = static_cast<int>(stride * 2);
        to = thread / kChunks * kPitch<DP> + chunk * 16;
    }
    // base(slot): where the slot's first row starts
    template <class F>
    __device__ void load(const Slot (&slots)[ROWS / kSlot], F&& base) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = wave_row + kRows * i, skipped = kRows * i % kSlot;
            Slot s = slots[kRows * i / kSlot];
            if constexpr (kRows > kSlot) {  // the waves of a step copy different slots
#pragma unroll
                for (int j = kRows * i / kSlot + 1; j < kRows * (i + 1) / kSlot; ++j) {
                    const bool here = at / kSlot == j;
                    s.row = here ? slots[j].row : s.row;
                    s.first = here ? slots[j].first : s.first;
                    s.left = here ? slots[j].left : s.left;
                }
            }
            auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base(s)), 0, 0x7fffffff, 0x00020000);
            held[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, row + skipped < s.left ? offset + step * skipped : kOut, 0, 0);
        }
    }
    // The first `valid` of ROWS rows that follow each other.
    __device__ void load_rows(const char* base, int valid) {
        auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, 0x7fffffff, 0x00020000);
        const int skipped = kRows > kSlot ? wave_row / kSlot * kSlot : 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int rows = kRows * i + skipped;
            held[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, row + rows < valid ? offset + step * rows : kOut, 0, 0);
        }
    }
    __device__ void store(char* tile) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (DP != 96 || mine) *reinterpret_cast<u32x4*>(tile + to + kRows * i * kPitch<DP>) = held[i];
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

// Writes a lane's column of a result, factor * x rounded, to elements 32 * part ... of its row. The halves of the wave that share a
// column exchange every other four elements, so that a store is of 16 bytes (8 bytes each: 32 requests of 512 tokens, 12 heads of
// 64, the keys' gradient 84 us where this takes 77).
template <class E>
__device__ __forceinline__ void store_column(char* row, const f32x16& x, int part, int hi, int d, float factor) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        typename E::T y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (typename E::T)(x[8 * p + j] * factor);
        const u32x4 z = *reinterpret_cast<u32x4*>(y);
        const auto a = __builtin_amdgcn_permlane32_swap(z[0], z[2], false, false);
        const auto b = __builtin_amdgcn_permlane32_swap(z[1], z[3], false, false);
        const int at = 32 * part + 16 * p + 8 * hi;
        if (at < d) *reinterpret_cast<u32x4*>(row + at * 2) = u32x4{a[0], b[0], a[1], b[1]};
    }
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

// The bank row of passage r of request b and how many positions it holds: none for a row outside the bank. No branch follows the
// loads, so that nothing waits for them here.
__device__ __forceinline__ int2 find_row(const AttendArgs& a, int b, int r) {
    int row = b * a.passages + r, count = a.length;
    if (a.rows) row = a.rows[b * a.rows_outer + r * a.rows_step];
    const bool there = row >= 0 && row < a.bank;
    row = there ? row : 0;
    if (a.lengths && a.bank) count = min(max(a.lengths[row], 0), a.length);
    return make_int2(row, there ? count : 0);
}
// A request's keys are counted in places: slots of its passages, empty ones included, passage by passage. A block holds the rows
// of the passages that its places [begin, end) lie in.
struct Places {
    int per_row, begin, end, r0;
    __device__ Places(const AttendArgs& a, int from, int count) {
        per_row = (a.length + kSlot - 1) / kSlot;
        begin = from;
        end = min(from + count, per_row * a.passages);
        r0 = begin < end ? begin / per_row : 0;
    }
    // A thread's entry of the block's table; a block has a thread for each.
    __device__ int2 look(const AttendArgs& a, int b, int thread) const {
        return begin < end ? find_row(a, b, min(r0 + thread, (end - 1) / per_row)) : make_int2(0, 0);
    }
    __device__ void put(int2 entry, int2* found, int thread) const {
        if (thread < kHeldPassages) found[thread] = entry;
    }
};

// Where a slot's first position starts, of a key head.
__device__ __forceinline__ const char* slot_start(const AttendView& v, const Slot& s, int head) {
    return static_cast<const char*>(v.p) + (s.row * v.outer + s.first * v.middle + head * v.head) * 2;
}
// Walks the slots that hold a key, SLOTS at a time. While a row lasts its next tile is reached by adding to two addresses: what a
// wave computes for itself between its tiles is on its critical path.
template <int SLOTS>
struct KeyWalk {
    Slot slots[SLOTS];  // of the tile
    bool run;           // they are full and follow each other in one row, from these addresses on
    const char *k, *v;

    const AttendArgs& a;
    const int2* found;
    int per_row, end, r0, head;
    int r, row, first, left;  // the passage, its row, the next position and how many are left
    const char *next_k, *next_v;

    __device__ KeyWalk(const AttendArgs& args, const Places& p, const int2* held, int kv_head)
        : a(args), found(held), per_row(p.per_row), end(p.end), r0(p.r0), head(kv_head), r(p.r0), row(0), first(0), left(0) {
        next_k = next_v = nullptr;
        if (p.begin < end) take((p.begin - p.r0 * per_row) * kSlot);
        else r = end;
    }
    __device__ void take(int from) {
        row = uniform(found[r - r0].x);
        left = min(uniform(found[r - r0].y), (end - r * per_row) * kSlot) - from;
        first = from;
        next_k = slot_start(a.k, {row, first, 0}, head);
        next_v = slot_start(a.v, {row, first, 0}, head);
    }
    __device__ void pass(int positions) {
        first += positions;
        left -= positions;
        next_k += positions * a.k.middle * 2;
        next_v += positions * a.v.middle * 2;
    }
    // Goes on to the next tile, empty slots at its end; false where none is left.
    __device__ bool next() {
        run = left >= SLOTS * kSlot;
        if (run) {
            k = next_k;
            v = next_v;
#pragma unroll
            for (int i = 0; i < SLOTS; ++i) slots[i] = {row, first + kSlot * i, kSlot};
            pass(SLOTS * kSlot);
            return true;
        }
#pragma unroll
        for (int i = 0; i < SLOTS; ++i) {
            while (left <= 0 && r * per_row < end) {
                if (++r * per_row < end) take(0);
            }
            slots[i] = {0, 0, 0};
            if (left > 0) {
                slots[i] = {row, first, min(left, kSlot)};
                pass(kSlot);
            }
        }
        return slots[0].left > 0;
    }
    template <class C>
    __device__ void load(C& ks, C& vs) const {
        if (run) {
            ks.load_rows(k, SLOTS * kSlot);
            vs.load_rows(v, SLOTS * kSlot);
        } else {
            ks.load(slots, [&](const Slot& s) { return slot_start(a.k, s, head); });
            vs.load(slots, [&](const Slot& s) { return slot_start(a.v, s, head); });
        }
    }
};
// Whether all of a tile's places hold a key, and the first and last position of any.
template <int SLOTS>
__device__ __forceinline__ bool whole(const Slot (&s)[SLOTS]) {
    bool all = true;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) all = all && s[i].left == kSlot;
    return all;
}
template <int SLOTS>
__device__ __forceinline__ int2 reach(const Slot (&s)[SLOTS]) {
    int2 x = make_int2(s[0].first, s[0].first);
#pragma unroll
    for (int i = 1; i < SLOTS; ++i)
        if (s[i].left) x = make_int2(min(x.x, s[i].first), max(x.y, s[i].first));
    return make_int2(x.x, x.y + kSlot - 1);
}

// Blocks that read the same keys (or queries) follow each other in the order of places, `each` to a group. The hardware deals
// block ids over the 8 XCDs in turn: two groups that follow each other, of neighbouring heads as a rule, go to one XCD, whose L2
// sees what they read again, and the pairs to the XCDs in turn, so that ragged requests load them alike; what is left over is cut
// into 8 runs. (9 requests of up to 1592 tokens over their own, 12 heads of 64: 103, 168 and 168 us for the forward pass, the
// queries' and the keys' gradient where all groups were cut into 8 runs, 96, 147 and 137 so; 32 of 512 each take the same time.)
__device__ __forceinline__ int xcd_place(int id, int total, int each) {
    each *= 2;
    const int whole = total / each / 8 * 8 * each;
    if (id < whole) {
        const int i = id / 8, group = i / each;
        return (group * 8 + id % 8) * each + (i - group * each);
    }
    id -= whole;
    const int q = (total - whole) / 8, extra = (total - whole) % 8, x = id % 8, i = id / 8;
    return whole + x * q + min(x, extra) + i;
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

// The biases at 16 of a lane's results, 8 for each of two slots. x0, x1: the distances at their tile_row(0, hi); STEP: how a
// distance changes from row to row.
template <int STEP, class F>
__device__ __forceinline__ void each_bias(const float* held, int far, int x0, int x1, F&& use) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
        const int x = part ? x1 : x0;
        const float* at = held + bias_index(far, STEP > 0 ? x : x - 14);
#pragma unroll
        for (int r = 0; r < 8; ++r) use(8 * part + r, at[STEP > 0 ? tile_row(r, 0) : 14 - tile_row(r, 0)]);
    }
}

// Where one run of instructions ends and the next begins.
__device__ __forceinline__ void between_runs() { __builtin_amdgcn_sched_barrier(0); }
// A run of N products of the matrix cores whose first operands come from LDS, READS reads each: read(i) is kept MOST products
// in front of product(i, ...), as a read takes about as long as three to four products. The order is asked of the compiler, and
// written out besides: where a kernel is short of registers the compiler goes back to the order as written, and with each read
// right before its product the queries' gradient of the wide tables took a tenth longer.
template <int N, int READS, int MOST, class R, class P>
__device__ __forceinline__ void products(R&& read, P&& product) {
    constexpr int ahead = MOST < N ? MOST : N;
    between_runs();
    s16x8 first[ahead];
#pragma unroll
    for (int i = 0; i < ahead; ++i) first[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        product(i, first[i % ahead]);
        if (i + ahead < N) first[i % ahead] = read(i + ahead);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, READS * ahead, 0);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i + ahead < N) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    between_runs();
}

// A block of 256 threads of those that follow the queries' gradient: d_q = scale * sum of the splits' parts, four elements a thread,
// or the table's gradient, one wave per (bucket, head).
template <class E>
__device__ __forceinline__ void join_queries(const AttendGradArgs& g, int block, int thread) {
    const AttendArgs& a = g.a;
    if (block < g.join_q) {
        const int groups = a.heads / a.pack, columns = a.tokens * a.pack, quads = a.d / 4;
        const int64_t rows = static_cast<int64_t>(a.batch) * groups * columns, at = static_cast<int64_t>(block) * 256 + thread;
        if (at >= rows * quads) return;
        const int64_t row = at / quads;
        const int e = static_cast<int>(at - row * quads) * 4;
        f32x4 x{};
#pragma unroll 4
        for (int i = 0; i < a.splits; ++i) x += *reinterpret_cast<const f32x4*>(a.part + (i * rows + row) * a.d + e);
        const int c = row % columns, group = row / columns % groups, b = row / columns / groups;
        const int token = c / a.pack, head = group * a.pack + c % a.pack;
        typename E::T z[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] = (typename E::T)(x[j] * g.scale);
        char* out = static_cast<char*>(g.d_q.p) + (b * g.d_q.outer + token * g.d_q.middle + head * g.d_q.head + e) * 2;
        *reinterpret_cast<u32x2*>(out) = *reinterpret_cast<u32x2*>(z);
        return;
    }
    const int lane = thread % 64, at = (block - g.join_q) * 4 + thread / 64;
    if (at >= a.heads * a.bias.buckets) return;
    const int head = at % a.heads, bucket = at / a.heads;
    float x = 0.f;
#pragma unroll 4
    for (int i = lane; i < g.table_parts; i += 64) x += g.table_part[(static_cast<int64_t>(i) * a.heads + head) * a.bias.buckets + bucket];
    x = wave_sum(x);
    if (lane == 0) static_cast<typename E::T*>(g.d_table)[at] = (typename E::T)x;
}

}  // namespace vk::attend
