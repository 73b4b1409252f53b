// The backward pass by tiles, in two kernels that each take the weights again from the logits and the forward's statistics:
//   P = exp(scale Q K^T + bias - lse),  dP = dO V^T,  dS = P (dP - delta),  delta = sum over d of dO O
//   queries: dQ = scale dS K, and the bias table's gradient, the sum of dS over the places of each bucket
//   keys:    dV = P^T dO,  dK = scale dS^T Q, summed over the query heads that share a key head
// Two kernels take 7 products where one would take 5, but each sums its own outputs in registers: no atomic sums in global
// memory, no second copy of dQ in 32 bits, and the same bits from every run. P and dS are rounded to the inputs' type where
// they become operands (the matrix instructions take 16 bits; in binary16 small dS need the loss scaling that training in
// that type uses anyway); statistics, dP, delta and all sums are held in 32 bits. delta is taken from the rounded output, as that
// is what a program has kept: its error, of 2^-9 of the output's size in bfloat16, is the same for all keys of a row. It shows where
// a row has few keys and dP - delta all but cancels; there, where one tile holds them all, delta is the sum of P dP, which is there
// by then. With more tiles that would take two more products.
//
// Measured: 32 requests of 512 tokens over their own, 12 heads of 64, a two-sided bias: queries 93 us, keys 77 us (415 and 670
// TFLOP/s of the products done), of which 30 and 14 us go by where no key is there: the reading of a block's own columns and
// the writing of its results, which all blocks do at about the same time; 4 of 2048 tokens: 135 and 131 us. 2 of 2048 tokens over
// 4 x 2048, 16 heads of 128, no bias: 395 and 610 us (1040 and 900 TFLOP/s). With heads of 64 the matrix cores are busy for 24 %
// and 35 % of the time, and the rest is VALU: exponentials, bias and the table's sums; with 128 for 51 % and 40 %, LDS for 34 % and
// 38 %, and what is left are waits: of a tile for its barrier, with two waves a SIMD, which registers limit.
#include "attend_tile.hpp"

namespace vk::attend {

// Adds dS of a 32 x 32 tile (lane: one query position, x: the distance of the tile's first key from the first query) to a
// wave's sums by distance, in a fixed order. Of each result, rows n and n + 1 in the two halves of the wave, the queries are turned
// by n lanes within a half: then lane j has the distances -j and 32 - j of every row (one more in the upper half), and adds what it
// is given to one of two sums. Past the ends of the buckets a sum goes to a register. (An LDS atomic for each element took 130
// clocks an instruction. Diagonals summed through a skewed tile in LDS took the same time, but 9 KB a wave: from far = 147 on only
// one block then had room on a compute unit, and 26 requests of 714 tokens and 162 keys, far 469, took 104 us where this takes 66.)
template <int FROM, int... R>
__device__ __forceinline__ void turn(const f32x16& ds, float (&x)[8], std::integer_sequence<int, R...>) {
    // lane j of 32 reads lane (j + n) % 32, n = tile_row(r, 0)
    ((x[R] = __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(ds[FROM + R]), 0xc000 | tile_row(FROM + R, 0) << 5))), ...);
}
__device__ __forceinline__ void add_diagonals(const f32x16& ds, float* sums, int far, int x, int lane, float& below, float& above) {
    float near = 0.f, further = 0.f;  // distance -j and 32 - j
    float turned[2][8];  // eight under way while eight are added
    turn<0>(ds, turned[0], std::make_integer_sequence<int, 8>());
    between_runs();
    turn<8>(ds, turned[1], std::make_integer_sequence<int, 8>());
    between_runs();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const bool over = lane % 32 >= 32 - tile_row(r, 0);
        near += over ? 0.f : turned[r / 8][r % 8];
        further += over ? turned[r / 8][r % 8] : 0.f;
    }
    // both sums of the lower half, and beside them those of the upper half, which belong to the lane before
    const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(near), __float_as_uint(further), false, false);
    const float sum = __uint_as_float(y[0]) + __int_as_float(__builtin_amdgcn_ds_bpermute((lane + 1) % 64 * 4, y[1]));
    const int place = x - lane % 32 + (lane & 32) + far + kPad;
    if (place < 0) below += sum;
    else if (place > 2 * far + 2 * kPad) above += sum;
    else sums[place] += sum;
    between_lanes();
}

// The first distance |x| of bucket j of a side.
__device__ __forceinline__ int bucket_begin(const AttendBias& s, int j) {
    const int exact = s.side / 2;
    return j <= exact ? j : j - exact - 1 < s.edges ? s.edge[j - exact - 1] : s.far + kPad + 1;
}

// With 32 elements a head three waves a SIMD: 32 requests of 512 tokens, 12 heads, 66 us where two take 78.
template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(256, DP <= 32 ? 3 : 2) void grad_q_kernel(AttendGradArgs g) {
    // with 128 elements a head two waves a SIMD have no registers for more
    constexpr int kSteps = DP / 16, kParts = DP / 32, kKeys = grad_keys(DP), kSubs = kKeys / 32, kSlots = kKeys / kSlot;
    const AttendArgs& a = g.a;
    __shared__ __align__(16) char tile[2][2][kTileBytes<DP, kKeys>];
    __shared__ int2 found[kHeldPassages];
    extern __shared__ float held[];  // the bias by distance; per wave its gradient's sums by distance

    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, hi = lane / 32;
    const int columns = a.tokens * a.pack, column_tiles = (columns + kColumns - 1) / kColumns, groups = a.heads / a.pack;
    int place = xcd_place(blockIdx.x, gridDim.x, column_tiles * a.splits);
    const int column_tile = place % column_tiles;
    place /= column_tiles;
    const int split = place % a.splits;
    place /= a.splits;
    const int group = place % groups, b = place / groups;
    const int kv_head = group * a.pack / (a.heads / a.kv_heads);

    const int c = column_tile * kColumns + wave * 32 + lane % 32;
    const int token = c / a.pack, head = group * a.pack + c % a.pack;
    const bool used = c < columns;
    const int64_t row = (static_cast<int64_t>(b) * a.heads + head) * a.tokens + token;
    auto at = [&](const AttendView& v) { return b * v.outer + token * v.middle + head * v.head; };
    const Places places(a, split * a.tiles_per_split * kSlots, a.tiles_per_split * kSlots);
    const int2 entry = places.look(a, b, thread);  // first of all, as the keys' loads wait for it
    s16x8 qf[kSteps], df[kSteps], of[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qf[i] = column(a.q, at(a.q), used, i, hi, a.d);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) df[i] = column(g.d_out, at(g.d_out), used, i, hi, a.d);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) of[i] = column(a.out, at(a.out), used, i, hi, a.d);
    float2 lse = a.lse[used ? row : 0];
    places.put(entry, found, thread);

    f32x16 dq[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) dq[i] = f32x16{};

    Copier<DP, kKeys, 256> ks, vs;
    ks.init(thread, a.k.middle, a.d);
    vs.init(thread, a.v.middle, a.d);
    __syncthreads();
    KeyWalk<kSlots> walk(a, places, found, kv_head);
    bool more = walk.next();
    int now = 0;
    if (more) walk.load(ks, vs);
    int position = 0;
    float below = 0.f, above = 0.f;
    bool large = false;
    float* sums = nullptr;
    if constexpr (BIAS) {
        const int distances = bias_places(a.bias.far);
        sums = held + (1 + wave) * distances;
        large = fill_biases<E>(a.bias, head, 1, a.scale, held, thread, 256);
        for (int i = thread; i < 4 * distances; i += 256) held[distances + i] = 0.f;
        position = token + a.q_start_all + (a.q_start ? a.q_start[b] : 0);
    }

    float delta = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const auto x = __builtin_bit_cast(typename E::x8, df[i]), y = __builtin_bit_cast(typename E::x8, of[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(static_cast<float>(x[j]), static_cast<float>(y[j]), delta);
    }
    delta = both_sum(delta);
    // rows without a key, and columns past the last: exp(x - inf) = 0
    lse = make_float2(!used || lse.x == -INFINITY ? INFINITY : lse.x, used ? lse.y * -kLog2e : 0.f);
    const float scale_log2 = a.scale * kLog2e;
    if (more) {
        ks.store(tile[0][0]);
        vs.store(tile[0][1]);
    }
    __syncthreads();
    const char *k, *v;
    // all but the first of a sub-tile's logits: dP's first step, and the others of both in turn
    auto logits = [&](f32x16 (&s)[kSubs], f32x16 (&dp)[kSubs]) {
        constexpr int kEach = 2 * kSteps - 1;
        products<kSubs * kEach, 1, 4>(
            [&](int i) { return straight<DP>(i % kEach % 2 ? k : v, 32 * (i / kEach), (i % kEach + 1) / 2, lane); },
            [&](int i, s16x8 x) {
                const int sub = i / kEach, step = (i % kEach + 1) / 2;
                if (i % kEach % 2) s[sub] = E::mfma(x, qf[step], s[sub]);
                else dp[sub] = E::mfma(x, df[step], dp[sub]);
            });
    };
    auto gather = [&](const f32x16& ds, int sub) {
        s16x8 y;
        products<2 * kParts, 2, 3>([&](int i) { return transposed<DP>(k, 32 * sub + 16 * (i / kParts), i % kParts, lane); },
                                   [&](int i, s16x8 x) {
                                       if (i % kParts == 0) y = rounded<E>(ds, i / kParts);
                                       dq[i % kParts] = E::mfma(x, y, dq[i % kParts]);
                                   });
    };
    // kAlone: one tile holds all keys of the rows
    auto run = [&](auto kind, auto single) {
        constexpr bool kLarge = decltype(kind)::value, kAlone = decltype(single)::value;
        while (more) {
            Slot slots[kSlots];
#pragma unroll
            for (int i = 0; i < kSlots; ++i) slots[i] = walk.slots[i];
            const bool full = walk.run || whole(slots);
            more = !kAlone && walk.next();
            if (more) walk.load(ks, vs);
            const int2 at_keys = reach(slots);
            k = tile[now][0];
            v = tile[now][1];
            f32x16 s[kSubs], dp[kSubs] = {};
            bool near = kLarge;  // the tile's keys do not share one bias
            float apart = 0.f;   // the bias they share
            int t0 = 0;
            if constexpr (BIAS) {
                t0 = __builtin_amdgcn_readfirstlane(position);
                if (!kLarge) near = !far_apart(a.bias, at_keys.x - (t0 + 31), at_keys.y - t0);
            }
            // the first product of each sum stands in the branch: beginning with zero costs no instruction there
            if (BIAS && !kLarge && near) {
#pragma unroll
                for (int sub = 0; sub < kSubs; ++sub) {
                    each_bias<1>(held, a.bias.far, slots[2 * sub].first + hi - position, slots[2 * sub + 1].first + hi - position,
                                 [&](int r, float x) { s[sub][r] = x; });
                    s[sub] = E::mfma(straight<DP>(k, 32 * sub, 0, lane), qf[0], s[sub]);
                }
            } else {
                if (BIAS && !kLarge) apart = held[bias_index(a.bias.far, at_keys.x - position)] * a.scale;
#pragma unroll
                for (int sub = 0; sub < kSubs; ++sub) s[sub] = E::mfma(straight<DP>(k, 32 * sub, 0, lane), qf[0], f32x16{});
            }
            logits(s, dp);
            if constexpr (kLarge) {
#pragma unroll
                for (int sub = 0; sub < kSubs; ++sub)
                    each_bias<1>(held, a.bias.far, slots[2 * sub].first + hi - position, slots[2 * sub + 1].first + hi - position,
                                 [&](int r, float x) {
                                     s[sub][r] = __builtin_fmaf(__builtin_fmaf(s[sub][r], a.scale, x) - lse.x, kLog2e, lse.y);
                                 });
            } else {
                const float shift = __builtin_fmaf(apart - lse.x, kLog2e, lse.y);
#pragma unroll
                for (int r = 0; r < 16 * kSubs; ++r) s[r / 16][r % 16] = __builtin_fmaf(s[r / 16][r % 16], scale_log2, shift);
            }
            if constexpr (kAlone) {
                float sum = 0.f;
#pragma unroll
                for (int r = 0; r < 16 * kSubs; ++r) {
                    const float p = __builtin_amdgcn_exp2f(s[r / 16][r % 16]);
                    sum = __builtin_fmaf(slot_row(r, hi) < slots[r / 8].left ? p : 0.f, dp[r / 16][r % 16], sum);
                }
                delta = both_sum(sum);
            }
#pragma unroll
            for (int r = 0; r < 16 * kSubs; ++r)
                s[r / 16][r % 16] = __builtin_amdgcn_exp2f(s[r / 16][r % 16]) * (dp[r / 16][r % 16] - delta);
            if (!full) {
#pragma unroll
                for (int r = 0; r < 16 * kSubs; ++r)
                    if (slot_row(r, hi) >= slots[r / 8].left) s[r / 16][r % 16] = 0.f;
            }
            if constexpr (BIAS) {
                if (near) {
                    // a sub-tile whose two slots do not follow each other goes by each on its own
#pragma unroll
                    for (int sub = 0; sub < kSubs; ++sub) {
                        const Slot &x = slots[2 * sub], &y = slots[2 * sub + 1];
                        if (y.left && y.first != x.first + kSlot) {
                            f32x16 one = s[sub];
#pragma unroll
                            for (int r = 0; r < 8; ++r) one[r] = 0.f;
                            add_diagonals(one, sums, a.bias.far, y.first - kSlot - t0, lane, below, above);
                            one = s[sub];
#pragma unroll
                            for (int r = 8; r < 16; ++r) one[r] = 0.f;
                            add_diagonals(one, sums, a.bias.far, x.first - t0, lane, below, above);
                        } else {
                            add_diagonals(s[sub], sums, a.bias.far, x.first - t0, lane, below, above);
                        }
                    }
                } else {
                    float all = 0.f;
#pragma unroll
                    for (int r = 0; r < 16 * kSubs; ++r) all += s[r / 16][r % 16];
                    if (at_keys.x < position) below += all;
                    else above += all;
                }
            }
#pragma unroll
            for (int sub = 0; sub < kSubs; ++sub) gather(s[sub], sub);
            if (more) {
                ks.store(tile[now ^ 1][0]);
                vs.store(tile[now ^ 1][1]);
            }
            __syncthreads();
            now ^= 1;
        }
    };
    auto each = [&](auto single) {
        if (BIAS && large) run(std::integral_constant<bool, BIAS>(), single);
        else run(std::false_type(), single);
    };
    KeyWalk<kSlots> ahead = walk;
    if (a.splits == 1 && !ahead.next()) each(std::true_type());
    else each(std::false_type());

    if (used && hi == 0 && split == 0) g.delta[row] = delta;
    if (used && a.splits > 1) {
        float* part = a.part + (((static_cast<int64_t>(split) * a.batch + b) * groups + group) * columns + c) * a.d;
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int quad = 0; quad < 4; ++quad) {
                const int e = 32 * i + mfma_row(4 * quad, hi);
                if (e < a.d)
                    *reinterpret_cast<f32x4*>(part + e) = f32x4{dq[i][4 * quad], dq[i][4 * quad + 1], dq[i][4 * quad + 2], dq[i][4 * quad + 3]};
            }
    } else if (used) {
        char* out = static_cast<char*>(g.d_q.p) + at(g.d_q) * 2;
#pragma unroll
        for (int i = 0; i < kParts; ++i) store_column<E>(out, dq[i], i, hi, a.d, g.scale);
    }
    if constexpr (BIAS) {
        const AttendBias& s = a.bias;
        const int distances = bias_places(s.far), zero = s.far + kPad;  // the place of distance 0
        below = wave_sum(below);
        above = wave_sum(above);
        if (lane == 0) {
            sums[0] += below;
            sums[distances - 1] += above;
        }
        __syncthreads();
        for (int i = thread; i < distances; i += 256) {
            float x = 0.f;
            for (int w = 1; w <= 4; ++w) x += held[w * distances + i];
            held[i] = x;
        }
        __syncthreads();
        for (int bucket = thread / 8; bucket < (s.buckets + 31) / 32 * 32; bucket += 32) {  // eight lanes each
            const int j = bucket % s.side, from = bucket_begin(s, j), to = j + 1 < s.side ? bucket_begin(s, j + 1) : zero + 1;
            float x = 0.f;
            if (bucket < s.side) {
                for (int y = from + thread % 8; y < to; y += 8) x += held[zero - y];
                if (!s.two_sided && j == 0)
                    for (int y = 1 + thread % 8; y <= zero; y += 8) x += held[zero + y];
            } else if (bucket < s.buckets) {
                for (int y = max(from, 1) + thread % 8; y < to; y += 8) x += held[zero + y];
            }
#pragma unroll
            for (int i = 1; i < 8; i *= 2) x += __shfl_xor(x, i);
            if (thread % 8 == 0 && bucket < s.buckets)
                g.table_part[(((static_cast<int64_t>(split) * a.batch + b) * column_tiles + column_tile) * a.heads + head) * s.buckets +
                             bucket] = x;
        }
    }
}

// Keys come in slots of 16 positions of a passage. A block takes eight of a request's slots that hold a key, in order, so that what
// ragged passages leave empty costs no products; and beside them it writes the zeros of the keys that are absent in the eight slots
// that would be its own if all were full. (8 requests of 256 tokens over 8 passages of up to 256 positions, 8 key heads of 128: 108 us
// with a block's own slots whatever they held, 94 so; 33 of 84 over 14 of up to 511: 161 and 136; blocks of one tile pay for the
// search, 217 of 27 over 4 of up to 48: 95 and 102.)
struct KeySlot {
    int row, first, left;
};
// The lane's of the wave's two slots, `slot` and the next. All lanes of the wave call it.
__device__ __forceinline__ KeySlot key_slot(const AttendArgs& a, int b, int slot, int per_row, int lane) {
    if (!a.lengths) {
        const int own = slot + lane % 32 / kSlot, passage = own / per_row, first = (own - passage * per_row) * kSlot;
        return passage < a.passages ? KeySlot{b * a.passages + passage, first, a.length - first} : KeySlot{0, 0, 0};
    }
    KeySlot x[2] = {};
    int before = 0, found = 0;
    for (int r0 = 0; r0 < a.passages && found < 2; r0 += 64) {
        const int count = r0 + lane < a.passages ? min(max(a.lengths[b * a.passages + r0 + lane], 0), a.length) : 0;
        const int slots = (count + kSlot - 1) / kSlot;
        const int upto = wave_sums(slots);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint64_t at = __ballot(before + upto > slot + i);
            if (found > i || !at) continue;
            const int l = __builtin_ctzll(at);
            const int n = slot + i - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(slots, l));
            x[i] = {b * a.passages + r0 + l, n * kSlot, __builtin_amdgcn_readlane(count, l) - n * kSlot};
            found = i + 1;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    if (found < 2) x[1].first = x[0].first;  // what is not there lies beside what is
    return lane % 32 < kSlot ? x[0] : x[1];
}
// Row and position of the lane's key in the slots as they would be if all were full, where it is past the row's length; else (0, -1).
__device__ __forceinline__ int2 absent_key(const AttendArgs& a, int b, int slot, int per_row, int lane) {
    const int own = slot + lane % 32 / kSlot, passage = own / per_row, key = (own - passage * per_row) * kSlot + lane % kSlot;
    if (!a.lengths || passage >= a.passages || key >= a.length) return make_int2(0, -1);
    const int row = b * a.passages + passage;
    return key < a.lengths[row] ? make_int2(0, -1) : make_int2(row, key);
}

// Writes a key's d_k or d_v, or a split's part of it.
template <class E, int DP>
__device__ __forceinline__ void store_key(const AttendGradArgs& g, bool value, int split, int row, int key, int kv_head, int hi,
                                          const f32x16 (&sum)[DP / 32]) {
    const AttendArgs& a = g.a;
    const AttendView& v = value ? g.d_v : g.d_k;
    if (g.kv_splits > 1) {
        float* part = g.kv_part + ((((value ? g.kv_splits : 0) + split) * a.bank + row) * a.length + key) * a.kv_heads * a.d + kv_head * a.d;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (int quad = 0; quad < 4; ++quad) {
                const int e = 32 * i + mfma_row(4 * quad, hi);
                if (e < a.d)
                    *reinterpret_cast<f32x4*>(part + e) = f32x4{sum[i][4 * quad], sum[i][4 * quad + 1], sum[i][4 * quad + 2], sum[i][4 * quad + 3]};
            }
    } else {
        char* out = static_cast<char*>(v.p) + (row * v.outer + key * v.middle + kv_head * v.head) * 2;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) store_column<E>(out, sum[i], i, hi, a.d, value ? 1.f : g.scale);
    }
}

// One block: 128 keys of a request and key head (8 slots), each wave 32 of them; walks the request's query tiles, head by head.
template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(256, 2) void grad_kv_kernel(AttendGradArgs g) {
    constexpr int kSteps = DP / 16, kParts = DP / 32, kQueries = grad_queries(DP);
    const AttendArgs& a = g.a;
    __shared__ __align__(16) char tile[2][2][kTileBytes<DP, kQueries>];
    // of each query, in the order of the products' rows: -lse / scale and -delta, with which the products' sums begin; for
    // large biases lse and -what its rounding left off * log2(e)
    __shared__ __align__(16) float stat[2][4][kQueries];
    extern __shared__ float bias_held[];

    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, hi = lane / 32;
    const int share = a.heads / a.kv_heads, per_row = (a.length + kSlot - 1) / kSlot;
    const int key_tiles = (per_row * a.passages + kColumns / kSlot - 1) / (kColumns / kSlot);
    const int keys = key_tiles * g.kv_splits * a.kv_heads * a.batch;
    if (static_cast<int>(blockIdx.x) >= keys) {
        join_queries<E>(g, blockIdx.x - keys, thread);
        return;
    }
    int place = xcd_place(blockIdx.x, keys, key_tiles * g.kv_splits);
    const int key_tile = place % key_tiles;
    place /= key_tiles;
    int split = 0;
    if (g.kv_splits > 1) {
        split = place % g.kv_splits;
        place /= g.kv_splits;
    }
    const int kv_head = place % a.kv_heads, b = place / a.kv_heads;
    const int slot = key_tile * (kColumns / kSlot) + wave * 2;
    const KeySlot mine = key_slot(a, b, slot, per_row, lane);
    const int row = mine.row, first_key = mine.first, key = first_key + lane % kSlot;
    const bool there = lane % kSlot < mine.left;
    const int2 absent = absent_key(a, b, slot, per_row, lane);
    if (absent.y >= 0) {
        const f32x16 none[kParts] = {};
        store_key<E, DP>(g, false, split, absent.x, absent.y, kv_head, hi, none);
        store_key<E, DP>(g, true, split, absent.x, absent.y, kv_head, hi, none);
    }

    f32x16 dk[kParts], dv[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) dk[i] = dv[i] = f32x16{};

    if (__syncthreads_or(there)) {
        s16x8 kf[kSteps], vf[kSteps];
        const float scale_log2 = a.scale * kLog2e, by_scale = 1.f / a.scale;
        const int start = BIAS ? a.q_start_all + (a.q_start ? uniform(a.q_start[b]) : 0) : 0;
        Copier<DP, kQueries, 256> qs, ds;
        qs.init(thread, a.q.middle, a.d);
        ds.init(thread, g.d_out.middle, a.d);
        float2 lse;
        float delta = 0.f;
        const int query_tiles = (a.tokens + kQueries - 1) / kQueries, begin = split * g.kv_tiles_per_split;
        int left = min(g.kv_tiles_per_split, query_tiles * share - begin);  // tiles
        int head = kv_head * share, first = 0;
        if (split) {
            head += begin / query_tiles;
            first = begin % query_tiles * kQueries;
        }
        auto load = [&] {
            const int valid = a.tokens - first;
            qs.load_rows(slot_start(a.q, {b, first, 0}, head), valid);
            ds.load_rows(slot_start(g.d_out, {b, first, 0}, head), valid);
            if (thread < kQueries) {
                const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.tokens + first + thread;
                // nothing is computed from them before store(): that would wait for all loads under way
                lse = thread < valid ? a.lse[at] : make_float2(-INFINITY, 0.f);
                delta = thread < valid ? g.delta[at] : 0.f;
            }
        };
        auto store = [&](int to) {
            qs.store(tile[to][0]);
            ds.store(tile[to][1]);
            if (thread < kQueries) {
                const int at = place_of(thread);
                const float value = lse.x == -INFINITY ? INFINITY : lse.x, low = lse.y * -kLog2e;
                stat[to][0][at] = (low * kLn2 - value) * by_scale;
                stat[to][1][at] = -delta;
                stat[to][2][at] = value;
                stat[to][3][at] = low;
            }
        };
        load();
        {
            const int64_t k = row * a.k.outer + key * a.k.middle + kv_head * a.k.head;
            const int64_t v = row * a.v.outer + key * a.v.middle + kv_head * a.v.head;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) kf[i] = column(a.k, k, there, i, hi, a.d);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) vf[i] = column(a.v, v, there, i, hi, a.d);
        }
        bool large = false;
        if constexpr (BIAS) {
            large = share > 1 && large_bias<E>(a.bias, kv_head * share, share, a.scale, thread, 256);
            if (large) fill_bias<E>(a.bias, head, 1.f, bias_held, thread, 256);
            else large = fill_biases<E>(a.bias, head, 1, a.scale, bias_held, thread, 256);
        }
        store(0);
        __syncthreads();
        int now = 0;
        bool more = left > 0;
        const char *q, *d;
        auto of = [&](int which, int sub, int quad) {
            return *reinterpret_cast<const f32x4*>(&stat[now][which][32 * sub + mfma_row(4 * quad, hi)]);
        };
        auto logits = [&](f32x16 (&s)[2], f32x16 (&dp)[2]) {
            products<4 * kSteps, 1, 4>([&](int i) { return straight<DP>(i % 2 ? d : q, 32 * (i / (2 * kSteps)), i / 2 % kSteps, lane); },
                                       [&](int i, s16x8 x) {
                                           const int sub = i / (2 * kSteps), step = i / 2 % kSteps;
                                           if (i % 2) dp[sub] = E::mfma(x, vf[step], dp[sub]);
                                           else s[sub] = E::mfma(x, kf[step], s[sub]);
                                       });
        };
        auto gather = [&](const f32x16 (&p)[2], const f32x16 (&ds)[2]) {
            s16x8 y, z;
            products<8 * kParts, 2, 3>([&](int i) { return transposed<DP>(i % 2 ? q : d, 16 * (i / (2 * kParts)), i / 2 % kParts, lane); },
                                       [&](int i, s16x8 x) {
                                           const int half = i / (2 * kParts), part = i / 2 % kParts;
                                           if (i % (2 * kParts) == 0) {
                                               y = rounded<E>(p[half / 2], half % 2);
                                               z = rounded<E>(ds[half / 2], half % 2);
                                           }
                                           if (i % 2) dk[part] = E::mfma(x, z, dk[part]);
                                           else dv[part] = E::mfma(x, y, dv[part]);
                                       });
        };
        auto run = [&](auto kind) {
            constexpr bool kLarge = decltype(kind)::value;
            while (more) {
                const int from = first;
                first += kQueries;
                bool turned = false;
                if (first >= a.tokens) {
                    first = 0;
                    ++head;
                    turned = true;
                }
                more = --left > 0;
                if (more) load();
                q = tile[now][0];
                d = tile[now][1];
                f32x16 s[2], dp[2];
#pragma unroll
                for (int quad = 0; quad < 8; ++quad) {
                    const f32x4 l = of(0, quad / 4, quad % 4), e = of(1, quad / 4, quad % 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[quad / 4][4 * (quad % 4) + j] = kLarge ? 0.f : l[j];
                        dp[quad / 4][4 * (quad % 4) + j] = e[j];
                    }
                }
                float apart = 0.f;  // a bias that all places of the tile share
                if constexpr (BIAS && !kLarge) {
                    const int x = __builtin_amdgcn_readfirstlane(first_key), y = __builtin_amdgcn_readlane(first_key, kSlot);
                    if (far_apart(a.bias, min(x, y) - (from + kQueries - 1 + start), max(x, y) + kSlot - 1 - (from + start))) {
                        apart = bias_held[bias_index(a.bias.far, key - (from + start))] * scale_log2;
                    } else {
#pragma unroll
                        for (int sub = 0; sub < 2; ++sub)
                            each_bias<-1>(bias_held, a.bias.far, key - (from + start + 32 * sub + hi), key - (from + start + 32 * sub + 16 + hi),
                                          [&](int r, float x) { s[sub][r] += x; });
                    }
                }
                logits(s, dp);
                if constexpr (kLarge) {
#pragma unroll
                    for (int sub = 0; sub < 2; ++sub) {
                        each_bias<-1>(bias_held, a.bias.far, key - (from + start + 32 * sub + hi), key - (from + start + 32 * sub + 16 + hi),
                                      [&](int r, float x) { s[sub][r] = __builtin_fmaf(s[sub][r], a.scale, x); });
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            s[sub][r] = __builtin_fmaf(s[sub][r] - of(2, sub, r / 4)[r % 4], kLog2e, of(3, sub, r / 4)[r % 4]);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 32; ++r)
                        s[r / 16][r % 16] = BIAS ? __builtin_fmaf(s[r / 16][r % 16], scale_log2, apart) : s[r / 16][r % 16] * scale_log2;
                }
#pragma unroll
                for (int r = 0; r < 32; ++r) {
                    s[r / 16][r % 16] = __builtin_amdgcn_exp2f(s[r / 16][r % 16]);
                    dp[r / 16][r % 16] *= s[r / 16][r % 16];
                }
                gather(s, dp);
                if (more) store(now ^ 1);
                if constexpr (BIAS) {
                    if (turned && more) {  // another head's bias, once every wave is done with this one's
                        __syncthreads();
                        fill_bias<E>(a.bias, head, kLarge ? 1.f : by_scale, bias_held, thread, 256);
                    }
                }
                __syncthreads();
                now ^= 1;
            }
        };
        if (BIAS && large) run(std::integral_constant<bool, BIAS>());
        else run(std::false_type());
    }

    if (there) {
        store_key<E, DP>(g, false, split, row, key, kv_head, hi, dk);
        store_key<E, DP>(g, true, split, row, key, kv_head, hi, dv);
    }
}

// The same for more than 64 elements a head, with query tiles of 32 rows. The work on 32 keys is dealt over two waves, as one
// wave's keys, values and two gradients would take more registers than two waves a SIMD may have:
//   the first:  S = Q K^T, P = exp(...), dV += dO^T P, and P to LDS in 32 bits
//   the second, one tile behind:  dP = dO V^T, dS = P (dP - delta), dK += Q^T dS
// Both take as many products; three tiles lie in LDS, one for each of them and one to be filled. (With a fourth tile and every
// half's two products of different tiles, so that no product waits for its own tile's exponentials: 635 -> 700 us then. 64 keys
// for two waves of twice the registers: 673.)
template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(512, 2) void grad_kv_pair_kernel(AttendGradArgs g) {
    constexpr int kSteps = DP / 16, kParts = DP / 32, kQueries = grad_queries(DP);
    const AttendArgs& a = g.a;
    __shared__ __align__(16) char tile[3][2][kTileBytes<DP, kQueries>];
    __shared__ f32x4 handed[2][4][4][64];  // P of a tile: by waves, quads of rows, lanes
    // of each query, in the order of the products' rows: -lse / scale and -delta, with which the products' sums begin; for
    // large biases lse and -what its rounding left off * log2(e)
    __shared__ __align__(16) float stat[3][4][kQueries];
    extern __shared__ float bias_held[];

    const int thread = threadIdx.x, lane = thread % 64, hi = lane / 32, wave = uniform(thread / 64) % 4;
    const bool second = uniform(thread / 256) != 0;
    const int share = a.heads / a.kv_heads, per_row = (a.length + kSlot - 1) / kSlot;
    const int key_tiles = (per_row * a.passages + kColumns / kSlot - 1) / (kColumns / kSlot);
    const int keys = key_tiles * g.kv_splits * a.kv_heads * a.batch;
    if (static_cast<int>(blockIdx.x) >= keys) {
        const int block = 2 * (blockIdx.x - keys) + (second ? 1 : 0);
        if (block < g.join_q + g.join_table) join_queries<E>(g, block, thread % 256);
        return;
    }
    int place = xcd_place(blockIdx.x, keys, key_tiles * g.kv_splits);
    const int key_tile = place % key_tiles;
    place /= key_tiles;
    int split = 0;
    if (g.kv_splits > 1) {
        split = place % g.kv_splits;
        place /= g.kv_splits;
    }
    const int kv_head = place % a.kv_heads, b = place / a.kv_heads;
    const int slot = key_tile * (kColumns / kSlot) + wave * 2;
    const KeySlot mine = key_slot(a, b, slot, per_row, lane);
    const int row = mine.row, first_key = mine.first, key = first_key + lane % kSlot;
    const bool there = lane % kSlot < mine.left;
    const int2 absent = absent_key(a, b, slot, per_row, lane);
    if (absent.y >= 0) {
        const f32x16 none[kParts] = {};
        store_key<E, DP>(g, !second, split, absent.x, absent.y, kv_head, hi, none);
    }

    f32x16 sum[kParts];  // dV or dK
#pragma unroll
    for (int i = 0; i < kParts; ++i) sum[i] = f32x16{};

    if (__syncthreads_or(there)) {
        s16x8 own[kSteps];  // V or K
        const float scale_log2 = a.scale * kLog2e, by_scale = 1.f / a.scale;
        const int start = BIAS ? a.q_start_all + (a.q_start ? uniform(a.q_start[b]) : 0) : 0;
        const int query_tiles = (a.tokens + kQueries - 1) / kQueries, first_tile = split * g.kv_tiles_per_split;
        const int tiles = min(g.kv_tiles_per_split, query_tiles * share - first_tile);
        const AttendView& rows = second ? g.d_out : a.q;  // each half of the block copies one of the two
        Copier<DP, kQueries, 256> copier;
        copier.init(thread % 256, rows.middle, a.d);
        float2 lse;
        float delta = 0.f;
        auto load = [&](int head, int first) {
            const int valid = a.tokens - first;
            copier.load_rows(slot_start(rows, {b, first, 0}, head), valid);
            if (thread < kQueries) {
                const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.tokens + first + thread;
                // nothing is computed from them before store(): that would wait for all loads under way
                lse = thread < valid ? a.lse[at] : make_float2(-INFINITY, 0.f);
                delta = thread < valid ? g.delta[at] : 0.f;
            }
        };
        auto store = [&](int to) {
            copier.store(tile[to][second]);
            if (thread < kQueries) {
                const int at = place_of(thread);
                const float value = lse.x == -INFINITY ? INFINITY : lse.x, low = lse.y * -kLog2e;
                stat[to][0][at] = (low * kLn2 - value) * by_scale;
                stat[to][1][at] = -delta;
                stat[to][2][at] = value;
                stat[to][3][at] = low;
            }
        };
        auto logits = [&](f32x16 s, const char* rows) {
            products<kSteps, 1, 4>([&](int i) { return straight<DP>(rows, 0, i, lane); }, [&](int i, s16x8 x) { s = E::mfma(x, own[i], s); });
            return s;
        };
        auto gather = [&](const f32x16& z, const char* rows) {
            s16x8 y;
            products<2 * kParts, 2, 3>([&](int i) { return transposed<DP>(rows, 16 * (i / kParts), i % kParts, lane); },
                                       [&](int i, s16x8 x) {
                                           if (i % kParts == 0) y = rounded<E>(z, i / kParts);
                                           sum[i % kParts] = E::mfma(x, y, sum[i % kParts]);
                                       });
        };
        int head = kv_head * share, first = 0;  // of the tile that is loaded next
        if (split) {
            head += first_tile / query_tiles;
            first = first_tile % query_tiles * kQueries;
        }
        load(head, first);
        {
            const AttendView& v = second ? a.v : a.k;
            const int64_t at = row * v.outer + key * v.middle + kv_head * v.head;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) own[i] = column(v, at, there, i, hi, a.d);
        }
        bool large = false;
        if constexpr (BIAS) {
            large = share > 1 && large_bias<E>(a.bias, kv_head * share, share, a.scale, thread, 512);
            if (large) fill_bias<E>(a.bias, head, 1.f, bias_held, thread, 512);
            else large = fill_biases<E>(a.bias, head, 1, a.scale, bias_held, thread, 512);
        }
        store(0);
        __syncthreads();
        // each half of the block has a loop of its own, with the same barriers
        auto run = [&](auto half, auto kind) {
            constexpr bool kSecond = decltype(half)::value, kLarge = decltype(kind)::value;
            int now = 0, before = 2, from = 0;
            for (int n = 0; n <= tiles; ++n) {
                const int after = now == 2 ? 0 : now + 1;
                from = first;
                first += kQueries;
                const bool turned = first >= a.tokens;
                if (turned) {
                    first = 0;
                    ++head;
                }
                if (n + 1 < tiles) load(head, first);
                between_runs();
                auto begin = [&](int at, int which) {
                    f32x16 x;
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = reinterpret_cast<const f32x4*>(&stat[at][which][mfma_row(r / 4 * 4, hi)])[0][r % 4];
                    return x;
                };
                if (!kSecond && n < tiles) {
                    f32x16 s = kLarge ? f32x16{} : begin(now, 0);
                    float apart = 0.f;  // a bias that all places of the tile share
                    if constexpr (BIAS && !kLarge) {
                        const int x = __builtin_amdgcn_readfirstlane(first_key), y = __builtin_amdgcn_readlane(first_key, kSlot);
                        if (far_apart(a.bias, min(x, y) - (from + kQueries - 1 + start), max(x, y) + kSlot - 1 - (from + start))) {
                            apart = bias_held[bias_index(a.bias.far, key - (from + start))] * scale_log2;
                        } else {
                            each_bias<-1>(bias_held, a.bias.far, key - (from + start + hi), key - (from + start + 16 + hi), [&](int r, float x) { s[r] += x; });
                        }
                    }
                    s = logits(s, tile[now][0]);
                    if constexpr (kLarge) {
                        const f32x16 l = begin(now, 2), low = begin(now, 3);
                        each_bias<-1>(bias_held, a.bias.far, key - (from + start + hi), key - (from + start + 16 + hi), [&](int r, float x) {
                            s[r] = __builtin_fmaf(__builtin_fmaf(s[r], a.scale, x) - l[r], kLog2e, low[r]);
                        });
                    } else {
#pragma unroll
                        for (int r = 0; r < 16; ++r) s[r] = BIAS ? __builtin_fmaf(s[r], scale_log2, apart) : s[r] * scale_log2;
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(s[r]);
#pragma unroll
                    for (int quad = 0; quad < 4; ++quad)
                        handed[n % 2][wave][quad][lane] = f32x4{s[4 * quad], s[4 * quad + 1], s[4 * quad + 2], s[4 * quad + 3]};
                    gather(s, tile[now][1]);
                } else if (kSecond && n > 0) {
                    f32x16 dp = logits(begin(before, 1), tile[before][1]);
#pragma unroll
                    for (int quad = 0; quad < 4; ++quad) {
                        const f32x4 p = handed[(n + 1) % 2][wave][quad][lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) dp[4 * quad + j] *= p[j];
                    }
                    gather(dp, tile[before][0]);
                }
                between_runs();
                if (n + 1 < tiles) store(after);
                if constexpr (BIAS) {
                    if (turned && n + 1 < tiles) {  // another head's bias, once every wave is done with this one's
                        __syncthreads();
                        fill_bias<E>(a.bias, head, kLarge ? 1.f : by_scale, bias_held, thread, 512);
                    }
                }
                __syncthreads();
                before = now;
                now = after;
            }
        };
        auto both = [&](auto kind) {
            if (second) run(std::true_type(), kind);
            else run(std::false_type(), kind);
        };
        if (BIAS && large) both(std::integral_constant<bool, BIAS>());
        else both(std::false_type());
    }

    if (there) store_key<E, DP>(g, !second, split, row, key, kv_head, hi, sum);
}

template <class E, int DP>
hipError_t launch_grad_q(const AttendGradArgs& g, hipStream_t stream) {
    const AttendArgs& a = g.a;
    const int64_t blocks = (static_cast<int64_t>(a.tokens) * a.pack + kColumns - 1) / kColumns * (a.heads / a.pack) * a.batch * a.splits;
    if (blocks > kMostBlocks) return hipErrorInvalidValue;
    const size_t lds = a.bias.table ? 5 * (2 * a.bias.far + 2 * kPad + 1) * sizeof(float) : 0;
    auto kernel = a.bias.table ? grad_q_kernel<E, DP, true> : grad_q_kernel<E, DP, false>;
    kernel<<<static_cast<unsigned>(blocks), 256, lds, stream>>>(g);
    return hipGetLastError();
}

template <class E, int DP>
hipError_t launch_grad_kv(const AttendGradArgs& g, hipStream_t stream) {
    const AttendArgs& a = g.a;
    const int64_t slots = static_cast<int64_t>((a.length + kSlot - 1) / kSlot) * a.passages;
    const int64_t joined = static_cast<int64_t>(g.join_q) + g.join_table;
    const int64_t blocks = (slots + kColumns / kSlot - 1) / (kColumns / kSlot) * a.kv_heads * a.batch * g.kv_splits +
                           (DP <= 64 ? joined : (joined + 1) / 2);
    if (blocks > kMostBlocks) return hipErrorInvalidValue;
    const size_t lds = a.bias.table ? (2 * a.bias.far + 2 * kPad + 1) * sizeof(float) : 0;
    if constexpr (DP <= 64) {  // two waves for 32 keys: 170 us where one took 142 then (4 x 2048 tokens, 12 heads of 64)
        auto kernel = a.bias.table ? grad_kv_kernel<E, DP, true> : grad_kv_kernel<E, DP, false>;
        kernel<<<static_cast<unsigned>(blocks), 256, lds, stream>>>(g);
    } else {  // one wave for 32 keys: 767 us where two took 603 then (2 x 2048 tokens over 4 x 2048, 16 heads of 128)
        auto kernel = a.bias.table ? grad_kv_pair_kernel<E, DP, true> : grad_kv_pair_kernel<E, DP, false>;
        kernel<<<static_cast<unsigned>(blocks), 512, lds, stream>>>(g);
    }
    return hipGetLastError();
}

}  // namespace vk::attend
