// The forward pass for few query columns (a new token, or a few, with the query heads that share a key head): what it takes is
// reading the states once. A block holds up to 32 columns; its eight waves walk the key tiles (32 rows) in turn, each with its
// own columns' maxima, sums and outputs, which are joined in LDS at the end, so most calls are one launch and few blocks keep
// many loads in flight: a wave has its next tile's K and V (16 KB at 128 elements a head) under way while it works on one. Nothing
// waits at a barrier in between. Products, roundings and the raised maximum are those of the tile kernel (attend_forward.inl).
//
// Measured, bound by the reading: one token of each of 32 requests over 100 x 256 positions, 8 key heads of 128: 530 us for
// 3.4 GB, 2.2 of them different, 6.3 TB/s; 128 requests over 10 x 200, 12 heads of 128: 260 us for 1.6 GB, 6.0 TB/s; 256 over as many,
// heads of 64: 290 us for 1.6 GB, 5.4 TB/s (a large copy: 5.0). 64 over 10 ragged rows of up to 100, 4 key heads of 128: 19 us
// for 68 MB, one round of one block a compute unit. One request over 10 x 64: 8 us, latency: records, lengths, states and the
// join follow each other.
#include <atomic>

#include "attend_tile.hpp"

namespace vk::attend {

template <int DP>
constexpr int kFewTiles = kFewWaves * 2 * kTileBytes<DP, kFewKeys>;
template <int DP>
constexpr bool kJoinFits = kFewWaves * 32 * (DP + 4) * 4 <= kFewTiles<DP>;
static_assert(kJoinFits<32> && kJoinFits<64> && kJoinFits<96> && kJoinFits<128>, "the waves' outputs are joined where the tiles were");

template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(64 * kFewWaves, DP <= 64 ? 4 : 2) void few_kernel(AttendArgs a) {
    constexpr int kSteps = DP / 16, kParts = DP / 32, kThreads = 64 * kFewWaves, kSlots = kFewKeys / kSlot;
    extern __shared__ __align__(16) char shared[];  // tiles of each wave; (row, positions) of the passages; the bias by distance
    const int thread = threadIdx.x, lane = thread % 64, wave = uniform(thread / 64), hi = lane / 32;
    const int columns = a.tokens * a.pack, column_tiles = (columns + 31) / 32, groups = a.heads / a.pack;
    int place = xcd_place(blockIdx.x, gridDim.x, column_tiles * a.splits);
    const int column_tile = place % column_tiles;
    place /= column_tiles;
    const int split = place % a.splits;
    place /= a.splits;
    const int group = place % groups, b = place / groups;
    const int kv_head = group * a.pack / (a.heads / a.kv_heads);

    const Places places(a, split * a.tiles_per_split * kSlots, a.tiles_per_split * kSlots);
    char* mine = shared + wave * 2 * kTileBytes<DP, kFewKeys>;
    int2* found = reinterpret_cast<int2*>(shared + kFewTiles<DP>);
    const int c = column_tile * 32 + lane % 32;
    const int token = c / a.pack, head = group * a.pack + c % a.pack;
    const bool used = c < columns;
    const int64_t q = b * a.q.outer + token * a.q.middle + head * a.q.head;
    const int2 entry = places.look(a, b, thread);  // first of all, as the keys' loads wait for it
    s16x8 qf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qf[i] = column(a.q, q, used, i, hi, a.d);
    places.put(entry, found, thread);
    const float* held = nullptr;
    int position = 0;
    if constexpr (BIAS) {
        float* all = reinterpret_cast<float*>(shared + kFewTiles<DP> + kHeldPassages * sizeof(int2));
        const int distances = bias_places(a.bias.far);
        for (int p = 0; p < a.pack; ++p) fill_bias<E>(a.bias, group * a.pack + p, 1.f, all + p * distances, thread, kThreads);
        held = all + (head - group * a.pack) * distances;
        position = token + a.q_start_all + (a.q_start ? a.q_start[b] : 0);
    }
    __syncthreads();

    f32x16 o[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) o[i] = f32x16{};
    float top = -INFINITY, total = 0.f;

    Copier<DP, kFewKeys, 64> ks, vs;
    ks.init(lane, a.k.middle, a.d);
    vs.init(lane, a.v.middle, a.d);
    // the wave's next place, its passage and slot; the wave takes kSlots places of every kFewWaves * kSlots
    int at = places.begin + wave * kSlots, r = places.per_row ? at / places.per_row : 0, step = at - r * places.per_row;
    Slot slots[kSlots];
    // goes on to the wave's next tile with a key, and sets its loads going
    auto load = [&] {
        while (at < places.end) {
            int any = 0;
#pragma unroll
            for (int i = 0; i < kSlots; ++i) {
                while (step >= places.per_row) {
                    step -= places.per_row;
                    ++r;
                }
                slots[i] = {0, 0, 0};
                if (at + i < places.end) {
                    const int2 x = found[r - places.r0];
                    slots[i] = {uniform(x.x), step * kSlot, min(max(uniform(x.y) - step * kSlot, 0), kSlot)};
                }
                any += slots[i].left;
                ++step;
            }
            at += kFewWaves * kSlots;
            step += (kFewWaves - 1) * kSlots;
            if (!any) continue;
            ks.load(slots, [&](const Slot& s) { return slot_start(a.k, s, kv_head); });
            vs.load(slots, [&](const Slot& s) { return slot_start(a.v, s, kv_head); });
            return true;
        }
        return false;
    };
    bool more = load();
    while (more) {
        ks.store(mine);
        vs.store(mine + kTileBytes<DP, kFewKeys>);
        between_lanes();
        const Slot here[kSlots] = {slots[0], slots[1]};
        more = load();

        f32x16 s{};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) s = E::mfma(straight<DP>(mine, 0, i, lane), qf[i], s);
        if constexpr (BIAS) {
            each_bias<1>(held, a.bias.far, here[0].first + hi - position, here[1].first + hi - position,
                         [&](int i, float x) { s[i] = __builtin_fmaf(s[i], a.scale, x); });
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] *= a.scale;
        }
        if (!whole(here)) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (slot_row(i, hi) >= here[i / 8].left) s[i] = -INFINITY;
        }
        float most = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, s[i]);
        most = both_max(most);
        if (__any(most > top + kSlack)) {
            const float raised = fmaxf(top, most);
            const float factor = raised == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((top - raised) * kLog2e);
            top = raised;
            total *= factor;
#pragma unroll
            for (int i = 0; i < kParts; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= factor;
        }
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f((s[i] - base) * kLog2e);
            total += s[i];
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const s16x8 p = rounded<E>(s, half);
#pragma unroll
            for (int i = 0; i < kParts; ++i)
                o[i] = E::mfma(transposed<DP>(mine + kTileBytes<DP, kFewKeys>, 16 * half, i, lane), p, o[i]);
        }
        between_lanes();
    }

    // the waves' parts, joined
    constexpr int kRow = DP + 4;
    float* parts = reinterpret_cast<float*>(shared);
    float2* stats = reinterpret_cast<float2*>(found);
    total = both_sum(total);
    __syncthreads();
    if (used) {
        float* to = parts + (wave * 32 + lane % 32) * kRow;
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int quad = 0; quad < 4; ++quad)
                *reinterpret_cast<f32x4*>(to + 32 * i + mfma_row(4 * quad, hi)) =
                    f32x4{o[i][4 * quad], o[i][4 * quad + 1], o[i][4 * quad + 2], o[i][4 * quad + 3]};
        if (hi == 0) stats[wave * 32 + lane] = make_float2(top, total);
    }
    __syncthreads();
    const int held_columns = min(columns - column_tile * 32, 32), quads = a.d / 4;
    for (int i = thread; i < held_columns * quads; i += kThreads) {
        const int x = i / quads, e = i % quads * 4;
        float most = -INFINITY, sum = 0.f;
        for (int w = 0; w < kFewWaves; ++w) most = fmaxf(most, stats[w * 32 + x].x);
        const float base = most == -INFINITY ? 0.f : most;
        f32x4 y{};
        for (int w = 0; w < kFewWaves; ++w) {
            const float2 s = stats[w * 32 + x];
            const float weight = __builtin_amdgcn_exp2f((s.x - base) * kLog2e);
            sum = __builtin_fmaf(weight, s.y, sum);
            y += weight * *reinterpret_cast<const f32x4*>(parts + (w * 32 + x) * kRow + e);
        }
        const int column = column_tile * 32 + x, t = column / a.pack, h = group * a.pack + column % a.pack;
        if (a.splits == 1) {
            const float factor = sum == 0.f ? 0.f : 1.f / sum;
            typename E::T z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) z[j] = (typename E::T)(y[j] * factor);
            char* out = static_cast<char*>(a.out.p) + (b * a.out.outer + t * a.out.middle + h * a.out.head + e) * 2;
            *reinterpret_cast<u32x2*>(out) = *reinterpret_cast<u32x2*>(z);
            if (a.lse && e == 0) a.lse[(static_cast<int64_t>(b) * a.heads + h) * a.tokens + t] = logarithm(most, sum);
        } else {
            const int64_t at = ((static_cast<int64_t>(split) * a.batch + b) * groups + group) * columns + column;
            if (e == 0) a.stat[at] = make_float2(most, sum);
            *reinterpret_cast<f32x4*>(a.part + at * a.d + e) = y;
        }
    }
}

template <class E, int DP>
hipError_t launch_few(const AttendArgs& a, hipStream_t stream) {
    const int64_t blocks = (static_cast<int64_t>(a.tokens) * a.pack + 31) / 32 * a.splits * (a.heads / a.pack) * a.batch;
    if (blocks > kMostBlocks) return hipErrorInvalidValue;
    const size_t lds = kFewTiles<DP> + kHeldPassages * sizeof(int2) +
                       (a.bias.table ? a.pack * (2 * a.bias.far + 2 * kPad + 1) * sizeof(float) : 0);
    auto kernel = a.bias.table ? few_kernel<E, DP, true> : few_kernel<E, DP, false>;
    // more LDS than a kernel may have unasked; asked for once a device, for any bias
    static std::atomic<uint64_t> asked[2];
    int device = 0;
    hipError_t e = hipGetDevice(&device);
    if (e != hipSuccess) return e;
    std::atomic<uint64_t>& done = asked[a.bias.table != nullptr];
    const uint64_t bit = uint64_t(1) << (device % 64);
    if (device >= 64 || !(done.load(std::memory_order_relaxed) & bit)) {
        e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                kFewTiles<DP> + static_cast<int>(kHeldPassages * sizeof(int2)) + kMostBiasBytes);
        if (e != hipSuccess) return e;
        done.fetch_or(bit, std::memory_order_relaxed);
    }
    kernel<<<static_cast<unsigned>(blocks), 64 * kFewWaves, lds, stream>>>(a);
    return hipGetLastError();
}

}  // namespace vk::attend
