// The forward pass by tiles: O = softmax(scale Q K^T + bias) V, one pass over the keys with the running maximum and sum.
//
// A block of four waves holds 128 query columns, each wave 32 of them, and walks the key tiles of its request; a key tile (64
// rows of K and of V) is staged in LDS for all four, the next one's loads in flight meanwhile. The products are taken
// transposed, S^T = K Q^T and O^T = V^T P^T: a lane then holds one query column of the logits, its maximum and sum need one
// exchange with the lane 32 further, and the rounded weights are the second product's operand where they are.
//
// P is rounded to the inputs' type for the second product (the matrix instructions take 16-bit operands); the sum that
// normalises it, the maximum and the output are held in 32 bits. The weights are relative to a maximum that is only raised
// when it grew by more than kSlack: the output's rescaling is rare, and P <= e^kSlack keeps its relative precision in either
// type.
//
// Measured, and what bounds it (cards differ by 5 %): 4 requests of 512 tokens over 10 x 512 positions, 16 heads of 64: 62 us and
// 7 for the join of three splits, 590 TFLOP/s. For each matrix instruction there are 10 others, two of them exponentials at a
// quarter of the rate: the matrix cores are busy for 28 % of the time and the other instructions set the pace (more waves a
// SIMD, which leaves each fewer registers, 77 us). 4096 tokens over 16 x 512, 16 heads of 128 over 4 key heads: 265 us,
// 970 TFLOP/s; 4.7 others for a matrix instruction, matrix cores 45 %, LDS 34 %. 256 x 128 tokens with a bias, 12 heads of 64, the
// keys of an encoder's own rows: 51 us for 164 MB, 3.2 TB/s: a block's two tiles are too few to hide its first loads.
#include "attend_tile.hpp"

namespace vk::attend {

template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(256, DP <= 64 ? 3 : 2) void forward_kernel(AttendArgs a) {
    constexpr int kSteps = DP / 16, kParts = DP / 32, kSlots = kKeyTile / kSlot;
    __shared__ __align__(16) char tile[2][2][kTileBytes<DP, kKeyTile>];
    __shared__ int2 found[kHeldPassages];
    extern __shared__ float bias_held[];

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
    const int64_t q = b * a.q.outer + token * a.q.middle + head * a.q.head;
    const Places places(a, split * a.tiles_per_split * kSlots, a.tiles_per_split * kSlots);
    // first what the keys' loads wait for; then all other loads are under way together
    places.put(places.look(a, b, thread), found, thread);

    f32x16 o[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) o[i] = f32x16{};
    float top = -INFINITY, total = 0.f;

    Copier<DP, kKeyTile, 256> ks, vs;
    ks.init(thread, a.k.middle, a.d);
    vs.init(thread, a.v.middle, a.d);
    __syncthreads();
    KeyWalk<kSlots> walk(a, places, found, kv_head);
    bool more = walk.next();
    int now = 0;
    if (more) walk.load(ks, vs);
    s16x8 qf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) qf[i] = column(a.q, q, used, i, hi, a.d);
    const float* held = nullptr;
    int position = 0;
    bool large = false;
    if constexpr (BIAS) {
        large = fill_biases<E>(a.bias, group * a.pack, a.pack, a.scale, bias_held, thread, 256);
        held = bias_held + (head - group * a.pack) * bias_places(a.bias.far);
        position = token + a.q_start_all + (a.q_start ? a.q_start[b] : 0);
    }
    if (more) {
        ks.store(tile[0][0]);
        vs.store(tile[0][1]);
    }
    __syncthreads();
    auto run = [&](auto kind) {
        constexpr bool kLarge = decltype(kind)::value;
        while (more) {
            Slot slots[kSlots];
#pragma unroll
            for (int i = 0; i < kSlots; ++i) slots[i] = walk.slots[i];
            const bool full = walk.run || whole(slots);
            more = walk.next();
            if (more) walk.load(ks, vs);

            f32x16 s[2];
            const char *k = tile[now][0], *v = tile[now][1];
            float apart = 0.f;  // a bias that all keys of the tile share
            bool near = false;  // the tile's keys do not share one bias
            int2 at{};
            if constexpr (BIAS && !kLarge) {
                // the wave's tokens lie between its first and last column's
                const int t0 = __builtin_amdgcn_readfirstlane(position), t1 = __builtin_amdgcn_readlane(position, 31);
                at = reach(slots);
                near = !far_apart(a.bias, at.x - t1, at.y - t0);
            }
            __builtin_amdgcn_s_setprio(1);
            // the first product of each sum stands in the branch: beginning with zero costs no instruction there
            if (BIAS && near) {
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) {
                    each_bias<1>(held, a.bias.far, slots[2 * sub].first + hi - position, slots[2 * sub + 1].first + hi - position,
                                 [&](int r, float x) { s[sub][r] = x; });
                    s[sub] = E::mfma(straight<DP>(k, 32 * sub, 0, lane), qf[0], s[sub]);
                }
            } else {
                if (BIAS && !kLarge) apart = held[bias_index(a.bias.far, at.x - position)] * a.scale;
#pragma unroll
                for (int sub = 0; sub < 2; ++sub) s[sub] = E::mfma(straight<DP>(k, 32 * sub, 0, lane), qf[0], f32x16{});
            }
            products<2 * kSteps - 2, 1, 3>(
                [&](int i) { return straight<DP>(k, 32 * (i / (kSteps - 1)), 1 + i % (kSteps - 1), lane); },
                [&](int i, s16x8 x) { s[i / (kSteps - 1)] = E::mfma(x, qf[1 + i % (kSteps - 1)], s[i / (kSteps - 1)]); });
            __builtin_amdgcn_s_setprio(0);
            if constexpr (kLarge) {
#pragma unroll
                for (int sub = 0; sub < 2; ++sub)
                    each_bias<1>(held, a.bias.far, slots[2 * sub].first + hi - position, slots[2 * sub + 1].first + hi - position,
                                 [&](int r, float x) { s[sub][r] = __builtin_fmaf(s[sub][r], a.scale, x); });
            }
            if (!full) {
#pragma unroll
                for (int r = 0; r < 32; ++r)
                    if (slot_row(r, hi) >= slots[r / 8].left) s[r / 16][r % 16] = -INFINITY;
            }
            float most = s[0][0];
#pragma unroll
            for (int r = 1; r < 32; ++r) most = fmaxf(most, s[r / 16][r % 16]);
            most = both_max(most);
            if (!kLarge) most = __builtin_fmaf(most, a.scale, apart);
            if (__any(most > top + kSlack)) {
                const float raised = fmaxf(top, most);
                const float factor = raised == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((top - raised) * kLog2e);
                top = raised;
                total *= factor;
#pragma unroll
                for (int i = 0; i < kParts; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[i][r] *= factor;
            }
            const float base = top == -INFINITY ? 0.f : top;
            // scale, shared bias and maximum go into the exponent's one step
            const float by = a.scale * kLog2e, shift = (apart - base) * kLog2e;
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const float x = s[r / 16][r % 16];
                s[r / 16][r % 16] = __builtin_amdgcn_exp2f(kLarge ? (x - base) * kLog2e : __builtin_fmaf(x, by, shift));
                total += s[r / 16][r % 16];
            }
            __builtin_amdgcn_s_setprio(1);
            s16x8 p;
            products<4 * kParts, 2, 3>([&](int i) { return transposed<DP>(v, 16 * (i / kParts), i % kParts, lane); },
                                       [&](int i, s16x8 x) {
                                           if (i % kParts == 0) p = rounded<E>(s[i / kParts / 2], i / kParts % 2);
                                           o[i % kParts] = E::mfma(x, p, o[i % kParts]);
                                       });
            __builtin_amdgcn_s_setprio(0);
            if (more) {
                ks.store(tile[now ^ 1][0]);
                vs.store(tile[now ^ 1][1]);
            }
            __syncthreads();
            now ^= 1;
        }
    };
    if (BIAS && large) run(std::integral_constant<bool, BIAS>());
    else run(std::false_type());

    total = both_sum(total);
    if (!used) return;
    if (a.splits == 1) {
        const float factor = total == 0.f ? 0.f : 1.f / total;
        char* out = static_cast<char*>(a.out.p) + (b * a.out.outer + token * a.out.middle + head * a.out.head) * 2;
#pragma unroll
        for (int i = 0; i < kParts; ++i) store_column<E>(out, o[i], i, hi, a.d, factor);
        if (a.lse && hi == 0)
            a.lse[(static_cast<int64_t>(b) * a.heads + head) * a.tokens + token] = logarithm(top, total);
    } else {
        const int64_t at = ((static_cast<int64_t>(split) * a.batch + b) * groups + group) * columns + c;
        if (hi == 0) a.stat[at] = make_float2(top, total);
        float* part = a.part + at * a.d;
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int quad = 0; quad < 4; ++quad) {
                const int e = 32 * i + mfma_row(4 * quad, hi);
                if (e >= a.d) continue;
                *reinterpret_cast<f32x4*>(part + e) = f32x4{o[i][4 * quad], o[i][4 * quad + 1], o[i][4 * quad + 2], o[i][4 * quad + 3]};
            }
    }
}

template <class E, int DP>
hipError_t launch_forward(const AttendArgs& a, hipStream_t stream) {
    const int64_t column_tiles = (static_cast<int64_t>(a.tokens) * a.pack + kColumns - 1) / kColumns;
    const int64_t blocks = column_tiles * a.splits * (a.heads / a.pack) * a.batch;
    if (blocks > kMostBlocks) return hipErrorInvalidValue;
    const size_t lds = a.bias.table ? a.pack * (2 * a.bias.far + 2 * kPad + 1) * sizeof(float) : 0;
    auto kernel = a.bias.table ? forward_kernel<E, DP, true> : forward_kernel<E, DP, false>;
    kernel<<<static_cast<unsigned>(blocks), 256, lds, stream>>>(a);
    return hipGetLastError();
}

}  // namespace vk::attend
