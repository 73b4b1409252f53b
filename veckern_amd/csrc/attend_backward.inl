// The backward pass by tiles, in two kernels that each take the weights again from the logits and the forward's statistics:
//   P = exp(scale Q K^T + bias - lse),  dP = dO V^T,  dS = P (dP - delta),  delta = sum over d of dO O
//   queries: dQ = scale dS K, and the bias table's gradient, the sum of dS over the places of each bucket
//   keys:    dV = P^T dO,  dK = scale dS^T Q, summed over the query heads that share a key head
// Two kernels take 7 products where one would take 5, but each sums its own outputs in registers: no atomic sums in global
// memory, no second copy of dQ in 32 bits, and the same bits from every run. P and dS are rounded to the inputs' type where
// they become operands (the matrix instructions take 16 bits; in binary16 small dS need the loss scaling that training in
// that type uses anyway); statistics, dP, delta and all sums are held in 32 bits.
#include "attend_tile.hpp"

namespace vk::attend {

template <class T>
__device__ __forceinline__ void store_four(void* p, int at, const f32x16& x, int quad, float factor) {
    T y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (T)(x[4 * quad + j] * factor);
    *reinterpret_cast<u32x2*>(static_cast<char*>(p) + at * 2) = *reinterpret_cast<u32x2*>(y);
}

// Adds dS of a 32 x 32 tile (lane: one query position) to the sums by distance. Each wave half owns an array, in which its
// lanes' places differ, and adds to it in program order; lanes beyond the far ends add to a register instead. So no two adds
// meet whose order is not fixed.
__device__ __forceinline__ void add_by_distance(const f32x16& ds, float* sums, int far, int x0, float& below, float& above) {
#pragma unroll
    for (int quad = 0; quad < 4; ++quad) {
        const int i = x0 + 8 * quad + far + 3;
        if (i >= 0 && i <= 2 * far + 3) {
#pragma unroll
            for (int j = 0; j < 4; ++j) unsafeAtomicAdd(sums + i + j, ds[4 * quad + j]);
        } else {
            const float all = (ds[4 * quad] + ds[4 * quad + 1]) + (ds[4 * quad + 2] + ds[4 * quad + 3]);
            if (i < 0) below += all;
            else above += all;
        }
    }
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int i = 1; i < 64; i *= 2) x += __shfl_xor(x, i);
    return x;
}

// The first distance |x| of bucket j of a side.
__device__ __forceinline__ int bucket_begin(const AttendBias& s, int j) {
    const int exact = s.side / 2;
    return j <= exact ? j : j - exact - 1 < s.edges ? s.edge[j - exact - 1] : s.far + 4;
}

template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(256, 2) void grad_q_kernel(AttendGradArgs g) {
    constexpr int kSteps = DP / 16, kParts = DP / 32;
    const AttendArgs& a = g.a;
    __shared__ s16x8 tile[2][2][kKeyTile * DP / 8];
    extern __shared__ float shared[];  // the bias by distance, then eight arrays of its gradient's sums

    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, hi = lane / 32;
    const int columns = a.tokens * a.pack, column_tiles = (columns + kColumns - 1) / kColumns, groups = a.heads / a.pack;
    int place = xcd_place(blockIdx.x, gridDim.x);
    const int column_tile = place % column_tiles;
    place /= column_tiles;
    const int group = place % groups, b = place / groups;
    const int kv_head = group * a.pack / (a.heads / a.kv_heads);

    const int c = column_tile * kColumns + wave * 32 + lane % 32;
    const int token = c / a.pack, head = group * a.pack + c % a.pack;
    const bool used = c < columns;
    const int64_t row = (static_cast<int64_t>(b) * a.heads + head) * a.tokens + token;
    auto at = [&](const AttendView& v) {
        return used ? static_cast<char*>(v.p) + (b * v.outer + token * v.middle + head * v.head) * 2 : nullptr;
    };
    s16x8 qf[kSteps], df[kSteps];
    float delta = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        qf[i] = column(at(a.q), i, hi, a.d);
        df[i] = column(at(g.d_out), i, hi, a.d);
        const auto x = __builtin_bit_cast(typename E::x8, df[i]);
        const auto y = __builtin_bit_cast(typename E::x8, column(at(a.out), i, hi, a.d));
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(static_cast<float>(x[j]), static_cast<float>(y[j]), delta);
    }
    delta = both_sum(delta);
    if (used && hi == 0) g.delta[row] = delta;
    // rows without a key, and columns past the last: exp(x - inf) = 0
    float2 lse = used ? a.lse[row] : make_float2(-INFINITY, 0.f);
    lse = make_float2(lse.x == -INFINITY ? INFINITY : lse.x, lse.y * -kLog2e);

    const float scale_log2 = a.scale * kLog2e;
    int position = 0;
    float below = 0.f, above = 0.f;
    float* sums = nullptr;
    if constexpr (BIAS) {
        const int places = bias_places(a.bias.far);
        fill_bias<E>(a.bias, head, shared, thread, 256);
        for (int i = thread; i < 8 * places; i += 256) shared[places + i] = 0.f;
        sums = shared + (1 + 2 * wave + hi) * places;
        position = token + a.q_start_all + (a.q_start ? a.q_start[b] : 0);
    }

    f32x16 dq[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) dq[i] = f32x16{};

    KeyWalk walk;
    walk.begin(a, b, 0, 0x7fffffff);
    Copier<DP, kKeyTile, 256> ks, vs;
    ks.init(thread, a.k.middle, a.d);
    vs.init(thread, a.v.middle, a.d);
    auto load = [&] {
        const int valid = walk.count - walk.first;
        ks.load(thread, static_cast<const char*>(a.k.p) + (walk.row * a.k.outer + walk.first * a.k.middle + kv_head * a.k.head) * 2, valid);
        vs.load(thread, static_cast<const char*>(a.v.p) + (walk.row * a.v.outer + walk.first * a.v.middle + kv_head * a.v.head) * 2, valid);
    };
    bool more = walk.valid();
    int now = 0;
    if (more) {
        load();
        ks.store(thread, tile[0][0]);
        vs.store(thread, tile[0][1]);
    }
    __syncthreads();
    while (more) {
        const int first = walk.first, left = walk.count - walk.first;
        walk.next(a);
        more = walk.valid();
        if (more) load();
        bool near = false, wide = false;
        float apart = 0.f;
        if constexpr (BIAS) {
            const int t0 = __builtin_amdgcn_readfirstlane(position), t1 = __builtin_amdgcn_readlane(position, 31);
            near = !far_apart(a.bias, first - t1, first + kKeyTile - 1 - t0);
            if (!near) {
                apart = shared[bias_index(a.bias.far, first - position)];
                wide = __any(fabsf(apart) > kLargeBias);
            }
        }
#pragma unroll
        for (int sub = 0; sub < 2; ++sub) {
            f32x16 s{}, dp{};
#pragma unroll
            for (int i = 0; i < kSteps; ++i) s = E::mfma(straight<DP>(tile[now][0], 32 * sub, i, lane), qf[i], s);
#pragma unroll
            for (int i = 0; i < kSteps; ++i) dp = E::mfma(straight<DP>(tile[now][1], 32 * sub, i, lane), df[i], dp);
            const int x0 = first + 32 * sub + 4 * hi - position;
            if (BIAS && near) {
                add_bias<1>(s, a.scale, shared, a.bias.far, x0);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r] - lse.x, kLog2e, lse.y);
            } else if (BIAS && wide) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(__builtin_fmaf(s[r], a.scale, apart) - lse.x, kLog2e, lse.y);
            } else {
                const float shift = __builtin_fmaf(apart - lse.x, kLog2e, lse.y);
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], scale_log2, shift);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float p = __builtin_amdgcn_exp2f(s[r]);
                if (left < kKeyTile && 32 * sub + row_of(r, hi) >= left) p = 0.f;
                s[r] = p * (dp[r] - delta);
            }
            if constexpr (BIAS) {
                if (near) {
                    add_by_distance(s, sums, a.bias.far, x0, below, above);
                } else {
                    float all = 0.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) all += s[r];
                    if (first < position) below += all;
                    else above += all;
                }
            }
#pragma unroll
            for (int step = 0; step < 2; ++step) {
                const s16x8 x = rounded<E>(s, step);
#pragma unroll
                for (int i = 0; i < kParts; ++i)
                    dq[i] = E::mfma(transposed<DP>(tile[now][0], 32 * sub + 16 * step, i, lane), x, dq[i]);
            }
        }
        if (more) {
            ks.store(thread, tile[now ^ 1][0]);
            vs.store(thread, tile[now ^ 1][1]);
        }
        __syncthreads();
        now ^= 1;
    }

    if (used) {
        char* out = at(g.d_q);
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int quad = 0; quad < 4; ++quad) {
                const int e = 32 * i + row_of(4 * quad, hi);
                if (e < a.d) store_four<typename E::T>(out, e, dq[i], quad, g.scale);
            }
    }
    if constexpr (BIAS) {
        const AttendBias& s = a.bias;
        const int places = bias_places(s.far);
        below = wave_sum(below);
        above = wave_sum(above);
        if (lane == 0) {  // this wave's lower array; its own adds came before
            sums[0] += below;
            sums[places - 1] += above;
        }
        __syncthreads();
        for (int i = thread; i < places; i += 256) {
            float x = 0.f;
            for (int w = 1; w <= 8; ++w) x += shared[w * places + i];
            shared[i] = x;
        }
        __syncthreads();
        for (int bucket = thread; bucket < s.buckets; bucket += 256) {
            const int j = bucket % s.side, from = bucket_begin(s, j), to = j + 1 < s.side ? bucket_begin(s, j + 1) : s.far + 4;
            float x = 0.f;
            if (bucket < s.side) {
                for (int y = from; y < to; ++y) x += shared[s.far + 3 - y];
                if (!s.two_sided && j == 0)
                    for (int y = 1; y <= s.far + 3; ++y) x += shared[s.far + 3 + y];
            } else {
                for (int y = max(from, 1); y < to; ++y) x += shared[s.far + 3 + y];
            }
            g.table_part[((static_cast<int64_t>(b) * column_tiles + column_tile) * a.heads + head) * s.buckets + bucket] = x;
        }
    }
}

// One block: 128 keys of a bank row and key head, each wave 32 of them; walks the request's query tiles, head by head.
template <class E, int DP, bool BIAS>
__global__ __launch_bounds__(256, 1) void grad_kv_kernel(AttendGradArgs g) {
    constexpr int kSteps = DP / 16, kParts = DP / 32, kQueries = 64;
    const AttendArgs& a = g.a;
    __shared__ s16x8 tile[2][2][kQueries * DP / 8];
    // of each query: lse and -what its rounding left off * log2(e); both as one in log2 units, negative; delta
    __shared__ __align__(16) float stat[2][4][kQueries];
    extern __shared__ float bias_held[];

    const int thread = threadIdx.x, lane = thread % 64, wave = thread / 64, hi = lane / 32;
    const int key_tiles = (a.length + kColumns - 1) / kColumns, share = a.heads / a.kv_heads;
    int place = xcd_place(blockIdx.x, gridDim.x);
    const int key_tile = place % key_tiles;
    place /= key_tiles;
    const int kv_head = place % a.kv_heads;
    const int row = place / a.kv_heads, b = row / a.passages;
    const int count = row_length(a, row);
    const int key = key_tile * kColumns + wave * 32 + lane % 32;
    const bool there = key < count;

    f32x16 dk[kParts], dv[kParts];
#pragma unroll
    for (int i = 0; i < kParts; ++i) dk[i] = dv[i] = f32x16{};

    if (key_tile * kColumns < count) {
        s16x8 kf[kSteps], vf[kSteps];
        {
            const char* k = there ? static_cast<const char*>(a.k.p) + (row * a.k.outer + key * a.k.middle + kv_head * a.k.head) * 2 : nullptr;
            const char* v = there ? static_cast<const char*>(a.v.p) + (row * a.v.outer + key * a.v.middle + kv_head * a.v.head) * 2 : nullptr;
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                kf[i] = column(k, i, hi, a.d);
                vf[i] = column(v, i, hi, a.d);
            }
        }
        const float scale_log2 = a.scale * kLog2e;
        const int start = BIAS ? a.q_start_all + (a.q_start ? uniform(a.q_start[b]) : 0) : 0;
        Copier<DP, kQueries, 256> qs, ds;
        qs.init(thread, a.q.middle, a.d);
        ds.init(thread, g.d_out.middle, a.d);
        float2 lse;
        float delta = 0.f;
        int head = kv_head * share, first = 0;
        auto load = [&] {
            const int valid = a.tokens - first;
            qs.load(thread, static_cast<const char*>(a.q.p) + (b * a.q.outer + first * a.q.middle + head * a.q.head) * 2, valid);
            ds.load(thread, static_cast<const char*>(g.d_out.p) + (b * g.d_out.outer + first * g.d_out.middle + head * g.d_out.head) * 2, valid);
            if (thread < kQueries) {
                const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.tokens + first + thread;
                lse = thread < valid ? a.lse[at] : make_float2(-INFINITY, 0.f);
                lse = make_float2(lse.x == -INFINITY ? INFINITY : lse.x, lse.y * -kLog2e);
                delta = thread < valid ? g.delta[at] : 0.f;
            }
        };
        auto store = [&](int to) {
            qs.store(thread, tile[to][0]);
            ds.store(thread, tile[to][1]);
            if (thread < kQueries) {
                stat[to][0][thread] = lse.x;
                stat[to][1][thread] = lse.y;
                stat[to][2][thread] = __builtin_fmaf(lse.x, -kLog2e, lse.y);
                stat[to][3][thread] = delta;
            }
        };
        load();
        if constexpr (BIAS) fill_bias<E>(a.bias, head, bias_held, thread, 256);
        store(0);
        __syncthreads();
        int now = 0;
        bool more = true;
        while (more) {
            const int from = first;
            first += kQueries;
            bool turned = false;
            if (first >= a.tokens) {
                first = 0;
                ++head;
                turned = true;
            }
            more = head < (kv_head + 1) * share;
            if (more) load();
            bool near = false;
            float apart = 0.f;
            bool wide = false;
            if constexpr (BIAS) {
                const int k0 = key_tile * kColumns + wave * 32;
                near = !far_apart(a.bias, k0 - (from + kQueries - 1 + start), k0 + 31 - (from + start));
                if (!near) {
                    apart = bias_held[bias_index(a.bias.far, key - (from + start))];
                    wide = __any(fabsf(apart) > kLargeBias);
                }
            }
#pragma unroll
            for (int sub = 0; sub < 2; ++sub) {
                f32x16 s{}, dp{};
#pragma unroll
                for (int i = 0; i < kSteps; ++i) s = E::mfma(straight<DP>(tile[now][0], 32 * sub, i, lane), kf[i], s);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) dp = E::mfma(straight<DP>(tile[now][1], 32 * sub, i, lane), vf[i], dp);
                if (BIAS && near) {
                    add_bias<-1>(s, a.scale, bias_held, a.bias.far, key - (from + start + 32 * sub + 4 * hi));
                } else if (BIAS && wide) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = __builtin_fmaf(s[r], a.scale, apart);
                }
                const bool added = BIAS && (near || wide);
                const float apart_log2 = apart * kLog2e;
#pragma unroll
                for (int quad = 0; quad < 4; ++quad) {
                    const f32x4 l = *reinterpret_cast<const f32x4*>(&stat[now][0][32 * sub + row_of(4 * quad, hi)]);
                    const f32x4 low = *reinterpret_cast<const f32x4*>(&stat[now][1][32 * sub + row_of(4 * quad, hi)]);
                    const f32x4 one = *reinterpret_cast<const f32x4*>(&stat[now][2][32 * sub + row_of(4 * quad, hi)]);
                    const f32x4 e = *reinterpret_cast<const f32x4*>(&stat[now][3][32 * sub + row_of(4 * quad, hi)]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int r = 4 * quad + j;
                        const float x = added ? __builtin_fmaf(s[r] - l[j], kLog2e, low[j])
                                              : __builtin_fmaf(s[r], scale_log2, BIAS ? apart_log2 + one[j] : one[j]);
                        s[r] = there ? __builtin_amdgcn_exp2f(x) : 0.f;
                        dp[r] = s[r] * (dp[r] - e[j]);
                    }
                }
#pragma unroll
                for (int step = 0; step < 2; ++step) {
                    const s16x8 p = rounded<E>(s, step), x = rounded<E>(dp, step);
#pragma unroll
                    for (int i = 0; i < kParts; ++i) {
                        dv[i] = E::mfma(transposed<DP>(tile[now][1], 32 * sub + 16 * step, i, lane), p, dv[i]);
                        dk[i] = E::mfma(transposed<DP>(tile[now][0], 32 * sub + 16 * step, i, lane), x, dk[i]);
                    }
                }
            }
            if (more) store(now ^ 1);
            if constexpr (BIAS) {
                if (turned && more) {  // another head's bias, once every wave is done with this one's
                    __syncthreads();
                    fill_bias<E>(a.bias, head, bias_held, thread, 256);
                }
            }
            __syncthreads();
            now ^= 1;
        }
    }

    if (key < a.length) {  // keys past the row's length have no gradient: zeros
        char* k = static_cast<char*>(g.d_k.p) + (row * g.d_k.outer + key * g.d_k.middle + kv_head * g.d_k.head) * 2;
        char* v = static_cast<char*>(g.d_v.p) + (row * g.d_v.outer + key * g.d_v.middle + kv_head * g.d_v.head) * 2;
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
            for (int quad = 0; quad < 4; ++quad) {
                const int e = 32 * i + row_of(4 * quad, hi);
                if (e >= a.d) continue;
                const f32x16 zero{};
                store_four<typename E::T>(k, e, there ? dk[i] : zero, quad, g.scale);
                store_four<typename E::T>(v, e, there ? dv[i] : zero, quad, 1.f);
            }
    }
}

template <class E, int DP>
hipError_t launch_grad_q(const AttendGradArgs& g, hipStream_t stream) {
    const AttendArgs& a = g.a;
    const int64_t blocks = (static_cast<int64_t>(a.tokens) * a.pack + kColumns - 1) / kColumns * (a.heads / a.pack) * a.batch;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    const size_t lds = a.bias.table ? 9 * (2 * a.bias.far + 7) * sizeof(float) : 0;
    auto kernel = a.bias.table ? grad_q_kernel<E, DP, true> : grad_q_kernel<E, DP, false>;
    kernel<<<static_cast<unsigned>(blocks), 256, lds, stream>>>(g);
    return hipGetLastError();
}

template <class E, int DP>
hipError_t launch_grad_kv(const AttendGradArgs& g, hipStream_t stream) {
    const AttendArgs& a = g.a;
    const int64_t blocks = static_cast<int64_t>((a.length + kColumns - 1) / kColumns) * a.kv_heads * a.bank;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    const size_t lds = a.bias.table ? (2 * a.bias.far + 7) * sizeof(float) : 0;
    auto kernel = a.bias.table ? grad_kv_kernel<E, DP, true> : grad_kv_kernel<E, DP, false>;
    kernel<<<static_cast<unsigned>(blocks), 256, lds, stream>>>(g);
    return hipGetLastError();
}

}  // namespace vk::attend
