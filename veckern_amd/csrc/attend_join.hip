// What follows the attention kernels where their work was split: the joined softmax of the splits of a row, the gradients'
// parts, and the bias table's gradient from the blocks' sums, if no block of the keys' gradient has joined that (join_queries in
// attend_tile.hpp). All sum in a fixed order. They read their input once: 4 to 5 us where
// that is little (a launch and two loads that follow each other), 7 us for three splits of 4 x 512 tokens, 16 heads of 64 (29 MB,
// 4.1 TB/s), 20 us for three runs of d_k and d_v of 12 x 213 states, 12 heads of 128 (94 MB).
#include "attend_tile.hpp"

namespace vk {
namespace attend {

// out = sum of exp(top_i - top) part_i / sum of exp(top_i - top) total_i over the splits i; a thread takes four elements of a row.
template <class E>
__global__ __launch_bounds__(256) void combine_kernel(AttendArgs a) {
    const int groups = a.heads / a.pack, columns = a.tokens * a.pack, quads = a.d / 4;
    const int64_t rows = static_cast<int64_t>(a.batch) * groups * columns, at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (at >= rows * quads) return;
    const int64_t row = at / quads;
    const int e = static_cast<int>(at - row * quads) * 4;
    float top = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) top = fmaxf(top, a.stat[i * rows + row].x);
    const float base = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    f32x4 x{};
#pragma unroll 4
    for (int i = 0; i < a.splits; ++i) {
        const float2 s = a.stat[i * rows + row];
        const float w = __builtin_amdgcn_exp2f((s.x - base) * kLog2e);
        total = __builtin_fmaf(w, s.y, total);
        x += w * *reinterpret_cast<const f32x4*>(a.part + (i * rows + row) * a.d + e);
    }
    const int c = row % columns, group = row / columns % groups, b = row / columns / groups;
    const int token = c / a.pack, head = group * a.pack + c % a.pack;
    const float factor = total == 0.f ? 0.f : 1.f / total;
    typename E::T z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = (typename E::T)(x[j] * factor);
    char* out = static_cast<char*>(a.out.p) + (b * a.out.outer + token * a.out.middle + head * a.out.head + e) * 2;
    *reinterpret_cast<u32x2*>(out) = *reinterpret_cast<u32x2*>(z);
    if (a.lse && e == 0) a.lse[(static_cast<int64_t>(b) * a.heads + head) * a.tokens + token] = logarithm(top, total);
}

// The first `joined` blocks: d_q and the table; the others: d_k and d_v alike, four elements a thread.
template <class E>
__global__ __launch_bounds__(256) void grad_join_kernel(AttendGradArgs g, int joined) {
    const AttendArgs& a = g.a;
    if (static_cast<int>(blockIdx.x) < joined) {
        join_queries<E>(g, blockIdx.x, threadIdx.x);
        return;
    }
    const int quads = a.d / 4;
    const int64_t states = a.bank * a.length * a.kv_heads, at = static_cast<int64_t>(blockIdx.x - joined) * 256 + threadIdx.x;
    if (at >= 2 * states * quads) return;
    const bool value = at >= states * quads;
    const int64_t state = at / quads - (value ? states : 0);
    const int e = static_cast<int>(at % quads) * 4;
    const float* part = g.kv_part + ((value ? g.kv_splits * states : 0) + state) * a.d + e;
    f32x4 x{};
#pragma unroll 4
    for (int i = 0; i < g.kv_splits; ++i) x += *reinterpret_cast<const f32x4*>(part + i * states * a.d);
    const int kv_head = state % a.kv_heads, key = state / a.kv_heads % a.length;
    const int64_t row = state / a.kv_heads / a.length;
    const AttendView& v = value ? g.d_v : g.d_k;
    typename E::T z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = (typename E::T)(x[j] * (value ? 1.f : g.scale));
    char* out = static_cast<char*>(v.p) + (row * v.outer + key * v.middle + kv_head * v.head + e) * 2;
    *reinterpret_cast<u32x2*>(out) = *reinterpret_cast<u32x2*>(z);
}

}  // namespace attend

hipError_t launch_attend_combine(const AttendArgs& a, int type, hipStream_t stream) {
    const int64_t blocks = (static_cast<int64_t>(a.batch) * a.heads * a.tokens * (a.d / 4) + 255) / 256;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    auto kernel = type == kAttendBf16 ? attend::combine_kernel<attend::Bf16> : attend::combine_kernel<attend::F16>;
    kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(a);
    return hipGetLastError();
}

hipError_t launch_attend_grad_join(const AttendGradArgs& g, int type, bool queries, hipStream_t stream) {
    const AttendArgs& a = g.a;
    const int joined = queries ? g.join_q + g.join_table : 0;
    const int64_t keys = g.kv_splits > 1 ? (2 * a.bank * a.length * a.kv_heads * (a.d / 4) + 255) / 256 : 0, blocks = joined + keys;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    if (!blocks) return hipSuccess;
    auto kernel = type == kAttendBf16 ? attend::grad_join_kernel<attend::Bf16> : attend::grad_join_kernel<attend::F16>;
    kernel<<<static_cast<unsigned>(blocks), 256, 0, stream>>>(g, joined);
    return hipGetLastError();
}

}  // namespace vk
