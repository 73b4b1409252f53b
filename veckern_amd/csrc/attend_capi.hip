// C ABI of the attention over found rows (vk_attend, vk_attend_backward): checks, the plan of a call, and its launches.
#include <algorithm>
#include <cmath>
#include <string>

#include "attend.hpp"
#include "errors.hpp"

namespace vk {

#define VK_ATTEND_INSTANCES(type, size)                                              \
    hipError_t attend_forward_##type##_##size(const AttendArgs& a, hipStream_t stream);     \
    hipError_t attend_few_##type##_##size(const AttendArgs& a, hipStream_t stream);         \
    hipError_t attend_grad_q_##type##_##size(const AttendGradArgs& g, hipStream_t stream);  \
    hipError_t attend_grad_kv_##type##_##size(const AttendGradArgs& g, hipStream_t stream);
VK_ATTEND_INSTANCES(bf16, 32)
VK_ATTEND_INSTANCES(bf16, 64)
VK_ATTEND_INSTANCES(bf16, 96)
VK_ATTEND_INSTANCES(bf16, 128)
VK_ATTEND_INSTANCES(f16, 32)
VK_ATTEND_INSTANCES(f16, 64)
VK_ATTEND_INSTANCES(f16, 96)
VK_ATTEND_INSTANCES(f16, 128)

// The instance of the type and of the next of 32, 64, 96 and 128 elements a head; a smaller head in a larger instance costs what
// the larger does. 16 x 512 tokens, 12 heads of 32, 64, 96, 128: forward 20, 26, 39, 45 us, gradients 48, 81, 132, 152; one token
// over 10 x 100 positions for 64 requests: 21, 37, 54, 80 us.
#define VK_ATTEND_PICK(name, type, d)                                                                                     \
    ((type) == kAttendBf16 ? ((d) <= 32 ? name##_bf16_32 : (d) <= 64 ? name##_bf16_64 : (d) <= 96 ? name##_bf16_96 : name##_bf16_128) \
                           : ((d) <= 32 ? name##_f16_32 : (d) <= 64 ? name##_f16_64 : (d) <= 96 ? name##_f16_96 : name##_f16_128))

hipError_t launch_attend_forward(const AttendArgs& a, int type, hipStream_t stream) {
    return VK_ATTEND_PICK(attend_forward, type, a.d)(a, stream);
}
hipError_t launch_attend_few(const AttendArgs& a, int type, hipStream_t stream) {
    return VK_ATTEND_PICK(attend_few, type, a.d)(a, stream);
}
hipError_t launch_attend_grad_q(const AttendGradArgs& g, int type, hipStream_t stream) {
    return VK_ATTEND_PICK(attend_grad_q, type, g.a.d)(g, stream);
}
hipError_t launch_attend_grad_kv(const AttendGradArgs& g, int type, hipStream_t stream) {
    return VK_ATTEND_PICK(attend_grad_kv, type, g.a.d)(g, stream);
}

}  // namespace vk

namespace {

using vk::AttendArgs;
using vk::AttendBias;
using vk::AttendGradArgs;
using vk::AttendView;
using vk::fail;
using vk::guarded;

void valid(bool condition, const char* message) {
    if (!condition) fail(VK_ERR_INVALID_ARGUMENT, message);
}

constexpr size_t kMost = (size_t(1) << 31) - 1;

// The bucket layout of vk_bias_bucket. The edge of bucket e + i is the least x with x >= e (max_distance / e)^(i / (n - e)):
// where that power is a whole number, the logarithms' rounding must not move the edge past it.
AttendBias bias_of(size_t buckets, size_t max_distance, bool two_sided) {
    valid(buckets <= 2 * vk::kMostEdges, "the bias has more than 256 buckets");
    valid(!two_sided || buckets % 2 == 0, "a two-sided bias needs an even number of buckets");
    AttendBias s;
    s.two_sided = two_sided;
    s.buckets = static_cast<int>(buckets);
    s.side = s.buckets / (two_sided ? 2 : 1);
    valid(s.side >= 2, "the bias needs at least two buckets a side");
    const int e = s.side / 2, w = s.side - e;
    valid(max_distance > static_cast<size_t>(e), "max_distance must exceed the buckets of one distance each");
    valid(max_distance <= vk::kMostDistance, "max_distance is more than 1024");
    s.edges = w - 1;
    for (int i = 1; i < w; ++i) {
        const long double x = e * std::pow(static_cast<long double>(max_distance) / e, static_cast<long double>(i) / w);
        const long double whole = std::round(x);
        s.edge[i - 1] = static_cast<int>(std::fabs(x - whole) < 1e-12L * x ? whole : std::ceil(x));
    }
    for (int i = s.edges; i < vk::kMostEdges; ++i) s.edge[i] = INT32_MAX;
    s.far = s.edges ? s.edge[s.edges - 1] : e;
    return s;
}

struct Dim {
    size_t outer, middle, head;
};

AttendView view_of(const vk_tensor& t, const Dim& size, const char* name) {
    const std::string n = name;
    const bool none = size.outer == 0 || size.middle == 0 || size.head == 0;
    AttendView v;
    v.p = t.data;
    const size_t sizes[3] = {size.outer, size.middle, size.head};
    int64_t stride[3];
    for (int i = 0; i < 3; ++i) {
        stride[i] = sizes[i] > 1 ? t.stride[i] : 0;
        if (stride[i] < 0 || stride[i] % 8) fail(VK_ERR_INVALID_ARGUMENT, n + ": strides must be multiples of 8 elements and not negative");
    }
    // a tile's rows are reached by 32-bit offsets
    if (stride[1] >= (int64_t(1) << 23)) fail(VK_ERR_INVALID_ARGUMENT, n + ": the stride between positions is 2^23 elements or more");
    if (!none && !t.data) fail(VK_ERR_INVALID_ARGUMENT, n + " is NULL");
    if (reinterpret_cast<uintptr_t>(t.data) % 16) fail(VK_ERR_INVALID_ARGUMENT, n + " is not 16-byte aligned");
    v.outer = stride[0];
    v.middle = stride[1];
    v.head = stride[2];
    return v;
}

// Checks a call's arguments; `out` only where the call has it.
AttendArgs args_of(const vk_attention* x, bool tensors) {
    valid(x != nullptr, "arguments are NULL");
    valid(x->type == VK_F16 || x->type == VK_BF16, "type must be VK_F16 or VK_BF16");
    valid(x->head_dim >= 8 && x->head_dim <= 128 && x->head_dim % 8 == 0, "head_dim must be a multiple of 8 and at most 128");
    valid(x->heads > 0 && x->kv_heads > 0 && x->heads % x->kv_heads == 0, "heads must be a multiple of kv_heads");
    valid(x->batch <= kMost && x->tokens <= kMost && x->passages <= kMost && x->length <= kMost && x->bank <= kMost && x->heads <= 65536,
          "a size is too large");
    valid(x->tokens * x->heads <= kMost / 2 && (x->length + vk::kSlot) / vk::kSlot * x->passages <= kMost / 16 &&
              x->length <= kMost / 2, "a size is too large");
    valid(std::isfinite(x->scale) && x->scale >= 0.f, "scale must be finite and not negative");
    valid(x->rows || x->bank == x->batch * x->passages, "without rows, bank must be batch * passages");
    valid(x->q_start > -(int64_t(1) << 30) && x->q_start < (int64_t(1) << 30), "q_start is out of range");
    AttendArgs a;
    a.batch = static_cast<int>(x->batch);
    a.tokens = static_cast<int>(x->tokens);
    a.heads = static_cast<int>(x->heads);
    a.kv_heads = static_cast<int>(x->kv_heads);
    a.d = static_cast<int>(x->head_dim);
    a.passages = static_cast<int>(x->passages);
    a.length = static_cast<int>(x->length);
    a.bank = static_cast<int64_t>(x->bank);
    a.scale = std::max(x->scale, 1e-37f);
    a.rows = x->rows;
    a.rows_outer = x->rows_stride[0];
    a.rows_step = x->rows_stride[1];
    a.lengths = x->lengths;
    a.q_start = x->q_starts;
    a.q_start_all = static_cast<int>(x->q_start);
    a.lse = reinterpret_cast<float2*>(x->lse);
    valid(reinterpret_cast<uintptr_t>(x->lse) % 8 == 0, "lse is not 8-byte aligned");
    if (x->table) {
        // its powers take microseconds: the thread's last layout is kept, by its three numbers
        static thread_local struct {
            size_t buckets = 0, max_distance = 0;
            bool two_sided = false;
            AttendBias bias;
        } last;
        if (last.buckets != x->buckets || last.max_distance != x->max_distance || last.two_sided != (x->two_sided != 0)) {
            last.bias = bias_of(x->buckets, x->max_distance, x->two_sided != 0);
            last.buckets = x->buckets;
            last.max_distance = x->max_distance;
            last.two_sided = x->two_sided != 0;
        }
        a.bias = last.bias;
        a.bias.table = x->table;
        a.bias.bucket_stride = x->table_stride[0];
        a.bias.head_stride = x->table_stride[1];
        valid(a.bias.bucket_stride >= 0 && a.bias.head_stride >= 0, "the bias table's strides must not be negative");
    }
    if (tensors) {
        const Dim q{x->batch, x->tokens, x->heads}, k{x->bank, x->length, x->kv_heads};
        a.q = view_of(x->q, q, "q");
        a.out = view_of(x->out, q, "out");
        a.k = view_of(x->k, k, "k");
        a.v = view_of(x->v, k, "v");
    }
    return a;
}

// Whether a call has so few columns for each key head that its time is the reading of the states. 64 requests over 10 x 100
// positions, 12 heads, by the kernel for few columns and by tiles: 32 columns of 64 elements 38 and 50 us, of 128 87 and 92; 64
// columns 51 and 49, 122 and 93.
bool few_columns(const AttendArgs& a) { return static_cast<int64_t>(a.tokens) * a.pack <= 32; }

// How long blocks of a kernel take, in microseconds as measured on this card: `start` for a block's first loads and its end,
// `tile` for each of its tiles where a compute unit has one block, and `shared` of that more for each further block.
struct Pace {
    int resident;  // blocks that a compute unit holds at once
    double start, tile, shared;
};

// Into how many runs of whole tiles, for different blocks, an axis of `tiles` tiles is split where that makes a call shorter: the
// runs' parts are joined by another launch (5 us) that reads what the runs wrote in 32 bits (part_bytes a run, both ways, at
// 3.5 TB/s). `blocks`: of one run; at_a_time: tiles that a block takes at once. At the pace of the tile kernel one split of 256
// blocks over 80 tiles of 64 elements a head took 107 us, two 75 + 6 and three, which fill the card, 63 + 7; of 18 blocks over 15
// tiles of 128, one 26 us, five 12 + 4 and fifteen 12 + 7.
int best_splits(int tiles, int least, int64_t blocks, const Pace& pace, int at_a_time, double part_bytes) {
    double best = 0;
    int splits = 1;
    for (int s = least; s <= std::max(least, std::min(tiles, 64)); ++s) {
        const int each = (tiles + s - 1) / s;
        if (s > least && (tiles + each - 1) / each != s) continue;
        const int64_t all = blocks * s, beside = std::max<int64_t>(1, std::min<int64_t>(pace.resident, (all + vk::kUnits - 1) / vk::kUnits));
        const double rounds = static_cast<double>((all + vk::kUnits * beside - 1) / (vk::kUnits * beside));
        const double time = rounds * (pace.start + (each + at_a_time - 1) / at_a_time * pace.tile * (1 + pace.shared * (beside - 1))) +
                            (s > 1 ? 5 + s * part_bytes / 3.5e6 : 0);
        if (s == least || time < best) {
            best = time;
            splits = each ? (tiles + each - 1) / each : 1;
        }
    }
    return splits;
}
void split_keys(AttendArgs& a, int keys, int64_t blocks, const Pace& pace, int at_a_time) {
    const int per_row = (a.length + vk::kSlot - 1) / vk::kSlot, per_tile = keys / vk::kSlot;
    const int tiles = static_cast<int>((static_cast<int64_t>(per_row) * a.passages + per_tile - 1) / per_tile);
    // a block holds the rows of kHeldPassages passages, and a run touches one more than it fills
    const int64_t most_tiles = std::max<int64_t>(1, static_cast<int64_t>(vk::kHeldPassages - 1) * per_row / per_tile);
    const int least = static_cast<int>(std::max<int64_t>(1, (tiles + most_tiles - 1) / most_tiles));
    a.splits = best_splits(tiles, least, blocks, pace, at_a_time, 8.0 * a.batch * a.heads * a.tokens * a.d);
    a.tiles_per_split = (tiles + a.splits - 1) / a.splits;
}

void plan_forward(AttendArgs& a) {
    const int share = a.heads / a.kv_heads;
    a.pack = share;
    if (a.bias.table && static_cast<size_t>(share) * (2 * a.bias.far + 2 * vk::kPad + 1) * sizeof(float) > vk::kMostBiasBytes) a.pack = 1;
    const int64_t columns = static_cast<int64_t>(a.tokens) * a.pack, rest = static_cast<int64_t>(a.heads / a.pack) * a.batch;
    const bool small = a.d <= 64;
    if (few_columns(a)) {
        split_keys(a, vk::kFewKeys, rest, small ? Pace{2, 6.5, 0.8, 0.5} : Pace{1, 6.5, 2, 0}, vk::kFewWaves);
    } else {
        split_keys(a, vk::kKeyTile, (columns + vk::kColumns - 1) / vk::kColumns * rest,
                   small ? Pace{3, 6, 1.27, 0.34} : Pace{2, 6, 1.33, 0.66}, 1);
    }
}
void plan_backward(AttendGradArgs& g) {
    AttendArgs& a = g.a;
    a.pack = a.bias.table ? 1 : a.heads / a.kv_heads;
    const int64_t columns = static_cast<int64_t>(a.tokens) * a.pack, rest = static_cast<int64_t>(a.heads / a.pack) * a.batch;
    split_keys(a, vk::grad_keys(a.d), (columns + vk::kColumns - 1) / vk::kColumns * rest,
               a.d <= 64 ? Pace{2, 10, 1.6, 0.5} : Pace{2, 10, 1.1, 0.5}, 1);
    if (a.rows) return;  // no gradient of the states
    const int queries = vk::grad_queries(a.d), tiles = (a.tokens + queries - 1) / queries * (a.heads / a.kv_heads);
    const int64_t slots = static_cast<int64_t>((a.length + vk::kSlot - 1) / vk::kSlot) * a.passages, per_block = vk::kColumns / vk::kSlot;
    g.kv_splits = best_splits(tiles, 1, (slots + per_block - 1) / per_block * a.kv_heads * a.batch,
                              a.d <= 64 ? Pace{2, 10, 1.4, 0.4} : Pace{1, 10, 1.25, 0}, 1,
                              16.0 * a.batch * a.passages * a.length * a.kv_heads * a.d);
    g.kv_tiles_per_split = (tiles + g.kv_splits - 1) / g.kv_splits;
}
size_t query_rows(const AttendArgs& a) { return static_cast<size_t>(a.batch) * a.heads * a.tokens; }
size_t align(size_t x) { return (x + 15) / 16 * 16; }
size_t part_bytes(const AttendArgs& a) { return a.splits == 1 ? 0 : align(a.splits * query_rows(a) * a.d * sizeof(float)); }
size_t forward_bytes(const AttendArgs& a) {
    return a.splits == 1 ? 0 : part_bytes(a) + a.splits * query_rows(a) * sizeof(float2);
}
int table_parts(const AttendArgs& a) { return (a.tokens + vk::kColumns - 1) / vk::kColumns * a.batch * a.splits; }
size_t table_bytes(const AttendArgs& a) {
    return a.bias.table ? align(static_cast<size_t>(table_parts(a)) * a.heads * a.bias.buckets * sizeof(float)) : 0;
}
size_t delta_bytes(const AttendArgs& a) { return align(query_rows(a) * sizeof(float)); }
size_t backward_bytes(const AttendGradArgs& g) {
    const AttendArgs& a = g.a;
    const size_t states = static_cast<size_t>(a.bank) * a.length * a.kv_heads;
    return delta_bytes(a) + table_bytes(a) + part_bytes(a) + (g.kv_splits == 1 ? 0 : 2 * g.kv_splits * states * a.d * sizeof(float));
}

void check_workspace(void* workspace, size_t bytes, size_t needed) {
    valid(bytes >= needed && (workspace || !needed), "the workspace is too small");
    valid(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace is not 16-byte aligned");
}

}  // namespace

VK_EXPORT int vk_bias_bucket(int64_t distance, size_t buckets, size_t max_distance, int two_sided, int* bucket) {
    return guarded([&] {
        valid(bucket != nullptr, "bucket is NULL");
        const AttendBias s = bias_of(buckets, max_distance, two_sided != 0);
        const int64_t far = s.far;
        const int x = static_cast<int>(std::min(std::max(distance, -far), far));
        const int a = two_sided ? std::abs(x) : std::max(-x, 0), e = s.side / 2;
        int b = a;
        if (a >= e) {
            b = e;
            for (int i = 0; i < s.edges; ++i) b += s.edge[i] <= a;
        }
        *bucket = b + (two_sided && distance > 0 ? s.side : 0);
    });
}

VK_EXPORT int vk_attend_workspace(const vk_attention* x, size_t* bytes) {
    return guarded([&] {
        valid(bytes != nullptr, "bytes is NULL");
        AttendArgs a = args_of(x, false);
        plan_forward(a);
        *bytes = forward_bytes(a);
    });
}

VK_EXPORT int vk_attend(const vk_attention* x, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        AttendArgs a = args_of(x, true);
        plan_forward(a);
        check_workspace(workspace, workspace_bytes, forward_bytes(a));
        if (!query_rows(a)) return;
        if (a.splits > 1) {
            a.part = static_cast<float*>(workspace);
            a.stat = reinterpret_cast<float2*>(static_cast<char*>(workspace) + part_bytes(a));
        }
        const auto on = static_cast<hipStream_t>(stream);
        VK_HIP(few_columns(a) ? vk::launch_attend_few(a, x->type, on) : vk::launch_attend_forward(a, x->type, on));
        if (a.splits > 1) VK_HIP(vk::launch_attend_combine(a, x->type, on));
    });
}

VK_EXPORT int vk_attend_backward_workspace(const vk_attention* x, size_t* bytes) {
    return guarded([&] {
        valid(bytes != nullptr, "bytes is NULL");
        AttendGradArgs g;
        g.a = args_of(x, false);
        plan_backward(g);
        *bytes = backward_bytes(g);
    });
}

VK_EXPORT int vk_attend_backward(const vk_attention* x, const vk_attention_grad* y, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    return guarded([&] {
        valid(y != nullptr, "gradients are NULL");
        AttendGradArgs g;
        g.a = args_of(x, true);
        AttendArgs& a = g.a;
        const Dim q{x->batch, x->tokens, x->heads}, k{x->bank, x->length, x->kv_heads};
        g.d_out = view_of(y->d_out, q, "d_out");
        g.d_q = view_of(y->d_q, q, "d_q");
        if (x->rows) {
            valid(!y->d_k.data && !y->d_v.data, "rows of a bank are constants: d_k and d_v must be NULL where rows is given");
        } else {
            g.d_k = view_of(y->d_k, k, "d_k");
            g.d_v = view_of(y->d_v, k, "d_v");
        }
        valid(!query_rows(a) || a.lse, "lse is NULL");
        valid(!a.bias.table || y->d_table, "d_table is NULL");
        valid(a.bias.table || !y->d_table, "d_table is given without a table");
        g.d_table = y->d_table;
        g.scale = x->scale;
        plan_backward(g);
        check_workspace(workspace, workspace_bytes, backward_bytes(g));
        char* at = static_cast<char*>(workspace);
        g.delta = reinterpret_cast<float*>(at);
        g.table_part = reinterpret_cast<float*>(at + delta_bytes(a));
        a.part = reinterpret_cast<float*>(at + delta_bytes(a) + table_bytes(a));
        g.kv_part = reinterpret_cast<float*>(at + delta_bytes(a) + table_bytes(a) + part_bytes(a));
        const auto on = static_cast<hipStream_t>(stream);
        const int64_t join_q = a.splits > 1 ? static_cast<int64_t>((query_rows(a) * (a.d / 4) + 255) / 256) : 0;
        valid(join_q < vk::kMostBlocks, "a size is too large");
        g.join_q = static_cast<int>(join_q);
        g.join_table = a.bias.table ? (a.heads * a.bias.buckets + 3) / 4 : 0;
        g.table_parts = table_parts(a);
        const bool states = !x->rows && x->bank && x->length;
        if (query_rows(a)) VK_HIP(vk::launch_attend_grad_q(g, x->type, on));
        if (states) VK_HIP(vk::launch_attend_grad_kv(g, x->type, on));
        VK_HIP(vk::launch_attend_grad_join(g, x->type, !states, on));
    });
}
