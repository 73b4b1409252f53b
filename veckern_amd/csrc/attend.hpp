// Attention over rows of encoder states: arguments and launches shared by the C ABI (attend_capi.hip) and the kernels
// (attend_forward*.hip, attend_backward*.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace vk {

constexpr int kMostEdges = 128;      // bucket edges of a one-sided bias of 256 buckets
constexpr int kMostDistance = 1024;  // largest max_distance: the bias by distance, and its gradient, are held in LDS
constexpr int kPad = 15;             // places at either end of the bias by distance (attend_tile.hpp)
constexpr int kMostBiasBytes = 16384;  // biases by distance of the heads that share a block's columns; else a head alone
constexpr int kSlot = 16;            // keys of a passage that stand together in a tile
constexpr int kKeyTile = 64;         // keys that a block of the tile kernels holds at once
constexpr int kFewWaves = 8, kFewKeys = 32;  // waves of a block of the few-columns kernel, keys of its tiles
constexpr int kHeldPassages = 256;   // passages that a block holds the rows of
constexpr int grad_keys(int d) { return d <= 64 ? 64 : 32; }  // keys of a tile of the query gradient
constexpr int grad_queries(int d) { return d <= 64 ? 64 : 32; }  // queries of a tile of the keys' and values' gradient
constexpr int kColumns = 128;        // query columns of a block of the tile kernels
constexpr int kUnits = 256;          // compute units of the card
constexpr int kMostBlocks = (1 << 30) - 1;  // of a grid that xcd_place() orders, which doubles the size of a group of blocks

// A tensor [outer][middle][head][d]: element strides, d contiguous.
struct AttendView {
    void* p = nullptr;
    int64_t outer = 0, middle = 0, head = 0;
};

// Position bias by buckets. The distance x = key position - query position falls into the bucket
//   (two-sided and x > 0 ? side : 0) + (a < side / 2 ? a : side / 2 + (number of edges <= a)),   a = |x| or max(-x, 0).
struct AttendBias {
    const void* table = nullptr;  // [buckets][heads], of the queries' type; nullptr: no bias
    int64_t bucket_stride = 0, head_stride = 0;
    int buckets = 0, side = 0, edges = 0;
    int far = 0;  // from this distance on, and beyond, the last bucket of a side
    bool two_sided = false;
    int edge[kMostEdges];
};

struct AttendArgs {
    AttendView q, k, v, out;      // q, out: [batch][tokens][heads][d]; k, v: [bank][length][kv_heads][d]
    float2* lse = nullptr;        // [batch][heads][tokens] (value, what its rounding left off); may be nullptr in the forward pass
    const int32_t* rows = nullptr;  // [batch][passages] by rows_outer, rows_step; nullptr: b * passages + r
    int64_t rows_outer = 0, rows_step = 0;
    const int32_t* lengths = nullptr;   // [bank]; nullptr: all `length`
    const int32_t* q_start = nullptr;   // [batch], added to q_start_all
    int q_start_all = 0;
    int batch = 0, tokens = 0, heads = 0, kv_heads = 0, d = 0, passages = 0, length = 0;
    int64_t bank = 0;
    float scale = 0.f;            // positive, so that -inf * scale is -inf (0 is taken as 1e-37)
    AttendBias bias;
    // How the work is laid out. pack: query heads of one key head that share a block's columns (column = token * pack + head).
    // splits: runs of the keys that different blocks take, each of tiles_per_split tiles.
    int pack = 1, splits = 1, tiles_per_split = 0;
    float* part = nullptr;   // splits > 1: [splits][batch][heads / pack][tokens * pack][d] unnormalised sums ... (d_q's parts alike)
    float2* stat = nullptr;  // ... and [splits][...][tokens * pack] (maximum, sum)
};

struct AttendGradArgs {
    AttendArgs a;                 // out: the forward's result, lse: its statistics
    AttendView d_out, d_q, d_k, d_v;
    float scale = 0.f;            // the logits' own, which may be 0
    float* delta = nullptr;       // workspace [batch][heads][tokens]
    float* table_part = nullptr;  // workspace [splits * batch * column tiles][heads][buckets]
    void* d_table = nullptr;      // [buckets][heads], contiguous
    // Runs of a key head's query tiles (head by head) that different blocks take for d_k and d_v.
    int kv_splits = 1, kv_tiles_per_split = 0;
    // Blocks of 256 threads that join d_q's parts and the table's partial sums, of which there are table_parts: those of d_q first.
    // They stand behind the blocks of the keys' gradient, which waits for what they need anyway, or, for rows of a bank, in a launch
    // of their own (3 requests of 77 tokens over 5 x 131, 6 heads of 80, bias, forward and backward: 51 us with that launch, 47 so).
    int join_q = 0, join_table = 0, table_parts = 0;
    float* kv_part = nullptr;     // kv_splits > 1: workspace [d_k, d_v][kv_splits][bank][length][kv_heads][d]
};

enum AttendType { kAttendF16 = 0, kAttendBf16 = 1 };

hipError_t launch_attend_forward(const AttendArgs& a, int type, hipStream_t stream);
hipError_t launch_attend_few(const AttendArgs& a, int type, hipStream_t stream);
hipError_t launch_attend_combine(const AttendArgs& a, int type, hipStream_t stream);
// Writes d_q, or its parts, delta and the table's partial sums.
hipError_t launch_attend_grad_q(const AttendGradArgs& g, int type, hipStream_t stream);
hipError_t launch_attend_grad_kv(const AttendGradArgs& g, int type, hipStream_t stream);
// Joins d_q's parts and the table's sums if `queries`, and the parts of d_k and d_v if there are any.
hipError_t launch_attend_grad_join(const AttendGradArgs& g, int type, bool queries, hipStream_t stream);

}  // namespace vk
