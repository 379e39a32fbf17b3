// Rules of the training operators that are arithmetic on sizes alone: plain C++, so that a test can hold them
// against what the kernels behind them assume, without a GPU.
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace cti {

constexpr int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// n / d for n < 2^31 by one multiplication (Granlund and Montgomery, 1994): m = floor(2^(31 + s) / d) + 1 with
// s = ceil(log2 d) is off by at most d <= 2^s, so n times that stays below 2^(31 + s).
struct ChunkDivide {
  uint32_t m, shift;
  static constexpr ChunkDivide by(uint32_t d) {
    uint32_t s = 0;
    while (s < 32 && (uint64_t{1} << s) < d) ++s;
    return {static_cast<uint32_t>((uint64_t{1} << (31 + s)) / d + 1), 31 + s};
  }
  constexpr uint32_t quotient(uint32_t n) const { return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> shift); }
};

// Where the 8 columns of the chunk at column c of a row of `cols` (8 or more) begin in the lookup: the row's last 8 for a chunk that
// would end behind it. (Nothing is added to c, which comes close to 2^31 in the widest rows.)
constexpr int chunk_start(int c, int cols) { return c <= cols - 8 ? c : cols - 8; }

constexpr int64_t kMostChunks = int64_t{1} << 30;  // of 8 columns, a launch

constexpr int kGradTile = 4096;
constexpr int64_t kGradMostIds = int64_t{1} << 30;        // ids and bags: 32-bit numbers, and launches below 2^32 threads
constexpr int64_t kGradMostRows = (int64_t{1} << 31) - 1;  // rows of all tables are fewer: the number itself is a key
constexpr int64_t kGradMostDim = int64_t{1} << 22;
constexpr int64_t kGradFillShare = 64 << 10;  // bytes that a workgroup fills
// Shares of the fill that one launch of the sort may take beside its own workgroups and stay below 2^32 threads: launches of 1,024
// threads have 256 workgroups at most (one, a range of keys each, or 64 digits each), launches of 512 one for each tile.
constexpr int64_t kGradMostShares = (int64_t{1} << 22) - 512;
constexpr int kGradDigitBits = 11, kGradDigits = 1 << kGradDigitBits;
constexpr int64_t kGradIdsAlone = 8192;    // in bags: ids that one workgroup finds and sorts
constexpr int64_t kGradIdsRanged = 32768;  // ids that are sorted by ranges of keys
constexpr int kGradPositionBits = 15, kGradKeyBits = 32 - kGradPositionBits;  // ids that one workgroup sorts
constexpr int64_t kGradTilesUnscanned = 16;
constexpr int64_t kGradHeadsUnscanned = 4096;

constexpr int kGradWalkCols = 64;  // narrower rows would leave most of a wavefront idle

struct GradPlan {
  int64_t tiles;
  int bits, digit_bits;
  bool walk;      // a wavefront for each run of ids, else lane groups
  int lane_cols;  // columns a lane
  int log_lanes, run, blocks;  // lanes of a group, ids of a group, blocks of 64 lanes' columns
  int64_t workgroups;
  int64_t ids[2], counts, totals, heads, last_rank, inv_len, partial, bytes;  // places in the workspace
};

// The gradient of n ids in tables of `rows` rows, the widest of `dim` columns; mean_bags: bags under mean pooling, else 0;
// even: all rows of grad have `dim` columns and lie one behind the other.
inline GradPlan grad_plan(int64_t n, int64_t mean_bags, int64_t dim, int elem_bytes, uint32_t rows, bool even) {
  GradPlan p{};
  p.tiles = ceil_div(n, kGradTile);
  while (p.bits < 32 && (rows >> p.bits)) ++p.bits;  // of the key `rows` itself
  const int passes = (p.bits + kGradDigitBits - 1) / kGradDigitBits;
  p.digit_bits = (p.bits + passes - 1) / passes;
  if (p.digit_bits < 2) p.digit_bits = 2;  // a thread holds four digits
  const int vec = 16 / elem_bytes;
  p.walk = even && dim >= kGradWalkCols;
  if (p.walk) {
    p.log_lanes = 6;
    p.lane_cols = 1;
    while (p.lane_cols < vec && 64 * p.lane_cols < dim) p.lane_cols *= 2;
    p.blocks = static_cast<int>(ceil_div(dim, 64 * p.lane_cols));
    // enough wavefronts to fill the card, ids enough for each to keep its loads in flight
    p.run = 128;
    while (p.run > 16 && ceil_div(n, p.run) * p.blocks < 4096) p.run /= 2;
  } else {
    p.lane_cols = vec;
    const int64_t vectors = ceil_div(dim, vec);
    while (p.log_lanes < 6 && (int64_t{1} << p.log_lanes) < vectors) ++p.log_lanes;
    p.blocks = static_cast<int>(ceil_div(vectors, 64));
    const int groups = 256 >> p.log_lanes;
    p.run = 2048 / groups < 32 ? 2048 / groups : 32;
    if (ceil_div(n, int64_t{groups} * p.run) * p.blocks < 1024) p.run = 8;
  }
  p.workgroups = ceil_div(n, int64_t{256 >> p.log_lanes} * p.run);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += ceil_div(bytes, 256) * 256;
    return here;
  };
  for (int i = 0; i < 2; ++i) p.ids[i] = take(n * 8);
  p.counts = take((p.tiles << p.digit_bits) * 4);
  p.totals = take(kGradDigits * 4);
  p.heads = take((p.workgroups + 1) * 4);
  p.last_rank = take(p.workgroups * 4);
  p.inv_len = take(mean_bags * 4);
  p.partial = take(p.workgroups * p.blocks * 2 * (int64_t{p.lane_cols} << p.log_lanes) * 4);
  p.bytes = at;
  return p;
}

// Bits of the ranges of keys by which n ids of `bits` bits are sorted in one launch, a workgroup for each range: 64 ranges (of
// 16,384 tokens 256 each), fewer where that leaves less than 64 ids each, and as many as leave a key its 17 bits next to a
// position. 0: by digits, in tiles.
inline int grad_range_bits(int64_t n, int bits) {
  if (n > kGradIdsRanged) return 0;
  int r = 6;
  while (r > 1 && (n >> r) < 64) --r;
  if (bits - r > kGradKeyBits) r = bits - kGradKeyBits;
  if (r >= bits) r = bits - 1;
  return r < 1 || r > 8 ? 0 : r;
}

// Bytes that every form of a gradient of these sizes fits in.
inline int64_t grad_workspace_bytes(int64_t n, int64_t mean_bags, int64_t dim, uint32_t rows) {
  int64_t most = 0;
  for (const int elem_bytes : {2, 4})
    for (const bool even : {false, true}) {
      const int64_t bytes = grad_plan(n, mean_bags, dim, elem_bytes, rows, even).bytes;
      most = bytes > most ? bytes : most;
    }
  return most;
}

// The register form of the norm with dropout: `lanes` threads hold a row, `chunks` chunks of 8 columns each (1, 2 or 4);
// lanes 0: the loop form. Measured (us): 4,096 columns by 256 threads of two chunks | 512 of one: 16,384 rows bf16 97.7 | 98.8,
// fp32 211 | 199; 65,536 rows of 1,021 by 64 threads of two | 128 of one: bf16 113 | 112, fp32 238 | 223.
struct TrainNormForm {
  int lanes, chunks;
};
inline TrainNormForm train_norm_form(int64_t cols, int elem_bytes) {
  const int64_t n = ceil_div(cols, 8);
  for (const int lanes : {8, 16, 32, 64})
    if (n <= lanes) return {lanes, 1};
  if (n <= 128) return {128, 1};
  if (n <= 256) return {256, 1};
  if (n <= 512) return elem_bytes == 4 ? TrainNormForm{512, 1} : TrainNormForm{256, 2};
  if (n <= 1024) return {512, 2};
  if (n <= 2048) return {512, 4};
  return {0, 0};
}
// The backward pass holds three arrays' chunks, the parameters' gradients and the next row's loads: one chunk a thread
// as far as 512 threads go (112 registers, four wavefronts a SIMD; 4,096 columns by 256 threads of two chunks take 187, two
// wavefronts: no faster), then two, then two of 1,024 threads with the gradients in LDS (2 x 16,384 fp32 numbers; in
// registers they spill: 4,096 rows of 14,336 bf16 164 us).
inline TrainNormForm train_norm_back_form(int64_t cols) {
  const int64_t n = ceil_div(cols, 8);
  for (const int lanes : {8, 16, 32, 64, 128, 256, 512})
    if (n <= lanes) return {lanes, 1};
  if (n <= 1024) return {512, 2};
  if (n <= 2048) return {1024, 2};
  return {0, 0};
}
// Workgroups of the backward pass: as many as are resident (each adds up gamma's and beta's gradients over its rows).
inline int64_t train_norm_workgroups(int64_t rows, int64_t cols) {
  const TrainNormForm f = train_norm_back_form(cols);
  const int64_t side = f.lanes > 0 && f.lanes < 256 ? 256 / f.lanes : 1;  // rows side by side
  // (wider rows: workgroups for each 2,048 columns, four a CU in all)
  const int64_t most = f.lanes == 0 ? ceil_div(1024, ceil_div(cols, 2048)) : f.lanes < 512 ? 1024 : f.chunks == 1 ? 512 : 256;
  const int64_t n = ceil_div(rows, side);
  return n < 1 ? 0 : ceil_div(n, ceil_div(n, most));  // as many rows to each
}
// Few rows: the parameters' gradients come from workgroups of the same launch that read all rows of some columns once more (from
// L2) instead of a second launch that adds up the first one's sums: 64 columns each where up to 256 threads hold a row (2,048
// columns), else 128. Backward passes one after another in a graph, one launch against two (us, fp16): 128 x 3,584 4.5 against 7.8,
// 256 x 8,192 7.6 against 15.8, 256 x 1,024 5.0 against 6.7, 255 x 1,021 6.7 against 7.4, 255 x 8,191 12.0 against 18.9; narrow odd
// rows are level (255 x 333: 7.0 and 7.2) or lose (255 x 77: 7.7 and 5.9). By calls the host takes 12 with one launch, 17 with
// two. More rows lose: in a graph 512 x 1,024 was 9.8 against 8.1 and 1,024 x 1,024 18.1 against 11.0 (128 columns each). 64 columns a
// workgroup for wide rows too: 256 x 3,584 8.1 for 6.6; 128 for all: 255 x 1,021 9.6 for 6.7.
constexpr int64_t kTrainNormFewRows = 256;
constexpr int train_norm_few_cols(int lanes) { return lanes <= 256 ? 64 : 128; }
inline bool train_norm_few(int64_t rows, int64_t cols) { return rows <= kTrainNormFewRows && cols <= 8192; }
inline int64_t train_norm_workspace_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || train_norm_few(rows, cols) ? 0 : train_norm_workgroups(rows, cols) * 2 * ceil_div(cols, 8) * 8 * 4;
}

}  // namespace cti
