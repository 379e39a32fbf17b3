// Embedding lookup with a scale, and the gradients of tables behind lookups and pooled bags, for MI355X
// (gfx950).
//
//   lookup:    out[i] = scale * W[clamp(id_i)]                    fp32, one rounding
//   gradient:  dW[v] = scale * sum_{i: clamp(id_i) = v} w_i g[u_i]
// u_i is the gradient's row that id i contributed to (the id's own position, or its bag), w_i is 1 or, under
// mean pooling, 1 / length of the bag. No contribution is added by an atomic: the ids are sorted (stably, so
// in order of position), and each table row's contributions are added in fp32 in an order that the sizes
// and the ids fix, rounded once. The same call gives the same bits in every run.
//
// 1. Keys: (table's first row number + clamped id, u) for each id; ids of the padding row and ids in no bag
//    get the key `total`, which sorts last and is dropped. Bags are found from their starts in the tile.
// 2. A radix sort by digits of at most 11 bits, least significant first, in tiles of 4,096: counts of every
//    tile, their sums over the tiles, then ranks within the tile (one ballot a bit finds the lanes of a
//    wavefront that hold the same digit), the tile put in order in LDS and written out in runs. Few tiles add
//    up the counts of the others themselves. Up to 32,768 ids are sorted in one launch, by ranges of keys; up to
//    8,192 ids in bags in the launch that finds their bags.
// 3. Sums: a workgroup takes a run of the sorted list, wavefronts (or, for narrow rows and tables of several
//    widths, lane groups that cover a row's columns) walk shares of it, several rows' loads in flight, and write
//    a table row where its key ends inside the share. What crosses shares is added in LDS, what crosses
//    workgroups goes to the workspace as fp32 rows, at most two a workgroup, and a second kernel adds these up.
//
// Measured (917,504 ids in 114,688 bags of 128 bf16 columns, Zipf ids of 2M rows, 146,000 of them hit): keys 13 us,
// sort 42, the rows' numbers 4, sums 42 (235 MB gathered from the memory-side cache; the pooling kernel takes 29 for
// the same rows in bags of 64, with a tenth of the rows to write), join 7. The sort is bound by its launches' latency
// (4 to 13 us each), the sums by the gather.
#include <stdint.h>

#include "ebag_train.h"

namespace cti {
namespace {

// ---------------------------------------------------------------------------------------------
// Lookup
// ---------------------------------------------------------------------------------------------
constexpr int kLookupThreads = 256;

struct LookupParams {
  const void* ids;
  const char* weight;
  char* out;
  int64_t rows;
  int64_t row_bytes;  // between rows of the table
  int32_t dim;
  int32_t ids64;
  uint32_t chunks;    // of this launch
  uint32_t per_row;   // chunks of 8 columns a row
  ChunkDivide div;
  float scale;
  int32_t stream_out;
};

// An id of either type, clamped to a table's rows.
__device__ __forceinline__ int64_t load_id(const void* ids, int32_t ids64, int64_t i, int64_t rows) {
  const int64_t id = ids64 ? static_cast<const int64_t*>(ids)[i] : static_cast<int64_t>(static_cast<const int32_t*>(ids)[i]);
  return clamp_i64(id, 0, rows - 1);
}

// A thread takes four chunks of 8 columns, their loads under way together (16,384 rows of 4,096 bf16 columns:
// 35 us, 4.9 TB/s of minimal bytes; one chunk a thread 38).
// Bound by HBM where the rows are many, by the latency of an id's load and a row's behind it where they are few.
// The last chunk of a row ends with it and overlaps the one before (the same values twice); rows of less than 8 columns are
// one chunk.
constexpr int kLookupChunks = 4;
template <typename T, typename OT>
__global__ void __launch_bounds__(kLookupThreads) lookup_kernel(const LookupParams p) {
  const uint32_t first = blockIdx.x * (kLookupThreads * kLookupChunks) + threadIdx.x;
  uint32_t row[kLookupChunks];
  int col[kLookupChunks];
  int64_t id[kLookupChunks];
  Chunk<T> x[kLookupChunks];
#pragma unroll
  for (int k = 0; k < kLookupChunks; ++k) {
    const uint32_t c = first + k * kLookupThreads, at = c < p.chunks ? c : p.chunks - 1;
    row[k] = p.div.quotient(at);
    col[k] = static_cast<int>(at - row[k] * p.per_row) * 8;
    if (p.dim >= 8) col[k] = chunk_start(col[k], p.dim);
    id[k] = load_id(p.ids, p.ids64, row[k], p.rows);
  }
#pragma unroll
  for (int k = 0; k < kLookupChunks; ++k) x[k].load(p.weight + id[k] * p.row_bytes, col[k], p.dim);
  with_stream(p.stream_out, [&](auto stream) {
#pragma unroll
    for (int k = 0; k < kLookupChunks; ++k) {
      if (first + k * kLookupThreads < p.chunks) {
        float v[8];
        x[k].unpack(v, col[k], p.dim);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= p.scale;
        store8<OT, decltype(stream)::value>(p.out + (static_cast<int64_t>(row[k]) * p.dim + col[k]) * Elem<OT>::kBytes, p.dim - col[k], v);
      }
    }
  });
}

// ---------------------------------------------------------------------------------------------
// Gradient: keys
// ---------------------------------------------------------------------------------------------
constexpr int kTile = kGradTile;  // keys a workgroup sorts
constexpr int kSortThreads = 512;
constexpr int kItems = kTile / kSortThreads;  // keys a thread
constexpr int kMaxFields = 64;

// Where the ids' bags and tables are.
struct GradSource {
  const void* ids;
  const void* val_offsets;  // reference layout: first id of each slot; NULL: global offsets
  const void* offsets;      // row offsets [F * (B + 1)], or global [F * B + 1]; NULL: a lookup, u_i = i
  float* inv_len;           // mean pooling: 1 / length of bag u is written here; NULL: sum
  int64_t n;
  int64_t batch;
  int64_t bags;             // F * B
  int32_t fields;
  int32_t ids64;
  int32_t offs64;
  int32_t per_field;        // base / rows below hold for each field; else base 0 and rows[0] for all
  uint32_t total;           // rows of all tables: the key of what is dropped
  ChunkDivide by_batch;
  int64_t padding;          // -1: none
  uint32_t base[kMaxFields];
  uint32_t rows[kMaxFields];
};

__device__ __forceinline__ int64_t load_off(const void* p, int32_t is64, int64_t i) {
  return is64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// First id of bag j = f * B + b, clipped to [0, n]; bag j's end is that of the next offset.
__device__ __forceinline__ int64_t bag_edge(const GradSource& s, int64_t j, int end) {
  int64_t v;
  if (s.val_offsets) {
    const int64_t f = s.by_batch.quotient(static_cast<uint32_t>(j));
    v = load_off(s.val_offsets, s.offs64, f) + load_off(s.offsets, s.offs64, j + f + end);
  } else {
    v = load_off(s.offsets, s.offs64, j + end);
  }
  return clamp_i64(v, 0, s.n);
}

// The key of an id of field f.
__device__ __forceinline__ uint32_t grad_key(const GradSource& s, int64_t id, int f) {
  const uint32_t at = s.per_field ? f : 0;
  id = clamp_i64(id, 0, static_cast<int64_t>(s.rows[at]) - 1);
  return id == s.padding ? s.total : s.base[at] + static_cast<uint32_t>(id);
}

constexpr int kMostBags = 8 * kTile;  // bags whose starts a tile looks through; with more, each id searches

// Keys and u of the tile's ids (THREADS * ITEMS): item k of a thread is the tile's id item_index(k). s_bag: a word for each.
template <int ITEMS = kItems>
__device__ __forceinline__ int item_index(int k) {
  return (static_cast<int>(threadIdx.x) / kWave) * (ITEMS * kWave) + k * kWave + lane_id();
}

// The ids' own loads are under way while their bags are found: the tile's first bag to within 512 by a search of 512
// places a step, the others by reading edges from there on, 1,024 at a time. Bag j's start is event 2 (j - lo) + 2 at its place,
// its end event 2 (j - lo) + 3 at the place behind; the largest event up to an id is its bag's start (even), or an
// end: the id lies in no bag. (Ends looked up id by id, a search of 64 places and one for the tile's last id:
// 917,504 ids in 114,688 bags 16 us, 13 so.)
template <int THREADS, int ITEMS>
__device__ __forceinline__ void tile_keys(const GradSource& s, int64_t tile, uint32_t* key, uint32_t* unit, int32_t* s_bag,
                                          int32_t* s_wave) {
  const int64_t first = tile * (THREADS * ITEMS);
  const int t = static_cast<int>(threadIdx.x);
  int64_t id[ITEMS];
  const auto load_ids = [&](auto type) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t i = first + item_index<ITEMS>(k);
      id[k] = static_cast<const decltype(type)*>(s.ids)[i < s.n ? i : s.n - 1];
    }
  };
  if (s.ids64) load_ids(int64_t{});
  else load_ids(int32_t{});
  if (!s.offsets) {
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const int64_t i = first + item_index<ITEMS>(k);
      key[k] = i < s.n ? grad_key(s, id[k], 0) : 0xffffffffu;
      unit[k] = static_cast<uint32_t>(i);
    }
    return;
  }
  const int64_t last = (first + THREADS * ITEMS < s.n ? first + THREADS * ITEMS : s.n) - 1;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) s_bag[t + k * THREADS] = 0;
  // bags that start at or before the first id: `lo` at least, `hi` at most
  int64_t lo = 0, hi = s.bags;
  while (hi - lo > THREADS) {  // lo grows or hi falls in every step, whatever the offsets hold
    const int64_t step = (hi - lo + THREADS - 1) / THREADS;
    const int64_t j = lo + step * (t + 1) - 1;  // the thread's last bag of its share
    const int started = __syncthreads_count(j < hi && bag_edge(s, j, 0) <= first);
    lo += step * started;
    if (lo + step - 1 < hi) hi = lo + step - 1;
  }
  lo = lo > 0 ? lo - 1 : 0;
  // edges of bags lo, lo + 1, ... until one starts behind the tile, two a thread; those before the tile leave nothing
  __syncthreads();
  int64_t begun = 0;
  bool scan = true;
  for (int64_t j0 = lo;; j0 += 2 * THREADS) {
    int64_t a[2], b[2];
    bool in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t j = j0 + h * THREADS + t;
      in[h] = j < s.bags;
      a[h] = in[h] ? bag_edge(s, j, 0) : 0;
      b[h] = in[h] ? bag_edge(s, j, 1) : 0;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      in[h] = in[h] && a[h] <= last;
      if (in[h] && b[h] > first) {
        const int32_t event = static_cast<int32_t>(j0 + h * THREADS + t - lo) * 2 + 2;
        const int64_t at = a[h] > first ? a[h] - first : 0;
        if (b[h] > a[h]) atomicMax(&s_bag[at], event);
        if (b[h] <= last) atomicMax(&s_bag[b[h] - first], event + 1);
      }
    }
    const int c = __syncthreads_count(in[1]);
    begun += 2 * c;
    if (c < THREADS) break;
    if (begun > kMostBags) {
      scan = false;
      break;
    }
  }
  if (scan) {
    constexpr int kRun = ITEMS;
    int32_t m[kRun], top = 0;
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const int32_t b = s_bag[t * kRun + k];
      top = b > top ? b : top;
      m[k] = top;
    }
    int32_t before = top;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int32_t o = shfl_i32(before, lane_id() - d);
      if (lane_id() >= d) before = o > before ? o : before;
    }
    if (lane_id() == kWave - 1) s_wave[t / kWave] = before;
    int32_t carry = shfl_i32(before, lane_id() - 1);
    if (lane_id() == 0) carry = 0;
    __syncthreads();
    for (int w = 0; w < t / kWave; ++w) carry = s_wave[w] > carry ? s_wave[w] : carry;
#pragma unroll
    for (int k = 0; k < kRun; ++k) s_bag[t * kRun + k] = m[k] > carry ? m[k] : carry;
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t i = first + item_index<ITEMS>(k);
    key[k] = 0xffffffffu;
    unit[k] = 0u;
    if (i >= s.n) continue;
    key[k] = s.total;
    int64_t j;
    if (scan) {
      const int32_t event = s_bag[item_index<ITEMS>(k)];
      if (event == 0 || event % 2) continue;  // in no bag
      j = lo + event / 2 - 1;
    } else {
      int64_t a = lo, b = s.bags;  // bags started at or before i
      while (a < b) {
        const int64_t mid = (a + b) / 2;
        if (bag_edge(s, mid, 0) <= i) a = mid + 1;
        else b = mid;
      }
      j = a - 1;
      if (j < 0 || i >= bag_edge(s, j, 1)) continue;
    }
    const int64_t f = s.by_batch.quotient(static_cast<uint32_t>(j));
    key[k] = grad_key(s, id[k], static_cast<int>(f));
    unit[k] = static_cast<uint32_t>((j - f * s.batch) * s.fields + f);
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient: rows without ids
// ---------------------------------------------------------------------------------------------
// What is written before the sums: zeros to whole tables, -1 to the compact form's numbers. It rides on the
// sort's launches, whose few workgroups wait on latency: workgroups behind the sort's take shares of 64 KiB.
constexpr int64_t kFillShare = kGradFillShare;
struct GradFill {
  char* data[kMaxFields];
  int64_t bytes[kMaxFields];       // rows * row_bytes
  int64_t row_bytes[kMaxFields];   // to be written
  int64_t row_stride[kMaxFields];  // bytes between rows
  int32_t tables;
  uint32_t value;
  int32_t sort_groups;  // workgroups of this launch that sort
  int32_t first_share;  // share of the first one behind them
};

__device__ __forceinline__ void fill_share(const GradFill& f, int64_t share) {
  int i = 0;
  for (; i < f.tables; ++i) {
    const int64_t shares = (f.bytes[i] + kFillShare - 1) / kFillShare;
    if (share < shares) break;
    share -= shares;
  }
  if (i == f.tables) return;
  char* const data = f.data[i];
  const int64_t a = share * kFillShare, b = a + kFillShare < f.bytes[i] ? a + kFillShare : f.bytes[i];
  const int t = static_cast<int>(threadIdx.x);
  if (f.row_stride[i] == f.row_bytes[i]) {
    const u32x4 v = {f.value, f.value, f.value, f.value};
    const int64_t whole = a + (b - a) / 16 * 16;
#pragma unroll 8
    for (int64_t at = a + t * 16; at < whole; at += blockDim.x * 16) *reinterpret_cast<u32x4_any*>(data + at) = v;
    for (int64_t at = whole + t * 2; at < b; at += blockDim.x * 2) *reinterpret_cast<uint16_t*>(data + at) = static_cast<uint16_t>(f.value);
  } else {
    for (int64_t at = a + t * 2; at < b; at += blockDim.x * 2) {
      const int64_t row = at / f.row_bytes[i];
      *reinterpret_cast<uint16_t*>(data + row * f.row_stride[i] + (at - row * f.row_bytes[i])) = static_cast<uint16_t>(f.value);
    }
  }
}

// Whether the workgroup is one behind the sort's; then its share is written.
__device__ __forceinline__ bool fills(const GradFill& f) {
  const int extra = static_cast<int>(blockIdx.x) - f.sort_groups;
  if (extra < 0) return false;
  fill_share(f, static_cast<int64_t>(f.first_share) + extra);
  return true;
}

// ---------------------------------------------------------------------------------------------
// Gradient: sort
// ---------------------------------------------------------------------------------------------
// (key, u) of every id. Digits of up to kGradDigitBits = 11 bits (21 bits, two million rows, in two passes: 917,504
// ids 55 us with their keys; in three of 7 bits, each tile adding up the counts of all tiles, 74).
typedef uint2 Pair;

// The tile of a workgroup: runs of tiles to each of the 8 XCDs, to which workgroups go in turn, so that what
// neighbouring tiles write side by side meets in one L2.
__device__ __forceinline__ int64_t tile_of(int64_t group, int64_t tiles) {
  const int64_t per = tiles / 8, more = tiles % 8, xcd = group % 8;
  return xcd * per + (xcd < more ? xcd : more) + group / 8;
}

// Exclusive sums over the workgroup's threads; s_scan: a word for each wavefront.
template <int THREADS>
__device__ __forceinline__ uint32_t group_scan(uint32_t v, uint32_t* s_scan) {
  const int t = static_cast<int>(threadIdx.x);
  uint32_t x = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = static_cast<uint32_t>(shfl_i32(static_cast<int>(x), lane_id() - d));
    if (lane_id() >= d) x += o;
  }
  __syncthreads();
  if (lane_id() == kWave - 1) s_scan[t / kWave] = x;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / kWave; ++w) before += w < t / kWave ? s_scan[w] : 0u;
  return before + x - v;
}

// Places of the tile's keys in the tile sorted by one digit (stable): place[k] of item k. s_hist: wavefronts << bits
// numbers, 16-byte aligned; s_start[d] is the first place of digit d. A thread holds digits 4 t to 4 t + 3; counts[4] of them are the tile's.
template <int THREADS, int ITEMS>
__device__ __forceinline__ void tile_places(const uint32_t* key, int shift, int bits, uint32_t* place, uint16_t* s_hist,
                                            uint32_t* s_start, uint32_t* s_scan) {
  const int t = static_cast<int>(threadIdx.x), w = t / kWave, digits = 1 << bits;
  const uint32_t mask = digits - 1;
  uint2* const hist4 = reinterpret_cast<uint2*>(s_hist);
  for (int i = t; i < THREADS / kWave * digits / 4; i += THREADS) hist4[i] = make_uint2(0u, 0u);
  __syncthreads();
  // the lanes with the same digit, of every item before the first one's turn, so that no ballot waits for LDS: where a
  // lane's bit is like the lane's own (m: its bit in every place), same & ~(ones ^ m) keeps it
  uint32_t lo[ITEMS], hi[ITEMS];
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) lo[k] = hi[k] = ~0u;
#pragma unroll
  for (int b = 0; b < kGradDigitBits; ++b) {
    if (b < bits) {
#pragma unroll
      for (int k = 0; k < ITEMS; ++k) {
        const uint32_t m = static_cast<uint32_t>(static_cast<int32_t>((key[k] >> shift) << (31 - b)) >> 31);
        const uint64_t ones = __ballot(m != 0u);
        lo[k] = __builtin_amdgcn_bitop3_b32(lo[k], static_cast<uint32_t>(ones), m, 0x90);
        hi[k] = __builtin_amdgcn_bitop3_b32(hi[k], static_cast<uint32_t>(ones >> 32), m, 0x90);
      }
    }
  }
  volatile uint16_t* const mine = s_hist + w * digits;
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t d = (key[k] >> shift) & mask;
    const uint32_t seen = mine[d];
    const uint32_t rank = __builtin_amdgcn_mbcnt_hi(hi[k], __builtin_amdgcn_mbcnt_lo(lo[k], 0u));  // lanes before this one
    place[k] = seen + rank;
    __builtin_amdgcn_wave_barrier();
    if (rank == 0) mine[d] = static_cast<uint16_t>(seen + static_cast<uint32_t>(__popc(lo[k]) + __popc(hi[k])));
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  uint32_t sum[4] = {0u, 0u, 0u, 0u};
  if (4 * t < digits) {
#pragma unroll
    for (int i = 0; i < THREADS / kWave; ++i) {
      const uint2 c = hist4[i * (digits / 4) + t];
      hist4[i * (digits / 4) + t] = make_uint2(sum[0] | (sum[1] << 16), sum[2] | (sum[3] << 16));
      sum[0] += c.x & 0xffffu, sum[1] += c.x >> 16, sum[2] += c.y & 0xffffu, sum[3] += c.y >> 16;
    }
  }
  uint32_t start = group_scan<THREADS>(sum[0] + sum[1] + sum[2] + sum[3], s_scan);
  if (4 * t < digits) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s_start[4 * t + i] = start;
      start += sum[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const uint32_t d = (key[k] >> shift) & mask;
    place[k] += s_start[d] + s_hist[w * digits + d];
  }
}

// All ids in one tile of up to kGradIdsAlone: keys and every digit in one launch (5,001 ids of 10 bits: 10 us, in two
// launches 15; 16,384 ids of 15 bits: 35 us in one workgroup, 37 in four launches of four).
template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) grad_sort_tile_kernel(const GradSource s, Pair* out, int all_bits, int digit_bits,
                                                                 const GradFill fill) {
  if (fills(fill)) return;
  constexpr int HIST = THREADS / kWave * kGradDigits;
  __shared__ Pair s_pair[THREADS * ITEMS > HIST / 4 ? THREADS * ITEMS : HIST / 4];  // the digits' numbers, then the pairs
  __shared__ uint32_t s_start[kGradDigits], s_scan[THREADS / kWave];
  uint16_t* const s_hist = reinterpret_cast<uint16_t*>(s_pair);
  uint32_t key[ITEMS], unit[ITEMS], place[ITEMS];
  tile_keys<THREADS, ITEMS>(s, 0, key, unit, reinterpret_cast<int32_t*>(s_pair), reinterpret_cast<int32_t*>(s_scan));
  __syncthreads();
  for (int shift = 0; shift < all_bits; shift += digit_bits) {
    tile_places<THREADS, ITEMS>(key, shift, digit_bits, place, s_hist, s_start, s_scan);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) s_pair[place[k]] = make_uint2(key[k], unit[k]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
      const Pair v = s_pair[item_index<ITEMS>(k)];
      key[k] = v.x;
      unit[k] = v.y;
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int i = item_index<ITEMS>(k);
    if (i < s.n) out[i] = make_uint2(key[k], unit[k]);
  }
}

// Up to kGradIdsRanged ids in one launch without counts: a workgroup for each range of keys (the `range_bits` top ones) reads
// all of them, keeps its own in LDS in their order, as (the key's other bits, position), sorts these and writes them behind the
// ids of the ranges before, which it has counted on the way. Nothing waits for another workgroup; a range that holds every
// id takes as long as one workgroup takes for them. (19 bits without a fill: 8,192 ids 10 us, 16,384 13, 32,768 19; with the sort's
// steps unrolled for a range of any size alone, their conditions held as scalars, 12, 16 and 25. Beside a fill of 131 MB, which
// takes 20 by itself, 16,384 ids in four tiles and four launches 37.)
constexpr int kRangeThreads = 1024, kRangeWaves = kRangeThreads / kWave;
static_assert(kGradIdsRanged <= (1 << kGradPositionBits), "a position has its bits");
template <int ITEMS>
__global__ void __launch_bounds__(kRangeThreads) grad_sort_ranges_kernel(const GradSource s, const Pair* in, Pair* out, int key_bits,
                                                                         const GradFill fill) {
  if (fills(fill)) return;
  // (8 bits where two workgroups, of which the other fills, then fit a CU)
  constexpr int DIGIT_BITS = ITEMS == 32 ? 9 : 8, DIGITS = 1 << DIGIT_BITS;
  __shared__ uint32_t s_val[kRangeThreads * ITEMS];
  __shared__ __align__(16) uint16_t s_hist[kRangeWaves * DIGITS];
  __shared__ uint32_t s_start[DIGITS], s_scan[kRangeWaves], s_count[2][kRangeWaves];
  const int t = static_cast<int>(threadIdx.x), w = t / kWave, n = static_cast<int>(s.n);
  const uint32_t range = blockIdx.x;
  // a wavefront reads `rows` times 64 ids side by side
  const int rows = (n + kRangeThreads - 1) / kRangeThreads;
  const int first = w * rows * kWave + lane_id(), end = (w + 1) * rows * kWave < n ? (w + 1) * rows * kWave : n;
  uint32_t v[ITEMS], kept = 0, mine = 0, below = 0;
  const auto read = [&](auto key_of) {
#pragma unroll
    for (int g = 0; g < ITEMS; g += 8) {  // (a condition an item would hold a scalar each)
      if (g < rows) {
#pragma unroll
        for (int k = g; k < g + 8; ++k) v[k] = key_of(first + k * kWave < end ? first + k * kWave : n - 1);
      }
    }
  };
  if (in) read([&](int i) { return in[i].x; });
  else if (s.ids64) read([&](int i) { return grad_key(s, static_cast<const int64_t*>(s.ids)[i], 0); });
  else read([&](int i) { return grad_key(s, static_cast<const int32_t*>(s.ids)[i], 0); });
#pragma unroll
  for (int g = 0; g < ITEMS; g += 8) {
    if (g < rows) {
#pragma unroll
      for (int k = g; k < g + 8; ++k) {
        const bool there = first + k * kWave < end;
        const uint32_t r = v[k] >> key_bits;
        const bool own = there && r == range;
        kept |= (own ? 1u : 0u) << k;
        mine += static_cast<uint32_t>(__popcll(__ballot(own)));
        below += static_cast<uint32_t>(__popcll(__ballot(there && r < range)));
      }
    }
  }
  if (lane_id() == 0) {
    s_count[0][w] = mine;
    s_count[1][w] = below;
  }
  __syncthreads();
  uint32_t at = 0, m = 0, base = 0;
#pragma unroll
  for (int i = 0; i < kRangeWaves; ++i) {
    at += i < w ? s_count[0][i] : 0u;
    m += s_count[0][i];
    base += s_count[1][i];
  }
#pragma unroll
  for (int g = 0; g < ITEMS; g += 8) {
    if (g < rows) {
#pragma unroll
      for (int k = g; k < g + 8; ++k) {
        const bool own = (kept >> k) & 1u;
        const uint64_t lanes = __ballot(own);
        const uint32_t place = at + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32),
                                                              __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0u));
        if (own) s_val[place] = ((v[k] & ((1u << key_bits) - 1u)) << kGradPositionBits) | static_cast<uint32_t>(first + k * kWave);
        at += static_cast<uint32_t>(__popcll(lanes));
      }
    }
  }
  __syncthreads();
  const int per = static_cast<int>((m + kRangeThreads - 1) / kRangeThreads);  // items a thread
  const int passes = (key_bits + DIGIT_BITS - 1) / DIGIT_BITS;
  const int digit_bits = passes > 0 ? ((key_bits + passes - 1) / passes < 2 ? 2 : (key_bits + passes - 1) / passes) : 0;
  const auto sort = [&](auto most) {
    constexpr int PER = decltype(most)::value;  // per <= PER; ranges are mostly small, and code that is skipped is still fetched
    for (int shift = 0; m > 1 && shift < key_bits; shift += digit_bits) {
      const int digits = 1 << digit_bits;
      const uint32_t mask = digits - 1;
      uint2* const hist4 = reinterpret_cast<uint2*>(s_hist);
      for (int i = t; i < kRangeWaves * digits / 4; i += kRangeThreads) hist4[i] = make_uint2(0u, 0u);
      __syncthreads();
      volatile uint16_t* const hist = s_hist + w * digits;
      uint32_t x[PER], place[PER];
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        if (k < per) {
          const uint32_t i = static_cast<uint32_t>((w * per + k) * kWave + lane_id());
          x[k] = i < m ? s_val[i] : ~0u;  // past the end: the largest digit, and last
          const uint32_t d = (x[k] >> (kGradPositionBits + shift)) & mask;
          uint32_t lo = ~0u, hi = ~0u;
#pragma unroll
          for (int b = 0; b < DIGIT_BITS; ++b) {
            if (b < digit_bits) {
              const uint32_t own = static_cast<uint32_t>(static_cast<int32_t>(d << (31 - b)) >> 31);
              const uint64_t ones = __ballot(own != 0u);
              lo = __builtin_amdgcn_bitop3_b32(lo, static_cast<uint32_t>(ones), own, 0x90);
              hi = __builtin_amdgcn_bitop3_b32(hi, static_cast<uint32_t>(ones >> 32), own, 0x90);
            }
          }
          const uint32_t seen = hist[d];
          const uint32_t rank = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0u));
          place[k] = seen + rank;
          __builtin_amdgcn_wave_barrier();
          if (rank == 0) hist[d] = static_cast<uint16_t>(seen + static_cast<uint32_t>(__popc(lo) + __popc(hi)));
          __builtin_amdgcn_wave_barrier();
        }
      }
      __syncthreads();
      uint32_t sum[4] = {0u, 0u, 0u, 0u};
      if (4 * t < digits) {
#pragma unroll
        for (int i = 0; i < kRangeWaves; ++i) {
          const uint2 c = hist4[i * (digits / 4) + t];
          hist4[i * (digits / 4) + t] = make_uint2(sum[0] | (sum[1] << 16), sum[2] | (sum[3] << 16));
          sum[0] += c.x & 0xffffu, sum[1] += c.x >> 16, sum[2] += c.y & 0xffffu, sum[3] += c.y >> 16;
        }
      }
      uint32_t start = group_scan<kRangeThreads>(sum[0] + sum[1] + sum[2] + sum[3], s_scan);
      if (4 * t < digits) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s_start[4 * t + i] = start;
          start += sum[i];
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        if (k < per) {
          const uint32_t d = (x[k] >> (kGradPositionBits + shift)) & mask;
          s_val[place[k] + s_start[d] + s_hist[w * digits + d]] = x[k];
        }
      }
      __syncthreads();
    }
  };
  if (per <= 2) sort(std::integral_constant<int, 2>{});
  else sort(std::integral_constant<int, ITEMS>{});
  for (uint32_t i = t; i < m; i += kRangeThreads) {
    const uint32_t x = s_val[i], position = x & ((1u << kGradPositionBits) - 1u);
    out[base + i] = make_uint2((range << key_bits) | (x >> kGradPositionBits), in ? in[position].y : position);
  }
}

__device__ __forceinline__ void tile_count(const uint32_t* key, int64_t live, int shift, int bits, uint32_t* counts,
                                           uint32_t* s_hist) {
  const int t = static_cast<int>(threadIdx.x), digits = 1 << bits;
  const uint32_t mask = digits - 1;
  for (int i = t; i < digits; i += kSortThreads) s_hist[i] = 0u;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kItems; ++k)
    if (item_index(k) < live) atomicAdd(&s_hist[(key[k] >> shift) & mask], 1u);
  __syncthreads();
  for (int i = t; i < digits; i += kSortThreads) counts[i] = s_hist[i];
}

// Fewer ids a tile where few ids are sorted by ranges, which need no tiles of 4,096: more workgroups, fewer bags for each (21,500
// ids in 7,168 bags beside half a fill of 72 MB: 15 us, so 11; 512 ids a tile 10.6).
constexpr int kRangeKeyItems = 2;
// Keys of every tile of ITEMS ids a thread and (tiles of 4,096) the counts of their first digit.
template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads) grad_keys_kernel(const GradSource s, Pair* out, uint32_t* counts, int bits,
                                                                 const GradFill fill) {
  if (fills(fill)) return;
  __shared__ int32_t s_bag[kSortThreads * ITEMS];
  __shared__ int32_t s_wave[kSortThreads / kWave];
  uint32_t key[ITEMS], unit[ITEMS];
  const int64_t tile = tile_of(blockIdx.x, fill.sort_groups), first = tile * (kSortThreads * ITEMS);
  tile_keys<kSortThreads, ITEMS>(s, tile, key, unit, s_bag, s_wave);
#pragma unroll
  for (int k = 0; k < ITEMS; ++k) {
    const int64_t i = first + item_index<ITEMS>(k);
    if (i < s.n) out[i] = make_uint2(key[k], unit[k]);
  }
  if constexpr (ITEMS == kItems) {
    __shared__ uint32_t s_hist[kGradDigits];
    tile_count(key, s.n - first, 0, bits, counts + (tile << bits), s_hist);
  }
}

__global__ void __launch_bounds__(kSortThreads) grad_count_kernel(const Pair* in, int64_t n, int shift, int bits, uint32_t* counts,
                                                                  const GradFill fill) {
  if (fills(fill)) return;
  __shared__ uint32_t s_hist[kGradDigits];
  uint32_t key[kItems];
  const int64_t tile = tile_of(blockIdx.x, fill.sort_groups), first = tile * kTile;
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = first + item_index(k);
    key[k] = in[i < n ? i : n - 1].x;
  }
  tile_count(key, n - first, shift, bits, counts + (tile << bits), s_hist);
}

// counts[tile][digit] -> how many of the digit lie in tiles before it; totals[digit]. A lane takes a digit, the wavefronts
// runs of tiles, up to kScanHeld of them in registers.
constexpr int kScanThreads = 1024, kScanWaves = kScanThreads / kWave, kScanHeld = 16;
__global__ void __launch_bounds__(kScanThreads) grad_scan_kernel(uint32_t* counts, uint32_t* totals, int64_t tiles, int bits,
                                                                 const GradFill fill) {
  if (fills(fill)) return;
  __shared__ uint32_t s_sum[kScanWaves][kWave];
  const int w = static_cast<int>(threadIdx.x) / kWave;
  const int64_t digit = static_cast<int64_t>(blockIdx.x) * kWave + lane_id(), digits = int64_t{1} << bits;
  const bool there = digit < digits;
  const int64_t per = (tiles + kScanWaves - 1) / kScanWaves;
  const int64_t a = per * w < tiles ? per * w : tiles, b = a + per < tiles ? a + per : tiles;
  uint32_t* const col = counts + digit;
  uint32_t held[kScanHeld], sum = 0;
  const bool hold = per <= kScanHeld;
  if (hold) {
#pragma unroll
    for (int k = 0; k < kScanHeld; ++k) held[k] = there && a + k < b ? col[(a + k) << bits] : 0u;
#pragma unroll
    for (int k = 0; k < kScanHeld; ++k) sum += held[k];
  } else if (there) {
#pragma unroll 8
    for (int64_t i = a; i < b; ++i) sum += col[i << bits];
  }
  s_sum[w][lane_id()] = sum;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kScanWaves; ++i) {
    const uint32_t c = s_sum[i][lane_id()];
    before += i < w ? c : 0u;
    all += c;
  }
  if (!there) return;
  if (w == 0) totals[digit] = all;
  if (hold) {
#pragma unroll
    for (int k = 0; k < kScanHeld; ++k) {
      if (a + k < b) col[(a + k) << bits] = before;
      before += held[k];
    }
  } else {
    for (int64_t i = a; i < b; ++i) {
      const uint32_t c = col[i << bits];
      col[i << bits] = before;
      before += c;
    }
  }
}

// One digit: the tile in order, written to its places. totals NULL: counts are the few tiles' own.
__global__ void __launch_bounds__(kSortThreads) grad_scatter_kernel(const Pair* in, Pair* out, int64_t n, int shift, int bits,
                                                                    const uint32_t* counts, const uint32_t* totals,
                                                                    const GradFill fill) {
  if (fills(fill)) return;
  __shared__ Pair s_pair[kTile];
  __shared__ __align__(16) uint16_t s_hist[kSortThreads / kWave * kGradDigits];
  __shared__ uint32_t s_start[kGradDigits], s_scan[kSortThreads / kWave];
  const int t = static_cast<int>(threadIdx.x), digits = 1 << bits;
  const int64_t tile = tile_of(blockIdx.x, fill.sort_groups), first = tile * kTile;
  uint32_t key[kItems], unit[kItems], place[kItems];
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int64_t i = first + item_index(k);
    const Pair v = in[i < n ? i : n - 1];
    key[k] = i < n ? v.x : 0xffffffffu;
    unit[k] = v.y;
  }
  uint4 before = make_uint4(0u, 0u, 0u, 0u), total = before;
  if (4 * t < digits) {
    const uint4* const c4 = reinterpret_cast<const uint4*>(counts);
    if (totals) {
      before = c4[tile * (digits / 4) + t];
      total = reinterpret_cast<const uint4*>(totals)[t];
    } else {
#pragma unroll 16
      for (int i = 0; i < fill.sort_groups; ++i) {
        const uint4 c = c4[i * (digits / 4) + t];
        const uint32_t m = i < tile ? ~0u : 0u;  // (a branch would wait for every load)
        total.x += c.x, total.y += c.y, total.z += c.z, total.w += c.w;
        before.x += c.x & m, before.y += c.y & m, before.z += c.z & m, before.w += c.w & m;
      }
    }
  }
  const uint32_t base = group_scan<kSortThreads>(total.x + total.y + total.z + total.w, s_scan);
  tile_places<kSortThreads, kItems>(key, shift, bits, place, s_hist, s_start, s_scan);
#pragma unroll
  for (int k = 0; k < kItems; ++k) s_pair[place[k]] = make_uint2(key[k], unit[k]);
  __syncthreads();
  if (4 * t < digits) {  // s_start becomes the way from a place in the tile to the place in the list
    uint32_t* const at = s_start + 4 * t;
    at[0] = base + before.x - at[0];
    at[1] = base + total.x + before.y - at[1];
    at[2] = base + total.x + total.y + before.z - at[2];
    at[3] = base + total.x + total.y + total.z + before.w - at[3];
  }
  __syncthreads();
  const int64_t live = n - first;
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int i = item_index(k);
    if (i < live) {  // keys past the end are the tile's last: their digit is the largest and they come last
      const Pair v = s_pair[i];
      out[s_start[(v.x >> shift) & (digits - 1)] + static_cast<uint32_t>(i)] = v;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Gradient: sums
// ---------------------------------------------------------------------------------------------
constexpr int kSumThreads = 256;
constexpr int kSumMost = 2048;  // ids a workgroup takes at most
constexpr int kSumAhead = 8;    // rows a lane group loads at once

struct SumParams {
  const char* grad;
  const Pair* ids;        // sorted
  const float* inv_len;
  const uint32_t* heads;  // compact: distinct keys that begin in each workgroup's run (or before it: scanned)
  int32_t heads_scanned;
  uint32_t* last_rank;    // compact: the last key's number of each workgroup's run
  char* out;              // dense (one table) or compact rows
  int64_t* rows_out;      // compact
  int64_t* count_out;
  float* partial;         // [columns' block][workgroup][2][slots]: what the run before began, what goes on behind
  int64_t n;
  int64_t grad_stride;    // elements between units' groups of `fields` (per-field), else dim
  uint32_t total;
  int32_t dim;            // the widest field's
  int32_t log_lanes;      // lanes that cover a block of columns, each with `lane_cols`
  int32_t lane_cols;
  int32_t out_dtype;
  int32_t run;            // ids a lane group
  int32_t workgroups;
  float scale;
  int32_t fields;
  int32_t per_field;      // tables in SumFields
  ChunkDivide by_fields;
};
// A table for each field.
struct SumFields {
  char* data[kMaxFields];
  int64_t stride[kMaxFields];
  uint32_t base[kMaxFields];
  int32_t dim[kMaxFields];
  int32_t col[kMaxFields];
};
struct NoFields {};

// Distinct keys that begin in each run of `ids`.
__global__ void __launch_bounds__(kSumThreads) grad_heads_kernel(const Pair* sorted, int64_t n, uint32_t total, int ids,
                                                                 uint32_t* heads) {
  __shared__ uint32_t s_sum[kSumThreads / kWave];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * ids;
  uint32_t c = 0;
  for (int i = static_cast<int>(threadIdx.x); i < ids; i += kSumThreads) {
    const int64_t at = first + i;
    if (at < n) {
      const uint32_t k = sorted[at].x;
      c += k < total && (at == 0 || sorted[at - 1].x != k) ? 1u : 0u;
    }
  }
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) c += static_cast<uint32_t>(shfl_i32(static_cast<int>(c), lane_id() ^ m));
  if (lane_id() == 0) s_sum[threadIdx.x / kWave] = c;
  __syncthreads();
  if (threadIdx.x == 0) {
    c = 0;
#pragma unroll
    for (int w = 0; w < kSumThreads / kWave; ++w) c += s_sum[w];
    heads[blockIdx.x] = c;
  }
}

// heads[i] -> their sum before i, heads[count] the whole: one workgroup.
__global__ void __launch_bounds__(kScanThreads) grad_heads_scan_kernel(uint32_t* heads, int64_t count) {
  __shared__ uint32_t s_sum[kScanThreads];
  const int t = static_cast<int>(threadIdx.x);
  const int64_t per = (count + kScanThreads - 1) / kScanThreads;
  const int64_t a = per * t < count ? per * t : count, b = a + per < count ? a + per : count;
  uint32_t sum = 0;
  for (int64_t i = a; i < b; ++i) sum += heads[i];
  s_sum[t] = sum;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < kScanThreads; ++i) {
    if (i == t) sum = before;
    before += s_sum[i];
  }
  if (t == 0) heads[count] = before;
  for (int64_t i = a; i < b; ++i) {
    const uint32_t c = heads[i];
    heads[i] = sum;
    sum += c;
  }
}

// The first of the `cols` columns of lane `lane` of block `block`; the last vector ends with the row and
// overlaps the one before it (both come to the same sums). A row narrower than a vector is lane 0's.
__device__ __forceinline__ int first_column(int block, int lane, int dim, int cols) {
  const int c = (block * kWave + lane) * cols;
  if (c >= dim) return -1;
  return c + cols <= dim ? c : (dim >= cols ? dim - cols : 0);
}

// f(OT{}) for the type of the sums (the walk below knows it when it is built: 45 us against 42, a key's end being a place in
// every unrolled step).
template <typename F>
__device__ __forceinline__ void with_out_type(const SumParams& p, F&& f) {
  if (p.out_dtype == CTI_EBAG_F32) f(float{});
  else if (p.out_dtype == CTI_EBAG_BF16) f(bf16_t{});
  else f(f16_t{});
}
// One element of a row of sums.
__device__ __forceinline__ void put_sum(const SumParams& p, char* row, int col, float v) {
  with_out_type(p, [&](auto o) { store_one(reinterpret_cast<decltype(o)*>(row) + col, v, false); });
}

template <typename T, typename FIELDS>
struct Sums {
  static constexpr int VEC = 16 / Elem<T>::kBytes;
  static constexpr bool kPerField = !std::is_same<FIELDS, NoFields>::value;

  // Element col of unit's row, and that row's width.
  __device__ static __forceinline__ const char* row(const SumParams& p, const FIELDS& fs, uint32_t unit, int* dim) {
    if constexpr (kPerField) {
      const uint32_t b = p.by_fields.quotient(unit), f = unit - b * static_cast<uint32_t>(p.fields);
      *dim = fs.dim[f];
      return p.grad + (static_cast<int64_t>(b) * p.grad_stride + fs.col[f]) * Elem<T>::kBytes;
    } else {
      *dim = p.dim;
      return p.grad + static_cast<int64_t>(unit) * p.dim * Elem<T>::kBytes;
    }
  }
  // The row that a key's sum goes to; rank: its number among the distinct keys.
  __device__ static __forceinline__ char* target(const SumParams& p, const FIELDS& fs, uint32_t key, uint32_t unit, uint32_t rank) {
    const int bytes = p.out_dtype == CTI_EBAG_F32 ? 4 : 2;
    if (p.rows_out) return p.out + static_cast<int64_t>(rank) * p.dim * bytes;
    if constexpr (kPerField) {
      const uint32_t f = unit - p.by_fields.quotient(unit) * static_cast<uint32_t>(p.fields);
      return fs.data[f] + static_cast<int64_t>(key - fs.base[f]) * fs.stride[f] * bytes;
    } else {
      return p.out + static_cast<int64_t>(key) * p.dim * bytes;
    }
  }
  __device__ static __forceinline__ int width(const SumParams& p, const FIELDS& fs, uint32_t unit) {
    if constexpr (kPerField) return fs.dim[unit - p.by_fields.quotient(unit) * static_cast<uint32_t>(p.fields)];
    else return p.dim;
  }
};

// Distinct keys that begin in the runs before this workgroup's, and all of them. s_sum: 2 * wavefronts words.
__device__ __forceinline__ uint32_t keys_begun(const SumParams& p, uint32_t* total, uint32_t (*s_sum)[kSumThreads / kWave]) {
  if (p.heads_scanned) {
    *total = p.heads[p.workgroups];
    return p.heads[blockIdx.x];
  }
  const int t = static_cast<int>(threadIdx.x);
  uint32_t all = 0, begun = 0;
#pragma unroll 8
  for (int i = t; i < p.workgroups; i += kSumThreads) {
    const uint32_t c = p.heads[i];
    all += c;
    begun += i < static_cast<int>(blockIdx.x) ? c : 0u;
  }
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    all += static_cast<uint32_t>(shfl_i32(static_cast<int>(all), lane_id() ^ m));
    begun += static_cast<uint32_t>(shfl_i32(static_cast<int>(begun), lane_id() ^ m));
  }
  if (lane_id() == 0) {
    s_sum[0][t / kWave] = all;
    s_sum[1][t / kWave] = begun;
  }
  __syncthreads();
  all = begun = 0;
#pragma unroll
  for (int w = 0; w < kSumThreads / kWave; ++w) {
    all += s_sum[0][w];
    begun += s_sum[1][w];
  }
  *total = all;
  return begun;
}

// A workgroup's run of the sorted ids: `run` for each of its kSumThreads >> log_lanes lane groups.
// blockIdx.x: the run; blockIdx.y: the block of 64 vectors of columns.
template <typename T, typename FIELDS>
__global__ void __launch_bounds__(kSumThreads) grad_sum_kernel(const SumParams p, const FIELDS fs) {
  using S = Sums<T, FIELDS>;
  constexpr int VEC = S::VEC;
  __shared__ uint32_t s_key[kSumMost + 2];  // one before, one behind
  __shared__ uint32_t s_unit[kSumMost];
  __shared__ uint32_t s_rank[kSumMost];
  __shared__ float s_part[2][kSumThreads * VEC];  // of each lane group: what a group before began; what goes on
  __shared__ uint8_t s_flag[2][kSumThreads];      // 1: there is one; 2: it goes on behind the group, too
  __shared__ uint32_t s_wave[kSumThreads / kWave], s_sum[2][kSumThreads / kWave];
  const int t = static_cast<int>(threadIdx.x), lanes = 1 << p.log_lanes, groups = kSumThreads >> p.log_lanes;
  const int ids = groups * p.run, block = static_cast<int>(blockIdx.y);
  const int64_t first = static_cast<int64_t>(blockIdx.x) * ids;
  const int live = static_cast<int>(p.n - first < ids ? p.n - first : ids);
  for (int i = t; i < live + 2; i += kSumThreads) {
    const int64_t at = first + i - 1;
    const Pair v = at >= 0 && at < p.n ? p.ids[at] : make_uint2(0xffffffffu, 0u);  // no key is that large
    s_key[i] = v.x;
    if (i > 0 && i <= live) s_unit[i - 1] = v.y;
  }
  uint32_t begun = 0;  // distinct keys before this run
  if (p.rows_out) {
    uint32_t all;
    begun = keys_begun(p, &all, s_sum);
    if (blockIdx.x == 0 && block == 0 && t == 0) *p.count_out = all;
  }
  __syncthreads();
  if (p.rows_out) {
    // s_rank[i]: the number of id i's key among all distinct ones
    const int per = (ids + kSumThreads - 1) / kSumThreads;
    const int a = t * per;
    uint32_t c = 0;
    for (int i = a; i < a + per && i < live; ++i) c += s_key[i + 1] < p.total && s_key[i + 1] != s_key[i] ? 1u : 0u;
    uint32_t x = c;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const uint32_t o = static_cast<uint32_t>(shfl_i32(static_cast<int>(x), lane_id() - d));
      if (lane_id() >= d) x += o;
    }
    if (lane_id() == kWave - 1) s_wave[t / kWave] = x;
    __syncthreads();
    uint32_t rank = begun + x - c;
    for (int w = 0; w < t / kWave; ++w) rank += s_wave[w];
    for (int i = a; i < a + per && i < live; ++i) {
      const uint32_t k = s_key[i + 1];
      if (k < p.total && k != s_key[i]) {
        if (block == 0) p.rows_out[rank] = k;
        ++rank;
      }
      s_rank[i] = rank - 1u;  // of a key that began before the run: begun - 1
    }
    if (a < live && live <= a + per && block == 0) p.last_rank[blockIdx.x] = rank - 1u;
    __syncthreads();
  }

  // Each lane group walks its ids. The row of a key is written where the key ends, unless it began in a group before.
  const int g = t >> p.log_lanes, lane = t & (lanes - 1);
  const int a = g * p.run, b = a + p.run < live ? a + p.run : live;
  int flag0 = 0, flag1 = 0;
  float acc[VEC];
  if (a < b) {
    uint32_t cur = s_key[a + 1];
    bool open = cur == s_key[a];  // began before
    int at = a;                   // an id of the current key
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    const auto finish = [&](int i) {  // the key of id i ends
      if (open) {
        flag0 = 1;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s_part[0][t * VEC + e] = acc[e];
      } else if (cur < p.total) {
        const uint32_t unit = s_unit[i];
        const int dim = S::width(p, fs, unit), c0 = first_column(block, lane, dim, VEC);
        if (c0 >= 0) {
          char* const row = S::target(p, fs, cur, unit, p.rows_out ? s_rank[i] : 0u);
          float v[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[e] = acc[e] * p.scale;
          with_out_type(p, [&](auto o) {
            store_vec<decltype(o), VEC>(row + static_cast<int64_t>(c0) * Elem<decltype(o)>::kBytes, dim - c0, v);
          });
        }
      }
      open = false;
    };
    for (int i0 = a; i0 < b; i0 += kSumAhead) {
      uint4 raw[kSumAhead];
      float w[kSumAhead];
#pragma unroll
      for (int u = 0; u < kSumAhead; ++u) {
        const int i = i0 + u;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        w[u] = 1.f;
        if (i < b && s_key[i + 1] < p.total) {
          const uint32_t unit = s_unit[i];
          int dim;
          const char* const row = S::row(p, fs, unit, &dim);
          const int c0 = first_column(block, lane, dim, VEC);
          if (c0 >= 0) raw[u] = load_raw<T, VEC>(row + static_cast<int64_t>(c0) * Elem<T>::kBytes, dim - c0);
          if (p.inv_len) w[u] = p.inv_len[unit];
        }
      }
#pragma unroll
      for (int u = 0; u < kSumAhead; ++u) {
        const int i = i0 + u;
        if (i < b) {
          const uint32_t k = s_key[i + 1];
          if (k != cur) {
            finish(at);
            cur = k;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
          }
          at = i;
          float v[VEC];
          unpack16(raw[u], v, T{});
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = __builtin_fmaf(v[e], w[u], acc[e]);
        }
      }
    }
    if (s_key[b + 1] == cur && cur < p.total) {  // goes on behind the group
      const int which = open ? 0 : 1;
      if (open) flag0 = 2;
      else flag1 = 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) s_part[which][t * VEC + e] = acc[e];
    } else {
      finish(at);
    }
  }
  if (lane == 0) {
    s_flag[0][g] = static_cast<uint8_t>(flag0);
    s_flag[1][g] = static_cast<uint8_t>(flag1);
  }
  __syncthreads();

  // Keys that cross lane groups, in the groups' order: a thread adds up one column's parts.
  const int slots = lanes * VEC;
  float* const mine = p.partial + (static_cast<int64_t>(block) * p.workgroups + blockIdx.x) * 2 * slots;
  for (int slot = t; slot < slots; slot += kSumThreads) {
    bool before = live > 0 && s_key[1] == s_key[0];  // the key began before this workgroup's run
    bool carrying = before;
    float carry = 0.f;
    const int l = slot / VEC, e = slot % VEC;
    for (int w = 0; w < groups; ++w) {
      const int f0 = s_flag[0][w];
      if (f0) {
        carry += s_part[0][w * slots + slot];
        if (f0 == 1) {
          if (before) {
            mine[slot] = carry;
          } else if (s_key[w * p.run + 1] < p.total) {
            const int i = w * p.run;
            const uint32_t unit = s_unit[i];
            const int dim = S::width(p, fs, unit), c0 = first_column(block, l, dim, VEC);
            if (c0 >= 0 && c0 + e < dim)
              put_sum(p, S::target(p, fs, s_key[i + 1], unit, p.rows_out ? s_rank[i] : 0u), c0 + e, carry * p.scale);
          }
          before = carrying = false;
          carry = 0.f;
        }
      }
      if (s_flag[1][w]) {
        carry = s_part[1][w * slots + slot];
        carrying = true;
      }
    }
    if (carrying) mine[before ? slot : slots + slot] = carry;
  }
}

// The same for rows of at least kWalkCols columns that lie one behind the other in grad: a whole wavefront
// walks its ids, so that keys, rows' addresses and the ends of keys are scalars: an id costs a load and its
// additions. (917,504 ids of 128 bf16 columns: 42 us. Lane groups of 16 lanes took 64, the end of a key in one of four
// groups stopping the others.) COLS columns a lane; a wavefront takes `run` ids, 128 at most.
constexpr int kWalkWaves = kSumThreads / kWave;
constexpr int kWalkBatches = 2;

// Addresses that went through lanes' registers are numbers: as pointers of no address space they would be loaded by flat
// instructions, which complete in no order, so that every wait is for all of them.
template <typename V>
using Global = __attribute__((address_space(1))) V;

template <typename T, int COLS>
struct LaneCols {  // COLS columns as loaded
  static constexpr int kBytes = COLS * Elem<T>::kBytes;
  static constexpr int kWords = (kBytes + 3) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const Global<char>* p) {
    if constexpr (kBytes == 2) w[0] = *reinterpret_cast<const Global<uint16_t>*>(p);
    else if constexpr (kBytes == 4) w[0] = *reinterpret_cast<const Global<u32_any>*>(p);
    else if constexpr (kBytes == 8) { const u32x2 v = *reinterpret_cast<const Global<u32x2_any>*>(p); w[0] = v.x, w[1] = v.y; }
    else { const u32x4 v = *reinterpret_cast<const Global<u32x4_any>*>(p); w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w; }
  }
  __device__ __forceinline__ float value(int e) const {
    if constexpr (Elem<T>::kBytes == 4) return __uint_as_float(w[e]);
    else if constexpr (std::is_same<T, bf16_t>::value) return __uint_as_float(e % 2 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
    else return f16_bits_to_f32(e % 2 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
  }
};

template <typename V, typename A>
__device__ __forceinline__ void put_global(Global<char>* p, V v) {
  *reinterpret_cast<Global<A>*>(p) = v;
}
template <typename OT, int COLS>
__device__ __forceinline__ void store_cols(Global<char>* p, const float* v) {
  constexpr int kBytes = COLS * Elem<OT>::kBytes;
  if constexpr (kBytes == 2) {
    put_global<uint16_t, uint16_t>(p, static_cast<uint16_t>(Packed<OT>::pair(v[0], 0.f)));
  } else {
    uint32_t w[kBytes / 4];
#pragma unroll
    for (int i = 0; i < kBytes / 4; ++i) {
      if constexpr (Elem<OT>::kBytes == 4) w[i] = __float_as_uint(v[i]);
      else w[i] = Packed<OT>::pair(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (kBytes == 4) {
      put_global<uint32_t, u32_any>(p, w[0]);
    } else if constexpr (kBytes == 8) {
      put_global<u32x2, u32x2_any>(p, u32x2{w[0], w[1]});
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 4; i += 4) put_global<u32x4, u32x4_any>(p + i * 4, u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]});
    }
  }
}

__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) {
  return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane));
}

// Wavefronts a SIMD that the registers leave room for: all of a launch of a million ids at once where an id's columns are few.
template <int BYTES>
constexpr int kWalkPerSimd = BYTES <= 4 ? 8 : 4;

template <typename T, typename OT, int COLS, bool MEAN>
__global__ void __launch_bounds__(kSumThreads, (kWalkPerSimd<COLS * Elem<T>::kBytes>)) grad_walk_kernel(const SumParams p, const SumFields fs) {
  constexpr int AHEAD = COLS * Elem<T>::kBytes >= 16 ? 8 : 16;  // rows whose loads are in flight
  __shared__ float s_part[2][kWalkWaves][kWave * COLS];
  __shared__ uint32_t s_flag[2][kWalkWaves], s_heads[kWalkWaves];
  __shared__ Global<char>* s_target[kWalkWaves];  // of each wavefront's first key
  __shared__ uint32_t s_sum[2][kSumThreads / kWave];
  const int t = static_cast<int>(threadIdx.x), lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(t / kWave);
  const int block = static_cast<int>(blockIdx.y);
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kWalkWaves + w) * p.run;  // the wavefront's
  const int64_t rest = p.n - first;
  const int have = rest <= 0 ? 0 : rest < p.run ? static_cast<int>(rest) : p.run;
  uint32_t key[kWalkBatches], unit[kWalkBatches];
  float weight[kWalkBatches];
  uint64_t begins[kWalkBatches];  // whose key is another than the id's before
  int live = 0;                   // ids that are not dropped: those come last
  uint32_t heads = 0;
  const uint32_t before = have && first > 0 ? p.ids[first - 1].x : 0xffffffffu;  // no key is that large
  const uint32_t behind = have && first + have < p.n ? p.ids[first + have].x : 0xffffffffu;
#pragma unroll
  for (int b = 0; b < kWalkBatches; ++b) {
    const int i = b * kWave + lane;
    const bool in = i < have;
    const Pair v = in ? p.ids[first + i] : make_uint2(0xffffffffu, 0u);
    key[b] = v.x;
    unit[b] = v.y;
  }
#pragma unroll
  for (int b = 0; b < kWalkBatches; ++b) {
    uint32_t prev = static_cast<uint32_t>(shfl_i32(static_cast<int>(key[b]), lane - 1));
    const uint32_t last = b == 0 ? before : lane_value(key[b > 0 ? b - 1 : 0], kWave - 1);
    if (lane == 0) prev = last;
    const bool kept = key[b] < p.total;
    begins[b] = __ballot(kept && key[b] != prev);
    live += __popcll(__ballot(kept));
    heads += static_cast<uint32_t>(__popcll(begins[b]));
    weight[b] = MEAN && kept ? p.inv_len[unit[b]] : 1.f;
  }
  const uint32_t first_key = lane_value(key[0], 0);
  bool open = live > 0 && before == first_key;  // the first key began before
  const int c0 = first_column(block, lane, p.dim, COLS);
  const uint32_t lane_at = static_cast<uint32_t>(c0 < 0 ? 0 : c0) * Elem<T>::kBytes;  // lanes without columns read the first
  uint64_t source[kWalkBatches];  // each id's row of grad
#pragma unroll
  for (int b = 0; b < kWalkBatches; ++b)
    source[b] = reinterpret_cast<uint64_t>(p.grad) + static_cast<uint64_t>(unit[b]) * (static_cast<uint64_t>(p.dim) * Elem<T>::kBytes);
  const auto of_lane = [&](uint64_t v, int i) {
    return reinterpret_cast<Global<char>*>((static_cast<uint64_t>(lane_value(static_cast<uint32_t>(v >> 32), i)) << 32) |
                                           lane_value(static_cast<uint32_t>(v), i));
  };
  LaneCols<T, COLS> rows[2][AHEAD];
  const auto fetch = [&](int b, int i0, LaneCols<T, COLS>* to) {
    const int last = (live - b * kWave < kWave ? live - b * kWave : kWave) - 1;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) to[u].load(of_lane(source[b], i0 + u < last ? i0 + u : last) + lane_at);
  };
  if (live > 0) fetch(0, 0, rows[0]);  // under way while the places of the sums are found
  uint32_t rank = 0;
  if (p.rows_out) {
    uint32_t all;
    if (lane == 0) s_heads[w] = heads;
    rank = keys_begun(p, &all, s_sum);
    if (p.heads_scanned) __syncthreads();
    if (blockIdx.x == 0 && block == 0 && t == 0) *p.count_out = all;
    for (int i = 0; i < w; ++i) rank += s_heads[i];
    rank = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(rank)));
  }
  // Where the sum of each id's key goes: a lane for an id, so that no key's end waits for its table's numbers.
  uint64_t target[kWalkBatches];
#pragma unroll
  for (int b = 0; b < kWalkBatches; ++b) {
    target[b] = 0;
    if (p.rows_out) {
      const uint32_t r = rank + static_cast<uint32_t>(__popcll(begins[b] & (~uint64_t{0} >> (kWave - 1 - lane)))) - 1u;
      if (block == 0 && ((begins[b] >> lane) & 1)) p.rows_out[r] = key[b];
      rank += static_cast<uint32_t>(__popcll(begins[b]));
      target[b] = reinterpret_cast<uint64_t>(p.out + static_cast<int64_t>(r) * p.dim * Elem<OT>::kBytes);
    } else if (key[b] < p.total) {
      target[b] = reinterpret_cast<uint64_t>(
          p.per_field ? Sums<T, SumFields>::target(p, fs, key[b], unit[b], 0u)
                      : p.out + static_cast<int64_t>(key[b]) * p.dim * Elem<OT>::kBytes);
    }
  }
  if (p.rows_out && block == 0 && have && lane == 0 && (w == kWalkWaves - 1 || rest <= p.run)) p.last_rank[blockIdx.x] = rank - 1u;
  uint32_t flag0 = 0, flag1 = 0;
  float acc[COLS];
#pragma unroll
  for (int e = 0; e < COLS; ++e) acc[e] = 0.f;
  Global<char>* const first_target = of_lane(target[0], 0);
  Global<char>* cur_target = first_target;
  const auto finish = [&]() {
    if (open) {
      flag0 = 1;
#pragma unroll
      for (int e = 0; e < COLS; ++e) s_part[0][w][lane * COLS + e] = acc[e];
      open = false;
    } else {
      float v[COLS];
#pragma unroll
      for (int e = 0; e < COLS; ++e) v[e] = acc[e] * p.scale;
      if (c0 >= 0) {
        store_cols<OT, COLS>(cur_target + static_cast<uint32_t>(c0) * Elem<OT>::kBytes, v);
      }
    }
#pragma unroll
    for (int e = 0; e < COLS; ++e) acc[e] = 0.f;
  };
#pragma unroll
  for (int b = 0; b < kWalkBatches; ++b) {
    const int now = live - b * kWave < kWave ? live - b * kWave : kWave;
    if (now <= 0) break;
    const auto add = [&](int i, const LaneCols<T, COLS>& row) {
      if ((begins[b] >> i) & 1) {
        if (b + i > 0) finish();
        cur_target = of_lane(target[b], i);
      }
      if constexpr (MEAN) {
        const float f = __uint_as_float(lane_value(__float_as_uint(weight[b]), i));
#pragma unroll
        for (int e = 0; e < COLS; ++e) acc[e] = __builtin_fmaf(row.value(e), f, acc[e]);
      } else {
#pragma unroll
        for (int e = 0; e < COLS; ++e) acc[e] += row.value(e);
      }
    };
    const auto add_all = [&](int i0, const LaneCols<T, COLS>* from) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (i0 + u < now) add(i0 + u, from[u]);
    };
    if (b > 0) fetch(b, 0, rows[0]);
    for (int i0 = 0; i0 < now; i0 += 2 * AHEAD) {
      if (i0 + AHEAD < now) fetch(b, i0 + AHEAD, rows[1]);
      add_all(i0, rows[0]);
      if (i0 + 2 * AHEAD < now) fetch(b, i0 + 2 * AHEAD, rows[0]);
      add_all(i0 + AHEAD, rows[1]);
    }
  }
  if (live > 0) {
    const uint32_t last_key = lane_value(live > kWave ? key[1] : key[0], (live - 1) % kWave);
    if (live == have && behind == last_key) {  // goes on behind the wavefront's ids
      const int which = open ? 0 : 1;
      if (open) flag0 = 2;
      else flag1 = 1;
#pragma unroll
      for (int e = 0; e < COLS; ++e) s_part[which][w][lane * COLS + e] = acc[e];
    } else {
      finish();
    }
  }
  if (lane == 0) {
    s_flag[0][w] = flag0;
    s_flag[1][w] = flag1;
    s_target[w] = first_target;
  }
  __syncthreads();

  // Keys that cross wavefronts, in their order; a thread adds up its columns' parts.
  constexpr int SLOTS = kWave * COLS;
  float* const mine = p.partial + (static_cast<int64_t>(block) * p.workgroups + blockIdx.x) * 2 * SLOTS;
  bool head = s_flag[0][0] != 0;  // the first key began before the workgroup's ids
  for (int slot = t; slot < SLOTS; slot += kSumThreads) {
    bool began = head, carrying = head;
    float carry = 0.f;
#pragma unroll
    for (int i = 0; i < kWalkWaves; ++i) {
      const uint32_t f0 = s_flag[0][i];
      if (f0) {
        carry += s_part[0][i][slot];
        if (f0 == 1) {
          if (began) {
            mine[slot] = carry;
          } else {
            const int at = first_column(block, slot / COLS, p.dim, COLS);
            if (at >= 0)
              {
              const float v = carry * p.scale;
              store_cols<OT, 1>(s_target[i] + static_cast<int64_t>(at + slot % COLS) * Elem<OT>::kBytes, &v);
            }
          }
          began = carrying = false;
          carry = 0.f;
        }
      }
      if (s_flag[1][i]) {
        carry = s_part[1][i][slot];
        carrying = true;
      }
    }
    if (carrying) mine[began ? slot : SLOTS + slot] = carry;
  }
}

// Keys that cross workgroups: the workgroup in whose run one begins and goes on adds up its own part and, in order of the
// runs, those of the runs it crosses.
template <typename FIELDS>
__global__ void __launch_bounds__(kSumThreads) grad_join_kernel(const SumParams p, const FIELDS fs) {
  using S = Sums<float, FIELDS>;  // (grad itself is not read)
  __shared__ float4 s_part[kSumThreads];
  const int t = static_cast<int>(threadIdx.x), lanes = 1 << p.log_lanes, groups = kSumThreads >> p.log_lanes;
  const int64_t ids = static_cast<int64_t>(groups) * p.run, first = static_cast<int64_t>(blockIdx.x) * ids;
  const int block = static_cast<int>(blockIdx.y);
  const int64_t next = first + ids;
  if (next >= p.n) return;
  // (all of these loads at once: each is a microsecond away)
  const int64_t h0 = (static_cast<int64_t>(blockIdx.x) + 1 + t) * ids;
  const uint32_t key = p.ids[next - 1].x, key_next = p.ids[next].x, key_first = p.ids[first].x;
  const uint32_t key_before = first > 0 ? p.ids[first - 1].x : 0xffffffffu;
  const uint32_t key_run = h0 < p.n ? p.ids[h0].x : 0xffffffffu;
  const uint32_t unit = p.ids[next - 1].y;
  const uint32_t rank = p.rows_out ? p.last_rank[blockIdx.x] : 0u;
  if (key >= p.total || key_next != key) return;           // ends with the run
  if (key_first == key && key_before == key) return;       // began in a run before
  // runs that begin with the key
  int follow = __syncthreads_count(key_run == key);
  for (int at = static_cast<int>(blockIdx.x) + 1 + kSumThreads; follow % kSumThreads == 0; at += kSumThreads) {
    const int64_t i = (static_cast<int64_t>(at) + t) * ids;
    const int c = __syncthreads_count(i < p.n && p.ids[i].x == key);
    follow += c;
    if (c < kSumThreads) break;
  }
  const int slots = lanes * p.lane_cols, quads = slots / 4, rows = kSumThreads / quads;  // rows of parts side by side
  const int64_t row_floats = 2 * static_cast<int64_t>(slots);
  const float* const mine = p.partial + (static_cast<int64_t>(block) * p.workgroups + blockIdx.x) * row_floats;
  const int q = t % quads, r = t / quads;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int h = r; h < follow; h += rows) {
    const float4 v = *reinterpret_cast<const float4*>(mine + (h + 1) * row_floats + q * 4);
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  s_part[t] = sum;
  __syncthreads();
  if (t >= quads) return;
  sum = *reinterpret_cast<const float4*>(mine + slots + q * 4);
  for (int i = 0; i < rows; ++i) {
    const float4 v = s_part[i * quads + q];
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  const int dim = S::width(p, fs, unit);
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
  char* const row = S::target(p, fs, key, unit, rank);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int slot = q * 4 + k, c0 = first_column(block, slot / p.lane_cols, dim, p.lane_cols);
    if (c0 >= 0 && c0 + slot % p.lane_cols < dim) put_sum(p, row, c0 + slot % p.lane_cols, v[k] * p.scale);
  }
}

// 1 / length of every bag (1 for empty ones: no id reads it).
__global__ void __launch_bounds__(256) grad_lengths_kernel(const GradSource s) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (j >= s.bags) return;
  const int64_t len = bag_edge(s, j, 1) - bag_edge(s, j, 0), f = s.by_batch.quotient(static_cast<uint32_t>(j));
  s.inv_len[(j - f * s.batch) * s.fields + f] = len > 0 ? 1.0f / static_cast<float>(len) : 1.0f;
}

__global__ void __launch_bounds__(kSortThreads) grad_fill_kernel(const GradFill f, int64_t* count_out) {
  fill_share(f, blockIdx.x);
  if (count_out && blockIdx.x == 0 && threadIdx.x == 0) *count_out = 0;
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
struct GradCall {
  GradSource src{};
  SumParams sum{};
  SumFields fields{};
  bool per_field = false;
  bool even = true;   // the units' rows lie one behind the other in grad, all of sum.dim columns
  bool walk = false;  // the plan's
  int32_t grad_dtype = 0, out_dtype = 0;
  int64_t capacity = 0;
  void* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

template <typename T, int COLS>
void launch_walk(const SumParams& p, const SumFields& fs, dim3 grid, hipStream_t s) {
  if constexpr (COLS * Elem<T>::kBytes <= 16) {
    with_type(p.out_dtype, [&](auto o) {
      using OT = decltype(o);
      if (p.inv_len) hipLaunchKernelGGL((grad_walk_kernel<T, OT, COLS, true>), grid, dim3(kSumThreads), 0, s, p, fs);
      else hipLaunchKernelGGL((grad_walk_kernel<T, OT, COLS, false>), grid, dim3(kSumThreads), 0, s, p, fs);
    });
  }
}
void launch_sums(const GradCall& c, int blocks, hipStream_t s) {
  const SumParams& p = c.sum;
  const dim3 grid(static_cast<unsigned>(p.workgroups), static_cast<unsigned>(blocks)), threads(kSumThreads);
  with_type(c.grad_dtype, [&](auto t) {
    using T = decltype(t);
    if (c.walk) {
      if (p.lane_cols == 1) launch_walk<T, 1>(p, c.fields, grid, s);
      else if (p.lane_cols == 2) launch_walk<T, 2>(p, c.fields, grid, s);
      else if (p.lane_cols == 4) launch_walk<T, 4>(p, c.fields, grid, s);
      else launch_walk<T, 8>(p, c.fields, grid, s);
    } else if (c.per_field) {
      hipLaunchKernelGGL((grad_sum_kernel<T, SumFields>), grid, threads, 0, s, p, c.fields);
    } else {
      hipLaunchKernelGGL((grad_sum_kernel<T, NoFields>), grid, threads, 0, s, p, NoFields{});
    }
  });
  if (p.workgroups == 1) return;
  if (c.per_field) hipLaunchKernelGGL((grad_join_kernel<SumFields>), grid, threads, 0, s, p, c.fields);
  else hipLaunchKernelGGL((grad_join_kernel<NoFields>), grid, threads, 0, s, p, NoFields{});
}

// The sort and the sums of a call whose arguments are checked.
int run_gradient(GradCall& c, hipStream_t s) {
  const int64_t n = c.src.n;
  const bool compact = c.sum.rows_out != nullptr;
  GradFill fill{};
  int64_t shares = 0;
  const auto fill_table = [&](char* data, int64_t rows, int64_t row_bytes, int64_t row_stride) {
    for (int k = 0; k < fill.tables; ++k)
      if (fill.data[k] == data) return;  // fields that share a table
    const int i = fill.tables++;
    fill.data[i] = data;
    fill.bytes[i] = rows * row_bytes;
    fill.row_bytes[i] = row_bytes;
    fill.row_stride[i] = row_stride;
    shares += (fill.bytes[i] + kFillShare - 1) / kFillShare;
  };
  const int eb = dtype_bytes(c.out_dtype);
  if (compact) {
    fill.value = 0xffffffffu;
    fill_table(reinterpret_cast<char*>(c.sum.rows_out), c.capacity, 8, 8);
  } else if (c.per_field) {
    for (int f = 0; f < c.src.fields; ++f)
      if (c.fields.data[f]) fill_table(c.fields.data[f], c.src.rows[f], static_cast<int64_t>(c.fields.dim[f]) * eb, c.fields.stride[f] * eb);
  } else {
    fill_table(c.sum.out, c.src.rows[0], static_cast<int64_t>(c.sum.dim) * eb, static_cast<int64_t>(c.sum.dim) * eb);
  }
  if (shares > kGradMostShares) return set_error(CTI_EBAG_EUNSUPPORTED, "a gradient of more than 2^38 - 2^25 bytes");
  if (n == 0) {
    hipLaunchKernelGGL(grad_fill_kernel, dim3(static_cast<unsigned>(shares > 0 ? shares : 1)), dim3(kSortThreads), 0, s, fill,
                       c.sum.count_out);
    return check_launch("gradient");
  }

  c.src.by_batch = ChunkDivide::by(static_cast<uint32_t>(c.src.batch));
  const GradPlan plan = grad_plan(n, c.src.inv_len ? c.src.bags : 0, c.sum.dim, dtype_bytes(c.grad_dtype), c.src.total, c.even);
  char* const ws = static_cast<char*>(c.workspace);
  Pair* const buf[2] = {reinterpret_cast<Pair*>(ws + plan.ids[0]), reinterpret_cast<Pair*>(ws + plan.ids[1])};
  uint32_t* const counts = reinterpret_cast<uint32_t*>(ws + plan.counts);
  uint32_t* const totals = reinterpret_cast<uint32_t*>(ws + plan.totals);
  if (c.src.inv_len) {
    c.src.inv_len = reinterpret_cast<float*>(ws + plan.inv_len);
    c.sum.inv_len = c.src.inv_len;
    hipLaunchKernelGGL(grad_lengths_kernel, dim3(static_cast<unsigned>((c.src.bags + 255) / 256)), dim3(256), 0, s, c.src);
  }
  // the shares of the fill are dealt to the sort's launches evenly
  const bool scan = plan.tiles > kGradTilesUnscanned;
  const bool bags = c.src.offsets != nullptr, alone = bags && n <= kGradIdsAlone;
  const int range_bits = alone ? 0 : grad_range_bits(n, plan.bits);
  const int launches = alone ? 1 : range_bits > 0 ? (bags ? 2 : 1)
                             : (scan ? 3 : 2) * static_cast<int>(ceil_div(plan.bits, plan.digit_bits));
  int launch = 0;
  const auto grid = [&](int64_t groups) {
    fill.sort_groups = static_cast<int32_t>(groups);
    fill.first_share = static_cast<int32_t>(shares * launch / launches);
    ++launch;
    return dim3(static_cast<unsigned>(groups + shares * launch / launches - fill.first_share));
  };
  const dim3 threads(kSortThreads);
  int at = 0;
  if (alone) {
    const dim3 g = grid(1);
    if (n <= 4096) hipLaunchKernelGGL((grad_sort_tile_kernel<512, 8>), g, threads, 0, s, c.src, buf[0], plan.bits, plan.digit_bits, fill);
    else hipLaunchKernelGGL((grad_sort_tile_kernel<1024, 8>), g, dim3(1024), 0, s, c.src, buf[0], plan.bits, plan.digit_bits, fill);
  } else if (range_bits > 0) {
    const Pair* keys = nullptr;
    if (bags) {
      const dim3 g = grid(ceil_div(n, kSortThreads * kRangeKeyItems));
      hipLaunchKernelGGL((grad_keys_kernel<kRangeKeyItems>), g, threads, 0, s, c.src, buf[0], static_cast<uint32_t*>(nullptr), 0, fill);
      keys = buf[0];
      at = 1;
    }
    const dim3 g = grid(int64_t{1} << range_bits);
    const int key_bits = plan.bits - range_bits;
    if (n <= 8 * kRangeThreads) hipLaunchKernelGGL((grad_sort_ranges_kernel<8>), g, dim3(kRangeThreads), 0, s, c.src, keys, buf[at], key_bits, fill);
    else if (n <= 16 * kRangeThreads) hipLaunchKernelGGL((grad_sort_ranges_kernel<16>), g, dim3(kRangeThreads), 0, s, c.src, keys, buf[at], key_bits, fill);
    else hipLaunchKernelGGL((grad_sort_ranges_kernel<32>), g, dim3(kRangeThreads), 0, s, c.src, keys, buf[at], key_bits, fill);
  } else {
    const int bits = plan.digit_bits;
    for (int shift = 0; shift < plan.bits; shift += bits) {
      dim3 g = grid(plan.tiles);
      if (shift == 0) hipLaunchKernelGGL((grad_keys_kernel<kItems>), g, threads, 0, s, c.src, buf[0], counts, bits, fill);
      else hipLaunchKernelGGL(grad_count_kernel, g, threads, 0, s, buf[at], n, shift, bits, counts, fill);
      if (scan) {
        g = grid(ceil_div(int64_t{1} << bits, kWave));
        hipLaunchKernelGGL(grad_scan_kernel, g, dim3(kScanThreads), 0, s, counts, totals, plan.tiles, bits, fill);
      }
      g = grid(plan.tiles);
      hipLaunchKernelGGL(grad_scatter_kernel, g, threads, 0, s, buf[at], buf[1 - at], n, shift, bits, counts,
                         scan ? totals : nullptr, fill);
      at = 1 - at;
    }
  }
  SumParams& p = c.sum;
  p.ids = buf[at];
  p.n = n;
  p.total = c.src.total;
  p.partial = reinterpret_cast<float*>(ws + plan.partial);
  c.walk = plan.walk;
  p.log_lanes = plan.log_lanes;
  p.lane_cols = plan.lane_cols;
  p.run = plan.run;
  p.workgroups = static_cast<int32_t>(plan.workgroups);
  p.fields = c.src.fields;
  p.per_field = c.per_field;
  p.by_fields = ChunkDivide::by(static_cast<uint32_t>(c.src.fields));
  if (compact) {
    uint32_t* const heads = reinterpret_cast<uint32_t*>(ws + plan.heads);
    p.heads = heads;
    p.last_rank = reinterpret_cast<uint32_t*>(ws + plan.last_rank);
    hipLaunchKernelGGL(grad_heads_kernel, dim3(static_cast<unsigned>(plan.workgroups)), dim3(kSumThreads), 0, s, p.ids, n, p.total,
                       static_cast<int>(plan.run * (kSumThreads >> plan.log_lanes)), heads);
    p.heads_scanned = plan.workgroups > kGradHeadsUnscanned;
    if (p.heads_scanned)
      hipLaunchKernelGGL(grad_heads_scan_kernel, dim3(1), dim3(kScanThreads), 0, s, heads, plan.workgroups);
  }
  p.out_dtype = c.out_dtype;
  launch_sums(c, plan.blocks, s);
  return check_launch("gradient");
}

// Checks that every form of the gradient shares. `rows`: of all tables; padding may be -1.
int check_gradient(int32_t grad_dtype, int32_t out_dtype, int32_t index_type, int64_t n, int64_t units, int64_t dim,
                   bool compact, const int64_t* count_out, int64_t rows, int64_t capacity) {
  if (!float_dtype(grad_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown gradient dtype code %d", grad_dtype);
  if (!float_dtype(out_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown output dtype code %d", out_dtype);
  if (index_type != CTI_EBAG_I64 && index_type != CTI_EBAG_I32) return set_error(CTI_EBAG_EINVAL, "unknown index type %d", index_type);
  if (n < 0) return set_error(CTI_EBAG_EINVAL, "the number of ids must be >= 0 (got %lld)", (long long)n);
  if (dim < 1) return set_error(CTI_EBAG_EINVAL, "dim must be >= 1 (got %lld)", (long long)dim);
  if (dim > kGradMostDim) return set_error(CTI_EBAG_EUNSUPPORTED, "dim %lld > 2^22", (long long)dim);
  if (rows < 1) return set_error(CTI_EBAG_EINVAL, "rows must be >= 1 (got %lld)", (long long)rows);
  if (rows >= kGradMostRows) return set_error(CTI_EBAG_EUNSUPPORTED, "%lld rows of tables (2^31 - 1 at most)", (long long)rows);
  if (n > kGradMostIds || units > kGradMostIds)
    return set_error(CTI_EBAG_EUNSUPPORTED, "%lld ids in %lld bags (2^30 of each at most)", (long long)n, (long long)units);
  if (compact != (count_out != nullptr)) return set_error(CTI_EBAG_EINVAL, "rows_out and count_out are given together or not at all");
  if (compact && capacity < (n < rows ? n : rows))
    return set_error(CTI_EBAG_EINVAL, "capacity %lld for the rows of %lld ids in tables of %lld", (long long)capacity, (long long)n,
                     (long long)rows);
  return CTI_EBAG_OK;
}

int check_workspace(const GradCall& c, int64_t bags, int64_t dim) {
  if (c.src.n == 0) return CTI_EBAG_OK;
  const int64_t need = grad_workspace_bytes(c.src.n, bags, dim, c.src.total);
  if (!c.workspace || c.workspace_bytes < need)
    return set_error(CTI_EBAG_EWORKSPACE, "workspace of %lld bytes, %lld needed", (long long)(c.workspace ? c.workspace_bytes : 0),
                     (long long)need);
  if (reinterpret_cast<uintptr_t>(c.workspace) % 16) return set_error(CTI_EBAG_EINVAL, "workspace is not 16-byte aligned");
  return CTI_EBAG_OK;
}

}  // namespace
}  // namespace cti

using namespace cti;

extern "C" int cti_ebag_lookup(const void* ids, int32_t index_type, int64_t n, const void* weight, int32_t dtype, int64_t rows,
                               int64_t row_stride, int32_t dim, float scale, void* out, int32_t out_dtype, void* stream) {
  clear_error();
  if (!float_dtype(dtype)) return set_error(CTI_EBAG_EINVAL, "unknown table dtype code %d", dtype);
  if (!float_dtype(out_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown output dtype code %d", out_dtype);
  if (index_type != CTI_EBAG_I64 && index_type != CTI_EBAG_I32) return set_error(CTI_EBAG_EINVAL, "unknown index type %d", index_type);
  if (n < 0) return set_error(CTI_EBAG_EINVAL, "the number of ids must be >= 0 (got %lld)", (long long)n);
  if (dim < 1) return set_error(CTI_EBAG_EINVAL, "dim must be >= 1 (got %d)", dim);
  if (rows < 1) return set_error(CTI_EBAG_EINVAL, "rows must be >= 1 (got %lld)", (long long)rows);
  if (row_stride < dim) return set_error(CTI_EBAG_EINVAL, "row_stride %lld < dim %d", (long long)row_stride, dim);
  if (n == 0) return CTI_EBAG_OK;
  if (!ids || !weight || !out) return set_error(CTI_EBAG_EINVAL, "NULL device pointer among ids/weight/out");
  LookupParams p;
  p.weight = static_cast<const char*>(weight);
  p.rows = rows;
  p.row_bytes = row_stride * dtype_bytes(dtype);
  p.dim = dim;
  p.ids64 = index_type == CTI_EBAG_I64;
  p.per_row = (static_cast<uint32_t>(dim) + 7) / 8;
  p.div = ChunkDivide::by(p.per_row);
  p.scale = scale;
  p.stream_out = n * dim * dtype_bytes(out_dtype) >= kStreamOutBytes;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t per_launch = kMostChunks / p.per_row;  // rows
  for (int64_t i = 0; i < n; i += per_launch) {
    const int64_t now = n - i < per_launch ? n - i : per_launch;
    p.ids = static_cast<const char*>(ids) + i * (p.ids64 ? 8 : 4);
    p.out = static_cast<char*>(out) + i * dim * dtype_bytes(out_dtype);
    p.chunks = static_cast<uint32_t>(now * p.per_row);
    const dim3 grid(static_cast<unsigned>(ceil_div(p.chunks, kLookupThreads * kLookupChunks))), block(kLookupThreads);
    with_types(dtype, out_dtype, [&](auto t, auto o) {
      hipLaunchKernelGGL((lookup_kernel<decltype(t), decltype(o)>), grid, block, 0, s, p);
    });
  }
  return check_launch("lookup");
}

extern "C" int64_t cti_ebag_backward_workspace_bytes(int64_t nnz, int64_t bags, int64_t rows, int32_t dim, int32_t pooling) {
  if (nnz <= 0 || bags < 0 || rows < 1 || dim < 1 || nnz > kGradMostIds || bags > kGradMostIds || rows >= kGradMostRows) return 0;
  const int64_t b = pooling == CTI_EBAG_MEAN ? bags : 0;
  return grad_workspace_bytes(nnz, b, dim, static_cast<uint32_t>(rows));
}

extern "C" int cti_ebag_lookup_backward(const void* grad, int32_t grad_dtype, const void* ids, int32_t index_type, int64_t n,
                                        int64_t rows, int32_t dim, float scale, int64_t padding_idx, void* out, int32_t out_dtype,
                                        int64_t* rows_out, int64_t* count_out, int64_t capacity, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_gradient(grad_dtype, out_dtype, index_type, n, n, dim, rows_out != nullptr, count_out, rows, capacity);
  if (rc != CTI_EBAG_OK) return rc;
  if (padding_idx < -1 || padding_idx >= rows)
    return set_error(CTI_EBAG_EINVAL, "padding_idx %lld outside [0, %lld)", (long long)padding_idx, (long long)rows);
  if ((n > 0 && (!grad || !ids)) || (!out && (n > 0 || !rows_out)))
    return set_error(CTI_EBAG_EINVAL, "NULL device pointer among grad/ids/out");
  GradCall c;
  c.src.ids = ids;
  c.src.n = n;
  c.src.batch = n;
  c.src.bags = n;
  c.src.fields = 1;
  c.src.ids64 = index_type == CTI_EBAG_I64;
  c.src.total = static_cast<uint32_t>(rows);
  c.src.padding = padding_idx;
  c.src.rows[0] = static_cast<uint32_t>(rows);
  c.sum.grad = static_cast<const char*>(grad);
  c.sum.dim = dim;
  c.sum.scale = scale;
  c.sum.out = static_cast<char*>(out);
  c.sum.rows_out = rows_out;
  c.sum.count_out = count_out;
  c.grad_dtype = grad_dtype;
  c.out_dtype = out_dtype;
  c.capacity = capacity;
  c.workspace = workspace;
  c.workspace_bytes = workspace_bytes;
  rc = check_workspace(c, 0, dim);
  return rc != CTI_EBAG_OK ? rc : run_gradient(c, static_cast<hipStream_t>(stream));
}

extern "C" int cti_ebag_fused_all_slots_backward(const void* grad, int32_t grad_dtype, const void* values, int32_t index_type,
                                                 const void* val_offsets, const void* row_offsets, int32_t offset_type,
                                                 int64_t batch_size, int32_t num_slots, int32_t emb_dim, int64_t max_idx,
                                                 int64_t nnz, int32_t pooling, int64_t padding_idx, void* out, int32_t out_dtype,
                                                 int64_t* rows_out, int64_t* count_out, int64_t capacity, void* workspace,
                                                 int64_t workspace_bytes, void* stream) {
  clear_error();
  if (batch_size < 0) return set_error(CTI_EBAG_EINVAL, "batch_size must be >= 0 (got %lld)", (long long)batch_size);
  if (num_slots < 0) return set_error(CTI_EBAG_EINVAL, "num_slots must be >= 0 (got %d)", num_slots);
  if (max_idx < 0) return set_error(CTI_EBAG_EINVAL, "max_idx must be >= 0 (got %lld)", (long long)max_idx);
  if (offset_type != CTI_EBAG_I64 && offset_type != CTI_EBAG_I32) return set_error(CTI_EBAG_EINVAL, "unknown offset type %d", offset_type);
  if (pooling != CTI_EBAG_SUM && pooling != CTI_EBAG_MEAN) return set_error(CTI_EBAG_EINVAL, "unknown pooling mode %d", pooling);
  if (batch_size > kGradMostIds) return set_error(CTI_EBAG_EUNSUPPORTED, "batch_size %lld (2^30 at most)", (long long)batch_size);
  if (max_idx >= kGradMostRows) return set_error(CTI_EBAG_EUNSUPPORTED, "max_idx %lld", (long long)max_idx);
  const int64_t rows = max_idx + 1, bags = batch_size * num_slots;
  int rc = check_gradient(grad_dtype, out_dtype, index_type, nnz, bags, emb_dim, rows_out != nullptr, count_out, rows, capacity);
  if (rc != CTI_EBAG_OK) return rc;
  if (padding_idx < -1 || padding_idx >= rows)
    return set_error(CTI_EBAG_EINVAL, "padding_idx %lld outside [0, %lld)", (long long)padding_idx, (long long)rows);
  const bool any = nnz > 0 && bags > 0;
  if ((any && (!grad || !values || !val_offsets || !row_offsets)) || (!out && (any || !rows_out)))
    return set_error(CTI_EBAG_EINVAL, "NULL device pointer among grad/values/val_offsets/row_offsets/out");
  GradCall c;
  c.src.ids = values;
  c.src.val_offsets = val_offsets;
  c.src.offsets = row_offsets;
  c.src.n = any ? nnz : 0;
  c.src.batch = batch_size;
  c.src.bags = bags;
  c.src.fields = num_slots > 0 ? num_slots : 1;
  c.src.ids64 = index_type == CTI_EBAG_I64;
  c.src.offs64 = offset_type == CTI_EBAG_I64;
  c.src.total = static_cast<uint32_t>(rows);
  c.src.padding = padding_idx;
  c.src.rows[0] = static_cast<uint32_t>(rows);
  c.src.inv_len = pooling == CTI_EBAG_MEAN ? static_cast<float*>(workspace) : nullptr;
  c.sum.grad = static_cast<const char*>(grad);
  c.sum.dim = emb_dim;
  c.sum.scale = 1.f;
  c.sum.out = static_cast<char*>(out);
  c.sum.rows_out = rows_out;
  c.sum.count_out = count_out;
  c.grad_dtype = grad_dtype;
  c.out_dtype = out_dtype;
  c.capacity = capacity;
  c.workspace = workspace;
  c.workspace_bytes = workspace_bytes;
  rc = check_workspace(c, pooling == CTI_EBAG_MEAN ? bags : 0, emb_dim);
  return rc != CTI_EBAG_OK ? rc : run_gradient(c, static_cast<hipStream_t>(stream));
}

extern "C" int cti_ebag_backward_fields(const void* grad, int32_t grad_dtype, int64_t grad_row_stride, const void* values,
                                        int32_t index_type, int64_t nnz, const int64_t* offsets, int64_t batch_size,
                                        int32_t num_fields, const cti_ebag_table* tables, uint64_t wanted, int32_t pooling,
                                        int64_t padding_idx, int32_t out_dtype, void* out, int64_t* rows_out, int64_t* count_out,
                                        int64_t capacity, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (batch_size < 0) return set_error(CTI_EBAG_EINVAL, "batch_size must be >= 0 (got %lld)", (long long)batch_size);
  if (num_fields < 1) return set_error(CTI_EBAG_EINVAL, "num_fields must be >= 1 (got %d)", num_fields);
  if (num_fields > kMaxFields) return set_error(CTI_EBAG_EUNSUPPORTED, "num_fields %d > %d", num_fields, kMaxFields);
  if (!tables) return set_error(CTI_EBAG_EINVAL, "tables is NULL");
  if (pooling != CTI_EBAG_SUM && pooling != CTI_EBAG_MEAN) return set_error(CTI_EBAG_EINVAL, "unknown pooling mode %d", pooling);
  if (batch_size > kGradMostIds) return set_error(CTI_EBAG_EUNSUPPORTED, "batch_size %lld (2^30 at most)", (long long)batch_size);
  if (num_fields < kMaxFields) wanted &= (uint64_t{1} << num_fields) - 1;
  if (!wanted) return set_error(CTI_EBAG_EINVAL, "no field has a gradient");
  const bool compact = rows_out != nullptr;
  const int first_wanted = __builtin_ctzll(wanted);
  GradCall c;
  c.per_field = true;
  int64_t rows = 0, dim = 0;
  for (int f = 0; f < num_fields; ++f) {
    const cti_ebag_table& t = tables[f];
    const bool with = (wanted >> f) & 1;
    if (with && t.rows < 1) return set_error(CTI_EBAG_EINVAL, "tables[%d].rows must be >= 1 (got %lld)", f, (long long)t.rows);
    if (t.dim < 1) return set_error(CTI_EBAG_EINVAL, "tables[%d].dim must be >= 1 (got %d)", f, t.dim);
    if (with && t.row_stride < t.dim)
      return set_error(CTI_EBAG_EINVAL, "tables[%d].row_stride %lld < dim %d", f, (long long)t.row_stride, t.dim);
    if (t.out_col < 0 || t.out_col + static_cast<int64_t>(t.dim) > grad_row_stride)
      return set_error(CTI_EBAG_EINVAL, "tables[%d]: columns [%d, %lld) outside the gradient's row of %lld", f, t.out_col,
                       (long long)t.out_col + t.dim, (long long)grad_row_stride);
    c.even = c.even && t.dim == tables[0].dim && t.out_col == static_cast<int64_t>(f) * t.dim;
    c.fields.dim[f] = t.dim;
    c.fields.col[f] = t.out_col;
    if (!with) continue;
    if (!t.data) return set_error(CTI_EBAG_EINVAL, "tables[%d].data is NULL", f);
    if (compact && t.dim != tables[first_wanted].dim)
      return set_error(CTI_EBAG_EUNSUPPORTED, "rows_out needs tables of one width (%d, %d)", tables[first_wanted].dim, t.dim);
    if (padding_idx < -1 || padding_idx >= t.rows)
      return set_error(CTI_EBAG_EINVAL, "padding_idx %lld outside tables[%d]", (long long)padding_idx, f);
    int same = f;
    for (int k = first_wanted; k < f && same == f; ++k)
      if (((wanted >> k) & 1) && tables[k].data == t.data) same = k;
    if (same < f && (tables[same].rows != t.rows || tables[same].dim != t.dim || tables[same].row_stride != t.row_stride))
      return set_error(CTI_EBAG_EINVAL, "tables[%d] and tables[%d] share data but not their shape", same, f);
    c.src.base[f] = same < f ? c.src.base[same] : static_cast<uint32_t>(rows);
    if (same == f) {
      if (t.rows >= kGradMostRows || rows + t.rows >= kGradMostRows)
        return set_error(CTI_EBAG_EUNSUPPORTED, "more than 2^31 - 2 rows of tables");
      rows += t.rows;
    }
    c.src.rows[f] = static_cast<uint32_t>(t.rows);
    c.fields.data[f] = static_cast<char*>(const_cast<void*>(t.data));
    c.fields.stride[f] = t.row_stride;
    c.fields.base[f] = c.src.base[f];
    if (t.dim > dim) dim = t.dim;
  }
  // Fields without a gradient: a table of one row, whose number is the dropped ids' key.
  for (int f = 0; f < num_fields; ++f) {
    if ((wanted >> f) & 1) continue;
    c.src.base[f] = static_cast<uint32_t>(rows);
    c.src.rows[f] = 1;
  }
  c.even = c.even && grad_row_stride == num_fields * dim;
  const int64_t bags = batch_size * num_fields;
  int rc = check_gradient(grad_dtype, out_dtype, index_type, nnz, bags, dim, compact, count_out, rows, capacity);
  if (rc != CTI_EBAG_OK) return rc;
  const bool any = nnz > 0 && bags > 0;
  if ((any && (!grad || !values || !offsets)) || (compact && any && !out))
    return set_error(CTI_EBAG_EINVAL, "NULL device pointer among grad/values/offsets/out");
  c.src.ids = values;
  c.src.offsets = offsets;
  c.src.n = any ? nnz : 0;
  c.src.batch = batch_size;
  c.src.bags = bags;
  c.src.fields = num_fields;
  c.src.ids64 = index_type == CTI_EBAG_I64;
  c.src.offs64 = 1;
  c.src.per_field = 1;
  c.src.total = static_cast<uint32_t>(rows);
  c.src.padding = padding_idx;
  c.src.inv_len = pooling == CTI_EBAG_MEAN ? static_cast<float*>(workspace) : nullptr;
  c.sum.grad = static_cast<const char*>(grad);
  c.sum.grad_stride = grad_row_stride;
  c.sum.dim = static_cast<int32_t>(dim);
  c.sum.scale = 1.f;
  c.sum.out = static_cast<char*>(out);
  c.sum.rows_out = rows_out;
  c.sum.count_out = count_out;
  c.grad_dtype = grad_dtype;
  c.out_dtype = out_dtype;
  c.capacity = capacity;
  c.workspace = workspace;
  c.workspace_bytes = workspace_bytes;
  rc = check_workspace(c, pooling == CTI_EBAG_MEAN ? bags : 0, dim);
  return rc != CTI_EBAG_OK ? rc : run_gradient(c, static_cast<hipStream_t>(stream));
}

extern "C" int cti_ebag_backward(const void* grad, int32_t grad_dtype, int64_t grad_row_stride, const void* values,
                                 int32_t index_type, int64_t nnz, const int64_t* offsets, int64_t batch_size, int32_t num_fields,
                                 const cti_ebag_table* tables, int32_t pooling, int64_t padding_idx, int32_t out_dtype, void* out,
                                 int64_t* rows_out, int64_t* count_out, int64_t capacity, void* workspace, int64_t workspace_bytes,
                                 void* stream) {
  return cti_ebag_backward_fields(grad, grad_dtype, grad_row_stride, values, index_type, nnz, offsets, batch_size, num_fields, tables,
                                  ~uint64_t{0}, pooling, padding_idx, out_dtype, out, rows_out, count_out, capacity, workspace,
                                  workspace_bytes, stream);
}
