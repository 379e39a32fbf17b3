// Matrix product in 8-bit integers for MI355X (gfx950), with a scale for each row of x (token) and each
// row of the weight (output channel), and its gated form:
//   t[m, n] = sum_k q[m, k] * w[n, k]                        (exact in int32: K <= kLinear8MaxK)
//   v[m, n] = (t[m, n] * scale[m]) * wscale[n] + bias[n]     (fp32)
//   plain:  y[m, n] = v[m, n]
//   gated:  y[m, n] = act(v[m, n]) * v[m, N + n]             (the weight's 2 N rows: gates, then values)
// with one rounding to y's type. Integer sums do not depend on their order, so results are bit for bit the
// same whatever the tiles and splits.
//
// The products run on v_mfma_i32_16x16x64_i8 with the weight as the first operand: lane l supplies
// w[n0 + l % 16][16 bytes] and q[m0 + l % 16][16 bytes], its 16 bytes being chunk l / 16 of 4 of a 64-byte
// step (any assignment of k to chunks will do as long as both operands use it), and receives
// t[m0 + l % 16][n0 + 4 (l / 16) + r], r < 4: four consecutive columns of one row.
//
// Forms, chosen by linear8_plan:
//   rows   few rows or few outputs: bound by reading the weight, or by the way to memory and back. A workgroup owns
//          16 rows by 16 columns (gated: 16 gates and their 16 values); its wavefronts split K, load both operands
//          straight to registers and add their sums through LDS.
//   rings  tiles through LDS, a ring of four steps loaded straight to it: 64 x 64, two to a CU; 128 x 64 and 128 x 128, one.
//   tiles  128 x 128 and 256 x 256 tiles, two steps in LDS, fragments read half a step ahead.
//   any    128 x 128 tiles of operands at any address and any width, through registers: without a workspace. With one,
//          operands of odd widths are copied to rows of whole steps first.
// Where tiles would leave CUs idle, K is split over workgroups, each writing int32 partial sums to the caller's
// workspace, added by a second kernel.
#include <stdint.h>

#include "ebag_device.h"
#include "ebag_internal.h"
#include "ebag_rules.h"

namespace cti {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef i32x4 i32x4_any __attribute__((aligned(1)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

constexpr int kStep = kLinear8Step;  // bytes of K per step
constexpr int kXcds = 8;

struct Linear8Params {
  const int8_t* x;      // [M, K]
  const float* scale;   // [M]
  const int8_t* w;      // [N or 2 N, K]
  const float* wscale;  // [N or 2 N]
  const void* bias;     // [N or 2 N] or NULL
  char* y;              // [M, N]
  int32_t* part;        // split K: int32 partial sums [splits, M, linear8_part_cols() (gated: twice)]; NULL: no split
  int64_t M;
  int32_t N;            // columns of y
  int32_t K;            // bytes of a row of x and w
  int32_t n_begin, n_end;  // columns of y of this launch
  int32_t tiles_m, tiles_n;
  int32_t split_steps;  // split K: steps per split; split s is blockIdx.y
  int32_t bias_dtype, y_dtype;
  int32_t gate;         // CTI_EBAG_GATE_*
};

// ---------------------------------------------------------------------------------------------
// Epilogue
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ float load_bias(const Linear8Params& p, int n) {
  const char* const b = static_cast<const char*>(p.bias);
  switch (p.bias_dtype) {
    case CTI_EBAG_F32: return Elem<float>::load(b + static_cast<int64_t>(n) * 4);
    case CTI_EBAG_BF16: return Elem<bf16_t>::load(b + static_cast<int64_t>(n) * 2);
    default: return Elem<f16_t>::load(b + static_cast<int64_t>(n) * 2);
  }
}

// act(g) in fp32: silu with exp(-|g|), which cannot overflow; gelu with erfc, without the cancellation of 1 + erf.
template <int GATE>
__device__ __forceinline__ float activate(float g) {
  if constexpr (GATE == CTI_EBAG_GATE_SILU) {
    const float e = expf(-fabsf(g));
    return (g < 0.f ? g * e : g) / (1.0f + e);
  } else if constexpr (GATE == CTI_EBAG_GATE_GELU) {
    return 0.5f * g * erfcf(g * -0.70710678118654752f);
  } else {
    return g < 0.f ? 0.f : g;  // NaN stays NaN
  }
}

// Weight scales and bias of C (a multiple of 4) consecutive columns from `row` of the weight on, `live` of which
// exist (1 at least; the others repeat the last).
template <int C>
struct Columns {
  float scale[C], bias[C];
  __device__ __forceinline__ void load(const Linear8Params& p, int row, int live) {
    if (live >= C) {
#pragma unroll
      for (int i = 0; i < C; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4_any*>(p.wscale + row + i);
#pragma unroll
        for (int r = 0; r < 4; ++r) scale[i + r] = v[r];
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) scale[i] = p.wscale[row + (i < live ? i : live - 1)];
    }
#pragma unroll
    for (int i = 0; i < C; ++i) bias[i] = 0.f;
    if (p.bias) {
#pragma unroll
      for (int i = 0; i < C; ++i) bias[i] = load_bias(p, row + (i < live ? i : live - 1));
    }
  }
  __device__ __forceinline__ float apply(int i, int t, float sm) const {
    return static_cast<float>(t) * sm * scale[i] + bias[i];
  }
};

// y[i], i < live, of C consecutive columns, rounded to YT.
template <typename YT, int C>
__device__ __forceinline__ void store_columns(char* y, int64_t at, const float* v, int live) {
  if constexpr (std::is_same<YT, float>::value) {
    float* const to = reinterpret_cast<float*>(y) + at;
    if (live >= C) {
#pragma unroll
      for (int i = 0; i < C; i += 4) *reinterpret_cast<f32x4_any*>(to + i) = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < C - 1; ++i)
        if (i < live) to[i] = v[i];
    }
  } else {
    uint32_t w[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; ++i)
      w[i] = std::is_same<YT, bf16_t>::value ? pack_bf16x2(v[2 * i], v[2 * i + 1]) : pack_f16x2(v[2 * i], v[2 * i + 1]);
    uint16_t* const to = reinterpret_cast<uint16_t*>(y) + at;
    if (live >= C) {
      if constexpr (C % 8 == 0) {
#pragma unroll
        for (int i = 0; i < C / 2; i += 4) *reinterpret_cast<u32x4_any*>(to + 2 * i) = u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]};
      } else {
#pragma unroll
        for (int i = 0; i < C / 2; i += 2) *reinterpret_cast<u32x2_any*>(to + 2 * i) = u32x2{w[i], w[i + 1]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < C - 1; ++i)
        if (i < live) to[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i % 2)));
    }
  }
}

// Runs f(gate) with the gate as a constant: one copy of what f unrolls for each.
template <bool GATED, typename F>
__device__ __forceinline__ void with_gate(const Linear8Params& p, F&& f) {
  if constexpr (!GATED) {
    f(std::integral_constant<int, CTI_EBAG_GATE_NONE>{});
  } else {
    switch (p.gate) {
      case CTI_EBAG_GATE_SILU: f(std::integral_constant<int, CTI_EBAG_GATE_SILU>{}); break;
      case CTI_EBAG_GATE_GELU: f(std::integral_constant<int, CTI_EBAG_GATE_GELU>{}); break;
      default: f(std::integral_constant<int, CTI_EBAG_GATE_RELU>{}); break;
    }
  }
}

// C consecutive columns of a row from the sums t (gated: gates) and u (values).
template <typename YT, int GATE, int C>
__device__ __forceinline__ void emit(const Linear8Params& p, int64_t m, int n, int live, float sm, const Columns<C>& a,
                                     const Columns<C>& b, const int* t, const int* u) {
  float v[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    v[i] = a.apply(i, t[i], sm);
    if constexpr (GATE != CTI_EBAG_GATE_NONE) v[i] = as_f32(activate<GATE>(v[i]) * b.apply(i, u[i], sm));
  }
  store_columns<YT, C>(p.y, m * p.N + n, v, live);
}

// A wavefront's sums to y, or to this split's partial sums: lane l holds rows m0 + R a + l % R, a < MI, and of each
// GROUPS times C columns side by side from col_of(g) on; sum(a, g, half, i) is the sum of column i of group g (half 1:
// of the gated form's values). Scales are loaded at once and before the first is used: one at a time, between the
// stores, they took 38 us a 256 x 256 tile, as long as 3,500 of K.
template <typename YT, bool GATED, int R, int MI, int GROUPS, int C, typename ColOf, typename Sum>
__device__ __forceinline__ void epilogue(const Linear8Params& p, int64_t m0, ColOf&& col_of, Sum&& sum, int split) {
  constexpr int H = GATED ? 2 : 1;
  const int row = lane_id() % R;
  if (p.part) {
    const int64_t cols = linear8_part_cols(p.n_end - p.n_begin), width = cols * H;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int n = col_of(g), live = p.n_end - n;
      if (live <= 0) continue;
      int32_t* const part = p.part + split * p.M * width + n - p.n_begin;
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        const int64_t m = m0 + a * R + row;
        if (m >= p.M) continue;
#pragma unroll
        for (int half = 0; half < H; ++half) {
          int32_t* const to = part + m * width + half * cols;
#pragma unroll
          for (int i = 0; i < C; i += 4) {
            // (a row's space is whole vectors: what lies past its columns is never used)
            if (i < live)
              *reinterpret_cast<i32x4*>(to + i) =
                  i32x4{sum(a, g, half, i), sum(a, g, half, i + 1), sum(a, g, half, i + 2), sum(a, g, half, i + 3)};
          }
        }
      }
    }
    return;
  }
  float sm[MI];
#pragma unroll
  for (int a = 0; a < MI; ++a) {
    const int64_t m = m0 + a * R + row;
    sm[a] = p.scale[m < p.M ? m : p.M - 1];
  }
  Columns<C> ca[GROUPS], cb[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int n = col_of(g), live = p.n_end - n;
    if (live <= 0) continue;
    ca[g].load(p, n, live);
    if constexpr (GATED) cb[g].load(p, p.N + n, live);
  }
  with_gate<GATED>(p, [&](auto gate) {
#pragma unroll
    for (int a = 0; a < MI; ++a) {
      const int64_t m = m0 + a * R + row;
      if (m >= p.M) continue;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) {  // a row's groups one after the other: they share cache lines
        const int n = col_of(g), live = p.n_end - n;
        if (live <= 0) continue;
        int t[C], u[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
          t[i] = sum(a, g, 0, i);
          u[i] = sum(a, g, H - 1, i);
        }
        emit<YT, decltype(gate)::value, C>(p, m, n, live, sm[a], ca[g], cb[g], t, u);
      }
    }
  });
}

// ---------------------------------------------------------------------------------------------
// Loads
// ---------------------------------------------------------------------------------------------
// 16 bytes of a row at byte k; what lies past K is zero. Rows start at any address (the vector loads of gfx950
// take any). A row's last bytes, if fewer than 16, are the end of its last 16 moved down: 40 rows of 333 by 1,000
// outputs took 17 us with them loaded one by one (rows of less than 16 bytes are).
__device__ __forceinline__ i32x4 load_chunk(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const i32x4_any*>(row + k);
  i32x4 v = {0, 0, 0, 0};
  if (k >= K) return v;
  if (K < 16) {
#pragma unroll
    for (int b = 0; b < 15; ++b)
      if (b < K) v[b / 4] |= static_cast<int>(static_cast<uint32_t>(static_cast<uint8_t>(row[b])) << (8 * (b % 4)));
    return v;
  }
  const i32x4 e = *reinterpret_cast<const i32x4_any*>(row + K - 16);
  const int by = k + 16 - K;  // bytes to drop, 1 to 15
  const uint32_t w[8] = {static_cast<uint32_t>(e[0]), static_cast<uint32_t>(e[1]), static_cast<uint32_t>(e[2]),
                         static_cast<uint32_t>(e[3]), 0u, 0u, 0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t lo = w[i], hi = w[i + 1];  // words i + by / 4 and the next
#pragma unroll
    for (int j = 1; j < 4; ++j) {
      lo = by / 4 == j ? w[i + j] : lo;
      hi = by / 4 == j ? w[i + j + 1 < 8 ? i + j + 1 : 7] : hi;
    }
    v[i] = static_cast<int>(__builtin_amdgcn_alignbyte(hi, lo, static_cast<uint32_t>(by) & 3u));
  }
  return v;
}

// ---------------------------------------------------------------------------------------------
// Few rows, or few outputs: 16 rows by 16 columns (gated: of gates and of values) a workgroup
// ---------------------------------------------------------------------------------------------
template <typename YT, int W, int U, bool GATED>
__global__ void __launch_bounds__(W * kWave) linear8_rows_kernel(const Linear8Params p) {
  constexpr int NT = GATED ? 2 : 1;
  __shared__ i32x4 s_acc[W][NT][kWave];
  const int t = static_cast<int>(threadIdx.x);
  const int lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int fr = lane & 15, fq = lane >> 4;
  const int tile_m = static_cast<int>(blockIdx.x) / p.tiles_n;
  const int n0 = p.n_begin + (static_cast<int>(blockIdx.x) - tile_m * p.tiles_n) * 16;
  const int64_t m0 = static_cast<int64_t>(tile_m) * 16;
  // columns past the last and rows past M repeat the last: not stored
  const int n = n0 + fr < p.n_end ? n0 + fr : p.n_end - 1;
  const int64_t m = m0 + fr < p.M ? m0 + fr : p.M - 1;
  const int8_t* const xrow = p.x + m * p.K;
  const int8_t* wrow[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) wrow[c] = p.w + (static_cast<int64_t>(c) * p.N + n) * p.K;
  i32x4 acc[NT];
#pragma unroll
  for (int c = 0; c < NT; ++c) acc[c] = i32x4{0, 0, 0, 0};
  // Steps of 128 bytes of K, of which the lane's two chunks are 32 bytes side by side; wavefront w takes steps w,
  // w + W, ..., U of them at a time with all their loads in flight (those past the last whole step load it again
  // and multiply by zero).
  // (K split over workgroups: of this split's steps)
  const int nk_all = p.K / kStep;
  const int ks0 = p.part ? static_cast<int>(blockIdx.y) * p.split_steps : 0;
  const int whole = p.part && ks0 + p.split_steps < nk_all ? ks0 + p.split_steps : nk_all;
  for (int s = ks0 + wave; s < whole; s += W * U) {
    i32x4 fw[U][NT][2], fx[U][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int su = s + u * W;
      const int k = (su < whole ? su : whole - 1) * kStep + fq * 32;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int c = 0; c < NT; ++c) fw[u][c][h] = *reinterpret_cast<const i32x4_any*>(wrow[c] + k + h * 16);
        fx[u][h] = *reinterpret_cast<const i32x4_any*>(xrow + k + h * 16);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // every load before the first product
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const i32x4 x = s + u * W < whole ? fx[u][h] : i32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NT; ++c) acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[u][c][h], x, acc[c], 0, 0, 0);
      }
  }
  if (p.K % kStep != 0 && wave == nk_all % W && (!p.part || blockIdx.y + 1 == gridDim.y)) {  // the rest of K
    const int k = nk_all * kStep + fq * 32;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const i32x4 x = load_chunk(xrow, k + h * 16, p.K);
#pragma unroll
      for (int c = 0; c < NT; ++c)
        acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(load_chunk(wrow[c], k + h * 16, p.K), x, acc[c], 0, 0, 0);
    }
  }
#pragma unroll
  for (int c = 0; c < NT; ++c) s_acc[wave][c][lane] = acc[c];
  __syncthreads();
  if (wave != 0) return;
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int i = 1; i < W; ++i) acc[c] += s_acc[i][c][lane];
  epilogue<YT, GATED, 16, 1, 1, 4>(p, m0, [&](int) { return n0 + fq * 4; },
                                   [&](int, int, int half, int i) { return acc[half][i]; }, static_cast<int>(blockIdx.y));
}

// ---------------------------------------------------------------------------------------------
// Tiles of operands at any address: BM rows by BN weight rows, WM x WN wavefronts
// ---------------------------------------------------------------------------------------------
// Tile i of the launch. Dispatch position i runs on XCD i % 8: each XCD gets a contiguous range of tiles
// (L2 is per XCD), which runs down kGroup row bands before it steps to the next column of tiles. A group of 6, no power
// of two, keeps what runs at a time off the same cache channels: 8192 x 2048 -> 16384 took 277 / 246 / 238 / 293 / 241 us with
// groups of 1 / 2 / 3 / 4 / 6, 16384 x 2048 -> 8192 291 / 255 / 253 / 243 / 236 and 288 with 8.
__device__ __forceinline__ void tile_of(const Linear8Params& p, int* tm, int* tn) {
  constexpr int kGroup = 6;
  const int total = p.tiles_m * p.tiles_n, i = static_cast<int>(blockIdx.x);
  const int xcd = i % kXcds, each = total / kXcds, more = total % kXcds;
  const int tile = xcd * each + (xcd < more ? xcd : more) + i / kXcds;
  const int per = kGroup * p.tiles_n;
  const int g = tile / per, rest = tile - g * per;
  const int rows = p.tiles_m - g * kGroup < kGroup ? p.tiles_m - g * kGroup : kGroup;
  *tm = g * kGroup + rest % rows;
  *tn = rest / rows;
}

template <typename YT, int BM, int BN, int WM, int WN, bool GATED>
__global__ void __launch_bounds__(WM * WN * kWave) linear8_tile_kernel(const Linear8Params p) {
  constexpr int THREADS = WM * WN * kWave;
  constexpr int TM = BM / WM, TN = BN / WN;     // a wavefront's rows and weight rows
  constexpr int MI = TM / 16, NI = TN / 16;
  constexpr int kChunks = kStep / 16;           // 16-byte chunks of a row and step
  constexpr int PX = BM * kChunks / THREADS, PW = BN * kChunks / THREADS;
  constexpr int kRowStep = THREADS / kChunks;
  constexpr int NO = GATED ? NI / 2 : NI;       // fragments of output columns
  constexpr int OUT = GATED ? BN / 2 : BN;      // output columns of the tile
  static_assert(kRowStep % 8 == 0 && BM % kRowStep == 0 && BN % kRowStep == 0, "tile shape");
  // rows of 128 bytes, chunk c of row r in slot c ^ (r & 7) (no bank conflicts)
  __shared__ i32x4 sX[2][BM * kChunks];
  __shared__ i32x4 sW[2][BN * kChunks];
  int tm, tn;
  tile_of(p, &tm, &tn);
  const int64_t m0 = static_cast<int64_t>(tm) * BM;
  const int n0 = p.n_begin + tn * OUT;
  const int t = static_cast<int>(threadIdx.x);
  const int lane = t & (kWave - 1), wave = t / kWave;
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, fq = lane >> 4;
  const int kc = t % kChunks, r0 = t / kChunks;

  // rows past M and weight rows past N repeat the last one: their products are not stored
  const int8_t* xrow[PX];
  const int8_t* wrow[PW];
#pragma unroll
  for (int q = 0; q < PX; ++q) {
    const int64_t m = m0 + r0 + q * kRowStep;
    xrow[q] = p.x + (m < p.M ? m : p.M - 1) * p.K;
  }
#pragma unroll
  for (int q = 0; q < PW; ++q) {
    const int j = r0 + q * kRowStep;  // row of the tile: wavefront column j / TN, fragment j % TN / 16
    int n, half = 0;
    if constexpr (GATED) {
      half = j % TN / (TN / 2);  // a wavefront's first half: gates, second half: their values
      n = n0 + j / TN * (TN / 2) + j % (TN / 2);
    } else {
      n = n0 + j;
    }
    wrow[q] = p.w + (static_cast<int64_t>(half) * p.N + (n < p.n_end ? n : p.n_end - 1)) * p.K;
  }
  const int nk_all = (p.K + kStep - 1) / kStep;
  const int ks0 = p.part ? static_cast<int>(blockIdx.y) * p.split_steps : 0;
  const int nk = p.part ? (nk_all - ks0 < p.split_steps ? nk_all - ks0 : p.split_steps) : nk_all;
  i32x4 rx[PX], rw[PW];
  const auto issue = [&](int s) {
    const int k = (ks0 + s) * kStep + kc * 16;
#pragma unroll
    for (int q = 0; q < PX; ++q) rx[q] = load_chunk(xrow[q], k, p.K);
#pragma unroll
    for (int q = 0; q < PW; ++q) rw[q] = load_chunk(wrow[q], k, p.K);
  };
  const auto put = [&](int buf) {
    const int slot = r0 * kChunks + (kc ^ (r0 & 7));
#pragma unroll
    for (int q = 0; q < PX; ++q) sX[buf][slot + q * kRowStep * kChunks] = rx[q];
#pragma unroll
    for (int q = 0; q < PW; ++q) sW[buf][slot + q * kRowStep * kChunks] = rw[q];
  };
  i32x4 acc[MI][NI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int c = 0; c < NI; ++c) acc[a][c] = i32x4{0, 0, 0, 0};
  issue(0);
  put(0);
  __syncthreads();
  for (int s = 0; s < nk; ++s) {
    if (s + 1 < nk) issue(s + 1);
    const int buf = s & 1;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int slot = (h * 4 + fq) ^ (fr & 7);
      i32x4 fw[NI], fx[MI];
#pragma unroll
      for (int c = 0; c < NI; ++c) fw[c] = sW[buf][(wn * TN + c * 16 + fr) * kChunks + slot];
#pragma unroll
      for (int a = 0; a < MI; ++a) fx[a] = sX[buf][(wm * TM + a * 16 + fr) * kChunks + slot];
#pragma unroll
      for (int a = 0; a < MI; ++a)
#pragma unroll
        for (int c = 0; c < NI; ++c)
          acc[a][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[c], fx[a], acc[a][c], 0, 0, 0);
    }
    if (s + 1 < nk) put(buf ^ 1);
    __syncthreads();
  }
  epilogue<YT, GATED, 16, MI, NO, 4>(p, m0 + wm * TM, [&](int g) { return n0 + wn * NO * 16 + g * 16 + fq * 4; },
                                     [&](int a, int g, int half, int i) { return acc[a][half * NO + g][i]; },
                                     static_cast<int>(blockIdx.y));
}

// ---------------------------------------------------------------------------------------------
// Large tiles (K a multiple of 16, 16-byte aligned operands): loads straight to LDS
// ---------------------------------------------------------------------------------------------
typedef __amdgpu_buffer_rsrc_t Rsrc;
__device__ __forceinline__ Rsrc make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0), static_cast<int>(bytes),
                                           0x00020000);  // raw buffer, 32-bit data format
}
// 16 bytes per lane straight to LDS, lane l's to lds + 16 l (lds the same for every lane).
__device__ __forceinline__ void load_lds(Rsrc r, i32x4* lds, uint32_t voff, uint32_t soff) {
#ifdef __HIP_DEVICE_COMPILE__  // the host pass has no 16-byte form
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, soff, 0, 0);
#endif
}
// Waits until at most N of this wavefront's loads are in flight, and for its LDS reads; then the barrier.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");  // no instruction: keeps the compiler's order
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4 << 14));  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Tiles of BM x BN with WM x WN wavefronts, a ring of four steps: a step's loads are issued three steps ahead. For
// tiles that are few, or short in K once it is split: what counts is bytes in flight, and for rounds that fill the card
// bytes from L2 (4096 x 3584 -> 512: 512 tiles of 64 x 64, two to a CU, load 32 KB for each product of 128 x 64 x 128 on a CU
// and take 15.2 us; 256 of 128 x 64 load 24 and take 12.7; 2048 x 5632 -> 2048 as 256 tiles of 128 x 128 26.7, its matrix
// cores busy half of that, 34 bytes a clock and CU loaded). Fragments read half a step ahead as below gained nothing here.
template <typename YT, int BM, int BN, int WM, int WN, bool GATED>
__global__ void __launch_bounds__(WM * WN * kWave, 1) linear8_ring_kernel(const Linear8Params p) {
  constexpr int WAVES = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN;
  constexpr int MI = TM / 16, NI = TN / 16;
  constexpr int kChunks = kStep / 16;
  constexpr int PX = BM / 8 / WAVES, PW = BN / 8 / WAVES;  // loads per thread and step, 8 rows a wavefront each
  constexpr int OUT = GATED ? BN / 2 : BN;
  constexpr int NO = GATED ? NI / 2 : NI;
  constexpr int G = std::is_same<YT, float>::value || NO < 2 ? 1 : 2;
  static_assert(PX >= 1 && PW >= 1 && NO >= 1 && (!GATED || PW == 1 || NI % 2 == 0), "tile shape");
  __shared__ i32x4 s0[(BM + BN) * kChunks], s1[(BM + BN) * kChunks], s2[(BM + BN) * kChunks], s3[(BM + BN) * kChunks];
  int tm, tn;
  tile_of(p, &tm, &tn);
  const int64_t m0 = static_cast<int64_t>(tm) * BM;
  const int n0 = p.n_begin + tn * OUT;
  const int t = static_cast<int>(threadIdx.x);
  const int lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, fq = lane >> 4;
  const int nk_all = (p.K + kStep - 1) / kStep;
  const int ks0 = p.part ? static_cast<int>(blockIdx.y) * p.split_steps : 0;
  const int nk = p.part ? (nk_all - ks0 < p.split_steps ? nk_all - ks0 : p.split_steps) : nk_all;

  const int64_t mrows = p.M - m0 < BM ? p.M - m0 : BM;
  const int64_t nrows = p.n_end - n0 < OUT ? p.n_end - n0 : OUT;
  const Rsrc xr = make_rsrc(p.x + m0 * p.K, static_cast<uint32_t>(mrows * p.K));
  const Rsrc wr = make_rsrc(p.w + static_cast<int64_t>(n0) * p.K, static_cast<uint32_t>(nrows * p.K));
  const Rsrc ur = make_rsrc(p.w + (static_cast<int64_t>(GATED ? p.N : 0) + n0) * p.K, static_cast<uint32_t>(nrows * p.K));
  uint32_t xoff[PX], woff[PW];
  const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int q = 0; q < PX; ++q) xoff[q] = static_cast<uint32_t>((wave * PX + q) * 8 + lane / 8) * p.K + chunk * 16;
#pragma unroll
  for (int q = 0; q < PW; ++q) {
    const int j = (wave * PW + q) * 8 + lane / 8, f = j % TN / 16 % NO, i = j % 16;
    const int c = j / TN * (NO * 16) + f / G * (16 * G) + 4 * G * (i / 4) + 4 * (f % G) + i % 4;
    woff[q] = static_cast<uint32_t>(c) * p.K + chunk * 16;
  }
  const auto issue = [&](int s, i32x4* to) {
    const int k = (ks0 + (s < nk ? s : nk - 1)) * kStep;  // later steps are never used
#pragma unroll
    for (int q = 0; q < PX; ++q) load_lds(xr, to + (wave * PX + q) * kWave, xoff[q], k);
#pragma unroll
    for (int q = 0; q < PW; ++q) {
      const int f = (wave * PW + q) / 2 % NI;
      load_lds(GATED && f >= NO ? ur : wr, to + BM * kChunks + (wave * PW + q) * kWave, woff[q], k);
    }
  };
  i32x4 acc[MI][NI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int c = 0; c < NI; ++c) acc[a][c] = i32x4{0, 0, 0, 0};
  constexpr int L = PX + PW;
  issue(0, s0);
  issue(1, s1);
  issue(2, s2);
  const auto step = [&](int s, const i32x4* mine, i32x4* free, auto endc) {
    constexpr bool end = decltype(endc)::value;
    wait_barrier<2 * L>();
    issue(s + 3, free);  // over step s - 1, which every wavefront has read
    const int left = p.K - (ks0 + s) * kStep;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int slot = fr * kChunks + ((h * 4 + fq) ^ (fr & 7));
      i32x4 fw[NI], fx[MI];
#pragma unroll
      for (int c = 0; c < NI; ++c) fw[c] = mine[BM * kChunks + (wn * TN + c * 16) * kChunks + slot];
#pragma unroll
      for (int a = 0; a < MI; ++a) fx[a] = mine[(wm * TM + a * 16) * kChunks + slot];
      if (end && left < kStep) {  // the rest of K
#pragma unroll
        for (int a = 0; a < MI; ++a)
          if (h * 64 + fq * 16 >= left) fx[a] = i32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int a = 0; a < MI; ++a)
#pragma unroll
        for (int c = 0; c < NI; ++c)
          acc[a][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[c], fx[a], acc[a][c], 0, 0, 0);
    }
  };
  constexpr std::integral_constant<bool, false> inside{};
  constexpr std::integral_constant<bool, true> end{};
  int s = 0;
  for (; s + 4 < nk; s += 4) {
    step(s, s0, s3, inside);
    step(s + 1, s1, s0, inside);
    step(s + 2, s2, s1, inside);
    step(s + 3, s3, s2, inside);
  }
  // one to four steps, the last of which may be the rest of K
  step(s, s0, s3, end);
  if (s + 1 < nk) {
    step(s + 1, s1, s0, end);
    if (s + 2 < nk) {
      step(s + 2, s2, s1, end);
      if (s + 3 < nk) step(s + 3, s3, s2, end);
    }
  }
  epilogue<YT, GATED, 16, MI, NO / G, 4 * G>(
      p, m0 + wm * TM, [&](int g) { return n0 + wn * (NO * 16) + g * (16 * G) + fq * (4 * G); },
      [&](int a, int g, int half, int i) { return acc[a][half * NO + g * G + i / 4][i % 4]; }, static_cast<int>(blockIdx.y));
}

// Asks the scheduler for P products with R LDS reads and L loads spread evenly between them.
template <int P, int R, int L, int I = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (I < P) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // product
    // reads come in the first three quarters: the next products need them
    constexpr int r = (I + 1) * R * 4 / (P * 3) > R ? R : (I + 1) * R * 4 / (P * 3);
    constexpr int r0 = I * R * 4 / (P * 3) > R ? R : I * R * 4 / (P * 3);
    if constexpr (r > r0) __builtin_amdgcn_sched_group_barrier(0x100, r - r0, 0);
    constexpr int l = (I + 1) * L / P, l0 = I * L / P;
    if constexpr (l > l0) __builtin_amdgcn_sched_group_barrier(0x20, l - l0, 0);
    interleave<P, R, L, I + 1>();
  }
}

template <typename YT, int BM, int BN, int WM, int WN, bool GATED, bool TAIL>
__global__ void __launch_bounds__(WM * WN * kWave, 1) linear8_big_kernel(const Linear8Params p) {
  constexpr int WAVES = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN;
  constexpr int MI = TM / 16, NI = TN / 16;
  constexpr int kChunks = kStep / 16;
  constexpr int PX = BM / 8 / WAVES, PW = BN / 8 / WAVES;  // loads per thread and step, 8 rows a wavefront each
  constexpr int OUT = GATED ? BN / 2 : BN;
  constexpr int NO = GATED ? NI / 2 : NI;    // fragments of output columns
  // G fragments of columns side by side, so that a lane holds 16 bytes of a row and four lanes store 64 in a row (32
  // bytes a lane, stored in two halves with gaps, took the same time)
  constexpr int G = std::is_same<YT, float>::value || NO < 2 ? 1 : 2;
  // rows of 128 bytes, chunk c of row r in slot c ^ (r & 7) (no bank conflicts)
  __shared__ i32x4 s0[(BM + BN) * kChunks], s1[(BM + BN) * kChunks];
  int tm, tn;
  tile_of(p, &tm, &tn);
  const int64_t m0 = static_cast<int64_t>(tm) * BM;
  const int n0 = p.n_begin + tn * OUT;
  const int t = static_cast<int>(threadIdx.x);
  const int lane = t & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const int wm = wave / WN, wn = wave % WN;
  const int fr = lane & 15, fq = lane >> 4;

  const int nk_all = (p.K + kStep - 1) / kStep;
  const int ks0 = p.part ? static_cast<int>(blockIdx.y) * p.split_steps : 0;
  const int nk = p.part ? (nk_all - ks0 < p.split_steps ? nk_all - ks0 : p.split_steps) : nk_all;

  // rows past M, weight rows past N and chunks past the last row's end lie past the buffers: nothing is read (a
  // chunk past the end of another row is the next row's; either is masked or multiplies what is not stored)
  const int64_t mrows = p.M - m0 < BM ? p.M - m0 : BM;
  const int64_t nrows = p.n_end - n0 < OUT ? p.n_end - n0 : OUT;
  const Rsrc xr = make_rsrc(p.x + m0 * p.K, static_cast<uint32_t>(mrows * p.K));
  const Rsrc wr = make_rsrc(p.w + static_cast<int64_t>(n0) * p.K, static_cast<uint32_t>(nrows * p.K));
  const Rsrc ur = make_rsrc(p.w + (static_cast<int64_t>(GATED ? p.N : 0) + n0) * p.K, static_cast<uint32_t>(nrows * p.K));
  // load q of wavefront w fills LDS rows 8 (w PX + q) .. + 8, lane l chunk l % 8 of row l / 8 there
  uint32_t xoff[PX], woff[PW];
  const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
  for (int q = 0; q < PX; ++q) xoff[q] = static_cast<uint32_t>((wave * PX + q) * 8 + lane / 8) * p.K + chunk * 16;
#pragma unroll
  for (int q = 0; q < PW; ++q) {
    // LDS row 16 f + i of a wavefront column holds column 4 G (i / 4) + 4 (f % G) + i % 4 of each 16 G (gated:
    // fragments f < NO gates, the others their values), so that a lane receives 4 G columns side by side
    const int j = (wave * PW + q) * 8 + lane / 8, f = j % TN / 16 % NO, i = j % 16;
    const int c = j / TN * (NO * 16) + f / G * (16 * G) + 4 * G * (i / 4) + 4 * (f % G) + i % 4;
    woff[q] = static_cast<uint32_t>(c) * p.K + chunk * 16;
  }
  const auto issue = [&](int s, i32x4* to) {
    const int k = (ks0 + (s < nk ? s : nk - 1)) * kStep;  // later steps are never used
#pragma unroll
    for (int q = 0; q < PX; ++q) load_lds(xr, to + (wave * PX + q) * kWave, xoff[q], k);
#pragma unroll
    for (int q = 0; q < PW; ++q) {
      const int f = (wave * PW + q) / 2 % NI;
      load_lds(GATED && f >= NO ? ur : wr, to + BM * kChunks + (wave * PW + q) * kWave, woff[q], k);
    }
  };
  i32x4 fx[2][MI], fw[2][NI];
  const auto read = [&](const i32x4* from, auto half) {
    constexpr int h = decltype(half)::value;
    const int slot = fr * kChunks + ((h * 4 + fq) ^ (fr & 7));
#pragma unroll
    for (int c = 0; c < NI; ++c) fw[h][c] = from[BM * kChunks + (wn * TN + c * 16) * kChunks + slot];
#pragma unroll
    for (int a = 0; a < MI; ++a) fx[h][a] = from[(wm * TM + a * 16) * kChunks + slot];
  };
  i32x4 acc[MI][NI];
#pragma unroll
  for (int a = 0; a < MI; ++a)
#pragma unroll
    for (int c = 0; c < NI; ++c) acc[a][c] = i32x4{0, 0, 0, 0};
  const auto multiply = [&](auto half) {
    constexpr int h = decltype(half)::value;
#pragma unroll
    for (int a = 0; a < MI; ++a)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int c = a & 1 ? NI - 1 - i : i;  // there and back: an operand changes at a time (0.5% at the power limit)
        acc[a][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h][c], fx[h][a], acc[a][c], 0, 0, 0);
      }
  };
  constexpr std::integral_constant<int, 0> first{};
  constexpr std::integral_constant<int, 1> second{};
  constexpr int L = PX + PW;
  issue(0, s0);
  issue(1, s1);
  wait_barrier<L>();
  read(s0, first);
  // Step s: the first half's fragments are in registers (or on their way), the second half's are read while the
  // first is multiplied. Once every wavefront has them and step s + 1 has arrived, the second half is multiplied
  // while step s + 2 is loaded over step s and the next step's first half is read.
  const auto step = [&](int s, i32x4* mine, const i32x4* next, auto endc) {
    constexpr bool end = decltype(endc)::value;
    const int left = p.K - (ks0 + s) * kStep;  // bytes of K from this step on
    const auto mask = [&](int h) {
      if (end && s == nk - 1 && left < kStep) {
#pragma unroll
        for (int a = 0; a < MI; ++a)
          if (h * 64 + fq * 16 >= left) fx[h][a] = i32x4{0, 0, 0, 0};
      }
    };
    mask(0);
    read(mine, second);
    multiply(first);
    interleave<MI * NI, MI + NI, 0>();
    wait_barrier<0>();
    mask(1);
    issue(s + 2, mine);
    read(next, first);
    multiply(second);
    interleave<MI * NI, MI + NI, L>();
    __builtin_amdgcn_sched_barrier(0);
  };
  // one way out of the loop: the compiler then knows at its head which loads to LDS are in flight, and adds no wait
  constexpr std::integral_constant<bool, false> inside{};
  constexpr std::integral_constant<bool, TAIL> end{};
  int s = 0;
  for (; s + 2 <= (TAIL ? nk - 1 : nk); s += 2) {
    step(s, s0, s1, inside);
    step(s + 1, s1, s0, inside);
  }
  if (s < nk) {
    step(s, s0, s1, end);
    if (TAIL && s + 1 < nk) step(s + 1, s1, s0, end);
  }
  epilogue<YT, GATED, 16, MI, NO / G, 4 * G>(
      p, m0 + wm * TM, [&](int g) { return n0 + wn * (NO * 16) + g * (16 * G) + fq * (4 * G); },
      [&](int a, int g, int half, int i) { return acc[a][half * NO + g * G + i / 4][i % 4]; }, static_cast<int>(blockIdx.y));
}

// Split K: the splits' sums added, scales, bias, gate and rounding as in the tiles' epilogue; 4 columns a thread.
constexpr int kReduceThreads = 256;
template <typename YT, bool GATED>
__global__ void __launch_bounds__(kReduceThreads) linear8_reduce_kernel(const Linear8Params p, int splits) {
  const int64_t cols = linear8_part_cols(p.n_end - p.n_begin), quads = cols / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kReduceThreads + threadIdx.x;
  const int64_t m = i / quads;
  if (m >= p.M) return;
  const int at = static_cast<int>(i - m * quads) * 4, n = p.n_begin + at, live = p.n_end - n;
  const int64_t width = cols * (GATED ? 2 : 1), each = p.M * width;
  int t[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int half = 0; half < (GATED ? 2 : 1); ++half) {
    const int32_t* const from = p.part + m * width + half * cols + at;
    constexpr int kAhead = 8;  // loads in flight
    for (int s = 0; s < splits; s += kAhead) {
      i32x4 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        v[j] = *reinterpret_cast<const i32x4*>(from + (s + j < splits ? s + j : splits - 1) * each);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) t[half][r] += s + j < splits ? v[j][r] : 0;
    }
  }
  Columns<4> ca, cb;
  ca.load(p, n, live);
  if constexpr (GATED) cb.load(p, p.N + n, live);
  with_gate<GATED>(p, [&](auto gate) {
    emit<YT, decltype(gate)::value, 4>(p, m, n, live, p.scale[m], ca, cb, t[0], t[1]);
  });
}

// Rows of K bytes at any address to rows of a whole number of steps, the rest zero: x, then the weight. A copy of both
// (read once, written once) costs less than tiles of operands that cannot be loaded straight to LDS.
constexpr int kPadThreads = 256;
__global__ void __launch_bounds__(kPadThreads) linear8_pad_kernel(const int8_t* x, const int8_t* w, int64_t x_rows,
                                                                  int64_t rows, int32_t K, int32_t chunks, i32x4* out) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kPadThreads + threadIdx.x;
  const int64_t row = i / chunks;
  if (row >= rows) return;
  const int8_t* const from = row < x_rows ? x + row * K : w + (row - x_rows) * K;
  out[i] = load_chunk(from, static_cast<int>(i - row * chunks) * 16, K);
}

// ---------------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------------
template <typename YT, bool GATED>
hipError_t launch_part(Linear8Params p, const Linear8Part& part, int32_t* work, hipStream_t s) {
  p.n_begin = part.n_begin;
  p.n_end = part.n_end;
  p.split_steps = part.steps;
  p.part = part.splits > 1 ? work : nullptr;
  const Linear8Tile tile = linear8_tile(part.form);
  const int out = GATED && part.form != kLinear8Rows ? tile.cols / 2 : tile.cols;
  p.tiles_m = static_cast<int32_t>(linear_ceil(p.M, tile.rows));
  p.tiles_n = static_cast<int32_t>(linear_ceil(p.n_end - p.n_begin, out));
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.tiles_m) * p.tiles_n), static_cast<unsigned>(part.splits));
  const auto go = [&](auto kernel, int waves) { hipLaunchKernelGGL(kernel, grid, dim3(waves * kWave), 0, s, p); };
  const bool whole = p.K % kStep == 0;
  switch (part.form) {
    case kLinear8Rows:
      // the steps of a split in one batch of loads where they are few
      switch (linear8_rows_waves(part.steps)) {
        case 4:
          if (part.steps <= 4) go(linear8_rows_kernel<YT, 4, 1, GATED>, 4);
          else if (part.steps <= 8) go(linear8_rows_kernel<YT, 4, 2, GATED>, 4);
          else go(linear8_rows_kernel<YT, 4, 4, GATED>, 4);
          break;
        case 8: go(linear8_rows_kernel<YT, 8, 4, GATED>, 8); break;
        default: go(linear8_rows_kernel<YT, 16, 4, GATED>, 16);
      }
      break;
    case kLinear8Any: go(linear8_tile_kernel<YT, 128, 128, 2, 2, GATED>, 4); break;
    case kLinear8Ring: go(linear8_ring_kernel<YT, 64, 64, 2, 2, GATED>, 4); break;
    case kLinear8Tile128:
      if (whole) go(linear8_big_kernel<YT, 128, 128, 2, 4, GATED, false>, 8);
      else go(linear8_big_kernel<YT, 128, 128, 2, 4, GATED, true>, 8);
      break;
    case kLinear8Tile256:
      if (whole) go(linear8_big_kernel<YT, 256, 256, 2, 4, GATED, false>, 8);
      else go(linear8_big_kernel<YT, 256, 256, 2, 4, GATED, true>, 8);
      break;
    case kLinear8RingTall: go(linear8_ring_kernel<YT, 128, 64, 4, 2, GATED>, 8); break;
    case kLinear8Ring128: go(linear8_ring_kernel<YT, 128, 128, 4, 2, GATED>, 8); break;
    case kLinear8Forms: return hipErrorInvalidValue;
  }
  if (p.part) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t threads = p.M * (linear8_part_cols(p.n_end - p.n_begin) / 4);
    hipLaunchKernelGGL((linear8_reduce_kernel<YT, GATED>), dim3(static_cast<unsigned>((threads + kReduceThreads - 1) / kReduceThreads)),
                       dim3(kReduceThreads), 0, s, p, part.splits);
  }
  return hipGetLastError();
}

template <typename YT, bool GATED>
hipError_t launch(Linear8Params p, const Linear8Plan& plan, char* work, hipStream_t s) {
  if (plan.padded) {
    const int64_t wrows = static_cast<int64_t>(p.N) * (GATED ? 2 : 1), rows = p.M + wrows;
    const int32_t to = static_cast<int32_t>(linear_ceil(p.K, kStep) * kStep), chunks = to / 16;
    hipLaunchKernelGGL(linear8_pad_kernel, dim3(static_cast<unsigned>(linear_ceil(rows * chunks, kPadThreads))),
                       dim3(kPadThreads), 0, s, p.x, p.w, p.M, rows, p.K, chunks, reinterpret_cast<i32x4*>(work));
    p.x = reinterpret_cast<const int8_t*>(work);
    p.w = p.x + p.M * to;
    p.K = to;
    work += rows * to;
  }
  // (parts run one after the other: they may share the space for partial sums)
  for (int i = 0; i < plan.parts; ++i) {
    const hipError_t e = launch_part<YT, GATED>(p, plan.part[i], reinterpret_cast<int32_t*>(work), s);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <bool GATED>
hipError_t launch_typed(const Linear8Params& p, const Linear8Plan& plan, char* work, hipStream_t s) {
  switch (p.y_dtype) {
    case CTI_EBAG_F32: return launch<float, GATED>(p, plan, work, s);
    case CTI_EBAG_BF16: return launch<bf16_t, GATED>(p, plan, work, s);
    default: return launch<f16_t, GATED>(p, plan, work, s);
  }
}

bool float_dtype(int32_t dt) { return dt == CTI_EBAG_F32 || dt == CTI_EBAG_BF16 || dt == CTI_EBAG_F16; }

}  // namespace
}  // namespace cti

using namespace cti;

static int64_t workspace_bytes(int64_t rows, int32_t cols, int32_t out_features, int32_t gate, bool aligned) {
  const bool gated = gate != CTI_EBAG_GATE_NONE;
  if (rows < 1 || rows > INT32_MAX || cols < 1 || cols > kLinear8MaxK || out_features < 1 ||
      out_features > linear8_max_out(gated) || gate < CTI_EBAG_GATE_NONE || gate > CTI_EBAG_GATE_RELU)
    return 0;
  return linear8_workspace_bytes(rows, out_features, cols, gated, aligned);
}

extern "C" int64_t cti_ebag_linear_int8_workspace_bytes(int64_t rows, int32_t cols, int32_t out_features, int32_t gate) {
  return workspace_bytes(rows, cols, out_features, gate, true);
}

extern "C" int64_t cti_ebag_linear_int8_workspace_bytes_unaligned(int64_t rows, int32_t cols, int32_t out_features,
                                                                  int32_t gate) {
  return workspace_bytes(rows, cols, out_features, gate, false);
}

extern "C" int cti_ebag_linear_int8(const int8_t* q, const float* scale, int64_t rows, int32_t cols, const int8_t* weight,
                                    const float* weight_scale, int32_t out_features, const void* bias,
                                    int32_t bias_dtype, int32_t gate, void* y, int32_t y_dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  clear_error();
  if (rows < 0) return set_error(CTI_EBAG_EINVAL, "rows must be >= 0 (got %lld)", (long long)rows);
  if (cols < 1) return set_error(CTI_EBAG_EINVAL, "cols must be >= 1 (got %d)", cols);
  if (out_features < 1) return set_error(CTI_EBAG_EINVAL, "out_features must be >= 1 (got %d)", out_features);
  if (gate < CTI_EBAG_GATE_NONE || gate > CTI_EBAG_GATE_RELU) return set_error(CTI_EBAG_EINVAL, "unknown gate %d", gate);
  if (!float_dtype(y_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown output dtype code %d", y_dtype);
  if (bias && !float_dtype(bias_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown bias dtype code %d", bias_dtype);
  if (workspace_bytes < 0) return set_error(CTI_EBAG_EINVAL, "workspace_bytes must be >= 0");
  if (cols > kLinear8MaxK)
    return set_error(CTI_EBAG_EUNSUPPORTED, "cols %d > %d (the int32 sums could overflow)", cols, kLinear8MaxK);
  if (out_features > kLinear8MaxN)
    return set_error(CTI_EBAG_EUNSUPPORTED, "out_features %d > %d", out_features, kLinear8MaxN);
  if (rows == 0) return CTI_EBAG_OK;
  if (rows > INT32_MAX) return set_error(CTI_EBAG_EUNSUPPORTED, "more than 2^31 - 1 rows (%lld)", (long long)rows);
  if (!q || !scale || !weight || !weight_scale || !y)
    return set_error(CTI_EBAG_EINVAL, "NULL device pointer among q/scale/weight/weight_scale/y");
  if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
    return set_error(CTI_EBAG_EINVAL, "workspace is not 16-byte aligned");
  const bool gated = gate != CTI_EBAG_GATE_NONE;
  if (out_features > linear8_max_out(gated))
    return set_error(CTI_EBAG_EUNSUPPORTED, "too many output tiles (%lld x %d)", (long long)rows, out_features);
  const bool aligned = cols % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(weight) % 16 == 0;
  const int64_t ws_bytes = workspace ? workspace_bytes : 0;
  const auto plan_of = [&](int64_t m) { return linear8_plan(m, out_features, cols, gated, aligned, ws_bytes); };
  // launches of `most` rows, and of those left
  const int64_t most = linear8_launch_rows(out_features, gated), rest = rows % most, whole = rows - rest;
  const Linear8Plan plan = whole ? plan_of(most) : Linear8Plan{}, last = rest ? plan_of(rest) : Linear8Plan{};
  Linear8Params p = {};
  p.w = weight;
  p.wscale = weight_scale;
  p.bias = bias;
  p.N = out_features;
  p.K = cols;
  p.bias_dtype = bias_dtype;
  p.y_dtype = y_dtype;
  p.gate = gate;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const work = static_cast<char*>(workspace);
  for (int64_t m = 0; m < rows; m += most) {
    const Linear8Plan& of = m < whole ? plan : last;
    p.M = m < whole ? most : rest;
    p.x = q + m * cols;
    p.scale = scale + m;
    p.y = static_cast<char*>(y) + m * out_features * dtype_bytes(y_dtype);
    const hipError_t e = gated ? launch_typed<true>(p, of, work, s) : launch_typed<false>(p, of, work, s);
    if (e != hipSuccess) return set_error(CTI_EBAG_EHIP, "linear launch failed: %s", hipGetErrorString(e));
  }
  return CTI_EBAG_OK;
}
