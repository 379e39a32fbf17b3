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
//   rows   few rows: bound by reading the weight once. A wavefront owns 16 columns (gated: 16 gates and
//          their 16 values) and a share of K, weights and rows straight to registers; the wavefronts of a
//          workgroup split K and add their sums through LDS.
//   tiles  both operands through LDS. When the tiles would leave CUs idle, K is split over workgroups,
//          each writing int32 partial sums to the caller's workspace, added by a second kernel.
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
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

constexpr int kStep = kLinear8Step;  // bytes of K per step
constexpr int kXcds = 8;

struct Linear8Params {
  const int8_t* x;      // [M, K]
  const float* scale;   // [M]
  const int8_t* w;      // [N or 2 N, K]
  const float* wscale;  // [N or 2 N]
  const void* bias;     // [N or 2 N] or NULL
  char* y;              // [M, N]
  int32_t* part;        // split K: int32 partial sums [splits, M, N or 2 N]; NULL: no split
  int64_t M;
  int32_t N;            // columns of y
  int32_t K;
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
    if constexpr (GATE != CTI_EBAG_GATE_NONE) v[i] = activate<GATE>(v[i]) * b.apply(i, u[i], sm);
  }
  store_columns<YT, C>(p.y, m * p.N + n, v, live);
}

// A wavefront's sums to y, or to this split's partial sums: lane l holds rows m0 + 16 a + l % 16 and of them C
// columns side by side from n on (`live` of which exist) in acc[a][f * C / 4 ..], gated: the values' behind the gates'.
// Scales are loaded at once and before the first is used: one at a time, between the stores, they took longer than
// 64 steps of products.
template <typename YT, bool GATED, int MI, int NO, int G, typename ColOf>
__device__ __forceinline__ void epilogue(const Linear8Params& p, int64_t m0, ColOf&& col_of,
                                         const i32x4 (&acc)[MI][GATED ? 2 * NO : NO], int split) {
  constexpr int C = 4 * G, GROUPS = NO / G;
  const int fr = lane_id() & 15;
  const auto sums = [&](int a, int f, int* t) {
#pragma unroll
    for (int i = 0; i < C; ++i) t[i] = acc[a][f + i / 4][i % 4];
  };
  if (p.part) {
    const int64_t width = static_cast<int64_t>(p.N) * (GATED ? 2 : 1);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      const int n = col_of(g), live = p.N - n;
      if (live <= 0) continue;
      int32_t* const part = p.part + split * p.M * width + n;
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        const int64_t m = m0 + a * 16 + fr;
        if (m >= p.M) continue;
#pragma unroll
        for (int half = 0; half < (GATED ? 2 : 1); ++half) {
          int32_t* const to = part + m * width + static_cast<int64_t>(half) * p.N;
#pragma unroll
          for (int i = 0; i < C; i += 4) {
            const i32x4 v = acc[a][half * NO + g * G + i / 4];
            if (live >= C) {
              *reinterpret_cast<i32x4_any*>(to + i) = v;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (i + r < live) to[i + r] = v[r];
            }
          }
        }
      }
    }
    return;
  }
  float sm[MI];
#pragma unroll
  for (int a = 0; a < MI; ++a) {
    const int64_t m = m0 + a * 16 + fr;
    sm[a] = p.scale[m < p.M ? m : p.M - 1];
  }
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int n = col_of(g), live = p.N - n;
    if (live <= 0) continue;
    Columns<C> ca, cb;
    ca.load(p, n, live);
    if constexpr (GATED) cb.load(p, p.N + n, live);
    with_gate<GATED>(p, [&](auto gate) {
#pragma unroll
      for (int a = 0; a < MI; ++a) {
        const int64_t m = m0 + a * 16 + fr;
        int t[C], u[C];
        sums(a, g * G, t);
        sums(a, (GATED ? NO : 0) + g * G, u);
        if (m < p.M) emit<YT, decltype(gate)::value, C>(p, m, n, live, sm[a], ca, cb, t, u);
      }
    });
  }
}

// ---------------------------------------------------------------------------------------------
// Loads
// ---------------------------------------------------------------------------------------------
// 16 bytes of a row at byte k; what lies past K is zero. Rows start at any address (the vector loads of
// gfx950 take any); only the row's last bytes, if fewer than 16, are loaded one by one.
__device__ __forceinline__ i32x4 load_chunk(const int8_t* row, int k, int K) {
  if (k + 16 <= K) return *reinterpret_cast<const i32x4_any*>(row + k);
  i32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int b = 0; b < 15; ++b)
    if (k + b < K) v[b / 4] |= static_cast<int>(static_cast<uint32_t>(static_cast<uint8_t>(row[k + b])) << (8 * (b % 4)));
  return v;
}

// ---------------------------------------------------------------------------------------------
// Few rows (M <= 16 MT)
// ---------------------------------------------------------------------------------------------
template <typename YT, int W, int MT, bool GATED>
__global__ void __launch_bounds__(W * kWave) linear8_rows_kernel(const Linear8Params p) {
  constexpr int NT = GATED ? 2 : 1;
  __shared__ i32x4 s_acc[W > 1 ? W : 1][MT * NT][kWave];
  const int t = static_cast<int>(threadIdx.x);
  const int lane = t & (kWave - 1), wave = t / kWave;
  const int fr = lane & 15, fq = lane >> 4;
  const int n0 = static_cast<int>(blockIdx.x) * 16;
  const int nr = n0 + fr < p.N ? n0 + fr : p.N - 1;  // columns past N repeat the last: not stored
  const int8_t* wrow[NT];
  const int8_t* xrow[MT];
#pragma unroll
  for (int c = 0; c < NT; ++c) wrow[c] = p.w + (static_cast<int64_t>(c) * p.N + nr) * p.K;
#pragma unroll
  for (int a = 0; a < MT; ++a) {
    const int64_t m = a * 16 + fr;
    xrow[a] = p.x + (m < p.M ? m : p.M - 1) * p.K;
  }
  i32x4 acc[NT][MT];
#pragma unroll
  for (int c = 0; c < NT; ++c)
#pragma unroll
    for (int a = 0; a < MT; ++a) acc[c][a] = i32x4{0, 0, 0, 0};
  // a step of 128 bytes: the lane's two chunks are 32 bytes side by side
  const int nk = (p.K + kStep - 1) / kStep;
  for (int s = wave; s < nk; s += W) {
    const int k = s * kStep + fq * 32;
    i32x4 fw[NT][2], fx[MT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int c = 0; c < NT; ++c) fw[c][h] = load_chunk(wrow[c], k + h * 16, p.K);
#pragma unroll
      for (int a = 0; a < MT; ++a) fx[a][h] = load_chunk(xrow[a], k + h * 16, p.K);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int a = 0; a < MT; ++a)
          acc[c][a] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[c][h], fx[a][h], acc[c][a], 0, 0, 0);
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int a = 0; a < MT; ++a) s_acc[wave][a * NT + c][lane] = acc[c][a];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 1; i < W; ++i) acc[c][a] += s_acc[i][a * NT + c][lane];
  }
  // lane l holds columns 4 (l / 16) .. + 4 of row l % 16
  i32x4 sums[MT][NT];
#pragma unroll
  for (int a = 0; a < MT; ++a)
#pragma unroll
    for (int c = 0; c < NT; ++c) sums[a][c] = acc[c][a];
  epilogue<YT, GATED, MT, 1, 1>(p, 0, [&](int) { return n0 + fq * 4; }, sums, 0);
}

// ---------------------------------------------------------------------------------------------
// Tiles: BM rows by BN weight rows, WM x WN wavefronts
// ---------------------------------------------------------------------------------------------
// Tile i of the launch. Dispatch position i runs on XCD i % 8: each XCD gets a contiguous range of tiles
// (L2 is per XCD), which runs down kGroup row bands before it steps to the next column of tiles.
__device__ __forceinline__ void tile_of(const Linear8Params& p, int* tm, int* tn) {
  constexpr int kGroup = 8;
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
  const int n0 = tn * OUT;
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
    wrow[q] = p.w + (static_cast<int64_t>(half) * p.N + (n < p.N ? n : p.N - 1)) * p.K;
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
  epilogue<YT, GATED, MI, NO, 1>(p, m0 + wm * TM, [&](int g) { return n0 + wn * NO * 16 + g * 16 + fq * 4; }, acc,
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

template <typename YT, int WM, int WN, bool GATED, bool TAIL>
__global__ void __launch_bounds__(WM * WN * kWave, 1) linear8_big_kernel(const Linear8Params p) {
  constexpr int BM = 256, BN = 256, WAVES = WM * WN;
  constexpr int TM = BM / WM, TN = BN / WN;
  constexpr int MI = TM / 16, NI = TN / 16;
  constexpr int kChunks = kStep / 16;
  constexpr int PX = BM / 8 / WAVES, PW = BN / 8 / WAVES;  // loads per thread and step, 8 rows a wavefront each
  constexpr int OUT = GATED ? BN / 2 : BN;
  constexpr int NO = GATED ? NI / 2 : NI;    // fragments of output columns
  constexpr int G = NO < 4 ? NO : 4;         // of them side by side: a lane holds 4 G columns of a row
  // rows of 128 bytes, chunk c of row r in slot c ^ (r & 7) (no bank conflicts)
  __shared__ i32x4 s0[(BM + BN) * kChunks], s1[(BM + BN) * kChunks];
  int tm, tn;
  tile_of(p, &tm, &tn);
  const int64_t m0 = static_cast<int64_t>(tm) * BM;
  const int n0 = tn * OUT;
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
  const int64_t nrows = p.N - n0 < OUT ? p.N - n0 : OUT;
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
    // LDS row 16 f + i of a wavefront column holds column 16 (i / 4) + 4 (f % 4) + i % 4 of 64 (gated: fragments
    // f < NO gates, the others their values), so that a lane receives 4 G columns side by side
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
      for (int c = 0; c < NI; ++c)
        acc[a][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[h][c], fx[h][a], acc[a][c], 0, 0, 0);
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
#pragma unroll
    for (int i = 0; i < (MI + NI) / 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 4, 0);    // products
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS reads
    }
    wait_barrier<0>();
    mask(1);
    issue(s + 2, mine);
    read(next, first);
    multiply(second);
#pragma unroll
    for (int i = 0; i < L / 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 3, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);   // load
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x8, 2, 0);
      __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
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
  epilogue<YT, GATED, MI, NO, G>(p, m0 + wm * TM, [&](int g) { return n0 + wn * (NO * 16) + g * (16 * G) + fq * (4 * G); },
                                 acc, static_cast<int>(blockIdx.y));
}

// Split K: the splits' sums added, scales, bias, gate and rounding as in the tiles' epilogue; 4 columns a thread.
constexpr int kReduceThreads = 256;
template <typename YT, bool GATED>
__global__ void __launch_bounds__(kReduceThreads) linear8_reduce_kernel(const Linear8Params p, int splits) {
  const int quads = (p.N + 3) / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kReduceThreads + threadIdx.x;
  const int64_t m = i / quads;
  if (m >= p.M) return;
  const int n = static_cast<int>(i - m * quads) * 4, live = p.N - n;
  const int64_t width = static_cast<int64_t>(p.N) * (GATED ? 2 : 1), each = p.M * width;
  int t[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
  for (int half = 0; half < (GATED ? 2 : 1); ++half) {
    const int32_t* const from = p.part + m * width + static_cast<int64_t>(half) * p.N + n;
    if (live >= 4) {
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const i32x4 v = *reinterpret_cast<const i32x4_any*>(from + s * each);
#pragma unroll
        for (int r = 0; r < 4; ++r) t[half][r] += v[r];
      }
    } else {
      for (int s = 0; s < splits; ++s)
#pragma unroll
        for (int r = 0; r < 3; ++r)
          if (r < live) t[half][r] += from[s * each + r];
    }
  }
  Columns<4> ca, cb;
  ca.load(p, n, live);
  if constexpr (GATED) cb.load(p, p.N + n, live);
  with_gate<GATED>(p, [&](auto gate) {
    emit<YT, decltype(gate)::value, 4>(p, m, n, live, p.scale[m], ca, cb, t[0], t[1]);
  });
}

// ---------------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------------
template <typename YT, bool GATED>
hipError_t launch(Linear8Params p, const Linear8Plan& plan, hipStream_t s) {
  if (plan.form == kLinear8Rows) {
    const dim3 grid(static_cast<unsigned>((p.N + 15) / 16));
    p.part = nullptr;
    if (p.M <= 16) hipLaunchKernelGGL((linear8_rows_kernel<YT, 8, 1, GATED>), grid, dim3(8 * kWave), 0, s, p);
    else hipLaunchKernelGGL((linear8_rows_kernel<YT, 8, 2, GATED>), grid, dim3(8 * kWave), 0, s, p);
    return hipGetLastError();
  }
  if (p.M > 1024 && p.K % 16 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0) {
    p.tiles_m = static_cast<int32_t>((p.M + 255) / 256);
    p.tiles_n = (p.N + (GATED ? 127 : 255)) / (GATED ? 128 : 256);
    p.part = nullptr;
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.tiles_m) * p.tiles_n));
    if (p.K % kStep == 0) hipLaunchKernelGGL((linear8_big_kernel<YT, 2, 4, GATED, false>), grid, dim3(8 * kWave), 0, s, p);
    else hipLaunchKernelGGL((linear8_big_kernel<YT, 2, 4, GATED, true>), grid, dim3(8 * kWave), 0, s, p);
    return hipGetLastError();
  }
  constexpr int BM = 128, BN = 128, OUT = GATED ? BN / 2 : BN;
  p.tiles_m = static_cast<int32_t>((p.M + BM - 1) / BM);
  p.tiles_n = (p.N + OUT - 1) / OUT;
  p.split_steps = plan.steps;
  if (plan.splits <= 1) p.part = nullptr;
  const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.tiles_m) * p.tiles_n), static_cast<unsigned>(plan.splits));
  hipLaunchKernelGGL((linear8_tile_kernel<YT, BM, BN, 2, 2, GATED>), grid, dim3(4 * kWave), 0, s, p);
  if (p.part) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t threads = p.M * ((p.N + 3) / 4);
    hipLaunchKernelGGL((linear8_reduce_kernel<YT, GATED>), dim3(static_cast<unsigned>((threads + kReduceThreads - 1) / kReduceThreads)),
                       dim3(kReduceThreads), 0, s, p, plan.splits);
  }
  return hipGetLastError();
}

template <bool GATED>
hipError_t launch_typed(const Linear8Params& p, const Linear8Plan& plan, hipStream_t s) {
  switch (p.y_dtype) {
    case CTI_EBAG_F32: return launch<float, GATED>(p, plan, s);
    case CTI_EBAG_BF16: return launch<bf16_t, GATED>(p, plan, s);
    default: return launch<f16_t, GATED>(p, plan, s);
  }
}

bool float_dtype(int32_t dt) { return dt == CTI_EBAG_F32 || dt == CTI_EBAG_BF16 || dt == CTI_EBAG_F16; }

}  // namespace
}  // namespace cti

using namespace cti;

extern "C" int64_t cti_ebag_linear_int8_workspace_bytes(int64_t rows, int32_t cols, int32_t out_features, int32_t gate) {
  if (rows < 1 || rows > INT32_MAX || cols < 1 || cols > kLinear8MaxK || out_features < 1 ||
      out_features > kLinear8MaxN || gate < CTI_EBAG_GATE_NONE || gate > CTI_EBAG_GATE_RELU)
    return 0;
  const bool gated = gate != CTI_EBAG_GATE_NONE;
  const Linear8Plan plan = linear8_plan(rows, out_features, cols, gated, INT64_MAX);
  return linear8_part_bytes(plan, rows, out_features, gated);
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
  const Linear8Plan plan = linear8_plan(rows, out_features, cols, gated, workspace ? workspace_bytes : 0);
  if (linear8_workgroups(plan, rows, out_features, gated) > INT32_MAX)
    return set_error(CTI_EBAG_EUNSUPPORTED, "too many output tiles (%lld x %d)", (long long)rows, out_features);
  Linear8Params p = {};
  p.x = q;
  p.scale = scale;
  p.w = weight;
  p.wscale = weight_scale;
  p.bias = bias;
  p.y = static_cast<char*>(y);
  p.part = static_cast<int32_t*>(workspace);
  p.M = rows;
  p.N = out_features;
  p.K = cols;
  p.bias_dtype = bias_dtype;
  p.y_dtype = y_dtype;
  p.gate = gate;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = gated ? launch_typed<true>(p, plan, s) : launch_typed<false>(p, plan, s);
  if (e != hipSuccess) return set_error(CTI_EBAG_EHIP, "linear launch failed: %s", hipGetErrorString(e));
  return CTI_EBAG_OK;
}
