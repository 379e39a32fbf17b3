// Dropout, and the layer norm with dropout and the residual's addition in it, forward and backward, for
// MI355X (gfx950).
//
//   dropout:   y = residual + keep(row, col) * x / (1 - p)
//   forward:   h = residual + keep * x / (1 - p), stored in x's type; y = (h - mean) * rstd * gamma + beta of
//              what is stored, so that the backward pass differentiates what the forward pass computed
//   backward:  z = (h - mean) * rstd, a = g * gamma
//              dh = rstd * (a - mean(a) - z * mean(a * z)) + grad_h      (the residual's gradient)
//              dx = keep * dh / (1 - p);  dgamma = sum over rows of g * z;  dbeta = sum over rows of g
// all in fp32 (sums too), one rounding to the outputs' types. The mask is never stored: it is a function of
// seed, offset, row and column.
//
// Bound by HBM, each array read or written once; the generator's multiplications come next. A row lies in
// the registers of 8 lanes (64 columns) to 512 threads (16,384 columns), chunks of 8 columns a thread; wider
// rows take a loop form. The backward pass adds up dgamma and dbeta over the rows of a workgroup, in registers
// or (8,193 to 16,384 columns) in LDS, which go to the workspace as one fp32 row each; a second kernel adds those
// up in their order (up to 256 rows of up to 8,192 columns: in the same launch, by workgroups that read the rows once
// more). No atomics: results are the same bits in every run.
//
// Measured (16,384 x 4,096 bf16; a read and a write of 1 GiB reach 6.25 TB/s here): dropout 44 us, with a residual 71 (6.1 and 5.7
// TB/s); forward with dropout and residual 95 (5.6); backward with grad_h and both gradients out 137 (4.9), and the
// parameters' sums 6.
#include <stdint.h>

#include "ebag_train.h"

namespace cti {
namespace {

// ---------------------------------------------------------------------------------------------
// Dropout
// ---------------------------------------------------------------------------------------------
constexpr int kDropThreads = 256;

struct DropParams {
  const char* x;
  const char* res;  // NULL: no residual
  char* y;
  int64_t cols;
  uint32_t first_row;
  uint32_t chunks;   // of this launch
  uint32_t per_row;
  ChunkDivide div;
  Dropout drop;
  int32_t stream_out;
};

template <typename T>
__global__ void __launch_bounds__(kDropThreads) dropout_kernel(const DropParams p) {
  const uint32_t c = blockIdx.x * kDropThreads + threadIdx.x;
  if (c >= p.chunks) return;
  const uint32_t row = p.div.quotient(c), chunk = c - row * p.per_row;
  const int cols = static_cast<int>(p.cols), col = static_cast<int>(chunk) * 8;
  const int64_t row_at = static_cast<int64_t>(row) * p.cols * Elem<T>::kBytes;
  Chunk<T> x, res;
  float v[8];
  x.load(p.x + row_at, col, cols);
  if (p.res) res.load(p.res + row_at, col, cols);
  x.unpack(v, col, cols);
  Dropout d = p.drop;
  if (d.threshold) {
    load_state(d);
    apply_dropout(d, p.first_row + row, chunk, v);
  }
  if (p.res) {
    float r[8];
    res.unpack(r, col, cols);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += r[e];
  }
  with_stream(p.stream_out, [&](auto stream) { store8<T, decltype(stream)::value>(p.y + row_at + static_cast<int64_t>(col) * Elem<T>::kBytes, cols - col, v); });
}

// ---------------------------------------------------------------------------------------------
// Norm
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ void round8(float* v) {
  if constexpr (std::is_same<T, bf16_t>::value) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t w = pack_bf16x2(v[e], v[e + 1]);
      v[e] = __uint_as_float(w << 16);
      v[e + 1] = __uint_as_float(w & 0xffff0000u);
    }
  } else if constexpr (std::is_same<T, f16_t>::value) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f16_bits_to_f32(f32_to_f16_bits(v[e]));
  }
}

// v + v of the lane across, by the cross-lane forms of the VALU: 5 steps of about 10 cycles where a trip through the LDS
// crossbar is 60 (16,384 x 4,096 bf16 backward, one reduction a row: see the kernel).
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over each LANES lanes side by side, the same bits in all of them: pairs, quads (permutations within four lanes), eights
// and sixteens (a row's halves, then the row, mirrored), rows and halves of the wavefront swapped.
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  static_assert(LANES == 8 || LANES == 16 || LANES == 32 || LANES == 64, "a power of two of lanes");
  v = add_dpp<0xb1>(v);   // lanes 1 0 3 2
  v = add_dpp<0x4e>(v);   // lanes 2 3 0 1
  v = add_dpp<0x141>(v);  // 7 - lane of each eight
  if constexpr (LANES >= 16) v = add_dpp<0x140>(v);  // 15 - lane of each sixteen
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LANES == 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// N sums over the LANES threads that hold a row, in a fixed order. s_red: N floats a wavefront that no thread still reads from
// another use (callers take turns between two: then one barrier is enough).
template <int LANES, int N>
__device__ __forceinline__ void row_sums(float* v, float* s_red) {
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lane_sum<(LANES < kWave ? LANES : kWave)>(v[k]);
  if constexpr (LANES > kWave) {
    constexpr int WAVES = LANES / kWave;
    float* const mine = s_red + threadIdx.x / LANES * (N * WAVES);  // the row's, of those side by side
    if (lane_id() == 0) {
#pragma unroll
      for (int k = 0; k < N; ++k) mine[k * WAVES + threadIdx.x % LANES / kWave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < WAVES; ++i) t += mine[k * WAVES + i];
      v[k] = t;
    }
  }
}

struct TrainNormParams {
  const char* x;
  const char* res;
  const void* gamma;
  const void* beta;
  char* h;  // NULL: h is x
  char* y;
  float* mean;
  float* rstd;
  int64_t rows;
  int64_t cols;
  uint32_t first_row;
  float eps;
  Dropout drop;
  int32_t param_dtype;
  int32_t stream_out;
};

template <int LANES>
struct Block {
  static constexpr int kThreads = LANES < 256 ? 256 : LANES;
  static constexpr int kSide = kThreads / LANES;  // rows side by side
  static constexpr int kReds = LANES <= kWave ? 1 : 2 * kThreads / kWave;  // one use of row_sums
};

template <typename T, int LANES, int K>
__global__ void __launch_bounds__(Block<LANES>::kThreads) train_norm_kernel(const TrainNormParams p) {
  __shared__ float s_red[2][Block<LANES>::kReds];
  const int t = static_cast<int>(threadIdx.x), lane = t % LANES;
  const int64_t want = static_cast<int64_t>(blockIdx.x) * Block<LANES>::kSide + t / LANES;
  const bool there = want < p.rows;  // the lanes of a row past the end take part in the shuffles
  const int64_t row = there ? want : p.rows - 1;
  const int cols = static_cast<int>(p.cols);
  const int64_t at = row * p.cols * Elem<T>::kBytes;
  Dropout d = p.drop;
  if (d.threshold) load_state(d);
  float v[K][8], s = 0.f;
  Chunk<T> x[K], r[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (lane + k * LANES) * 8;
    x[k].load(p.x + at, c, cols);
    if (p.res) r[k].load(p.res + at, c, cols);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (lane + k * LANES) * 8;
    x[k].unpack(v[k], c, cols);
    if (d.threshold) apply_dropout(d, p.first_row + static_cast<uint32_t>(row), static_cast<uint32_t>(c / 8), v[k]);
    if (p.res) {
      float w[8];
      r[k].unpack(w, c, cols);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] += w[e];
    }
    if (p.h) {
      round8<T>(v[k]);
      if (there && c < cols)
        with_stream(p.stream_out, [&](auto st) { store8<T, decltype(st)::value>(p.h + at + c * Elem<T>::kBytes, cols - c, v[k]); });
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[k][e];  // columns past the row are +0: dropped or kept
  }
  const float n = static_cast<float>(cols);
  row_sums<LANES, 1>(&s, s_red[0]);
  const float mean = s / n;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (lane + k * LANES) * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[k][e] = c + e < cols ? v[k][e] - mean : 0.f;
      q += v[k][e] * v[k][e];
    }
  }
  row_sums<LANES, 1>(&q, s_red[1]);
  const float rstd = 1.0f / __builtin_sqrtf(q / n + p.eps);
  if (!there) return;
  if (lane == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  with_stream(p.stream_out, [&](auto st) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (lane + k * LANES) * 8;
      if (c < cols) {
        float gm[8], bt[8];
        load_params8(p.gamma, p.param_dtype, c, cols, gm);
        load_params8(p.beta, p.param_dtype, c, cols, bt);
#pragma unroll
        for (int e = 0; e < 8; ++e) gm[e] = v[k][e] * rstd * gm[e] + bt[e];
        store8<T, decltype(st)::value>(p.y + at + c * Elem<T>::kBytes, cols - c, gm);
      }
    }
  });
}

// Rows of any width: a workgroup reads its row three times (h is made again each time).
constexpr int kWideThreads = 1024;
template <typename T>
__device__ __forceinline__ void wide_h(const TrainNormParams& p, const Dropout& d, int64_t row, int64_t c, float* v) {
  const int64_t at = (row * p.cols + c) * Elem<T>::kBytes;
  const int live = p.cols - c < 8 ? static_cast<int>(p.cols - c) : 8;
  load8<T>(p.x + at, live, v);
  if (d.threshold) apply_dropout(d, p.first_row + static_cast<uint32_t>(row), static_cast<uint32_t>(c / 8), v);
  if (p.res) {
    float w[8];
    load8<T>(p.res + at, live, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += w[e];
  }
  if (p.h) round8<T>(v);
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) train_norm_wide_kernel(const TrainNormParams p) {
  __shared__ float s_red[2][kWideThreads / kWave];
  const int64_t row = blockIdx.x, t = threadIdx.x;
  Dropout d = p.drop;
  if (d.threshold) load_state(d);
  float s = 0.f, v[8];
  for (int64_t c = t * 8; c < p.cols; c += kWideThreads * 8) {
    wide_h<T>(p, d, row, c, v);
    if (p.h) store8<T>(p.h + (row * p.cols + c) * Elem<T>::kBytes, p.cols - c < 8 ? static_cast<int>(p.cols - c) : 8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[e];
  }
  const float n = static_cast<float>(p.cols);
  row_sums<kWideThreads, 1>(&s, s_red[0]);
  const float mean = s / n;
  float q = 0.f;
  for (int64_t c = t * 8; c < p.cols; c += kWideThreads * 8) {
    wide_h<T>(p, d, row, c, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = c + e < p.cols ? v[e] - mean : 0.f;
      q += w * w;
    }
  }
  row_sums<kWideThreads, 1>(&q, s_red[1]);
  const float rstd = 1.0f / __builtin_sqrtf(q / n + p.eps);
  if (t == 0) {
    p.mean[row] = mean;
    p.rstd[row] = rstd;
  }
  for (int64_t c = t * 8; c < p.cols; c += kWideThreads * 8) {
    const int live = p.cols - c < 8 ? static_cast<int>(p.cols - c) : 8;
    float gm[8], bt[8];
    wide_h<T>(p, d, row, c, v);
    load_params8(p.gamma, p.param_dtype, static_cast<int>(c), static_cast<int>(p.cols), gm);
    load_params8(p.beta, p.param_dtype, static_cast<int>(c), static_cast<int>(p.cols), bt);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (v[e] - mean) * rstd * gm[e] + bt[e];
    store8<T>(p.y + (row * p.cols + c) * Elem<T>::kBytes, live, v);
  }
}

// ---------------------------------------------------------------------------------------------
// Norm, backward
// ---------------------------------------------------------------------------------------------
struct NormBackParams {
  const char* g;
  const char* h;
  const char* grad_h;  // NULL: none
  const float* mean;
  const float* rstd;
  const void* gamma;
  char* dh;  // NULL: not asked for (or the same as dx)
  char* dx;
  float* partial;  // [workgroup][dgamma, dbeta][whole chunks]
  char* dgamma;    // few rows: written by the workgroups behind the first row_groups
  char* dbeta;
  int64_t rows;
  int64_t cols;
  Dropout drop;
  int32_t param_dtype;
  int32_t stream_out;
  int32_t row_groups;  // workgroups that take rows
};

// gamma's and beta's gradients of COLS columns over all rows: COLS / 8 threads take a row's chunks, the others further
// rows; their sums are added in order. s_sum: 16 floats a thread.
// Rounds of rows in fours whose loads are under way together, the last ones' too: rows past the end are the last one again, and
// left out. (In a loop over each thread's own rows, unrolled by 8, what is left over is loaded row by row: 255 rows of 1,021
// columns 12.4 us, 6.7 so, 256 rows of 1,024 7.4 and 5.0.)
template <typename T, int THREADS, bool WHOLE, int COLS>
__device__ __forceinline__ void few_rows_columns(const NormBackParams& p, int block, float* s_sum) {
  constexpr int WIDE = COLS / 8, SIDE = THREADS / WIDE, AHEAD = 4;
  const int t = static_cast<int>(threadIdx.x), lane = t % WIDE, cols = static_cast<int>(p.cols), rows = static_cast<int>(p.rows);
  const int c = block * COLS + lane * 8;
  float sums[16] = {};
  if (c < cols) {
    for (int base = 0; base < rows; base += AHEAD * SIDE) {
      Chunk<T, WHOLE> gc[AHEAD], hc[AHEAD];
      float mean[AHEAD], rstd[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (base + u * SIDE < rows) {
          const int want = base + u * SIDE + t / WIDE, row = want < rows ? want : rows - 1;
          const int64_t at = static_cast<int64_t>(row) * p.cols * Elem<T>::kBytes;
          gc[u].load(p.g + at, c, cols);
          hc[u].load(p.h + at, c, cols);
          mean[u] = p.mean[row];
          rstd[u] = p.rstd[row];
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (base + u * SIDE < rows) {
          const bool there = base + u * SIDE + t / WIDE < rows;
          float g[8], h[8];
          gc[u].unpack(g, c, cols);
          hc[u].unpack(h, c, cols);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sums[e] += there ? g[e] * ((h[e] - mean[u]) * rstd[u]) : 0.f;
            sums[8 + e] += there ? g[e] : 0.f;
          }
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) s_sum[e * THREADS + t] = sums[e];
  __syncthreads();
  if (t >= 2 * WIDE) return;
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = 0.f;
    for (int r = 0; r < SIDE; ++r) v[e] += s_sum[((t / WIDE) * 8 + e) * THREADS + r * WIDE + lane];
  }
  if (c >= cols) return;
  char* const out = t < WIDE ? p.dgamma : p.dbeta;
  if (p.param_dtype == CTI_EBAG_F32) store8<float>(out + static_cast<int64_t>(c) * 4, cols - c, v);
  else if (p.param_dtype == CTI_EBAG_BF16) store8<bf16_t>(out + static_cast<int64_t>(c) * 2, cols - c, v);
  else store8<f16_t>(out + static_cast<int64_t>(c) * 2, cols - c, v);
}

// FEW: the parameters' gradients are the workgroups' behind the first row_groups (a kernel of its own: as a branch of this one
// their registers leave the rows a wavefront less a SIMD, 4,096 x 3,584 bf16 28 -> 36 us).
template <typename T, int LANES, int K, bool WHOLE, bool FEW>
__global__ void __launch_bounds__(Block<LANES>::kThreads) train_norm_back_kernel(const NormBackParams p) {
  constexpr int SIDE = Block<LANES>::kSide;
  __shared__ float s_red[2][Block<LANES>::kReds];
  int turn = 0;
  constexpr bool IN_LDS = LANES == 1024;
  __shared__ float s_acc[FEW ? 16 * Block<LANES>::kThreads : SIDE > 1 ? 2 * Block<LANES>::kThreads * 8 * K : 1];
  if constexpr (FEW) {
    if (static_cast<int>(blockIdx.x) >= p.row_groups) {
      few_rows_columns<T, Block<LANES>::kThreads, WHOLE, train_norm_few_cols(LANES)>(p, static_cast<int>(blockIdx.x) - p.row_groups, s_acc);
      return;
    }
  }
  const int t = static_cast<int>(threadIdx.x), lane = t % LANES;
  const int cols = static_cast<int>(p.cols);
  const float n = static_cast<float>(cols);
  Dropout d = p.drop;
  if (d.threshold) load_state(d);
  // The next row's loads are under way while this one is worked on (fp32 rows of 1,024 threads leave no registers for it).
  constexpr bool AHEAD = LANES < 1024 || Elem<T>::kBytes == 2;
  // gamma's and beta's gradients: in registers, or in LDS where a thread's are the float4s of its chunks, four arrays of them
  __shared__ float4 s_sums[IN_LDS ? 4 * LANES * K : 1];
  float dgamma[IN_LDS ? 1 : K][8], dbeta[IN_LDS ? 1 : K][8], gamma[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (lane + k * LANES) * 8;
    if constexpr (IN_LDS) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s_sums[(j * K + k) * LANES + lane] = make_float4(0.f, 0.f, 0.f, 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dgamma[k][e] = dbeta[k][e] = 0.f;
    }
    load_params8(p.gamma, p.param_dtype, c, cols, gamma[k]);
  }
  const int64_t step = static_cast<int64_t>(p.row_groups) * SIDE;
  struct Row {
    Chunk<T, WHOLE> g[K], h[K], gh[K];
    float mean, rstd;
  };
  const auto fetch = [&](int64_t row, Row& r, bool all = true) {
    const int64_t at = row * p.cols * Elem<T>::kBytes;
    r.mean = p.mean[row];
    r.rstd = p.rstd[row];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (lane + k * LANES) * 8;
      r.g[k].load(p.g + at, c, cols);
      r.h[k].load(p.h + at, c, cols);
      if (all && p.grad_h) r.gh[k].load(p.grad_h + at, c, cols);
    }
  };
  // whole rounds of rows: a group past the last row repeats it and leaves its results out
  const int64_t mine = static_cast<int64_t>(blockIdx.x) * SIDE + t / LANES;
  Row now, next;
  if constexpr (AHEAD) fetch(mine < p.rows ? mine : p.rows - 1, now);
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * SIDE; base < p.rows; base += step) {
    const int64_t row = base + t / LANES;
    const bool there = row < p.rows;
    if constexpr (AHEAD) {
      if (base + step < p.rows) fetch(row + step < p.rows ? row + step : p.rows - 1, next);
    } else {
      fetch(there ? row : p.rows - 1, now, false);
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (lane + k * LANES) * 8;
      float g[8], h[8];
      now.g[k].unpack(g, c, cols);
      now.h[k].unpack(h, c, cols);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = WHOLE ? c < cols : c + e < cols;
        const float z = (h[e] - now.mean) * now.rstd, a = g[e] * gamma[k][e];
        s[0] += in ? a : 0.f;
        s[1] += in ? a * z : 0.f;
        if constexpr (IN_LDS) {
          h[e] = g[e] * z;
        } else if (there) {  // (of columns past the row: left out below)
          dgamma[k][e] += g[e] * z;
          dbeta[k][e] += g[e];
        }
      }
      if constexpr (IN_LDS) {  // one row a workgroup: it is there
        const auto add = [&](int j, const float* v) {
          float4& at = s_sums[(j * K + k) * LANES + lane];
          const float4 o = at;
          at = make_float4(o.x + v[0], o.y + v[1], o.z + v[2], o.w + v[3]);
        };
        add(0, h), add(1, h + 4), add(2, g), add(3, g + 4);
      }
    }
    row_sums<LANES, 2>(s, s_red[turn]);
    turn ^= 1;
    if constexpr (AHEAD) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        now.g[k].forget();
        now.h[k].forget();
      }
    } else {
      fetch(there ? row : p.rows - 1, now);
    }
    const float m0 = s[0] / n, m1 = s[1] / n;
    if (there) {
      const int64_t at = row * p.cols * Elem<T>::kBytes;
      with_stream(p.stream_out, [&](auto st) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (lane + k * LANES) * 8;
          if (c < cols) {
            float g[8], h[8], v[8];
            now.g[k].unpack(g, c, cols);
            now.h[k].unpack(h, c, cols);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float z = (h[e] - now.mean) * now.rstd;
              v[e] = now.rstd * (g[e] * gamma[k][e] - m0 - z * m1);
            }
            if (p.grad_h) {
              now.gh[k].unpack(g, c, cols);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] += g[e];
            }
            if (p.dh) store8<T, decltype(st)::value>(p.dh + at + c * Elem<T>::kBytes, cols - c, v);
            if (d.threshold) apply_dropout(d, static_cast<uint32_t>(row), static_cast<uint32_t>(c / 8), v);
            store8<T, decltype(st)::value>(p.dx + at + c * Elem<T>::kBytes, cols - c, v);
          }
        }
      });
    }
    if constexpr (AHEAD) now = next;
  }
  if constexpr (FEW) return;
  // the workgroup's sums: of the rows side by side through LDS, in their order
  const int64_t width = ceil_div(p.cols, 8) * 8;
  float* const out = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * width;
  if constexpr (SIDE > 1) {
    const int wide = LANES * K * 8;
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = (lane + k * LANES) * 8 + e;
        s_acc[(t / LANES) * wide + c] = dgamma[k][e];
        s_acc[(SIDE + t / LANES) * wide + c] = dbeta[k][e];
      }
    }
    __syncthreads();
    for (int i = t; i < 2 * wide; i += Block<LANES>::kThreads) {
      const int which = i / wide, c = i % wide;
      float sum = 0.f;
      for (int r = 0; r < SIDE; ++r) sum += s_acc[(which * SIDE + r) * wide + c];
      if (c < width) out[which * width + c] = sum;
    }
  } else if constexpr (IN_LDS) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (lane + k * LANES) * 8;
      if (c < cols) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          *reinterpret_cast<float4*>(out + (j / 2) * width + c + (j % 2) * 4) = s_sums[(j * K + k) * LANES + lane];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (lane + k * LANES) * 8;
      if (c < cols) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          *reinterpret_cast<float4*>(out + c + e) = make_float4(dgamma[k][e], dgamma[k][e + 1], dgamma[k][e + 2], dgamma[k][e + 3]);
          *reinterpret_cast<float4*>(out + width + c + e) = make_float4(dbeta[k][e], dbeta[k][e + 1], dbeta[k][e + 2], dbeta[k][e + 3]);
        }
      }
    }
  }
}

// Rows of any width: a workgroup a row, read twice (the second time from L2) ...
template <typename T>
__global__ void __launch_bounds__(kWideThreads) train_norm_back_wide_kernel(const NormBackParams p) {
  __shared__ float s_red[2][2 * kWideThreads / kWave];
  int turn = 0;
  const int t = static_cast<int>(threadIdx.x), cols = static_cast<int>(p.cols);
  const float n = static_cast<float>(cols);
  Dropout d = p.drop;
  if (d.threshold) load_state(d);
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.mean[row], rstd = p.rstd[row];
    const int64_t at = row * p.cols * Elem<T>::kBytes;
    float s[2] = {0.f, 0.f}, g[8], h[8], gamma[8];
    const auto load = [&](int c) {
      Chunk<T> gc, hc;
      gc.load(p.g + at, c, cols);
      hc.load(p.h + at, c, cols);
      load_params8(p.gamma, p.param_dtype, c, cols, gamma);
      gc.unpack(g, c, cols);
      hc.unpack(h, c, cols);
    };
    for (int c = t * 8; c < cols; c += kWideThreads * 8) {
      load(c);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float z = c + e < cols ? (h[e] - mean) * rstd : 0.f, a = g[e] * gamma[e];
        s[0] += a;
        s[1] += a * z;
      }
    }
    row_sums<kWideThreads, 2>(s, s_red[turn]);
    turn ^= 1;
    const float m0 = s[0] / n, m1 = s[1] / n;
    for (int c = t * 8; c < cols; c += kWideThreads * 8) {
      load(c);
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = rstd * (g[e] * gamma[e] - m0 - (h[e] - mean) * rstd * m1);
      if (p.grad_h) {
        Chunk<T> gh;
        gh.load(p.grad_h + at, c, cols);
        gh.unpack(g, c, cols);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += g[e];
      }
      const int64_t to = at + static_cast<int64_t>(c) * Elem<T>::kBytes;
      if (p.dh) store8<T>(p.dh + to, cols - c, v);
      if (d.threshold) apply_dropout(d, static_cast<uint32_t>(row), static_cast<uint32_t>(c / 8), v);
      store8<T>(p.dx + to, cols - c, v);
    }
  }
}
// ... and the parameters' gradients of 2,048 columns over a share of the rows (blockIdx.y), read once more.
constexpr int kColumnThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kColumnThreads) train_norm_columns_kernel(const NormBackParams p) {
  const int cols = static_cast<int>(p.cols);
  const int64_t first = (static_cast<int64_t>(blockIdx.x) * kColumnThreads + threadIdx.x) * 8;
  if (first >= cols) return;
  const int c = static_cast<int>(first);
  float dgamma[8] = {}, dbeta[8] = {};
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const int64_t at = row * p.cols * Elem<T>::kBytes;
    Chunk<T> gc, hc;
    gc.load(p.g + at, c, cols);
    hc.load(p.h + at, c, cols);
    const float mean = p.mean[row], rstd = p.rstd[row];
    float g[8], h[8];
    gc.unpack(g, c, cols);
    hc.unpack(h, c, cols);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dgamma[e] += g[e] * ((h[e] - mean) * rstd);
      dbeta[e] += g[e];
    }
  }
  const int64_t width = ceil_div(p.cols, 8) * 8;
  float* const out = p.partial + static_cast<int64_t>(blockIdx.y) * 2 * width + c;
#pragma unroll
  for (int e = 0; e < 8; e += 4) {
    *reinterpret_cast<float4*>(out + e) = make_float4(dgamma[e], dgamma[e + 1], dgamma[e + 2], dgamma[e + 3]);
    *reinterpret_cast<float4*>(out + width + e) = make_float4(dbeta[e], dbeta[e + 1], dbeta[e + 2], dbeta[e + 3]);
  }
}

// dgamma (blockIdx.y 0) and dbeta (1): the workgroups' sums, ROWS of them side by side, then those in order. 64 for many
// (1,024 workgroups' of 1,021 columns: 16 side by side 7.9 us, 64 5.9; 128 workgroups' of 3,584: 3.3 and 4.6).
constexpr int kParamQuads = 16;
template <typename PT, int ROWS>
__global__ void __launch_bounds__(ROWS * kParamQuads) train_norm_params_kernel(const float* partial, int workgroups, int64_t cols,
                                                                               char* dgamma, char* dbeta) {
  __shared__ float4 s_sum[ROWS * kParamQuads];
  const int t = static_cast<int>(threadIdx.x), q = t % kParamQuads, r = t / kParamQuads;
  const int64_t width = ceil_div(cols, 8) * 8, c = (static_cast<int64_t>(blockIdx.x) * kParamQuads + q) * 4;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < width) {
    const float* const from = partial + static_cast<int64_t>(blockIdx.y) * width + c;
#pragma unroll 8
    for (int w = r; w < workgroups; w += ROWS) {
      const float4 v = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(w) * 2 * width);
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
  }
  s_sum[t] = sum;
  __syncthreads();
  if (r != 0 || c >= cols) return;
  for (int i = 1; i < ROWS; ++i) {
    const float4 v = s_sum[i * kParamQuads + q];
    sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
  }
  const float v[4] = {sum.x, sum.y, sum.z, sum.w};
  store_vec<PT, 4>((blockIdx.y ? dbeta : dgamma) + c * Elem<PT>::kBytes, cols - c < 4 ? static_cast<int>(cols - c) : 4, v);
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
// f(LANES, K) for the register form of a width, as types.
template <int V>
using Const = std::integral_constant<int, V>;
template <typename F>
void with_form(const TrainNormForm& form, F&& f) {
  if (form.lanes == 8) f(Const<8>{}, Const<1>{});
  else if (form.lanes == 16) f(Const<16>{}, Const<1>{});
  else if (form.lanes == 32) f(Const<32>{}, Const<1>{});
  else if (form.lanes == 64) f(Const<64>{}, Const<1>{});
  else if (form.lanes == 128) f(Const<128>{}, Const<1>{});
  else if (form.lanes == 256 && form.chunks == 1) f(Const<256>{}, Const<1>{});
  else if (form.lanes == 256) f(Const<256>{}, Const<2>{});
  else if (form.chunks == 1) f(Const<512>{}, Const<1>{});
  else if (form.chunks == 2) f(Const<512>{}, Const<2>{});
  else f(Const<512>{}, Const<4>{});
}

template <typename F>
void with_back_form(const TrainNormForm& form, F&& f) {
  if (form.lanes == 8) f(Const<8>{}, Const<1>{});
  else if (form.lanes == 16) f(Const<16>{}, Const<1>{});
  else if (form.lanes == 32) f(Const<32>{}, Const<1>{});
  else if (form.lanes == 64) f(Const<64>{}, Const<1>{});
  else if (form.lanes == 128) f(Const<128>{}, Const<1>{});
  else if (form.lanes == 256) f(Const<256>{}, Const<1>{});
  else if (form.lanes == 512 && form.chunks == 1) f(Const<512>{}, Const<1>{});
  else if (form.lanes == 512) f(Const<512>{}, Const<2>{});
  else f(Const<1024>{}, Const<2>{});
}

int check_norm(int64_t rows, int64_t cols, int32_t dtype, int32_t param_dtype) {
  if (rows < 0) return set_error(CTI_EBAG_EINVAL, "rows must be >= 0 (got %lld)", (long long)rows);
  if (cols < 1) return set_error(CTI_EBAG_EINVAL, "cols must be >= 1 (got %lld)", (long long)cols);
  if (!float_dtype(dtype)) return set_error(CTI_EBAG_EINVAL, "unknown dtype code %d", dtype);
  if (!float_dtype(param_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown parameter dtype code %d", param_dtype);
  if (rows > INT32_MAX) return set_error(CTI_EBAG_EUNSUPPORTED, "more than 2^31 - 1 rows (%lld)", (long long)rows);
  if (cols > INT32_MAX / 8) return set_error(CTI_EBAG_EUNSUPPORTED, "more than 2^28 - 1 columns (%lld)", (long long)cols);
  return CTI_EBAG_OK;
}

}  // namespace
}  // namespace cti

using namespace cti;

extern "C" int cti_ebag_dropout(const void* x, const void* residual, void* y, int64_t rows, int64_t cols, int32_t dtype, double p,
                                uint64_t seed, uint64_t offset, const int64_t* state, void* stream) {
  clear_error();
  const int rc = check_norm(rows, cols, dtype, dtype);
  if (rc != CTI_EBAG_OK) return rc;
  DropParams a{};
  if (!set_dropout(&a.drop, p, seed, offset, state)) return set_error(CTI_EBAG_EINVAL, "p must be in [0, 1] (got %g)", p);
  if (rows == 0) return CTI_EBAG_OK;
  if (!x || !y) return set_error(CTI_EBAG_EINVAL, "NULL device pointer among x/y");
  const int64_t row_bytes = cols * dtype_bytes(dtype);
  a.cols = cols;
  a.per_row = static_cast<uint32_t>(ceil_div(cols, 8));
  a.div = ChunkDivide::by(a.per_row);
  a.stream_out = rows * row_bytes >= kStreamOutBytes;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t per_launch = kMostChunks / a.per_row;  // rows
  for (int64_t r = 0; r < rows; r += per_launch) {
    const int64_t now = rows - r < per_launch ? rows - r : per_launch;
    a.x = static_cast<const char*>(x) + r * row_bytes;
    a.res = residual ? static_cast<const char*>(residual) + r * row_bytes : nullptr;
    a.y = static_cast<char*>(y) + r * row_bytes;
    a.first_row = static_cast<uint32_t>(r);
    a.chunks = static_cast<uint32_t>(now * a.per_row);
    const dim3 grid((a.chunks + kDropThreads - 1) / kDropThreads), block(kDropThreads);
    with_type(dtype, [&](auto t) { hipLaunchKernelGGL((dropout_kernel<decltype(t)>), grid, block, 0, s, a); });
  }
  return check_launch("dropout");
}

extern "C" int cti_ebag_dropout_layernorm(const void* x, const void* residual, void* h, void* y, int64_t rows, int64_t cols,
                                          int32_t dtype, const void* gamma, const void* beta, int32_t param_dtype, float eps, double p,
                                          uint64_t seed, uint64_t offset, const int64_t* state, float* mean, float* rstd,
                                          void* stream) {
  clear_error();
  const int rc = check_norm(rows, cols, dtype, param_dtype);
  if (rc != CTI_EBAG_OK) return rc;
  if (!(eps >= 0.f)) return set_error(CTI_EBAG_EINVAL, "eps must be >= 0");
  TrainNormParams a{};
  if (!set_dropout(&a.drop, p, seed, offset, state)) return set_error(CTI_EBAG_EINVAL, "p must be in [0, 1] (got %g)", p);
  const bool plain = !residual && a.drop.threshold == 0;
  if (rows == 0) return CTI_EBAG_OK;
  if (!x || !y || !gamma || !beta || !mean || !rstd)
    return set_error(CTI_EBAG_EINVAL, "NULL device pointer among x/y/gamma/beta/mean/rstd");
  if (!plain && !h) return set_error(CTI_EBAG_EINVAL, "h is NULL: a call with dropout or a residual writes it");
  const int64_t row_bytes = cols * dtype_bytes(dtype);
  a.gamma = gamma;
  a.beta = beta;
  a.cols = cols;
  a.eps = eps;
  a.param_dtype = param_dtype;
  a.stream_out = rows * row_bytes >= kStreamOutBytes;
  const TrainNormForm form = train_norm_form(cols, dtype_bytes(dtype));
  const int threads = form.lanes == 0 ? kWideThreads : form.lanes < 256 ? 256 : form.lanes;
  const int side = form.lanes > 0 && form.lanes < 256 ? 256 / form.lanes : 1;
  const int64_t per_launch = (int64_t{1} << 31) / threads * side;  // rows: below 2^32 threads
  const hipStream_t s = static_cast<hipStream_t>(stream);
  for (int64_t r = 0; r < rows; r += per_launch) {
    a.rows = rows - r < per_launch ? rows - r : per_launch;
    a.x = static_cast<const char*>(x) + r * row_bytes;
    a.res = residual ? static_cast<const char*>(residual) + r * row_bytes : nullptr;
    a.h = h ? static_cast<char*>(h) + r * row_bytes : nullptr;
    a.y = static_cast<char*>(y) + r * row_bytes;
    a.mean = mean + r;
    a.rstd = rstd + r;
    a.first_row = static_cast<uint32_t>(r);
    const dim3 grid(static_cast<unsigned>(ceil_div(a.rows, side))), block(threads);
    with_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (form.lanes == 0) {
        hipLaunchKernelGGL((train_norm_wide_kernel<T>), grid, block, 0, s, a);
      } else {
        with_form(form, [&](auto lanes, auto k) {
          hipLaunchKernelGGL((train_norm_kernel<T, decltype(lanes)::value, decltype(k)::value>), grid, block, 0, s, a);
        });
      }
    });
  }
  return check_launch("dropout_layernorm");
}

extern "C" int64_t cti_ebag_dropout_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols < 1 || rows > INT32_MAX || cols > INT32_MAX / 8 ? 0 : train_norm_workspace_bytes(rows, cols);
}

extern "C" int cti_ebag_dropout_layernorm_backward(const void* grad, const void* h, const void* grad_h, const float* mean,
                                                   const float* rstd, int64_t rows, int64_t cols, int32_t dtype, const void* gamma,
                                                   int32_t param_dtype, double p, uint64_t seed, uint64_t offset,
                                                   const int64_t* state, void* dx, void* dresidual, void* dgamma, void* dbeta,
                                                   void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  const int rc = check_norm(rows, cols, dtype, param_dtype);
  if (rc != CTI_EBAG_OK) return rc;
  NormBackParams a{};
  if (!set_dropout(&a.drop, p, seed, offset, state)) return set_error(CTI_EBAG_EINVAL, "p must be in [0, 1] (got %g)", p);
  if (!dgamma || !dbeta || (rows > 0 && (!grad || !h || !mean || !rstd || !gamma || !dx)))
    return set_error(CTI_EBAG_EINVAL, "NULL device pointer among grad/h/mean/rstd/gamma/dx/dgamma/dbeta");
  const int64_t need = train_norm_workspace_bytes(rows, cols);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(CTI_EBAG_EWORKSPACE, "workspace of %lld bytes, %lld needed", (long long)(workspace ? workspace_bytes : 0),
                     (long long)need);
  if (need > 0 && reinterpret_cast<uintptr_t>(workspace) % 16) return set_error(CTI_EBAG_EINVAL, "workspace is not 16-byte aligned");
  a.g = static_cast<const char*>(grad);
  a.h = static_cast<const char*>(h);
  a.grad_h = static_cast<const char*>(grad_h);
  a.mean = mean;
  a.rstd = rstd;
  a.gamma = gamma;
  a.dh = static_cast<char*>(dresidual);
  a.dx = static_cast<char*>(dx);
  a.partial = static_cast<float*>(workspace);
  a.rows = rows;
  a.cols = cols;
  a.param_dtype = param_dtype;
  a.stream_out = rows * cols * dtype_bytes(dtype) >= kStreamOutBytes;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const TrainNormForm form = train_norm_back_form(cols);
  const int64_t workgroups = rows > 0 ? train_norm_workgroups(rows, cols) : 0;
  const bool few = rows > 0 && train_norm_few(rows, cols);
  a.dgamma = static_cast<char*>(dgamma);
  a.dbeta = static_cast<char*>(dbeta);
  a.row_groups = static_cast<int32_t>(workgroups);
  const dim3 grid(static_cast<unsigned>(workgroups + (few ? ceil_div(cols, train_norm_few_cols(form.lanes)) : 0)));
  const dim3 block(form.lanes == 0 ? kWideThreads : form.lanes < 256 ? 256 : form.lanes);
  if (rows > 0) {
    with_type(dtype, [&](auto t) {
      using T = decltype(t);
      if (form.lanes == 0) {
        const unsigned blocks = static_cast<unsigned>(ceil_div(cols, kColumnThreads * 8));
        hipLaunchKernelGGL((train_norm_back_wide_kernel<T>), dim3(static_cast<unsigned>(rows < 4096 ? rows : 4096)), block, 0, s, a);
        hipLaunchKernelGGL((train_norm_columns_kernel<T>), dim3(blocks, static_cast<unsigned>(workgroups)), dim3(kColumnThreads), 0, s, a);
      } else {
        with_back_form(form, [&](auto lanes, auto k) {
          constexpr int LANES = decltype(lanes)::value, K = decltype(k)::value;
          if (few) {
            if constexpr (LANES < 1024) {  // up to 8,192 columns
              if (cols % 8 == 0) hipLaunchKernelGGL((train_norm_back_kernel<T, LANES, K, true, true>), grid, block, 0, s, a);
              else hipLaunchKernelGGL((train_norm_back_kernel<T, LANES, K, false, true>), grid, block, 0, s, a);
            }
          } else if (cols % 8 == 0) {
            hipLaunchKernelGGL((train_norm_back_kernel<T, LANES, K, true, false>), grid, block, 0, s, a);
          } else {
            hipLaunchKernelGGL((train_norm_back_kernel<T, LANES, K, false, false>), grid, block, 0, s, a);
          }
        });
      }
    });
  }
  if (few) return check_launch("dropout_layernorm_backward");
  with_type(param_dtype, [&](auto pt) {
    using PT = decltype(pt);
    const dim3 sums(static_cast<unsigned>(ceil_div(cols, kParamQuads * 4)), 2);
    const int n = static_cast<int>(workgroups);
    char* const dg = static_cast<char*>(dgamma);
    char* const db = static_cast<char*>(dbeta);
    if (n <= 256) hipLaunchKernelGGL((train_norm_params_kernel<PT, 16>), sums, dim3(16 * kParamQuads), 0, s, a.partial, n, cols, dg, db);
    else hipLaunchKernelGGL((train_norm_params_kernel<PT, 64>), sums, dim3(64 * kParamQuads), 0, s, a.partial, n, cols, dg, db);
  });
  return check_launch("dropout_layernorm_backward");
}
