// Row norms with int8 output for MI355X (gfx950): the residual's addition, LayerNorm or root-mean-square
// norm, and the quantisation of the normalised row in one pass.
//
//   h = x + residual                                (fp32; residual_out = h rounded to x's type)
//   RMS:   y = h * rstd * gamma,                    rstd = 1 / sqrt(sum(h^2) / cols + eps)
//   Layer: y = (h - mean) * rstd * gamma + beta,    rstd = 1 / sqrt(sum((h - mean)^2) / cols + eps)
//   m = max_j |y_j|, s = max(m * RN32(1/127), 1e-8), q_j = clamp(rint(y_j / s), -128, 127)
// all in fp32 (h is not rounded before the norm reads it), the quantisation the one of
// quantize_embedding_int8 (online_best/infer.py:895-901). A row whose statistics or normalised values are
// not all finite gets the scale NaN and q = 0, so that what is computed from it is NaN, and only that.
//
// Bound by HBM: per element x and the residual are read once and residual_out and one byte written. A
// workgroup holds its row in registers as 16-byte vectors between the sum, the maximum and the output, so
// nothing is read twice. gamma and beta come from L1 / L2.
// Widths that are not whole vectors: the last vector ends with the row and overlaps the one before it;
// elements it shares are left out of the sums and written twice with the same value (stores come after a
// reduction over the whole row, so residual_out may be x or residual). Addresses need no more than the
// element's alignment (the vector loads of gfx950 take any).
#include <stdint.h>

#include <initializer_list>

#include "ebag_device.h"
#include "ebag_internal.h"
#include "ebag_rules.h"

namespace cti {
namespace {

constexpr int kLoopThreads = 256;

struct Norm8Params {
  const char* x;
  const char* res;  // NULL: no residual
  char* res_out;
  const void* gamma;
  const void* beta;  // layer only
  int8_t* q;
  float* scale;
  int64_t cols;
  float eps;
  int32_t layer;       // LayerNorm, else root-mean-square norm
  int32_t stream_out;  // residual_out is at least kStreamOutBytes: non-temporal stores
};

// VEC parameters from element c0 on, as loaded: 8, 16 or 32 bytes.
template <typename PT, int VEC>
struct Params {
  static constexpr int kBytes = VEC * Elem<PT>::kBytes;
  uint4 raw[kBytes > 16 ? kBytes / 16 : 1];
  __device__ __forceinline__ void load(const void* p, int64_t c0) {
    const char* const base = static_cast<const char*>(p) + c0 * Elem<PT>::kBytes;
    if constexpr (kBytes == 8) {
      const u32x2 u = *reinterpret_cast<const u32x2_any*>(base);
      raw[0] = make_uint4(u.x, u.y, 0u, 0u);
    } else {
#pragma unroll
      for (int h = 0; h < kBytes / 16; ++h) raw[h] = load16_any(base + h * 16);
    }
  }
  __device__ __forceinline__ void unpack(float* out) const {
    constexpr int N = 16 / Elem<PT>::kBytes;
    float t[N];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      if (e % N == 0) unpack16(raw[e / N], t, PT{});
      out[e] = t[e % N];
    }
  }
};

// The larger of m and every |v|, NaN if any is: one instruction for two of them.
template <int N>
__device__ __forceinline__ float top_of(float m, const float* v) {
#pragma unroll
  for (int e = 0; e < N; e += 2)
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(v[e]), __builtin_fabsf(v[e + 1])), m);
  return m;
}

// The scale of a row whose largest |y| has these bits; NaN for infinity and NaN.
__device__ __forceinline__ float scale_of(uint32_t bits) {
  const float s = __uint_as_float(bits) * (1.0f / 127.0f);
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return s < 1e-8f ? 1e-8f : s;
}

// RN32(v / s), given inv = RN32(1 / s), where the quotient is neither tiny nor huge (for others a number that rounds to the
// same byte): v * inv is within 1.5 last places, one correction by the exact remainder brings it within one, and from
// there a correction with the reciprocal rounded to nearest gives the quotient rounded to nearest (Markstein, 1990).
__device__ __forceinline__ float quotient(float v, float s, float inv) {
  float y = v * inv;
  y = __builtin_fmaf(__builtin_fmaf(-y, s, v), inv, y);
  return __builtin_fmaf(__builtin_fmaf(-y, s, v), inv, y);
}

constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: a sum with it leaves the nearest integer (ties to even) in the low byte

template <int VEC>
__device__ __forceinline__ void store_low_bytes(int8_t* dst, const uint32_t* t, bool live) {
  uint32_t w[VEC / 4];
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) {
    const uint32_t* const b = t + 4 * i;
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
    w[i] = live ? __builtin_amdgcn_perm(hi, lo, 0x05040100u) : 0u;
  }
  if constexpr (VEC == 4) *reinterpret_cast<u32_any*>(dst) = w[0];
  else *reinterpret_cast<u32x2_any*>(dst) = u32x2{w[0], w[1]};
}

// VEC bytes rint(RN32(v / s)), given inv = RN32(1 / s); |v / s| <= 127 (1 + 2^-22). A product with a reciprocal is exact
// inside the addition of kMagic. It is taken twice: three last places below inv are at most (1 / s) (1 - 2^-24), three above
// at least (1 / s) (1 + 2^-24), so |RN32(v / s)| lies between the two products, and where their nearest integers agree it is
// the quotient's (they are compared by 16 bits). Else (an element in 50,000, more where bf16 values meet weights of 1 and
// lie in the middle itself) the vector is stored again from the quotients. (One product, its bytes off by one next to the
// middle: 16,384 x 1,024 bf16 13.3 us, 13.7 so; LayerNorm 4,096 x 3,584 12.3 and 12.7; what HBM bounds takes as long.)
// `live` false (the row's scale is NaN): zeros.
template <int VEC>
__device__ __forceinline__ void store_quantised(int8_t* dst, const float* v, float s, float inv, bool live) {
  const float lo_inv = __uint_as_float(__float_as_uint(inv) - 3u), hi_inv = __uint_as_float(__float_as_uint(inv) + 3u);
  uint32_t t[VEC], apart = 0u;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    t[e] = __float_as_uint(__builtin_fmaf(v[e], lo_inv, kMagic));
    apart = __builtin_amdgcn_sad_u16(t[e], __float_as_uint(__builtin_fmaf(v[e], hi_inv, kMagic)), apart);
  }
  store_low_bytes<VEC>(dst, t, live);
  if (__builtin_expect(apart != 0u, 0)) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = __float_as_uint(quotient(v[e], s, inv) + kMagic);
    store_low_bytes<VEC>(dst, t, live);
  }
}

// 1 / sqrt(var + eps); NaN where the sum of squares left fp32's range (it would give a row of zeros).
__device__ __forceinline__ float rstd_of(float var, float eps) {
  const float r = 1.0f / __builtin_sqrtf(var + eps);
  return var < __builtin_inff() ? r : __uint_as_float(0x7fc00000u);
}

// One 16-byte vector of rounded values.
__device__ __forceinline__ u32x4 pack16(const float* v, float) {
  return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
__device__ __forceinline__ u32x4 pack16(const float* v, bf16_t) {
  return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ u32x4 pack16(const float* v, f16_t) {
  return u32x4{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7])};
}

// One row per workgroup of WAVES wavefronts, the row in registers: thread t holds vectors
// t, t + THREADS, ... (K of them). At least one whole vector per row.
template <typename T, typename PT, int K, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave) norm8_rows_kernel(const Norm8Params p) {
  constexpr int VEC = 16 / Elem<T>::kBytes;
  constexpr int THREADS = WAVES * kWave;
  constexpr bool kEarly = K <= 2;  // gamma and beta are loaded with x where registers allow
  __shared__ float s_sum[WAVES];
  __shared__ uint32_t s_max[WAVES];
  const int64_t row = blockIdx.x;
  const int t = static_cast<int>(threadIdx.x);
  const int cols = static_cast<int>(p.cols);
  const int nfull = cols / VEC, rest = cols % VEC;
  const int nvec = nfull + (rest != 0);
  const int64_t at = row * p.cols;
  const auto first = [&](int i) { return i < nfull ? i * VEC : cols - VEC; };  // vector i's first column

  uint4 rx[K], rr[K];
  Params<PT, VEC> gm[kEarly ? K : 1], bt[kEarly ? K : 1];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = t + k * THREADS;
    rx[k] = rr[k] = make_uint4(0u, 0u, 0u, 0u);
    if (i < nvec) {
      rx[k] = load16_any(p.x + (at + first(i)) * Elem<T>::kBytes);
      if (p.res) rr[k] = load16_any(p.res + (at + first(i)) * Elem<T>::kBytes);
      if constexpr (kEarly) {
        gm[k].load(p.gamma, first(i));
        if (p.layer) bt[k].load(p.beta, first(i));
      }
    }
  }
  float v[K][VEC];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    unpack16(rx[k], v[k], T{});
    if (p.res) {
      float r[VEC];
      unpack16(rr[k], r, T{});
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[k][e] += r[e];
    }
  }
  // f over the elements that count: not those that the last vector shares with the one before it, and where `beyond`
  // is set not those of vectors past the row (which hold 0)
  const auto each = [&](bool beyond, auto&& f) {
    if (rest == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (beyond && t + k * THREADS >= nvec) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(v[k][e], true);
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = t + k * THREADS;
        const int shared = i < nfull ? 0 : (i < nvec ? VEC - rest : (beyond ? VEC : 0));
#pragma unroll
        for (int e = 0; e < VEC; ++e) f(v[k][e], e >= shared);
      }
    }
  };
  const float n = static_cast<float>(cols);
  float mean = 0.f, s = 0.f;
  if (p.layer) {
    each(false, [&](float& x, bool counts) { s += counts ? x : 0.f; });
    mean = block_sum<WAVES>(s, s_sum) / n;
    s = 0.f;
    each(true, [&](float& x, bool counts) {
      const float d = counts ? x - mean : 0.f;
      s = __builtin_fmaf(d, d, s);
    });
  } else {
    each(false, [&](float& x, bool counts) {
      const float c = counts ? x : 0.f;
      s = __builtin_fmaf(c, c, s);
    });
  }
  s = block_sum<WAVES>(s, s_sum) / n;
  const float rstd = rstd_of(s, p.eps);
  if (p.res) {
    with_stream(p.stream_out, [&](auto stream) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int i = t + k * THREADS;
        if (i < nvec) {
          u32x4_any* const dst = reinterpret_cast<u32x4_any*>(p.res_out + (at + first(i)) * Elem<T>::kBytes);
          if constexpr (decltype(stream)::value) __builtin_nontemporal_store(pack16(v[k], T{}), dst);
          else *dst = pack16(v[k], T{});
        }
      }
    });
  }
  float top = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = t + k * THREADS;
    if (i < nvec) {
      float g[VEC], b[VEC];
      if constexpr (!kEarly) {
        gm[0].load(p.gamma, first(i));
        if (p.layer) bt[0].load(p.beta, first(i));
      }
      gm[kEarly ? k : 0].unpack(g);
      if (p.layer) {
        bt[kEarly ? k : 0].unpack(b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = __builtin_fmaf((v[k][e] - mean) * rstd, g[e], b[e]);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[k][e] = v[k][e] * rstd * g[e];
      }
      top = top_of<VEC>(top, v[k]);
    }
  }
  const float sc = scale_of(block_max_bits<WAVES>(__float_as_uint(top) & 0x7fffffffu, s_max));
  if (t == 0) p.scale[row] = sc;
  const float inv = 1.0f / sc;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = t + k * THREADS;
    if (i < nvec) store_quantised<VEC>(p.q + at + first(i), v[k], sc, inv, sc == sc);
  }
}

// Narrow rows: a group of 1 << lg lanes holds a row, a vector a lane; a wavefront has 64 >> lg rows side by side.
// (262,144 rows of 64 bf16 with a residual: 101.5 us with a wavefront for each, 26 so.)
constexpr int kNarrowWaves = 4;
template <typename T, typename PT>
__global__ void __launch_bounds__(kNarrowWaves * kWave) norm8_narrow_kernel(const Norm8Params p, int64_t rows, int lg) {
  constexpr int VEC = 16 / Elem<T>::kBytes;
  const int lane = lane_id(), i = lane & ((1 << lg) - 1);
  const int64_t row = ((static_cast<int64_t>(blockIdx.x) * kNarrowWaves + threadIdx.x / kWave) << (6 - lg)) + (lane >> lg);
  const int cols = static_cast<int>(p.cols);
  const int nfull = cols / VEC, rest = cols % VEC;
  const bool live = row < rows && i < nfull + (rest != 0);  // (lanes stay: the sums are taken across lanes)
  const int first = i < nfull ? i * VEC : cols - VEC;
  const int64_t at = row * cols + first;
  uint4 rx = make_uint4(0u, 0u, 0u, 0u), rr = rx;
  Params<PT, VEC> gm = {}, bt = {};
  if (live) {
    rx = load16_any(p.x + at * Elem<T>::kBytes);
    if (p.res) rr = load16_any(p.res + at * Elem<T>::kBytes);
    gm.load(p.gamma, first);
    if (p.layer) bt.load(p.beta, first);
  }
  float v[VEC];
  unpack16(rx, v, T{});
  if (p.res) {
    float r[VEC];
    unpack16(rr, r, T{});
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] += r[e];
  }
  const auto group_sum = [&](float s) {
    for (int m = 1; m < (1 << lg); m <<= 1) s += shfl_xor_f32(s, m);
    return s;
  };
  const int shared = !live ? VEC : (i == nfull ? VEC - rest : 0);  // elements that do not count
  const float n = static_cast<float>(cols);
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const float c = e >= shared ? v[e] : 0.f;
    s = p.layer ? s + c : __builtin_fmaf(c, c, s);
  }
  s = group_sum(s) / n;
  float mean = 0.f;
  if (p.layer) {
    mean = s;
    s = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float d = e >= shared ? v[e] - mean : 0.f;
      s += d * d;
    }
    s = group_sum(s) / n;
  }
  const float rstd = rstd_of(s, p.eps);
  if (live && p.res) {
    u32x4_any* const dst = reinterpret_cast<u32x4_any*>(p.res_out + at * Elem<T>::kBytes);
    if (p.stream_out) __builtin_nontemporal_store(pack16(v, T{}), dst);
    else *dst = pack16(v, T{});
  }
  float g[VEC], b[VEC];
  gm.unpack(g);
  bt.unpack(b);
#pragma unroll
  for (int e = 0; e < VEC; ++e)
    v[e] = p.layer ? __builtin_fmaf((v[e] - mean) * rstd, g[e], b[e]) : v[e] * rstd * g[e];
  uint32_t top = live ? __float_as_uint(top_of<VEC>(0.f, v)) & 0x7fffffffu : 0u;
  for (int m = 1; m < (1 << lg); m <<= 1) {
    const uint32_t o = static_cast<uint32_t>(shfl_i32(static_cast<int>(top), lane ^ m));
    top = o > top ? o : top;
  }
  const float sc = scale_of(top);
  if (live) {
    if (i == 0) p.scale[row] = sc;
    store_quantised<VEC>(p.q + at, v, sc, 1.0f / sc, sc == sc);
  }
}

// Rows of less than a vector or more than the registers hold: the row is read four times; residual_out is
// written last, each element by the thread that has read it.
template <typename T, typename PT>
__global__ void __launch_bounds__(kLoopThreads) norm8_loop_kernel(const Norm8Params p) {
  constexpr int kWaves = kLoopThreads / kWave;
  __shared__ float s_sum[kWaves];
  __shared__ uint32_t s_max[kWaves];
  const int64_t row = blockIdx.x, at = row * p.cols;
  const auto h = [&](int64_t c) {
    float v = Elem<T>::load(p.x + (at + c) * Elem<T>::kBytes);
    if (p.res) v += Elem<T>::load(p.res + (at + c) * Elem<T>::kBytes);
    return v;
  };
  const float n = static_cast<float>(p.cols);
  float mean = 0.f, s = 0.f;
  if (p.layer) {
    for (int64_t c = threadIdx.x; c < p.cols; c += kLoopThreads) s += h(c);
    mean = block_sum<kWaves>(s, s_sum) / n;
    s = 0.f;
  }
  for (int64_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float d = h(c) - mean;
    s += d * d;
  }
  const float rstd = rstd_of(block_sum<kWaves>(s, s_sum) / n, p.eps);
  const auto y = [&](int64_t c, float hc) {
    const float v = (hc - mean) * rstd * Elem<PT>::load(static_cast<const char*>(p.gamma) + c * Elem<PT>::kBytes);
    return p.layer ? v + Elem<PT>::load(static_cast<const char*>(p.beta) + c * Elem<PT>::kBytes) : v;
  };
  uint32_t top = 0u;
  for (int64_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const uint32_t a = __float_as_uint(y(c, h(c))) & 0x7fffffffu;
    top = a > top ? a : top;
  }
  const float sc = scale_of(block_max_bits<kWaves>(top, s_max));
  if (threadIdx.x == 0) p.scale[row] = sc;
  T* const ro = reinterpret_cast<T*>(p.res_out);
  for (int64_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float hc = h(c);
    p.q[at + c] = sc == sc ? static_cast<int8_t>(rintf(y(c, hc) / sc)) : static_cast<int8_t>(0);
    if (p.res) store_one(ro + at + c, hc, false);
  }
}

template <typename T, typename PT>
hipError_t launch_norm8_rows(const Norm8Params& p, int64_t rows, hipStream_t s) {
  constexpr int VEC = 16 / Elem<T>::kBytes;
  const Norm8Form form = norm8_form(rows, p.cols, VEC);
  const dim3 grid(static_cast<unsigned>(rows));
  const auto rows_form = [&](auto k, auto waves) {
    constexpr int K = decltype(k)::value, W = decltype(waves)::value;
    if (form.vectors == K && form.waves == W)
      hipLaunchKernelGGL((norm8_rows_kernel<T, PT, K, W>), grid, dim3(W * kWave), 0, s, p);
  };
  using std::integral_constant;
  constexpr integral_constant<int, 1> n1{};
  constexpr integral_constant<int, 2> n2{};
  constexpr integral_constant<int, 4> n4{};
  constexpr integral_constant<int, 8> n8{};
  constexpr integral_constant<int, 16> n16{};
  if (form.vectors == 0) {
    hipLaunchKernelGGL((norm8_loop_kernel<T, PT>), grid, dim3(kLoopThreads), 0, s, p);
  } else if (form.waves == 0) {
    int lg = 0;
    while ((VEC << lg) < p.cols) ++lg;
    const int64_t per = static_cast<int64_t>(kNarrowWaves) << (6 - lg);
    hipLaunchKernelGGL((norm8_narrow_kernel<T, PT>), dim3(static_cast<unsigned>((rows + per - 1) / per)),
                       dim3(kNarrowWaves * kWave), 0, s, p, rows, lg);
  } else {
    rows_form(n1, n1);
    rows_form(n1, n2);
    rows_form(n1, n4);
    rows_form(n1, n8);
    rows_form(n2, n4);
    rows_form(n2, n8);
    rows_form(n2, n16);
    rows_form(n4, n8);
    rows_form(n4, n16);
  }
  return hipGetLastError();
}

// A launch has fewer than 2^32 threads: at most so many rows of up to 1,024 threads in one.
constexpr int64_t kNorm8Rows = UINT32_MAX / 1024;
template <typename T, typename PT>
hipError_t launch_norm8(Norm8Params p, int64_t rows, hipStream_t s) {
  for (; rows > kNorm8Rows; rows -= kNorm8Rows) {
    const hipError_t e = launch_norm8_rows<T, PT>(p, kNorm8Rows, s);
    if (e != hipSuccess) return e;
    const int64_t bytes = kNorm8Rows * p.cols * Elem<T>::kBytes;
    p.x += bytes;
    if (p.res) {
      p.res += bytes;
      p.res_out += bytes;
    }
    p.q += kNorm8Rows * p.cols;
    p.scale += kNorm8Rows;
  }
  return launch_norm8_rows<T, PT>(p, rows, s);
}

template <typename T>
hipError_t launch_norm8_typed(int32_t pdt, const Norm8Params& p, int64_t rows, hipStream_t s) {
  switch (pdt) {
    case CTI_EBAG_F32: return launch_norm8<T, float>(p, rows, s);
    case CTI_EBAG_BF16: return launch_norm8<T, bf16_t>(p, rows, s);
    default: return launch_norm8<T, f16_t>(p, rows, s);
  }
}

bool float_dtype(int32_t dt) { return dt == CTI_EBAG_F32 || dt == CTI_EBAG_BF16 || dt == CTI_EBAG_F16; }

}  // namespace
}  // namespace cti

using namespace cti;

extern "C" int cti_ebag_norm_int8(int32_t kind, const void* x, const void* residual, void* residual_out, int64_t rows,
                                  int64_t cols, int32_t dtype, const void* gamma, const void* beta,
                                  int32_t param_dtype, float eps, int8_t* q, float* scale, void* stream) {
  clear_error();
  if (kind != CTI_EBAG_RMS_NORM && kind != CTI_EBAG_LAYER_NORM) return set_error(CTI_EBAG_EINVAL, "unknown norm %d", kind);
  if (rows < 0) return set_error(CTI_EBAG_EINVAL, "rows must be >= 0 (got %lld)", (long long)rows);
  if (cols < 1) return set_error(CTI_EBAG_EINVAL, "cols must be >= 1 (got %lld)", (long long)cols);
  if (!float_dtype(dtype)) return set_error(CTI_EBAG_EINVAL, "unknown dtype code %d", dtype);
  if (!float_dtype(param_dtype)) return set_error(CTI_EBAG_EINVAL, "unknown parameter dtype code %d", param_dtype);
  if (!(eps >= 0.f)) return set_error(CTI_EBAG_EINVAL, "eps must be >= 0");
  if ((residual != nullptr) != (residual_out != nullptr))
    return set_error(CTI_EBAG_EINVAL, "residual and residual_out must be given together (or neither)");
  if (rows == 0) return CTI_EBAG_OK;
  if (rows > INT32_MAX) return set_error(CTI_EBAG_EUNSUPPORTED, "more than 2^31 - 1 rows (%lld)", (long long)rows);
  if (!x || !q || !scale || !gamma) return set_error(CTI_EBAG_EINVAL, "NULL device pointer among x/gamma/q/scale");
  if (kind == CTI_EBAG_LAYER_NORM && !beta) return set_error(CTI_EBAG_EINVAL, "beta is NULL");
  if (residual) {
    // the output replaces an input element by element, or lies apart from both
    const uintptr_t bytes = static_cast<uintptr_t>(rows) * cols * dtype_bytes(dtype), o = reinterpret_cast<uintptr_t>(residual_out);
    for (const void* in : {x, residual}) {
      const uintptr_t i = reinterpret_cast<uintptr_t>(in);
      if (o != i && o < i + bytes && i < o + bytes)
        return set_error(CTI_EBAG_EINVAL, "residual_out overlaps x or residual without being it");
    }
  }
  Norm8Params p;
  p.x = static_cast<const char*>(x);
  p.res = static_cast<const char*>(residual);
  p.res_out = static_cast<char*>(residual_out);
  p.gamma = gamma;
  p.beta = beta;
  p.q = q;
  p.scale = scale;
  p.cols = cols;
  p.eps = eps;
  p.layer = kind == CTI_EBAG_LAYER_NORM;
  p.stream_out = rows * cols * dtype_bytes(dtype) >= kStreamOutBytes;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e;
  switch (dtype) {
    case CTI_EBAG_F32: e = launch_norm8_typed<float>(param_dtype, p, rows, s); break;
    case CTI_EBAG_BF16: e = launch_norm8_typed<bf16_t>(param_dtype, p, rows, s); break;
    default: e = launch_norm8_typed<f16_t>(param_dtype, p, rows, s); break;
  }
  if (e != hipSuccess) return set_error(CTI_EBAG_EHIP, "norm launch failed: %s", hipGetErrorString(e));
  return CTI_EBAG_OK;
}
