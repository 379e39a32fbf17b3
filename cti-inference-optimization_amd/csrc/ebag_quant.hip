// Row quantisation of an embedding table to int8 for MI355X (gfx950), as the reference's
// quantize_embedding_int8 (online_best/infer.py:895-901) evaluates on the device:
//   m = max_j |w[r, j]|                 (fp32; exact in any order)
//   s = max(m * RN32(1/127), 1e-8)      (torch divides a device tensor by a Python scalar as a
//                                        multiply by the scalar's fp32 reciprocal; then
//                                        torch.clamp(scale, min=1e-8))
//   q[r, j] = clamp(rint(w[r, j] / s), -128, 127)   (IEEE fp32 division, round half to even)
// Results are bit-identical to that expression for finite tables. In a table, NaN is left out of m (and becomes q = 0);
// rows of activations may not lose it (nan_rows): one with NaN or infinity in it gets the scale NaN and q = 0.
//
// A streaming pass: each element is read once and written once as a byte. Bound by HBM (2M rows of
// 128 bf16: 512 MB read, 264 MB written), so a lane group reads its row as 16-byte vectors, keeps
// it in registers between the maximum and the quantisation, and a wavefront has several rows in
// flight (quantize_rows_kernel). One wavefront per row with 2-byte loads, the row read twice and an
// IEEE division per element took 638 us on that table; this form takes 147 (5.3 TB/s).
#include <stdint.h>

#include "ebag_device.h"
#include "ebag_internal.h"

namespace cti {
namespace {

constexpr int kQuantThreads = 256;
constexpr int kQuantRowsPerBlock = kQuantThreads / kWave;  // wavefronts per workgroup
// Row sets a wavefront of the chunk form has in flight: 4 loads per lane.
constexpr int rows_in_flight(int chunks_per_lane) { return 4 / chunks_per_lane; }

// The largest of m and every |v|, NaN if any is. (v_maximum3_f32: two elements an instruction.)
template <int N>
__device__ __forceinline__ float max_abs(float m, const float* v) {
  if constexpr (N == 1) return __builtin_elementwise_maximum(m, __builtin_fabsf(v[0]));
#pragma unroll
  for (int e = 0; e + 1 < N; e += 2)
    m = __builtin_elementwise_maximum(__builtin_elementwise_maximum(__builtin_fabsf(v[e]), __builtin_fabsf(v[e + 1])), m);
  return m;
}
// The largest of m and of the |v| that are not NaN: taken again where a table's row has NaN.
template <int N>
__device__ __forceinline__ float max_abs_numbers(float m, const float* v) {
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, __builtin_fabsf(v[e]));
  return m;
}
// The bits of such a maximum: ordered as the values are, NaN above infinity, so that maxima over lanes keep it.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t max_bits(float m) { return __float_as_uint(m) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t bits, bool nan_rows) {
  const float s = __uint_as_float(bits) * (1.0f / 127.0f);
  if (nan_rows && bits >= kInfBits) return __uint_as_float(0x7fc00000u);
  return s < 1e-8f ? 1e-8f : s;
}

// Any width and alignment: one wavefront per row, the row read twice.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_loop_kernel(const char* w, int64_t rows, int64_t dim,
                                                                       int64_t row_stride, bool nan_rows, int8_t* q,
                                                                       float* scale) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kQuantRowsPerBlock + threadIdx.x / kWave;
  if (row >= rows) return;  // uniform over the wavefront
  const int lane = lane_id();
  const char* wr = w + row * row_stride * Elem<T>::kBytes;
  float m = 0.f;
  for (int64_t c = lane; c < dim; c += kWave) {
    const float v = Elem<T>::load(wr + c * Elem<T>::kBytes);
    m = max_abs<1>(m, &v);
  }
  uint32_t top = block_max_bits<1>(max_bits(m), nullptr);
  if (top > kInfBits && !nan_rows) {  // the same in every lane
    m = 0.f;
    for (int64_t c = lane; c < dim; c += kWave) {
      const float v = Elem<T>::load(wr + c * Elem<T>::kBytes);
      m = max_abs_numbers<1>(m, &v);
    }
    top = block_max_bits<1>(max_bits(m), nullptr);
  }
  const float s = row_scale(top, nan_rows);
  if (lane == 0) scale[row] = s;
  int8_t* qr = q + row * dim;
  for (int64_t c = lane; c < dim; c += kWave) {
    float v = rintf(Elem<T>::load(wr + c * Elem<T>::kBytes) / s);
    v = v < -128.f ? -128.f : (v > 127.f ? 127.f : v);
    qr[c] = static_cast<int8_t>(v);
  }
}

// ---------------------------------------------------------------------------------------------
// Rows as chunks of C elements (one load of C * sizeof(T) bytes): a group of 1 << lg lanes holds a
// row, lane l chunks l, l + (1 << lg), ... (K of them); a wavefront quantises 64 >> lg rows side by
// side and kRows such sets at a time, all loads issued before the first is used.
// ---------------------------------------------------------------------------------------------
// C elements of T as loaded (C * sizeof(T) = 2, 4, 8 or 16 bytes).
template <int BYTES>
struct Chunk;
template <>
struct Chunk<2> { typedef uint16_t type; };
template <>
struct Chunk<4> { typedef uint32_t type; };
template <>
struct Chunk<8> { typedef u32x2 type; };
template <>
struct Chunk<16> { typedef u32x4 type; };

template <typename T, int C>
__device__ __forceinline__ void unpack_chunk(const typename Chunk<C * Elem<T>::kBytes>::type& raw, float* v) {
  constexpr int BYTES = C * Elem<T>::kBytes;
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  if constexpr (BYTES <= 4) w.x = raw;
  else if constexpr (BYTES == 8) w = make_uint4(raw.x, raw.y, 0u, 0u);
  else w = make_uint4(raw.x, raw.y, raw.z, raw.w);
  float t[16 / Elem<T>::kBytes];
  unpack16(w, t, T{});
#pragma unroll
  for (int e = 0; e < C; ++e) v[e] = t[e];
}

// Maximum over each aligned group of 1 << lg lanes, in every lane of the group: lane moves inside 16 lanes on the VALU
// (DPP), across them through LDS.
__device__ __forceinline__ uint32_t group_max(uint32_t m, int lg) {
  const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
  const auto dpp = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  const auto other = [](uint32_t x, int by) { return static_cast<uint32_t>(shfl_i32(static_cast<int>(x), lane_id() ^ by)); };
  if (lg > 0) m = larger(m, dpp(m, std::integral_constant<int, 0xb1>{}));   // quad_perm: lane ^ 1
  if (lg > 1) m = larger(m, dpp(m, std::integral_constant<int, 0x4e>{}));   // quad_perm: lane ^ 2
  if (lg > 2) m = larger(m, dpp(m, std::integral_constant<int, 0x141>{}));  // row_half_mirror
  if (lg > 3) m = larger(m, dpp(m, std::integral_constant<int, 0x140>{}));  // row_mirror
  if (lg > 4) m = larger(m, other(m, 16));
  if (lg > 5) m = larger(m, other(m, 32));
  return m;
}

template <typename T, int C, int K>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const char* w, int64_t rows, int32_t chunks,
                                                                       int64_t row_bytes, int lg, bool nan_rows, int8_t* q,
                                                                       float* scale) {
  using V = typename Chunk<C * Elem<T>::kBytes>::type;
  constexpr int kRows = rows_in_flight(K);
  const int lane = lane_id();
  const int g = lane >> lg, sl = lane & ((1 << lg) - 1);
  const int R = kWave >> lg;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * kQuantRowsPerBlock + threadIdx.x / kWave;
  const int64_t r0 = wave * (R * kRows) + g;
  V raw[kRows][K];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int64_t row = r0 + u * R;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k << lg) + sl;
      raw[u][k] = V{};
      if (row < rows && c < chunks) raw[u][k] = __builtin_nontemporal_load(reinterpret_cast<const V*>(w + row * row_bytes) + c);
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int64_t row = r0 + u * R;
    float v[K][C];
    float m = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      unpack_chunk<T, C>(raw[u][k], v[k]);
      m = max_abs<C>(m, v[k]);
    }
    uint32_t top = group_max(max_bits(m), lg);
    if (__builtin_expect(__ballot(top > kInfBits) != 0 && !nan_rows, 0)) {  // (a whole wavefront: lanes read each other)
      m = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) m = max_abs_numbers<C>(m, v[k]);
      top = group_max(max_bits(m), lg);
    }
    const float s = row_scale(top, nan_rows);
    const float inv = 1.0f / s;
    if (row < rows && sl == 0) scale[row] = s;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k << lg) + sl;
      uint32_t b[C];
      quantize_chunk<C>(v[k], s, inv, b);
      if (row < rows && c < chunks) {
        int8_t* const dst = q + (row * chunks + c) * C;
        if constexpr (C == 1) {
          *dst = static_cast<int8_t>(b[0]);
        } else if constexpr (C == 2) {
          *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(b[0] | (b[1] << 8));
        } else {
          uint32_t word[C / 4];
#pragma unroll
          for (int i = 0; i < C / 4; ++i)
            word[i] = b[4 * i] | (b[4 * i + 1] << 8) | (b[4 * i + 2] << 16) | (b[4 * i + 3] << 24);
          if constexpr (C == 4) __builtin_nontemporal_store(word[0], reinterpret_cast<uint32_t*>(dst));
          else __builtin_nontemporal_store(u32x2{word[0], word[1]}, reinterpret_cast<u32x2*>(dst));
        }
      }
    }
  }
}

// Chunks of C elements when the rows, the base pointers and the width allow loads of that size,
// and the row is at most 4 chunks per lane of a wavefront (single elements: 2; 200,000 rows of 129 /
// 191 / 255 bf16 took 62 / 68 / 82 us at 4, the loop kernel 59 / 64 / 79); false: not this form.
template <typename T, int C>
bool launch_chunks(const char* w, int64_t rows, int64_t dim, int64_t row_stride, bool nan_rows, int8_t* q, float* scale,
                   hipStream_t s) {
  constexpr int BYTES = C * Elem<T>::kBytes;
  if (dim % C != 0 || (row_stride * Elem<T>::kBytes) % BYTES != 0 || reinterpret_cast<uintptr_t>(w) % BYTES != 0 ||
      reinterpret_cast<uintptr_t>(q) % C != 0 || dim / C > (C == 1 ? 2 : 4) * kWave)
    return false;
  const int32_t chunks = static_cast<int32_t>(dim / C);
  const int K = chunks <= kWave ? 1 : (chunks <= 2 * kWave ? 2 : 4);
  int lg = 0;
  while ((K << lg) < chunks) ++lg;
  const int64_t per_block = static_cast<int64_t>(kQuantRowsPerBlock) * (kWave >> lg) * rows_in_flight(K);
  const dim3 grid(static_cast<unsigned>((rows + per_block - 1) / per_block)), block(kQuantThreads);
  const int64_t rb = row_stride * Elem<T>::kBytes;
  if (K == 1) hipLaunchKernelGGL((quantize_rows_kernel<T, C, 1>), grid, block, 0, s, w, rows, chunks, rb, lg, nan_rows, q, scale);
  if (K == 2) hipLaunchKernelGGL((quantize_rows_kernel<T, C, 2>), grid, block, 0, s, w, rows, chunks, rb, lg, nan_rows, q, scale);
  if constexpr (C > 1) {
    if (K == 4) hipLaunchKernelGGL((quantize_rows_kernel<T, C, 4>), grid, block, 0, s, w, rows, chunks, rb, lg, nan_rows, q, scale);
  }
  return true;
}

// Rows wider than a wavefront holds: a workgroup of WAVES wavefronts holds its row in registers, thread t vectors t,
// t + THREADS, ... (K of them), at any alignment; the last vector ends with the row and overlaps the one before it where
// the row is no whole number of them (the bytes both store are the same). 2,048 rows of 5,632 bf16: 57.7 us in the
// loop kernel (one wavefront a row, 2-byte loads, the row read twice), 10.2 in this; one row of 4,096: 18.6 and 5.0.
// Up to 128 vectors take two wavefronts (200,000 rows of 257 fp32: 94 us in the loop kernel, 102 by four wavefronts of
// which three are idle, 67 by two; of 1,021 bf16 410, 182 and 134).
template <typename T, int K, int WAVES>
__global__ void __launch_bounds__(WAVES * kWave) quantize_wide_kernel(const char* w, int32_t dim, int64_t row_bytes,
                                                                      bool nan_rows, int8_t* q, float* scale) {
  constexpr int VEC = 16 / Elem<T>::kBytes, THREADS = WAVES * kWave;
  __shared__ uint32_t s_max[WAVES];
  const int64_t row = blockIdx.x;
  const char* const wr = w + row * row_bytes;
  const int t = static_cast<int>(threadIdx.x), whole = dim / VEC, vecs = whole + (dim % VEC != 0);
  const auto first = [&](int i) { return i < whole ? i * VEC : dim - VEC; };  // vector i's first column
  uint4 raw[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = t + k * THREADS;
    raw[k] = make_uint4(0u, 0u, 0u, 0u);
    if (i < vecs) raw[k] = load16_any(wr + static_cast<int64_t>(first(i)) * Elem<T>::kBytes);
  }
  float v[K][VEC];
  float m = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    unpack16(raw[k], v[k], T{});
    m = max_abs<VEC>(m, v[k]);
  }
  uint32_t top = block_max_bits<WAVES>(max_bits(m), s_max);
  if (__builtin_expect(top > kInfBits && !nan_rows, 0)) {  // the same in every thread
    m = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) m = max_abs_numbers<VEC>(m, v[k]);
    __syncthreads();  // every wavefront has read the first maximum
    top = block_max_bits<WAVES>(max_bits(m), s_max);
  }
  const float s = row_scale(top, nan_rows);
  const float inv = 1.0f / s;
  if (t == 0) scale[row] = s;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int i = t + k * THREADS;
    if (i < vecs) {
      uint32_t b[VEC];
      quantize_chunk<VEC>(v[k], s, inv, b);
      store_bytes<VEC>(q + row * dim + first(i), b);
    }
  }
}

template <typename T>
bool launch_wide(const char* w, int64_t rows, int64_t dim, int64_t row_stride, bool nan_rows, int8_t* q, float* scale,
                 hipStream_t s) {
  constexpr int VEC = 16 / Elem<T>::kBytes;
  const int64_t vecs = (dim + VEC - 1) / VEC;
  if (vecs <= kWave || vecs > 64 * kWave) return false;
  const int64_t rb = row_stride * Elem<T>::kBytes;
  const auto go = [&](auto k, auto waves) {
    constexpr int W = decltype(waves)::value;
    constexpr int64_t kRows = UINT32_MAX / (W * kWave);  // a launch has fewer than 2^32 threads
    for (int64_t r = 0; r < rows; r += kRows) {
      const dim3 grid(static_cast<unsigned>(rows - r < kRows ? rows - r : kRows));
      hipLaunchKernelGGL((quantize_wide_kernel<T, decltype(k)::value, W>), grid, dim3(W * kWave), 0, s, w + r * rb,
                         static_cast<int32_t>(dim), rb, nan_rows, q + r * dim, scale + r);
    }
  };
  constexpr std::integral_constant<int, 1> n1{};
  constexpr std::integral_constant<int, 2> n2{};
  constexpr std::integral_constant<int, 4> n4{};
  constexpr std::integral_constant<int, 16> n16{};
  if (vecs <= 2 * kWave) go(n1, n2);
  else if (vecs <= 4 * kWave) go(n1, n4);
  else if (vecs <= 8 * kWave) go(n2, n4);
  else if (vecs <= 16 * kWave) go(n4, n4);
  else if (vecs <= 32 * kWave) go(n2, n16);
  else go(n4, n16);
  return true;
}

// The widest chunks that fit; wider rows than they cover take the wide kernel, what that does not cover either the
// loop kernel.
template <typename T>
void launch_quantize(const char* w, int64_t rows, int64_t dim, int64_t row_stride, bool nan_rows, int8_t* q, float* scale,
                     hipStream_t s) {
  constexpr int kMax = 16 / Elem<T>::kBytes;
  if (launch_chunks<T, kMax>(w, rows, dim, row_stride, nan_rows, q, scale, s)) return;
  if (launch_chunks<T, kMax / 2>(w, rows, dim, row_stride, nan_rows, q, scale, s)) return;
  if (launch_chunks<T, kMax / 4>(w, rows, dim, row_stride, nan_rows, q, scale, s)) return;
  if constexpr (kMax == 8) {
    if (launch_chunks<T, 1>(w, rows, dim, row_stride, nan_rows, q, scale, s)) return;
  }
  if (launch_wide<T>(w, rows, dim, row_stride, nan_rows, q, scale, s)) return;
  const dim3 grid(static_cast<unsigned>((rows + kQuantRowsPerBlock - 1) / kQuantRowsPerBlock)), block(kQuantThreads);
  hipLaunchKernelGGL((quantize_rows_loop_kernel<T>), grid, block, 0, s, w, rows, dim, row_stride, nan_rows, q, scale);
}

// ---------------------------------------------------------------------------------------------
// The way back: out[r, j] = q[r, j] * scale[r] in fp32, rounded once to the output type.
// Both arrays are contiguous, so a chunk is as many consecutive elements as 16 bytes of output hold, wherever rows
// begin and end in them, and a wavefront's chunks are side by side (with 64 bytes a lane in four stores, 8,192 x 8,192
// to fp32 took 202 us). Bound by HBM (one byte read and 2 or 4 written an element).
// ---------------------------------------------------------------------------------------------
constexpr int kDequantChunks = 4;  // per thread

template <typename T, typename I>
__global__ void __launch_bounds__(kQuantThreads) dequantize_rows_kernel(const int8_t* q, const float* scale, I total,
                                                                        I dim, char* out, int32_t stream_out) {
  constexpr int C = 16 / Elem<T>::kBytes;
  using V = std::conditional_t<C == 4, u32_any, u32x2_any>;
  const I first = static_cast<I>(blockIdx.x) * (kQuantThreads * kDequantChunks) + threadIdx.x;
  V raw[kDequantChunks];
#pragma unroll
  for (int u = 0; u < kDequantChunks; ++u) {
    const I e0 = (first + u * kQuantThreads) * C;
    raw[u] = V{};
    if (e0 + C <= total) raw[u] = *reinterpret_cast<const V*>(q + e0);
  }
#pragma unroll
  for (int u = 0; u < kDequantChunks; ++u) {
    const I e0 = (first + u * kQuantThreads) * C;
    if (e0 >= total) return;
    I row = e0 / dim;
    I left = dim - (e0 - row * dim);  // elements of this row from e0 on
    T* const dst = reinterpret_cast<T*>(out) + e0;
    if (e0 + C > total) {
      for (I e = 0; e < total - e0; ++e, --left) {
        if (left == 0) {
          ++row;
          left = dim;
        }
        store_one(dst + e, as_f32(static_cast<float>(q[e0 + e]) * scale[row]), false);
      }
      return;
    }
    float s = scale[row], v[C];
#pragma unroll
    for (int e = 0; e < C; ++e) {
      uint32_t w;
      if constexpr (C == 4) w = raw[u];
      else w = raw[u][e / 4];
      v[e] = static_cast<float>(static_cast<int8_t>(w >> (8 * (e % 4))));
    }
    if (left >= C) {
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] = as_f32(v[e] * s);
    } else {
#pragma unroll
      for (int e = 0; e < C; ++e, --left) {
        if (left == 0) {
          s = scale[++row];
          left = dim;
        }
        v[e] = as_f32(v[e] * s);
      }
    }
    with_stream(stream_out, [&](auto stream) { store_out<C>(dst, v, decltype(stream)::value); });
  }
}

template <typename T>
void launch_dequantize(const int8_t* q, const float* scale, int64_t total, int64_t dim, char* out, hipStream_t s) {
  constexpr int64_t kPer = int64_t{kQuantThreads} * kDequantChunks * (16 / Elem<T>::kBytes);
  const dim3 grid(static_cast<unsigned>((total + kPer - 1) / kPer)), block(kQuantThreads);
  const int32_t stream_out = total * Elem<T>::kBytes >= kStreamOutBytes;
  if (total + kPer <= UINT32_MAX)
    hipLaunchKernelGGL((dequantize_rows_kernel<T, uint32_t>), grid, block, 0, s, q, scale, static_cast<uint32_t>(total),
                       static_cast<uint32_t>(dim), out, stream_out);
  else
    hipLaunchKernelGGL((dequantize_rows_kernel<T, uint64_t>), grid, block, 0, s, q, scale, static_cast<uint64_t>(total),
                       static_cast<uint64_t>(dim), out, stream_out);
}

}  // namespace
}  // namespace cti

using namespace cti;

extern "C" int cti_ebag_dequantize_int8(const int8_t* q, const float* scale, int64_t rows, int64_t dim, void* out,
                                        int32_t out_dtype, void* stream) {
  clear_error();
  if (out_dtype != CTI_EBAG_F32 && out_dtype != CTI_EBAG_BF16 && out_dtype != CTI_EBAG_F16)
    return set_error(CTI_EBAG_EINVAL, "unknown dtype code %d", out_dtype);
  if (rows < 0) return set_error(CTI_EBAG_EINVAL, "rows must be >= 0 (got %lld)", (long long)rows);
  if (dim < 1) return set_error(CTI_EBAG_EINVAL, "dim must be >= 1 (got %lld)", (long long)dim);
  if (rows == 0) return CTI_EBAG_OK;
  if (!q || !scale || !out) return set_error(CTI_EBAG_EINVAL, "NULL device pointer among q/scale/out");
  // a launch has fewer than 2^32 threads
  const int64_t most = UINT32_MAX / kQuantThreads * (int64_t{kQuantThreads} * kDequantChunks * 16 / dtype_bytes(out_dtype));
  if (rows > most / dim)
    return set_error(CTI_EBAG_EUNSUPPORTED, "more than %lld elements (%lld x %lld)", (long long)most, (long long)rows, (long long)dim);
  if (reinterpret_cast<uintptr_t>(out) % dtype_bytes(out_dtype) != 0)
    return set_error(CTI_EBAG_EINVAL, "out is not aligned to its elements");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* const o = static_cast<char*>(out);
  switch (out_dtype) {
    case CTI_EBAG_F32: launch_dequantize<float>(q, scale, rows * dim, dim, o, s); break;
    case CTI_EBAG_BF16: launch_dequantize<bf16_t>(q, scale, rows * dim, dim, o, s); break;
    default: launch_dequantize<f16_t>(q, scale, rows * dim, dim, o, s); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(CTI_EBAG_EHIP, "dequantize launch failed: %s", hipGetErrorString(e));
  return CTI_EBAG_OK;
}

static int quantize(const void* weight, int32_t dtype, int64_t rows, int64_t dim, int64_t row_stride, bool nan_rows,
                    int8_t* q, float* scale, void* stream) {
  clear_error();
  if (dtype != CTI_EBAG_F32 && dtype != CTI_EBAG_BF16 && dtype != CTI_EBAG_F16)
    return set_error(CTI_EBAG_EINVAL, "unknown dtype code %d", dtype);
  if (rows < 0) return set_error(CTI_EBAG_EINVAL, "rows must be >= 0 (got %lld)", (long long)rows);
  if (dim < 1) return set_error(CTI_EBAG_EINVAL, "dim must be >= 1 (got %lld)", (long long)dim);
  if (row_stride < dim) return set_error(CTI_EBAG_EINVAL, "row_stride %lld < dim %lld", (long long)row_stride, (long long)dim);
  if (rows == 0) return CTI_EBAG_OK;
  if (!weight || !q || !scale) return set_error(CTI_EBAG_EINVAL, "NULL device pointer among weight/q/scale");
  const int64_t blocks = (rows + kQuantRowsPerBlock - 1) / kQuantRowsPerBlock;
  if (blocks > INT32_MAX) return set_error(CTI_EBAG_EUNSUPPORTED, "too many rows (%lld)", (long long)rows);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const char* w = static_cast<const char*>(weight);
  switch (dtype) {
    case CTI_EBAG_F32: launch_quantize<float>(w, rows, dim, row_stride, nan_rows, q, scale, s); break;
    case CTI_EBAG_BF16: launch_quantize<bf16_t>(w, rows, dim, row_stride, nan_rows, q, scale, s); break;
    default: launch_quantize<f16_t>(w, rows, dim, row_stride, nan_rows, q, scale, s); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error(CTI_EBAG_EHIP, "quantize launch failed: %s", hipGetErrorString(e));
  return CTI_EBAG_OK;
}

extern "C" int cti_ebag_quantize_int8(const void* weight, int32_t dtype, int64_t rows, int64_t dim,
                                      int64_t row_stride, int8_t* q, float* scale, void* stream) {
  return quantize(weight, dtype, rows, dim, row_stride, false, q, scale, stream);
}

extern "C" int cti_ebag_quantize_activations_int8(const void* x, int32_t dtype, int64_t rows, int64_t dim,
                                                  int64_t row_stride, int8_t* q, float* scale, void* stream) {
  return quantize(x, dtype, rows, dim, row_stride, true, q, scale, stream);
}
