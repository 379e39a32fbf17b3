// Device helpers shared by the training operators: chunks of 8 columns of any type at any address, types
// chosen at run time, and the counter-based generator of dropout.
#pragma once

#include "ebag_device.h"
#include "ebag_internal.h"
#include "ebag_train_rules.h"

namespace cti {

// The first `live` (8 at most) of 8 elements at p, the rest +0.
template <typename T>
__device__ __forceinline__ void load8(const char* p, int live, float* v) {
  if (live >= 8) {
    if constexpr (Elem<T>::kBytes == 4) {
      unpack16(load16_any(p), v, T{});
      unpack16(load16_any(p + 16), v + 4, T{});
    } else {
      unpack16(load16_any(p), v, T{});
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < live ? Elem<T>::load(p + e * Elem<T>::kBytes) : 0.f;
  }
}

// 8 columns of a row from column c on, as loaded; what lies past the row's `cols` is +0. Rows of at least 8 columns are read
// by whole vectors, at any address: a chunk past the row's end as the last 8 columns, moved to their places when they are
// unpacked. (Read one by one, they would be waited for in a branch, and every other load with them.)
// WHOLE: the row's width is a multiple of 8 (columns from the row's end on are its last 8, for lanes that leave them out).
template <typename T, bool WHOLE = false>
struct Chunk {
  static constexpr int kVecs = Elem<T>::kBytes / 2;
  uint4 raw[kVecs];
  __device__ __forceinline__ void load(const char* row, int c, int cols) {
    if (WHOLE || cols >= 8) {
      const char* const p = row + static_cast<int64_t>(c + 8 <= cols ? c : cols - 8) * Elem<T>::kBytes;
#pragma unroll
      for (int i = 0; i < kVecs; ++i) raw[i] = load16_any(p + i * 16);
    } else {
      uint32_t w[4 * kVecs] = {};
#pragma unroll
      for (int e = 0; e < 7; ++e) {
        if (c + e < cols) {
          const char* const p = row + (c + e) * Elem<T>::kBytes;
          if constexpr (Elem<T>::kBytes == 4) w[e] = *reinterpret_cast<const uint32_t*>(p);
          else w[e / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p)) << (16 * (e % 2));
        }
      }
#pragma unroll
      for (int i = 0; i < kVecs; ++i) raw[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
  __device__ __forceinline__ void unpack(float* v, int c, int cols) const {
    constexpr int VEC = 16 / Elem<T>::kBytes, N = 4 * kVecs;
    if (WHOLE || c + 8 <= cols || cols < 8) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) unpack16(raw[i], v + i * VEC, T{});
      return;
    }
    const int by = c + 8 - cols < 8 ? c + 8 - cols : 8;  // columns to move by
    uint32_t w[N];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) w[4 * i] = raw[i].x, w[4 * i + 1] = raw[i].y, w[4 * i + 2] = raw[i].z, w[4 * i + 3] = raw[i].w;
#pragma unroll
    for (int step = 8; step * Elem<T>::kBytes >= 4; step /= 2) {
      const int words = step * Elem<T>::kBytes / 4;
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = by & step ? (i + words < N ? w[i + words] : 0u) : w[i];
    }
    if constexpr (Elem<T>::kBytes == 2) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = by & 1 ? (w[i] >> 16) | (i + 1 < N ? w[i + 1] << 16 : 0u) : w[i];
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) unpack16(make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]), v + i * VEC, T{});
  }
  // What was unpacked before is forgotten, and unpacked again when it is needed: else the compiler keeps both forms.
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) asm("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z), "+v"(raw[i].w));
  }
};

// One vector of 16 bytes, as loaded, of which the first `live` elements are there.
template <typename T, int VEC>
__device__ __forceinline__ uint4 load_raw(const char* p, int live) {
  if (live >= VEC) return load16_any(p);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (e < live) {
      if constexpr (Elem<T>::kBytes == 4) w[e] = *reinterpret_cast<const uint32_t*>(p + e * 4);
      else w[e / 2] |= static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(p + e * 2)) << (16 * (e % 2));
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T>
struct Packed;
template <>
struct Packed<float> {
  __device__ static __forceinline__ uint32_t pair(float a, float) { return __float_as_uint(a); }
};
template <>
struct Packed<bf16_t> {
  __device__ static __forceinline__ uint32_t pair(float a, float b) { return pack_bf16x2(a, b); }
};
template <>
struct Packed<f16_t> {
  __device__ static __forceinline__ uint32_t pair(float a, float b) { return pack_f16x2(a, b); }
};

template <bool STREAM, typename V, typename A>
__device__ __forceinline__ void put_any(char* p, V v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<A*>(p));
  else *reinterpret_cast<A*>(p) = v;
}

// The first `live` of N values (N is 4 or 8), rounded to T, at any address.
template <typename T, int N, bool STREAM = false>
__device__ __forceinline__ void store_vec(char* p, int live, const float* v) {
  constexpr int kWords = N * Elem<T>::kBytes / 4;
  if (live >= N) {
    uint32_t w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      if constexpr (Elem<T>::kBytes == 4) w[i] = Packed<T>::pair(v[i], 0.f);
      else w[i] = Packed<T>::pair(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (kWords == 2) {
      put_any<STREAM, u32x2, u32x2_any>(p, u32x2{w[0], w[1]});
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) put_any<STREAM, u32x4, u32x4_any>(p + i * 4, u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]});
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < live) store_one(reinterpret_cast<T*>(p) + e, v[e], false);
  }
}
template <typename T, bool STREAM = false>
__device__ __forceinline__ void store8(char* p, int live, const float* v) {
  store_vec<T, 8, STREAM>(p, live, v);
}

// f(T{}) for the element type of a code that has been checked.
template <typename F>
inline void with_type(int32_t dtype, F&& f) {
  switch (dtype) {
    case CTI_EBAG_F32: f(float{}); break;
    case CTI_EBAG_BF16: f(bf16_t{}); break;
    default: f(f16_t{}); break;
  }
}
// 8 parameters of a type known at run time, from column c on.
__device__ __forceinline__ void load_params8(const void* p, int32_t dtype, int c, int cols, float* v) {
  const auto load = [&](auto t) {
    Chunk<decltype(t)> x;
    x.load(static_cast<const char*>(p), c, cols);
    x.unpack(v, c, cols);
  };
  if (dtype == CTI_EBAG_F32) load(float{});
  else if (dtype == CTI_EBAG_BF16) load(bf16_t{});
  else load(f16_t{});
}

template <typename F>
inline void with_types(int32_t a, int32_t b, F&& f) {
  with_type(a, [&](auto t) { with_type(b, [&](auto o) { f(t, o); }); });
}

inline bool float_dtype(int32_t dt) { return dt == CTI_EBAG_F32 || dt == CTI_EBAG_BF16 || dt == CTI_EBAG_F16; }

// ---------------------------------------------------------------------------------------------
// Dropout's mask. Philox4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as
// 1, 2, 3, 2011): four words for each counter (row, chunk of 8 columns, offset) and key (seed), 16 bits of
// them for each column. A column is dropped where its 16 bits are below `threshold` = round(65536 p), and
// kept ones are multiplied by 65536 / (65536 - threshold): the mean is exact for the p that is drawn. 16 bits
// rather than 32 halve the generator's multiplications, which would bound 16-bit types, not memory.
// ---------------------------------------------------------------------------------------------
struct Dropout {
  uint64_t seed;
  uint64_t offset;
  const int64_t* state;  // NULL, or two numbers on the device that are added to seed and offset
  uint32_t threshold;    // 0: nothing is dropped; 65536: everything
  float factor;
};

// Seed and offset with the state's, once a thread.
__device__ __forceinline__ void load_state(Dropout& d) {
  if (d.state) {
    d.seed += static_cast<uint64_t>(d.state[0]);
    d.offset += static_cast<uint64_t>(d.state[1]);
  }
}

__device__ __forceinline__ void apply_dropout(const Dropout& d, uint32_t row, uint32_t chunk, float* v) {
  uint32_t c0 = row, c1 = chunk, c2 = static_cast<uint32_t>(d.offset), c3 = static_cast<uint32_t>(d.offset >> 32);
  uint32_t k0 = static_cast<uint32_t>(d.seed), k1 = static_cast<uint32_t>(d.seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xd2511f53u, b = static_cast<uint64_t>(c2) * 0xcd9e8d57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9e3779b9u;
    k1 += 0xbb67ae85u;
  }
  const uint32_t w[4] = {c0, c1, c2, c3};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    // selected, not multiplied by 0: what is dropped is +0, NaN and infinities too
    v[2 * j] = (w[j] & 0xffffu) >= d.threshold ? v[2 * j] * d.factor : 0.f;
    v[2 * j + 1] = (w[j] >> 16) >= d.threshold ? v[2 * j + 1] * d.factor : 0.f;
  }
}

// The threshold and factor of a probability in [0, 1]; false for others (NaN among them).
inline bool set_dropout(Dropout* d, double p, uint64_t seed, uint64_t offset, const int64_t* state) {
  if (!(p >= 0.0 && p <= 1.0)) return false;
  d->threshold = static_cast<uint32_t>(p * 65536.0 + 0.5);
  d->factor = d->threshold < 65536u ? static_cast<float>(65536.0 / (65536.0 - d->threshold)) : 0.f;
  d->seed = seed;
  d->offset = offset;
  d->state = state;
  return true;
}

}  // namespace cti
