// Row access of the model operators (layer norm, distillation, attention): 16-byte chunks of a row that may start
// on any element, with the row's ragged end handled element by element, and reductions over a wave.
#pragma once

#include <type_traits>

#include "common.hpp"

namespace bgx {

// Elements per 16-byte chunk and the conversions of one chunk.
template <typename T>
struct Chunk;
template <>
struct Chunk<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};
template <>
struct Chunk<bf16_t> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(f32x2_to_bf16x2_bits(f[0], f[1]), f32x2_to_bf16x2_bits(f[2], f[3]),
                      f32x2_to_bf16x2_bits(f[4], f[5]), f32x2_to_bf16x2_bits(f[6], f[7]));
  }
};
template <>
struct Chunk<f16_t> {
  static constexpr int N = 8;
  // both at once (v_cvt_pk_f16_f32, to nearest even); converted one by one they would take three instructions
  __device__ static uint32_t pair(float lo, float hi) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
  }
  __device__ static void unpack(const uint4& v, float* f) {
    const f16x8 h = __builtin_bit_cast(f16x8, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)h[i];
  }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(pair(f[0], f[1]), pair(f[2], f[3]), pair(f[4], f[5]), pair(f[6], f[7]));
  }
};

// The element type of a 16-byte chunk decides how far its address may be from a 16-byte boundary: global memory
// takes vector accesses at any element, so rows of odd length need no path of their own.
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
typedef raw4 raw4_by2 __attribute__((aligned(2)));
typedef raw4 raw4_by4 __attribute__((aligned(4)));
template <typename T>
using raw4_any = typename std::conditional<sizeof(T) == 2, raw4_by2, raw4_by4>::type;

template <typename T>
__device__ inline uint4 load_chunk_any(const T* p) {
  typedef __attribute__((address_space(1))) const raw4_any<T>* global_ptr;
  const raw4 v = *(global_ptr)(uintptr_t)p;
  return make_uint4(v.x, v.y, v.z, v.w);
}
template <typename T>
__device__ inline void store_chunk_any(T* p, const uint4& v) {
  typedef __attribute__((address_space(1))) raw4_any<T>* global_ptr;
  *(global_ptr)(uintptr_t)p = raw4{v.x, v.y, v.z, v.w};
}

// The same, STREAM: past the caches.  For results of this many bytes or more: they do not fit the memory-side cache
// (256 MB) beside what they were made from, whoever reads them next reads memory anyway, and lines that linger there
// are written back under the next kernel's reads (measured on 4096 x 50304 bf16 logits: the forward pass after a
// backward pass 102 -> 80 us, the backward pass itself 157 us either way).
constexpr int64_t STREAM_BYTES = 128ll << 20;
template <bool STREAM, typename T>
__device__ inline void store_chunk(T* p, const uint4& v) {
  if constexpr (STREAM) {
    typedef __attribute__((address_space(1))) raw4_any<T>* global_ptr;
    __builtin_nontemporal_store((raw4_any<T>)raw4{v.x, v.y, v.z, v.w}, (global_ptr)(uintptr_t)p);
  } else {
    store_chunk_any(p, v);
  }
}

template <typename T>
__device__ inline uint32_t load_bits(const T* p) {
  if constexpr (sizeof(T) == 4)
    return *reinterpret_cast<const uint32_t*>(p);
  else
    return *reinterpret_cast<const uint16_t*>(p);
}
template <typename T>
__device__ inline void store_bits(T* p, uint32_t b) {
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<uint32_t*>(p) = b;
  else
    *reinterpret_cast<uint16_t*>(p) = (uint16_t)b;
}

// Elements col .. col + N - 1 of a row of `len` elements; what lies past the end reads as zero and is not touched.
template <typename T>
__device__ inline uint4 load_chunk_tail(const T* row, int64_t col, int64_t len) {
  constexpr int N = Chunk<T>::N;
  if (col + N <= len) return load_chunk_any(row + col);
  uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (col + e < len) {
      const uint32_t b = load_bits(row + col + e);
      if constexpr (sizeof(T) == 4)
        w[e] = b;
      else
        w[e >> 1] |= (e & 1) ? (b << 16) : b;
    }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ inline void store_chunk_tail(T* row, int64_t col, int64_t len, const uint4& v) {
  constexpr int N = Chunk<T>::N;
  if (col + N <= len) {
    store_chunk_any(row + col, v);
    return;
  }
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (col + e < len) {
      if constexpr (sizeof(T) == 4)
        store_bits(row + col + e, w[e]);
      else
        store_bits(row + col + e, (e & 1) ? (w[e >> 1] >> 16) : (w[e >> 1] & 0xffffu));
    }
}

// Sum / maximum over the 64 lanes of a wave; every lane gets the result, formed in the same order on every lane: within
// 16 lanes by lane permutations that the operand read applies, then across the 16s and the halves.
template <int CTRL>
__device__ inline float dpp_of(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <typename OP>
__device__ inline float wave_reduce(float v, OP op) {
  v = op(v, dpp_of<0xb1>(v));   // lane ^ 1
  v = op(v, dpp_of<0x4e>(v));   // lane ^ 2
  v = op(v, dpp_of<0x141>(v));  // mirrored within 8: the other four
  v = op(v, dpp_of<0x140>(v));  // mirrored within 16: the other eight
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ inline float wave_sum(float v) {
  return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ inline float wave_max(float v) {
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace bgx
