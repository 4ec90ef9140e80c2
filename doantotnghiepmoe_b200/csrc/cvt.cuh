// Element types of the operators that take more than one: loads widen to
// fp32, stores round once, to nearest even.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace moe {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// Two values rounded into one word, the first in the low half.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&v);
}

// V = 8 or 1 elements of a row, as they lie in memory: what a thread holds of a
// row that is still on its way.
template <typename T, int V>
struct Piece {
  uint32_t w[V == 8 ? 2 * sizeof(T) : 1];

  // Elements c .. c + V - 1; zeros from n on (with V = 8, n is a multiple of 8
  // and the address 16-byte aligned).
  __device__ __forceinline__ void load(const T *p, int c, int n) {
    if constexpr (V == 8) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        *reinterpret_cast<uint4 *>(w + 4 * i) =
            c < n ? reinterpret_cast<const uint4 *>(p + c)[i] : make_uint4(0, 0, 0, 0);
    } else {
      *reinterpret_cast<T *>(w) = c < n ? p[c] : T(0.0f);
    }
  }
  // The same from shared memory (V = 8).
  __device__ __forceinline__ void load_shared(const uint8_t *p, int c, int n) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i)
      *reinterpret_cast<uint4 *>(w + 4 * i) =
          c < n ? reinterpret_cast<const uint4 *>(p + c * sizeof(T))[i] : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (uint32_t &u : w) u = 0;
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    } else {
      return to_f32(reinterpret_cast<const T *>(w)[i]);
    }
  }
};

// 8 consecutive elements, the pointer 16-byte aligned.
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{}),
                                               pack2(v[4], v[5], T{}), pack2(v[6], v[7], T{}));
  }
}

}  // namespace moe
