// MXFP4: blocks of 32 consecutive values of a row share one power-of-two
// scale, and each value is a 4-bit E2M1 number (sign, 0 0.5 1 1.5 2 3 4 6).
//
//   s = 2^(floor(log2 max|x|) - 2), at least 2^-127, stored as the byte
//       log2(s) + 127 (E8M0; 255 stands for NaN)
//   q = x / s rounded to the nearest E2M1 value, ties to the even code, held
//       at 6 past it (max|x| / s lies in [4, 8))
//
// x / s is exact (a power of two), so the codes are a function of the values
// alone.  A block with an infinity or a NaN gets the scale byte 255 and zero
// codes: it decodes to NaN.  Layout: codes [rows][16 ceil(k / 32)], element
// 2i of a row in the low nibble; scales [rows][4 ceil(k / 128)], the bytes
// behind the last block zero; values behind k are zeros.
//
// Both directions move each byte once and are bound by HBM.  A warp takes
// 256 values of a row (8 a lane, one 16-byte load of 16-bit values): a block
// is 4 lanes, its maximum two shuffles, and a lane stores its 8 codes as one
// word, so a warp's store is 128 contiguous bytes.
#include <algorithm>

#include "../../include/moe_b200.h"
#include "common.cuh"
#include "cvt.cuh"
#include "ops.h"

namespace moe {
namespace {

constexpr int kQThreads = 256, kSpan = 256;  // values of a warp's unit

// Codes of eight values already divided by the scale, value i in nibble i.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// The value of E2M1 code c, exactly.
__device__ __forceinline__ float e2m1_value(uint32_t c) {
  const uint32_t m = c & 7u;
  // m = 1 is 0.5; from 2 on, exponent m >> 1 and one fraction bit, as in fp32
  const float v = m < 2u ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
  return (c & 8u) ? -v : v;
}

__device__ __forceinline__ float e8m0_value(uint32_t b) {
  if (b == 255u) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(b ? b << 23 : 1u << 22);
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_span(const T *row, int c, int k, float (&v)[8]) {
  if (VEC && c + 8 <= k) {
    load8(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < k ? to_f32(row[c + i]) : 0.0f;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQThreads) mxfp4_quantize_kernel(Mxfp4Quant a) {
  const int lane = threadIdx.x & 31;
  const int spans = (a.k + kSpan - 1) / kSpan, nb = (a.k + 31) / 32;
  const int ldc = mxfp4_code_stride(a.k), lds = mxfp4_scale_stride(a.k);
  const long long units = (long long)a.rows * spans;
  const long long step = (long long)gridDim.x * (kQThreads / 32);
  for (long long u = (long long)blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5); u < units;
       u += step) {
    const int r = (int)(u / spans), c = (int)(u % spans) * kSpan + lane * 8, blk = c / 32;
    int src = r;
    if (a.index) {
      src = a.index[r];
      if (src < 0 || src >= a.src_rows) {
        if (lane == 0) set_status(a.status, kStatusBadRoute);
        src = -1;
      }
    }
    float v[8] = {};
    if (src >= 0) load_span<T, VEC>(reinterpret_cast<const T *>(a.x) + src * a.ld_x, c, a.k, v);
    // as integers, |NaN| > infinity > every finite |v|
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t ex = m >> 23;  // floor(log2 max) + 127 (0 for subnormal numbers)
    const uint32_t sb = ex == 255u ? 255u : (ex > 2u ? ex - 2u : 0u);
    const float inv = __uint_as_float((254u - min(sb, 252u)) << 23);  // 2^(127 - sb), normal
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = ex == 255u ? 0.0f : v[i] * inv;
    const uint32_t q = e2m1x8(v);
    if (blk < nb) *reinterpret_cast<uint32_t *>(a.codes + (int64_t)r * ldc + c / 2) = q;
    if ((lane & 3) == 0 && blk < lds) a.scales[(int64_t)r * lds + blk] = blk < nb ? sb : 0;
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQThreads) mxfp4_dequantize_kernel(Mxfp4Dequant a) {
  const int lane = threadIdx.x & 31;
  const int spans = (a.k + kSpan - 1) / kSpan;
  const int ldc = mxfp4_code_stride(a.k), lds = mxfp4_scale_stride(a.k);
  const long long units = (long long)a.rows * spans;
  const long long step = (long long)gridDim.x * (kQThreads / 32);
  for (long long u = (long long)blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5); u < units;
       u += step) {
    const int64_t r = u / spans;
    const int c = (int)(u % spans) * kSpan + lane * 8;
    if (c >= a.k) continue;
    const uint32_t q = *reinterpret_cast<const uint32_t *>(a.codes + r * ldc + c / 2);
    const float s = e8m0_value(a.scales[r * lds + c / 32]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = e2m1_value(q >> (4 * i) & 15u) * s;
    T *o = reinterpret_cast<T *>(a.out) + r * a.ld_out + c;
    if (VEC && c + 8 <= a.k) {
      store8(o, v);
    } else {
      for (int i = 0; i < 8 && c + i < a.k; ++i) o[i] = from_f32<T>(v[i]);
    }
  }
}

int span_grid(int rows, int k, int sm_count) {
  const long long units = (long long)rows * ((k + kSpan - 1) / kSpan);
  return (int)std::min<long long>((units + kQThreads / 32 - 1) / (kQThreads / 32),
                                  (long long)sm_count * 8);
}

template <typename T>
cudaError_t quantize_t(const Mxfp4Quant &a, cudaStream_t s) {
  const bool vec = ((uintptr_t)a.x & 15) == 0 && (a.ld_x * sizeof(T)) % 16 == 0;
  const int grid = span_grid(a.rows, a.k, a.sm_count);
  if (vec) mxfp4_quantize_kernel<T, true><<<grid, kQThreads, 0, s>>>(a);
  else mxfp4_quantize_kernel<T, false><<<grid, kQThreads, 0, s>>>(a);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_t(const Mxfp4Dequant &a, cudaStream_t s) {
  const bool vec = ((uintptr_t)a.out & 15) == 0 && (a.ld_out * sizeof(T)) % 16 == 0;
  const int grid = span_grid(a.rows, a.k, a.sm_count);
  if (vec) mxfp4_dequantize_kernel<T, true><<<grid, kQThreads, 0, s>>>(a);
  else mxfp4_dequantize_kernel<T, false><<<grid, kQThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mxfp4_quantize(const Mxfp4Quant &a, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  if (a.dtype == MOE_DT_F32) return quantize_t<float>(a, s);
  return a.dtype == MOE_DT_BF16 ? quantize_t<__nv_bfloat16>(a, s) : quantize_t<__half>(a, s);
}

cudaError_t launch_mxfp4_dequantize(const Mxfp4Dequant &a, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  if (a.dtype == MOE_DT_F32) return dequantize_t<float>(a, s);
  return a.dtype == MOE_DT_BF16 ? dequantize_t<__nv_bfloat16>(a, s) : dequantize_t<__half>(a, s);
}

}  // namespace moe
