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
// Both directions move each byte once and are bound by HBM, with the issue slots
// close behind, so 16-bit values stay packed: the maximum of a block is taken
// on pairs of magnitudes, and codes become bf16 by byte lookups (prmt) and one
// packed multiplication by the scale.  A warp quantises 512 values of a row at a
// time, two such spans in flight: a lane has half a block (8 values a lane took 93
// instructions for them), so that its maximum is one shuffle, and stores 16
// codes.  It dequantises 256 at a time, four in flight: 8 codes a lane, whose
// bf16 values are one 16-byte store.  Rows go to warps, or their parts to several
// (a power of two) where rows are few.  196608 x 2048 bf16 values on B200: 158 us to
// quantise (6.4 TB/s), 182 us back (5.6 TB/s).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/moe_b200.h"
#include "common.cuh"
#include "cvt.cuh"
#include "ops.h"

namespace moe {
namespace {

constexpr int kQThreads = 256;
// Values of a warp's step, and steps whose loads are issued together.
constexpr int kQuantSpan = 512, kQuantFlight = 2, kSpan = 256, kFlight = 4;

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

__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {  // of 16-bit halves
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Sixteen values of a row, half a block, as they lie in memory.
template <typename T>
struct Half {
  uint32_t w[4 * sizeof(T)];

  template <bool VEC>
  __device__ __forceinline__ void load(const T *row, int c, int k) {
    if (VEC && c + 16 <= k) {
      const uint4 *p = reinterpret_cast<const uint4 *>(row + c);
#pragma unroll
      for (int i = 0; i < (int)sizeof(T); ++i) *reinterpret_cast<uint4 *>(w + 4 * i) = __ldg(p + i);
    } else {
      T *e = reinterpret_cast<T *>(w);
#pragma unroll
      for (int i = 0; i < 16; ++i) e[i] = c + i < k ? row[c + i] : T(0.0f);
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
      return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    else return to_f32(reinterpret_cast<const T *>(w)[i]);
  }
  // The exponent field of the largest magnitude of the two lanes' 32 values in
  // fp32 (any NaN counts above infinity, as an integer): on pairs of 16-bit
  // magnitudes where the values are that.
  __device__ __forceinline__ uint32_t top_exponent() const {
    if constexpr (sizeof(T) == 2) {
      uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 8; ++i) m = max2(m, w[i] & 0x7fff7fffu);
      m = max2(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m & 0xffffu, m >> 16);
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        return m >> 7;
      } else {
        return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))) >> 23;
      }
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) m = max(m, w[i] & 0x7fffffffu);
      return max(m, __shfl_xor_sync(0xffffffffu, m, 1)) >> 23;
    }
  }
};

// A warp's rows and spans: parts = 1 << shift warps share a row.
struct SpanWalk {
  int lane, part, parts;
  long long row, step;
  __device__ __forceinline__ explicit SpanWalk(int shift) {
    const long long w = (long long)blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5);
    lane = threadIdx.x & 31;
    parts = 1 << shift;
    part = (int)(w & (parts - 1));
    row = w >> shift;
    step = ((long long)gridDim.x * (kQThreads / 32)) >> shift;
    if (row >= step) row = LLONG_MAX / 2;  // a part of a row's warps only: no work
  }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQThreads) mxfp4_quantize_kernel(Mxfp4Quant a, int shift) {
  const SpanWalk sw(shift);
  const int spans = (a.k + kQuantSpan - 1) / kQuantSpan, nb = (a.k + 31) / 32;
  const int ldc = mxfp4_code_stride(a.k), lds = mxfp4_scale_stride(a.k);
  for (long long r = sw.row; r < a.rows; r += sw.step) {
    long long src = r;
    if (a.index) {
      src = a.index[r];
      if (src < 0 || src >= a.src_rows) {
        if (sw.lane == 0) set_status(a.status, kStatusBadRoute);
        src = -1;
      }
    }
    const T *row = reinterpret_cast<const T *>(a.x) + src * a.ld_x;
    uint8_t *codes = a.codes + r * ldc, *scales = a.scales + r * lds;
    for (int s0 = sw.part; s0 < spans; s0 += kQuantFlight * sw.parts) {
      Half<T> x[kQuantFlight];
#pragma unroll
      for (int f = 0; f < kQuantFlight; ++f)
        x[f].template load<VEC>(row, (s0 + f * sw.parts) * kQuantSpan + sw.lane * 16,
                                src < 0 ? 0 : a.k);
#pragma unroll
      for (int f = 0; f < kQuantFlight; ++f) {
        const int c = (s0 + f * sw.parts) * kQuantSpan + sw.lane * 16, blk = c / 32;
        if (s0 + f * sw.parts >= spans) break;  // warp-uniform
        const uint32_t ex = x[f].top_exponent();  // floor(log2 max) + 127, 0 if subnormal
        const uint32_t sb = max(ex, 2u) - 2u;
        const float inv = __uint_as_float((254u - sb) << 23);  // 2^(127 - sb), a normal number
        float v[2][8];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i / 8][i % 8] = x[f].value(i) * inv;
        const bool bad = ex == 255u;
        const uint2 q = bad ? make_uint2(0u, 0u) : make_uint2(e2m1x8(v[0]), e2m1x8(v[1]));
        if (blk < nb) *reinterpret_cast<uint2 *>(codes + c / 2) = q;
        if ((sw.lane & 1) == 0 && blk < lds)
          scales[blk] = (uint8_t)(blk >= nb ? 0u : bad ? 255u : sb);
      }
    }
  }
}

// __byte_perm with all four bits of each selector.
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t s) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(s));
  return r;
}

// The bf16 of the eight codes in q, codes 2i and 2i + 1 in word i.  The high and
// low bytes of 0 0.5 1 1.5 2 3 4 6 are looked up by the codes' low three bits;
// with the fourth bit set a lookup repeats the byte's top bit instead, which
// makes 0xff of 0x80 and so the sign.
__device__ __forceinline__ void e2m1x8_bf16(uint32_t q, uint32_t (&w)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t t = q >> (16 * h), sel = t & 0x7777u;
    const uint32_t sg = prmt(0x80808080u, 0x80808080u, t);
    const uint32_t hi = __byte_perm(0x3f3f3f00u, 0x40404040u, sel) | (sg << 7 & 0x80808080u);
    const uint32_t lo = __byte_perm(0xc0800000u, 0xc0804000u, sel);
    w[2 * h] = __byte_perm(lo, hi, 0x5140);
    w[2 * h + 1] = __byte_perm(lo, hi, 0x7362);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kQThreads) mxfp4_dequantize_kernel(Mxfp4Dequant a, int shift) {
  const SpanWalk sw(shift);
  const int spans = (a.k + kSpan - 1) / kSpan;
  const int ldc = mxfp4_code_stride(a.k), lds = mxfp4_scale_stride(a.k);
  for (long long r = sw.row; r < a.rows; r += sw.step) {
    const uint8_t *codes = a.codes + r * ldc, *scales = a.scales + r * lds;
    T *row = reinterpret_cast<T *>(a.out) + r * a.ld_out;
    for (int s0 = sw.part; s0 < spans; s0 += kFlight * sw.parts) {
      uint32_t q[kFlight], sb[kFlight];
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int c = (s0 + f * sw.parts) * kSpan + sw.lane * 8;
        q[f] = c < a.k ? __ldg(reinterpret_cast<const uint32_t *>(codes + c / 2)) : 0u;
        sb[f] = c < a.k ? __ldg(scales + c / 32) : 0u;
      }
#pragma unroll
      for (int f = 0; f < kFlight; ++f) {
        const int c = (s0 + f * sw.parts) * kSpan + sw.lane * 8;
        if (c >= a.k) break;
        uint32_t w[4];
        e2m1x8_bf16(q[f], w);
        // 2^(sb - 127) as a bf16: exponent bits, the subnormal 2^-127, or NaN
        const uint32_t sc = sb[f] == 255u ? 0x7fffu : sb[f] ? sb[f] << 7 : 0x40u;
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
          const uint32_t s2 = sc | sc << 16;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 p = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&w[i]),
                                             *reinterpret_cast<const __nv_bfloat162 *>(&s2));
            w[i] = *reinterpret_cast<const uint32_t *>(&p);
          }
          if (VEC && c + 8 <= a.k) {
            *reinterpret_cast<uint4 *>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
            for (int i = 0; i < 8 && c + i < a.k; ++i)
              row[c + i] = reinterpret_cast<const __nv_bfloat16 *>(w)[i];
          }
        } else {
          const float s = __uint_as_float(sc << 16);
          float v[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16) * s;
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * s;
          }
          if (VEC && c + 8 <= a.k) {
            store8(row + c, v);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c + i < a.k) row[c + i] = from_f32<T>(v[i]);
          }
        }
      }
    }
  }
}

// Warps of a row, as a shift: 1, or a power of two up to its spans while the
// rows alone would leave the GPU's warps idle; and the grid.
int row_split(int rows, int k, int span, int sm_count, int *grid) {
  const long long warps = (long long)sm_count * 8 * (kQThreads / 32);
  const int spans = (k + span - 1) / span;
  int shift = 0;
  while ((2 << shift) <= spans && ((long long)rows << (shift + 1)) <= warps) ++shift;
  const long long blocks = (((long long)rows << shift) + kQThreads / 32 - 1) / (kQThreads / 32);
  *grid = (int)std::min<long long>(blocks, (long long)sm_count * 8);
  return shift;
}

template <typename T>
cudaError_t quantize_t(const Mxfp4Quant &a, cudaStream_t s) {
  const bool vec = ((uintptr_t)a.x & 15) == 0 && (a.ld_x * sizeof(T)) % 16 == 0;
  int grid;
  const int shift = row_split(a.rows, a.k, kQuantSpan, a.sm_count, &grid);
  if (vec) mxfp4_quantize_kernel<T, true><<<grid, kQThreads, 0, s>>>(a, shift);
  else mxfp4_quantize_kernel<T, false><<<grid, kQThreads, 0, s>>>(a, shift);
  return cudaGetLastError();
}

template <typename T>
cudaError_t dequantize_t(const Mxfp4Dequant &a, cudaStream_t s) {
  const bool vec = ((uintptr_t)a.out & 15) == 0 && (a.ld_out * sizeof(T)) % 16 == 0;
  int grid;
  const int shift = row_split(a.rows, a.k, kSpan, a.sm_count, &grid);
  if (vec) mxfp4_dequantize_kernel<T, true><<<grid, kQThreads, 0, s>>>(a, shift);
  else mxfp4_dequantize_kernel<T, false><<<grid, kQThreads, 0, s>>>(a, shift);
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
