// Matrix products grouped by expert, on the SIMT pipes: the form for operands
// that the tensor-core kernel's copies cannot take (a base address or a row
// stride that is not a multiple of 16 bytes).
//
// D(i, j) = sum_l A(i, l) B(j, l), every product and sum in fp32.  A 64 x 64
// tile of D per CTA of 256 threads, 4 x 4 sums a thread, 16 steps of l staged
// in shared memory as fp32; any strides.  Bound by the FMA pipe and its
// shared-memory reads (two 16-byte reads for 16 multiply-adds): 7.7 ms for 32768
// rows, n = 1536, k = 2048 (27 TFLOP/s) where the tensor cores take 0.21 ms.
#include <algorithm>

#include "../../include/moe_b200.h"
#include "cvt.cuh"
#include "ops.h"
#include "segments.cuh"

namespace moe {
namespace {

constexpr int kT = 64, kL = 16, kSimpleThreads = 256;

template <typename T>
struct StridedRows {
  const T *p;
  int64_t si, sl;
  __device__ __forceinline__ float operator()(int i, int l) const {
    return to_f32(p[i * si + l * sl]);
  }
};

// One tile: D rows [i0, i0 + 64) of ni, columns [j0, j0 + 64) of nj.
template <typename LA, typename LB, typename Store>
__device__ __forceinline__ void simple_tile(float (&sa)[kL][kT + 4], float (&sb)[kL][kT + 4],
                                            LA la, LB lb, int i0, int ni, int j0, int nj, int nl,
                                            Store store) {
  const int t = threadIdx.x, ti = t / 16 * 4, tj = t % 16 * 4;
  float acc[4][4] = {};
  for (int l0 = 0; l0 < nl; l0 += kL) {
#pragma unroll
    for (int u = 0; u < kT * kL / kSimpleThreads; ++u) {
      const int q = t + u * kSimpleThreads, i = q / kL, l = q % kL;
      sa[l][i] = (i0 + i < ni && l0 + l < nl) ? la(i0 + i, l0 + l) : 0.0f;
      sb[l][i] = (j0 + i < nj && l0 + l < nl) ? lb(j0 + i, l0 + l) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int l = 0; l < kL; ++l) {
      const float4 a = *reinterpret_cast<const float4 *>(&sa[l][ti]);
      const float4 b = *reinterpret_cast<const float4 *>(&sb[l][tj]);
      const float av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int x = 0; x < 4; ++x)
#pragma unroll
        for (int y = 0; y < 4; ++y) acc[x][y] = fmaf(av[x], bv[y], acc[x][y]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int y = 0; y < 4; ++y)
      if (i0 + ti + x < ni && j0 + tj + y < nj) store(i0 + ti + x, j0 + tj + y, acc[x][y]);
}

__device__ __forceinline__ void store_as(void *out, int dtype, int64_t at, float v) {
  if (dtype == MOE_DT_F32) reinterpret_cast<float *>(out)[at] = v;
  else if (dtype == MOE_DT_BF16) reinterpret_cast<__nv_bfloat16 *>(out)[at] = from_f32<__nv_bfloat16>(v);
  else reinterpret_cast<__half *>(out)[at] = from_f32<__half>(v);
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kSimpleThreads) grouped_simple_kernel(GroupedArgs a) {
  __shared__ SegTable seg;
  __shared__ __align__(16) float sa[kL][kT + 4], sb[kL][kT + 4];
  if (threadIdx.x < 32) build_segments(seg, a.seg_off, a.E, a.R, kT, kT, a.status);
  __syncthreads();
  const T *x = reinterpret_cast<const T *>(a.x), *w = reinterpret_cast<const T *>(a.w),
          *d = reinterpret_cast<const T *>(a.dout);
  const int nj = KIND == kGroupedFwd ? a.n : a.k, tj = (nj + kT - 1) / kT;
  const int ti_w = (a.n + kT - 1) / kT;
  const long long total = KIND == kGroupedWgrad ? (long long)a.E * ti_w * tj
                                                : (long long)seg.total * tj;
  for (long long it = blockIdx.x; it < total; it += gridDim.x) {
    const int j0 = (int)(it % tj) * kT, g = (int)(it / tj);
    if (KIND == kGroupedWgrad) {
      const int e = g / ti_w, i0 = g % ti_w * kT;
      const int64_t r0 = seg.off[e];
      simple_tile(sa, sb, StridedRows<T>{d + r0 * a.ld_out, 1, a.ld_out},
                  StridedRows<T>{x + r0 * a.ld_x, 1, a.ld_x}, i0, a.n, j0, a.k, seg.rows(e),
                  [&](int i, int j, float v) {
                    store_as(a.out, a.out_dtype, e * a.es_w + i * a.ld_w + j, v);
                  });
    } else {
      const int e = seg.expert_of(g, a.E);  // tiles of kT rows
      const int i0 = (g - seg.tile0[e]) * kT;
      const int64_t r0 = seg.off[e];
      if (KIND == kGroupedFwd)
        simple_tile(sa, sb, StridedRows<T>{x + r0 * a.ld_x, a.ld_x, 1},
                    StridedRows<T>{w + e * a.es_w, a.ld_w, 1}, i0, seg.rows(e), j0, a.n, a.k,
                    [&](int i, int j, float v) {
                      store_as(a.out, a.out_dtype, (r0 + i) * a.ld_out + j, v);
                    });
      else
        simple_tile(sa, sb, StridedRows<T>{d + r0 * a.ld_out, a.ld_out, 1},
                    StridedRows<T>{w + e * a.es_w, 1, a.ld_w}, i0, seg.rows(e), j0, a.k, a.n,
                    [&](int i, int j, float v) {
                      store_as(a.out, a.out_dtype, (r0 + i) * a.ld_x + j, v);
                    });
    }
    __syncthreads();
  }
}

template <typename T>
cudaError_t launch_t(GroupedKind kind, const GroupedArgs &a, cudaStream_t s) {
  const long long nj = ((kind == kGroupedFwd ? a.n : a.k) + kT - 1) / kT;
  const long long ni =
      kind == kGroupedWgrad ? (long long)a.E * ((a.n + kT - 1) / kT) : a.R / kT + std::min(a.E, a.R);
  const int grid = (int)std::min<long long>(ni * nj, (long long)a.sm_count * 4);
  if (kind == kGroupedFwd) grouped_simple_kernel<T, kGroupedFwd><<<grid, kSimpleThreads, 0, s>>>(a);
  else if (kind == kGroupedDgrad)
    grouped_simple_kernel<T, kGroupedDgrad><<<grid, kSimpleThreads, 0, s>>>(a);
  else grouped_simple_kernel<T, kGroupedWgrad><<<grid, kSimpleThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_grouped_simple(GroupedKind kind, const GroupedArgs &a, cudaStream_t s) {
  return a.dtype == MOE_DT_BF16 ? launch_t<__nv_bfloat16>(kind, a, s) : launch_t<__half>(kind, a, s);
}

}  // namespace moe
