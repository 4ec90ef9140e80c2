// Launchers of the expert-product, MXFP4 and block-norm operators (grouped.cu,
// grouped_tc.cu, mxfp4.cu, block_norm.cu), called from ops_abi.cu.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

namespace moe {

enum GroupedKind { kGroupedFwd = 0, kGroupedDgrad = 1, kGroupedWgrad = 2 };

// One grouped product, as the kernels see it: D = A B^T for each expert,
//   forward  D [rows, n] : A = x [rows, k],     B = w[e] [n, k]
//   dgrad    D [rows, k] : A = dout [rows, n],  B = w[e]^T
//   wgrad    D [n, k]    : A = dout^T,          B = x^T, over the expert's rows
struct GroupedArgs {
  const void *x, *w, *dout;  // the operands that the kind reads
  void *out;
  const int32_t *seg_off;
  int E, R, n, k;
  int dtype, out_dtype;              // MOE_DT_F16 / BF16, and F32 for out
  int64_t ld_x, ld_w, es_w, ld_out;  // row strides of [rows, k], [n, k], [rows, n]; expert stride
  int sm_count;
  uint32_t *status;
};

cudaError_t launch_grouped_simple(GroupedKind kind, const GroupedArgs &a, cudaStream_t s);
// The tensor-core form, for 16-byte aligned operands (grouped_tc_ok).
bool grouped_tc_ok(GroupedKind kind, const GroupedArgs &a);
cudaError_t launch_grouped_tc(GroupedKind kind, const GroupedArgs &a, cudaStream_t s);

// ---- MXFP4 ---------------------------------------------------------------
struct Mxfp4Quant {
  const void *x;
  int dtype;           // MOE_DT_F32 / F16 / BF16
  int64_t ld_x;
  const int32_t *index;  // source row of each output row, or null
  int src_rows, rows, k;
  uint8_t *codes, *scales;
  int sm_count;
  uint32_t *status;
};
struct Mxfp4Dequant {
  const uint8_t *codes, *scales;
  int rows, k;
  void *out;
  int dtype;
  int64_t ld_out;
  int sm_count;
};
struct Mxfp4Args {
  const uint8_t *xc, *xs, *wc, *ws;
  void *out;
  const int32_t *seg_off;
  int E, R, n, k, out_dtype;
  int64_t ld_out;
  int sm_count;
  uint32_t *status;
};
constexpr int mxfp4_code_stride(int k) { return (k + 31) / 32 * 16; }
constexpr int mxfp4_scale_stride(int k) { return (k + 127) / 128 * 4; }

cudaError_t launch_mxfp4_quantize(const Mxfp4Quant &a, cudaStream_t s);
cudaError_t launch_mxfp4_dequantize(const Mxfp4Dequant &a, cudaStream_t s);
cudaError_t launch_mxfp4_mm(const Mxfp4Args &a, cudaStream_t s);

// ---- norms around a block --------------------------------------------------
struct BlockNormArgs {
  int rows, H, res_dtype, dtype;
  int64_t ld_res, ld_blk;
  int post;
  float scale, eps;
  const void *x, *y;             // forward: residual in; backward: residual out
  const float *w_pre, *w_post, *gate;
  void *x_out, *h;               // forward results
  const void *dx_out, *dh;       // backward inputs
  void *dx, *dy;
  float *dw_pre, *dw_post, *dgate, *partial;
  int sm_count;
  uint32_t *status;
};
cudaError_t launch_block_norm(const BlockNormArgs &a, cudaStream_t s);
cudaError_t launch_block_norm_backward(const BlockNormArgs &a, cudaStream_t s);
// CTAs of the backward pass, each with 2 H partial sums.
int block_norm_backward_ctas(int rows, int H, int sm_count);
constexpr int kMaxNormWidth = 16384;

}  // namespace moe
