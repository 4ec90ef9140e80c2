// C ABI of the expert-product, MXFP4 and block-norm operators: argument
// checks and launches.  A refused call launches nothing and leaves its reason
// in moe_last_error().  No operator keeps device memory of its own, so calls
// on different streams and captured graphs do not share any state but the
// handle's status word.
#include "handle.h"
#include "ops.h"

using namespace moe;
using namespace moe::host;

namespace {

constexpr int kMaxWidth = 1 << 20;
constexpr int kMaxRows = INT32_MAX - 4096;  // a tile behind the last row has a number
constexpr int64_t kMaxStride = (int64_t)1 << 36;  // elements: byte strides fit a tensor map

template <typename... A>
moe_status refuse(moe_handle *h, const char *fmt, A... args) {
  set_err(h->err, fmt, args...);
  return MOE_ERR_INVALID;
}

size_t type_size(int dt) { return dt == MOE_DT_F32 ? 4 : 2; }
bool half_type(int dt) { return dt == MOE_DT_F16 || dt == MOE_DT_BF16; }
bool float_type(int dt) { return half_type(dt) || dt == MOE_DT_F32; }
// The stride of a tensor with at most one row addresses nothing, so it neither
// keeps a call from 16-byte accesses nor reaches a tensor map.
int64_t row_stride(int rows, int64_t ld, int width) {
  return rows > 1 ? ld : ((int64_t)width + 7) / 8 * 8;
}
bool misaligned(const void *p, size_t to) { return ((uintptr_t)p & (to - 1)) != 0; }

template <typename F>
moe_status launch(moe_handle *h, const char *name, void *stream, int launches, F &&f) {
  DeviceGuard g(h->device);
  cudaStream_t s = pick(h, stream);
  cudaEvent_t p0 = h->prof.begin(s);
  const cudaError_t e = f(s);
  h->prof.end(name, p0, s);
  if (e != cudaSuccess) return cuda_fail(h, e, name);
  h->last_launches = launches;
  return MOE_OK;
}

moe_status check_grouped(moe_handle *h, const moe_grouped_desc *d, GroupedArgs &a) {
  if (d->num_experts < 1 || d->num_experts > kMaxExperts)
    return refuse(h, "expert count %d outside [1, %d]", d->num_experts, kMaxExperts);
  if (d->rows < 0 || d->rows > kMaxRows)
    return refuse(h, "row count %d outside [0, %d]", d->rows, kMaxRows);
  if (d->n < 1 || d->n > kMaxWidth || d->k < 1 || d->k > kMaxWidth)
    return refuse(h, "widths n = %d, k = %d outside [1, %d]", d->n, d->k, kMaxWidth);
  if (!half_type(d->dtype)) return refuse(h, "operand type %d is neither F16 nor BF16", d->dtype);
  if (d->out_dtype != d->dtype && d->out_dtype != MOE_DT_F32)
    return refuse(h, "result type %d is neither the operands' type nor F32", d->out_dtype);
  a.ld_x = row_stride(d->rows, d->ld_x, d->k);
  a.ld_w = row_stride(d->n, d->ld_w, d->k);
  a.ld_out = row_stride(d->rows, d->ld_out, d->n);
  if (a.ld_x < d->k || a.ld_w < d->k || a.ld_out < d->n)
    return refuse(h, "a row stride is smaller than its row (k = %d, n = %d)", d->k, d->n);
  if (a.ld_x > kMaxStride || a.ld_w > kMaxStride || a.ld_out > kMaxStride ||
      d->expert_stride > kMaxStride)
    return refuse(h, "a stride is above %lld elements", (long long)kMaxStride);
  if (d->num_experts > 1 && d->expert_stride < (d->n - 1) * a.ld_w + d->k)
    return refuse(h, "expert stride %lld is smaller than one expert", (long long)d->expert_stride);
  a.E = d->num_experts;
  a.R = d->rows;
  a.n = d->n;
  a.k = d->k;
  a.dtype = d->dtype;
  a.out_dtype = d->out_dtype;
  a.es_w = d->num_experts > 1 ? d->expert_stride : d->n * a.ld_w;
  a.sm_count = h->sm_count;
  a.status = h->status;
  return MOE_OK;
}

moe_status run_grouped(moe_handle *h, GroupedKind kind, const char *name, GroupedArgs &a,
                       const int32_t *d_seg_off, void *stream) {
  const size_t sz = type_size(a.dtype);
  if (misaligned(a.x, sz) || misaligned(a.w, sz) || misaligned(a.dout, sz) ||
      misaligned(a.out, type_size(a.out_dtype)) || misaligned(d_seg_off, 4))
    return refuse(h, "a pointer is not aligned to its elements");
  a.seg_off = d_seg_off;
  if (a.R == 0 && kind != kGroupedWgrad) {
    h->last_launches = 0;
    return MOE_OK;
  }
  return launch(h, name, stream, 1,
                [&](cudaStream_t s) {
                  return grouped_tc_ok(kind, a) ? launch_grouped_tc(kind, a, s)
                                                : launch_grouped_simple(kind, a, s);
                });
}

}  // namespace

extern "C" void *moe_get_stream(moe_handle *h) {
  if (!h) return nullptr;
  std::lock_guard<std::mutex> lock(h->mu);
  return h->stream;
}

extern "C" moe_status moe_grouped_mm(moe_handle *h, const moe_grouped_desc *d, const void *d_x,
                                     const void *d_w, const int32_t *d_seg_off, void *d_out,
                                     void *stream) {
  if (!h || !d || !d_w || !d_seg_off || (d->rows > 0 && (!d_x || !d_out))) return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  GroupedArgs a{};
  const moe_status st = check_grouped(h, d, a);
  if (st != MOE_OK) return st;
  a.x = d_x;
  a.w = d_w;
  a.out = d_out;
  return run_grouped(h, kGroupedFwd, "grouped_mm", a, d_seg_off, stream);
}

extern "C" moe_status moe_grouped_mm_dgrad(moe_handle *h, const moe_grouped_desc *d,
                                           const void *d_dout, const void *d_w,
                                           const int32_t *d_seg_off, void *d_dx, void *stream) {
  if (!h || !d || !d_w || !d_seg_off || (d->rows > 0 && (!d_dout || !d_dx)))
    return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  GroupedArgs a{};
  const moe_status st = check_grouped(h, d, a);
  if (st != MOE_OK) return st;
  a.dout = d_dout;
  a.w = d_w;
  a.out = d_dx;
  return run_grouped(h, kGroupedDgrad, "grouped_mm_dgrad", a, d_seg_off, stream);
}

extern "C" moe_status moe_grouped_mm_wgrad(moe_handle *h, const moe_grouped_desc *d,
                                           const void *d_dout, const void *d_x,
                                           const int32_t *d_seg_off, void *d_dw, void *stream) {
  if (!h || !d || !d_dw || !d_seg_off || (d->rows > 0 && (!d_dout || !d_x)))
    return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  GroupedArgs a{};
  const moe_status st = check_grouped(h, d, a);
  if (st != MOE_OK) return st;
  a.dout = d_dout;
  a.x = d_x;
  a.out = d_dw;
  return run_grouped(h, kGroupedWgrad, "grouped_mm_wgrad", a, d_seg_off, stream);
}

// ---------------------------------------------------------------------------
// MXFP4
// ---------------------------------------------------------------------------
extern "C" size_t moe_mxfp4_code_stride(int k) { return k > 0 ? (size_t)mxfp4_code_stride(k) : 0; }
extern "C" size_t moe_mxfp4_scale_stride(int k) {
  return k > 0 ? (size_t)mxfp4_scale_stride(k) : 0;
}

extern "C" moe_status moe_mxfp4_quantize(moe_handle *h, const void *d_x, int dtype, int64_t ld_x,
                                         int src_rows, const int32_t *d_index, int rows, int k,
                                         uint8_t *d_codes, uint8_t *d_scales, void *stream) {
  if (!h || (rows > 0 && (!d_codes || !d_scales || (src_rows > 0 && !d_x))))
    return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  if (!float_type(dtype)) return refuse(h, "type %d is none of F32, F16 and BF16", dtype);
  ld_x = row_stride(src_rows, ld_x, k);
  if (rows < 0 || src_rows < 0 || k < 1 || k > kMaxWidth || ld_x < k || ld_x > kMaxStride)
    return refuse(h, "rows %d of %d, width %d, row stride %lld", rows, src_rows, k,
                  (long long)ld_x);
  if (!d_index && rows > src_rows)
    return refuse(h, "%d rows of %d without an index", rows, src_rows);
  if (misaligned(d_x, type_size(dtype)) || misaligned(d_index, 4) || misaligned(d_codes, 16) ||
      misaligned(d_scales, 4))
    return refuse(h, "a pointer is not aligned (codes to 16 bytes, scales to 4)");
  Mxfp4Quant a{d_x, dtype, ld_x, d_index, src_rows, rows, k, d_codes, d_scales, h->sm_count,
               h->status};
  h->last_launches = 0;
  if (rows == 0) return MOE_OK;
  return launch(h, "mxfp4_quantize", stream, 1,
                [&](cudaStream_t s) { return launch_mxfp4_quantize(a, s); });
}

extern "C" moe_status moe_mxfp4_dequantize(moe_handle *h, const uint8_t *d_codes,
                                           const uint8_t *d_scales, int rows, int k, void *d_out,
                                           int dtype, int64_t ld_out, void *stream) {
  if (!h || (rows > 0 && (!d_codes || !d_scales || !d_out))) return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  if (!float_type(dtype)) return refuse(h, "type %d is none of F32, F16 and BF16", dtype);
  ld_out = row_stride(rows, ld_out, k);
  if (rows < 0 || k < 1 || k > kMaxWidth || ld_out < k || ld_out > kMaxStride)
    return refuse(h, "rows %d, width %d, row stride %lld", rows, k, (long long)ld_out);
  if (misaligned(d_out, type_size(dtype)) || misaligned(d_codes, 16) || misaligned(d_scales, 4))
    return refuse(h, "a pointer is not aligned (codes to 16 bytes, scales to 4)");
  Mxfp4Dequant a{d_codes, d_scales, rows, k, d_out, dtype, ld_out, h->sm_count};
  h->last_launches = 0;
  if (rows == 0) return MOE_OK;
  return launch(h, "mxfp4_dequantize", stream, 1,
                [&](cudaStream_t s) { return launch_mxfp4_dequantize(a, s); });
}

extern "C" moe_status moe_grouped_mm_mxfp4(moe_handle *h, int num_experts, int rows, int n, int k,
                                           const uint8_t *d_xcodes, const uint8_t *d_xscales,
                                           const uint8_t *d_wcodes, const uint8_t *d_wscales,
                                           const int32_t *d_seg_off, void *d_out, int out_dtype,
                                           int64_t ld_out, void *stream) {
  if (!h || !d_wcodes || !d_wscales || !d_seg_off ||
      (rows > 0 && (!d_xcodes || !d_xscales || !d_out)))
    return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  if (num_experts < 1 || num_experts > kMaxExperts)
    return refuse(h, "expert count %d outside [1, %d]", num_experts, kMaxExperts);
  if (rows < 0 || rows > kMaxRows || n < 1 || n > kMaxWidth || k < 1 || k > kMaxWidth)
    return refuse(h, "rows %d, widths n = %d, k = %d", rows, n, k);
  if (!float_type(out_dtype)) return refuse(h, "type %d is none of F32, F16 and BF16", out_dtype);
  ld_out = row_stride(rows, ld_out, n);
  if (ld_out < n || ld_out > kMaxStride)
    return refuse(h, "row stride %lld of a row of %d", (long long)ld_out, n);
  if (misaligned(d_xcodes, 16) || misaligned(d_wcodes, 16) || misaligned(d_xscales, 4) ||
      misaligned(d_wscales, 4) || misaligned(d_seg_off, 4) ||
      misaligned(d_out, type_size(out_dtype)))
    return refuse(h, "a pointer is not aligned (codes to 16 bytes, scales to 4)");
  Mxfp4Args a{d_xcodes, d_xscales, d_wcodes, d_wscales, d_out,   d_seg_off, num_experts,
              rows,     n,         k,        out_dtype, ld_out, h->sm_count, h->status};
  h->last_launches = 0;
  if (rows == 0) return MOE_OK;
  return launch(h, "grouped_mm_mxfp4", stream, 1,
                [&](cudaStream_t s) { return launch_mxfp4_mm(a, s); });
}

// ---------------------------------------------------------------------------
// Norms around a block
// ---------------------------------------------------------------------------
namespace {

moe_status check_norm(moe_handle *h, const moe_block_norm_desc *d, BlockNormArgs &a) {
  if (d->rows < 0 || d->hidden < 1 || d->hidden > kMaxNormWidth)
    return refuse(h, "rows %d, width %d (at most %d)", d->rows, d->hidden, kMaxNormWidth);
  if (!float_type(d->res_dtype) || !float_type(d->dtype) ||
      (d->res_dtype != d->dtype && d->res_dtype != MOE_DT_F32))
    return refuse(h, "residual type %d with block type %d: the same, or an F32 residual",
                  d->res_dtype, d->dtype);
  a.ld_res = row_stride(d->rows, d->ld_res, d->hidden);
  a.ld_blk = row_stride(d->rows, d->ld_block, d->hidden);
  if (a.ld_res < d->hidden || a.ld_blk < d->hidden || a.ld_res > kMaxStride ||
      a.ld_blk > kMaxStride)
    return refuse(h, "row strides %lld, %lld of a row of %d", (long long)d->ld_res,
                  (long long)d->ld_block, d->hidden);
  if (!(d->eps >= 0.0f)) return refuse(h, "eps is negative or not a number");
  a.rows = d->rows;
  a.H = d->hidden;
  a.res_dtype = d->res_dtype;
  a.dtype = d->dtype;
  a.post = d->post_norm != 0;
  a.scale = d->residual_scale;
  a.eps = d->eps;
  a.sm_count = h->sm_count;
  a.status = h->status;
  return MOE_OK;
}

}  // namespace

extern "C" moe_status moe_block_norm(moe_handle *h, const moe_block_norm_desc *d, const void *d_x,
                                     const void *d_y, const float *d_w_post, const float *d_gate,
                                     const float *d_w_pre, void *d_x_out, void *d_h,
                                     void *stream) {
  if (!h || !d || (d->rows > 0 && (!d_x || (!d_x_out && !d_h)))) return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  BlockNormArgs a{};
  const moe_status st = check_norm(h, d, a);
  if (st != MOE_OK) return st;
  const size_t rs = type_size(d->res_dtype), bs = type_size(d->dtype);
  if (misaligned(d_x, rs) || misaligned(d_x_out, rs) || misaligned(d_y, bs) ||
      misaligned(d_h, bs) || misaligned(d_w_post, 4) || misaligned(d_w_pre, 4) ||
      misaligned(d_gate, 4))
    return refuse(h, "a pointer is not aligned to its elements");
  a.x = d_x;
  a.y = d_y;
  a.w_post = d_w_post;
  a.w_pre = d_w_pre;
  a.gate = d_gate;
  a.x_out = d_x_out;
  a.h = d_h;
  h->last_launches = 0;
  if (a.rows == 0) return MOE_OK;
  return launch(h, "block_norm", stream, 1,
                [&](cudaStream_t s) { return launch_block_norm(a, s); });
}

extern "C" size_t moe_block_norm_backward_workspace(const moe_handle *h, int rows, int hidden) {
  if (!h || rows < 0 || hidden < 1 || hidden > kMaxNormWidth) return 0;
  return (size_t)block_norm_backward_ctas(rows, hidden, h->sm_count) * 2 * hidden * sizeof(float);
}

extern "C" moe_status moe_block_norm_backward(moe_handle *h, const moe_block_norm_desc *d,
                                              const void *d_dx_out, const void *d_dh,
                                              const void *d_x_out, const void *d_y,
                                              const float *d_w_post, const float *d_gate,
                                              const float *d_w_pre, void *d_dx, void *d_dy,
                                              float *d_dw_post, float *d_dgate, float *d_dw_pre,
                                              void *d_workspace, size_t workspace_bytes,
                                              void *stream) {
  if (!h || !d || !d_workspace || (d->rows > 0 && (!d_x_out || !d_dx || (!d_dx_out && !d_dh))))
    return MOE_ERR_INVALID;
  std::lock_guard<std::mutex> lock(h->mu);
  BlockNormArgs a{};
  const moe_status st = check_norm(h, d, a);
  if (st != MOE_OK) return st;
  if ((d_y != nullptr) != (d_dy != nullptr) && d->rows > 0)
    return refuse(h, "the block's output and its gradient come together");
  if (!d_y && (d_dw_post || d_dgate) && d->rows > 0)
    return refuse(h, "gradients of the gate or the post-norm's gain need the block's output");
  if (!a.post && d_dw_post) return refuse(h, "the gradient of a post-norm's gain without one");
  const size_t rs = type_size(d->res_dtype), bs = type_size(d->dtype);
  if (misaligned(d_dx_out, rs) || misaligned(d_x_out, rs) || misaligned(d_dx, rs) ||
      misaligned(d_dh, bs) || misaligned(d_y, bs) || misaligned(d_dy, bs) ||
      misaligned(d_w_post, 4) || misaligned(d_gate, 4) || misaligned(d_w_pre, 4) ||
      misaligned(d_dw_post, 4) || misaligned(d_dgate, 4) || misaligned(d_dw_pre, 4) ||
      misaligned(d_workspace, 4))
    return refuse(h, "a pointer is not aligned to its elements");
  const size_t need =
      (size_t)block_norm_backward_ctas(a.rows, a.H, a.sm_count) * 2 * a.H * sizeof(float);
  if (workspace_bytes < need)
    return refuse(h, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  a.x = d_x_out;
  a.y = d_y;
  a.w_post = d_w_post;
  a.w_pre = d_w_pre;
  a.gate = d_gate;
  a.dx_out = d_dx_out;
  a.dh = d_dh;
  a.dx = d_dx;
  a.dy = d_dy;
  a.dw_post = d_dw_post;
  a.dgate = d_dgate;
  a.dw_pre = d_dw_pre;
  a.partial = reinterpret_cast<float *>(d_workspace);
  return launch(h, "block_norm_backward", stream, d_dw_pre || d_dw_post ? 2 : 1,
                [&](cudaStream_t s) { return launch_block_norm_backward(a, s); });
}
