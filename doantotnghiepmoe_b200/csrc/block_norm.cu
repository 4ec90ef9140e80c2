// The norms before and after a block, fused with the block's gate and the
// residual scale, and their backward pass.
//
// Forward, a row x of the residual stream and y of the block's output:
//   z  = y / rms(y) * w_post        (z = y without a post-norm)
//   x' = a x + g z                  rms(v) = sqrt(sum v^2 / H + eps)
//   h  = x' / rms(x') * w_pre       (the next block's input)
// Backward, with c = dh w_pre, rq = 1 / rms(x'), rp = 1 / rms(y):
//   D  = dx' + rq c - x' rq^3 <c, x'> / H
//   dx = a D         dw_pre  = sum over rows of dh x' rq
//   S  = <D w_post, y>
//   dy = g rp (D w_post - y rp^2 S / H)      dgate = rp S
//   dw_post = sum over rows of g D y rp
// (without a post-norm dy = g D and dgate = <D, y>).
//
// Every statistic and sum is fp32; x' is normalised before it is rounded to
// its type.  Both passes move each value once and are bound by HBM: a row
// stays in the registers of one CTA (8 consecutive values a thread and step)
// from its loads to its stores, with two block sums forward (sum y^2, then
// sum x'^2) and two backward (sum x'^2, <c, x'>, sum y^2 together, then S).
// The gains' gradients are summed in registers over the rows of a CTA, whose
// sums a second kernel adds in a fixed order.
#include <algorithm>

#include "../../include/moe_b200.h"
#include "common.cuh"
#include "cvt.cuh"
#include "ops.h"

namespace moe {
namespace {

constexpr int kMaxThreads = 256;

// Sums of N values over the block; every thread gets them.  Two alternating
// halves of `buf`, so that one barrier a call is enough.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*buf)[kMaxThreads / 32], int &flip) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int d = 16; d; d >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
  if (nw == 1) return;
  float(*b)[kMaxThreads / 32] = buf + flip * 4;
  flip ^= 1;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) b[i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float s = 0.0f;
    for (int w = 0; w < nw; ++w) s += b[i][w];
    v[i] = s;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_v(T *p, int c, int H, const float (&v)[V]) {
  if (c >= H) return;
  if constexpr (V == 8) store8(p + c, v);
  else p[c] = from_f32<T>(v[0]);
}

// A gain's values, or ones.
template <int V>
__device__ __forceinline__ void load_gain(Piece<float, V> &w, const float *g, int c, int H) {
  if (g) {
    w.load(g, c, H);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) w.w[i] = __float_as_uint(1.0f);
  }
}

template <typename TX, typename TY, int V, int NE>
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(BlockNormArgs a) {
  __shared__ float buf[8][kMaxThreads / 32];
  int flip = 0;
  const int64_t r = blockIdx.x;
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool post = a.y && a.post;
  // everything a row needs is on its way before the first sum
  Piece<TX, V> x[NE];
  Piece<TY, V> y[NE];
  Piece<float, V> wq[NE], wp[NE];
#pragma unroll
  for (int n = 0; n < NE; ++n) {
    const int c = (n * blockDim.x + threadIdx.x) * V;
    if (a.y) y[n].load(reinterpret_cast<const TY *>(a.y) + r * a.ld_blk, c, H);
    else y[n].clear();
    x[n].load(reinterpret_cast<const TX *>(a.x) + r * a.ld_res, c, H);
    load_gain<V>(wp[n], post ? a.w_post : nullptr, c, H);
    load_gain<V>(wq[n], a.w_pre, c, H);
  }
  float g = a.y && a.gate ? a.gate[r] : 1.0f;
  if (post) {
    float s[1] = {0.0f};
#pragma unroll
    for (int n = 0; n < NE; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] = fmaf(y[n][i], y[n][i], s[0]);
    block_sums(s, buf, flip);
    g *= __frsqrt_rn(s[0] * inv_h + a.eps);
  }
  float xo[NE][V], s[1] = {0.0f};
#pragma unroll
  for (int n = 0; n < NE; ++n) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      xo[n][i] = x[n][i] * a.scale;
      if (a.y) xo[n][i] = fmaf(g * wp[n][i], y[n][i], xo[n][i]);
      s[0] = fmaf(xo[n][i], xo[n][i], s[0]);
    }
    if (a.x_out)
      store_v<TX, V>(reinterpret_cast<TX *>(a.x_out) + r * a.ld_res,
                     (n * blockDim.x + threadIdx.x) * V, H, xo[n]);
  }
  if (!a.h) return;
  block_sums(s, buf, flip);
  const float rq = __frsqrt_rn(s[0] * inv_h + a.eps);
#pragma unroll
  for (int n = 0; n < NE; ++n) {
#pragma unroll
    for (int i = 0; i < V; ++i) xo[n][i] *= rq * wq[n][i];
    store_v<TY, V>(reinterpret_cast<TY *>(a.h) + r * a.ld_blk,
                   (n * blockDim.x + threadIdx.x) * V, H, xo[n]);
  }
}

// What the backward pass reads of a row.
template <typename TX, typename TY, int V>
struct BwdRow {
  Piece<TX, V> x, d;
  Piece<TY, V> c, y;
  __device__ __forceinline__ void load(const BlockNormArgs &a, int64_t r, int at) {
    const int H = r < a.rows ? a.H : 0;
    x.load(reinterpret_cast<const TX *>(a.x) + r * a.ld_res, at, H);
    if (a.dx_out) d.load(reinterpret_cast<const TX *>(a.dx_out) + r * a.ld_res, at, H);
    else d.clear();
    if (a.dh) c.load(reinterpret_cast<const TY *>(a.dh) + r * a.ld_blk, at, H);
    else c.clear();
    if (a.y) y.load(reinterpret_cast<const TY *>(a.y) + r * a.ld_blk, at, H);
    else y.clear();
  }
};

template <typename TX, typename TY, int V, int NE>
__global__ void __launch_bounds__(kMaxThreads) block_norm_bwd_kernel(BlockNormArgs a) {
  __shared__ float buf[8][kMaxThreads / 32];
  int flip = 0;
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool post = a.y && a.post;
  // The next row is loaded before this one's sums where its registers allow.
  constexpr bool kAhead = V * NE <= 8;
  float wpre[NE][V] = {}, wpost[NE][V] = {};  // sums of the gains' gradients
  Piece<float, V> gq[NE], gp[NE];
  BwdRow<TX, TY, V> next[NE];
#pragma unroll
  for (int n = 0; n < NE; ++n) {
    const int at = (n * blockDim.x + threadIdx.x) * V;
    if (kAhead) {
      load_gain<V>(gq[n], a.w_pre, at, H);
      load_gain<V>(gp[n], post ? a.w_post : nullptr, at, H);
      next[n].load(a, blockIdx.x, at);
    }
  }
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    BwdRow<TX, TY, V> row[NE];
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      const int at = (n * blockDim.x + threadIdx.x) * V;
      if (kAhead) {
        row[n] = next[n];
        next[n].load(a, r + gridDim.x, at);
      } else {
        row[n].load(a, r, at);
        load_gain<V>(gq[n], a.w_pre, at, H);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[0] = fmaf(row[n].x[i], row[n].x[i], s[0]);
        s[1] = fmaf(row[n].c[i] * gq[n][i], row[n].x[i], s[1]);
        s[2] = fmaf(row[n].y[i], row[n].y[i], s[2]);
      }
    }
    block_sums(s, buf, flip);
    const float rq = a.dh ? __frsqrt_rn(s[0] * inv_h + a.eps) : 0.0f;
    const float rp = post ? __frsqrt_rn(s[2] * inv_h + a.eps) : 1.0f;
    const float kx = rq * rq * rq * s[1] * inv_h;
    const float g = a.y && a.gate ? a.gate[r] : 1.0f;
    float t[1] = {0.0f}, d[NE][V];
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      const int at = (n * blockDim.x + threadIdx.x) * V;
      if (!kAhead) {
        load_gain<V>(gq[n], a.w_pre, at, H);
        load_gain<V>(gp[n], post ? a.w_post : nullptr, at, H);
      }
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = row[n].x[i], c = row[n].c[i];
        wpre[n][i] = fmaf(c, x * rq, wpre[n][i]);
        d[n][i] = fmaf(rq, c * gq[n][i], row[n].d[i]) - kx * x;
        o[i] = a.scale * d[n][i];
        wpost[n][i] = fmaf(g * d[n][i], row[n].y[i] * rp, wpost[n][i]);
        d[n][i] *= gp[n][i];
        t[0] = fmaf(d[n][i], row[n].y[i], t[0]);
      }
      store_v<TX, V>(reinterpret_cast<TX *>(a.dx) + r * a.ld_res, at, H, o);
    }
    if (!a.y) continue;
    float ky = 0.0f;
    if (post || a.dgate) {
      block_sums(t, buf, flip);
      if (post) ky = rp * rp * t[0] * inv_h;
      if (a.dgate && threadIdx.x == 0) a.dgate[r] = rp * t[0];
    }
#pragma unroll
    for (int n = 0; n < NE; ++n) {
#pragma unroll
      for (int i = 0; i < V; ++i) d[n][i] = g * rp * (d[n][i] - ky * row[n].y[i]);
      store_v<TY, V>(reinterpret_cast<TY *>(a.dy) + r * a.ld_blk,
                     (n * blockDim.x + threadIdx.x) * V, H, d[n]);
    }
  }
  float *part = a.partial + (int64_t)blockIdx.x * 2 * H;
#pragma unroll
  for (int n = 0; n < NE; ++n)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (n * blockDim.x + threadIdx.x) * V + i;
      if (c < H) {
        part[c] = wpre[n][i];
        part[H + c] = wpost[n][i];
      }
    }
}

// dw[c] = the sum over the CTAs' partial sums, in an order that their number
// fixes: a warp a chain of every 32nd, then the chains one after another.
__global__ void __launch_bounds__(1024) block_norm_gains_kernel(const float *part, int ctas, int H,
                                                                float *dw_pre, float *dw_post) {
  __shared__ float sm[32][33];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float s = 0.0f;
  if (c < 2 * H) {
#pragma unroll 4
    for (int g = w; g < ctas; g += 32) s += part[(int64_t)g * 2 * H + c];
  }
  sm[w][lane] = s;
  __syncthreads();
  if (w || c >= 2 * H) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) s += sm[i][lane];
  if (c < H) {
    if (dw_pre) dw_pre[c] = s;
  } else if (dw_post) {
    dw_post[c - H] = s;
  }
}

// Threads of a row: whole warps that cover it once, 256 at most.
int row_threads(int H, int v) {
  const int need = (H + v - 1) / v;
  return std::min(kMaxThreads, (need + 31) / 32 * 32);
}

// Calls f(integral V, integral NE) for a row of H values: V = 8 where every
// pointer and row stride allows 16-byte accesses and H is a multiple of 8.
template <typename F>
cudaError_t by_width(int H, bool vec, F &&f) {
  const int ne = (H + (vec ? 8 : 1) * kMaxThreads - 1) / ((vec ? 8 : 1) * kMaxThreads);
  if (vec) {
    if (ne <= 1) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    if (ne <= 2) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    if (ne <= 4) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
  }
  if (ne <= 4) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  if (ne <= 8) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
  if (ne <= 16) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 64>{});
}

template <typename F>
cudaError_t by_types(int res, int blk, F &&f) {
  if (res == MOE_DT_BF16) return f(__nv_bfloat16{}, __nv_bfloat16{});
  if (res == MOE_DT_F16) return f(__half{}, __half{});
  if (blk == MOE_DT_BF16) return f(float{}, __nv_bfloat16{});
  if (blk == MOE_DT_F16) return f(float{}, __half{});
  return f(float{}, float{});
}

bool aligned16(std::initializer_list<const void *> ps) {
  uintptr_t u = 0;
  for (const void *p : ps) u |= (uintptr_t)p;
  return (u & 15) == 0;
}

bool vec_ok(const BlockNormArgs &a) {
  return a.H % 8 == 0 && a.ld_res % 8 == 0 && a.ld_blk % 8 == 0 &&
         aligned16({a.x, a.y, a.w_pre, a.w_post, a.x_out, a.h, a.dx_out, a.dh, a.dx, a.dy});
}

}  // namespace

int block_norm_backward_ctas(int rows, int H, int sm_count) {
  (void)H;
  return std::max(1, std::min(rows, sm_count * 3));
}

cudaError_t launch_block_norm(const BlockNormArgs &a, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  const bool vec = vec_ok(a);
  return by_types(a.res_dtype, a.dtype, [&](auto tx, auto ty) {
    return by_width(a.H, vec, [&](auto v, auto ne) {
      block_norm_kernel<decltype(tx), decltype(ty), v(), ne()>
          <<<a.rows, row_threads(a.H, v()), 0, s>>>(a);
      return cudaGetLastError();
    });
  });
}

cudaError_t launch_block_norm_backward(const BlockNormArgs &a, cudaStream_t s) {
  const int ctas = block_norm_backward_ctas(a.rows, a.H, a.sm_count);
  const bool vec = vec_ok(a);
  cudaError_t e = by_types(a.res_dtype, a.dtype, [&](auto tx, auto ty) {
    return by_width(a.H, vec, [&](auto v, auto ne) {
      block_norm_bwd_kernel<decltype(tx), decltype(ty), v(), ne()>
          <<<ctas, row_threads(a.H, v()), 0, s>>>(a);
      return cudaGetLastError();
    });
  });
  if (e != cudaSuccess || (!a.dw_pre && !a.dw_post)) return e;
  block_norm_gains_kernel<<<(2 * a.H + 31) / 32, 1024, 0, s>>>(a.partial, ctas, a.H, a.dw_pre,
                                                             a.dw_post);
  return cudaGetLastError();
}

}  // namespace moe
