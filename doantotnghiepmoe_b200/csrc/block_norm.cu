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
//   t  = <D w_post, y rp>
//   dy = g rp (D w_post - y rp t / H)        dgate = t
//   dw_post = sum over rows of g D y rp
// (without a post-norm dy = g D and dgate = <D, y>).
//
// Every statistic and sum is fp32; x' is normalised before it is rounded to
// its type.  Both passes move each value once and are bound by HBM: a row
// stays in the registers of one CTA (8 consecutive values a thread and step)
// from its loads to its stores, with two block sums forward (sum y^2, then
// sum x'^2) and two backward (sum x'^2, <c, x'>, sum y^2 together, then t).
// Forward, a CTA a row: 4096 x 2048 (fp32 residual, bf16 block) in 21 us, 4.8 TB/s
// (a ring of rows in a few persistent CTAs took 24).  Backward, where a CTA sums
// the gains' gradients over its rows in registers: while there are more rows than
// CTAs it keeps a ring of rows in shared memory full by bulk copies, up to 4
// ahead.  8192 x 2048 bf16 in 61 us, 3.3 TB/s, half of the issue slots busy (with
// one row ahead in registers 73); a second kernel adds the CTAs' sums in a fixed
// order, 8 us.
#include <algorithm>

#include "../../include/moe_b200.h"
#include "common.cuh"
#include "cvt.cuh"
#include "ops.h"
#include "tma_ptx.cuh"

namespace moe {
namespace {

constexpr int kMaxThreads = 256, kBwdThreads = 128;
constexpr int kMaxRing = 4;  // rows ahead

// Rows on their way into shared memory.  A row is up to four tensors' rows one
// behind the other; a CTA's rows are r, r + gridDim.x, ...
struct RowRing {
  uint8_t *mem;
  uint64_t *full;
  int *failed;
  uint32_t row_bytes;
  int stages;
  const uint8_t *src[4];
  int64_t stride[4];
  uint32_t bytes[4];

  __device__ __forceinline__ RowRing(uint8_t *m, uint64_t *f, int *fail, int n)
      : mem(m), full(f), failed(fail), row_bytes(0), stages(n) {}
  __device__ __forceinline__ void tensor(int i, const void *p, int64_t row_stride, uint32_t n) {
    src[i] = reinterpret_cast<const uint8_t *>(p);
    stride[i] = row_stride;
    bytes[i] = p ? n : 0;
    row_bytes += bytes[i];
  }
  __device__ __forceinline__ uint32_t offset(int i) const {
    uint32_t o = 0;
    for (int j = 0; j < i; ++j) o += bytes[j];
    return o;
  }
  __device__ __forceinline__ void issue(int s, int64_t r) {  // one thread
    tma::mbar_expect_tx(&full[s], row_bytes);
    uint8_t *dst = mem + (size_t)s * row_bytes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!bytes[i]) continue;
      tma::load_bulk(dst, src[i] + r * stride[i], &full[s], bytes[i]);
      dst += bytes[i];
    }
  }
  __device__ __forceinline__ void start(int64_t rows) {
    if (threadIdx.x == 0) {
      for (int s = 0; s < stages; ++s) tma::mbar_init(&full[s], 1);
      *failed = 0;
      tma::fence_mbar_init();
      for (int s = 0; s < stages; ++s)
        if (blockIdx.x + (int64_t)s * gridDim.x < rows) issue(s, blockIdx.x + (int64_t)s * gridDim.x);
    }
    __syncthreads();
  }
  // Behind a barrier that follows the reads of stage s: the row that takes its
  // place, and the stage after it.
  __device__ __forceinline__ void refill(int &s, uint32_t &use, int64_t r, int64_t rows) {
    if (threadIdx.x == 0 && r + (int64_t)stages * gridDim.x < rows)
      issue(s, r + (int64_t)stages * gridDim.x);
    if (++s == stages) {
      s = 0;
      ++use;
    }
  }
  // Copies in flight land before the CTA exits after a failed wait.
  __device__ __forceinline__ void finish(uint32_t *status) {
    if (!*(volatile int *)failed) return;
    if (threadIdx.x == 0) {
      set_status(status, kStatusTimeout);
      for (int s = 0; s < stages; ++s)
        for (uint32_t p = 0; p < 2; ++p) tma::mbar_wait(&full[s], p, nullptr, tma::kWaitCycles / 64);
    }
    __syncthreads();
  }
  // A row that does not arrive in time is recorded; the threads leave together
  // behind their next barrier.
  __device__ __forceinline__ const uint8_t *wait(int s, uint32_t use) {
    if (!tma::mbar_try(&full[s], use & 1) && !tma::mbar_wait(&full[s], use & 1, failed)) *failed = 1;
    return mem + (size_t)s * row_bytes;
  }
};

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
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(const BlockNormArgs a) {
  __shared__ float buf[8][kMaxThreads / 32];
  int flip = 0;
  const int64_t r = blockIdx.x;
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool post = a.y && a.post;
  // everything the row needs is on its way before the first sum
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

// RING: rows through shared memory; else straight into registers.
template <typename TX, typename TY, int V, int NE, bool RING>
__global__ void __launch_bounds__(V == 1 ? kMaxThreads : kBwdThreads,
                                  V == 1 ? (NE <= 4 ? 4 : 1) : V * NE <= 16 ? 4 : 1)
    block_norm_bwd_kernel(const BlockNormArgs a, int stages) {
  __shared__ float buf[8][kMaxThreads / 32];
  __shared__ uint64_t full[kMaxRing];
  __shared__ int failed;
  extern __shared__ __align__(16) uint8_t ring_mem[];
  int flip = 0;
  const int H = a.H;
  const float inv_h = 1.0f / (float)H;
  const bool post = a.y && a.post;
  RowRing ring(ring_mem, full, &failed, stages);
  if (RING) {
    ring.tensor(0, a.x, a.ld_res * sizeof(TX), H * sizeof(TX));
    ring.tensor(1, a.dx_out, a.ld_res * sizeof(TX), H * sizeof(TX));
    ring.tensor(2, a.dh, a.ld_blk * sizeof(TY), H * sizeof(TY));
    ring.tensor(3, a.y, a.ld_blk * sizeof(TY), H * sizeof(TY));
    ring.start(a.rows);
  }
  const uint32_t od = ring.offset(1), oc = ring.offset(2), oy = ring.offset(3);
  // The gains stay in registers where a thread has little of the row.
  constexpr bool kKeep = V * NE <= 16;
  Piece<float, V> gq[NE], gp[NE];
  if (kKeep) {
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      load_gain<V>(gq[n], a.w_pre, (n * blockDim.x + threadIdx.x) * V, H);
      load_gain<V>(gp[n], post ? a.w_post : nullptr, (n * blockDim.x + threadIdx.x) * V, H);
    }
  }
  float wpre[NE][V] = {}, wpost[NE][V] = {};  // sums of the gains' gradients
  TX *dx_row = reinterpret_cast<TX *>(a.dx) + blockIdx.x * a.ld_res;
  TY *dy_row = reinterpret_cast<TY *>(a.dy) + blockIdx.x * a.ld_blk;
  int st = 0;
  uint32_t use = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    Piece<TX, V> x[NE], dx[NE];
    Piece<TY, V> ch[NE], y[NE];
    const uint8_t *mem = RING ? ring.wait(st, use) : nullptr;
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      const int at = (n * blockDim.x + threadIdx.x) * V;
      if constexpr (RING) {
        x[n].load_shared(mem, at, H);
        if (a.dx_out) dx[n].load_shared(mem + od, at, H);
        if (a.dh) ch[n].load_shared(mem + oc, at, H);
        if (a.y) y[n].load_shared(mem + oy, at, H);
      } else {
        x[n].load(reinterpret_cast<const TX *>(a.x) + r * a.ld_res, at, H);
        if (a.dx_out) dx[n].load(reinterpret_cast<const TX *>(a.dx_out) + r * a.ld_res, at, H);
        if (a.dh) ch[n].load(reinterpret_cast<const TY *>(a.dh) + r * a.ld_blk, at, H);
        if (a.y) y[n].load(reinterpret_cast<const TY *>(a.y) + r * a.ld_blk, at, H);
      }
      if (!a.dx_out) dx[n].clear();
      if (!a.dh) ch[n].clear();
      if (!a.y) y[n].clear();
    }
    if (RING) {
      __syncthreads();  // the row is in registers
      if (*(volatile int *)&failed) break;
      ring.refill(st, use, r, a.rows);
    }
    float s[3] = {0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      if (!kKeep) load_gain<V>(gq[n], a.w_pre, (n * blockDim.x + threadIdx.x) * V, H);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xv = x[n][i], yv = y[n][i];
        s[0] = fmaf(xv, xv, s[0]);
        s[1] = fmaf(gq[n][i], ch[n][i] * xv, s[1]);
        s[2] = fmaf(yv, yv, s[2]);
      }
    }
    block_sums(s, buf, flip);
    const float rq = a.dh ? __frsqrt_rn(s[0] * inv_h + a.eps) : 0.0f;
    const float rp = post ? __frsqrt_rn(s[2] * inv_h + a.eps) : 1.0f;
    // The row enters as x rq and y rp, which are of size one: rq^3 alone leaves fp32's
    // range for rows above 1e12 or, without eps, below 1e-13, whose sums do not.
    const float kx = rq * s[1] * inv_h * rq;
    const float g = a.y && a.gate ? a.gate[r] : 1.0f;
    float t[1] = {0.0f}, d[NE][V];
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      const int at = (n * blockDim.x + threadIdx.x) * V;
      if (!kKeep) {
        load_gain<V>(gq[n], a.w_pre, at, H);
        load_gain<V>(gp[n], post ? a.w_post : nullptr, at, H);
      }
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float xn = rq * x[n][i], c = ch[n][i];
        wpre[n][i] = fmaf(c, xn, wpre[n][i]);
        const float D = fmaf(-kx, xn, fmaf(rq, c * gq[n][i], dx[n][i]));
        const float Dy = D * (rp * y[n][i]);
        o[i] = a.scale * D;
        wpost[n][i] = fmaf(g, Dy, wpost[n][i]);
        t[0] = fmaf(gp[n][i], Dy, t[0]);
        d[n][i] = D * gp[n][i];
      }
      store_v<TX, V>(dx_row, at, H, o);
    }
    dx_row += (int64_t)gridDim.x * a.ld_res;
    if (!a.y) continue;
    const float grp = g * rp;
    float ky = 0.0f;
    if (post || a.dgate) {
      block_sums(t, buf, flip);
      if (post) ky = -rp * (t[0] * inv_h);
      if (a.dgate && threadIdx.x == 0) a.dgate[r] = t[0];
    }
#pragma unroll
    for (int n = 0; n < NE; ++n) {
#pragma unroll
      for (int i = 0; i < V; ++i) d[n][i] = grp * fmaf(ky, y[n][i], d[n][i]);
      store_v<TY, V>(dy_row, (n * blockDim.x + threadIdx.x) * V, H, d[n]);
    }
    dy_row += (int64_t)gridDim.x * a.ld_blk;
  }
  if (RING) ring.finish(a.status);
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

size_t type_bytes(int dt) { return dt == MOE_DT_F32 ? 4 : 2; }

// The backward pass in CTAs that fill an SM's registers and whose rings share its
// shared memory: narrow rows take small CTAs, and many.  A thread has 8 or 16
// values of a row in pieces of 8, or, of rows without 16-byte alignment, 4 single
// ones (8 a thread took 190 us for 6420 rows of 1001 values, 4 take 86).
constexpr size_t kMaxRingBytes = 56 * 1024;  // of a CTA: a quarter of an SM's 224 KB
struct BwdShape {
  int threads, per_sm;
  size_t ring_bytes;
  BwdShape(int H, bool vec)
      : threads(!vec ? std::min(kMaxThreads, (H + 127) / 128 * 32) : H > 512 ? kBwdThreads : 64),
        per_sm(H > 512 ? 4 : H > 256 ? 8 : 16),
        ring_bytes(kMaxRingBytes * 4 / per_sm) {}
};

// Threads of a row: whole warps that cover it once, 256 at most.
int row_threads(int H, int v, int most) {
  const int need = (H + v - 1) / v;
  return std::min(most, (need + 31) / 32 * 32);
}

// Calls f(integral V, integral NE) for a row of H values: V = 8 where every
// pointer and row stride allows 16-byte accesses and H is a multiple of 8.
template <typename F>
cudaError_t by_width(int H, bool vec, int threads, F &&f) {
  const int v = vec ? 8 : 1, ne = (H + v * threads - 1) / (v * threads);
  if (vec) {
    if (ne <= 1) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 1>{});
    if (ne <= 2) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    if (ne <= 4) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    if (ne <= 8) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 16>{});
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
  return std::max(1, std::min(rows, sm_count * BwdShape(H, true).per_sm));
}

cudaError_t launch_block_norm(const BlockNormArgs &a, cudaStream_t s) {
  if (a.rows <= 0) return cudaSuccess;
  return by_types(a.res_dtype, a.dtype, [&](auto tx, auto ty) {
    return by_width(a.H, vec_ok(a), kMaxThreads, [&](auto v, auto ne) {
      if constexpr (v() * ne() > 64) return cudaErrorInvalidValue;  // wider than kMaxNormWidth
      else
        block_norm_kernel<decltype(tx), decltype(ty), v(), ne()>
            <<<a.rows, row_threads(a.H, v(), kMaxThreads), 0, s>>>(a);
      return cudaGetLastError();
    });
  });
}

cudaError_t launch_block_norm_backward(const BlockNormArgs &a, cudaStream_t s) {
  const int ctas = block_norm_backward_ctas(a.rows, a.H, a.sm_count);
  const bool vec = vec_ok(a);
  const size_t row = (size_t)a.H * (type_bytes(a.res_dtype) * (a.dx_out ? 2 : 1) +
                                    type_bytes(a.dtype) * ((a.dh ? 1 : 0) + (a.y ? 1 : 0)));
  const BwdShape shape(a.H, vec);
  const int stages =
      vec && a.rows > ctas ? (int)std::min<size_t>(kMaxRing, shape.ring_bytes / row) : 0;
  cudaError_t e = by_types(a.res_dtype, a.dtype, [&](auto tx, auto ty) {
    return by_width(a.H, vec, shape.threads, [&](auto v, auto ne) {
      const int threads = row_threads(a.H, v(), shape.threads);
      if constexpr (v() == 8) {
        if (stages >= 2) {
          auto *kernel = block_norm_bwd_kernel<decltype(tx), decltype(ty), v(), ne(), true>;
          // One bound for every width: the attribute belongs to the kernel, which all
          // handles and host threads of the process launch, and a smaller one set
          // between another call's own and its launch would refuse that launch.
          const cudaError_t attr = cudaFuncSetAttribute(
              kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxRingBytes);
          if (attr != cudaSuccess) return attr;
          kernel<<<ctas, threads, stages * row, s>>>(a, stages);
          return cudaGetLastError();
        }
      }
      block_norm_bwd_kernel<decltype(tx), decltype(ty), v(), ne(), false>
          <<<ctas, threads, 0, s>>>(a, 0);
      return cudaGetLastError();
    });
  });
  if (e != cudaSuccess || (!a.dw_pre && !a.dw_post)) return e;
  block_norm_gains_kernel<<<(2 * a.H + 31) / 32, 1024, 0, s>>>(a.partial, ctas, a.H, a.dw_pre,
                                                             a.dw_post);
  return cudaGetLastError();
}

}  // namespace moe
