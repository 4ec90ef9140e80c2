// Grouped product of MXFP4 operands on the tensor cores: out[r, m] = sum over
// the blocks b of K of sx[r, b] sw[m, b] <qx[r, b], qw[m, b]> as
// tcgen05.mma kind::mxf4, which takes the 4-bit codes and the scale bytes as
// they lie in memory and adds in fp32 (cut off, not rounded): nothing is decoded.
//
// The shape of the kernel is that of grouped_tc.cu: weights on the M side,
// an expert's rows on the N side in tiles that are any multiple of 16, one
// persistent CTA an SM, a ring of TMA stages that runs on across items, two
// accumulator buffers.  A stage is 256 elements of K: 128-byte rows of codes
// of 128 weight rows and up to 192 rows of x.
//
// The MMA reads the scales from TMEM, one 32-bit column for 32 rows and 4
// blocks (128 elements of K), in the order of the rows' lanes.  Scale bytes
// lie by row in memory; four warps, each at another stage, fetch 4 of them at
// a time and store them in the order that a 32-row copy to TMEM takes: word
// (r % 32) * 4 + r / 32 of a 512-byte group.  192 rows of N rather than 256 leave
// room in TMEM for a set of scales a stage beside the two buffers: a stage is
// filled again only once its MMAs are done, and so its set is free with it.
//
// Measured on B200 (128 experts, n = 1536, k = 2048): 32768 rows 89 us, 0.32 GB of
// DRAM traffic and 0.88 GB from L2 into the SMs, tensor pipe 29%.  The fullest SM goes
// through 160 steps of 36 KB on average, 960 cycles each; at the 54 bytes a cycle that
// the copies of a single CTA reach they are 670 of those.  64 rows 27 us, 107 MB of
// weights at 3.9 TB/s, of which the first 4 us pass before the first stage has landed.
#include <cuda.h>

#include <algorithm>

#include "expert_tc.h"
#include "ops.h"
#include "segments.cuh"
#include "tc_ptx.cuh"

namespace moe {
namespace {

using namespace tcp;

constexpr int kTM = 128;
// Rows of x in a tile.  A draining warp that adds parts (below) holds 32 columns for
// each 128 of them, and its registers have room for one such turn.
constexpr int tile_rows(bool parts) { return parts ? 128 : 192; }
constexpr int kTN = tile_rows(false);
// An addition to a sum in TMEM takes 64 of K and is cut off rather than rounded.
// Against 64 bits, values of blocks with different scales, of the result's norm: one
// sum of K = 1024 1.6e-7, 2048 2.9e-7, 4096 5.6e-7, 16384 2.5e-6, 262144 5.4e-5 (7.8e-5
// of one sign).  So an fp32 result is summed over at most 2048 of K at a time, where
// fp32 sums that round lose as much (2.9e-7 for a library product of the decoded
// values), and an fp16 one over 2^17, a tenth of half its step; bf16 loses less than
// that over every width.  In steps of 256 of K:
__host__ __device__ constexpr int sum_limit(int out_dtype) {
  return out_dtype == MOE_DT_F32 ? 8 : out_dtype == MOE_DT_F16 ? 512 : 4096;
}
constexpr uint32_t kABytes = kTM * 128;
constexpr int kMaxStages = 8;
constexpr int kGroup = 512;            // scale bytes of 128 rows and 4 blocks
constexpr int kScaleBytes = 6 * kGroup;  // of a stage: 2 groups of w, 2 x 2 of x
constexpr int kSetCols = 24;             // TMEM columns of a stage's scales
constexpr uint32_t kTmemCols = 512;
// A warp comes to a stage every time round or less often, never two rounds late:
// the parity of a wait names one round only.
constexpr int kScaleWarps = 4;
static_assert(kScaleWarps <= 4, "the fewest stages of a ring");
constexpr int kMxThreads = kThreads + 32 * kScaleWarps;
constexpr uint32_t kRingBytes = 4 * (kABytes + kTN * 128 + kScaleBytes) + 32 * 1024;
constexpr size_t kSmem = 1024 + sizeof(Pipe<kMaxStages>) + sizeof(SegTable) + 16 + kRingBytes +
                         kEpiWarps * kDrainBytes;
static_assert(kSmem <= 232448, "shared memory");

// A lane's scale words of a step (256 elements of K): words 2 kb and 2 kb + 1 of
// rows 32 i + lane of w (i < 4) and of x (i - 4).
struct Scales {
  uint2 u[10];
  bool wide;  // more than 128 rows of x
};

struct Maps {
  CUtensorMap w, x[3];  // x in boxes of 64, 32 and 16 rows
  FastDiv by_m;         // by the tiles of M
};

// PARTS: K is longer than one sum may be.
template <bool PARTS>
__global__ void __launch_bounds__(kMxThreads, 1)
    mxfp4_tc_kernel(const __grid_constant__ Maps maps, const Mxfp4Args a) {
  extern __shared__ uint8_t smem_raw[];
  using P = Pipe<kMaxStages>;
  P &pp = *reinterpret_cast<P *>(smem_raw);
  SegTable &seg = *reinterpret_cast<SegTable *>(smem_raw + sizeof(P));
  uint8_t *tiles = align1024(smem_raw + sizeof(P) + sizeof(SegTable));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    pp.init(1 + 32);  // a copying warp (for both), a scale warp's lanes
    tma::prefetch_map(&maps.w);
    for (int i = 0; i < 3; ++i) tma::prefetch_map(&maps.x[i]);
  }
  if (warp == 1) tmem_alloc(&pp.tmem_base, kTmemCols);
  if (warp == 3) build_segments(seg, a.seg_off, a.E, a.R, tile_rows(PARTS), 16, a.status);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();

  // The largest tile decides the stages' size and how many fit, and the columns of
  // an accumulator buffer: 4 stages with 192 rows of x, 8 with the few rows of a
  // decode batch, whose stages hold the weights and little else.
  const int most = (seg.most + 15) & ~15;
  const uint32_t stage_bytes = kABytes + ((uint32_t)most * 128u + 1023u & ~1023u);
  const int acc_cols = (most + 31) & ~31;
  const int stages = min(min(kMaxStages, (int)(kRingBytes / (stage_bytes + kScaleBytes))),
                         ((int)kTmemCols - 2 * acc_cols) / kSetCols);
  uint8_t *scales = tiles + stages * stage_bytes;
  const int nM = (a.n + kTM - 1) / kTM, nk = (a.k + 255) / 256;
  int part = nk;  // steps of one sum: equal parts
  if (PARTS) {
    const int limit = sum_limit(a.out_dtype), parts = (nk + limit - 1) / limit;
    part = (nk + parts - 1) / parts;
  }
  const int total = seg.total * nM;
  struct Item {
    int e, m0, c0, nc;
  };
  const auto item = [&](int w) {
    Item it;
    const int g = maps.by_m.div(w);
    it.m0 = (w - g * nM) * kTM;
    it.e = seg.expert_of(g, a.E);
    const int sz = seg.size[it.e], at = (g - seg.tile0[it.e]) * sz;
    it.c0 = seg.off[it.e] + at;
    it.nc = min(sz, seg.rows(it.e) - at);
    return it;
  };

  if (warp == 0 || warp == 2) {
    Ring ring(stages);
    bool ok = true;
    for (int w = blockIdx.x; w < total && ok; w += gridDim.x) {
      const Item it = item(w);
      const int rows = (it.nc + 15) & ~15;
      for (int kb = 0; kb < nk; ++kb, ring.next()) {
        const int s = ring.s;
        ok = ring.use == 0 || pp.wait_warp(&pp.empty[s], (ring.use - 1) & 1);
        if (!ok) break;
        if (elect_one()) {
          uint8_t *st = tiles + s * stage_bytes;
          uint64_t *bar = &pp.full[s];
          if (warp == 0) {
            tma::mbar_expect_tx(bar, kABytes + rows * 128u);
            tma::load_3d(st, &maps.w, bar, kb * 128, it.m0, it.e);
          } else {
            st += kABytes;
            for (int r = 0; r + 64 <= rows; r += 64)
              tma::load_3d(st + r * 128, &maps.x[0], bar, kb * 128, it.c0 + r, 0);
            if (rows & 32)
              tma::load_3d(st + (rows & 192) * 128, &maps.x[1], bar, kb * 128,
                           it.c0 + (rows & 192), 0);
            if (rows & 16)
              tma::load_3d(st + (rows & 224) * 128, &maps.x[2], bar, kb * 128,
                           it.c0 + (rows & 224), 0);
          }
        }
        __syncwarp();
      }
    }
    if (!ok) pp.drain(ring);
  } else if (warp == 1) {
    // E2M1 operands, E8M0 scales, M = 128
    const uint32_t idesc0 = (1u << 7) | (1u << 10) | (1u << 23) | ((uint32_t)(kTM >> 4) << 24);
    const uint32_t sf0 = pp.tmem_base + 2 * acc_cols;
    Ring ring(stages);
    int j = 0;
    for (int w = blockIdx.x; w < total; w += gridDim.x, ++j) {
      const Item it = item(w);
      if (j >= 2 && !pp.wait_warp(&pp.tempty[j & 1], ((j >> 1) - 1) & 1)) break;
      fence_after_sync();
      uint32_t d = pp.tmem_base + (uint32_t)((j & 1) * acc_cols);
      const uint32_t idesc = idesc0 | ((uint32_t)((it.nc + 15) >> 4) << 18);
      bool ok = true;
      int first = 0;  // step that opens the running sum
      for (int kb = 0; kb < nk; ++kb, ring.next()) {
        const int s = ring.s;
        if (PARTS && kb == first + part) {  // the next part, in the other buffer
          if (elect_one()) commit(&pp.tfull[j & 1]);
          ++j;
          ok = j < 2 || pp.wait_warp(&pp.tempty[j & 1], ((j >> 1) - 1) & 1);
          if (!ok) break;
          fence_after_sync();
          d = pp.tmem_base + (uint32_t)((j & 1) * acc_cols);
          first = kb;
        }
        if (!pp.wait_warp(&pp.full[s], ring.use & 1)) {
          ok = false;
          break;
        }
        fence_after_sync();
        if (elect_one()) {
          const uint32_t base = su32(tiles + s * stage_bytes);
          const uint64_t sd = rows16_desc(su32(scales + s * kScaleBytes));
          const uint64_t wd = sw128_desc(base, 16, 1024), xd = sw128_desc(base + kABytes, 16, 1024);
          const uint32_t sfa = sf0 + (uint32_t)s * kSetCols, sfb = sfa + 8;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            cp_scales(sfa + 4 * g, sd + (g * kGroup >> 4));
            cp_scales(sfb + 8 * g, sd + ((2 + 2 * g) * kGroup >> 4));
            if (it.nc > 128) cp_scales(sfb + 8 * g + 4, sd + ((3 + 2 * g) * kGroup >> 4));
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t id = (uint32_t)(k & 1) * 2;  // bytes 0-1 or 2-3 of a scale word
            mma_mxf4(d, wd + 2 * k, xd + 2 * k, idesc | (id << 4) | (id << 29), sfa + 4 * (k >> 1),
                     sfb + 8 * (k >> 1), (kb > first || k > 0) ? 1u : 0u);
          }
          commit(&pp.empty[s]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) commit(&pp.tfull[j & 1]);
    }
    if (elect_one()) commit(&pp.done);
  } else if (warp < 3 + kScaleWarps) {
    const int words = mxfp4_scale_stride(a.k) / 4;
    const uint32_t *xs = reinterpret_cast<const uint32_t *>(a.xs);
    const uint32_t *ws = reinterpret_cast<const uint32_t *>(a.ws);
    // both words of a step in one load, where that is aligned
    const bool even = words % 2 == 0 && (((uintptr_t)xs | (uintptr_t)ws) & 7) == 0;
    // This warp's steps are every kScaleWarps-th; the next one's words are loaded
    // before this one's are stored.
    int w = blockIdx.x, kb = warp - 3, it_w = -1;
    Item it{};
    Scales cur, next;
    const auto advance = [&] {  // to the item that holds step kb; false behind the last
      for (; kb >= nk && w < total; kb -= nk) w += gridDim.x;
      if (w >= total) return false;
      if (w != it_w) {
        it = item(w);
        it_w = w;
      }
      return true;
    };
    const auto load = [&](Scales &v) {
      const uint32_t *wrow = ws + ((int64_t)it.e * a.n + it.m0) * words + 2 * kb + lane * words;
      const uint32_t *xrow = xs + (int64_t)it.c0 * words + 2 * kb + lane * words;
      const bool two = 2 * kb + 1 < words;
#pragma unroll
      for (int i = 0; i < 10; ++i) {
        const int r0 = (i < 4 ? i : i - 4) * 32, left = (i < 4 ? a.n - it.m0 : it.nc) - r0;
        const uint32_t *p = (i < 4 ? wrow : xrow) + r0 * words;
        uint2 u = make_uint2(0u, 0u);
        if (left > 0) {  // warp-uniform
          if (lane < left) {
            if (two && even) {
              u = __ldg(reinterpret_cast<const uint2 *>(p));
            } else {
              u.x = __ldg(p);
              if (two) u.y = __ldg(p + 1);
            }
          }
        }
        v.u[i] = u;
      }
      v.wide = it.nc > 128;
    };
    bool more = advance();
    if (more) load(cur);
    Ring ring(stages);
    for (int i = 3; i < warp; ++i) ring.next();
    while (more) {
      kb += kScaleWarps;
      more = advance();
      if (more) load(next);
      const int s = ring.s;
      const uint32_t use = ring.use;
      if (use > 0 && !pp.wait_warp(&pp.empty[s], (use - 1) & 1)) break;
      uint4 *dst = reinterpret_cast<uint4 *>(scales + s * kScaleBytes) + lane;
      const uint2(&u)[10] = cur.u;
      dst[0] = make_uint4(u[0].x, u[1].x, u[2].x, u[3].x);
      dst[32] = make_uint4(u[0].y, u[1].y, u[2].y, u[3].y);
      dst[64] = make_uint4(u[4].x, u[5].x, u[6].x, u[7].x);
      dst[128] = make_uint4(u[4].y, u[5].y, u[6].y, u[7].y);
      if (cur.wide) {
        dst[96] = make_uint4(u[8].x, u[9].x, 0u, 0u);
        dst[160] = make_uint4(u[8].y, u[9].y, 0u, 0u);
      }
      tma::fence_proxy_async_smem();  // before the tensor cores' proxy reads them
      tma::mbar_arrive(&pp.full[s]);
      cur = next;
#pragma unroll
      for (int i = 0; i < kScaleWarps; ++i) ring.next();
    }
  } else {
    const int ew = warp - 3 - kScaleWarps, quarter = warp & 3, grp = ew >> 2;
    uint32_t *buf32 = reinterpret_cast<uint32_t *>(tiles + kRingBytes + ew * kDrainBytes);
    int j = 0;
    for (int w = blockIdx.x; w < total; w += gridDim.x) {
      const Item it = item(w);
      const int m = it.m0 + quarter * 32;
      const int64_t at = it.c0 * a.ld_out + m;
      const uint32_t lanes = pp.tmem_base + ((uint32_t)(32 * quarter) << 16);
      if constexpr (PARTS) {
        Sums<1> sums;
        sums.zero();
        bool ok = true;
        for (int kb = 0; kb < nk; kb += part, ++j) {
          ok = pp.wait_warp(&pp.tfull[j & 1], (j >> 1) & 1);
          if (!ok) break;
          fence_after_sync();
          sums.add(lanes + (uint32_t)((j & 1) * acc_cols), it.nc, grp * 32);
          fence_before_sync();
          __syncwarp();
          if (lane == 0) tma::mbar_arrive(&pp.tempty[j & 1]);
        }
        if (!ok) break;
        sums.store(it.nc, grp * 32, a.n - m, a.out, a.out_dtype, at, a.ld_out, buf32);
      } else {
        const int buf = j & 1;
        if (!pp.wait_warp(&pp.tfull[buf], (j >> 1) & 1)) break;
        ++j;
        fence_after_sync();
        for (int c = grp * 32; c < it.nc; c += kTurnCols) {
          Sums<1> sums;
          sums.take(lanes + (uint32_t)(buf * acc_cols), it.nc, c);
          sums.store(it.nc, c, a.n - m, a.out, a.out_dtype, at, a.ld_out, buf32);
        }
        fence_before_sync();
        __syncwarp();
        if (lane == 0) tma::mbar_arrive(&pp.tempty[buf]);
      }
    }
  }
  if (threadIdx.x == 32) tma::mbar_wait(&pp.done, 0, nullptr);  // no MMA still runs
  fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && pp.abort_flag) set_status(a.status, kStatusTimeout);
  if (warp == 1) tmem_dealloc(pp.tmem_base, kTmemCols);
}

template <bool PARTS>
cudaError_t launch_as(const Maps &maps, const Mxfp4Args &a, cudaStream_t s) {
  const cudaError_t attr = cudaFuncSetAttribute(
      mxfp4_tc_kernel<PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  if (attr != cudaSuccess) return attr;
  const long long items = (long long)(a.R / tile_rows(PARTS) + std::min(a.E, a.R)) *
                          ((a.n + kTM - 1) / kTM);
  if (items > INT32_MAX / 2) return cudaErrorInvalidValue;  // item numbers are 32-bit
  mxfp4_tc_kernel<PARTS><<<(int)std::min<long long>(items, a.sm_count), kMxThreads, kSmem, s>>>(
      maps, a);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_mxfp4_mm(const Mxfp4Args &a, cudaStream_t s) {
  if (a.R <= 0) return cudaSuccess;
  const uint64_t row = (uint64_t)mxfp4_code_stride(a.k);
  Maps maps;
  bool ok = tc::encode_map3d(&maps.w, a.wc, row, (uint64_t)a.n, (uint64_t)a.E, row, row * a.n, kTM);
  for (int i = 0; i < 3; ++i)
    ok = ok && tc::encode_map3d(&maps.x[i], a.xc, row, (uint64_t)a.R, 1, row, row, 64 >> i);
  if (!ok) return cudaErrorInvalidValue;
  maps.by_m = FastDiv((a.n + kTM - 1) / kTM);
  return (a.k + 255) / 256 > sum_limit(a.out_dtype) ? launch_as<true>(maps, a, s)
                                                    : launch_as<false>(maps, a, s);
}

}  // namespace moe
