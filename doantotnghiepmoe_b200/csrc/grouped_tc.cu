// Matrix products grouped by expert on the tensor cores (tcgen05).
//
// For each expert D = P Q^T with fp32 sums in TMEM, the M side (128 lanes)
// along the contiguous axis of the result and the N side along its rows:
//   forward  out[r, m] = sum_k  w[m, k]    x[r, k]       P = w (K-major),  Q = x (K-major)
//   dgrad    dx[r, m]  = sum_n  w[n, m]    dout[r, n]    P = w (MN-major), Q = dout (K-major)
//   wgrad    dw[n, m]  = sum_r  x[r, m]    dout[r, n]    P = x (MN-major), Q = dout (MN-major)
// No operand is transposed in memory: the MMA takes either major order out of
// 128-byte swizzled tiles.  The rows of an expert are on the N side of the
// first two, where an MMA may be any multiple of 16 wide, so a tile costs what
// its rows are and not a full 128 (a decoded token pays 16 columns).
//
// One persistent CTA an SM walks the items (128 of M x up to 256 of N): one
// thread keeps a ring of 4 stages (48 KB: 64 elements of K of both sides) full
// by TMA across items, one warp issues the MMAs into two accumulator buffers
// of 256 TMEM columns, and 16 warps drain one while the other fills.  Tiles
// that reach past a segment read other experts' rows and drop their columns;
// in wgrad, where the rows are summed, the rows of the last K step that belong
// to others are zeroed in shared memory before the MMA (zeros alone would not
// do on one side: 0 x NaN).  Every wait is bounded, as in expert_tc.cu.
#include <cuda.h>

#include <algorithm>

#include "expert_tc.h"
#include "ops.h"
#include "segments.cuh"
#include "tc_ptx.cuh"

namespace moe {
namespace {

using namespace tcp;

constexpr int kTM = 128, kTN = 256, kTK = 64;  // tile; kTK elements are 128 bytes
constexpr int kStages = 4;
constexpr uint32_t kABytes = kTM * 128, kStageBytes = (kTM + kTN) * 128;
constexpr int kBoxRows = 32;                 // N-side rows of one copy (K-major)
constexpr uint32_t kMnBox = kTK * 128;       // one copy of an MN-major side: 64 of M or N
constexpr size_t kSmem = 1024 + sizeof(Pipe<kStages>) + sizeof(SegTable) + 16 +
                         (size_t)kStages * kStageBytes + kEpiWarps * kDrainBytes;
static_assert(kSmem <= 232448, "shared memory");

struct Item {
  int e, m0;  // expert, first M index
  int c0, nc; // first N index (a row, or a column of dout) and how many
  int row0;   // wgrad: first row of the expert
  int len;    // extent of the summed axis
};

template <int KIND>
struct Work {
  const GroupedArgs &a;
  const SegTable &seg;
  int nM, nN;
  int total;
  __device__ __forceinline__ Work(const GroupedArgs &a_, const SegTable &s) : a(a_), seg(s) {
    nM = ((KIND == kGroupedFwd ? a.n : a.k) + kTM - 1) / kTM;
    nN = (a.n + kTN - 1) / kTN;
    total = KIND == kGroupedWgrad ? a.E * nM * nN : seg.total * nM;
  }
  __device__ __forceinline__ Item item(int w) const {
    Item it;
    const int g = w / nM;
    it.m0 = (w - g * nM) * kTM;
    if (KIND == kGroupedWgrad) {
      it.e = g / nN;
      it.c0 = g % nN * kTN;
      it.nc = min(kTN, a.n - it.c0);
      it.row0 = seg.off[it.e];
      it.len = seg.rows(it.e);
    } else {
      it.e = seg.expert_of(g, a.E);
      const int cnt = seg.rows(it.e), nt = seg.tile0[it.e + 1] - seg.tile0[it.e];
      const int sz = tile_rows(cnt, nt), t = g - seg.tile0[it.e];
      it.c0 = seg.off[it.e] + t * sz;
      it.nc = min(sz, cnt - t * sz);
      it.row0 = 0;
      it.len = KIND == kGroupedFwd ? a.k : a.n;
    }
    return it;
  }
};

template <int KIND>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_tc_kernel(const __grid_constant__ CUtensorMap mapP,
                      const __grid_constant__ CUtensorMap mapQ, GroupedArgs a) {
  constexpr bool kPMn = KIND != kGroupedFwd, kQMn = KIND == kGroupedWgrad;
  extern __shared__ uint8_t smem_raw[];
  using P = Pipe<kStages>;
  P &pp = *reinterpret_cast<P *>(smem_raw);
  SegTable &seg = *reinterpret_cast<SegTable *>(smem_raw + sizeof(P));
  uint8_t *tiles = align1024(smem_raw + sizeof(P) + sizeof(SegTable));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) pp.init(1);
  if (warp == 1) tmem_alloc(&pp.tmem_base, 2 * kTN);
  if (warp == 2) build_segments(seg, a.seg_off, a.E, a.R, kTN, a.status);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const Work<KIND> work(a, seg);

  if (warp == 0) {
    int q = 0;
    bool ok = true;
    for (int w = blockIdx.x; w < work.total && ok; w += gridDim.x) {
      const Item it = work.item(w);
      const int nk = (it.len + kTK - 1) / kTK;
      const int nbox = kQMn ? (it.nc + 63) / 64 : (it.nc + kBoxRows - 1) / kBoxRows;
      const uint32_t bytes = kABytes + nbox * (kQMn ? kMnBox : kBoxRows * 128u);
      for (int kb = 0; kb < nk; ++kb, ++q) {
        const int s = q % kStages, use = q / kStages;
        ok = use == 0 || pp.wait_warp(&pp.empty[s], (use - 1) & 1);
        if (!ok) break;
        if (elect_one()) {
          uint8_t *st = tiles + s * kStageBytes;
          tma::mbar_expect_tx(&pp.full[s], bytes);
          const int kr = it.row0 + kb * kTK;  // first row of K of an MN-major tile
          if (kPMn) {
            for (int i = 0; i < 2; ++i)
              tma::load_3d(st + i * kMnBox, &mapP, &pp.full[s], (it.m0 + 64 * i) * 2, kr,
                           kQMn ? 0 : it.e);
          } else {
            tma::load_3d(st, &mapP, &pp.full[s], kb * 128, it.m0, it.e);
          }
          for (int i = 0; i < nbox; ++i) {
            if (kQMn)
              tma::load_3d(st + kABytes + i * kMnBox, &mapQ, &pp.full[s], (it.c0 + 64 * i) * 2, kr,
                           0);
            else
              tma::load_3d(st + kABytes + i * kBoxRows * 128, &mapQ, &pp.full[s], kb * 128,
                           it.c0 + i * kBoxRows, 0);
          }
        }
        __syncwarp();
      }
    }
    if (!ok) pp.drain(q);
  } else if (warp == 1) {
    // fp32 sums, both operands of one type, M = 128
    const uint32_t fmt = a.dtype == MOE_DT_BF16 ? 1u : 0u;
    const uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)kPMn << 15) |
                            ((uint32_t)kQMn << 16) | ((uint32_t)(kTM >> 4) << 24);
    int q = 0, j = 0;
    for (int w = blockIdx.x; w < work.total; w += gridDim.x) {
      const Item it = work.item(w);
      const int nk = (it.len + kTK - 1) / kTK;
      if (nk == 0) continue;
      const int buf = j & 1;
      if (j >= 2 && !pp.wait_warp(&pp.tempty[buf], ((j >> 1) - 1) & 1)) break;
      fence_after_sync();
      const uint32_t d = pp.tmem_base + (uint32_t)(buf * kTN);
      const uint32_t idesc = idesc0 | ((uint32_t)((it.nc + 15) >> 4) << 18);
      bool ok = true;
      for (int kb = 0; kb < nk; ++kb, ++q) {
        const int s = q % kStages;
        if (!pp.wait_warp(&pp.full[s], (q / kStages) & 1)) {
          ok = false;
          break;
        }
        uint8_t *st = tiles + s * kStageBytes;
        const int left = it.len - kb * kTK;  // elements of K that belong to the sum
        int steps = kTK / 16;
        if (kQMn && left < kTK) {
          steps = (left + 15) / 16;
          const int nbox = 2 + (it.nc + 63) / 64, zr = steps * 16 - left;
          for (int i = lane; i < nbox * zr * 8; i += 32) {
            const int box = i / (zr * 8), r = left + i / 8 % zr;
            *reinterpret_cast<uint4 *>(st + box * kMnBox + r * 128 + i % 8 * 16) =
                make_uint4(0, 0, 0, 0);
          }
          tma::fence_proxy_async_smem();
          __syncwarp();
        }
        fence_after_sync();
        if (elect_one()) {
          const uint32_t base = su32(st);
          const uint64_t pd = kPMn ? sw128_desc(base, kMnBox, 1024) : sw128_desc(base, 16, 1024);
          const uint64_t qd = kQMn ? sw128_desc(base + kABytes, kMnBox, 1024)
                                   : sw128_desc(base + kABytes, 16, 1024);
          // 16 elements of K further: 32 bytes of a row, or 16 rows of 128 bytes
          constexpr uint64_t kPStep = (kPMn ? 2048 : 32) >> 4, kQStep = (kQMn ? 2048 : 32) >> 4;
          if (steps == kTK / 16) {
#pragma unroll
            for (int k = 0; k < kTK / 16; ++k)
              mma_f16(d, pd + k * kPStep, qd + k * kQStep, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          } else {
            for (int k = 0; k < steps; ++k)
              mma_f16(d, pd + k * kPStep, qd + k * kQStep, idesc, (kb > 0 || k > 0) ? 1u : 0u);
          }
          commit(&pp.empty[s]);
        }
        __syncwarp();
      }
      if (!ok) break;
      if (elect_one()) commit(&pp.tfull[buf]);
      ++j;
    }
    if (elect_one()) commit(&pp.done);
  } else if (warp >= 2) {
    const int quarter = warp & 3, grp = (warp - 2) >> 2;
    uint32_t *buf32 = reinterpret_cast<uint32_t *>(tiles + kStages * kStageBytes +
                                                   (warp - 2) * kDrainBytes);
    const int M = KIND == kGroupedFwd ? a.n : a.k;
    const int64_t ld = KIND == kGroupedFwd ? a.ld_out : KIND == kGroupedDgrad ? a.ld_x : a.ld_w;
    int j = 0;
    for (int w = blockIdx.x; w < work.total; w += gridDim.x) {
      const Item it = work.item(w);
      const int m = it.m0 + quarter * 32;
      const int64_t at = (KIND == kGroupedWgrad ? it.e * a.es_w : 0) + it.c0 * ld + m;
      const bool some = it.len > 0;
      const int buf = j & 1;
      if (some) {
        if (!pp.wait_warp(&pp.tfull[buf], (j >> 1) & 1)) break;
        fence_after_sync();
        ++j;
      }
      const uint32_t trow =
          pp.tmem_base + (uint32_t)(buf * kTN) + ((uint32_t)(32 * quarter) << 16);
      drain_tile(trow, some, it.nc, grp, M - m, a.out, a.out_dtype, at, ld, buf32);
      if (some) {
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
  if (warp == 1) tmem_dealloc(pp.tmem_base, 2 * kTN);
}

template <int KIND>
cudaError_t launch_kind(const CUtensorMap &p, const CUtensorMap &q, const GroupedArgs &a,
                        cudaStream_t s) {
  static const cudaError_t attr = cudaFuncSetAttribute(
      grouped_tc_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  if (attr != cudaSuccess) return attr;
  const long long nM = ((KIND == kGroupedFwd ? a.n : a.k) + kTM - 1) / kTM;
  const long long g = KIND == kGroupedWgrad ? (long long)a.E * ((a.n + kTN - 1) / kTN)
                                            : a.R / kTN + std::min(a.E, a.R);
  if (g * nM > INT32_MAX / 2) return cudaErrorInvalidValue;  // item numbers are 32-bit
  const int grid = (int)std::min<long long>(g * nM, a.sm_count);
  grouped_tc_kernel<KIND><<<grid, kThreads, kSmem, s>>>(p, q, a);
  return cudaGetLastError();
}

}  // namespace

bool grouped_tc_ok(GroupedKind kind, const GroupedArgs &a) {
  const uintptr_t base = (uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.dout;
  const int64_t strides = (kind != kGroupedDgrad ? a.ld_x : 0) |
                          (kind != kGroupedFwd ? a.ld_out : 0) |
                          (kind != kGroupedWgrad ? (a.ld_w | a.es_w) : 0);
  return a.R > 0 && base % 16 == 0 && strides % 8 == 0;
}

cudaError_t launch_grouped_tc(GroupedKind kind, const GroupedArgs &a, cudaStream_t s) {
  CUtensorMap p, q;
  const auto rows_map = [&](CUtensorMap *m, const void *t, int width, int64_t ld, int box) {
    return tc::encode_map3d(m, t, (uint64_t)width * 2, (uint64_t)a.R, 1, (uint64_t)ld * 2,
                            (uint64_t)ld * 2, (uint32_t)box);
  };
  bool ok;
  if (kind == kGroupedWgrad) {
    ok = rows_map(&p, a.x, a.k, a.ld_x, kTK) && rows_map(&q, a.dout, a.n, a.ld_out, kTK);
  } else {
    ok = tc::encode_map3d(&p, a.w, (uint64_t)a.k * 2, (uint64_t)a.n, (uint64_t)a.E,
                          (uint64_t)a.ld_w * 2, (uint64_t)a.es_w * 2,
                          kind == kGroupedFwd ? kTM : kTK);
    ok = ok && (kind == kGroupedFwd ? rows_map(&q, a.x, a.k, a.ld_x, kBoxRows)
                                    : rows_map(&q, a.dout, a.n, a.ld_out, kBoxRows));
  }
  if (!ok) return cudaErrorInvalidValue;
  if (kind == kGroupedFwd) return launch_kind<kGroupedFwd>(p, q, a, s);
  if (kind == kGroupedDgrad) return launch_kind<kGroupedDgrad>(p, q, a, s);
  return launch_kind<kGroupedWgrad>(p, q, a, s);
}

}  // namespace moe
