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
// A pair of CTAs (cta_group::2) works on one tile of 256 of M x up to 256 of N:
// each CTA loads its 128 of M and half of the N side and keeps 128 rows of D.
// Against a CTA's own 128 x 256 tile this moves 32 KB rather than 48 KB from L2
// for the same products, and L2 to SM traffic is what bounded that kernel (54
// bytes a cycle and SM).  One persistent CTA an SM: two warps keep a ring of
// stages full by TMA across items (6 blocks of 64 elements of K of both sides, or
// more of smaller tiles), the even CTA's issuing warp issues the pair's MMAs into
// two accumulator buffers of 256 TMEM columns, and 16 warps of each CTA drain one
// while the other fills.  The odd CTA's issuing warp passes on that its stage has
// landed.  Tiles that reach past a segment read other experts' rows and drop their
// columns; in wgrad, where the rows are summed, the last K step's rows beyond the
// expert's must be zeros on both sides (0 x NaN): that step's copies are cut to
// 16, 4 and 1 rows, and the rows up to the MMA's 16 come from behind the tensor's
// last row, where a copy reads zeros.  (Zeroing them in shared memory cost the
// step two fences, 2000 cycles in the even CTA and 11000 in the odd one while
// results were stored.)  Every wait on a barrier in memory is bounded, as in
// expert_tc.cu.
//
// Measured on B200 (32768 rows of 128 experts, bf16): forward n = 1536, k = 2048
// 208 us, 1.04 GB of DRAM traffic at 5.0 TB/s and 2.2 GB from L2 into the SMs, which
// alone takes 164 us; dgrad n = 2048, k = 768 113 us (5.1 TB/s); wgrad of it 160 us,
// of which its 403 MB of results bound the drains.  512 rows of 64 experts, n =
// 2048, k = 1024, fp32 result: 50 us, 5.4 TB/s of weights.
#include <cuda.h>

#include <algorithm>

#include "expert_tc.h"
#include "ops.h"
#include "segments.cuh"
#include "tc_ptx.cuh"

namespace moe {
namespace {

using namespace tcp;

constexpr int kTM = 256, kTN = 256, kTK = 64;  // tile of a pair; kTK elements are 128 bytes
constexpr uint32_t kABytes = kTM / 2 * 128;  // of a CTA and a block of kTK
constexpr uint32_t kRingBytes = 6 * (kTM + kTN) / 2 * 128;
// A stage holds kSub blocks of kTK: two halve the waits and commits, which a
// decoded token pays one by one (15.2 -> 13.5 us); wgrad's sums over an expert's
// rows are often shorter than two blocks (279 us with one, 284 with two).
template <int KIND>
constexpr int kSubOf = KIND == kGroupedWgrad ? 1 : 2;
constexpr int kMaxStages = 10;
// The tensor cores cut each addition to a sum in TMEM off rather than round it, so the
// error grows with the additions, 16 of K each.  Against 64 bits, of the result's norm,
// normal bf16 (fp16) values: one sum of K = 256 2.3e-7 (3.4e-7), 512 4.7e-7 (6.4e-7),
// 1024 1.0e-6 (1.3e-6), 4096 4.4e-6 (4.9e-6), 65536 7.6e-5; values of one sign: 1024
// 6.9e-7 (5.8e-6), 65536 3.8e-4 (4.2e-4).  A result is therefore summed over at most
// sum_limit of K at a time, in equal parts, and the draining warps add the parts,
// rounded, in their registers.  For an fp32 result 256 is the longest part with which
// normal values lose no more than in fp32 sums that round, at the usual lengths (K =
// 1024, parts of 128 / 256 / 512: 1.3e-7, 2.3e-7, 4.7e-7 in bf16, where a library
// product has 2.5e-7; 2.0e-7, 3.4e-7, 6.5e-7 in fp16, where it has 5.7e-7; only fp16
// values of one sign lose more, 1.1e-6 to its 4.8e-7).  Its price against one sum: 512
// rows of 64 experts, n = 2048, k = 1024 47.2 -> 50.0 us, prefill with an fp32 result
// 232 -> 253 us (128: 53 and 275).  Results of 16 bits lose more to their own rounding
// up to the lengths below, where a sum of one sign is short by a tenth of half a step
// of the type.  The draining form is another kernel for each of the two (Parts), so
// that it holds the stores of its type alone.
enum Parts { kWhole, kPartsF32, kPartsHalf };
__host__ __device__ constexpr int sum_limit(int out_dtype) {
  return out_dtype == MOE_DT_F32 ? 256 : out_dtype == MOE_DT_F16 ? 8192 : 65536;
}
constexpr uint32_t kMnBox = kTK * 128;    // one copy of an MN-major side: 64 of M or N

// Tensor maps: the M side and the N side with rows in boxes of several heights.
//   forward, dgrad  p[0] all of a tile; q[0..2] 64, 32 and 16 rows
//   wgrad           p[0..3], q[0..3]: 64, 16, 4 and 1 rows
struct Maps {
  CUtensorMap p[4], q[4];
  FastDiv by_m, by_n;  // by the tiles of M, and of N in wgrad
};
constexpr size_t kSmem = 1024 + sizeof(Pipe<kMaxStages>) + sizeof(SegTable) + 16 + kRingBytes +
                         kEpiWarps * kDrainBytes;
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
  const Maps &maps;
  int nM, nN;
  int total;
  __device__ __forceinline__ Work(const GroupedArgs &a_, const SegTable &s, const Maps &m)
      : a(a_), seg(s), maps(m) {
    nM = ((KIND == kGroupedFwd ? a.n : a.k) + kTM - 1) / kTM;
    nN = (a.n + kTN - 1) / kTN;
    total = KIND == kGroupedWgrad ? a.E * nM * nN : seg.total * nM;
  }
  __device__ __forceinline__ Item item(int w) const {
    Item it;
    const int g = maps.by_m.div(w);
    it.m0 = (w - g * nM) * kTM;
    if (KIND == kGroupedWgrad) {
      it.e = maps.by_n.div(g);
      it.c0 = (g - it.e * nN) * kTN;
      it.nc = min(kTN, a.n - it.c0);
      it.row0 = seg.off[it.e];
      it.len = seg.rows(it.e);
    } else {
      it.e = seg.expert_of(g, a.E);
      const int sz = seg.size[it.e], at = (g - seg.tile0[it.e]) * sz;
      it.c0 = seg.off[it.e] + at;
      it.nc = min(sz, seg.rows(it.e) - at);
      it.row0 = 0;
      it.len = KIND == kGroupedFwd ? a.k : a.n;
    }
    return it;
  }
};

// The copies of an MN-major side's K step: rows [row, row + 64) of `boxes`
// columns of 64 elements from col on, or, where only left < 64 of them belong
// to the sum, those and zeros up to a multiple of 16.  zero: a row behind the
// tensor.
__device__ __forceinline__ void load_mn(uint8_t *st, const CUtensorMap (&m)[4], uint64_t *bar,
                                        int col, int boxes, int row, int left, int zero) {
  if (left >= kTK) {
    for (int i = 0; i < boxes; ++i)
      tma::load_3d(st + i * kMnBox, &m[0], bar, (col + 64 * i) * 2, row, 0);
    return;
  }
  for (int i = 0; i < boxes; ++i) {
    const int x = (col + 64 * i) * 2;
    uint8_t *dst = st + i * kMnBox;
    int r = 0;
    for (; r + 16 <= left; r += 16) tma::load_3d(dst + r * 128, &m[1], bar, x, row + r, 0);
    if (r == left) continue;
    const int end = r + 16;
    for (; r + 4 <= left; r += 4) tma::load_3d(dst + r * 128, &m[2], bar, x, row + r, 0);
    for (; r & 3 || r < left; ++r)
      tma::load_3d(dst + r * 128, &m[3], bar, x, r < left ? row + r : zero, 0);
    for (; r < end; r += 4) tma::load_3d(dst + r * 128, &m[2], bar, x, zero, 0);
  }
}

// PARTS: the result's sums may be cut into parts.  In wgrad the host knows
// only that an expert may have that many rows; the items of those that have fewer
// drain as in the other form (the odd gradients of 1332 rows over 72 experts: 71.2
// us with every item held in registers first, 68.3 so).
template <int KIND, Parts PARTS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    grouped_tc_kernel(const __grid_constant__ Maps maps, const GroupedArgs a) {
  constexpr bool kPMn = KIND != kGroupedFwd, kQMn = KIND == kGroupedWgrad;
  constexpr int kSub = kSubOf<KIND>;
  extern __shared__ uint8_t smem_raw[];
  using P = Pipe<kMaxStages>;
  P &pp = *reinterpret_cast<P *>(smem_raw);
  SegTable &seg = *reinterpret_cast<SegTable *>(smem_raw + sizeof(P));
  uint8_t *tiles = align1024(smem_raw + sizeof(P) + sizeof(SegTable));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  // full: the M side's copying warp (for both), and the odd CTA's stage in the
  // even one; tempty: both CTAs drain
  if (threadIdx.x == 0) {
    pp.init(rank == 0 ? 2 : 1, 2 * kEpiWarps);
    for (int i = 0; i < (kQMn ? 4 : 1); ++i) tma::prefetch_map(&maps.p[i]);
    for (int i = 0; i < (kQMn ? 4 : 3); ++i) tma::prefetch_map(&maps.q[i]);
  }
  if (warp == 1) tmem_alloc_pair(&pp.tmem_base, 2 * kTN);
  if (warp == 3) build_segments(seg, a.seg_off, a.E, a.R, kTN, 32, a.status);
  fence_before_sync();
  __syncthreads();
  cluster_sync();
  fence_after_sync();
  const Work<KIND> work(a, seg, maps);
  // The largest tile's N side decides the stages' size and with it how many fit:
  // with the few rows of a decode batch they hold the weights alone, and more of
  // them are on their way.
  const int half_most = (min(kQMn ? a.n : seg.most, kTN) + 31) / 32 * 16;
  const uint32_t sub_bytes =
      kABytes + (kQMn ? (uint32_t)(half_most + 63) / 64 * kMnBox : half_most * 128u);
  const uint32_t stage_bytes = kSub * sub_bytes;
  const int stages = min(kMaxStages, (int)(kRingBytes / stage_bytes));
  const auto part_of = [&](int len) {  // how much of K = len goes into one sum
    const int limit = sum_limit(PARTS == kPartsF32 ? MOE_DT_F32 : a.out_dtype);
    if (PARTS == kWhole || len <= limit) return len;
    const int parts = (len + limit - 1) / limit;
    return ((len + parts - 1) / parts + 127) & ~127;  // whole stages
  };

  if (warp == 0 || warp == 2) {
    Ring ring(stages);
    bool ok = true;
    for (int w = pair; w < work.total && ok; w += pairs) {
      const Item it = work.item(w);
      const int half = (it.nc + 31) / 32 * 16, c0 = it.c0 + rank * half, m0 = it.m0 + rank * 128;
      const int boxes = (half + 63) / 64;  // of an MN-major N side
      for (int k0 = 0; k0 < it.len; k0 += kSub * kTK, ring.next()) {
        ok = ring.use == 0 || pp.wait_warp(&pp.empty[ring.s], (ring.use - 1) & 1);
        if (!ok) break;
        if (elect_one()) {
          uint8_t *st = tiles + ring.s * stage_bytes;
          uint64_t *bar = &pp.full[ring.s];
          const int left = it.len - k0;  // of the summed axis
          if (warp == 0)
            tma::mbar_expect_tx(
                bar, kQMn ? (2 + boxes) * 128u * min(kSub * kTK, (left + 15) & ~15)
                          : (kABytes + half * 128u) * (left > kTK ? kSub : 1));
          for (int sub = 0; sub < kSub; ++sub, st += sub_bytes) {
            if (sub * kTK >= left) break;
            const int k = k0 + sub * kTK;
            if (warp == 0) {
              if (KIND == kGroupedFwd) {
                tma::load_3d(st, &maps.p[0], bar, k * 2, m0, it.e);
              } else if (KIND == kGroupedDgrad) {
                tma::load_3d(st, &maps.p[0], bar, m0 * 2, k, it.e);
                tma::load_3d(st + kMnBox, &maps.p[0], bar, m0 * 2 + 128, k, it.e);
              } else {
                load_mn(st, maps.p, bar, m0, 2, it.row0 + k, left - sub * kTK, a.R);
              }
            } else {
              uint8_t *sq = st + kABytes;
              if (kQMn) {
                load_mn(sq, maps.q, bar, c0, boxes, it.row0 + k, left - sub * kTK, a.R);
              } else {
                if (half & 192) tma::load_3d(sq, &maps.q[0], bar, k * 2, c0, 0);
                if (half & 128) tma::load_3d(sq + 64 * 128, &maps.q[0], bar, k * 2, c0 + 64, 0);
                if (half & 32)
                  tma::load_3d(sq + (half & 64) * 128, &maps.q[1], bar, k * 2, c0 + (half & 64), 0);
                if (half & 16)
                  tma::load_3d(sq + (half & 96) * 128, &maps.q[2], bar, k * 2, c0 + (half & 96), 0);
              }
            }
          }
        }
        __syncwarp();
      }
    }
    if (!ok) pp.drain(ring);
  } else if (warp == 1) {
    // fp32 sums, both operands of one type, M = 256
    const uint32_t fmt = a.dtype == MOE_DT_BF16 ? 1u : 0u;
    const uint32_t idesc0 = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)kPMn << 15) |
                            ((uint32_t)kQMn << 16) | ((uint32_t)(kTM >> 4) << 24);
    // 16 elements of K further: 32 bytes of a row, or 16 rows of 128 bytes
    constexpr uint64_t kPStep = (kPMn ? 2048 : 32) >> 4, kQStep = (kQMn ? 2048 : 32) >> 4;
    const uint64_t pd0 = sw128_desc(su32(tiles), kPMn ? kMnBox : 16, 1024);
    const uint64_t qd0 = sw128_desc(su32(tiles) + kABytes, kQMn ? kMnBox : 16, 1024);
    Ring ring(stages);
    int j = 0;
    for (int w = pair; w < work.total; w += pairs) {
      const Item it = work.item(w);
      if (it.len == 0) continue;
      const uint32_t idesc = idesc0 | ((uint32_t)((it.nc + 31) >> 5) << 19);
      const int part = part_of(it.len);
      uint32_t d = 0;
      bool ok = true;
      int next = 0, more = 0;  // where the next part begins; 0: the part's first MMA
      for (int k0 = 0; k0 < it.len; k0 += kSub * kTK, ring.next()) {
        if (k0 == next) {
          if (k0 > 0) {
            if (rank == 0 && elect_one()) commit_pair(&pp.tfull[j & 1]);
            ++j;
          }
          ok = rank != 0 || j < 2 || pp.wait_warp(&pp.tempty[j & 1], ((j >> 1) - 1) & 1);
          if (!ok) break;
          d = pp.tmem_base + (uint32_t)((j & 1) * kTN);
          next = part < it.len - k0 ? k0 + part : it.len;
          more = 0;
        }
        if (!pp.wait_warp(&pp.full[ring.s], ring.use & 1)) {
          ok = false;
          break;
        }
        fence_after_sync();
        if (rank != 0) {
          if (elect_one()) arrive_at(&pp.full[ring.s], 0);
        } else if (elect_one()) {
          const uint64_t at = (uint64_t)(ring.s * (stage_bytes >> 4));
          const int left = it.len - k0;
          if (left >= kSub * kTK || (!kQMn && left > kTK)) {
#pragma unroll
            for (int k = 0; k < kSub * kTK / 16; ++k) {
              const uint64_t sub = at + (uint64_t)(k / (kTK / 16)) * (sub_bytes >> 4);
              mma_f16_pair(d, pd0 + sub + k % (kTK / 16) * kPStep,
                           qd0 + sub + k % (kTK / 16) * kQStep, idesc, (more || k > 0) ? 1u : 0u);
            }
          } else {
            // forward and dgrad: one block of kTK, the rest of it zeros; wgrad: the
            // rows there are, in steps of 16
            const int steps = kQMn ? (left + 15) / 16 : kTK / 16;
            for (int k = 0; k < steps; ++k) {
              const uint64_t sub = at + (uint64_t)(k / (kTK / 16)) * (sub_bytes >> 4);
              mma_f16_pair(d, pd0 + sub + k % (kTK / 16) * kPStep,
                           qd0 + sub + k % (kTK / 16) * kQStep, idesc, (more || k > 0) ? 1u : 0u);
            }
          }
          commit_pair(&pp.empty[ring.s]);
        }
        more = 1;
        __syncwarp();
      }
      if (!ok) break;
      if (rank == 0 && elect_one()) commit_pair(&pp.tfull[j & 1]);
      ++j;
    }
    // no MMA still runs, and no arrival is on its way, when the pair goes on
    if (rank == 0 && elect_one()) commit_pair(&pp.done);
    __syncwarp();
    tma::mbar_wait(&pp.done, 0, nullptr);
  } else {
    const int quarter = warp & 3, grp = (warp - 3) >> 2;
    uint32_t *buf32 = reinterpret_cast<uint32_t *>(tiles + kRingBytes + (warp - 3) * kDrainBytes);
    const int out_dtype = PARTS == kPartsF32 ? MOE_DT_F32 : a.out_dtype;
    const int M = KIND == kGroupedFwd ? a.n : a.k;
    const int64_t ld = KIND == kGroupedFwd ? a.ld_out : KIND == kGroupedDgrad ? a.ld_x : a.ld_w;
    int j = 0;
    for (int w = pair; w < work.total; w += pairs) {
      const Item it = work.item(w);
      const int m = it.m0 + rank * 128 + quarter * 32;
      const int64_t at = (KIND == kGroupedWgrad ? it.e * a.es_w : 0) + it.c0 * ld + m;
      const uint32_t lanes = pp.tmem_base + ((uint32_t)(32 * quarter) << 16);
      if (PARTS != kWhole && part_of(it.len) < it.len) {
        const int part = part_of(it.len);
        Sums<kTN / kTurnCols> sums;
        sums.zero();
        bool ok = true;
        for (int k0 = 0; k0 < it.len; k0 += part, ++j) {
          ok = pp.wait_warp(&pp.tfull[j & 1], (j >> 1) & 1);
          if (!ok) break;
          fence_after_sync();
          if (m < M) sums.add(lanes + (uint32_t)((j & 1) * kTN), it.nc, grp * 32);
          fence_before_sync();
          __syncwarp();
          if (lane == 0) arrive_at(&pp.tempty[j & 1], 0);
        }
        if (!ok) break;
        if (m < M) sums.store(it.nc, grp * 32, M - m, a.out, out_dtype, at, ld, buf32);
        continue;
      }
      const bool some = it.len > 0;
      const int buf = j & 1;
      if (some) {
        if (!pp.wait_warp(&pp.tfull[buf], (j >> 1) & 1)) break;
        fence_after_sync();
        ++j;
      }
      for (int c = grp * 32; c < it.nc && m < M; c += kTurnCols) {
        Sums<1> sums;
        sums.zero();
        if (some) sums.take(lanes + (uint32_t)(buf * kTN), it.nc, c);
        sums.store(it.nc, c, M - m, a.out, out_dtype, at, ld, buf32);
      }
      if (some) {
        fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_at(&pp.tempty[buf], 0);
      }
    }
  }
  __syncwarp();
  fence_before_sync();
  cluster_sync();
  if (threadIdx.x == 0 && pp.abort_flag) set_status(a.status, kStatusTimeout);
  if (warp == 1) tmem_dealloc_pair(pp.tmem_base, 2 * kTN);
}

template <int KIND, Parts PARTS>
cudaError_t launch_as(const Maps &maps, const GroupedArgs &a, int grid, cudaStream_t s) {
  const cudaError_t attr = cudaFuncSetAttribute(
      grouped_tc_kernel<KIND, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
  if (attr != cudaSuccess) return attr;
  grouped_tc_kernel<KIND, PARTS><<<grid, kThreads, kSmem, s>>>(maps, a);
  return cudaGetLastError();
}

template <int KIND>
cudaError_t launch_kind(const Maps &maps, const GroupedArgs &a, cudaStream_t s) {
  const long long nM = ((KIND == kGroupedFwd ? a.n : a.k) + kTM - 1) / kTM;
  const long long g = KIND == kGroupedWgrad ? (long long)a.E * ((a.n + kTN - 1) / kTN)
                                            : a.R / kTN + std::min(a.E, a.R);
  if (g * nM > INT32_MAX / 2) return cudaErrorInvalidValue;  // item numbers are 32-bit
  const int grid = 2 * (int)std::min<long long>(g * nM, a.sm_count / 2);
  const int longest = KIND == kGroupedFwd ? a.k : KIND == kGroupedDgrad ? a.n : a.R;
  if (longest <= sum_limit(a.out_dtype)) return launch_as<KIND, kWhole>(maps, a, grid, s);
  return a.out_dtype == MOE_DT_F32 ? launch_as<KIND, kPartsF32>(maps, a, grid, s)
                                   : launch_as<KIND, kPartsHalf>(maps, a, grid, s);
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
  Maps maps;
  const auto rows_map = [&](CUtensorMap *m, const void *t, int width, int64_t ld, int box) {
    return tc::encode_map3d(m, t, (uint64_t)width * 2, (uint64_t)a.R, 1, (uint64_t)ld * 2,
                            (uint64_t)ld * 2, (uint32_t)box);
  };
  bool ok = true;
  if (kind == kGroupedWgrad) {
    const int heights[4] = {kTK, 16, 4, 1};
    for (int i = 0; i < 4; ++i)
      ok = ok && rows_map(&maps.p[i], a.x, a.k, a.ld_x, heights[i]) &&
           rows_map(&maps.q[i], a.dout, a.n, a.ld_out, heights[i]);
  } else {
    const bool fwd = kind == kGroupedFwd;
    ok = tc::encode_map3d(&maps.p[0], a.w, (uint64_t)a.k * 2, (uint64_t)a.n, (uint64_t)a.E,
                          (uint64_t)a.ld_w * 2, (uint64_t)a.es_w * 2, fwd ? kTM / 2 : kTK);
    for (int i = 0; i < 3; ++i)
      ok = ok && rows_map(&maps.q[i], fwd ? a.x : a.dout, fwd ? a.k : a.n,
                          fwd ? a.ld_x : a.ld_out, 64 >> i);
  }
  if (!ok) return cudaErrorInvalidValue;
  maps.by_m = FastDiv(((kind == kGroupedFwd ? a.n : a.k) + kTM - 1) / kTM);
  maps.by_n = FastDiv((a.n + kTN - 1) / kTN);
  if (kind == kGroupedFwd) return launch_kind<kGroupedFwd>(maps, a, s);
  if (kind == kGroupedDgrad) return launch_kind<kGroupedDgrad>(maps, a, s);
  return launch_kind<kGroupedWgrad>(maps, a, s);
}

}  // namespace moe
