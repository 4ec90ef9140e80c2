// PTX wrappers of the tensor-core instructions (tcgen05), and, for the grouped
// products, their descriptors and the barriers of a persistent kernel with two
// copying warps, one issuing warp and kEpiWarps draining warps.
#pragma once

#include <cstdint>

#include "../../include/moe_b200.h"
#include "common.cuh"
#include "cvt.cuh"
#include "tma_ptx.cuh"

namespace moe {
namespace tcp {

using tma::su32;

__device__ __forceinline__ void tmem_alloc(uint32_t *dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   su32(dst_smem)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
// True for one lane of a converged warp, the same one each time.  The issuing
// code sits behind this rather than behind lane == 0: the tensor and copy
// instructions take uniform registers, and only here does the compiler know
// that a single lane runs them (measured: 107 cycles an MMA behind lane == 0).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void fence_after_sync() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_before_sync() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
// Arrives on bar once every MMA and copy this thread issued has completed.
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          su32(bar))
      : "memory");
}
// D (+)= (A sA) (B sB)^T of E2M1 operands with an E8M0 scale for 32 elements of
// K, fp32 sums; 64 elements of K.  sfa / sfb: TMEM columns of the scales.
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, "
      "[%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// 32 rows of 16 bytes of shared memory into 4 TMEM columns, the same in each
// quarter of the lanes; ordered before later MMAs of this thread.
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t sdesc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc)
               : "memory");
}
// 32 accumulator columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]),
        "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Shared-memory matrix descriptor (version 1) of a 128-byte swizzled operand.
//   K-major:  8-row x 128-byte atoms, `sbo` bytes apart along M or N; lbo unused.
//   MN-major: 128 bytes of M or N by 8 rows of K an atom, `sbo` bytes apart
//             along K and `lbo` bytes apart along M or N.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) |
         ((uint64_t)(sbo >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Descriptor of 32 rows of 16 bytes back to back (no swizzle): groups of 8 rows
// 128 bytes apart.
__device__ __forceinline__ uint64_t rows16_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}


// Warps: 0 copies the M side, 1 issues the MMAs, 2 copies the N side (a copy
// takes 60 to 70 cycles to issue, and one warp for both was the bound), and
// then, behind any others of a kernel, the draining warps.
constexpr int kEpiWarps = 16;  // four a TMEM lane quarter
constexpr int kThreads = 96 + 32 * kEpiWarps;

// A position in a ring of `stages`: the stage, and how often the ring went round.
struct Ring {
  int stages, s = 0;
  uint32_t use = 0;
  __device__ __forceinline__ explicit Ring(int n) : stages(n) {}
  __device__ __forceinline__ void next() {
    if (++s == stages) {
      s = 0;
      ++use;
    }
  }
};

// S: the most stages that a ring may have.
template <int S>
struct Pipe {
  uint64_t full[S], empty[S];  // stages of the shared-memory ring
  uint64_t tfull[2], tempty[2];  // accumulator buffers
  uint64_t done;                 // every MMA of this CTA has completed
  uint32_t tmem_base;
  int abort_flag;

  __device__ __forceinline__ void init(uint32_t full_count, uint32_t tempty_count = kEpiWarps) {
    for (int s = 0; s < S; ++s) {
      tma::mbar_init(&full[s], full_count);
      tma::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tma::mbar_init(&tfull[b], 1);
      tma::mbar_init(&tempty[b], tempty_count);
    }
    tma::mbar_init(&done, 1);
    abort_flag = 0;
    tma::fence_mbar_init();
  }
  // After an abort: the copies in flight land before the CTA may exit (a bounded
  // wait for the last use of each stage).
  __device__ __forceinline__ void drain(const Ring &r) {
    for (int s = 0; s < r.stages; ++s) {
      const uint32_t uses = r.use + (s < r.s ? 1 : 0);
      if (uses) tma::mbar_wait(&full[s], (uses - 1) & 1, nullptr, tma::kWaitCycles / 64);
    }
  }
  // A whole warp's bounded wait; false (for every lane) once any role gave up.
  __device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, tma::mbar_try(bar, parity))) return true;  // the usual case
    const bool ok = tma::mbar_wait(bar, parity, &abort_flag);
    if (__all_sync(0xffffffffu, ok)) return true;
    abort_flag = 1;
    return false;
  }
};

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
  return reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// The epilogue of a tile: column c of the accumulator is row c of the result,
// and lane l of a quarter its element m + l.  A warp's 32 lanes would store 64
// bytes of a 16-bit row at a time (measured: 14 cycles a store, the bound of
// wgrad), so 16 columns (8 of an fp32 result) at a time go through 1 KB of shared
// memory of the warp's own and leave as 16 bytes a lane, whole sectors of 8
// rows (4) a store.  16-bit values go as pairs of columns, one word a lane, and
// are parted on the way out.
constexpr int kDrainBytes = 1024;  // of shared memory, for each draining warp

// 8 (4 of fp32) elements of a row, of which the first `left` are inside it.
template <typename T>
__device__ __forceinline__ void store_piece(T *p, uint4 v, int left) {
  constexpr int kN = 16 / sizeof(T);
  if (left >= kN) {
    *reinterpret_cast<uint4 *>(p) = v;
  } else {
    const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (i < left) p[i] = e[i];
  }
}

// Columns c .. c + 31 of the accumulator (v), row c of the result at out; the
// warp's elements of a row start at out and `left` of its 32 are inside.
template <typename T>
__device__ __forceinline__ void store_cols(T *out, int64_t ld, int nc, int left, bool vec,
                                           uint32_t *buf, const uint32_t (&v)[32]) {
  const int lane = threadIdx.x & 31;
  if (!vec) {  // rows that do not start on 16 bytes: a lane's own element of each
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (i < nc && lane < left) out[i * ld + lane] = from_f32<T>(__uint_as_float(v[i]));
    __syncwarp();
    return;
  }
  const bool whole = nc >= 32 && left >= 32;  // nothing to leave out
  if constexpr (sizeof(T) == 2) {
    const int p = lane / 4, m = lane % 4 * 8;
    T *row = out + 2 * p * ld + m;
#pragma unroll
    for (int h = 0; h < 2; ++h, row += 16 * ld) {
      if (16 * h >= nc) break;  // warp-uniform
#pragma unroll
      for (int i = 0; i < 8; ++i)
        buf[i * 32 + lane] = pack2(__uint_as_float(v[16 * h + 2 * i]),
                                   __uint_as_float(v[16 * h + 2 * i + 1]), T{});
      __syncwarp();
      const uint4 a = *reinterpret_cast<const uint4 *>(buf + p * 32 + m);
      const uint4 b = *reinterpret_cast<const uint4 *>(buf + p * 32 + m + 4);
      const uint4 lo =
          make_uint4(__byte_perm(a.x, a.y, 0x5410), __byte_perm(a.z, a.w, 0x5410),
                     __byte_perm(b.x, b.y, 0x5410), __byte_perm(b.z, b.w, 0x5410));
      const uint4 hi =
          make_uint4(__byte_perm(a.x, a.y, 0x7632), __byte_perm(a.z, a.w, 0x7632),
                     __byte_perm(b.x, b.y, 0x7632), __byte_perm(b.z, b.w, 0x7632));
      if (whole) {
        *reinterpret_cast<uint4 *>(row) = lo;
        *reinterpret_cast<uint4 *>(row + ld) = hi;
      } else {
        const int i = 16 * h + 2 * p;
        if (i < nc) store_piece(row, lo, left - m);
        if (i + 1 < nc) store_piece(row + ld, hi, left - m);
      }
      __syncwarp();
    }
  } else {
    const int r = lane / 8, m = lane % 8 * 4;
    T *row = out + r * ld + m;
#pragma unroll
    for (int h = 0; h < 4; ++h, row += 8 * ld) {
      if (8 * h >= nc) break;  // warp-uniform
#pragma unroll
      for (int i = 0; i < 8; ++i) buf[i * 32 + lane] = v[8 * h + i];
      __syncwarp();
      const uint4 lo = *reinterpret_cast<const uint4 *>(buf + r * 32 + m);
      const uint4 hi = *reinterpret_cast<const uint4 *>(buf + (r + 4) * 32 + m);
      if (whole) {
        *reinterpret_cast<uint4 *>(row) = lo;
        *reinterpret_cast<uint4 *>(row + 4 * ld) = hi;
      } else {
        if (8 * h + r < nc) store_piece(row, lo, left - m);
        if (8 * h + r + 4 < nc) store_piece(row + 4 * ld, hi, left - m);
      }
      __syncwarp();
    }
  }
}

// What a draining warp holds of a tile: the four groups of warps take its columns
// in turns of 32, of which it holds kTurns.
constexpr int kTurnCols = kEpiWarps / 4 * 32;
template <int kTurns>
struct Sums {
  uint32_t v[kTurns][32];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int t = 0; t < kTurns; ++t)
#pragma unroll
      for (int i = 0; i < 32; ++i) v[t][i] = 0;
  }
  // Columns c0 .. c0 + 31 and so on out of TMEM.
  __device__ __forceinline__ void take(uint32_t trow, int nc, int c0) {
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int c = c0 + t * kTurnCols;
      if (c >= nc) break;  // warp-uniform
      tmem_ld32(trow + c, v[t]);
    }
    tmem_wait_ld();
  }
  // The same, added to what is held.
  __device__ __forceinline__ void add(uint32_t trow, int nc, int c0) {
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int c = c0 + t * kTurnCols;
      if (c >= nc) break;  // warp-uniform
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t u[16];
        tmem_ld16(trow + c + 16 * h, u);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i)
          v[t][16 * h + i] =
              __float_as_uint(__uint_as_float(v[t][16 * h + i]) + __uint_as_float(u[i]));
      }
    }
  }
  // at: the offset of the tile's element (row 0, m0 + 32 quarter).
  __device__ __forceinline__ void store(int nc, int c0, int left, void *out, int out_dtype,
                                        int64_t at, int64_t ld, uint32_t *buf) const {
    const int size = out_dtype == MOE_DT_F32 ? 4 : 2;
    const bool vec = (((uintptr_t)out + at * size) & 15) == 0 && ((ld * size) & 15) == 0;
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const int c = c0 + t * kTurnCols;
      if (c >= nc) break;  // warp-uniform
      if (out_dtype == MOE_DT_F32)
        store_cols(reinterpret_cast<float *>(out) + at + c * ld, ld, nc - c, left, vec, buf, v[t]);
      else if (out_dtype == MOE_DT_BF16)
        store_cols(reinterpret_cast<__nv_bfloat16 *>(out) + at + c * ld, ld, nc - c, left, vec,
                   buf, v[t]);
      else
        store_cols(reinterpret_cast<__half *>(out) + at + c * ld, ld, nc - c, left, vec, buf, v[t]);
    }
  }
};

// ---- pairs of CTAs (clusters of two, cta_group::2) ---------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}
// Arrives on the barrier at the same place in CTA `rank` of the cluster.  What it
// tells of is copies and tensor memory, which their own mechanisms order, never
// plain stores (release and acquire at cluster scope on every step made the pair
// kernel 2.5 times slower).
__device__ __forceinline__ void arrive_at(uint64_t *bar, uint32_t rank) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %0, %1;\n\t"
      "mbarrier.arrive.shared::cluster.b64 _, [a];\n\t}" ::"r"(su32(bar)),
      "r"(rank)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t *dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   su32(dst_smem)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}
// As commit, on the barrier at the same place in both CTAs of the pair.
__device__ __forceinline__ void commit_pair(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
      "[%0], %1;" ::"r"(su32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// D (+)= A B^T of f16 or bf16 operands, fp32 sums; 16 elements of K, M = 256 over the
// pair: each CTA's shared memory holds its 128 rows of A and its half of the rows of
// B, at the same places, and its TMEM 128 rows of D.
__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

}  // namespace tcp
}  // namespace moe
