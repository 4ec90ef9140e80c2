// PTX wrappers of the tensor-core instructions (tcgen05) that the grouped
// products use, their descriptors, and the barriers of a persistent kernel
// with one copying thread, one issuing warp and kEpiWarps draining warps.
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
// D (+)= A B^T of f16 or bf16 operands, fp32 sums; 16 elements of K.
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
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

constexpr int kEpiWarps = 8;                   // two a TMEM lane quarter
constexpr int kThreads = 64 + 32 * kEpiWarps;  // and the copying and issuing warps

template <int S>
struct Pipe {
  uint64_t full[S], empty[S];  // stages of the shared-memory ring
  uint64_t tfull[2], tempty[2];  // accumulator buffers
  uint64_t done;                 // every MMA of this CTA has completed
  uint32_t tmem_base;
  int abort_flag;
  int consumed;  // stages that the issuing warp has taken

  __device__ __forceinline__ void init(uint32_t full_count) {
    for (int s = 0; s < S; ++s) {
      tma::mbar_init(&full[s], full_count);
      tma::mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tma::mbar_init(&tfull[b], 1);
      tma::mbar_init(&tempty[b], kEpiWarps);
    }
    tma::mbar_init(&done, 1);
    abort_flag = 0;
    consumed = 0;
    tma::fence_mbar_init();
  }
  // A whole warp's bounded wait; false (for every lane) once any role gave up.
  __device__ __forceinline__ bool wait_warp(uint64_t *bar, uint32_t parity) {
    const bool ok = tma::mbar_wait(bar, parity, &abort_flag);
    if (__all_sync(0xffffffffu, ok)) return true;
    abort_flag = 1;
    return false;
  }
};

__device__ __forceinline__ uint8_t *align1024(uint8_t *p) {
  return reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(p) + 1023) & ~uintptr_t(1023));
}

// Writes a tile's sums: column c of the accumulator is row c of the result,
// and lane l of a quarter its element m0 + l.  Called by the 8 draining warps,
// grp the half of the columns (in turns of 32) that this warp takes.
template <typename T>
__device__ __forceinline__ void store_cols(T *out, int64_t ld, int c, int nc,
                                           const uint32_t (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (c + i < nc) out[(c + i) * ld] = from_f32<T>(__uint_as_float(v[i]));
}
__device__ __forceinline__ void drain_tile(uint32_t trow, bool some, int nc, int grp, bool inside,
                                           void *out, int out_dtype, int64_t at, int64_t ld) {
  for (int c = grp * 32; c < nc; c += 64) {
    uint32_t v[32];
    if (some) {
      tmem_ld32(trow + c, v);
      tmem_wait_ld();
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0;
    }
    if (inside) {
      if (out_dtype == MOE_DT_F32) store_cols(reinterpret_cast<float *>(out) + at, ld, c, nc, v);
      else if (out_dtype == MOE_DT_BF16)
        store_cols(reinterpret_cast<__nv_bfloat16 *>(out) + at, ld, c, nc, v);
      else store_cols(reinterpret_cast<__half *>(out) + at, ld, c, nc, v);
    }
    __syncwarp();  // the next load is the whole warp's
  }
}

// Rows of the t-th of nt row tiles of an expert with cnt rows: equal tiles, a
// multiple of 16 (the MMA's step of N), so that 300 rows become 160 + 140
// rather than 256 + 44.  No tile is empty: nt is ceil(cnt / (a multiple of 16)).
__device__ __forceinline__ int tile_rows(int cnt, int nt) {
  return ((cnt + nt - 1) / nt + 15) & ~15;
}

}  // namespace tcp
}  // namespace moe
