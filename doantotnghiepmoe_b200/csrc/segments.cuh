// The row segments of a by-expert permutation as work items of the grouped
// products: expert e owns rows [seg_off[e], seg_off[e + 1]).
//
// The offsets are device data that a caller may have got wrong, so the table
// holds them clamped into [0, R] and made non-decreasing (each such change
// sets kStatusBadRoute): no product reads or writes outside its R rows.
#pragma once

#include "common.cuh"

namespace moe {

struct SegTable {
  int32_t off[kMaxExperts + 1];
  int32_t tile0[kMaxExperts + 1];  // row tiles of the experts before e
  int32_t total;                   // row tiles of all experts
  int32_t most;                    // no tile has more rows

  int32_t size[kMaxExperts];       // rows of an expert's tiles (the last may have fewer)

  __device__ __forceinline__ int rows(int e) const { return off[e + 1] - off[e]; }

  // Expert of row tile g < total: the last e with tile0[e] <= g, which has rows.
  // Called by a whole warp: 32 experts eight apart, then the eight between.
  __device__ __forceinline__ int expert_of(int g, int E) const {
    const int lane = threadIdx.x & 31;
    const int a = lane * 8;
    const int hi = __popc(__ballot_sync(0xffffffffu, a < E && tile0[min(a, E)] <= g)) - 1;
    const int b = hi * 8 + (lane & 7);
    const uint32_t in = __ballot_sync(0xffffffffu, b < E && tile0[min(b, E)] <= g);
    return hi * 8 + __popc(in & 0xffu) - 1;
  }
};

// Division of 0 <= w < 2^31 by a number known on the host: w d rounded down is
// w m / 2^s with m = 2^s / d rounded up, s = 31 + ceil(log2 d).
struct FastDiv {
  uint32_t mul;
  int shift;
  __host__ explicit FastDiv(int d = 1) {
    int l = 0;
    while ((1ll << l) < d) ++l;
    shift = 31 + l;
    mul = (uint32_t)(((1ull << shift) + d - 1) / (uint64_t)d);
  }
  __device__ __forceinline__ int div(int w) const {
    return (int)(((uint64_t)(uint32_t)w * mul) >> shift);
  }
};

// Fills the table; called by one whole warp, before a block barrier.  Lane l
// handles experts 8 l .. 8 l + 7 and the running maximum and the tile counts
// are joined by warp scans.  bn: the most rows of a tile.
//
// An expert's tiles are equal, a multiple of `step` rows (that of the MMA's N), so
// that 300 rows in tiles of 256 at most become 160 + 140 rather than 256 + 44.
// None is empty: with nt = ceil(rows / bn) tiles and bn at least 8 steps, nt - 1
// tiles of rows / nt + step rows never cover the rows, and from 8 tiles on the
// size is bn.
__device__ __forceinline__ void build_segments(SegTable &t, const int32_t *seg_off, int E, int R,
                                               int bn, int step, uint32_t *status) {
  constexpr int kPer = kMaxExperts / 32;
  const int lane = threadIdx.x & 31;
  const int first = seg_off[0];
  int raw[kPer], v[kPer];
  bool bad = first < 0 || first > R;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane * kPer + j;
    raw[j] = e < E ? seg_off[e + 1] : 0;
  }
  int run = min(max(first, 0), R);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    run = max(run, min(max(raw[j], 0), R));
    v[j] = run;
  }
  int top = run;  // inclusive maximum over the lanes so far
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, top, d);
    if (lane >= d) top = max(top, o);
  }
  int prev = __shfl_up_sync(0xffffffffu, top, 1);
  if (lane == 0) prev = min(max(first, 0), R);
  int tiles = 0, most = 0, off0[kPer], t0[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane * kPer + j;
    v[j] = max(v[j], prev);
    off0[j] = j ? v[j - 1] : prev;
    t0[j] = tiles;
    if (e < E) {
      bad |= raw[j] != v[j];
      tiles += (v[j] - off0[j] + bn - 1) / bn;
      most = max(most, v[j] - off0[j]);
    }
  }
  int sum = tiles;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += o;
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane * kPer + j;
    if (e < E) {
      t.off[e] = off0[j];
      const int nt = j + 1 < kPer ? t0[j + 1] - t0[j] : tiles - t0[j];
      const int cnt = v[j] - off0[j], each = nt > 1 ? (cnt + nt - 1) / nt : cnt;
      t.size[e] = (each + step - 1) / step * step;
      t.tile0[e] = sum - tiles + t0[j];
      if (e == E - 1) t.off[E] = v[j];
    }
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 31) {
    t.total = t.tile0[E] = sum;
    t.most = min(most, bn);
  }
  if (bad) set_status(status, kStatusBadRoute);
}

}  // namespace moe
