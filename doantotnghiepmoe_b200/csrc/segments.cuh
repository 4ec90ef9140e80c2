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

  __device__ __forceinline__ int rows(int e) const { return off[e + 1] - off[e]; }

  // Expert of row tile g < total: the last e with tile0[e] <= g that has rows.
  __device__ __forceinline__ int expert_of(int g, int E) const {
    int lo = 0, hi = E;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (tile0[mid] <= g) lo = mid;
      else hi = mid;
    }
    return lo;
  }
};

// Fills the table; called by one whole warp, before a block barrier.  Lane l
// handles experts 8 l .. 8 l + 7 and the running maximum and the tile counts
// are joined by warp scans.  bn: the most rows of a tile.
__device__ __forceinline__ void build_segments(SegTable &t, const int32_t *seg_off, int E, int R,
                                               int bn, uint32_t *status) {
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
