// Equal shares of a list of key chunks: the schedule of the split-K kernels over
// KV caches whose lengths are on the device.
//
// A schedule S has B sequences; sequence b holds S::chunks(b) chunks (all its KV
// heads and row tiles), in (sequence, head, tile, key) order.  The C chunks of
// all sequences form one list, and worker w of the first NW = min(the grid's, C)
// takes the contiguous range [w C / NW, (w + 1) C / NW): every worker reads the
// same number of chunks (to one), whatever the lengths, and none has an empty
// range.
#pragma once

#include "kf_common.h"

namespace kf {

__device__ __forceinline__ int wave_sum_int(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return __builtin_amdgcn_readfirstlane(v);
}

// Total chunks C (wavefront-uniform).
template <typename S>
__device__ __forceinline__ int total_chunks(const S& s, int lane) {
  int tot = 0;
  for (int b0 = 0; b0 < s.B; b0 += 64)
    tot += wave_sum_int(b0 + lane < s.B ? s.chunks(b0 + lane) : 0);
  return tot;
}

// Sequence holding chunk c of the list (0 <= c < C) and the index of its first
// chunk, the chunks of the sequences before it.  Wavefront-uniform.
template <typename S>
__device__ __forceinline__ void locate_chunk(const S& s, int c, int lane, int& b_out,
                                             int& base_out) {
  int run = 0;
  b_out = 0;
  base_out = 0;
  for (int b0 = 0; b0 < s.B; b0 += 64) {
    const int b = b0 + lane;
    const int n = b < s.B ? s.chunks(b) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(n > 0 && run + incl - n <= c && c < run + incl);
    if (m) {
      const int l = (int)__builtin_ctzll(m);
      b_out = b0 + l;
      base_out = run + __shfl(incl - n, l, 64);
      b_out = __builtin_amdgcn_readfirstlane(b_out);
      base_out = __builtin_amdgcn_readfirstlane(base_out);
      return;
    }
    run += __builtin_amdgcn_readfirstlane(__shfl(incl, 63, 64));
  }
}

// floor(x / d) for 0 <= x < 2^53 and 0 < d < 2^31: the double quotient is
// within one of the exact one (its relative error is below 2^-52 and x / d <
// 2^53), so one correction step either way makes it exact, in far fewer
// instructions than a 64-bit integer division.
__device__ __forceinline__ int64_t floor_div(int64_t x, int64_t d) {
  int64_t q = (int64_t)((double)x / (double)d);
  if (q * d > x)
    --q;
  else if ((q + 1) * d <= x)
    ++q;
  return q;
}

// First chunk of worker w's range, floor(w C / NW).
__device__ __forceinline__ int range_start(int w, int C, int NW) {
  return (int)floor_div((int64_t)w * C, NW);
}

// The worker whose range holds chunk c: the largest w with w C / NW <= c.
__device__ __forceinline__ int chunk_owner(int c, int C, int NW) {
  return (int)floor_div(((int64_t)c + 1) * NW - 1, C);
}

}  // namespace kf
