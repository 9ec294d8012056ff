// 16-bit rows that begin anywhere: a warp whose lanes hold eight consecutive
// values each reads and writes them in aligned 16-byte accesses, in which a
// lane's eight are its own piece's end and its neighbour's beginning.  (Values
// one by one, 2 bytes a lane, took three times as long as aligned rows.)
#pragma once
#include <cstdint>

namespace tac {

// The eight values from place `by` (0..7, one for the whole warp) on of sixteen.
__device__ __forceinline__ uint4 eight_from(const uint4& a, const uint4& b, int by) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (by & 4) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (by & 2) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const uint32_t sel = by & 1 ? 0x5432 : 0x3210;
  return make_uint4(__byte_perm(w[0], w[1], sel), __byte_perm(w[1], w[2], sel), __byte_perm(w[2], w[3], sel), __byte_perm(w[3], w[4], sel));
}

__device__ __forceinline__ uint4 of_next_lane(const uint4& a) {
  return make_uint4(__shfl_down_sync(0xffffffffu, a.x, 1), __shfl_down_sync(0xffffffffu, a.y, 1), __shfl_down_sync(0xffffffffu, a.z, 1),
                    __shfl_down_sync(0xffffffffu, a.w, 1));
}

// Values [0, n) of the eight, zeros behind them.
__device__ __forceinline__ uint4 first_of(uint4 a, int n) {
  if (n >= 8) return a;
  auto word = [&](uint32_t w, int i) { return n >= i + 2 ? w : n == i + 1 ? w & 0xffffu : 0u; };
  return make_uint4(word(a.x, 0), word(a.y, 2), word(a.z, 4), word(a.w, 6));
}

// Whole warps: lane i has the eight values from p = (lane 0's) + 8 i on, of which the row still has `left` (also none or
// fewer); zeros for the rest.  Bytes beside the row are read only in 16-byte pieces that hold some of it.
__device__ __forceinline__ uint4 load8_any(const uint16_t* p, int left) {
  const int off = int(reinterpret_cast<uintptr_t>(p) >> 1) & 7;          // values from the aligned place to p
  const uint4* q = reinterpret_cast<const uint4*>(p - off);
  uint4 own = make_uint4(0, 0, 0, 0), last = own;
  if (left + off > 0) own = *q;                  // no read-only load: the row may be written by this kernel later
  if (off == 0) return first_of(own, left);
  if ((threadIdx.x & 31) == 31 && left > 8 - off) last = q[1];
  uint4 next = of_next_lane(own);
  if ((threadIdx.x & 31) == 31) next = last;
  return first_of(eight_from(own, next, off), left);
}

// The same places written; values from `left` on are not.
__device__ __forceinline__ void store8_any(uint16_t* p, const uint4& v, int left) {
  const int off = int(reinterpret_cast<uintptr_t>(p) >> 1) & 7, head = (8 - off) & 7, lane = threadIdx.x & 31;
  auto some = [](uint16_t* d, const uint4& a, int n) {                   // n < 8 of them
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 7; ++i)
      if (i < n) d[i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
  };
  const uint4 moved = off ? eight_from(v, of_next_lane(v), head) : v;
  const int n = lane == 31 && off ? min(8 - head, left - head) : left - head;    // the last lane's neighbour is another warp's
  if (n >= 8) *reinterpret_cast<uint4*>(p + head) = moved;
  else some(p + head, moved, n);
  if (lane == 0) some(p, v, min(head, left));
}

}  // namespace tac
