// Rows that begin anywhere, counted in 16-bit values: a warp whose lanes hold
// eight consecutive ones each reads and writes them in aligned 16-byte accesses,
// in which a lane's eight are its own piece's end and its neighbour's beginning.
// Rows of float32 are such rows of two values each.  (One value a lane and load
// took three times as long as aligned rows.)
#pragma once
#include <cstdint>
#include <type_traits>

namespace tac {

// Values [0, n) of the eight, zeros behind them.
__device__ __forceinline__ uint4 first_of(uint4 a, int n) {
  if (n >= 8) return a;
  auto word = [&](uint32_t w, int i) { return n >= i + 2 ? w : n == i + 1 ? w & 0xffffu : 0u; };
  return make_uint4(word(a.x, 0), word(a.y, 2), word(a.z, 4), word(a.w, 6));
}

// Whole warps: `chunks` (at most CH) times 32 lanes of eight values from p on, lane i of chunk c at p + 256 c + 8 i, of which
// the row still has `left` (also none).  Reading is split, so that many loads are under way before the first is waited for:
// load() takes the aligned pieces that the chunks begin in, and the one in which the last of them ends; values() gives the
// eight of each lane, zeros behind the row.  Bytes beside the row are read only in pieces that hold some of it, and of a
// piece that two warps share each uses its own values, so that other warps may write theirs meanwhile.
template <int CH>
struct AnySpan {
  uint4 v[CH], tail;
  int off;                             // values from the aligned place to p

  // Places 2 S + odd to 2 S + odd + 7 of a lane's eight and those behind them, which are the next lane's, or the next chunk's.
  template <int S>
  __device__ __forceinline__ uint4 behind(int c, int chunks, uint32_t odd) const {
    const uint4 over = c + 1 < CH && c + 1 < chunks ? v[c + 1 < CH ? c + 1 : c] : tail;
    const bool first = (threadIdx.x & 31) == 0;
    const int from = (threadIdx.x + 1) & 31;
    uint32_t w[8] = {v[c].x, v[c].y, v[c].z, v[c].w};
    w[4] = __shfl_sync(0xffffffffu, first ? over.x : v[c].x, from);
    if (S >= 1) w[5] = __shfl_sync(0xffffffffu, first ? over.y : v[c].y, from);
    if (S >= 2) w[6] = __shfl_sync(0xffffffffu, first ? over.z : v[c].z, from);
    if (S >= 3) w[7] = __shfl_sync(0xffffffffu, first ? over.w : v[c].w, from);
    const uint32_t sel = odd ? 0x5432 : 0x3210;
    return make_uint4(__byte_perm(w[S], w[S + 1], sel), __byte_perm(w[S + 1], w[S + 2], sel), __byte_perm(w[S + 2], w[S + 3], sel),
                      __byte_perm(w[S + 3], w[S + 4], sel));
  }
  // f(integral constant S) for places from `by` (0..7, the warp's) on
  template <typename F>
  __device__ __forceinline__ static void shifted(int by, F f) {
    switch (by >> 1) {
      case 0: return f(std::integral_constant<int, 0>());
      case 1: return f(std::integral_constant<int, 1>());
      case 2: return f(std::integral_constant<int, 2>());
      default: return f(std::integral_constant<int, 3>());
    }
  }
  __device__ __forceinline__ void load(const uint16_t* p, int chunks, int left) {
    const int lane = threadIdx.x & 31;
    off = int(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
    const uint4* q = reinterpret_cast<const uint4*>(p - off) + lane;     // no read-only loads: the row may be written later
#pragma unroll
    for (int c = 0; c < CH; ++c) v[c] = c < chunks && left + off > 256 * c + 8 * lane ? q[32 * c] : make_uint4(0, 0, 0, 0);
    tail = lane == 0 && off && left + off > 256 * chunks ? q[32 * chunks] : make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(int chunks, int left) {
    if (off) {
      shifted(off, [&](auto by) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (c < chunks) v[c] = behind<by.value>(c, chunks, off & 1);   // v[c + 1] is still as it was read
      });
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (left < 256 * (c + 1)) v[c] = first_of(v[c], left - 256 * c - 8 * int(threadIdx.x & 31));
  }
  // The lanes' values to such places; those from `left` on are not written.
  __device__ __forceinline__ void store(uint16_t* p, int chunks, int left) {
    const int lane = threadIdx.x & 31;
    off = int(reinterpret_cast<uintptr_t>(p) >> 1) & 7;
    const int head = (8 - off) & 7;
    auto some = [](uint16_t* d, const uint4& a, int n) {                 // n < 8 of them
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 7; ++i)
        if (i < n) d[i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
    };
    tail = make_uint4(0, 0, 0, 0);               // another warp's
    shifted(head, [&](auto by) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (c >= chunks) break;
        uint16_t* d = p + 256 * c + 8 * lane + head;
        const uint4 moved = off ? behind<by.value>(c, chunks, head & 1) : v[c];
        int n = left - 256 * c - 8 * lane - head;
        if (off && lane == 31 && c + 1 == chunks) n = min(n, 8 - head);
        if (n >= 8) *reinterpret_cast<uint4*>(d) = moved;
        else some(d, moved, n);
      }
    });
    if (lane == 0) some(p, v[0], min(head, left));
  }
};

}  // namespace tac
