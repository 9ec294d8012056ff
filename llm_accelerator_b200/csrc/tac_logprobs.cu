// Log-probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits, in one read of the logits.
//
// With m the largest logit, d = x - m, S = sum e^d and T = sum e^d d:
//   log p(v) = (x_v - m) - ln S,   entropy = ln S - T / S,
// in which nothing cancels (all d <= 0).  A thread keeps (m, S, T) of what it
// has read about an m that its largest value may pass by kSlack, and rescales
// them when it does more; such triples join into one, about the row's largest.
//
// The k likeliest: k of the threads' largest values give a lower bound on the
// k-th largest logit (where a warp has the row and k is most of its lanes, k of
// the largest values of their stretches: 2000 x 5000 with k = 32 takes 19 us so,
// 116 with a bound that hundreds of values reach).  Only stretches whose largest
// value reaches the bound are read again, from L1 or L2, and what does is
// collected.  The few collected entries are placed by counting how many order
// before each.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/taccel_b200.h"
#include "tac_launch.cuh"
#include "tac_sm100.cuh"

namespace {

using namespace tac;

constexpr int kMostTop = 32, kMostCtas = 8;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct LpParams {
  const void* x;
  int64_t ld;
  const void* tokens;
  int tok64;
  int M, V, top;
  float* lp;
  float* entropy;
  float* top_lp;
  int32_t* top_ids;
};

// 16 bytes that will not be read again, or only a few of them
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 u;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}
__device__ __forceinline__ float ninf() { return __uint_as_float(0xff800000u); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {     // NaN where either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// Orders as the values do, NaN above all, -0 with 0; 0 orders below every value.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
constexpr uint32_t kLeastKey = ~0xff800000u;     // of -inf
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? (key == 0xffffffffu ? 0x7fc00000u : key ^ 0x80000000u) : ~key);
}
// Orders by value, then the lowest index first.
__device__ __forceinline__ uint64_t entry(uint32_t key, int64_t i) { return uint64_t(key) << 32 | (0xffffffffu - uint32_t(i)); }

struct Sums {
  float m, s, t;             // m -inf: nothing yet, s = t = 0
};
// The same sums about another m, at least their own: e^-200 is 0, and d stays finite.
__device__ __forceinline__ void about(Sums& a, float m) {
  const float d = a.m == ninf() ? 0.f : max_nan(a.m - m, -200.f), f = ex2(d * kLog2e);
  a.t = fmaf(d, a.s, a.t) * f;
  a.s *= f;
  a.m = m;
}
// The sums of neighbouring lanes, in all of them, about the largest of their `m`, which is no less than what theirs are about.
template <int LANES>
__device__ __forceinline__ Sums join(Sums a, float m) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  about(a, m);
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  return a;
}

// Pairs of float32 values in one register pair.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 of_pair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4, kLow = 0;   // values of 16 bytes, lowest bits of a key that say nothing
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return __ldg(static_cast<const float*>(p) + i); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ void values(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  template <int NV>
  static __device__ __forceinline__ float largest(const uint4 (&u)[NV]) {
    float m = __uint_as_float(u[0].x);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      m = max_nan(max_nan(m, __uint_as_float(u[i].x)), max_nan(max_nan(__uint_as_float(u[i].y), __uint_as_float(u[i].z)), __uint_as_float(u[i].w)));
    return m;
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8, kLow = 13;
  static __device__ __forceinline__ float one(const void* p, int64_t i) {
    return __half2float(__ushort_as_half(__ldg(static_cast<const uint16_t*>(p) + i)));
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ __half2 pair(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
  static __device__ __forceinline__ void values(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(pair(w[j]));
      v[2 * j] = f.x, v[2 * j + 1] = f.y;
    }
  }
  template <int NV>
  static __device__ __forceinline__ float largest(const uint4 (&u)[NV]) {
    __half2 m = pair(u[0].x);
#pragma unroll
    for (int i = 0; i < NV; ++i) m = __hmax2_nan(__hmax2_nan(m, pair(u[i].x)), __hmax2_nan(__hmax2_nan(pair(u[i].y), pair(u[i].z)), pair(u[i].w)));
    const float2 f = __half22float2(m);
    return max_nan(f.x, f.y);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8, kLow = 16;
  static __device__ __forceinline__ float one(const void* p, int64_t i) {
    return __uint_as_float(uint32_t(__ldg(static_cast<const uint16_t*>(p) + i)) << 16);
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ __nv_bfloat162 pair(uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); }
  static __device__ __forceinline__ void values(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
  template <int NV>
  static __device__ __forceinline__ float largest(const uint4 (&u)[NV]) {
    __nv_bfloat162 m = pair(u[0].x);
#pragma unroll
    for (int i = 0; i < NV; ++i) m = __hmax2_nan(__hmax2_nan(m, pair(u[i].x)), __hmax2_nan(__hmax2_nan(pair(u[i].y), pair(u[i].z)), pair(u[i].w)));
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&m);
    return max_nan(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
  }
};

// Adds the values of NV loads, `apart` from `from` on, to a thread's sums; the
// largest of them.  The sums stay
// about a value that the largest may pass by kSlack: they are rescaled a few
// times a row, not in every call.  What passes it costs precision: exponents of
// up to kSlack log2 e are rounded where the largest one's would be 0, and
// moving the sums takes kSlack S from a t of both signs.  Entropies of 4096 x
// 50257 BF16, a few logits of a row far above the rest, are off by 2.5e-7 (root
// of the mean square; at most 1.1e-6) with a slack of 4, 2 or none, by 3.1e-7
// (2.5e-6) with 8 and 9.8e-7 (6.7e-6) with 16; 77 us with each of them, and 888
// rows take 22.6 with none, 22.3 with 4, 22.1 with 16.  A value of
// -inf makes e^d d, and with it t, a NaN; and c is rounded by half its last
// place, which all terms' exponents share and e^-over makes good while it is 64
// at most, below kLargest (further on it can pass all exponents that float32
// has).  Otherwise, and in the rest of the row, each difference is taken, and
// lifted, by itself (2000 x 50257, one token in 64 unmasked in every third row:
// 43 us, 56 while each group of a row was tried first; 4096 x 50257 with -10^9
// for all but one token in 64 77 us, with -10^10, which some lanes of a warp
// meet first and others do not, 122).
// Eight values cost about 36 instructions and eight exponentials (16 a clock and
// SM): 46 us for 4096 x 50257, whose bytes take 63.
constexpr float kSlack = 4.f, kLargest = 2147483648.f;
template <typename T>
__device__ __forceinline__ void take_each(Sums& a, const uint4& u) {
  constexpr int N = Vec<T>::kN;
  float v[N];
  Vec<T>::values(u, v);
  const uint64_t minus_m = pair_of(-a.m, -a.m);
  uint64_t s = 0, t = 0;
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 dd = of_pair(add2(pair_of(v[j], v[j + 1]), minus_m));
    const float d0 = max_nan(dd.x, -200.f), d1 = max_nan(dd.y, -200.f);
    const uint64_t e = pair_of(ex2(d0 * kLog2e), ex2(d1 * kLog2e));
    s = add2(s, e);
    t = fma2(e, pair_of(d0, d1), t);
  }
  const float2 ss = of_pair(s), tt = of_pair(t);
  a.s += ss.x + ss.y;
  a.t += tt.x + tt.y;
}
template <typename T, int NV, bool HELD>
__device__ __forceinline__ float take(Sums& a, const uint4 (&u)[NV], const uint4* from, int apart, bool& by_each) {
  constexpr int N = Vec<T>::kN;
  const float m = Vec<T>::template largest<NV>(u);
  if (m == ninf()) {
    by_each = true;                              // a masked row: sooner than at its first value, which other lanes have elsewhere
    return m;
  }
  if (!(m <= a.m + kSlack)) about(a, max_nan(a.m, m));   // a NaN too
  if (by_each) {
#pragma unroll
    for (int i = 0; i < NV; ++i) take_each<T>(a, u[i]);
    return m;
  }
  // y = x log2 e - c with c = m log2 e rounded, which the same correction for all values makes good
  const float c = a.m * kLog2e, over = fmaf(a.m, kLog2e, -c);
  const uint64_t minus_c = pair_of(-c, -c), log2e = pair_of(kLog2e, kLog2e);
  uint64_t s = 0, t = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float v[N];
    Vec<T>::values(u[i], v);
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      const uint64_t y = fma2(pair_of(v[j], v[j + 1]), log2e, minus_c);
      const float2 yy = of_pair(y);
      const uint64_t e = pair_of(ex2(yy.x), ex2(yy.y));
      s = add2(s, e);
      t = fma2(e, y, t);
    }
  }
  const float2 ss = of_pair(s), tt = of_pair(t);
  const float s1 = ss.x + ss.y, t1 = tt.x + tt.y;
  if (fabsf(t1) < __uint_as_float(0x7f800000u) && fabsf(c) < kLargest) {
    const float f = ex2(-over);
    a.s = fmaf(s1, f, a.s);
    a.t = fmaf(fmaf(-over, s1, t1) * f, kLn2, a.t);
  } else {
    by_each = true;
#pragma unroll
    for (int i = 0; i < NV; ++i) take_each<T>(a, HELD ? u[i] : __ldg(from + i * apart));   // held, they cost the loop 16 registers
  }
  return m;
}

// One row's share: elements [e0, e1), of which whole aligned 16-byte pieces
// [c0, c1) are read by the threads in turn and what is left of either end one
// by one.
struct Share {
  const void* row;
  int64_t e0, e1, first;     // first: the element at which piece 0 begins
  int c0, c1;
};

// The thread's elements above `least` (all where it is NaN) and some others, each once: f(value, index); false ends it.
template <typename T, int NT, typename F>
__device__ __forceinline__ void each(const Share& s, float least, F f) {
  constexpr int N = Vec<T>::kN, kAtOnce = 4;
  const int64_t v0 = s.first + int64_t(s.c0) * N, v1 = s.first + int64_t(s.c1) * N;
  if (int64_t i = s.e0 + threadIdx.x; i < v0 && !f(Vec<T>::one(s.row, i), i)) return;
  if (int64_t i = v1 + threadIdx.x; i < s.e1 && !f(Vec<T>::one(s.row, i), i)) return;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(s.row) + s.first);
#pragma unroll 1
  for (int c = s.c0 + threadIdx.x; c < s.c1; c += kAtOnce * NT) {
    uint4 u[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) u[q] = c + q * NT < s.c1 ? __ldg(p + c + q * NT) : Vec<T>::none();
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      if (c + q * NT >= s.c1) return;
      if (Vec<T>::template largest<1>({u[q]}) <= least) continue;
      float v[N];
      Vec<T>::values(u[q], v);
      const int64_t i = s.first + int64_t(c + q * NT) * N;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!f(v[j], i + j)) return;
    }
  }
}

// Kept small: what shared memory takes of an SM is lost to the loads in flight,
// which land in L1 (4096 x 50257: 78 us with 92 KB an SM, 83 with 175, 97 with
// all that shared memory may have).
template <int NT>                      // threads of a row
struct LpShared {
  static constexpr int kWarps = NT / 32, kMostOfWarp = kMostTop / kWarps + 2;
  static constexpr int kRoom = 320;              // collected entries: all of a share that leaves a thread without any
  static constexpr int kSlots = NT == 256 ? 4 : NT == 128 ? 8 : 16;    // largest values that a thread keeps, of as many stretches of its pieces
  static constexpr int kList = 256;              // stretches that are read again
  uint64_t list[kMostTop];             // the share's k first, in order
  uint32_t bounds[kMostOfWarp * kWarps], bound;
  Sums warp_sums[kWarps];
  int count, stretches, found[kWarps];
  uint64_t best[kWarps];
  float largest[kSlots * NT];
  uint16_t stretch[kList];
  __align__(16) uint64_t room[kRoom];
};
struct LpParts {                       // of the CTAs of a cluster, in CTA 0
  __align__(16) uint64_t lists[kMostCtas * kMostTop];
  uint64_t joined[kMostTop];
  Sums sums[kMostCtas];
};

// A key that at least k of a warp's, and few more, reach: the largest there is unless exactly k reach a smaller one, found
// bit by bit.  key(i): the lane's of n times 32, at most kMost of them; kLow: how many of the lowest bits say nothing.
template <int kLow, int kMost, typename F>
__device__ __forceinline__ uint32_t reached_by(int k, int n, F key) {
  uint32_t q[kMost], least = 0;
#pragma unroll
  for (int i = 0; i < kMost; ++i) q[i] = i < n ? key(i) : 0u;
  for (int bit = 31; bit >= kLow; --bit) {
    const uint32_t t = least | 1u << bit;
    int count = 0;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < n) count += __popc(__ballot_sync(0xffffffffu, q[i] >= t));
    if (count >= k) least = t;
    if (count == k) break;
  }
  return least & 0x80000000u ? least : least | ((1u << kLow) - 1);      // of values below 0 those bits are set
}

// Places the n entries of `from` (16-byte aligned) that order among the first k into list[0 .. k).
template <int NT>
__device__ __forceinline__ void place(const uint64_t* from, int n, int k, uint64_t* list) {
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t e = from[i];
    int before = 0, j = 0;
#pragma unroll 4
    for (; j + 1 < n; j += 2) {
      const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(from + j);
      before += int(o.x > e) + int(o.y > e);
    }
    if (j < n) before += from[j] > e;
    if (e && before < k) list[before] = e;
  }
}

// The same for the n collected ones.  A warp that has many first leaves out those that cannot be among the k.
template <typename T, int NT>
__device__ __forceinline__ void place_room(LpShared<NT>& sm, int n, int k) {
  if constexpr (NT == 32) {
    const int lane = threadIdx.x;
    if (n > 64) {
      const uint32_t least = reached_by<Vec<T>::kLow, LpShared<NT>::kRoom / 32>(k, (n + 31) / 32, [&](int i) {
        return i * 32 + lane < n ? uint32_t(sm.room[i * 32 + lane] >> 32) : 0u;
      });
      int left = 0;
      for (int i = 0; i < n; i += 32) {
        const uint64_t e = i + lane < n ? sm.room[i + lane] : 0;
        const bool stays = uint32_t(e >> 32) >= least && i + lane < n;
        const uint32_t who = __ballot_sync(0xffffffffu, stays);
        __syncwarp();                            // read before one of them is written over
        if (stays) sm.room[left + __popc(who & ((1u << lane) - 1))] = e;
        left += __popc(who);
      }
      n = left;
      __syncwarp();
    }
  }
  place<NT>(sm.room, n, k, sm.list);
}

// An entry of key `least` or more to sm.room, while there is room; false once it is full.
template <int NT>
__device__ __forceinline__ bool keep(LpShared<NT>& sm, uint32_t least, float v, int64_t i) {
  const uint32_t key = key_of(v);
  if (key < least) return true;
  const int at = atomicAdd(&sm.count, 1);
  if (at < LpShared<NT>::kRoom) sm.room[at] = entry(key, i);
  return at < LpShared<NT>::kRoom;
}

// The bound is -inf, as in a row with fewer than k unmasked values, or more
// entries or stretches reach it than there is room for, as where many are equal:
// those above the bound, then of those at the bound the first, in the order of
// their indices.
template <typename T, int NT>
__device__ __noinline__ void first_k_rare(LpShared<NT>& sm, const Share& s, int k, uint32_t mine, bool any, uint32_t bound) {
  constexpr int kWarps = NT / 32, kRoom = LpShared<NT>::kRoom;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  if (threadIdx.x == 0) sm.count = 0;
  __syncthreads();
  if (bound != 0xffffffffu && any && mine > bound)
    each<T, NT>(s, value_of(bound), [&](float v, int64_t i) { return keep<NT>(sm, bound + 1, v, i); });
  __syncthreads();
  int n = sm.count;
  if (n <= kRoom) {
    place_room<T, NT>(sm, n, k);
    for (int64_t base = s.e0; n < k && base < s.e1; base += NT) {
      const int64_t i = base + threadIdx.x;
      const bool hit = i < s.e1 && key_of(Vec<T>::one(s.row, i)) == bound;
      const uint32_t who = __ballot_sync(0xffffffffu, hit);
      __syncthreads();                           // the last round's counts have been read
      if (lane == 0) sm.found[warp] = __popc(who);
      __syncthreads();
      int at = n + __popc(who & ((1u << lane) - 1));
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += sm.found[w];
        n += sm.found[w];
      }
      if (hit && at < k) sm.list[at] = entry(bound, i);
    }
    __syncthreads();
    return;
  }
  // Most of the largest values in few threads: one entry a pass.
  uint64_t last = ~0ull;
  for (int r = 0; r < k; ++r) {
    uint64_t best = 0;
    each<T, NT>(s, __uint_as_float(0x7fc00000u), [&](float v, int64_t i) {
      const uint64_t e = entry(key_of(v), i);
      if (e < last && e > best) best = e;
      return true;
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    __syncthreads();
    if (lane == 0) sm.best[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) best = max(best, sm.best[w]);
    if (threadIdx.x == 0) sm.list[r] = best;
    last = best;
    if (!best) break;                            // every thread's
  }
  __syncthreads();
}

// The share's k first entries to sm.list; largest: of the thread's elements, sm.largest: of its stretches of 2^log_stretch
// pieces each.
template <typename T, int NT>
__device__ __forceinline__ void first_k(LpShared<NT>& sm, const Share& s, int k, float largest, bool any, int slots, int log_stretch) {
  constexpr int N = Vec<T>::kN, kWarps = NT / 32, kRoom = LpShared<NT>::kRoom, kList = LpShared<NT>::kList;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t mine = any ? key_of(largest) : 0u;
  // The k-th of some threads' largest values is a bound: those of each warp's first few threads, at least k in all.
  const int each_warp = min(k, (k + kWarps - 1) / kWarps + 2), some = each_warp * kWarps;
  uint32_t q = mine, bound = 0;
  if (kWarps == 1 && k > 20) {                   // of 32 threads too low a bound: the largest values of their stretches
    bound = reached_by<Vec<T>::kLow, LpShared<NT>::kSlots>(k, slots, [&](int i) { return key_of(sm.largest[i * NT + lane]); });
  } else {
    for (int i = 0; i < each_warp; ++i) {
      bound = __reduce_max_sync(0xffffffffu, q);
      const uint32_t who = __ballot_sync(0xffffffffu, q == bound);
      if (lane == __ffs(who) - 1) {
        q = 0;
        if (kWarps > 1) sm.bounds[warp * each_warp + i] = bound;
      }
    }
  }
  if (threadIdx.x < kMostTop) sm.list[threadIdx.x] = 0;
  if (threadIdx.x == 0) sm.count = sm.stretches = 0;
  __syncthreads();
  if constexpr (kWarps > 1) {
    if (int(threadIdx.x) < some) {
      const uint32_t v = sm.bounds[threadIdx.x];
      int before = 0;
#pragma unroll 4
      for (int i = 0; i < some; i += kWarps) {
#pragma unroll
        for (int j = 0; j < kWarps; ++j) before += sm.bounds[i + j] > v || (sm.bounds[i + j] == v && i + j < int(threadIdx.x));
      }
      if (before == k - 1) sm.bound = v;
    }
    __syncthreads();
    bound = sm.bound;
  }
  // Fewer than k threads have more than -inf: what is above it, and of those at -inf the first.
  if (bound <= kLeastKey) return first_k_rare<T, NT>(sm, s, k, mine, any, kLeastKey);
  // What reaches the bound lies in a few stretches, which all threads read again together.
  const float low = value_of(bound);             // NaN where only NaN are first
  if (any && mine >= bound) {
    for (int i = 0; i < slots; ++i)
      if (!(sm.largest[i * NT + threadIdx.x] < low)) {
        const int at = atomicAdd(&sm.stretches, 1);
        if (at < kList) sm.stretch[at] = uint16_t(i * NT + threadIdx.x);
      }
    if (threadIdx.x < N) {                       // the ends
      const int64_t i = s.e0 + threadIdx.x, j = s.first + int64_t(s.c1) * N + threadIdx.x;
      if (i < s.first + int64_t(s.c0) * N) keep<NT>(sm, bound, Vec<T>::one(s.row, i), i);
      if (j < s.e1) keep<NT>(sm, bound, Vec<T>::one(s.row, j), j);
    }
  }
  __syncthreads();
  const int stretches = sm.stretches;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(s.row) + s.first);
  const int reread = min(stretches, kList) << log_stretch;
  auto piece = [&](int t) {
    const int of = sm.stretch[t >> log_stretch];
    return s.c0 + of % NT + ((of / NT << log_stretch) + (t & ((1 << log_stretch) - 1))) * NT;
  };
  if constexpr (kWarps == 1) {
    int count = sm.count;
    for (int t = lane; t - lane < reread && count <= kRoom; t += NT) {
      const int c = t < reread ? piece(t) : s.c1;
      const uint4 u = c < s.c1 ? __ldg(p + c) : Vec<T>::none();
      if (__all_sync(0xffffffffu, Vec<T>::template largest<1>({u}) < low)) continue;
      float v[N];
      Vec<T>::values(u, v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t key = key_of(v[j]), who = __ballot_sync(0xffffffffu, key >= bound);
        const int at = count + __popc(who & ((1u << lane) - 1));
        if (key >= bound && at < kRoom) sm.room[at] = entry(key, s.first + int64_t(c) * N + j);
        count += __popc(who);
      }
    }
    __syncwarp();
    if (lane == 0) sm.count = count;
  } else
  for (int t = threadIdx.x; t < reread; t += NT) {
    const int c = piece(t);
    if (c >= s.c1) continue;
    const uint4 u = __ldg(p + c);
    if (Vec<T>::template largest<1>({u}) < low) continue;
    if (*static_cast<volatile int*>(&sm.count) > kRoom) break;
    float v[N];
    Vec<T>::values(u, v);
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) hits |= uint32_t(!(v[j] < low)) << j;
    for (; hits; hits &= hits - 1) {
      const int j = __ffs(hits) - 1;
      float x = v[0];
#pragma unroll
      for (int q = 1; q < N; ++q) x = j == q ? v[q] : x;
      keep<NT>(sm, bound, x, s.first + int64_t(c) * N + j);
    }
  }
  __syncthreads();
  const int n = sm.count;
  if (n <= kRoom && stretches <= kList) {
    place_room<T, NT>(sm, n, k);
    __syncthreads();
    return;
  }
  first_k_rare<T, NT>(sm, s, k, mine, any, bound);
}

template <typename T, bool CLUSTER>
__device__ __forceinline__ Share share_of(const LpParams& p, int64_t row, int rank, int log_ctas) {
  Share s;
  s.row = static_cast<const T*>(p.x) + row * p.ld;
  const int64_t off = (16 - (reinterpret_cast<uintptr_t>(s.row) & 15)) & 15;
  s.first = min(int64_t(off / sizeof(T)), int64_t(p.V));
  const int pieces = int((p.V - s.first) / Vec<T>::kN);
  s.c0 = 0, s.c1 = pieces, s.e0 = 0, s.e1 = p.V;
  if (CLUSTER) {
    s.c0 = int(int64_t(pieces) * rank >> log_ctas), s.c1 = int(int64_t(pieces) * (rank + 1) >> log_ctas);
    if (rank) s.e0 = s.first + int64_t(s.c0) * Vec<T>::kN;
    if (rank + 1 != 1 << log_ctas) s.e1 = s.first + int64_t(s.c1) * Vec<T>::kN;
  }
  return s;
}

// NT threads a row, or a cluster of CTAs of 256 where there are few: CTA 0
// then joins the parts, which the others write into its shared memory.
constexpr int kAtOnce = 4;             // loads of a thread in flight

template <typename T, int NT, bool CLUSTER>
__global__ void __launch_bounds__(NT, CLUSTER ? 4 : NT == 32 ? 32 : 1536 / NT) logprobs_kernel(LpParams p, int log_ctas) {
  constexpr int N = Vec<T>::kN, kWarps = NT / 32;
  __shared__ LpShared<NT> sm;
  const int ctas = CLUSTER ? 1 << log_ctas : 1, rank = CLUSTER ? blockIdx.x & (ctas - 1) : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = CLUSTER ? blockIdx.x >> log_ctas : blockIdx.x;
  after_previous();
  let_next();
  if (CLUSTER) sm100::cluster_arrive();         // CTA 0's shared memory may be written once it runs
  const Share s = share_of<T, CLUSTER>(p, row, rank, log_ctas);
  float token_x = __uint_as_float(0x7fc00000u);  // a token outside the vocabulary has no probability
  if (rank == 0 && threadIdx.x == 0) {
    const int64_t tok = p.tok64 ? __ldg(static_cast<const int64_t*>(p.tokens) + row) : __ldg(static_cast<const int32_t*>(p.tokens) + row);
    if (tok >= 0 && tok < p.V) token_x = Vec<T>::one(s.row, tok);
  }
  // the ends, fewer than N elements each
  float v0 = ninf(), v1 = ninf();
  if (const int64_t i = s.e0 + threadIdx.x; i < s.first + int64_t(s.c0) * N) v0 = Vec<T>::one(s.row, i);
  if (const int64_t i = s.first + int64_t(s.c1) * N + threadIdx.x; i < s.e1) v1 = Vec<T>::one(s.row, i);

  Sums a{ninf(), 0.f, 0.f};
  bool by_each = false;
  const uint4* pieces = reinterpret_cast<const uint4*>(static_cast<const T*>(s.row) + s.first);
  // stretches of 2^log_stretch pieces a thread, at most kSlots of them
  const int groups = ((s.c1 - s.c0 + NT - 1) / NT + kAtOnce - 1) / kAtOnce;
  int log_groups = 0;
  while (groups > LpShared<NT>::kSlots << log_groups) ++log_groups;
  // a warp's short row: each piece
  const bool single = NT == 32 && s.c1 - s.c0 <= kAtOnce * NT;
  const int log_stretch = single ? 0 : log_groups + 2;
  const int slots = single ? (s.c1 - s.c0 + NT - 1) / NT : (groups + (1 << log_groups) - 1) >> log_groups;
  static_assert(kAtOnce == 4, "log_stretch");
  int c = s.c0 + threadIdx.x, group = 0;
  float most = ninf(), largest = ninf();         // of the stretch, of all
#pragma unroll 1
  for (; c + (kAtOnce - 1) * NT < s.c1; c += kAtOnce * NT) {
    uint4 u[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) u[i] = load_once(pieces + c + i * NT);
    most = max_nan(most, take<T, kAtOnce, CLUSTER>(a, u, pieces + c, NT, by_each));
    if (single) {
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) sm.largest[i * NT + threadIdx.x] = Vec<T>::template largest<1>({u[i]});
      ++group;
      largest = most;
    } else if ((++group & ((1 << log_groups) - 1)) == 0) {
      sm.largest[((group - 1) >> log_groups) * NT + threadIdx.x] = most;
      largest = max_nan(largest, most);
      most = ninf();
    }
  }
  {
    uint4 u[kAtOnce - 1][1];
#pragma unroll
    for (int i = 0; i < kAtOnce - 1; ++i) u[i][0] = c + i * NT < s.c1 ? load_once(pieces + c + i * NT) : Vec<T>::none();
#pragma unroll
    for (int i = 0; i < kAtOnce - 1; ++i) {
      const float of = c + i * NT < s.c1 ? take<T, 1, CLUSTER>(a, u[i], pieces + c + i * NT, 0, by_each) : ninf();
      if (single && group == 0 && i < slots) sm.largest[i * NT + threadIdx.x] = of;
      most = max_nan(most, of);
    }
    if (single && group == 0 && slots == kAtOnce) sm.largest[(kAtOnce - 1) * NT + threadIdx.x] = ninf();
    if (!single && group >> log_groups < slots) sm.largest[(group >> log_groups) * NT + threadIdx.x] = most;
    largest = max_nan(largest, most);
  }
  if (threadIdx.x < N) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x = i ? v1 : v0;
      if (x == ninf()) continue;
      about(a, max_nan(a.m, x));
      largest = max_nan(largest, x);
      const float d = max_nan(x - a.m, -200.f), e = ex2(d * kLog2e);
      a.s += e;
      a.t = fmaf(e, d, a.t);
    }
  }
  a = join<32>(a, largest);
  if (lane == 0) sm.warp_sums[warp] = a;
  if (p.top) {
    // has this thread any element?
    const bool any = s.c0 + int(threadIdx.x) < s.c1 || s.e0 + threadIdx.x < s.first + int64_t(s.c0) * N ||
                     s.first + int64_t(s.c1) * N + threadIdx.x < s.e1;
    first_k<T, NT>(sm, s, p.top, largest, any, slots, log_stretch);
  } else {
    __syncthreads();
  }
  if (!CLUSTER && warp) return;                  // one warp has lanes for all results
  Sums all = join<kWarps>(sm.warp_sums[lane % kWarps], sm.warp_sums[lane % kWarps].m);
  const uint64_t* list = sm.list;
  if constexpr (CLUSTER) {
    __shared__ LpParts parts;
    __syncwarp();
    sm100::cluster_wait();
    if (warp == 0) {
      if (lane < 3) {
        const float v = lane == 0 ? all.m : lane == 1 ? all.s : all.t;
        asm volatile("st.shared::cluster.f32 [%0], %1;\n" ::"r"(sm100::mapa_shared(&parts.sums[rank].m + lane, 0)), "f"(v) : "memory");
      }
    } else if (warp == 1 && lane < p.top) {
      asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(sm100::mapa_shared(&parts.lists[rank * p.top + lane], 0)), "l"(sm.list[lane])
                   : "memory");
    }
    __syncwarp();
    sm100::cluster_sync();
    if (rank != 0) return;
    all = lane % kMostCtas < ctas ? parts.sums[lane % kMostCtas] : Sums{ninf(), 0.f, 0.f};
    all = join<kMostCtas>(all, all.m);
    if (p.top) {
      place<NT>(parts.lists, ctas * p.top, p.top, parts.joined);
      list = parts.joined;
      __syncthreads();
    }
  }
  const float log_s = logf(all.s);
  if (threadIdx.x == 0) {
    p.lp[row] = (token_x - all.m) - log_s;
    p.entropy[row] = log_s - all.t / all.s;
  }
  if (int(threadIdx.x) < p.top) {
    const uint64_t e = list[threadIdx.x];
    p.top_lp[row * p.top + threadIdx.x] = (value_of(uint32_t(e >> 32)) - all.m) - log_s;
    p.top_ids[row * p.top + threadIdx.x] = int32_t(0xffffffffu - uint32_t(e));
  }
}

template <typename T, int NT, bool CLUSTER>
int launch_rows(const LpParams& p, int log_ctas, cudaStream_t st) {
  if ((int64_t(p.M) << log_ctas) > 0x7fffffff) return TAC_E_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.M) << log_ctas);
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1u << log_ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER ? 2 : 1;
  return status(cudaLaunchKernelEx(&cfg, logprobs_kernel<T, NT, CLUSTER>, p, log_ctas));
}

template <typename T>
int launch_logprobs(const LpParams& p, cudaStream_t st) {
  static int sms_of[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  if (!sms_of[dev]) {
    if (int e = status(cudaDeviceGetAttribute(&sms_of[dev], cudaDevAttrMultiProcessorCount, dev))) return e;
  }
  // CTAs a row, two, four or eight of 256 threads: while all run at once, four an SM, if each thread has 12 loads; with
  // fewer, for which picking tokens in more CTAs costs more than it gives, two while there are three an SM, four while there
  // are two and eight while there is one and no more than 20 are picked.  Microseconds in one, two, four, eight of them, 16-bit
  // logits, none / 32 picked:
  //    20 x 50257     5.9 /  9.5    4.8 /  8.3    4.0 /  8.1    4.3 / 10.6
  //    20 x 121000   11.3 / 15.1    7.4 / 11.3    5.3 /  9.3    4.7 / 11.1
  //   105 x 50257     6.8 / 10.3    6.0 /  9.7    6.1 / 11.1    9.2 / 21.7
  //   224 x 121000   20.6 / 25.1   15.9 / 21.0   17.4 / 26.9   24.0 / 43.7
  //    41 x 243278   31.3 / 37.1   17.6 / 22.4   11.2 / 16.0    9.6 / 17.4
  const int sms = sms_of[dev], pieces = p.V / Vec<T>::kN;
  const auto pays = [&](int log) {
    const int64_t ctas = int64_t(p.M) << log, loads = (pieces >> log) / 256;
    return loads >= 12 ? ctas <= 4 * sms : loads >= 4 && ctas <= (4 - log) * sms && (log < 3 || p.top <= 20);
  };
  int log_ctas = 0;
  while (2 << log_ctas <= kMostCtas && pays(log_ctas + 1)) ++log_ctas;
  // Four rows for some SMs and three for others: halves even that out where 16-bit logits are bound by their exponentials (500
  // x 121000 in 29 against 38 us with none picked, 35 against 43 with 20; 590 rows in 32 against 38).  Elsewhere rows in one
  // CTA each are faster: 400 x 121000 in 24.2 against 25.6 us, 660 in 38.2 against 39.0, float32 500 x 121000 in 45 against 46.
  if (sizeof(T) == 2 && !log_ctas && p.M > 3 * sms && p.M <= 4 * sms && pieces >= 2 * 24 * 256) log_ctas = 1;
  if (log_ctas) return launch_rows<T, 256, true>(p, log_ctas, st);
  // A warp a row, which needs no barrier, for short rows: those of two groups of loads, and where there are rows for many
  // warps an SM those of twelve (five, where no tokens are picked) unless many are picked, for which four warps have the
  // better bound.  Against four warps a row, microseconds with five tokens picked (with 20; with none), 16-bit logits:
  //   1000 x 1000  5.4 / 5.6   20000 x 1000  28 / 57   2000 x 2600  7.7 / 10.4 (10.9 / 11.8; 5.4 / 6.4), masked rows
  //   among them 9.2 / 11.3 (17.6 / 12.8)   1300 x 5000  9.6 / 9.0   4000 x 5000  16.8 / 20.4 (23.8 / 23.3; 14.3 / 14.1)
  //   4000 x 9000  24.1 / 25.5 (33.9 / 29.3; 21.9 / 18.7)   20000 x 12000  106 / 114   4096 x 50257  91 / 78
  const int most = p.M < 12 * sms || p.top > 8 ? 2 : p.top ? 12 : 5;
  if (pieces <= 32 * most * kAtOnce) return launch_rows<T, 32, false>(p, 0, st);
  // Eight warps a row while those of four would not fill the SMs: 400 x 50257 in 14.3 against 18.8 us, 888 x 50257 in 22.1
  // against 23.4 (4096 rows 81 against 78).
  if (p.M <= 6 * sms && pieces >= 4 * 256) return launch_rows<T, 256, false>(p, 0, st);
  return launch_rows<T, 128, false>(p, 0, st);
}

}  // namespace

extern "C" int tac_token_logprobs(const void* X, int type, int64_t ldx, const void* tokens, int tokens_64, int M, int V, int top,
                                  float* logprob, float* entropy, float* top_logprobs, int32_t* top_ids, void* stream) {
  const int e = type == TAC_F32 ? 4 : 2;
  auto aligned = [](const void* q, uintptr_t n) { return (reinterpret_cast<uintptr_t>(q) & (n - 1)) == 0; };
  if (!X || !tokens || !logprob || !entropy || (type != TAC_F32 && type != TAC_F16 && type != TAC_BF16) || M <= 0 || V <= 0 ||
      (M > 1 && ldx < V) || top < 0 || top > kMostTop || top > V || (top && (!top_logprobs || !top_ids)))
    return TAC_E_ARGUMENT;
  if (!aligned(X, e) || !aligned(tokens, tokens_64 ? 8 : 4) || !aligned(logprob, 4) || !aligned(entropy, 4) ||
      !aligned(top_logprobs, 4) || !aligned(top_ids, 4))
    return TAC_E_ARGUMENT;
  LpParams p{};
  p.x = X, p.ld = ldx;
  p.tokens = tokens, p.tok64 = tokens_64 != 0;
  p.M = M, p.V = V, p.top = top;
  p.lp = logprob, p.entropy = entropy, p.top_lp = top_logprobs, p.top_ids = top_ids;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (type == TAC_F32) return launch_logprobs<float>(p, st);
  if (type == TAC_F16) return launch_logprobs<__half>(p, st);
  return launch_logprobs<__nv_bfloat16>(p, st);
}
