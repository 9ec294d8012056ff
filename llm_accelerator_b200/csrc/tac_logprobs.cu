// Log-probabilities of given tokens, the entropy and the likeliest tokens of
// rows of logits, in one read of the logits.
//
// With m the largest logit, d = (x - m) log2 e, S = sum 2^d and T = sum 2^d d:
//   log p(v) = (x_v - m) - ln S,   entropy = ln S - ln 2 * T / S,
// in which nothing cancels (all d <= 0).  A thread keeps (m, S, T) of what it
// has read, rescaled as its m grows; two such triples join into one.
//
// The k likeliest: k of the threads' largest values give a lower bound on the
// k-th largest logit, so only threads whose largest value reaches the bound
// read their share again (from L1 or L2) and collect what does.  The few
// collected entries are placed by counting how many order before each.
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

constexpr int kThreads = 256, kWarps = kThreads / 32, kMostTop = 32, kMostCtas = 8;
constexpr int kRoom = kThreads * 8 + 64;   // collected entries: all of a share that leaves a thread without any
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
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? (key == 0xffffffffu ? 0x7fc00000u : key ^ 0x80000000u) : ~key);
}
// Orders by value, then the lowest index first.
__device__ __forceinline__ uint64_t entry(uint32_t key, int64_t i) { return uint64_t(key) << 32 | (0xffffffffu - uint32_t(i)); }

struct Sums {
  float m, s, t;             // m -inf: nothing yet, s = t = 0
};
__device__ __forceinline__ void add_scaled(Sums& a, float m, float s, float t) {
  if (m == ninf()) return;
  const float d = max_nan((m - a.m) * kLog2e, -200.f), f = ex2(d);   // -200: 2^d is 0, and d stays finite
  a.s = fmaf(s, f, a.s);
  a.t = fmaf(fmaf(d, s, t), f, a.t);
}
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  Sums r{max_nan(a.m, b.m), 0.f, 0.f};
  add_scaled(r, a.m, a.s, a.t);
  add_scaled(r, b.m, b.s, b.t);
  return r;
}

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  static __device__ __forceinline__ float one(const void* p, int64_t i) { return __ldg(static_cast<const float*>(p) + i); }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ void values(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ float largest(const uint4& u) {
    return max_nan(max_nan(__uint_as_float(u.x), __uint_as_float(u.y)), max_nan(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
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
  static __device__ __forceinline__ float largest(const uint4& u) {
    const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(pair(u.x), pair(u.y)), __hmax2_nan(pair(u.z), pair(u.w))));
    return max_nan(f.x, f.y);
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
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
  static __device__ __forceinline__ float largest(const uint4& u) {
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(pair(u.x), pair(u.y)), __hmax2_nan(pair(u.z), pair(u.w)));
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&m);
    return max_nan(__uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
  }
};

// Adds NV loads' values to a thread's sums.
template <typename T, int NV>
__device__ __forceinline__ void take(Sums& a, const uint4 (&u)[NV]) {
  float m = Vec<T>::largest(u[0]);
#pragma unroll
  for (int i = 1; i < NV; ++i) m = max_nan(m, Vec<T>::largest(u[i]));
  if (m == ninf()) return;
  if (!(m <= a.m)) {                             // a NaN too
    Sums r{max_nan(a.m, m), 0.f, 0.f};
    add_scaled(r, a.m, a.s, a.t);
    a = r;
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float v[Vec<T>::kN];
    Vec<T>::values(u[i], v);
#pragma unroll
    for (int j = 0; j < Vec<T>::kN; ++j) {
      const float d = max_nan((v[j] - a.m) * kLog2e, -200.f), e = ex2(d);
      a.s += e;
      a.t = fmaf(e, d, a.t);
    }
  }
}

// One row's share: elements [e0, e1), of which whole aligned 16-byte pieces
// [c0, c1) are read by the threads in turn and what is left of either end one
// by one.
struct Share {
  const void* row;
  int64_t e0, e1, first;     // first: the element at which piece 0 begins
  int c0, c1;
};

// The thread's elements, each once: f(value, index); false ends it.
template <typename T, typename F>
__device__ __forceinline__ void each(const Share& s, F f) {
  constexpr int N = Vec<T>::kN;
  const int64_t v0 = s.first + int64_t(s.c0) * N, v1 = s.first + int64_t(s.c1) * N;
  if (int64_t i = s.e0 + threadIdx.x; i < v0 && !f(Vec<T>::one(s.row, i), i)) return;
  if (int64_t i = v1 + threadIdx.x; i < s.e1 && !f(Vec<T>::one(s.row, i), i)) return;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(s.row) + s.first);
  for (int c = s.c0 + threadIdx.x; c < s.c1; c += kThreads) {
    float v[N];
    Vec<T>::values(__ldg(p + c), v);
    const int64_t i = s.first + int64_t(c) * N;
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (!f(v[j], i + j)) return;
  }
}

struct LpShared {
  uint64_t list[kMostTop];             // the share's k first, in order
  Sums sums;
  uint32_t bound[kWarps];
  Sums warp_sums[kWarps];
  int count, found[kWarps];
  uint64_t best[kWarps];
  uint64_t room[kRoom];
};

// Places the n entries of `from` that order among the first k into list[0 .. k).
__device__ __forceinline__ void place(const uint64_t* from, int n, int k, uint64_t* list) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t e = from[i];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) before += from[j] > e;
    if (e && before < k) list[before] = e;
  }
}

// The share's k first entries to sm.list; largest: of the thread's elements.
template <typename T>
__device__ void first_k(LpShared& sm, const Share& s, int k, float largest, bool any) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t mine = any ? key_of(largest) : 0u;
  // In each warp ceil(k / warps) threads hold a value of its bound or more: k at least of the least of the bounds.
  uint32_t q = mine, bound = 0;
  for (int i = 0; i < (k + kWarps - 1) / kWarps; ++i) {
    bound = __reduce_max_sync(0xffffffffu, q);
    const uint32_t who = __ballot_sync(0xffffffffu, q == bound);
    if (lane == __ffs(who) - 1) q = 0;
  }
  if (lane == 0) sm.bound[warp] = bound;
  if (threadIdx.x < kMostTop) sm.list[threadIdx.x] = 0;
  if (threadIdx.x == 0) sm.count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) bound = min(bound, sm.bound[w]);
  auto collect = [&](uint32_t least) {           // entries of this key or more, up to the room
    if (any && mine >= least)
      each<T>(s, [&](float v, int64_t i) {
        const uint32_t key = key_of(v);
        if (key < least) return true;
        const int at = atomicAdd(&sm.count, 1);
        if (at < kRoom) sm.room[at] = entry(key, i);
        return at < kRoom;
      });
    __syncthreads();
    return sm.count;
  };
  int n = collect(bound);
  if (n <= kRoom) {
    place(sm.room, n, k, sm.list);
    __syncthreads();
    return;
  }
  // Many equal values (a row with fewer than k unmasked ones): those above the bound, then of those at the bound the
  // first, in the order of their indices.
  __syncthreads();
  if (threadIdx.x == 0) sm.count = 0;
  __syncthreads();
  n = bound == 0xffffffffu ? 0 : collect(bound + 1);
  if (n <= kRoom) {
    place(sm.room, n, k, sm.list);
    for (int64_t base = s.e0; n < k && base < s.e1; base += kThreads) {
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
    each<T>(s, [&](float v, int64_t i) {
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

// One cluster of CTAs a row (one CTA where there are many rows); CTA 0 joins
// the parts.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(LpParams p, int ctas) {
  constexpr int N = Vec<T>::kN, kAtOnce = 4;
  __shared__ LpShared sm;
  const int64_t row = blockIdx.x / ctas;
  const int rank = blockIdx.x % ctas, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Share s;
  s.row = static_cast<const T*>(p.x) + row * p.ld;
  const int64_t off = (16 - (reinterpret_cast<uintptr_t>(s.row) & 15)) & 15;
  s.first = min(int64_t(off / sizeof(T)), int64_t(p.V));
  const int pieces = int((p.V - s.first) / N);
  s.c0 = int(int64_t(pieces) * rank / ctas), s.c1 = int(int64_t(pieces) * (rank + 1) / ctas);
  s.e0 = rank == 0 ? 0 : s.first + int64_t(s.c0) * N;
  s.e1 = rank == ctas - 1 ? p.V : s.first + int64_t(s.c1) * N;

  float token_x = __uint_as_float(0x7fc00000u);  // a token outside the vocabulary has no probability
  if (rank == 0 && threadIdx.x == 0) {
    const int64_t tok = p.tok64 ? __ldg(static_cast<const int64_t*>(p.tokens) + row) : __ldg(static_cast<const int32_t*>(p.tokens) + row);
    if (tok >= 0 && tok < p.V) token_x = Vec<T>::one(s.row, tok);
  }

  Sums a{ninf(), 0.f, 0.f};
  const uint4* pieces_p = reinterpret_cast<const uint4*>(static_cast<const T*>(s.row) + s.first);
  int c = s.c0 + threadIdx.x;
  for (; c + (kAtOnce - 1) * kThreads < s.c1; c += kAtOnce * kThreads) {
    uint4 u[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) u[i] = __ldg(pieces_p + c + i * kThreads);
    take<T, kAtOnce>(a, u);
  }
  {
    uint4 u[kAtOnce - 1];
#pragma unroll
    for (int i = 0; i < kAtOnce - 1; ++i) u[i] = c + i * kThreads < s.c1 ? __ldg(pieces_p + c + i * kThreads) : Vec<T>::none();
    // the ends, fewer than N elements each
    float v0 = ninf(), v1 = ninf();
    if (const int64_t i = s.e0 + threadIdx.x; i < s.first + int64_t(s.c0) * N) v0 = Vec<T>::one(s.row, i);
    if (const int64_t i = s.first + int64_t(s.c1) * N + threadIdx.x; i < s.e1) v1 = Vec<T>::one(s.row, i);
    take<T, kAtOnce - 1>(a, u);
    if (threadIdx.x < N) a = join(a, join(Sums{v0, 1.f, 0.f}, Sums{v1, 1.f, 0.f}));
  }
  const float largest = a.m;

  auto warp_join = [](Sums v) {
#pragma unroll
    for (int o = 16; o; o >>= 1)
      v = join(v, Sums{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
                       __shfl_xor_sync(0xffffffffu, v.t, o)});
    return v;
  };
  a = warp_join(a);
  if (lane == 0) sm.warp_sums[warp] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    Sums r = sm.warp_sums[0];
    for (int w = 1; w < kWarps; ++w) r = join(r, sm.warp_sums[w]);
    sm.sums = r;
  }
  if (p.top) {
    // has this thread any element?
    const bool any = s.c0 + int(threadIdx.x) < s.c1 || s.e0 + threadIdx.x < s.first + int64_t(s.c0) * N ||
                     s.first + int64_t(s.c1) * N + threadIdx.x < s.e1;
    first_k<T>(sm, s, p.top, largest, any);
  } else {
    __syncthreads();
  }

  Sums all = sm.sums;
  uint64_t* list = sm.list;
  if (ctas > 1) {
    __syncwarp();
    sm100::cluster_sync();
    if (rank == 0) {
      auto remote32 = [](const void* q, int r) {
        uint32_t v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(sm100::mapa_shared(q, r)) : "memory");
        return v;
      };
      for (int r = 1; r < ctas; ++r)
        all = join(all, Sums{__uint_as_float(remote32(&sm.sums.m, r)), __uint_as_float(remote32(&sm.sums.s, r)),
                             __uint_as_float(remote32(&sm.sums.t, r))});
      if (p.top) {
        // every share's list, then the first of all of them behind it
        const int n = ctas * p.top;
        for (int i = threadIdx.x; i < n; i += kThreads) {
          const uint64_t* q = &sm.list[i % p.top];
          uint64_t v;
          asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(sm100::mapa_shared(q, i / p.top)) : "memory");
          sm.room[i] = v;
        }
        list = sm.room + kMostCtas * kMostTop;
        __syncthreads();
        place(sm.room, n, p.top, list);
        __syncthreads();
      }
    }
    __syncwarp();
    sm100::cluster_sync();                       // no CTA leaves while CTA 0 reads its shared memory
    if (rank != 0) return;
  }
  const float log_s = logf(all.s);
  if (threadIdx.x == 0) {
    p.lp[row] = (token_x - all.m) - log_s;
    p.entropy[row] = log_s - kLn2 * (all.t / all.s);
  }
  if (int(threadIdx.x) < p.top) {
    const uint64_t e = list[threadIdx.x];
    p.top_lp[row * p.top + threadIdx.x] = (value_of(uint32_t(e >> 32)) - all.m) - log_s;
    p.top_ids[row * p.top + threadIdx.x] = int32_t(0xffffffffu - uint32_t(e));
  }
}

template <typename T>
int launch_logprobs(const LpParams& p, cudaStream_t st) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return TAC_E_CUDA;
  // CTAs a row: up to eight while all find a place at once, with two loads a thread or more
  int ctas = 1;
  while (ctas < kMostCtas && int64_t(p.M) * ctas * 2 <= 4 * sms && p.V >= 2 * ctas * 2 * kThreads * Vec<T>::kN) ctas *= 2;
  if (int64_t(p.M) * ctas > 0x7fffffff) return TAC_E_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(p.M) * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1;
  return status(cudaLaunchKernelEx(&cfg, logprobs_kernel<T>, p, ctas));
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
