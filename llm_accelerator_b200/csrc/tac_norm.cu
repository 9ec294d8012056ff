// Root-mean-square norm of rows with the residual's addition, its form with
// INT8 codes and a scale for each row, and what such codes stand for.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/taccel_b200.h"
#include "tac_launch.cuh"
#include "tac_rows.cuh"

namespace {

using namespace tac;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool type_ok(int t) { return t == TAC_F32 || t == TAC_F16 || t == TAC_BF16; }
int elem(int type) { return type == TAC_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// N consecutive values in 16-byte accesses.
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float (&v)[N]) {
  constexpr int kPer = 16 / sizeof(T);
  static_assert(N % kPer == 0, "whole accesses");
#pragma unroll
  for (int i = 0; i < N; i += kPer) {
    union {
      uint4 u;
      T t[kPer];
    } a;
    a.u = *reinterpret_cast<const uint4*>(p + i);
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[i + j] = to_f(a.t[j]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float (&v)[N]) {
  constexpr int kPer = 16 / sizeof(T);
  static_assert(N % kPer == 0, "whole accesses");
#pragma unroll
  for (int i = 0; i < N; i += kPer) {
    union {
      uint4 u;
      T t[kPer];
    } a;
#pragma unroll
    for (int j = 0; j < kPer; ++j) from_f(a.t[j], v[i + j]);
    *reinterpret_cast<uint4*>(p + i) = a.u;
  }
}

// The values of 16 bytes as float32 and back.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& u, float (&v)[16 / sizeof(T)]) {
  const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int j = 0; j < int(16 / sizeof(T)); ++j) v[j] = to_f(t[j]);
}
template <typename T>
__device__ __forceinline__ uint4 pack(const float (&v)[16 / sizeof(T)]) {
  uint4 u;
  T* t = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int j = 0; j < int(16 / sizeof(T)); ++j) from_f(t[j], v[j]);
  return u;
}

struct NormParams {
  const void* x;
  const void* r;             // or null
  void* h;                   // where there is an r
  const void* w;
  void* y;                   // rows of the input's type, or codes
  float* scale;              // of codes
  int64_t ldx, ldr, ldh;
  int w_type, w_vec;         // w_vec: the weight is aligned to 16 bytes
  int M, K;
  int ldq;                   // columns of the codes, K rounded up to 16
  float eps;
};

__device__ __forceinline__ float half_of(const NormParams& p, uint16_t b) {
  return p.w_type == TAC_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float(uint32_t(b) << 16);
}
// The weights of columns k to k + VEC, 0 past K.  The type is asked for once and
// not at each load, which would wait for the one before it.
template <int VEC>
__device__ __forceinline__ void weights(const NormParams& p, int k, float (&w)[VEC]) {
  const bool whole = p.w_vec && k + VEC <= p.K;
  if (p.w_type == TAC_F32) {
    const float* a = static_cast<const float*>(p.w) + k;
    if (whole) {
      load_n<float, VEC>(a, w);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) w[j] = k + j < p.K ? __ldg(a + j) : 0.f;
    }
  } else {
    const uint16_t* a = static_cast<const uint16_t*>(p.w) + k;
    uint16_t b[VEC];
    if (VEC == 8 && whole) {
      *reinterpret_cast<uint4*>(b) = __ldg(reinterpret_cast<const uint4*>(a));
    } else if (VEC == 4 && whole) {
      *reinterpret_cast<uint2*>(b) = __ldg(reinterpret_cast<const uint2*>(a));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) b[j] = k + j < p.K ? __ldg(a + j) : uint16_t(0);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[j] = half_of(p, b[j]);
  }
}

// What a row's sums give: the factor of h * w, and for codes the factor of y
// and the scale.  max_bits: the largest magnitude of h * w as bits, in which
// infinities and NaN order above every finite value.
struct RowNorm {
  float rstd, inv, scale;
};
template <bool I8>
__device__ __forceinline__ RowNorm row_norm(const NormParams& p, float ss, uint32_t max_bits) {
  RowNorm n;
  n.rstd = __frsqrt_rn(ss / float(p.K) + p.eps);
  n.inv = n.scale = 0.f;
  if (I8) {
    const float top = __uint_as_float(max_bits) * n.rstd;
    const bool finite = top < __uint_as_float(0x7f800000u);      // false for NaN too
    const float t = fmaxf(top, 1e-8f);
    n.inv = finite ? __fdiv_rn(127.0f, t) : 0.f;
    n.scale = finite ? __fdiv_rn(t, 127.0f) : __uint_as_float(0x7fc00000u);
  }
  return n;
}

// The low byte is the code of y = hw * rstd; 0 in a row without a scale.
__device__ __forceinline__ uint32_t code_bits(float hw, const RowNorm& n) {
  const float q = __fmul_rn(__fmul_rn(hw, n.rstd), n.inv);
  return n.inv == 0.f ? 0u : __float_as_uint(__fadd_rn(q, 12582912.f));   // 1.5 * 2^23: rounds to whole numbers
}

template <int WPR>
__device__ __forceinline__ void reduce_row(float& ss, uint32_t& mb) {
#pragma unroll
  for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  mb = __reduce_max_sync(0xffffffffu, mb);
  if constexpr (WPR > 1) {
    __shared__ float red_s[WPR];
    __shared__ uint32_t red_m[WPR];
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) red_s[warp] = ss, red_m[warp] = mb;
    __syncthreads();
    ss = 0.f;
    mb = 0;
#pragma unroll
    for (int w = 0; w < WPR; ++w) ss += red_s[w], mb = max(mb, red_m[w]);
  }
}

// The weighed values h * w of one load, and what they add to the row's sums.
template <bool I8, int VEC>
__device__ __forceinline__ void weigh(const NormParams& p, int k, float (&v)[VEC], float& ss, uint32_t& mb) {
  float w[VEC];
  weights<VEC>(p, k, w);
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    ss = fmaf(v[j], v[j], ss);
    v[j] *= w[j];
    if (I8) mb = max(mb, __float_as_uint(v[j]) & 0x7fffffffu);
  }
}

// Their codes; 0 for values past the row, which are 0.
template <int VEC>
__device__ __forceinline__ void store_codes(uint8_t* q, const float (&v)[VEC], const RowNorm& n) {
#pragma unroll
  for (int j = 0; j < VEC; j += 4) {
    const uint32_t lo = __byte_perm(code_bits(v[j], n), code_bits(v[j + 1], n), 0x0040);
    const uint32_t hi = __byte_perm(code_bits(v[j + 2], n), code_bits(v[j + 3], n), 0x0040);
    reinterpret_cast<uint32_t*>(q)[j / 4] = __byte_perm(lo, hi, 0x5410);
  }
}

// A thread's share of a row: CH loads of 16 bytes, VEC values each, the c-th
// from at(c) on.  ANY: the row begins and ends anywhere, and a warp's loads
// follow one another, which AnySpan needs; otherwise the row is a whole number
// of aligned loads, which the warps take in turn.
template <typename T, bool ANY, int CH>
struct RowShare {
  static constexpr int VEC = 16 / sizeof(T);
  int K, first, step, chunks;          // of chunks that hold any of the row, the first `chunks` at most

  // `warps` warps share columns [k, K)
  __device__ __forceinline__ RowShare(int K, int k, int warp, int warps) : K(K) {
    const int lane = threadIdx.x & 31;
    if (ANY) {
      chunks = min(CH, ((K - k + VEC - 1) / VEC + 32 * warps - 1) / (32 * warps));
      first = k + (warp * chunks * 32 + lane) * VEC;
      step = 32 * VEC;
    } else {
      chunks = CH;
      first = k + (warp * 32 + lane) * VEC;
      step = 32 * warps * VEC;
    }
  }
  __device__ __forceinline__ int at(int c) const { return first + c * step; }
  __device__ __forceinline__ bool live(int c) const { return (!ANY || c < chunks) && at(c) < K; }

  // what the row has from `begin` on, or more than the share holds, in 16-bit values
  __device__ __forceinline__ int units(int begin) const { return min(K - begin, (CH + 1) * 32 * VEC) * int(sizeof(T) / 2); }

  // x (+ r) to v; h = x + r out where there is one
  __device__ __forceinline__ void sum(const T* x, const T* r, T* h, float (&v)[CH][VEC]) const {
    if constexpr (ANY) {
      const int begin = first - int(threadIdx.x & 31) * VEC, left = units(begin);
      AnySpan<CH> a, b;
      a.load(reinterpret_cast<const uint16_t*>(x + begin), chunks, left);
      if (r) b.load(reinterpret_cast<const uint16_t*>(r + begin), chunks, left);
      a.values(chunks, left);
#pragma unroll
      for (int c = 0; c < CH; ++c) unpack<T>(a.v[c], v[c]);
      if (r) {
        b.values(chunks, left);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          float t[VEC];
          unpack<T>(b.v[c], t);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[c][j] += t[j];
        }
      }
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (live(c)) load_n<T, VEC>(x + at(c), v[c]);
      if (r) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
          if (live(c)) {
            float t[VEC];
            load_n<T, VEC>(r + at(c), t);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[c][j] += t[j];
          }
      }
    }
    if (h) store(h, v);
  }
  __device__ __forceinline__ void store(T* y, const float (&v)[CH][VEC]) const {
    if constexpr (ANY) {
      const int begin = first - int(threadIdx.x & 31) * VEC;
      AnySpan<CH> a;
#pragma unroll
      for (int c = 0; c < CH; ++c) a.v[c] = pack<T>(v[c]);
      a.store(reinterpret_cast<uint16_t*>(y + begin), chunks, units(begin));
    } else {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (live(c)) store_n<T, VEC>(y + at(c), v[c]);
    }
  }
};

// WPR warps a row (one: four rows a CTA), CH loads of 16 bytes a thread.  A row
// is read once and stays in registers as h * w: the sum of h^2 and the largest
// |h * w| are reduced together, because the norm's factor is the same for the
// whole row, so that one exchange among the warps gives both the norm and the
// codes' scale.  h goes out, rounded, as soon as it is there; the norm is of the
// unrounded sum.
template <typename T, bool ANY, bool I8, int WPR, int CH>
__global__ void __launch_bounds__(WPR == 1 ? 128 : 32 * WPR, WPR == 16 ? 2 : 1) norm_kernel(NormParams p) {
  using Row = RowShare<T, ANY, CH>;
  constexpr int VEC = Row::VEC, kLanes = 32 * WPR;
  after_previous();
  let_next();
  const int64_t row = WPR == 1 ? int64_t(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= p.M) return;                        // a whole warp (WPR 1); otherwise none
  const Row s(p.K, 0, WPR == 1 ? 0 : threadIdx.x >> 5, WPR);
  float v[CH][VEC];
  float ss = 0.f;
  uint32_t mb = 0;
  s.sum(static_cast<const T*>(p.x) + row * p.ldx, p.r ? static_cast<const T*>(p.r) + row * p.ldr : nullptr,
        p.r ? static_cast<T*>(p.h) + row * p.ldh : nullptr, v);
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (s.live(c)) weigh<I8, VEC>(p, s.at(c), v[c], ss, mb);
  reduce_row<WPR>(ss, mb);
  const RowNorm n = row_norm<I8>(p, ss, mb);
  if constexpr (!I8) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[c][j] *= n.rstd;
    s.store(static_cast<T*>(p.y) + row * p.K, v);
  } else {
    uint8_t* q = static_cast<uint8_t*>(p.y) + row * p.ldq;
    const int t = threadIdx.x % kLanes;
    if (t == 0) p.scale[row] = n.scale;
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (s.live(c)) store_codes<VEC>(q + s.at(c), v[c], n);
    for (int k = (p.K + VEC - 1) / VEC * VEC + t; k < p.ldq; k += kLanes) q[k] = 0;      // the padding columns
  }
}

// Rows too long for registers: they are read again for the results.  h is
// written then, so that it may lie over the residual.
constexpr int kLongWarps = 16, kLongLoads = 2;
template <typename T, bool I8>
__global__ void __launch_bounds__(32 * kLongWarps, 2) norm_long_kernel(NormParams p) {
  using Row = RowShare<T, true, kLongLoads>;
  constexpr int VEC = Row::VEC, kStep = 32 * kLongWarps * kLongLoads * VEC;
  after_previous();
  let_next();
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5;
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = p.r ? static_cast<const T*>(p.r) + row * p.ldr : nullptr;
  float ss = 0.f;
  uint32_t mb = 0;
  for (int k = 0; k < p.K; k += kStep) {
    const Row s(p.K, k, warp, kLongWarps);
    float v[kLongLoads][VEC];
    s.sum(x, r, nullptr, v);
#pragma unroll
    for (int c = 0; c < kLongLoads; ++c)
      if (s.live(c)) weigh<I8, VEC>(p, s.at(c), v[c], ss, mb);
  }
  reduce_row<kLongWarps>(ss, mb);
  const RowNorm n = row_norm<I8>(p, ss, mb);
  uint8_t* q = I8 ? static_cast<uint8_t*>(p.y) + row * p.ldq : nullptr;
  if (I8 && threadIdx.x == 0) p.scale[row] = n.scale;
  for (int k = 0; k < p.K; k += kStep) {
    const Row s(p.K, k, warp, kLongWarps);
    float v[kLongLoads][VEC];
    s.sum(x, r, r ? static_cast<T*>(p.h) + row * p.ldh : nullptr, v);
#pragma unroll
    for (int c = 0; c < kLongLoads; ++c) {
      if (!s.live(c)) continue;
      weigh<I8, VEC>(p, s.at(c), v[c], ss, mb);
      if constexpr (I8) store_codes<VEC>(q + s.at(c), v[c], n);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[c][j] *= n.rstd;
    }
    if constexpr (!I8) s.store(static_cast<T*>(p.y) + row * p.K, v);
  }
  if constexpr (I8)
    for (int k = (p.K + VEC - 1) / VEC * VEC + threadIdx.x; k < p.ldq; k += 32 * kLongWarps) q[k] = 0;
}

// As few warps a row as hold it in four loads a thread, of one, two, four,
// eight and sixteen (with one, four and sixteen alone, rows whose threads have
// two loads or fewer leave too little under way: 2784 x 6560 BF16 to INT8 takes
// 26 us in eight warps, 39 in sixteen).
template <typename T, bool ANY, bool I8>
int launch_rows(const NormParams& p, cudaStream_t st) {
  constexpr int kOf = 64 / sizeof(T);            // values of four loads
  if (p.K <= 32 * kOf) return launch_behind(norm_kernel<T, ANY, I8, 1, 4>, unsigned(p.M + 3u) / 4, 128, 0, st, p);
  if (p.K <= 64 * kOf) return launch_behind(norm_kernel<T, ANY, I8, 2, 4>, p.M, 64, 0, st, p);
  if (p.K <= 128 * kOf) return launch_behind(norm_kernel<T, ANY, I8, 4, 4>, p.M, 128, 0, st, p);
  if (p.K <= 256 * kOf) return launch_behind(norm_kernel<T, ANY, I8, 8, 4>, p.M, 256, 0, st, p);
  if (p.K <= 512 * kOf) return launch_behind(norm_kernel<T, ANY, I8, 16, 4>, p.M, 512, 0, st, p);
  if constexpr (sizeof(T) == 4) {                // as 16-bit rows, to 16384; eight loads and their shifts need too many registers
    if (p.K <= 1024 * kOf) return launch_behind(norm_kernel<T, ANY, I8, ANY ? 32 : 16, ANY ? 4 : 8>, p.M, ANY ? 1024 : 512, 0, st, p);
  }
  return launch_behind(norm_long_kernel<T, I8>, p.M, 32 * kLongWarps, 0, st, p);
}

template <typename T, bool I8>
int launch_norm(const NormParams& p, cudaStream_t st) {
  auto whole = [&](const void* a, int64_t ld) { return aligned(a, 16) && (p.M == 1 || ld * int64_t(sizeof(T)) % 16 == 0); };
  const bool loads = p.K % (16 / int(sizeof(T))) == 0 && whole(p.x, p.ldx) && (!p.r || (whole(p.r, p.ldr) && whole(p.h, p.ldh))) &&
                     (I8 || whole(p.y, p.K));
  if (loads) return launch_rows<T, false, I8>(p, st);
  return launch_rows<T, true, I8>(p, st);
}

template <bool I8>
int pick_norm(NormParams p, int type, cudaStream_t st) {
  if (type == TAC_F32) return launch_norm<float, I8>(p, st);
  if (type == TAC_F16) return launch_norm<__half, I8>(p, st);
  return launch_norm<__nv_bfloat16, I8>(p, st);
}

// Checks that both forms share.
int check_norm(const void* X, int type, int64_t ldx, const void* R, int64_t ldr, const void* H, int64_t ldh, const void* W,
               int w_type, const void* Y, float eps, int M, int K) {
  if (!X || !W || !Y || !type_ok(type) || !type_ok(w_type) || M <= 0 || K <= 0 || K > (1 << 30) || !R != !H ||
      (H && H == Y))
    return TAC_E_ARGUMENT;
  if (M > 1 && (ldx < K || (R && (ldr < K || ldh < K)))) return TAC_E_ARGUMENT;
  const int e = elem(type);
  if (!aligned(X, e) || (R && (!aligned(R, e) || !aligned(H, e))) || !aligned(W, elem(w_type))) return TAC_E_ARGUMENT;
  return eps >= 0.f && eps <= 1e30f ? TAC_OK : TAC_E_ARGUMENT;   // NaN is neither
}

NormParams norm_params(const void* X, int type, int64_t ldx, const void* R, int64_t ldr, void* H, int64_t ldh, const void* W,
                       int w_type, void* Y, float* scale, float eps, int M, int K) {
  NormParams p{};
  p.x = X, p.r = R, p.h = H, p.w = W, p.y = Y, p.scale = scale;
  p.ldx = ldx, p.ldr = ldr, p.ldh = ldh;
  p.w_type = w_type, p.w_vec = aligned(W, 16);
  p.M = M, p.K = K, p.ldq = int((int64_t(K) + 15) / 16 * 16);
  p.eps = eps;
  return p;
}

// ---- the values of codes ---------------------------------------------------------------------------------------------
constexpr int kDqThreads = 256, kDqRows = 4;

// Eight codes of each of four rows a thread, all loads first (8192 x 4096 to
// BF16: 14.6 us; one row a thread takes 20); a row is cut into `cuts` CTAs.  VEC:
// aligned rows; otherwise 16-bit ones are written by whole warps (tac_rows.cuh).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kDqThreads) dequant_rows_kernel(const int8_t* __restrict__ Q, int ldq,
                                                                  const float* __restrict__ scale, T* __restrict__ Y, int M, int K,
                                                                  uint32_t cuts) {
  after_previous();
  let_next();
  const uint32_t group = blockIdx.x / cuts;
  const int64_t row = int64_t(group) * kDqRows;
  const int k = int((blockIdx.x - group * cuts) * kDqThreads + threadIdx.x) * 8;
  constexpr bool kAny = !VEC && sizeof(T) == 2;
  if (kAny ? k - int(threadIdx.x & 31) * 8 >= K : k >= K) return;        // whole warps, where they write together
  const int rows = int(min(int64_t(kDqRows), M - row));
  uint2 u[kDqRows];
  float s[kDqRows];
#pragma unroll
  for (int r = 0; r < kDqRows; ++r) {
    if (r >= rows) break;
    s[r] = __ldg(scale + row + r);
    u[r] = make_uint2(0, 0);
    if (k < K) u[r] = __ldg(reinterpret_cast<const uint2*>(Q + (row + r) * ldq + k));
  }
#pragma unroll
  for (int r = 0; r < kDqRows; ++r) {
    if (r >= rows) break;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = float(int8_t((j < 4 ? u[r].x : u[r].y) >> (8 * (j & 3)))) * s[r];
    T* y = Y + (row + r) * K + k;
    if constexpr (VEC) {
      store_n<T, 8>(y, v);
    } else if constexpr (kAny) {
      AnySpan<1> a;
      a.v[0] = pack<T>(v);
      const int before = int(threadIdx.x & 31) * 8;
      a.store(reinterpret_cast<uint16_t*>(y - before), 1, K - k + before);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) y[j] = v[j];
    }
  }
}

template <typename T>
int launch_dequant(const int8_t* Q, int ldq, const float* scale, T* Y, int M, int K, cudaStream_t st) {
  const int64_t per = kDqThreads * 8, cuts = (K + per - 1) / per, ctas = (int64_t(M) + kDqRows - 1) / kDqRows * cuts;
  if (ctas > 0x7fffffff) return TAC_E_ARGUMENT;
  if (K % 8 == 0 && aligned(Y, 16))
    return launch_behind(dequant_rows_kernel<T, true>, unsigned(ctas), kDqThreads, 0, st, Q, ldq, scale, Y, M, K, uint32_t(cuts));
  return launch_behind(dequant_rows_kernel<T, false>, unsigned(ctas), kDqThreads, 0, st, Q, ldq, scale, Y, M, K, uint32_t(cuts));
}

}  // namespace

extern "C" int tac_rms_norm(const void* X, int type, int64_t ldx, const void* R, int64_t ldr, void* H, int64_t ldh,
                            const void* W, int w_type, float eps, void* Y, int M, int K, void* stream) {
  if (int s = check_norm(X, type, ldx, R, ldr, H, ldh, W, w_type, Y, eps, M, K)) return s;
  if (!aligned(Y, elem(type))) return TAC_E_ARGUMENT;
  return pick_norm<false>(norm_params(X, type, ldx, R, ldr, H, ldh, W, w_type, Y, nullptr, eps, M, K), type,
                          static_cast<cudaStream_t>(stream));
}

extern "C" int tac_rms_norm_i8(const void* X, int type, int64_t ldx, const void* R, int64_t ldr, void* H, int64_t ldh,
                               const void* W, int w_type, float eps, int8_t* Q, float* scale, int M, int K, void* stream) {
  if (int s = check_norm(X, type, ldx, R, ldr, H, ldh, W, w_type, Q, eps, M, K)) return s;
  if (!scale || !aligned(Q, 16) || !aligned(scale, 4)) return TAC_E_ARGUMENT;
  return pick_norm<true>(norm_params(X, type, ldx, R, ldr, H, ldh, W, w_type, Q, scale, eps, M, K), type,
                         static_cast<cudaStream_t>(stream));
}

extern "C" int tac_dequantize_rows_i8(const int8_t* Q, const float* scale, void* Y, int y_type, int M, int K, void* stream) {
  if (!Q || !scale || !Y || !type_ok(y_type) || M <= 0 || K <= 0 || K > (1 << 30) || !aligned(Q, 16) || !aligned(scale, 4) ||
      !aligned(Y, elem(y_type)))
    return TAC_E_ARGUMENT;
  const int ldq = (K + 15) / 16 * 16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (y_type == TAC_F32) return launch_dequant(Q, ldq, scale, static_cast<float*>(Y), M, K, st);
  if (y_type == TAC_F16) return launch_dequant(Q, ldq, scale, static_cast<__half*>(Y), M, K, st);
  return launch_dequant(Q, ldq, scale, static_cast<__nv_bfloat16*>(Y), M, K, st);
}
