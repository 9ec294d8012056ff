// INT8 linear layers with a scale for each token and output channel: the row
// quantiser, the scaled product (tac_w8a8.cuh) and both in one call.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/taccel_b200.h"
#include "tac_launch.cuh"
#include "tac_tmap.h"
#include "tac_w8a8.cuh"

namespace tac {
int* gemm_fault_word();
}

namespace {

using namespace tac;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool type_ok(int t) { return t == TAC_F32 || t == TAC_F16 || t == TAC_BF16; }

int sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (!sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    sms[dev] = n;
  }
  return sms[dev];
}

int* fault_word() {
  static int* words[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return nullptr;
  if (!words[dev]) words[dev] = gemm_fault_word();
  return words[dev];
}

// ---- row quantiser --------------------------------------------------------------------------------------------------
// t = max(max |x|, 1e-8), scale = t / 127, q = rint(x * (127 / t)) in float32;
// a row that holds an infinity or a NaN gets the scale NaN.  The maximum is
// taken over the magnitudes' bits, in which infinities and NaN order above
// every finite value.
constexpr int kQrThreads = 128;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

struct RowScale {
  float inv, scale;
  bool finite;
};
__device__ __forceinline__ RowScale row_scale(uint32_t max_bits) {
  RowScale r;
  r.finite = max_bits < 0x7f800000u;
  const float t = fmaxf(__uint_as_float(max_bits), 1e-8f);
  r.inv = r.finite ? __fdiv_rn(127.0f, t) : 0.f;
  r.scale = r.finite ? __fdiv_rn(t, 127.0f) : __uint_as_float(0x7fc00000u);
  return r;
}

// Lets the product that follows start early: at once when these rows leave SMs free, else when they are done (its
// CTAs would take the registers that the rest of this grid needs).
__device__ __forceinline__ void release_dependents(bool early) {
  if (early == (gridDim.x <= 148)) asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

// Any alignment and length: two reads of the row.
template <typename T>
__global__ void __launch_bounds__(kQrThreads) quant_rows_kernel(const T* __restrict__ X, int64_t ldx,
                                                                int8_t* __restrict__ Q, int ldq,
                                                                float* __restrict__ scale, int K) {
  __shared__ uint32_t red[kQrThreads / 32];
  release_dependents(true);
  const int64_t row = blockIdx.x;
  const T* x = X + row * ldx;
  int8_t* q = Q + row * ldq;
  uint32_t mb = 0;
  for (int k = threadIdx.x; k < K; k += kQrThreads) mb = max(mb, __float_as_uint(to_f(x[k])) & 0x7fffffffu);
  mb = __reduce_max_sync(0xffffffffu, mb);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mb;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQrThreads / 32; ++w) mb = max(mb, red[w]);
  const RowScale r = row_scale(mb);
  if (threadIdx.x == 0) scale[row] = r.scale;
  for (int k = threadIdx.x; k < ldq; k += kQrThreads) {
    int v = 0;
    if (k < K && r.finite) v = __float2int_rn(__fmul_rn(to_f(x[k]), r.inv));
    q[k] = int8_t(v);
  }
  release_dependents(false);
}

// 16-bit rows of whole 16-byte chunks: a row is read once, eight chunks a
// thread at most, by one warp (K up to 2048) or four.  Bound by the bytes,
// 2 read and 1 written a value; the rounding is one addition of 1.5 * 2^23,
// after which the low byte is the code, and a byte permutation packs four
// (a convert instruction a value alone took as long as the memory).
// 8192 x 4096: 18.5 us, 5.4 TB/s.
template <typename T, int WPR>
__global__ void __launch_bounds__(kQrThreads) quant_rows_vec_kernel(const T* __restrict__ X, int64_t ldx,
                                                                    int8_t* __restrict__ Q, int ldq,
                                                                    float* __restrict__ scale, int M, int K) {
  constexpr int kChunks = 8, kLanes = 32 * WPR, kRows = kQrThreads / kLanes;
  __shared__ uint32_t red[kQrThreads / 32];
  release_dependents(true);
  const int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / kLanes;
  const int t = threadIdx.x % kLanes, chunks = K / 8;
  if (WPR == 1 && row >= M) return;              // a whole warp
  const uint4* x = reinterpret_cast<const uint4*>(X + row * ldx);
  uint4 v[kChunks];
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    v[i] = make_uint4(0, 0, 0, 0);
    if (t + i * kLanes < chunks) v[i] = __ldg(x + t + i * kLanes);
  }
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                               __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu)));
  }
  uint32_t mb = __reduce_max_sync(0xffffffffu, max(m2 & 0xffffu, m2 >> 16));
  if (WPR > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mb;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQrThreads / 32; ++w) mb = max(mb, red[w]);
  }
  // a 16-bit magnitude as float32: infinities and NaN stay above every finite value
  auto f32 = [](uint32_t h) {
    return sizeof(T) == 2 && std::is_same<T, __half>::value ? __half2float(__ushort_as_half(uint16_t(h))) : __uint_as_float(h << 16);
  };
  const RowScale r = row_scale(__float_as_uint(f32(mb)) & 0x7fffffffu);
  if (t == 0) scale[row] = r.scale;
  auto code = [&](uint32_t h) { return __float_as_uint(__fadd_rn(__fmul_rn(f32(h & 0xffffu), r.inv), 12582912.f)); };
  uint2* q = reinterpret_cast<uint2*>(Q + row * ldq);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    if (t + i * kLanes >= chunks) break;
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    uint32_t o[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t a = __byte_perm(code(w[2 * j]), code(w[2 * j] >> 16), 0x0040);
      const uint32_t b = __byte_perm(code(w[2 * j + 1]), code(w[2 * j + 1] >> 16), 0x0040);
      o[j] = r.finite ? __byte_perm(a, b, 0x5410) : 0u;
    }
    q[t + i * kLanes] = make_uint2(o[0], o[1]);
  }
  if (K % 16 && t == 0) q[chunks] = make_uint2(0, 0);   // the padding columns
  release_dependents(false);
}

template <typename T>
int quant_rows_16(const T* X, int64_t ldx, int8_t* Q, int ldq, float* scale, int M, int K, cudaStream_t st) {
  const bool vec = K % 8 == 0 && K <= 8192 && aligned(X, 16) && (M == 1 || ldx % 8 == 0);
  if (vec && K <= 2048) return launch(quant_rows_vec_kernel<T, 1>, (M + 3) / 4, kQrThreads, 0, st, X, ldx, Q, ldq, scale, M, K);
  if (vec) return launch(quant_rows_vec_kernel<T, 4>, M, kQrThreads, 0, st, X, ldx, Q, ldq, scale, M, K);
  return launch(quant_rows_kernel<T>, M, kQrThreads, 0, st, X, ldx, Q, ldq, scale, K);
}

int launch_quant_rows(const void* X, int type, int64_t ldx, int8_t* Q, float* scale, int M, int K, cudaStream_t st) {
  const int ldq = (K + 15) / 16 * 16;
  if (type == TAC_F32) return launch(quant_rows_kernel<float>, M, kQrThreads, 0, st, static_cast<const float*>(X), ldx, Q, ldq, scale, K);
  if (type == TAC_F16) return quant_rows_16(static_cast<const __half*>(X), ldx, Q, ldq, scale, M, K, st);
  return quant_rows_16(static_cast<const __nv_bfloat16*>(X), ldx, Q, ldq, scale, M, K, st);
}

// ---- scaled product -------------------------------------------------------------------------------------------------
bool map_rows(CUtensorMap* m, const int8_t* base, int K, int rows, int box_rows) {
  const cuuint64_t dims[2] = {cuuint64_t(K), cuuint64_t(rows)}, strides[1] = {cuuint64_t(K)};
  const cuuint32_t box[2] = {128, cuuint32_t(box_rows)};
  return tmap_encode_u8(m, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

constexpr int kSkMaxSmem = 224 * 1024;

// CTAs that share a tile's K blocks: as many as find an SM each, with eight K blocks or more a CTA (two for 16 tokens,
// whose partial sums are few).  Measured, four CTAs a tile against one: 64 x 4096 x 1024 loses 1.1 us of 7, 64 x 4096 x
// 4096 gains 1.2 of 12, 1 x 4096 x 4096 2.3 of 10; more CTAs than SMs cost 1 x 4096 x 1024 1.7 us.
int splits(int64_t tiles, int k_blocks, int tn, int sms) {
  int split = 1;
  while (split < 8 && 2 * split * (tn > 16 ? 8 : 2) <= k_blocks && tiles * split * 2 <= sms) split *= 2;
  return split;
}

template <int YT>
int launch_splitk(const int8_t* A, const int8_t* Bt, W8Params p, cudaStream_t st) {
  static bool smem_set[64] = {};
  int dev = 0;
  const int sms = sm_count();
  if (!sms || cudaGetDevice(&dev) != cudaSuccess) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (int e = status(cudaFuncSetAttribute(w8_splitk_kernel<YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSkMaxSmem))) return e;
    smem_set[dev] = true;
  }
  p.k_blocks = (p.K + 127) / 128;
  p.tn = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
  const int64_t tiles = int64_t((p.N + 127) / 128) * ((p.M + p.tn - 1) / p.tn);
  const int split = splits(tiles, p.k_blocks, p.tn, sms);
  const int per = (p.k_blocks + split - 1) / split, sb = sk_stage_bytes(p.tn);
  // in flight: 96 KB where two CTAs share an SM, else twice that
  p.stages = std::min(std::min(per, 8), std::max(2, (tiles * split > sms ? 96 : 190) * 1024 / sb));
  const int part = split > 1 ? sk_part_bytes(p.tn) : 0;
  CUtensorMap tw, ta;
  if (!map_rows(&tw, Bt, p.K, p.N, 128) || !map_rows(&ta, A, p.K, p.M, p.tn)) return TAC_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + 127) / 128, (p.M + p.tn - 1) / p.tn, split);
  cfg.blockDim = dim3(kSkThreads);
  cfg.dynamicSmemBytes = std::max(p.stages * sb, part) + 1024;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (split > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = 1;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = split;
  }
  if (p.after_rows) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  return status(cudaLaunchKernelEx(&cfg, w8_splitk_kernel<YT>, tw, ta, p));
}

// Tokens of a pair tile: the multiple of 32 that leaves the least work on the
// fullest pair, a tile's time going with its tokens plus a constant share for
// filling 256 channels of weights.
int pair_tokens(int M, int N, int clusters, int* waves) {
  const int64_t wt = (N + 255) / 256;
  int best = 0;
  double cost = 0;
  for (int tn = 256; tn >= 64; tn -= 32) {
    const int64_t tiles = wt * ((M + tn - 1) / tn);
    const double c = double((tiles + clusters - 1) / clusters) * (tn + 32);
    if (!best || c < cost) best = tn, cost = c, *waves = int((tiles + clusters - 1) / clusters);
  }
  return best;
}

// Largest number of CTA pairs that run at once; 0 where none does.
template <int YT>
int pair_clusters(int dev) {
  static int clusters[64];
  static bool done[64] = {};
  if (!done[dev]) {
    int n = 0;
    const int sms = sm_count();
    if (cudaFuncSetAttribute(w8_pair_kernel<YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg::kSmem) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * (sms / 2));
      cfg.blockDim = dim3(PairCfg::kThreads);
      cfg.dynamicSmemBytes = PairCfg::kSmem;
      if (cudaOccupancyMaxActiveClusters(&n, w8_pair_kernel<YT>, &cfg) != cudaSuccess) n = 0;
    }
    cudaGetLastError();
    clusters[dev] = std::min(n, sms / 2);
    done[dev] = true;
  }
  return clusters[dev];
}

template <int YT>
int launch_pair(const int8_t* A, const int8_t* Bt, W8Params p, int clusters, int tn, cudaStream_t st) {
  W8PairParams pp{};
  p.tn = tn;
  p.k_blocks = (p.K + 127) / 128;
  pp.g = p;
  pp.w_tiles = (p.N + 255) / 256;
  pp.t_tiles = (p.M + tn - 1) / tn;
  CUtensorMap tw, ta;
  if (!map_rows(&tw, Bt, p.K, p.N, 128) || !map_rows(&ta, A, p.K, p.M, tn / 2)) return TAC_E_CUDA;
  const int64_t tiles = int64_t(pp.w_tiles) * pp.t_tiles;
  if (tiles > (1 << 30)) return TAC_E_ARGUMENT;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * int(std::min<int64_t>(tiles, clusters)));
  cfg.blockDim = dim3(PairCfg::kThreads);
  cfg.dynamicSmemBytes = PairCfg::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.after_rows ? 1 : 0;
  return status(cudaLaunchKernelEx(&cfg, w8_pair_kernel<YT>, tw, ta, pp));
}

// Checks that both products share; also the limits of 32-bit sums and of the grid.
int check_product(const void* Bt, const void* b_scale, int b_type, const void* bias, int bias_type, const void* Y,
                  int y_type, int M, int N, int K) {
  if (!Bt || !b_scale || !Y || M <= 0 || N <= 0 || K <= 0) return TAC_E_ARGUMENT;
  if ((b_type != TAC_F32 && b_type != TAC_F16) || !type_ok(y_type) || (bias && !type_ok(bias_type))) return TAC_E_ARGUMENT;
  auto elem = [](int type) { return type == TAC_F32 ? 4 : 2; };
  if (!aligned(Y, elem(y_type)) || !aligned(b_scale, elem(b_type)) || (bias && !aligned(bias, elem(bias_type)))) return TAC_E_ARGUMENT;
  if (K >= (1 << 17) || M > (1 << 20) || N > (1 << 30) || !aligned(Bt, 16)) return TAC_E_ARGUMENT;   // |sum| <= K * 128^2 < 2^31
  return TAC_OK;
}

template <int YT>
int pick_product(const int8_t* A, const int8_t* Bt, const W8Params& p, cudaStream_t st) {
  int dev = 0, waves = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  const int clusters = pair_clusters<YT>(dev);
  if (p.M > 128 && clusters > 0) {
    const int tn = pair_tokens(p.M, p.N, clusters, &waves);
    if (int64_t((p.N + 255) / 256) * ((p.M + tn - 1) / tn) * 2 >= clusters) return launch_pair<YT>(A, Bt, p, clusters, tn, st);
  }
  return launch_splitk<YT>(A, Bt, p, st);
}

int run_product(const int8_t* A, const int8_t* Bt, const float* a_scale, const void* b_scale, int b_type,
                const void* bias, int bias_type, void* Y, int y_type, int M, int N, int K, bool after_rows, cudaStream_t st) {
  W8Params p{};
  p.after_rows = after_rows;
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.bias = bias;
  p.y = Y;
  p.b_type = b_type;
  p.bias_type = bias_type;
  p.M = M;
  p.N = N;
  p.K = K;
  if (!(p.fault = fault_word())) return TAC_E_CUDA;
  return y_type == TAC_F32 ? pick_product<0>(A, Bt, p, st) : y_type == TAC_F16 ? pick_product<1>(A, Bt, p, st) : pick_product<2>(A, Bt, p, st);
}

static_assert(kRowsMostK / 128 * kRowsMost * 128 + 2 * kSkWBytes + 1024 <= kSkMaxSmem, "whole rows and a ring fit");

// Few rows: one launch is possible, with no workspace.
bool few_rows(int M, int K) { return M <= kRowsMost && K <= kRowsMostK; }

// Where one launch is faster than the quantiser and the product, for a call that the host waits for: it spares the second
// launch and the workspace (5.5 us a call, 3 us of latency), but its 128 threads quantise every row in each of the N / 128
// CTAs before the first MMA, and whole rows of long K leave an SM one CTA.  On the device alone it is behind everywhere, by
// 0.8 us where a CTA has few values and by 250 where it has 131,072.  Microseconds, one launch against two, on the device
// and for a call alone:
//    1 x 4096 x 1024    7.0 / 5.8   22.6 / 25.7      1 x 28672 x 1024    9.1 /  9.1   24.5 / 28.8
//   16 x 4096 x 1024    9.7 / 6.4   25.2 / 26.4      8 x 28672 x 1024   14.8 /  9.1   30.1 / 28.4
//    4 x 4096 x 4096   12.0 / 8.8   27.6 / 28.6      1 x 28672 x 4096   34.0 / 22.0
//    8 x 4096 x 4096   15.1 / 8.8   31.2 / 28.9      1 x 10240 x 8192   27.0 / 19.4
//    1 x 4096 x 8192   13.7 / 11.0  29.0 / 31.0     16 x 28672 x 8192  292.3 / 41.7
// (N x K behind the rows.)
bool one_launch(int M, int N, int K, int sms) {
  if (!few_rows(M, K)) return false;
  const int64_t tiles = (int64_t(N) + 127) / 128;
  const int k_blocks = (K + 127) / 128, split = splits(tiles, k_blocks, kRowsMost, sms);
  return M * 128 * ((k_blocks + split - 1) / split) <= (tiles > sms ? 2048 : 4096);
}

template <int YT>
int launch_rows(W8RowsParams pp, const int8_t* Bt, cudaStream_t st) {
  static bool smem_set[64] = {};
  int dev = 0;
  const int sms = sm_count();
  if (!sms || cudaGetDevice(&dev) != cudaSuccess) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (int e = status(cudaFuncSetAttribute(w8_rows_kernel<YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSkMaxSmem))) return e;
    smem_set[dev] = true;
  }
  W8Params& p = pp.g;
  p.tn = kRowsMost;
  p.k_blocks = (p.K + 127) / 128;
  const int64_t tiles = (p.N + 127) / 128;
  const int split = splits(tiles, p.k_blocks, p.tn, sms);
  const int per = (p.k_blocks + split - 1) / split;
  // weights in flight: four stages where two CTAs share an SM, else eight, of what the rows' codes leave (five of 64 blocks)
  const int rows_bytes = per * kRowsMost * 128;
  p.stages = std::min({per, tiles * split > sms ? 4 : 8, (kSkMaxSmem - 1024 - rows_bytes) / kSkWBytes});
  CUtensorMap tw;
  if (!map_rows(&tw, Bt, p.K, p.N, 128)) return TAC_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(uint32_t(tiles), 1, split);
  cfg.blockDim = dim3(kSkThreads);
  cfg.dynamicSmemBytes = p.stages * kSkWBytes + rows_bytes + 1024;   // the partial sums (10 KB) fit the first stage
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = split;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1;
  return status(cudaLaunchKernelEx(&cfg, w8_rows_kernel<YT>, tw, pp));
}

uint64_t align256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

}  // namespace

extern "C" int tac_quantize_rows_i8(const void* X, int x_type, int64_t ldx, int8_t* Q, float* scale, int M, int K,
                                    void* stream) {
  if (!X || !Q || !scale || !type_ok(x_type) || M <= 0 || K <= 0 || (M > 1 && ldx < K) || !aligned(Q, 16) ||
      !aligned(X, x_type == TAC_F32 ? 4 : 2) || !aligned(scale, 4))
    return TAC_E_ARGUMENT;
  return launch_quant_rows(X, x_type, ldx, Q, scale, M, K, static_cast<cudaStream_t>(stream));
}

extern "C" int tac_gemm_i8_scaled(const int8_t* A, const int8_t* Bt, const float* a_scale, const void* b_scale,
                                  int b_scale_type, const void* bias, int bias_type, void* Y, int y_type, int M, int N,
                                  int K, void* stream) {
  if (!A || !a_scale || K % 16 || !aligned(A, 16) || !aligned(a_scale, 4)) return TAC_E_ARGUMENT;
  if (int s = check_product(Bt, b_scale, b_scale_type, bias, bias_type, Y, y_type, M, N, K)) return s;
  return run_product(A, Bt, a_scale, b_scale, b_scale_type, bias, bias_type, Y, y_type, M, N, K, false,
                     static_cast<cudaStream_t>(stream));
}

namespace {
// Codes and scales of M rows.
uint64_t rows_bytes(int M, int K) { return align256(uint64_t(M) * ((uint64_t(K) + 15) / 16 * 16)) + align256(uint64_t(M) * 4); }
}  // namespace

extern "C" uint64_t tac_linear_w8a8_workspace_bytes(int M, int K) {
  return M <= 0 || K <= 0 || few_rows(M, K) ? 0 : rows_bytes(M, K);
}

extern "C" uint64_t tac_linear_w8a8_best_workspace_bytes(int M, int N, int K) {
  return M <= 0 || N <= 0 || K <= 0 || one_launch(M, N, K, sm_count()) ? 0 : rows_bytes(M, K);
}

extern "C" int tac_linear_w8a8(const void* X, int x_type, int64_t ldx, const int8_t* Bt, const void* b_scale,
                               int b_scale_type, const void* bias, int bias_type, void* Y, int y_type, void* workspace,
                               uint64_t workspace_bytes, int M, int N, int K, void* stream) {
  if (!X || !type_ok(x_type) || (M > 1 && ldx < K) || !aligned(X, x_type == TAC_F32 ? 4 : 2)) return TAC_E_ARGUMENT;
  if (int s = check_product(Bt, b_scale, b_scale_type, bias, bias_type, Y, y_type, M, N, K)) return s;
  const int Kp = (K + 15) / 16 * 16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool room = workspace && aligned(workspace, 256) && workspace_bytes >= rows_bytes(M, K);
  if (few_rows(M, K) && !(room && !one_launch(M, N, K, sm_count()))) {
    W8RowsParams pp{};
    pp.g.b_scale = b_scale, pp.g.b_type = b_scale_type;
    pp.g.bias = bias, pp.g.bias_type = bias_type;
    pp.g.y = Y;
    pp.g.M = M, pp.g.N = N, pp.g.K = Kp;
    if (!(pp.g.fault = fault_word())) return TAC_E_CUDA;
    pp.x = X, pp.x_type = x_type, pp.ldx = ldx, pp.k_real = K;
    pp.x_vec = x_type != TAC_F32 && aligned(X, 16) && (M == 1 || ldx % 8 == 0);
    return y_type == TAC_F32 ? launch_rows<0>(pp, Bt, st) : y_type == TAC_F16 ? launch_rows<1>(pp, Bt, st) : launch_rows<2>(pp, Bt, st);
  }
  if (!room) return TAC_E_ARGUMENT;
  int8_t* q = static_cast<int8_t*>(workspace);
  float* s = reinterpret_cast<float*>(q + align256(uint64_t(M) * Kp));
  if (int e = launch_quant_rows(X, x_type, ldx, q, s, M, K, st)) return e;
  return run_product(q, Bt, s, b_scale, b_scale_type, bias, bias_type, Y, y_type, M, N, Kp, true, st);
}
