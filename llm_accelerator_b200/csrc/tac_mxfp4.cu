// 4-bit microscaled rows (E2M1 codes, blocks of 32 values with a power of two
// each): the row quantiser, the values of such rows, their products
// (tac_mxfp4.cuh) and linear layers of floating-point rows.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "../../include/taccel_b200.h"
#include "tac_launch.cuh"
#include "tac_mxfp4.cuh"
#include "tac_tmap.h"

namespace tac {
int* gemm_fault_word();
}

namespace {

using namespace tac;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
bool type_ok(int t) { return t == TAC_F32 || t == TAC_F16 || t == TAC_BF16; }
int elem(int type) { return type == TAC_F32 ? 4 : 2; }

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

int64_t blocks_of(int64_t K) { return (K + 31) / 32; }
int64_t code_bytes(int64_t rows, int64_t K) { return rows * blocks_of(K) * 16; }
int64_t scale_bytes(int64_t rows, int64_t K) { return (rows + 127) / 128 * mx_pieces(K) * 512; }

// ---- row quantiser --------------------------------------------------------------------------------------------------
// scale byte = max(floor(log2 max |x|) - 2 + 127, 0), codes E2M1(x / 2^(byte -
// 127)) to the nearest, ties to the even code, magnitudes at most 6; a block
// with an infinity or a NaN gets the byte 255 (NaN) and codes 0.  Powers of two
// divide exactly, so nothing here rounds but the code itself.
template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ void load8(const T* x, int k, int K, bool vec, float (&v)[8]) {
  if (vec && k + 8 <= K) {
    constexpr int kPer = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += kPer) {
      union {
        uint4 u;
        T t[kPer];
      } a;
      a.u = __ldg(reinterpret_cast<const uint4*>(x + k + i));
#pragma unroll
      for (int j = 0; j < kPer; ++j) v[i + j] = to_f(a.t[j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_f(x[k + j]) : 0.f;
  }
}

// Largest magnitude of a block whose four lanes hold eight values each, as bits: infinities and NaN order above all others.
__device__ __forceinline__ uint32_t block_max(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 2));
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t max_bits) {
  const uint32_t e = max_bits >> 23;
  return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}
// Eight codes, value 0 in the lowest four bits.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], uint32_t byte) {
  if (byte == 255) return 0u;
  const float inv = __uint_as_float((254u - byte) << 23);
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}\n"
      : "=r"(r)
      : "f"(v[0] * inv), "f"(v[1] * inv), "f"(v[2] * inv), "f"(v[3] * inv), "f"(v[4] * inv), "f"(v[5] * inv), "f"(v[6] * inv),
        "f"(v[7] * inv));
  return r;
}

// A warp takes 256 columns of the four rows whose scales share 16 bytes (lane +
// 0, 32, 64, 96 of 128): a lane eight values of each, four lanes a block.
constexpr int kQmThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kQmThreads) mx_quant_kernel(const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int M, int K, int vec, int64_t tasks,
                                                              int k_stages) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int64_t task = int64_t(blockIdx.x) * (kQmThreads / 32) + (threadIdx.x >> 5);
  if (task >= tasks) return;                     // a whole warp
  const int lane = threadIdx.x & 31;
  const int chunk = int(task % k_stages), r = int(task / k_stages % 32);
  const int64_t tile = task / k_stages / 32;
  const int k = chunk * kMxStageK + lane * 8;
  const int64_t ldc = int64_t((K + 31) / 32) * 16;
  float v[4][8];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t m = tile * 128 + g * 32 + r;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[g][j] = 0.f;
    if (m < M) load8(X + m * ldx, k, K, vec, v[g]);
  }
  uint32_t word[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int64_t m = tile * 128 + g * 32 + r;
    const uint32_t byte = scale_byte(block_max(v[g]));
    const uint32_t c = codes8(v[g], byte);
    if (m < M && k / 2 < ldc) *reinterpret_cast<uint32_t*>(codes + m * ldc + k / 2) = c;
    // the bytes of a lane's four blocks, lanes 0 and 16 of each half
    uint32_t b = byte << (8 * ((lane >> 2) & 3));
    b |= __shfl_xor_sync(0xffffffffu, b, 4);
    word[g] = b | __shfl_xor_sync(0xffffffffu, b, 8);
  }
  if ((lane & 15) == 0)
    *reinterpret_cast<uint4*>(scales + ((tile * k_stages + chunk) * 2 + (lane >> 4)) * 512 + r * 16) =
        make_uint4(word[0], word[1], word[2], word[3]);
}

int launch_quant(const void* X, int type, int64_t ldx, uint8_t* codes, uint8_t* scales, int M, int K, cudaStream_t st) {
  const int k_stages = int(mx_pieces(K) / 2);
  const int64_t tasks = (int64_t(M) + 127) / 128 * 32 * k_stages, ctas = (tasks + kQmThreads / 32 - 1) / (kQmThreads / 32);
  if (ctas > 0x7fffffff) return TAC_E_ARGUMENT;
  const int vec = aligned(X, 16) && (M == 1 || (ldx * elem(type)) % 16 == 0);
  const auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    return launch(mx_quant_kernel<T>, unsigned(ctas), kQmThreads, 0, st, x, ldx, codes, scales, M, K, vec, tasks, k_stages);
  };
  if (type == TAC_F32) return go(static_cast<const float*>(X));
  if (type == TAC_F16) return go(static_cast<const __half*>(X));
  return go(static_cast<const __nv_bfloat16*>(X));
}

// ---- values ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void from_f(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }

// Two codes' values as halves (exact).
__device__ __forceinline__ __half2 e2m1x2(uint32_t byte) {
  uint32_t r;
  asm("{\n\t.reg .b8 b, t;\n\tmov.b32 {b, t, t, t}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}\n" : "=r"(r) : "r"(byte));
  return *reinterpret_cast<const __half2*>(&r);
}

// Eight values a thread; a row is cut into `cuts` CTAs.
template <typename T>
__global__ void __launch_bounds__(kQmThreads) mx_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                               T* __restrict__ Y, int K, int vec, int cuts, int k_stages) {
  const int64_t m = blockIdx.x / cuts;
  const int k = ((blockIdx.x % cuts) * kQmThreads + threadIdx.x) * 8;
  if (k >= K) return;
  const int64_t ldc = int64_t((K + 31) / 32) * 16;
  const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(codes + m * ldc + k / 2));
  const int kb = k / 32;
  const uint32_t byte = __ldg(scales + ((m / 128) * k_stages * 2 + kb / 4) * 512 + (m % 32) * 16 + (m % 128) / 32 * 4 + kb % 4);
  // 2^(byte - 127); the byte 0 is half the smallest normal number, 255 NaN
  const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
  T* y = Y + m * K + k;
  union {
    uint4 u[8 * sizeof(T) / 16];
    T t[8];
  } a;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(e2m1x2((c >> (8 * j)) & 0xffu));
    from_f(a.t[2 * j], f.x * s);
    from_f(a.t[2 * j + 1], f.y * s);
  }
  if (vec) {
#pragma unroll
    for (int i = 0; i < int(8 * sizeof(T) / 16); ++i) reinterpret_cast<uint4*>(y)[i] = a.u[i];
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < K) y[j] = a.t[j];
  }
}

// ---- products -------------------------------------------------------------------------------------------------------
bool map_rows(CUtensorMap* m, const uint8_t* base, int K, int rows, int box_rows) {
  const cuuint64_t bytes = cuuint64_t(blocks_of(K) * 16);
  const cuuint64_t dims[2] = {bytes, cuuint64_t(rows)}, strides[1] = {bytes};
  const cuuint32_t box[2] = {128, cuuint32_t(box_rows)};
  return tmap_encode_u8(m, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

constexpr int kMxMaxSmem = 224 * 1024;

// CTAs that share a tile's stages: as many as find an SM each, with four stages or more a CTA (one for 16 tokens).
int splits(int64_t tiles, int k_stages, int tn, int sms) {
  int split = 1;
  while (split < 8 && 2 * split * (tn > 16 ? 4 : 1) <= k_stages && tiles * split * 2 <= sms) split *= 2;
  return split;
}

struct MxOperands {
  const uint8_t* a_codes;
  const uint8_t* b_codes;
  int K;
};

template <int YT>
int launch_splitk(const MxOperands& o, MxParams p, cudaStream_t st) {
  static bool smem_set[64] = {};
  int dev = 0;
  const int sms = sm_count();
  if (!sms || cudaGetDevice(&dev) != cudaSuccess) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (int e = status(cudaFuncSetAttribute(mx_splitk_kernel<YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMxMaxSmem))) return e;
    smem_set[dev] = true;
  }
  p.tn = p.M <= 16 ? 16 : p.M <= 32 ? 32 : p.M <= 64 ? 64 : 128;
  const int64_t tiles = int64_t((p.N + 127) / 128) * ((p.M + p.tn - 1) / p.tn);
  const int split = splits(tiles, p.k_stages, p.tn, sms);
  const int per = (p.k_stages + split - 1) / split, sb = mx_sk_stage_bytes(p.tn);
  // in flight: 96 KB where two CTAs share an SM, else twice that
  p.stages = std::min(std::min(per, kMxSkStages), std::max(2, (tiles * split > sms ? 96 : 190) * 1024 / sb));
  const int part = split > 1 ? mx_sk_part_bytes(p.tn) : 0;
  CUtensorMap tw, ta;
  if (!map_rows(&tw, o.b_codes, o.K, p.N, 128) || !map_rows(&ta, o.a_codes, o.K, p.M, p.tn)) return TAC_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.N + 127) / 128, (p.M + p.tn - 1) / p.tn, split);
  cfg.blockDim = dim3(kMxSkThreads);
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
  return status(cudaLaunchKernelEx(&cfg, mx_splitk_kernel<YT>, tw, ta, p));
}

// Checks that both products share; also the limits of the grids.
int check_product(const void* b_codes, const void* b_scales, const void* bias, int bias_type, const void* Y, int y_type, int M, int N,
                  int K) {
  if (!b_codes || !b_scales || !Y || M <= 0 || N <= 0 || K <= 0 || !type_ok(y_type) || (bias && !type_ok(bias_type))) return TAC_E_ARGUMENT;
  if (!aligned(b_codes, 16) || !aligned(b_scales, 16) || !aligned(Y, elem(y_type)) || (bias && !aligned(bias, elem(bias_type))))
    return TAC_E_ARGUMENT;
  return M > (1 << 20) || N > (1 << 30) || K > (1 << 24) ? TAC_E_ARGUMENT : TAC_OK;
}

int run_product(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales, const void* bias,
                int bias_type, void* Y, int y_type, int M, int N, int K, bool after_rows, cudaStream_t st) {
  MxParams p{};
  p.a_scale = a_scales, p.b_scale = b_scales;
  p.bias = bias, p.bias_type = bias_type;
  p.y = Y;
  p.M = M, p.N = N;
  p.k_stages = int(mx_pieces(K) / 2);
  p.after_rows = after_rows;
  if (!(p.fault = fault_word())) return TAC_E_CUDA;
  const MxOperands o{a_codes, b_codes, K};
  return y_type == TAC_F32 ? launch_splitk<0>(o, p, st) : y_type == TAC_F16 ? launch_splitk<1>(o, p, st) : launch_splitk<2>(o, p, st);
}

uint64_t align256(uint64_t v) { return (v + 255) & ~uint64_t(255); }

}  // namespace

extern "C" uint64_t tac_mxfp4_code_bytes(int rows, int K) { return rows <= 0 || K <= 0 ? 0 : uint64_t(code_bytes(rows, K)); }
extern "C" uint64_t tac_mxfp4_scale_bytes(int rows, int K) { return rows <= 0 || K <= 0 ? 0 : uint64_t(scale_bytes(rows, K)); }

extern "C" int tac_mxfp4_quantize(const void* X, int x_type, int64_t ldx, uint8_t* codes, uint8_t* scales, int M, int K, void* stream) {
  if (!X || !codes || !scales || !type_ok(x_type) || M <= 0 || K <= 0 || K > (1 << 24) || (M > 1 && ldx < K) || !aligned(codes, 16) ||
      !aligned(scales, 16) || !aligned(X, elem(x_type)))
    return TAC_E_ARGUMENT;
  return launch_quant(X, x_type, ldx, codes, scales, M, K, static_cast<cudaStream_t>(stream));
}

extern "C" int tac_mxfp4_values(const uint8_t* codes, const uint8_t* scales, void* Y, int y_type, int M, int K, void* stream) {
  if (!codes || !scales || !Y || !type_ok(y_type) || M <= 0 || K <= 0 || K > (1 << 24) || !aligned(codes, 16) || !aligned(scales, 16) ||
      !aligned(Y, elem(y_type)))
    return TAC_E_ARGUMENT;
  const int64_t cuts = (int64_t(K) + kQmThreads * 8 - 1) / (kQmThreads * 8);
  if (M * cuts > 0x7fffffff) return TAC_E_ARGUMENT;
  const int vec = K % 8 == 0 && aligned(Y, 16), k_stages = int(mx_pieces(K) / 2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto* y) {
    using T = std::remove_pointer_t<decltype(y)>;
    return launch(mx_values_kernel<T>, unsigned(M * cuts), kQmThreads, 0, st, codes, scales, y, K, vec, int(cuts), k_stages);
  };
  if (y_type == TAC_F32) return go(static_cast<float*>(Y));
  if (y_type == TAC_F16) return go(static_cast<__half*>(Y));
  return go(static_cast<__nv_bfloat16*>(Y));
}

extern "C" int tac_mxfp4_gemm(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales,
                              const void* bias, int bias_type, void* Y, int y_type, int M, int N, int K, void* stream) {
  if (!a_codes || !a_scales || !aligned(a_codes, 16) || !aligned(a_scales, 16)) return TAC_E_ARGUMENT;
  if (int s = check_product(b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K)) return s;
  return run_product(a_codes, a_scales, b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K, false, static_cast<cudaStream_t>(stream));
}

extern "C" uint64_t tac_linear_mxfp4_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return align256(code_bytes(M, K)) + align256(scale_bytes(M, K));
}

extern "C" int tac_linear_mxfp4(const void* X, int x_type, int64_t ldx, const uint8_t* b_codes, const uint8_t* b_scales, const void* bias,
                                int bias_type, void* Y, int y_type, void* workspace, uint64_t workspace_bytes, int M, int N, int K,
                                void* stream) {
  if (!X || !type_ok(x_type) || (M > 1 && ldx < K) || !aligned(X, elem(x_type))) return TAC_E_ARGUMENT;
  if (int s = check_product(b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K)) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < tac_linear_mxfp4_workspace_bytes(M, N, K)) return TAC_E_ARGUMENT;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + align256(code_bytes(M, K));
  if (int e = launch_quant(X, x_type, ldx, codes, scales, M, K, st)) return e;
  return run_product(codes, scales, b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K, true, st);
}
