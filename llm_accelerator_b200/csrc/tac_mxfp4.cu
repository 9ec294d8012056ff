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
#include "tac_rows.cuh"
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
// A warp takes 256 columns of the four rows whose scales share 16 bytes (lane +
// 0, 32, 64, 96 of 128): a lane eight values of each, four lanes a block.
// Bound by instructions until 16-bit magnitudes were compared in pairs, the four
// rows' scale bytes changed places in two exchanges and places were 32 bits
// (8192 x 4096: 15.5 us, 5.5 TB/s; 21 with 123 instructions for eight values).
constexpr int kQmThreads = 256;
// ANY: 16-bit rows that begin anywhere.
template <typename T, bool ANY>
__global__ void __launch_bounds__(kQmThreads) mx_quant_kernel(const T* __restrict__ X, int64_t ldx, uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int M, int K, int vec, uint32_t tasks,
                                                              uint32_t k_stages) {
  after_previous();
  let_next();
  const uint32_t task = blockIdx.x * (kQmThreads / 32) + (threadIdx.x >> 5);
  if (task >= tasks) return;                     // a whole warp
  const int lane = threadIdx.x & 31;
  const uint32_t line = task / k_stages, chunk = task - line * k_stages;
  const int tile = int(line >> 5), r = int(line & 31), k = int(chunk) * kMxStageK + lane * 8, m0 = tile * 128 + r;
  const int ldc = (K + 31) / 32 * 16;
  const T* x = X + m0 * ldx + k;
  MxHeld<T> held[4];
  if constexpr (ANY) {
    AnySpan<1> rows[4];
    const int left = K - int(chunk) * kMxStageK;
#pragma unroll
    for (int g = 0; g < 4; ++g)                  // a row behind the last has nothing left
      rows[g].load(reinterpret_cast<const uint16_t*>(x - lane * 8 + g * 32 * ldx), 1, m0 + g * 32 < M ? left : -8);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      rows[g].values(1, left);
      held[g].u[0] = rows[g].v[0];
    }
  } else {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      held[g].clear();
      if (m0 + g * 32 < M) held[g].load(x + g * 32 * ldx, K - k, vec);
    }
  }
  uint8_t* c = codes + int64_t(m0) * ldc + k / 2;
  uint32_t bytes = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const uint32_t byte = scale_byte(held[g].block_exponent());
    bytes |= byte << (8 * g);
    float v[8];
    held[g].values(v);
    const uint32_t w = codes8(v, byte);
    if (m0 + g * 32 < M && k / 2 < ldc) *reinterpret_cast<uint32_t*>(c + int64_t(g) * 32 * ldc) = w;
  }
  // byte g of block b's lanes (b = lane / 4 % 4) becomes byte b of lanes g: a 4 x 4 transposition, halves and then quarters
  uint32_t o = __shfl_xor_sync(0xffffffffu, bytes, 8);
  bytes = lane & 8 ? __byte_perm(o, bytes, 0x7632) : __byte_perm(bytes, o, 0x5410);
  o = __shfl_xor_sync(0xffffffffu, bytes, 4);
  bytes = lane & 4 ? __byte_perm(o, bytes, 0x7351) : __byte_perm(bytes, o, 0x6240);
  if ((lane & 3) == 0)
    *reinterpret_cast<uint32_t*>(scales + ((int64_t(tile) * k_stages + chunk) * 2 + (lane >> 4)) * 512 + r * 16 + (lane & 12)) = bytes;
}

int64_t quant_tasks(int M, int k_stages) { return (int64_t(M) + 127) / 128 * 32 * k_stages; }
int64_t quant_ctas(int M, int k_stages) { return (quant_tasks(M, k_stages) + kQmThreads / 32 - 1) / (kQmThreads / 32); }

bool vec_rows(const void* X, int type, int64_t ldx, int M) { return aligned(X, 16) && (M == 1 || (ldx * elem(type)) % 16 == 0); }

int launch_quant(const void* X, int type, int64_t ldx, uint8_t* codes, uint8_t* scales, int M, int K, cudaStream_t st) {
  const int k_stages = int(mx_pieces(K) / 2);
  const int64_t tasks = quant_tasks(M, k_stages), ctas = quant_ctas(M, k_stages);
  if (tasks > 0x7fffffff) return TAC_E_ARGUMENT;             // rows of 4 TB
  const int vec = vec_rows(X, type, ldx, M);
  const auto go = [&](auto* x) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    if constexpr (sizeof(T) == 2) {
      if (!vec)
        return launch_behind(mx_quant_kernel<T, true>, unsigned(ctas), kQmThreads, 0, st, x, ldx, codes, scales, M, K, vec,
                             uint32_t(tasks), uint32_t(k_stages));
    }
    return launch_behind(mx_quant_kernel<T, false>, unsigned(ctas), kQmThreads, 0, st, x, ldx, codes, scales, M, K, vec,
                         uint32_t(tasks), uint32_t(k_stages));
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

// A warp has 256 columns of the eight rows whose scales share 32 bytes (two
// neighbours, and those 32, 64 and 96 behind them): a lane eight values of each.
// 8192 x 4096 to BF16: 16.5 us, 5.1 TB/s, bound by the writes; with one row a
// thread 21.  Float32 values are not a lane's eight but one of each block, 6111
// x 7579 in 36 us (eight a lane one by one took 184, in 16 bytes where rows
// allow it 49).
constexpr int kQmRows = 8;
__device__ __forceinline__ int64_t quant_row(int64_t tile, int pair, int g) { return tile * 128 + (g >> 1) * 32 + pair * 2 + (g & 1); }

template <typename T>
__global__ void __launch_bounds__(kQmThreads) mx_values_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                               T* __restrict__ Y, int M, int K, int vec, uint32_t tasks, uint32_t k_stages) {
  after_previous();
  let_next();
  const uint32_t task = blockIdx.x * (kQmThreads / 32) + (threadIdx.x >> 5);
  if (task >= tasks) return;
  const int lane = threadIdx.x & 31;
  const uint32_t line = task / k_stages, chunk = task - line * k_stages;
  const int64_t tile = line >> 4;
  const int pair = int(line & 15), k = int(chunk) * kMxStageK + lane * 8;
  const int64_t ldc = int64_t((K + 31) / 32) * 16;
  const uint4* sp = reinterpret_cast<const uint4*>(scales + ((tile * k_stages + chunk) * 2 + (lane >> 4)) * 512 + pair * 32);
  const uint4 even = __ldg(sp), odd = __ldg(sp + 1);
  const uint32_t word[kQmRows] = {even.x, odd.x, even.y, odd.y, even.z, odd.z, even.w, odd.w};
  uint32_t c[kQmRows];
#pragma unroll
  for (int g = 0; g < kQmRows; ++g) {
    const int64_t m = quant_row(tile, pair, g);
    c[g] = m < M && k < K ? __ldg(reinterpret_cast<const uint32_t*>(codes + m * ldc + k / 2)) : 0u;
  }
#pragma unroll
  for (int g = 0; g < kQmRows; ++g) {
    const int64_t m = quant_row(tile, pair, g);
    if (m >= M) continue;                        // whole warps
    const uint32_t byte = (word[g] >> (8 * ((lane >> 2) & 3))) & 0xffu;
    // 2^(byte - 127); the byte 0 is half the smallest normal number, 255 NaN
    const float s = byte == 255 ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float(byte << 23) : __uint_as_float(0x00400000u);
    if constexpr (sizeof(T) == 4) {              // a block of 32 columns at a time, for runs of 128 bytes wherever rows begin
      const int k0 = int(chunk) * kMxStageK + lane;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t of = __shfl_sync(0xffffffffu, c[g], j * 4 + (lane >> 3));
        const float2 f = __half22float2(e2m1x2((of >> (4 * (lane & 6))) & 0xffu));
        const float v = (lane & 1 ? f.y : f.x) * __shfl_sync(0xffffffffu, s, j * 4);
        if (k0 + j * 32 < K) Y[m * K + k0 + j * 32] = v;
      }
    } else {
      T* y = Y + m * K + k;
      union {
        uint4 u;
        T t[8];
      } a;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(e2m1x2((c[g] >> (8 * j)) & 0xffu));
        from_f(a.t[2 * j], f.x * s);
        from_f(a.t[2 * j + 1], f.y * s);
      }
      if (vec) {
        if (k < K) *reinterpret_cast<uint4*>(y) = a.u;
      } else {
        AnySpan<1> row;
        row.v[0] = a.u;
        row.store(reinterpret_cast<uint16_t*>(y - lane * 8), 1, K - int(chunk) * kMxStageK);
      }
    }
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
  bool spread;               // pairs without a tile keep the quantiser's CTAs apart
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
  const int part = split > 1 ? std::max(mx_sk_part_bytes(p.tn), sm100::tmem_least_smem(mx_sk_cols(p.tn, p.stages))) : 0;
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
  attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  return status(cudaLaunchKernelEx(&cfg, mx_splitk_kernel<YT>, tw, ta, p));
}

// Scales of rows as 32-bit words: a box is a stage of `pieces` times 128 rows; rows past the last read as 0.
bool map_scales(CUtensorMap* m, const uint8_t* base, int k_stages, int rows, int pieces) {
  const cuuint64_t dims[2] = {cuuint64_t(k_stages) * (kMxSfBytes / 4), cuuint64_t((rows + 127) / 128)};
  const cuuint64_t strides[1] = {cuuint64_t(k_stages) * kMxSfBytes};
  const cuuint32_t box[2] = {kMxSfBytes / 4, cuuint32_t(pieces)};
  return tmap_encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// Tokens of a pair tile: the number that leaves the least work on the fullest
// pair.  A stage costs, in nanoseconds: mostly its operands' loads.  The costs are
// those of long K; the epilogue is not in them.
int pair_tokens(int M, int N, int clusters) {
  constexpr int kStageCost[4] = {273, 315, 436, 499};      // 64, 128, 192, 256 tokens (4096^3)
  const int64_t wt = (N + 255) / 256;
  int best = 0;
  int64_t cost = 0;
  for (int tn = 256; tn >= 64; tn -= 64) {
    const int64_t tiles = wt * ((M + tn - 1) / tn), c = (tiles + clusters - 1) / clusters * kStageCost[tn / 64 - 1];
    if (!best || c < cost) best = tn, cost = c;
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
    if (cudaFuncSetAttribute(mx_pair_kernel<YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, MxPairCfg::kSmem) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(2 * (sms / 2));
      cfg.blockDim = dim3(MxPairCfg::kThreads);
      cfg.dynamicSmemBytes = MxPairCfg::kSmem;
      if (cudaOccupancyMaxActiveClusters(&n, mx_pair_kernel<YT>, &cfg) != cudaSuccess) n = 0;
    }
    cudaGetLastError();
    clusters[dev] = std::min(n, sms / 2);
    done[dev] = true;
  }
  return clusters[dev];
}

template <int YT>
int launch_pair(const MxOperands& o, MxParams p, int clusters, int tn, cudaStream_t st) {
  MxPairParams pp{};
  p.tn = tn;
  pp.g = p;
  pp.w_tiles = (p.N + 255) / 256;
  pp.t_tiles = (p.M + tn - 1) / tn;
  CUtensorMap tw, ta, tws, tas;
  if (!map_rows(&tw, o.b_codes, o.K, p.N, 128) || !map_rows(&ta, o.a_codes, o.K, p.M, tn / 2) ||
      !map_scales(&tws, p.b_scale, p.k_stages, p.N, 1) || !map_scales(&tas, p.a_scale, p.k_stages, p.M, tn > 128 ? 2 : 1))
    return TAC_E_CUDA;
  const int64_t tiles = int64_t(pp.w_tiles) * pp.t_tiles;
  if (tiles > (1 << 30)) return TAC_E_ARGUMENT;
  // Behind the quantiser this kernel starts while that one runs, but not on an SM that holds two of its CTAs.  Where it has one
  // for each SM at most, pairs without a tile keep the last call's SMs from being free, on which the quantiser's CTAs would
  // gather: 300 x 9000 x 768 in 7.2 us, 9.3 without them (float32 rows 7.7 and 8.9).  The quantiser of 16-bit rows that begin
  // anywhere has 58 registers a thread, with which not even one CTA fits beside a pair's, and gains nothing (500 x 8192 x 512
  // in 8.3 us with them, 7.6 without).
  const bool fill = o.spread && quant_ctas(p.M, p.k_stages) <= 2 * clusters && tiles * 2 > clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * int(fill ? clusters : std::min<int64_t>(tiles, clusters)));
  cfg.blockDim = dim3(MxPairCfg::kThreads);
  cfg.dynamicSmemBytes = MxPairCfg::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return status(cudaLaunchKernelEx(&cfg, mx_pair_kernel<YT>, tw, ta, tws, tas, pp));
}

// Pairs from 65 tokens on, unless K is long and there are tiles for fewer than
// an eighth of the pairs: a stage costs a pair 0.23 us, sharing K 3 us.
// Microseconds, pairs / split K:
//   64 x 4096 x 4096    7.9 /  7.7   100 x 4096 x 4096    8.2 / 10.6   128 x 16384 x 4096  11.8 / 12.4
//   20 x 50257 x 768    8.1 /  6.8   100 x 50257 x 768   10.6 / 13.6    85 x 250 x 2048     5.0 /  6.9
//   85 x 250 x 4096     6.9 /  7.9   200 x 60 x 4096      6.7 /  8.7    85 x 640 x 8192    10.4 /  8.7
// (M x N x K.)
constexpr int kPairStages = 24;
template <int YT>
int pick_product(const MxOperands& o, const MxParams& p, cudaStream_t st) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  const int clusters = p.M > 64 ? pair_clusters<YT>(dev) : 0;
  if (clusters > 0) {
    const int tn = pair_tokens(p.M, p.N, clusters);
    if (p.k_stages <= kPairStages || int64_t((p.N + 255) / 256) * ((p.M + tn - 1) / tn) * 8 >= clusters) return launch_pair<YT>(o, p, clusters, tn, st);
  }
  return launch_splitk<YT>(o, p, st);
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
                int bias_type, void* Y, int y_type, int M, int N, int K, bool after_rows, bool spread, cudaStream_t st) {
  MxParams p{};
  p.a_scale = a_scales, p.b_scale = b_scales;
  p.bias = bias, p.bias_type = bias_type;
  p.y = Y;
  p.M = M, p.N = N;
  p.k_stages = int(mx_pieces(K) / 2);
  p.after_rows = after_rows;
  if (!(p.fault = fault_word())) return TAC_E_CUDA;
  const MxOperands o{a_codes, b_codes, K, spread};
  return y_type == TAC_F32 ? pick_product<0>(o, p, st) : y_type == TAC_F16 ? pick_product<1>(o, p, st) : pick_product<2>(o, p, st);
}

// ---- few rows -------------------------------------------------------------------------------------------------------
struct MxRowsShape {
  int tn, split, per;        // tokens of a tile, CTAs that share a tile's stages, stages of a CTA at most
  int64_t w_tiles, t_tiles;
};
// The largest tile of at most 64 rows of which each CTA quantises its part at once, if there is a CTA for each SM at most;
// else tn is 0.  (More rows are faster in two launches: 300 x 768 x 768 in 5.5 us, 6.8 in one.)
MxRowsShape rows_shape(int M, int N, int K, int sms) {
  MxRowsShape r{};
  if (M > 64) return r;
  r.w_tiles = (int64_t(N) + 127) / 128;
  const int k_stages = int(mx_pieces(K) / 2);
  for (int tn = M <= 16 ? 16 : M <= 32 ? 32 : 64; tn >= 16; tn /= 2) {
    r.t_tiles = (M + tn - 1) / tn;
    const int64_t tiles = r.w_tiles * r.t_tiles;
    if (tiles > sms) break;
    r.split = splits(tiles, k_stages, tn, sms);
    r.per = (k_stages + r.split - 1) / r.split;
    if (r.per * std::min(M, tn) * 32 <= 256 * kMxRowsHeld) {
      r.tn = tn;
      break;
    }
  }
  return r;
}

bool one_launch(int M, int N, int K, int sms) { return sms && rows_shape(M, N, K, sms).tn; }

template <typename T, int YT>
int launch_rows_as(MxRowsParams pp, const MxOperands& o, cudaStream_t st) {
  static bool smem_set[64] = {};
  int dev = 0;
  const int sms = sm_count();
  if (!sms || cudaGetDevice(&dev) != cudaSuccess) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (int e = status(cudaFuncSetAttribute(mx_rows_kernel<T, YT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMxMaxSmem))) return e;
    smem_set[dev] = true;
  }
  MxParams& p = pp.g;
  const MxRowsShape r = rows_shape(p.M, p.N, o.K, sms);
  p.tn = r.tn;
  const int rows = r.per * mx_rows_bytes(r.tn), sb = kMxWBytes + kMxSfBytes;
  p.stages = std::min({r.per, kMxSkStages, (kMxMaxSmem - 1024 - rows) / sb});     // the rows are 192 KB at most, of one token
  const int part = r.split > 1 ? std::max(mx_sk_part_bytes(r.tn), sm100::tmem_least_smem(mx_sk_cols(r.tn, p.stages))) : 0;
  CUtensorMap tw;
  if (!map_rows(&tw, o.b_codes, o.K, p.N, 128)) return TAC_E_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(r.w_tiles), unsigned(r.t_tiles), r.split);
  cfg.blockDim = dim3(kMxRowsThreads);
  cfg.dynamicSmemBytes = std::max(p.stages * sb + rows, part) + 1024;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = r.split;
  cfg.attrs = attr;
  cfg.numAttrs = r.split > 1 ? 2 : 1;
  return status(cudaLaunchKernelEx(&cfg, mx_rows_kernel<T, YT>, tw, pp));
}

template <typename T>
int launch_rows(const MxRowsParams& pp, const MxOperands& o, int y_type, cudaStream_t st) {
  return y_type == TAC_F32 ? launch_rows_as<T, 0>(pp, o, st) : y_type == TAC_F16 ? launch_rows_as<T, 1>(pp, o, st) : launch_rows_as<T, 2>(pp, o, st);
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
  const int vec = K % 8 == 0 && aligned(Y, 16), k_stages = int(mx_pieces(K) / 2);
  const int64_t tasks = (int64_t(M) + 127) / 128 * 16 * k_stages, ctas = (tasks + kQmThreads / 32 - 1) / (kQmThreads / 32);
  if (tasks > 0x7fffffff) return TAC_E_ARGUMENT;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const auto go = [&](auto* y) {
    using T = std::remove_pointer_t<decltype(y)>;
    return launch_behind(mx_values_kernel<T>, unsigned(ctas), kQmThreads, 0, st, codes, scales, y, M, K, vec, uint32_t(tasks),
                  uint32_t(k_stages));
  };
  if (y_type == TAC_F32) return go(static_cast<float*>(Y));
  if (y_type == TAC_F16) return go(static_cast<__half*>(Y));
  return go(static_cast<__nv_bfloat16*>(Y));
}

extern "C" int tac_mxfp4_gemm(const uint8_t* a_codes, const uint8_t* a_scales, const uint8_t* b_codes, const uint8_t* b_scales,
                              const void* bias, int bias_type, void* Y, int y_type, int M, int N, int K, void* stream) {
  if (!a_codes || !a_scales || !aligned(a_codes, 16) || !aligned(a_scales, 16)) return TAC_E_ARGUMENT;
  if (int s = check_product(b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K)) return s;
  return run_product(a_codes, a_scales, b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K, false, false, static_cast<cudaStream_t>(stream));
}

extern "C" uint64_t tac_linear_mxfp4_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || one_launch(M, N, K, sm_count())) return 0;
  return align256(code_bytes(M, K)) + align256(scale_bytes(M, K));
}

extern "C" int tac_linear_mxfp4(const void* X, int x_type, int64_t ldx, const uint8_t* b_codes, const uint8_t* b_scales, const void* bias,
                                int bias_type, void* Y, int y_type, void* workspace, uint64_t workspace_bytes, int M, int N, int K,
                                void* stream) {
  if (!X || !type_ok(x_type) || (M > 1 && ldx < K) || !aligned(X, elem(x_type))) return TAC_E_ARGUMENT;
  if (int s = check_product(b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K)) return s;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (one_launch(M, N, K, sm_count())) {
    MxRowsParams pp{};
    pp.g.b_scale = b_scales;
    pp.g.bias = bias, pp.g.bias_type = bias_type;
    pp.g.y = Y;
    pp.g.M = M, pp.g.N = N;
    pp.g.k_stages = int(mx_pieces(K) / 2);
    if (!(pp.g.fault = fault_word())) return TAC_E_CUDA;
    pp.x = X, pp.ldx = ldx, pp.K = K;
    pp.x_vec = vec_rows(X, x_type, ldx, M);
    const MxOperands o{nullptr, b_codes, K, false};
    return x_type == TAC_F32   ? launch_rows<float>(pp, o, y_type, st)
           : x_type == TAC_F16 ? launch_rows<__half>(pp, o, y_type, st)
                               : launch_rows<__nv_bfloat16>(pp, o, y_type, st);
  }
  if (!workspace || !aligned(workspace, 256) || workspace_bytes < tac_linear_mxfp4_workspace_bytes(M, N, K)) return TAC_E_ARGUMENT;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + align256(code_bytes(M, K));
  if (int e = launch_quant(X, x_type, ldx, codes, scales, M, K, st)) return e;
  return run_product(codes, scales, b_codes, b_scales, bias, bias_type, Y, y_type, M, N, K, true,
                     x_type == TAC_F32 || vec_rows(X, x_type, ldx, M), st);
}
