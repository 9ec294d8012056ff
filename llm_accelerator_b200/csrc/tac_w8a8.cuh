// INT8 products with a scale for each token and each output channel:
//   y[m, n] = (sum_k A[m, k] Bt[n, k]) * a_scale[m] * b_scale[n] (+ bias[n])
// A [M, K] and Bt [N, K] int8, both K-major; int32 sums, a float32 epilogue
// and one rounding to the output's type.
//
// Orientation: the 128 rows of the MMA are output channels and its columns
// are tokens, so the token tile is any multiple of 16 (few padded tokens in a
// ragged batch), a thread of the epilogue holds one channel (its scale and
// bias sit in registers), and a warp stores 32 consecutive channels of one
// token whatever the alignment of N.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "tac_sm100.cuh"

namespace tac {

enum W8Fault : int { W8_TIMEOUT_EMPTY = 11, W8_TIMEOUT_FULL = 12, W8_TIMEOUT_ACC = 13, W8_TIMEOUT_DRAIN = 14 };

// float32 value of element i of a TAC_F32 / TAC_F16 / TAC_BF16 array
__device__ __forceinline__ float ld_any(const void* p, int type, int64_t i) {
  if (type == 0) return __ldg(static_cast<const float*>(p) + i);
  const uint16_t b = __ldg(static_cast<const uint16_t*>(p) + i);
  return type == 1 ? __half2float(__ushort_as_half(b)) : __uint_as_float(uint32_t(b) << 16);
}

__device__ __forceinline__ void st_any(void* p, int type, int64_t i, float v) {
  if (type == 0) static_cast<float*>(p)[i] = v;
  else if (type == 1) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

struct W8Params {
  const float* a_scale;
  const void* b_scale;
  const void* bias;          // or null
  void* y;
  int b_type, bias_type, y_type;
  int M, N, K;
  int k_blocks;              // 128-byte blocks of K
  int tn;                    // tokens of a tile
  int stages;
  int* fault;
};

__device__ __forceinline__ float w8_value(int acc, float as, float bs, float bias, bool has_bias) {
  const float y = __fmul_rn(__fmul_rn(__int2float_rn(acc), as), bs);
  return has_bias ? __fadd_rn(y, bias) : y;
}

// ---- split-K over a cluster -----------------------------------------------------------------------------------------
// A 128-channel x tn-token tile for each cluster of S CTAs; CTA r sums its
// share of the K blocks, leaves the int32 partial sums in its shared memory,
// and after a cluster barrier finishes every S-th token from all S partials
// (integer sums: the split never changes a result).  For products with too
// few tiles for 148 SMs, where streaming the weights is the work.
//   warp 0      TMA loads of both operands, warp 1 MMAs, warps 2..5 epilogue.
constexpr int kSkThreads = 192;
constexpr int kSkWBytes = 128 * 128;

__host__ __device__ constexpr int sk_stage_bytes(int tn) { return kSkWBytes + tn * 128; }

__global__ void __launch_bounds__(kSkThreads)
    w8_splitk_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, W8Params p) {
  constexpr int kMaxStages = 8;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], acc_bar;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ float as_s[256];

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128, m0 = blockIdx.y * p.tn;
  const int nsplit = gridDim.z, rank = blockIdx.z;
  const int kb0 = int(int64_t(p.k_blocks) * rank / nsplit), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / nsplit);
  const int S = p.stages, stage_bytes = sk_stage_bytes(p.tn);
  const uint32_t cols = p.tn <= 32 ? 32 : p.tn <= 64 ? 64 : p.tn <= 128 ? 128 : 256;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full_bar[s], 1);
      sm100::mbar_init(&empty_bar[s], 1);
    }
    sm100::mbar_init(&acc_bar, 1);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  if (warp == 1) sm100::tmem_alloc(&tmem_base, cols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t s = it % S, ph = (it / S) & 1;
        if (!sm100::mbar_wait(&empty_bar[s], ph ^ 1, p.fault, W8_TIMEOUT_EMPTY) || *abort_v) {
          *abort_v = 1;
          break;
        }
        uint8_t* st = smem + s * stage_bytes;
        sm100::mbar_arrive_expect_tx(&full_bar[s], stage_bytes);
        sm100::tma_load_2d(st, &tm_w, kb * 128, n0, &full_bar[s]);
        sm100::tma_load_2d(st + kSkWBytes, &tm_a, kb * 128, m0, &full_bar[s]);
      }
      // the copies still in flight land before the CTA goes on
      const uint32_t first = it > uint32_t(S) ? it - S : 0;
      for (uint32_t j = first; j < it; ++j)
        sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, W8_TIMEOUT_DRAIN);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = sm100::idesc_i8(128, p.tn, 0);
      uint32_t it = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const uint32_t s = it % S, ph = (it / S) & 1;
        if (!sm100::mbar_wait(&full_bar[s], ph, p.fault, W8_TIMEOUT_FULL) || *abort_v) {
          *abort_v = 1;
          break;
        }
        sm100::tc_fence_after();
        const uint32_t w_addr = sm100::smem_u32(smem + s * stage_bytes);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          sm100::mma_i8(tmem, sm100::smem_desc_sw128(w_addr + k * 32, 16, 1024),
                        sm100::smem_desc_sw128(w_addr + kSkWBytes + k * 32, 16, 1024), idesc, (kb > kb0) || k);
        sm100::mma_commit(&empty_bar[s]);
      }
      // arrives once every MMA has completed, also after a failed wait
      sm100::mma_commit(&acc_bar);
      sm100::mbar_wait(&acc_bar, 0, p.fault, W8_TIMEOUT_DRAIN);
    }
    __syncwarp();
  }
  const int row = (warp & 3) * 32 + lane;     // TMEM lane = channel of the tile (warps 2..5)
  const int n = n0 + row;
  float bs = 0.f, bias = 0.f;
  const bool has_bias = p.bias != nullptr;
  bool acc_ok = false;
  if (warp >= 2) {
    if (n < p.N) {
      bs = ld_any(p.b_scale, p.b_type, n);
      if (has_bias) bias = ld_any(p.bias, p.bias_type, n);
    }
    for (int i = threadIdx.x - 64; i < p.tn; i += 128) as_s[i] = m0 + i < p.M ? __ldg(p.a_scale + m0 + i) : 0.f;
    asm volatile("bar.sync 1, 128;\n" ::: "memory");   // as_s, among the epilogue's warps
    acc_ok = sm100::mbar_wait(&acc_bar, 0, p.fault, W8_TIMEOUT_ACC);
    __syncwarp();
    sm100::tc_fence_after();
  }
  const uint32_t t_addr = tmem + (uint32_t((warp & 3) * 32) << 16);
  if (nsplit == 1) {
    if (warp >= 2 && acc_ok) {
      for (int c = 0; c < p.tn; c += 32) {
        uint32_t v[32];
        __syncwarp();
        sm100::tmem_ld32(t_addr + c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int m = m0 + c + j;
          if (c + j < p.tn && m < p.M && n < p.N)
            st_any(p.y, p.y_type, int64_t(m) * p.N + n, w8_value(int(v[j]), as_s[c + j], bs, bias, has_bias));
        }
      }
    }
  } else {
    int* part = reinterpret_cast<int*>(smem);            // [tn][128], over the stages: every copy and MMA has ended
    if (warp >= 2) {
      for (int c = 0; c < p.tn; c += 32) {
        uint32_t v[32];
        __syncwarp();
        sm100::tmem_ld32(t_addr + c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < p.tn) part[(c + j) * 128 + row] = int(v[j]);
      }
    }
    sm100::cluster_sync();
    if (warp >= 2) {
      for (int c = rank; c < p.tn; c += nsplit) {
        const int m = m0 + c;
        if (m >= p.M) break;
        int acc = 0;
        for (int r = 0; r < nsplit; ++r) {
          int v;
          asm volatile("ld.shared::cluster.s32 %0, [%1];\n" : "=r"(v) : "r"(sm100::mapa_shared(part + c * 128 + row, r)));
          acc += v;
        }
        if (n < p.N) st_any(p.y, p.y_type, int64_t(m) * p.N + n, w8_value(acc, as_s[c], bs, bias, has_bias));
      }
    }
    sm100::cluster_sync();   // no CTA leaves while another reads its partial sums
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, cols);
  }
}

}  // namespace tac
