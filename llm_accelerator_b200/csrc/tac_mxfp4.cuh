// Products of 4-bit microscaled rows:
//   y[m, n] = sum_k A[m, k] B[n, k] (+ bias[n])
// A [M, K] and B [N, K] E2M1 codes, two a byte and K-major, each 32 values
// along K with one power of two (E8M0).  tcgen05 kind::mxf4 multiplies codes
// and scales and sums in float32; one rounding to the output's type.
//
// Orientation: the 128 rows of the MMA are channels (B) and its columns tokens
// (A), as in the INT8 products: few padded tokens in a ragged batch, a thread
// of the epilogue holds one channel, and a warp stores 32 consecutive channels
// of one token whatever the alignment of N.
//
// Scales lie in memory as TMEM wants them: for each 128 rows and 128 columns
// (four blocks) one piece of 512 bytes, 16 bytes for each of 32 lanes, in it
// the four blocks' bytes of rows lane, lane + 32, lane + 64, lane + 96.  Pieces
// of 128 rows follow each other along K, an even number of them, so that a
// stage of 256 columns is 1024 bytes that one bulk copy brings to shared
// memory and two tcgen05.cp to four columns each of TMEM.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "tac_launch.cuh"
#include "tac_sm100.cuh"

namespace tac {

enum MxFault : int { MX_TIMEOUT_EMPTY = 21, MX_TIMEOUT_FULL = 22, MX_TIMEOUT_ACC = 23, MX_TIMEOUT_DRAIN = 24 };

constexpr int kMxStageK = 256;       // columns of a stage: 128 bytes of codes, 1024 of scales for 128 rows
constexpr int kMxSfBytes = 1024;

// 512-byte pieces of scales along K for each 128 rows
__host__ __device__ constexpr int64_t mx_pieces(int64_t K) { return (K + kMxStageK - 1) / kMxStageK * 2; }

struct MxParams {
  const uint8_t* a_scale;    // tokens'
  const uint8_t* b_scale;    // channels'
  const void* bias;          // or null
  void* y;
  int bias_type;
  int M, N;
  int k_stages;              // stages of 256 columns
  int tn;                    // tokens of a tile
  int stages;                // of the ring
  int* fault;
  int after_rows;            // launched behind the row quantiser, which may still run: A and its scales wait for its end
};

// ---- PTX ------------------------------------------------------------------------------------------------------------
namespace sm100 {

// Instruction descriptor of kind::mxf4 with block scales: E2M1 operands (code 1), E8M0 scales (bit 23), both K-major.
// sf: which half of a scale word the MMA's 64 columns take (0 or 2).
__host__ __device__ constexpr uint32_t idesc_mxf4(uint32_t M, uint32_t N, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | ((N >> 3) << 17) | (1u << 23) | ((M >> 4) << 24) | (sf << 29);
}

// D(tmem) [+]= A x B with scales in TMEM, 64 columns; issued by one thread.
__device__ __forceinline__ void mma_mxf4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t sf_a,
                                         uint32_t sf_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(sf_a), "r"(sf_b));
}

// One 512-byte piece of scales from shared memory to four columns, for all four quarters of TMEM's lanes.
__device__ __forceinline__ void cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc));
}

// The same on CTA pairs: the MMA reads both CTAs' operands at its own offsets, and the copy takes each CTA's piece to its
// own TMEM.
__device__ __forceinline__ void mma_mxf4_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t sf_a,
                                              uint32_t sf_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(sf_a), "r"(sf_b));
}
__device__ __forceinline__ void cp_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n" ::"r"(taddr), "l"(desc));
}

// Shared-memory descriptor of such a piece: rows of 16 bytes one after the other, no swizzle.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t saddr) {
  return uint64_t((saddr >> 4) & 0x3FFF) | (uint64_t(1) << 16) | (uint64_t(128 >> 4) << 32) | (uint64_t(1) << 46);
}

}  // namespace sm100

// ---- epilogue -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float mx_ld(const void* p, int type, int64_t i) {
  if (type == 0) return __ldg(static_cast<const float*>(p) + i);
  const uint16_t b = __ldg(static_cast<const uint16_t*>(p) + i);
  return type == 1 ? __half2float(__ushort_as_half(b)) : __uint_as_float(uint32_t(b) << 16);
}

template <int YT>
__device__ __forceinline__ void mx_st(void* p, int64_t i, float v) {
  if constexpr (YT == 0) static_cast<float*>(p)[i] = v;
  else if constexpr (YT == 1) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

template <int YT>
__device__ __forceinline__ uint32_t mx_pair(float lo, float hi) {
  if constexpr (YT == 1) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// Results of 32 tokens (m ..) and a warp's 32 channels, of which this lane has
// one, where p.N has it.  What bounds these stores is the way out of the SM, in
// requests and in 32-byte sectors (1.4 cycles each): with an odd N a row's
// 16-bit channels go one by one, 64 bytes in one request, because pairs would
// leave the ends of every second row to requests of their own (836 x 49977 x
// 160: 37 us, 45 in pairs).
template <int YT>
__device__ __forceinline__ void mx_store_singles(const MxParams& p, const uint32_t (&v)[32], int m, int n, float bias) {
  const int left = n < p.N ? p.M - m : 0;
  if constexpr (YT == 0) {
    float* dst = static_cast<float*>(p.y) + int64_t(m) * p.N + n;
#pragma unroll
    for (int j = 0; j < 32; ++j, dst += p.N)
      asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\t@p st.global.f32 [%0], %1;\n\t}\n" ::"l"(dst),
                   "f"(__uint_as_float(v[j]) + bias), "r"(left), "r"(j)
                   : "memory");
  } else {
    uint16_t* dst = static_cast<uint16_t*>(p.y) + int64_t(m) * p.N + n;
    uint32_t two = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j, dst += p.N) {
      two = j & 1 ? two >> 16 : mx_pair<YT>(__uint_as_float(v[j]) + bias, __uint_as_float(v[j + 1 < 32 ? j + 1 : j]) + bias);
      asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\t@p st.global.b16 [%0], %1;\n\t}\n" ::"l"(dst),
                   "h"(uint16_t(two)), "r"(left), "r"(j)
                   : "memory");
    }
  }
}

// With an even N in pairs of channels, half the stores (836 x 49978 x 160: 33 us):
// of two tokens the even lanes store one's pairs and the odd lanes the other's,
// and lanes exchange what their neighbours store, of four tokens at a time.
// Exchanges go before the stores, behind which each would wait.
template <int YT>
__device__ __forceinline__ void mx_store_pairs(const MxParams& p, const uint32_t (&v)[32], int m, int n, float bias) {
  const int odd = threadIdx.x & 1;
  uint16_t* dst = static_cast<uint16_t*>(p.y) + int64_t(m + odd) * p.N + n - odd;
  const int64_t step = 2 * int64_t(p.N);
  const uint32_t give = odd ? 0x5410 : 0x7632, sel0 = odd ? 0x3254 : 0x5410, sel1 = odd ? 0x3276 : 0x7610;
  uint32_t mine[16], other[8];       // the first token's result low, the second's high; the neighbour's of two pairs of tokens
#pragma unroll
  for (int j = 0; j < 16; ++j) mine[j] = mx_pair<YT>(__uint_as_float(v[2 * j]) + bias, __uint_as_float(v[2 * j + 1]) + bias);
#pragma unroll
  for (int j = 0; j < 8; ++j) other[j] = __shfl_xor_sync(0xffffffffu, __byte_perm(mine[2 * j], mine[2 * j + 1], give), 1);
  const int left = p.M - m - odd;
#pragma unroll
  for (int j = 0; j < 16; ++j, dst += step)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\t@p st.global.b32 [%0], %1;\n\t}\n" ::"l"(dst),
                 "r"(__byte_perm(mine[j], other[j >> 1], j & 1 ? sel1 : sel0)), "r"(left), "r"(2 * j)
                 : "memory");
}

// 32 tokens (m .. m + 31) of a warp's 32 consecutive channels (n its own); v the sums.
template <int YT>
__device__ __forceinline__ void mx_store32(const MxParams& p, const uint32_t (&v)[32], int m, int n, float bias) {
  const bool all_channels = n - int(threadIdx.x & 31) + 32 <= p.N;
  if (YT != 0 && all_channels && ((p.N | int(reinterpret_cast<uintptr_t>(p.y) >> 1)) & 1) == 0) mx_store_pairs<YT>(p, v, m, n, bias);
  else mx_store_singles<YT>(p, v, m, n, bias);
}

// ---- split-K over a cluster -----------------------------------------------------------------------------------------
// A 128-channel x tn-token tile for each cluster of S CTAs; CTA r sums its
// share of the stages, leaves the float32 partial sums in its shared memory,
// and after a cluster barrier finishes every S-th token from all S partials,
// in the order of the ranks.  For products with too few tiles for 148 SMs,
// where streaming the weights is the work.
//   warp 0      loads, warp 1 MMAs, warps 2..5 epilogue.
// A stage's scales have columns of TMEM of their own, so a copy never meets
// an MMA that still reads the last ones.
constexpr int kMxSkThreads = 192;
constexpr int kMxWBytes = 128 * 128;
constexpr int kMxSkStages = 8;

// TMEM: the sums' columns (read in chunks of 32), then 16 of scales a stage.
__host__ __device__ constexpr int mx_sk_sf_col(int tn) { return tn < 32 ? 32 : tn; }
__host__ __device__ constexpr int mx_sk_cols(int tn, int stages) {
  const int need = mx_sk_sf_col(tn) + 16 * stages;
  return need <= 64 ? 64 : need <= 128 ? 128 : 256;
}
__host__ __device__ constexpr int mx_sk_stage_bytes(int tn) { return kMxWBytes + tn * 128 + 2 * kMxSfBytes; }

// Partial sums of a split tile in shared memory: [128 channels][tn + 4], the padding against bank conflicts.
__host__ __device__ constexpr int mx_sk_part_bytes(int tn) { return 128 * (tn + 4) * 4; }

// CTA `rank`'s share of the tokens from the partial sums of NS CTAs, in the order of the ranks.  Eight reads of four tokens
// are under way at once: one after the other, 16 waits for other CTAs' memory made a split of 128 tokens 4 us slower.
template <int YT, int NS>
__device__ __forceinline__ void mx_sum_parts(const MxParams& p, const float* mine, int n, int m0, int rank, float bias) {
  constexpr int kAtOnce = 8 / NS;
  const int per = max(4, p.tn / NS), first = rank * per, last = min(min(first + per, p.tn), p.M - m0);
  uint32_t base[NS];
#pragma unroll
  for (int r = 0; r < NS; ++r) base[r] = sm100::mapa_shared(mine + first, r);
  for (int c = first; c < last; c += 4 * kAtOnce) {
    float4 v[kAtOnce][NS];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
#pragma unroll
      for (int r = 0; r < NS; ++r) {
        v[q][r] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (c + 4 * q < last)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                       : "=f"(v[q][r].x), "=f"(v[q][r].y), "=f"(v[q][r].z), "=f"(v[q][r].w)
                       : "r"(base[r] + (c - first + 4 * q) * 4)
                       : "memory");
      }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) {
      float acc[4] = {};
#pragma unroll
      for (int r = 0; r < NS; ++r) acc[0] += v[q][r].x, acc[1] += v[q][r].y, acc[2] += v[q][r].z, acc[3] += v[q][r].w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = c + 4 * q + j;
        if (t < last && n < p.N) mx_st<YT>(p.y, int64_t(m0 + t) * p.N + n, acc[j] + bias);
      }
    }
  }
}

// The tile's results, or the CTA's partial sums to shared memory (over its stages: every copy and MMA has ended) and,
// after the cluster's barrier, CTA r's share of the tokens from all partials.  All threads of the CTA.
template <int YT>
__device__ __forceinline__ void mx_splitk_finish(const MxParams& p, uint8_t* smem, uint32_t tmem, int warp, int row, int n, int m0,
                                                 int rank, int nsplit, float bias, bool acc_ok) {
  const bool epi = warp >= 2 && warp < 6;
  const uint32_t t_addr = tmem + (uint32_t((warp & 3) * 32) << 16);
  if (nsplit == 1) {
    if (epi && acc_ok)
      for (int c = 0; c < p.tn; c += 32) {
        uint32_t v[32];
        __syncwarp();
        sm100::tmem_ld32(t_addr + c, v);
        mx_store32<YT>(p, v, m0 + c, n, bias);   // a tile of 16 tokens has no more than 16 rows before M
      }
    return;
  }
  float* const mine = reinterpret_cast<float*>(smem) + row * (p.tn + 4);
  if (epi) {
    for (int c = 0; c < p.tn; c += 32) {
      uint32_t v[32];
      __syncwarp();
      sm100::tmem_ld32(t_addr + c, v);
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        if (c + j < p.tn) *reinterpret_cast<uint4*>(mine + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    }
  }
  __syncwarp();
  sm100::cluster_sync();
  if (epi) {
    if (nsplit == 2) mx_sum_parts<YT, 2>(p, mine, n, m0, rank, bias);
    else if (nsplit == 4) mx_sum_parts<YT, 4>(p, mine, n, m0, rank, bias);
    else mx_sum_parts<YT, 8>(p, mine, n, m0, rank, bias);
  }
  __syncwarp();
  // No CTA leaves while another reads its partial sums.  Relaxed: what was read has been summed, and a release would wait for
  // the stores of the results.
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");
  sm100::cluster_wait();
}

// The four MMAs of a stage, and before them its scales' copies.  w_sf, a_sf: shared memory; sf: TMEM columns of the stage.
__device__ __forceinline__ void mx_stage_mma(uint32_t tmem, uint32_t sf, uint64_t dw, uint64_t da, uint64_t w_sf, uint64_t a_sf,
                                             uint32_t idesc0, uint32_t idesc2, bool first) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    sm100::cp_scales(sf + 4 * j, w_sf + j * (512 >> 4));
    sm100::cp_scales(sf + 8 + 4 * j, a_sf + j * (512 >> 4));
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    sm100::mma_mxf4(tmem, dw + 2 * k, da + 2 * k, k & 1 ? idesc2 : idesc0, sf + 4 * (k >> 1), sf + 8 + 4 * (k >> 1), !first || k);
}

template <int YT>
__global__ void __launch_bounds__(kMxSkThreads)
    mx_splitk_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, MxParams p) {
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[kMxSkStages], empty_bar[kMxSkStages], acc_bar;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128, m0 = blockIdx.y * p.tn;
  const int nsplit = gridDim.z, rank = blockIdx.z;
  const int kb0 = int(int64_t(p.k_stages) * rank / nsplit), kb1 = int(int64_t(p.k_stages) * (rank + 1) / nsplit);
  const int S = p.stages, stage_bytes = mx_sk_stage_bytes(p.tn);
  const int sf_off = kMxWBytes + p.tn * 128;     // of a stage: channels' scales, then tokens'
  const uint8_t* w_scale = p.b_scale + int64_t(n0 / 128) * p.k_stages * kMxSfBytes;
  const uint8_t* a_scale = p.a_scale + int64_t(m0 / 128) * p.k_stages * kMxSfBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full_bar[s], 1);
      sm100::mbar_init(&empty_bar[s], 1);
    }
    sm100::mbar_init(&acc_bar, 1);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  const int cols = mx_sk_cols(p.tn, S);
  if (warp == 1) sm100::tmem_alloc(&tmem_base, cols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;
  // Behind the row quantiser, which has seen the kernels before it complete, the weights are there already.
  if (!p.after_rows) after_previous();
  let_next();

  if (warp == 0) {
    uint32_t s = 0, ph = 1, issued = 0;
    auto weights = [&](int i, int kb) {
      uint8_t* st = smem + i * stage_bytes;
      sm100::mbar_arrive_expect_tx(&full_bar[i], stage_bytes);
      sm100::tma_load_2d(st, &tm_w, kb * 128, n0, &full_bar[i]);
      sm100::bulk_g2s(st + sf_off, w_scale + int64_t(kb) * kMxSfBytes, kMxSfBytes, &full_bar[i]);
    };
    // the first stages' weights need not wait for the rows
    const int early = min(S, kb1 - kb0);
    if (sm100::elect_one())
      for (int i = 0; i < early; ++i) weights(i, kb0 + i);
    __syncwarp();
    after_previous();
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&empty_bar[s], ph, abort_v, p.fault, MX_TIMEOUT_EMPTY)) break;
      if (sm100::elect_one()) {
        uint8_t* st = smem + s * stage_bytes;
        if (kb - kb0 >= early) weights(s, kb);
        sm100::tma_load_2d(st + kMxWBytes, &tm_a, kb * 128, m0, &full_bar[s]);
        sm100::bulk_g2s(st + sf_off + kMxSfBytes, a_scale + int64_t(kb) * kMxSfBytes, kMxSfBytes, &full_bar[s]);
      }
      __syncwarp();
      ++issued;
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // the copies still in flight land before the CTA goes on
    for (uint32_t j = issued > uint32_t(S) ? issued - S : 0; j < issued; ++j)
      sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, MX_TIMEOUT_DRAIN);
  } else if (warp == 1) {
    const uint32_t idesc0 = sm100::idesc_mxf4(128, p.tn, 0), idesc2 = sm100::idesc_mxf4(128, p.tn, 2);
    const uint64_t w0 = sm100::smem_desc_sw128(sm100::smem_u32(smem), 16, 1024);
    const uint64_t sf0 = sm100::smem_desc_scales(sm100::smem_u32(smem) + sf_off);
    uint32_t s = 0, ph = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&full_bar[s], ph, abort_v, p.fault, MX_TIMEOUT_FULL)) break;
      sm100::tc_fence_after();
      const uint64_t dw = w0 + s * (stage_bytes >> 4), sf = sf0 + s * (stage_bytes >> 4);
      if (sm100::elect_one()) {
        mx_stage_mma(tmem, tmem + mx_sk_sf_col(p.tn) + 16 * s, dw, dw + (kMxWBytes >> 4), sf, sf + (kMxSfBytes >> 4), idesc0, idesc2, kb == kb0);
        sm100::mma_commit(&empty_bar[s]);
      }
      __syncwarp();
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // arrives once every MMA has completed, also after a failed wait
    if (sm100::elect_one()) sm100::mma_commit(&acc_bar);
    __syncwarp();
    sm100::mbar_wait(&acc_bar, 0, p.fault, MX_TIMEOUT_DRAIN);
  }
  const int row = (warp & 3) * 32 + lane;     // TMEM lane = channel of the tile (warps 2..5)
  const int n = n0 + row;
  float bias = 0.f;
  bool acc_ok = false;
  if (warp >= 2) {
    if (n < p.N && p.bias) bias = mx_ld(p.bias, p.bias_type, n);
    acc_ok = sm100::mbar_wait_warp(&acc_bar, 0, abort_v, p.fault, MX_TIMEOUT_ACC);
    __syncwarp();
    sm100::tc_fence_after();
  }
  mx_splitk_finish<YT>(p, smem, tmem, warp, row, n, m0, rank, nsplit, bias, acc_ok);
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, cols);
  }
}

// ---- rows to codes --------------------------------------------------------------------------------------------------
// Eight values of a row held as they were loaded: 16-bit ones in one register quadruple, float32 ones in two.
template <typename T>
struct MxHeld {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* x, int left, bool vec) {     // `left` values of the row from x on
    if (vec && left >= 8) {
#pragma unroll
      for (int i = 0; i < int(sizeof(T) / 2); ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(x) + i);
    } else {
      T* t = reinterpret_cast<T*>(u);
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = j < left ? x[j] : T(0.f);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) u[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const T* t = reinterpret_cast<const T*>(u);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = float(t[j]);
  }
  // Exponent bits of the largest magnitude, as float32, of the block that four neighbouring lanes hold.  Magnitudes are
  // compared as whole numbers, in which infinities and NaN order above all others.
  __device__ __forceinline__ uint32_t block_exponent() const {
    uint32_t m;
    if constexpr (sizeof(T) == 2) {
      const uint32_t m2 = __vmaxu2(__vmaxu2(u[0].x & 0x7fff7fffu, u[0].y & 0x7fff7fffu), __vmaxu2(u[0].z & 0x7fff7fffu, u[0].w & 0x7fff7fffu));
      m = max(m2 & 0xffffu, m2 >> 16);
    } else {
      m = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        m = max(m, max(max(u[i].x & 0x7fffffffu, u[i].y & 0x7fffffffu), max(u[i].z & 0x7fffffffu, u[i].w & 0x7fffffffu)));
    }
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    if constexpr (std::is_same<T, __half>::value) return __float_as_uint(__half2float(__ushort_as_half(uint16_t(m)))) >> 23;
    return sizeof(T) == 2 ? m >> 7 : m >> 23;
  }
};

__device__ __forceinline__ uint32_t scale_byte(uint32_t exponent) { return exponent == 255 ? 255u : max(exponent, 2u) - 2; }
// Eight codes, value 0 in the lowest four bits.
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], uint32_t byte) {
  const float inv = __uint_as_float((254u - byte) << 23);        // of 255 a NaN
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
  return byte == 255 ? 0u : r;
}

// ---- the split-K product of few floating-point rows, quantised in the kernel -----------------------------------------
// One launch for a decode step.  A block's scale needs no more than the block,
// so each CTA quantises just the columns that it multiplies, straight into the
// swizzled operand; the first weights are on their way meanwhile.  All of its
// values are in flight at once, eight loads of eight a thread at most: read
// four by four, each wait for memory cost 1.4 us.  Rows past M keep what was
// there: a token's column of the result depends on no other.
//   warp 0      weights, warp 1 MMAs, warps 2..9 rows, warps 2..5 epilogue.
constexpr int kMxRowsThreads = 64 + 256, kMxRowsHeld = 8;

struct MxRowsParams {
  MxParams g;
  const void* x;
  int x_vec;                 // rows of whole, aligned 16-byte pieces
  int64_t ldx;
  int K;                     // columns of x
};

// Bytes of a stage's rows: codes of tn tokens and their scales.
__host__ __device__ constexpr int mx_rows_bytes(int tn) { return tn * 128 + kMxSfBytes; }

template <typename T, int YT>
__global__ void __launch_bounds__(kMxRowsThreads) mx_rows_kernel(const __grid_constant__ CUtensorMap tm_w, MxRowsParams pp) {
  MxParams p = pp.g;
  const int m0 = blockIdx.y * p.tn;
  p.M = min(p.M, m0 + p.tn);                     // of this tile: a TMEM load may bring columns behind its own
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[kMxSkStages], empty_bar[kMxSkStages], rows_bar, acc_bar;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128, nsplit = gridDim.z, rank = blockIdx.z;
  const int kb0 = int(int64_t(p.k_stages) * rank / nsplit), kb1 = int(int64_t(p.k_stages) * (rank + 1) / nsplit);
  constexpr int kStageBytes = kMxWBytes + kMxSfBytes;
  const int S = p.stages, row_bytes = mx_rows_bytes(p.tn);
  uint8_t* const rows_sm = smem + S * kStageBytes;      // [stage][tn rows of 128 bytes, swizzled; scales]
  const uint8_t* w_scale = p.b_scale + int64_t(n0 / 128) * p.k_stages * kMxSfBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full_bar[s], 1);
      sm100::mbar_init(&empty_bar[s], 1);
    }
    sm100::mbar_init(&rows_bar, 8);
    sm100::mbar_init(&acc_bar, 1);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  const int cols = mx_sk_cols(p.tn, S);
  if (warp == 1) sm100::tmem_alloc(&tmem_base, cols);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;
  after_previous();
  let_next();

  if (warp == 0) {
    uint32_t s = 0, ph = 1, issued = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&empty_bar[s], ph, abort_v, p.fault, MX_TIMEOUT_EMPTY)) break;
      if (sm100::elect_one()) {
        uint8_t* st = smem + s * kStageBytes;
        sm100::mbar_arrive_expect_tx(&full_bar[s], kStageBytes);
        sm100::tma_load_2d(st, &tm_w, kb * 128, n0, &full_bar[s]);
        sm100::bulk_g2s(st + kMxWBytes, w_scale + int64_t(kb) * kMxSfBytes, kMxSfBytes, &full_bar[s]);
      }
      __syncwarp();
      ++issued;
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // the copies still in flight land before the CTA goes on
    for (uint32_t j = issued > uint32_t(S) ? issued - S : 0; j < issued; ++j)
      sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, MX_TIMEOUT_DRAIN);
  } else if (warp == 1) {
    const uint32_t idesc0 = sm100::idesc_mxf4(128, p.tn, 0), idesc2 = sm100::idesc_mxf4(128, p.tn, 2);
    const uint64_t w0 = sm100::smem_desc_sw128(sm100::smem_u32(smem), 16, 1024);
    const uint64_t ws0 = sm100::smem_desc_scales(sm100::smem_u32(smem) + kMxWBytes);
    const uint64_t r0 = sm100::smem_desc_sw128(sm100::smem_u32(rows_sm), 16, 1024);
    const uint64_t rs0 = sm100::smem_desc_scales(sm100::smem_u32(rows_sm) + p.tn * 128);
    const bool rows = sm100::mbar_wait_warp(&rows_bar, 0, abort_v, p.fault, MX_TIMEOUT_FULL);
    uint32_t s = 0, ph = 0;
    for (int kb = kb0; rows && kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&full_bar[s], ph, abort_v, p.fault, MX_TIMEOUT_FULL)) break;
      sm100::tc_fence_after();
      const uint64_t ring = s * (kStageBytes >> 4), at = (kb - kb0) * (row_bytes >> 4);
      if (sm100::elect_one()) {
        mx_stage_mma(tmem, tmem + mx_sk_sf_col(p.tn) + 16 * s, w0 + ring, r0 + at, ws0 + ring, rs0 + at, idesc0, idesc2, kb == kb0);
        sm100::mma_commit(&empty_bar[s]);
      }
      __syncwarp();
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // arrives once every MMA has completed, also after a failed wait
    if (sm100::elect_one()) sm100::mma_commit(&acc_bar);
    __syncwarp();
    sm100::mbar_wait(&acc_bar, 0, p.fault, MX_TIMEOUT_DRAIN);
  } else {
    // items of eight values, 32 a row and stage: a warp's 32 are one row's of one stage, four lanes a block
    const int of_stage = (p.M - m0) * 32, items = (kb1 - kb0) * of_stage;
    const T* x = static_cast<const T*>(pp.x) + m0 * pp.ldx;
    const int t = threadIdx.x - 64;
    MxHeld<T> held[kMxRowsHeld];
    int stage[kMxRowsHeld], m[kMxRowsHeld];
#pragma unroll
    for (int j = 0; j < kMxRowsHeld; ++j) {
      const int i = t + j * 256;
      if (i - lane >= items) break;            // whole warps
      stage[j] = i / of_stage, m[j] = (i - stage[j] * of_stage) >> 5;
      const int k = (kb0 + stage[j]) * kMxStageK + lane * 8;
      held[j].load(x + m[j] * pp.ldx + k, pp.K - k, pp.x_vec);
    }
#pragma unroll
    for (int j = 0; j < kMxRowsHeld; ++j) {
      if (t + j * 256 - lane >= items) break;
      float v[8];
      held[j].values(v);
      const uint32_t byte = scale_byte(held[j].block_exponent());
      uint8_t* codes = rows_sm + stage[j] * row_bytes;
      *reinterpret_cast<uint32_t*>(codes + m[j] * 128 + ((((lane >> 2) ^ m[j]) & 7) << 4) + (lane & 3) * 4) = codes8(v, byte);
      if ((lane & 3) == 0)
        codes[p.tn * 128 + (lane >> 4) * 512 + (m[j] & 31) * 16 + (m[j] >> 5) * 4 + ((lane >> 2) & 3)] = uint8_t(byte);
    }
    sm100::fence_proxy_async();
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(&rows_bar);
  }
  const int row = (warp & 3) * 32 + lane;     // TMEM lane = channel of the tile (warps 2..5)
  const int n = n0 + row;
  float bias = 0.f;
  bool acc_ok = false;
  if (warp >= 2) {
    if (n < p.N && p.bias) bias = mx_ld(p.bias, p.bias_type, n);
    acc_ok = sm100::mbar_wait_warp(&acc_bar, 0, abort_v, p.fault, MX_TIMEOUT_ACC);
    __syncwarp();
    sm100::tc_fence_after();
  }
  mx_splitk_finish<YT>(p, smem, tmem, warp, row, n, m0, rank, nsplit, bias, acc_ok);
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, cols);
  }
}

// ---- CTA pairs ------------------------------------------------------------------------------------------------------
// 256 channels x tn tokens a pair of CTAs (cta_group::2): each CTA stages 128
// channels of the weights and half of the tokens, its channels' scales and all
// tokens', and gets its 128 channels of the result in its own TMEM.
// Persistent: warp 0 loads, warp 1 issues copies and MMAs, 16 warps are the
// epilogue, under the next tile's MMAs.
//   TMEM holds two accumulators and the scales of several stages.  Two of 256
// columns would fill it: they overlap by 64, which the epilogue reads first, so
// that the next tile's MMAs wait for a quarter of it only.  A stage's scales
// take the columns of an earlier stage once that one's MMAs have completed.
//   Bound by the operands' way into the SM, 91 bytes a nanosecond at most
// (measured with loads alone, on one SM as on all), and by the copies of scales
// between the MMAs: 16384 x 8192 x 8192 takes 405 us (5.4 PFLOP/s), 356 without
// these copies, 322 without the operands' loads, 284 without both; 4096^3 takes
// 31.5.  Copying a stage ahead of the MMAs made nothing faster, the last round's
// tiles in halves 4096^3 by 1.5 %.
//   Outputs wider than K is deep are bound by the epilogue (333 x 50257 x 768: 17
// us, 12 without stores); 16-byte stores out of shared memory, for runs of 256
// bytes, took 20 and for even rows 3.5 us longer than pairs.
//   88 registers, so that a CTA of the quantiser of aligned 16-bit rows (32 a
// thread) fits beside it in each quarter of the SM's (five warps' of the 18, two
// of its): this kernel is then in place when the rows are quantised.  (333 x
// 50257 x 768 from BF16 rows: 18.1 us, 20.7 with the 96 that the compiler would
// take.)  The quantisers of float32 rows (48) and of 16-bit rows that begin
// anywhere (58) do not fit.
struct MxPairCfg {
  static constexpr int kStages = 6;
  static constexpr int kStageBytes = 2 * 16384 + 3 * kMxSfBytes;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kEpi = 512;     // epilogue threads: four warps a quadrant of TMEM, a fourth of the tokens each
  static constexpr int kThreads = 64 + kEpi;
};
static_assert(sm100::tmem_alone(MxPairCfg::kSmem), "two clusters could wait for each other's TMEM");

struct MxPairParams {
  MxParams g;
  int w_tiles, t_tiles;      // 256-channel tiles, token tiles
};

template <int YT>
__global__ void __cluster_dims__(2, 1, 1) __maxnreg__(88)
    mx_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a,
                   const __grid_constant__ CUtensorMap tm_ws, const __grid_constant__ CUtensorMap tm_as, MxPairParams pp) {
  constexpr int S = MxPairCfg::kStages;
  const MxParams& p = pp.g;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], acc_full[2], acc_empty[2], drain_bar;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = sm100::cluster_ctarank();
  const int cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
  const int half = p.tn / 2, total = pp.w_tiles * pp.t_tiles;
  const bool overlap = p.tn == 256;
  const int acc1 = overlap ? 192 : p.tn;         // column of the second accumulator
  // Tokens' scales come in pieces of 128 rows: two for 192 or 256 tokens, which begin at a multiple of 64.
  const int pieces = p.tn > 128 ? 2 : 1, sf0 = acc1 + p.tn, sf_cols = 8 + 8 * pieces, sf_sets = min(S, (512 - sf0) / sf_cols);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full_bar[s], 1);
      sm100::mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      sm100::mbar_init(&acc_full[b], 1);
      sm100::mbar_init(&acc_empty[b], 2 * MxPairCfg::kEpi / 32);   // the epilogue warps of both CTAs
    }
    sm100::mbar_init(&drain_bar, 1);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  if (warp == 1) sm100::tmem_alloc_pair(&tmem_base, 512);
  sm100::tc_fence_before();
  sm100::cluster_sync();   // barriers and TMEM of both CTAs exist before any remote use
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;
  after_previous();
  let_next();

  if (warp == 0) {
    uint32_t s = 0, ph = 1, issued = 0;
    bool go = true;
    for (int tile = cid; go && tile < total; tile += ncl) {
      const int n0 = tile / pp.t_tiles * 256 + int(rank) * 128, mt = tile % pp.t_tiles * p.tn, m0 = mt + int(rank) * half;
      for (int kb = 0; kb < p.k_stages; ++kb) {
        go = sm100::mbar_wait_warp(&empty_bar[s], ph, abort_v, p.fault, MX_TIMEOUT_EMPTY);
        if (!go) break;
        if (sm100::elect_one()) {
          if (rank == 0) sm100::mbar_arrive_expect_tx(&full_bar[s], 2 * (16384 + half * 128 + (1 + pieces) * kMxSfBytes));
          const uint32_t bar0 = sm100::mapa_shared(&full_bar[s], 0);
          uint8_t* st = smem + s * MxPairCfg::kStageBytes;
          sm100::tma_load_2d_pair(st, &tm_w, kb * 128, n0, bar0);
          sm100::tma_load_2d_pair(st + 16384, &tm_a, kb * 128, m0, bar0);
          sm100::tma_load_2d_pair(st + 32768, &tm_ws, kb * (kMxSfBytes / 4), n0 / 128, bar0);
          sm100::tma_load_2d_pair(st + 32768 + kMxSfBytes, &tm_as, kb * (kMxSfBytes / 4), mt / 128, bar0);
        }
        __syncwarp();
        ++issued;
        if (++s == S) s = 0, ph ^= 1;
      }
    }
    if (rank == 0) {
      // both CTAs' copies of the stages still in flight land on these barriers
      for (uint32_t j = issued > uint32_t(S) ? issued - S : 0; j < issued; ++j)
        sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, MX_TIMEOUT_DRAIN);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc0 = sm100::idesc_mxf4(256, p.tn, 0), idesc2 = sm100::idesc_mxf4(256, p.tn, 2);
      const uint64_t w0 = sm100::smem_desc_sw128(sm100::smem_u32(smem), 16, 1024);
      const uint64_t ws0 = sm100::smem_desc_scales(sm100::smem_u32(smem) + 32768);
      uint32_t s = 0, ph = 0, local = 0, set = 0, used = 0;     // used: stages issued so far
      uint32_t old = 0, old_ph = 0;                             // the stage whose scales had this stage's columns
      for (int tile = cid; tile < total; tile += ncl, ++local) {
        const uint32_t b = local & 1;
        // the accumulator's last tile has been read, or where they overlap the first part of the other one's
        const uint32_t wb = overlap ? b ^ 1 : b, wph = overlap ? ((local - 1) >> 1) & 1 : ((local >> 1) & 1) ^ 1;
        if (!(overlap && local == 0) && !sm100::mbar_wait_warp(&acc_empty[wb], wph, abort_v, p.fault, MX_TIMEOUT_ACC)) break;
        sm100::tc_fence_after();
        const uint32_t acc = tmem + b * acc1;
        const int mt = tile % pp.t_tiles * p.tn, off = (mt & 127) / 32;
        bool ok = true;
        for (int kb = 0; kb < p.k_stages; ++kb) {
          if (sf_sets < S && used >= uint32_t(sf_sets)) {
            ok = sm100::mbar_wait_warp(&empty_bar[old], old_ph, abort_v, p.fault, MX_TIMEOUT_ACC);
            if (!ok) break;
            if (++old == S) old = 0, old_ph ^= 1;
          }
          ok = sm100::mbar_wait_warp(&full_bar[s], ph, abort_v, p.fault, MX_TIMEOUT_FULL);
          if (!ok) break;
          sm100::tc_fence_after();
          const uint64_t dw = w0 + s * (MxPairCfg::kStageBytes >> 4), ds = ws0 + s * (MxPairCfg::kStageBytes >> 4);
          const uint32_t sf = tmem + sf0 + set * sf_cols;
          if (sm100::elect_one()) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              sm100::cp_scales_pair(sf + 4 * j, ds + j * (512 >> 4));
              for (int r = 0; r < pieces; ++r)
                sm100::cp_scales_pair(sf + 8 + 4 * (j * pieces + r), ds + ((1 + r) * kMxSfBytes + j * 512) / 16);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
              sm100::mma_mxf4_pair(acc, dw + 2 * k, dw + (16384 >> 4) + 2 * k, k & 1 ? idesc2 : idesc0, sf + 4 * (k >> 1),
                                   sf + 8 + 4 * (k >> 1) * pieces + off, (kb | k) != 0);
            sm100::mma_commit_pair(&empty_bar[s], 0x3);
          }
          __syncwarp();
          ++used;
          if (++set == uint32_t(sf_sets)) set = 0;
          if (++s == S) s = 0, ph ^= 1;
        }
        if (!ok) break;
        if (sm100::elect_one()) sm100::mma_commit_pair(&acc_full[b], 0x3);
        __syncwarp();
      }
      // every MMA issued must finish before either CTA releases TMEM
      if (sm100::elect_one()) sm100::mma_commit_pair(&drain_bar, 0x3);
      __syncwarp();
    }
    sm100::mbar_wait(&drain_bar, 0, p.fault, MX_TIMEOUT_DRAIN);
  } else {
    const int row = (warp & 3) * 32 + lane;
    const uint32_t acc_empty0_0 = sm100::mapa_shared(&acc_empty[0], 0), acc_empty0_1 = sm100::mapa_shared(&acc_empty[1], 0);
    const int part = (warp - 2) >> 2;
    uint32_t local = 0;
    // a tile's first token and this thread's channel; from one tile to the next without a division, which every warp
    // would do between its stores and its next wait
    const int step_w = ncl / pp.t_tiles, step_t = ncl % pp.t_tiles;
    int t_next = cid % pp.t_tiles, n_next = cid / pp.t_tiles * 256 + int(rank) * 128 + row;
    // the bias of a tile is loaded while the tile before it is finished
    float bias = p.bias && n_next < p.N ? mx_ld(p.bias, p.bias_type, n_next) : 0.f;
    for (int tile = cid; tile < total; tile += ncl, ++local) {
      const uint32_t b = local & 1, aph = (local >> 1) & 1;
      const int n = n_next, m0 = t_next * p.tn, tokens = min(p.tn, p.M - m0);
      const float bias_now = bias;
      t_next += step_t;
      n_next += step_w * 256;
      if (t_next >= pp.t_tiles) t_next -= pp.t_tiles, n_next += 256;
      if (p.bias && tile + ncl < total && n_next < p.N) bias = mx_ld(p.bias, p.bias_type, n_next);
      if (!sm100::mbar_wait_warp(&acc_full[b], aph, abort_v, p.fault, MX_TIMEOUT_ACC)) break;
      sm100::tc_fence_after();
      // Relaxed: as a release the arrival would wait for the warp's stores of this tile and the last.
      auto release = [&] {
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0)
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(b ? acc_empty0_1 : acc_empty0_0) : "memory");
      };
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        // Overlapping accumulators: the columns that the next tile's take are the upper half's of the first one and the
        // lower half's of the second one, and go first.
        const int k = overlap ? i ^ int(b) ^ 1 : i, c = part * 32 + k * 128;
        const bool live = c < tokens;
        uint32_t v[32];
        __syncwarp();
        if (live) sm100::tmem_ld32(tmem + (uint32_t((warp & 3) * 32) << 16) + b * acc1 + c, v);
        if (i == (overlap ? 0 : 1)) release();
        if (live) mx_store32<YT>(p, v, m0 + c, n, bias_now);
      }
    }
  }

  sm100::tc_fence_before();
  __syncwarp();
  sm100::cluster_sync();   // no CTA leaves while its peer may still touch its shared memory or TMEM
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc_pair(tmem, 512);
  }
}

}  // namespace tac
