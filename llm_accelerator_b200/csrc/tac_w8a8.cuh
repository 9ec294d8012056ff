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

// the same in two steps: the element's bits (the load is still under way), and their value
__device__ __forceinline__ uint32_t ld_bits(const void* p, int type, int64_t i) {
  return type == 0 ? __ldg(static_cast<const uint32_t*>(p) + i) : uint32_t(__ldg(static_cast<const uint16_t*>(p) + i));
}
__device__ __forceinline__ float bits_value(uint32_t b, int type) {
  return type == 0 ? __uint_as_float(b) : type == 1 ? __half2float(__ushort_as_half(uint16_t(b))) : __uint_as_float(b << 16);
}

template <int YT>
__device__ __forceinline__ void st_y(void* p, int64_t i, float v) {
  if constexpr (YT == 0) static_cast<float*>(p)[i] = v;
  else if constexpr (YT == 1) static_cast<__half*>(p)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

struct W8Params {
  const float* a_scale;
  const void* b_scale;
  const void* bias;          // or null
  void* y;
  int b_type, bias_type;
  int M, N, K;
  int k_blocks;              // 128-byte blocks of K
  int tn;                    // tokens of a tile
  int stages;
  int* fault;
  int after_rows;            // launched while the row quantiser may still run: A and a_scale wait for its end
};

__device__ __forceinline__ void wait_rows() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

__device__ __forceinline__ float w8_value(int acc, float as, float bs, float bias) {
  return fmaf(__fmul_rn(__int2float_rn(acc), as), bs, bias);   // bias 0 where there is none
}

// The 16-bit case of w8_store32.
template <int YT, bool ODD>
__device__ __forceinline__ void w8_store_pairs(const W8Params& p, const uint32_t (&v)[32], const float* as, int m, int n,
                                               float bs, float bias, uint32_t base_odd) {
  const int lane = threadIdx.x & 31;
  // the token of a pair whose row is word-aligned at an even channel: the first one, or with an odd N that of that parity
  const uint32_t first = ODD ? (base_odd ^ uint32_t(m & 1)) : 0u;   // the warp's first channel is even
  const bool mine_first = (lane & 1) == 0;                          // even lanes store the aligned token
  const int tok = mine_first ? int(first) : int(first ^ 1u);
  uint16_t* dst = static_cast<uint16_t*>(p.y) + int64_t(m + tok) * p.N + n - (mine_first || ODD ? 0 : 1);
  uint16_t* edge = static_cast<uint16_t*>(p.y) + int64_t(m + int(first ^ 1u)) * p.N + n;
  const int64_t step = 2 * int64_t(p.N);
  const bool has_next = !ODD || lane != 31, is_edge = lane == 0 || lane == 31;
  const uint32_t edge_shift = first ? 0 : 16;
  const uint32_t sel = ODD ? (tok ? 0x7632 : 0x5410) : (mine_first ? 0x5410 : 0x3276);
  // all exchanges first: between the stores each would wait behind them
  uint32_t mine[16], other[16];      // the first token's result low, the second's high
#pragma unroll
  for (int j = 0; j < 16; j += 2) {
    const float4 a = *reinterpret_cast<const float4*>(as + 2 * j);
    const float aa[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float y0 = w8_value(int(v[2 * (j + i)]), aa[2 * i], bs, bias), y1 = w8_value(int(v[2 * (j + i) + 1]), aa[2 * i + 1], bs, bias);
      if constexpr (YT == 1) {
        const __half2 h = __floats2half2_rn(y0, y1);
        mine[j + i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(y0, y1);
        mine[j + i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      other[j + i] = ODD ? __shfl_down_sync(0xffffffffu, mine[j + i], 1) : __shfl_xor_sync(0xffffffffu, mine[j + i], 1);
    }
  }
  // predicated: a branch for each costs more than the store.  Of the pairs' rows, those below M are stored.
  const int left = p.M - m - tok, left_edge = is_edge ? p.M - m - int(first ^ 1u) : 0, left_here = has_next ? left : 0;
#pragma unroll
  for (int j = 0; j < 16; ++j, dst += step, edge += step) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\t@p st.global.b32 [%0], %1;\n\t}\n" ::"l"(dst),
                 "r"(__byte_perm(mine[j], other[j], sel)), "r"(left_here), "r"(2 * j)
                 : "memory");
    if constexpr (ODD)
      asm volatile("{\n\t.reg .pred p;\n\tsetp.gt.s32 p, %2, %3;\n\t@p st.global.b16 [%0], %1;\n\t}\n" ::"l"(edge),
                   "h"(uint16_t(mine[j] >> edge_shift)), "r"(left_edge), "r"(2 * j)
                   : "memory");
  }
}

// 32 tokens (m .. m + 31) of a warp's 32 consecutive channels (n its own):
// v the sums, as their scales (shared memory, 16-byte aligned).  A thread has
// one channel, so 16-bit results are exchanged with the next lane and stored
// in pairs: of two tokens, the even lanes store one's pairs and the odd lanes
// the other's.  Where N is odd every second row begins between two words; its
// pairs are those of an odd lane and the next, its first and last channel go
// alone (3 us of 24 at 333 x 50257 x 768; collecting them for one store of all
// rows took as long).  Exchanges go before the stores, behind which each would
// wait (29 us).  (Four warps with an element's own 16-bit store and 30
// instructions each took 91 us at 4096^3, the MMAs 34.)
template <int YT>
__device__ __forceinline__ void w8_store32(const W8Params& p, const uint32_t (&v)[32], const float* as, int m, int n,
                                           float bs, float bias) {
  const int lane = threadIdx.x & 31, n_warp = n - lane;
  const bool all_channels = n_warp + 32 <= p.N, inside = all_channels && m + 32 <= p.M;
  const uint32_t base_odd = uint32_t(reinterpret_cast<uintptr_t>(p.y) >> 1) & 1;
  if (YT == 0 && inside) {
    float* dst = static_cast<float*>(p.y) + int64_t(m) * p.N + n;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 a = *reinterpret_cast<const float4*>(as + j);
      const float aa[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i, dst += p.N) *dst = w8_value(int(v[j + i]), aa[i], bs, bias);
    }
  } else if (YT != 0 && all_channels && ((p.N & 1) || !base_odd)) {
    if (p.N & 1) w8_store_pairs<YT, true>(p, v, as, m, n, bs, bias, base_odd);
    else w8_store_pairs<YT, false>(p, v, as, m, n, bs, bias, 0u);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (m + j < p.M && n < p.N) st_y<YT>(p.y, int64_t(m + j) * p.N + n, w8_value(int(v[j]), as[j], bs, bias));
  }
}

// ---- split-K over a cluster -----------------------------------------------------------------------------------------
// A 128-channel x tn-token tile for each cluster of S CTAs; CTA r sums its
// share of the K blocks, leaves the int32 partial sums in its shared memory,
// and after a cluster barrier finishes every S-th token from all S partials
// (integer sums: the split never changes a result).  For products with too
// few tiles for 148 SMs, where streaming the weights is the work.
//   warp 0      TMA loads of both operands, warp 1 MMAs, warps 2..5 epilogue.
// Bound by latency at these sizes: 64 x 4096 x 1024 takes 5.6 us, 0.7 of them
// for its bytes; launch, TMA, MMA and store each wait for the one before.
constexpr int kSkThreads = 192;
constexpr int kSkWBytes = 128 * 128;

__host__ __device__ constexpr int sk_stage_bytes(int tn) { return kSkWBytes + tn * 128; }

// Partial sums of a split tile in shared memory: [128 channels][tn + 4], so that a channel's tokens are read 16 bytes at
// a time from the other CTAs and the padding spreads the channels over the banks.
__host__ __device__ constexpr int sk_part_bytes(int tn) { return 128 * (tn + 4) * 4; }

// The end of both split-K kernels: the tile's results, or the CTA's partial sums to shared memory (over its stages:
// every copy and MMA has ended) and, after the cluster's barrier, CTA r's share of the tokens from all partials.
// (Reading the others' partials a word at a time took 12 us where one CTA alone took 7; pushing them a word at a time
// was no better.)  All threads of the CTA.
template <int YT>
__device__ __forceinline__ void w8_splitk_finish(const W8Params& p, uint8_t* smem, uint32_t tmem, const float* as_s, int warp,
                                                 int row, int n, int m0, int rank, int nsplit, float bs, float bias,
                                                 bool acc_ok) {
  const uint32_t t_addr = tmem + (uint32_t((warp & 3) * 32) << 16);
  if (nsplit == 1) {
    if (warp >= 2 && acc_ok) {
      for (int c = 0; c < p.tn; c += 32) {
        uint32_t v[32];
        __syncwarp();
        sm100::tmem_ld32(t_addr + c, v);
        // a tile of 16 tokens has no more than 16 rows before M
        w8_store32<YT>(p, v, as_s + c, m0 + c, n, bs, bias);
      }
    }
    return;
  }
  int* const mine = reinterpret_cast<int*>(smem) + row * (p.tn + 4);
  if (warp >= 2) {
    for (int c = 0; c < p.tn; c += 32) {
      uint32_t v[32];
      __syncwarp();
      sm100::tmem_ld32(t_addr + c, v);
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        if (c + j < p.tn) *reinterpret_cast<int4*>(mine + c + j) = make_int4(int(v[j]), int(v[j + 1]), int(v[j + 2]), int(v[j + 3]));
    }
  }
  __syncwarp();
  sm100::cluster_sync();
  const int per = max(4, p.tn / nsplit), first = rank * per;    // tokens of this CTA
  if (warp >= 2 && first < p.tn) {
    uint32_t base[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) base[r] = sm100::mapa_shared(mine + first, r < nsplit ? r : 0);
    for (int k = 0; k < per; k += 4) {
      if (m0 + first + k >= p.M) break;
      int4 v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        v[r] = make_int4(0, 0, 0, 0);
        if (r < nsplit)
          asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];\n"
                       : "=r"(v[r].x), "=r"(v[r].y), "=r"(v[r].z), "=r"(v[r].w)
                       : "r"(base[r] + k * 4)
                       : "memory");
      }
      int acc[4] = {};
#pragma unroll
      for (int r = 0; r < 8; ++r) acc[0] += v[r].x, acc[1] += v[r].y, acc[2] += v[r].z, acc[3] += v[r].w;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = first + k + j, m = m0 + tok;
        if (m < p.M && n < p.N) st_y<YT>(p.y, int64_t(m) * p.N + n, w8_value(acc[j], as_s[tok], bs, bias));
      }
    }
  }
  __syncwarp();
  sm100::cluster_sync();                         // no CTA leaves while another reads its partial sums
}

template <int YT>
__global__ void __launch_bounds__(kSkThreads)
    w8_splitk_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, W8Params p) {
  constexpr int kMaxStages = 8;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], acc_bar;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ __align__(16) float as_s[256];

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
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
    uint32_t s = 0, ph = 1, issued = 0;
    // the first stages' weights need not wait for the rows
    const int early = min(S, kb1 - kb0);
    if (sm100::elect_one())
      for (int i = 0; i < early; ++i) {
        sm100::mbar_arrive_expect_tx(&full_bar[i], stage_bytes);
        sm100::tma_load_2d(smem + i * stage_bytes, &tm_w, (kb0 + i) * 128, n0, &full_bar[i]);
      }
    __syncwarp();
    wait_rows();
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&empty_bar[s], ph, abort_v, p.fault, W8_TIMEOUT_EMPTY)) break;
      if (sm100::elect_one()) {
        uint8_t* st = smem + s * stage_bytes;
        if (kb - kb0 >= early) {
          sm100::mbar_arrive_expect_tx(&full_bar[s], stage_bytes);
          sm100::tma_load_2d(st, &tm_w, kb * 128, n0, &full_bar[s]);
        }
        sm100::tma_load_2d(st + kSkWBytes, &tm_a, kb * 128, m0, &full_bar[s]);
      }
      __syncwarp();
      ++issued;
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // the copies still in flight land before the CTA goes on
    for (uint32_t j = issued > uint32_t(S) ? issued - S : 0; j < issued; ++j)
      sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, W8_TIMEOUT_DRAIN);
  } else if (warp == 1) {
    const uint32_t idesc = sm100::idesc_i8(128, p.tn, 0);
    const uint64_t w0 = sm100::smem_desc_sw128(sm100::smem_u32(smem), 16, 1024);
    uint32_t s = 0, ph = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&full_bar[s], ph, abort_v, p.fault, W8_TIMEOUT_FULL)) break;
      sm100::tc_fence_after();
      const uint64_t dw = w0 + s * (stage_bytes >> 4);
      if (sm100::elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          sm100::mma_i8(tmem, dw + 2 * k, dw + (kSkWBytes >> 4) + 2 * k, idesc, (kb > kb0) || k);
        sm100::mma_commit(&empty_bar[s]);
      }
      __syncwarp();
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // arrives once every MMA has completed, also after a failed wait
    if (sm100::elect_one()) sm100::mma_commit(&acc_bar);
    __syncwarp();
    sm100::mbar_wait(&acc_bar, 0, p.fault, W8_TIMEOUT_DRAIN);
  }
  const int row = (warp & 3) * 32 + lane;     // TMEM lane = channel of the tile (warps 2..5)
  const int n = n0 + row;
  float bs = 0.f, bias = 0.f;
  bool acc_ok = false;
  if (warp >= 2) {
    if (n < p.N) {
      bs = ld_any(p.b_scale, p.b_type, n);
      if (p.bias) bias = ld_any(p.bias, p.bias_type, n);
    }
    wait_rows();
    for (int i = threadIdx.x - 64; i < p.tn; i += 128) as_s[i] = m0 + i < p.M ? __ldg(p.a_scale + m0 + i) : 0.f;
    asm volatile("bar.sync 1, 128;\n" ::: "memory");   // as_s, among the epilogue's warps
    acc_ok = sm100::mbar_wait_warp(&acc_bar, 0, abort_v, p.fault, W8_TIMEOUT_ACC);
    __syncwarp();
    sm100::tc_fence_after();
  }
  w8_splitk_finish<YT>(p, smem, tmem, as_s, warp, row, n, m0, rank, nsplit, bs, bias, acc_ok);
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, cols);
  }
}

// ---- the same for few floating-point rows, quantised in the kernel ----------------------------------------------------
// One launch for a decode step: while the first stages of weights are on their
// way, the epilogue's warps take the largest magnitude of each row over this
// CTA's K blocks, the cluster's CTAs tell each other theirs, and the rows'
// codes go straight into the swizzled operand, which stays in shared memory.
// For a call that the host waits for, a launch of its own for the quantiser
// costs more than reading the rows once for each 128 channels, as long as they
// are few thousand values (one_launch has both sides; 1 x 4096 x 1024: 7.0 us
// on the device with weights out of HBM, 6.6 with weights in L2).
constexpr int kRowsMost = 16, kRowsMostK = 8192;

struct W8RowsParams {
  W8Params g;
  const void* x;
  int x_type, x_vec;         // x_vec: 16-bit rows of whole 16-byte chunks
  int64_t ldx;
  int k_real;                // columns of x
};

__device__ __forceinline__ void load8(const W8RowsParams& p, int m, int k, float (&v)[8]) {
  const int64_t i = m * p.ldx + k;
  if (p.x_vec && k + 8 <= p.k_real) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + i));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t h = (w[j / 2] >> (16 * (j & 1))) & 0xffffu;
      v[j] = p.x_type == 1 ? __half2float(__ushort_as_half(uint16_t(h))) : __uint_as_float(h << 16);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < p.k_real ? ld_any(p.x, p.x_type, i + j) : 0.f;
  }
}

template <int YT>
__global__ void __launch_bounds__(kSkThreads) w8_rows_kernel(const __grid_constant__ CUtensorMap tm_w, W8RowsParams pp) {
  constexpr int kMaxStages = 8, kTn = kRowsMost;
  const W8Params& p = pp.g;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], acc_bar, rows_bar;
  __shared__ uint32_t tmem_base, row_max[kTn], all_max[8][kTn];
  __shared__ int abort_flag;
  __shared__ __align__(16) float as_s[32];       // a chunk of the epilogue is 32 tokens wide
  __shared__ float inv_s[kTn];

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * 128, nsplit = gridDim.z, rank = blockIdx.z;
  const int kb0 = int(int64_t(p.k_blocks) * rank / nsplit), kb1 = int(int64_t(p.k_blocks) * (rank + 1) / nsplit);
  const int S = p.stages;
  uint8_t* const rows_sm = smem + S * kSkWBytes;  // [K block][16 rows][128 bytes], swizzled

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full_bar[s], 1);
      sm100::mbar_init(&empty_bar[s], 1);
    }
    sm100::mbar_init(&acc_bar, 1);
    sm100::mbar_init(&rows_bar, 4);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  if (threadIdx.x < kTn) row_max[threadIdx.x] = 0;
  if (threadIdx.x < 32) as_s[threadIdx.x] = 0.f;
  if (warp == 1) sm100::tmem_alloc(&tmem_base, 32);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;
  // The maxima go into the other CTAs' shared memory, which may be written once every CTA of the cluster runs: it says so
  // here, and the wait below lies behind the rows' loads.
  if (nsplit > 1) sm100::cluster_arrive();

  const int early = min(S, kb1 - kb0);
  const int t = threadIdx.x - 64, per = (kb1 - kb0) * 16, items = p.M * per;   // 8-value chunks of this CTA's columns
  constexpr int kHeld = 4;                       // chunks that a thread keeps from the maximum to the codes; it reads the rest again
  float held[kHeld][8];
  auto item = [&](int i, float (&v)[8]) {
    const int m = i / per;
    load8(pp, m, kb0 * 128 + (i - m * per) * 8, v);
    return m;
  };
  auto largest = [&](int i, int m, const float (&v)[8]) {
    uint32_t mb = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) mb = max(mb, __float_as_uint(v[j]) & 0x7fffffffu);
    // 16 lanes of one row first: a row has a multiple of 16 chunks, so of a warp's 32 all or the lower half are items
    const uint32_t lanes = (i | 31) < items ? 0xffffffffu : 0x0000ffffu;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) mb = max(mb, __shfl_xor_sync(lanes, mb, o));
    if ((lane & 15) == 0) atomicMax(&row_max[m], mb);
  };
  if (warp == 0) {
    if (sm100::elect_one())
      for (int i = 0; i < early; ++i) {
        sm100::mbar_arrive_expect_tx(&full_bar[i], kSkWBytes);
        sm100::tma_load_2d(smem + i * kSkWBytes, &tm_w, (kb0 + i) * 128, n0, &full_bar[i]);
      }
    __syncwarp();
  } else if (warp >= 2) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (t + k * 128 < items) item(t + k * 128, held[k]);
    for (int i = t; i < per * 8; i += 128) reinterpret_cast<uint4*>(rows_sm)[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (t + k * 128 < items) largest(t + k * 128, (t + k * 128) / per, held[k]);
    for (int i = t + kHeld * 128; i < items; i += 128) {
      float v[8];
      const int m = item(i, v);
      largest(i, m, v);
    }
    asm volatile("bar.sync 1, 128;\n" ::: "memory");
    __syncwarp();
    if (nsplit > 1) sm100::cluster_wait();
    // this CTA's maxima to every CTA of the cluster
    for (int i = t; i < kTn * nsplit; i += 128)
      asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(sm100::mapa_shared(&all_max[rank][i % kTn], i / kTn)), "r"(row_max[i % kTn])
                   : "memory");
  }
  __syncwarp();
  if (nsplit > 1) {
    if (warp < 2) sm100::cluster_wait();         // of the first arrival, which the other warps have waited for
    sm100::cluster_sync();
  } else {
    __syncthreads();
  }

  if (warp == 0) {
    uint32_t s = 0, ph = 1, issued = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&empty_bar[s], ph, abort_v, p.fault, W8_TIMEOUT_EMPTY)) break;
      if (kb - kb0 >= early && sm100::elect_one()) {
        sm100::mbar_arrive_expect_tx(&full_bar[s], kSkWBytes);
        sm100::tma_load_2d(smem + s * kSkWBytes, &tm_w, kb * 128, n0, &full_bar[s]);
      }
      __syncwarp();
      ++issued;
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // the copies still in flight land before the CTA goes on
    for (uint32_t j = issued > uint32_t(S) ? issued - S : 0; j < issued; ++j)
      sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, W8_TIMEOUT_DRAIN);
  } else if (warp == 1) {
    const uint32_t idesc = sm100::idesc_i8(128, kTn, 0);
    const uint64_t w0 = sm100::smem_desc_sw128(sm100::smem_u32(smem), 16, 1024);
    const uint64_t r0 = sm100::smem_desc_sw128(sm100::smem_u32(rows_sm), 16, 1024);
    const bool rows = sm100::mbar_wait_warp(&rows_bar, 0, abort_v, p.fault, W8_TIMEOUT_FULL);
    uint32_t s = 0, ph = 0;
    for (int kb = kb0; rows && kb < kb1; ++kb) {
      if (!sm100::mbar_wait_warp(&full_bar[s], ph, abort_v, p.fault, W8_TIMEOUT_FULL)) break;
      sm100::tc_fence_after();
      const uint64_t dw = w0 + s * (kSkWBytes >> 4), dr = r0 + (kb - kb0) * (kTn * 128 >> 4);
      if (sm100::elect_one()) {
#pragma unroll
        for (int k = 0; k < 4; ++k) sm100::mma_i8(tmem, dw + 2 * k, dr + 2 * k, idesc, (kb > kb0) || k);
        sm100::mma_commit(&empty_bar[s]);
      }
      __syncwarp();
      if (++s == uint32_t(S)) s = 0, ph ^= 1;
    }
    // arrives once every MMA has completed, also after a failed wait
    if (sm100::elect_one()) sm100::mma_commit(&acc_bar);
    __syncwarp();
    sm100::mbar_wait(&acc_bar, 0, p.fault, W8_TIMEOUT_DRAIN);
  }
  const int row = (warp & 3) * 32 + lane;
  const int n = n0 + row;
  float bs = 0.f, bias = 0.f;
  bool acc_ok = false;
  if (warp >= 2) {
    if (t < p.M) {
      uint32_t mb = 0;
      for (int r = 0; r < nsplit; ++r) mb = max(mb, all_max[r][t]);
      const bool finite = mb < 0x7f800000u;
      const float top = fmaxf(__uint_as_float(mb), 1e-8f);
      inv_s[t] = finite ? __fdiv_rn(127.0f, top) : __uint_as_float(0x7fc00000u);
      as_s[t] = finite ? __fdiv_rn(top, 127.0f) : __uint_as_float(0x7fc00000u);
    }
    asm volatile("bar.sync 1, 128;\n" ::: "memory");   // inv_s, as_s, and the zeros of rows_sm
    auto codes = [&](int i, const float (&v)[8]) {
      const int m = i / per, c = i - m * per;    // c: 8-value chunk of the row
      const float inv = inv_s[m];
      if (!(inv == inv)) return;                 // a row without a scale: its codes stay 0
      uint32_t b[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(__fadd_rn(__fmul_rn(v[j], inv), 12582912.f));   // rounds; low byte = code
      // block c / 16, 16-byte chunk (c / 2) % 8, its half c % 2
      *reinterpret_cast<uint2*>(rows_sm + (c >> 4) * (kTn * 128) + (m >> 3) * 1024 + (m & 7) * 128 + ((((c >> 1) & 7) ^ (m & 7)) << 4) +
                                (c & 1) * 8) =
          make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                     __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
      if (t + k * 128 < items) codes(t + k * 128, held[k]);
    for (int i = t + kHeld * 128; i < items; i += 128) {
      float v[8];
      item(i, v);
      codes(i, v);
    }
    sm100::fence_proxy_async();
    __syncwarp();
    if (lane == 0) sm100::mbar_arrive(&rows_bar);
    if (n < p.N) {
      bs = ld_any(p.b_scale, p.b_type, n);
      if (p.bias) bias = ld_any(p.bias, p.bias_type, n);
    }
    acc_ok = sm100::mbar_wait_warp(&acc_bar, 0, abort_v, p.fault, W8_TIMEOUT_ACC);
    __syncwarp();
    sm100::tc_fence_after();
  }
  w8_splitk_finish<YT>(p, smem, tmem, as_s, warp, row, n, 0, rank, nsplit, bs, bias, acc_ok);
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 32);
  }
}

// ---- CTA pairs ------------------------------------------------------------------------------------------------------
// 256 channels x tn tokens a pair of CTAs (cta_group::2): each CTA stages 128
// channels of the weights and half of the tokens, 32 KB a 128-byte K block at
// most, and gets its 128 channels of the result in its own TMEM.  Persistent,
// two accumulators, the last tile's epilogue under the next one's MMAs.  Warp 0
// loads, warp 1 issues the MMAs, 16 warps are the epilogue; waits as in
// tac_gemm_tc2.cuh, and no load uses multicast.  Both issuing warps run their
// loops whole and one elected lane issues, so that descriptors stay in uniform
// registers (4096^3: 87 us with a single thread's loop, 49 with this).
// 4096^3: 2800 TOPS, tensor pipe 80 % busy, L2 hit rate 84 %.  Outputs wider
// than K is deep are bound by the stores (333 x 50257 x 768: 24 us).
struct PairCfg {
  static constexpr int kStages = 6;
  static constexpr int kStageBytes = 2 * 16384;
  static constexpr int kSmem = kStages * kStageBytes + 1024;
  static constexpr int kEpi = 512;     // epilogue threads: four warps a quadrant of TMEM, a fourth of the tokens each
  static constexpr int kThreads = 64 + kEpi;
};

struct W8PairParams {
  W8Params g;
  int w_tiles, t_tiles;      // 256-channel tiles, token tiles
};

template <int YT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairCfg::kThreads, 1)
    w8_pair_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, W8PairParams pp) {
  constexpr int S = PairCfg::kStages;
  const W8Params& p = pp.g;
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t full_bar[S], empty_bar[S], acc_full[2], acc_empty[2], drain_bar;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  __shared__ __align__(16) float as_s[PairCfg::kEpi / 32][64];

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t rank = sm100::cluster_ctarank();
  const int cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
  const int half = p.tn / 2, total = pp.w_tiles * pp.t_tiles;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      sm100::mbar_init(&full_bar[s], 1);
      sm100::mbar_init(&empty_bar[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      sm100::mbar_init(&acc_full[b], 1);
      sm100::mbar_init(&acc_empty[b], 2 * PairCfg::kEpi / 32);   // the epilogue warps of both CTAs
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

  if (warp == 0) {
    uint32_t s = 0, ph = 1, issued = 0;
    wait_rows();
    bool go = true;
    for (int tile = cid; go && tile < total; tile += ncl) {
      const int n0 = tile / pp.t_tiles * 256 + int(rank) * 128, m0 = tile % pp.t_tiles * p.tn + int(rank) * half;
      for (int kb = 0; kb < p.k_blocks; ++kb) {
        go = sm100::mbar_wait_warp(&empty_bar[s], ph, abort_v, p.fault, W8_TIMEOUT_EMPTY);
        if (!go) break;
        if (sm100::elect_one()) {
          if (rank == 0) sm100::mbar_arrive_expect_tx(&full_bar[s], 2 * (16384 + half * 128));
          const uint32_t bar0 = sm100::mapa_shared(&full_bar[s], 0);
          uint8_t* st = smem + s * PairCfg::kStageBytes;
          sm100::tma_load_2d_pair(st, &tm_w, kb * 128, n0, bar0);
          sm100::tma_load_2d_pair(st + 16384, &tm_a, kb * 128, m0, bar0);
        }
        __syncwarp();
        ++issued;
        if (++s == S) s = 0, ph ^= 1;
      }
    }
    if (rank == 0) {
      // both CTAs' copies of the stages still in flight land on these barriers
      for (uint32_t j = issued > uint32_t(S) ? issued - S : 0; j < issued; ++j)
        sm100::mbar_wait(&full_bar[j % S], (j / S) & 1, p.fault, W8_TIMEOUT_DRAIN);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = sm100::idesc_i8(256, p.tn, 0);
      const uint64_t w0 = sm100::smem_desc_sw128(sm100::smem_u32(smem), 16, 1024);
      uint32_t s = 0, ph = 0, local = 0;
      for (int tile = cid; tile < total; tile += ncl, ++local) {
        const uint32_t b = local & 1, aph = (local >> 1) & 1;
        if (!sm100::mbar_wait_warp(&acc_empty[b], aph ^ 1, abort_v, p.fault, W8_TIMEOUT_ACC)) break;
        sm100::tc_fence_after();
        bool ok = true;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          ok = sm100::mbar_wait_warp(&full_bar[s], ph, abort_v, p.fault, W8_TIMEOUT_FULL);
          if (!ok) break;
          sm100::tc_fence_after();
          const uint64_t dw = w0 + s * (PairCfg::kStageBytes >> 4);
          if (sm100::elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              sm100::mma_i8_pair(tmem + b * 256, dw + 2 * k, dw + (16384 >> 4) + 2 * k, idesc, (kb | k) != 0);
            sm100::mma_commit_pair(&empty_bar[s], 0x3);
          }
          __syncwarp();
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
    sm100::mbar_wait(&drain_bar, 0, p.fault, W8_TIMEOUT_DRAIN);
  } else {
    const int row = (warp & 3) * 32 + lane;
    const uint32_t acc_empty0_0 = sm100::mapa_shared(&acc_empty[0], 0), acc_empty0_1 = sm100::mapa_shared(&acc_empty[1], 0);
    const int part = (warp - 2) >> 2;
    uint32_t local = 0;
    wait_rows();
    // a tile's scales are loaded while the tile before it is finished: its channel's, and a token's of each of the
    // warp's (at most two) chunks of 32, which go through the warp's own piece of shared memory
    uint32_t bs = 0, bias = 0;
    float as[2] = {0.f, 0.f};
    // a tile's first token and this thread's channel; from one tile to the next without a division, which every warp
    // would do between its stores and its next wait
    const int step_w = ncl / pp.t_tiles, step_t = ncl % pp.t_tiles;
    int t_next = cid % pp.t_tiles, n_next = cid / pp.t_tiles * 256 + int(rank) * 128 + row;
    auto scales = [&] {
      const int n = n_next, m0 = t_next * p.tn;
      bs = bias = 0;
      if (n < p.N) {
        bs = ld_bits(p.b_scale, p.b_type, n);
        if (p.bias) bias = ld_bits(p.bias, p.bias_type, n);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int tok = part * 32 + k * (PairCfg::kEpi / 4) + lane;
        as[k] = tok < p.tn && m0 + tok < p.M ? __ldg(p.a_scale + m0 + tok) : 0.f;
      }
    };
    scales();                                    // cid < total: there are no more pairs than tiles
    for (int tile = cid; tile < total; tile += ncl, ++local) {
      const uint32_t b = local & 1, aph = (local >> 1) & 1;
      const int n = n_next, m0 = t_next * p.tn;
      const float bs_now = bits_value(bs, p.b_type), bias_now = bits_value(bias, p.bias_type);
      __syncwarp();                              // the warp is done with its last scales
      as_s[warp - 2][lane] = as[0];
      as_s[warp - 2][32 + lane] = as[1];
      __syncwarp();
      t_next += step_t;
      n_next += step_w * 256;
      if (t_next >= pp.t_tiles) t_next -= pp.t_tiles, n_next += 256;
      if (tile + ncl < total) scales();
      if (!sm100::mbar_wait_warp(&acc_full[b], aph, abort_v, p.fault, W8_TIMEOUT_ACC)) break;
      sm100::tc_fence_after();
      // The accumulator is free once its values are in registers.  The arrival is relaxed: as a release it would wait
      // for the warp's stores of this tile and the last.
      auto release = [&] {
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0)
          asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(b ? acc_empty0_1 : acc_empty0_0) : "memory");
      };
      const int chunks = min(2, max(0, (min(p.tn, p.M - m0) - part * 32 + PairCfg::kEpi / 4 - 1) / (PairCfg::kEpi / 4)));
      if (chunks == 0) release();
#pragma unroll 1
      for (int k = 0; k < chunks; ++k) {
        const int c = part * 32 + k * (PairCfg::kEpi / 4);
        uint32_t v[32];
        __syncwarp();
        sm100::tmem_ld32(tmem + (uint32_t((warp & 3) * 32) << 16) + b * 256 + c, v);
        if (k == chunks - 1) release();
        w8_store32<YT>(p, v, as_s[warp - 2] + 32 * k, m0 + c, n, bs_now, bias_now);
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
