// 4-bit paged key / value cache: append, read back, attention (tac_kv4.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/taccel_b200.h"
#include "tac_kv4.cuh"
#include "tac_kv4_rows.cuh"
#include "tac_kv4_tc.cuh"

namespace tac {
int* gemm_fault_word();
}

namespace {

using namespace tac;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int status() { return cudaGetLastError() == cudaSuccess ? TAC_OK : TAC_E_CUDA; }

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

// ---- append and read ------------------------------------------------------------------------------------------------
// D / 8 lanes a row, eight values (one word of codes) a lane.
constexpr int kRowThreads = 256;

struct RowArgs {
  Kv4Cache c;
  Kv4Seqs s;
  const void* x[2];
  int64_t tok[2], head[2];
  float* out[2];
  int type, vec;
};

// Position of new token `tok` and its sequence; false where it has none.
__device__ __forceinline__ bool token_place(const Kv4Seqs& s, int tok, int64_t cap, int& b, int64_t& pos) {
  b = tok;
  if (s.indptr) {
    int lo = 0, hi = s.batch;          // the last b with indptr[b] <= tok
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(s.indptr + mid) <= tok) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
  }
  if (b >= s.batch) return false;
  const Kv4Seq q = kv4_seq(s, b, cap);
  if (tok < q.q0 || tok >= q.q0 + q.n) return false;
  pos = int64_t(q.p0) + (tok - q.q0);
  return pos >= 0 && pos < cap;
}

// Index of the cache row of (b, pos, head), or -1.
__device__ __forceinline__ int64_t cache_row(const Kv4Cache& c, const Kv4Seqs& s, int b, int64_t pos, int head) {
  const int page = __ldg(s.table + int64_t(b) * s.width + (pos >> c.page_shift));
  if (page < 0 || page >= c.num_pages) return -1;
  return (int64_t(page) * c.heads + head) * c.page_size + (pos & (c.page_size - 1));
}

__device__ __forceinline__ float elem(const void* p, int type, int64_t i) {
  if (type == TAC_F32) return __ldg(static_cast<const float*>(p) + i);
  const uint16_t u = __ldg(static_cast<const uint16_t*>(p) + i);
  return type == TAC_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float(uint32_t(u) << 16);
}

template <int D>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(RowArgs a) {
  constexpr int L = D / 8;
  const int sub = threadIdx.x % L;
  const int64_t rows = int64_t(a.s.total) * a.c.heads * 2;
  const int64_t cap = int64_t(a.s.width) * a.c.page_size;
  const int64_t step = int64_t(gridDim.x) * (kRowThreads / L);
  // whole warps stay in the loop together: its shuffles name every lane
  for (int64_t i0 = int64_t(blockIdx.x) * (kRowThreads / L); i0 < rows; i0 += step) {
    const int64_t i = i0 + threadIdx.x / L;
    int64_t row = -1;
    float v[8] = {};
    const int which = int(i & 1);
    if (i < rows) {
      const int head = int((i >> 1) % a.c.heads), tok = int((i >> 1) / a.c.heads);
      int b;
      int64_t pos;
      if (token_place(a.s, tok, cap, b, pos)) row = cache_row(a.c, a.s, b, pos, head);
      if (row >= 0) {
        const int64_t e = tok * a.tok[which] + head * a.head[which] + sub * 8;
        if (a.vec && a.type != TAC_F32) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x[which]) + e));
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint16_t h = uint16_t(w[j / 2] >> (16 * (j & 1)));
            v[j] = a.type == TAC_F16 ? __half2float(__ushort_as_half(h)) : __uint_as_float(uint32_t(h) << 16);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = elem(a.x[which], a.type, e + j);
        }
      }
    }
    float lo = 0.f, hi = 0.f;
    uint32_t mag = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo = fminf(lo, v[j]);
      hi = fmaxf(hi, v[j]);
      mag = max(mag, __float_as_uint(v[j]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, o));
    }
    if (row < 0) continue;
    const float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
    uint32_t word, codes = 0;
    if (mag >= 0x7f800000u || s > 3.3e38f) {     // not finite: the row reads as NaN
      word = 0x7fc00000u;
    } else if (s == 0.f) {
      word = 0;
    } else {
      const float z = fminf(rintf(__fdiv_rn(-lo, s)), 15.f);   // a subnormal s may be far from (hi - lo) / 15
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = fminf(fmaxf(rintf(__fdiv_rn(v[j], s)) + z, 0.f), 15.f);
        codes |= uint32_t(c) << (4 * j);
      }
      word = __float_as_uint(s) | uint32_t(z);
    }
    reinterpret_cast<uint32_t*>((which ? a.c.vc : a.c.kc) + row * (D / 2))[sub] = codes;
    if (sub == 0) (which ? a.c.vp : a.c.kp)[row] = word;
  }
}

template <int D>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(RowArgs a) {
  constexpr int L = D / 8;
  const int sub = threadIdx.x % L;
  const int64_t rows = int64_t(a.s.total) * a.c.heads * 2;
  const int64_t cap = int64_t(a.s.width) * a.c.page_size;
  for (int64_t i = int64_t(blockIdx.x) * (kRowThreads / L) + threadIdx.x / L; i < rows;
       i += int64_t(gridDim.x) * (kRowThreads / L)) {
    const int which = int(i & 1), head = int((i >> 1) % a.c.heads), tok = int((i >> 1) / a.c.heads);
    int b;
    int64_t pos, row = -1;
    if (token_place(a.s, tok, cap, b, pos)) row = cache_row(a.c, a.s, b, pos, head);
    float v[8] = {};
    if (row >= 0) {
      const uint32_t codes = __ldg(reinterpret_cast<const uint32_t*>((which ? a.c.vc : a.c.kc) + row * (D / 2)) + sub);
      const uint32_t word = __ldg((which ? a.c.vp : a.c.kp) + row);
      const float s = kv4_scale(word), z = float(word & 0xffffu);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(s, float((codes >> (4 * j)) & 15u) - z);
    }
    float4* dst = reinterpret_cast<float4*>(a.out[which] + (int64_t(tok) * a.c.heads + head) * D + sub * 8);
    dst[0] = make_float4(v[0], v[1], v[2], v[3]);
    dst[1] = make_float4(v[4], v[5], v[6], v[7]);
  }
}

// ---- checks ---------------------------------------------------------------------------------------------------------
int take_cache(const tac_kv4_cache* c, Kv4Cache& out) {
  if (!c || !c->k_codes || !c->v_codes || !c->k_params || !c->v_params || c->num_pages <= 0 || c->heads <= 0 ||
      c->heads > 65536 || (c->head_dim != 64 && c->head_dim != 128))
    return TAC_E_ARGUMENT;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return TAC_E_ARGUMENT;
  if (!aligned(c->k_codes, 16) || !aligned(c->v_codes, 16) || !aligned(c->k_params, 16) || !aligned(c->v_params, 16))
    return TAC_E_ARGUMENT;
  // rows of codes are counted in 32 bits (2^32 rows of 64 values are 128 GB)
  if (int64_t(c->num_pages) * c->heads * c->page_size >= (int64_t(1) << 32)) return TAC_E_ARGUMENT;
  out = {c->k_codes, c->v_codes, c->k_params, c->v_params, c->num_pages, c->page_size, c->heads, 0};
  while ((1 << out.page_shift) < c->page_size) ++out.page_shift;
  return TAC_OK;
}

int take_seqs(const int32_t* table, const int32_t* lens, const int32_t* indptr, int batch, int width, int total,
              const Kv4Cache& c, Kv4Seqs& out) {
  if (!table || !lens || batch <= 0 || width <= 0 || total <= 0) return TAC_E_ARGUMENT;
  if (!indptr && total != batch) return TAC_E_ARGUMENT;
  if (int64_t(width) * c.page_size > (1 << 30)) return TAC_E_ARGUMENT;
  out = {table, lens, indptr, batch, width, total};
  return TAC_OK;
}

int rows_grid(const RowArgs& a, int D) {
  const int64_t rows = int64_t(a.s.total) * a.c.heads * 2, per = kRowThreads / (D / 8);
  return int(std::min<int64_t>((rows + per - 1) / per, int64_t(sm_count()) * 8));
}

// ---- attention ------------------------------------------------------------------------------------------------------
// Rows of a unit: 8 while they hold the query rows of one key-value head of an average sequence, else 16.
int rows_tiles(int batch, int total, int group) { return int64_t(total) * group <= int64_t(8) * batch ? 1 : 2; }

// The workspace is sized for the most CTAs that a launch can have, on any device.
constexpr int kMaxSms = 160;
static_assert(kMaxSms * 2 <= 1024, "kv4_join_kernel holds a weight for each CTA");

uint64_t rows_workspace(int D, int nt) {
  const uint64_t grid = uint64_t(kMaxSms) * rows_ctas(D, nt);
  return grid * 2 * (8 * nt) * (D + 2) * sizeof(float) + grid * sizeof(int4);
}

template <int D, int NT>
int launch_rows(Kv4RowsParams p, void* workspace, cudaStream_t st) {
  const int grid = std::min(sm_count(), kMaxSms) * rows_ctas(D, NT);
  // Contexts of up to four tiles are not worth the second launch that joining pieces takes.
  // Tiles are counted in 31 bits; a batch that could have more goes by units.
  const double capacity = double(p.s.width) * p.c.page_size;
  const double most = (double(p.s.total) * p.hq / (8 * NT) + double(p.s.batch) * p.c.heads) * (capacity / kRowsTile + 1);
  p.split = capacity > 4 * kRowsTile && most < 2147483648.0;
  p.cuts = static_cast<int4*>(workspace);
  p.part = reinterpret_cast<float*>(p.cuts + grid);
  static bool smem_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (cudaFuncSetAttribute(kv4_rows_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, rows_smem(D, NT)) !=
        cudaSuccess)
      return TAC_E_CUDA;
    smem_set[dev] = true;
  }
  kv4_rows_kernel<D, NT><<<grid, kRowsThreads, rows_smem(D, NT), st>>>(p);
  if (int s = status()) return s;
  if (!p.split) return TAC_OK;
  // launched while the first kernel still runs; it waits for that kernel's end before it reads
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid - 1, 8 * NT);
  cfg.blockDim = dim3(D);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<D, NT>, p) == cudaSuccess ? TAC_OK : TAC_E_CUDA;
}

// Prompt chunks: 256 rows a CTA, from 32 rows a sequence and key-value head on.
bool use_tc(int batch, int total, int group) { return int64_t(total) * group > int64_t(32) * batch; }

template <int D, bool BF16>
int launch_tc(const Kv4RowsParams& r, cudaStream_t st) {
  static bool smem_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (cudaFuncSetAttribute(kv4_tc_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, tc_smem(D)) != cudaSuccess)
      return TAC_E_CUDA;
    smem_set[dev] = true;
  }
  Kv4TcParams p{};
  p.r = r;
  p.fault = gemm_fault_word();
  if (!p.fault) return TAC_E_CUDA;
  p.blocks = int((int64_t(r.s.total) * r.group + kTcRows - 1) / kTcRows) + r.s.batch;
  if (int64_t(p.blocks) * r.c.heads > (int64_t(1) << 31) - 1) return TAC_E_ARGUMENT;
  kv4_tc_kernel<D, BF16><<<p.blocks * r.c.heads, kTcThreads, tc_smem(D), st>>>(p);
  return status();
}

}  // namespace

extern "C" int tac_kv4_append(const tac_kv4_cache* cache, const int32_t* page_table, const int32_t* lens,
                              const int32_t* indptr, int batch, int width, int total, const void* K, int64_t k_tok,
                              int64_t k_head, const void* V, int64_t v_tok, int64_t v_head, int type, void* stream) {
  RowArgs a{};
  if (int s = take_cache(cache, a.c)) return s;
  if (int s = take_seqs(page_table, lens, indptr, batch, width, total, a.c, a.s)) return s;
  if (!K || !V || (type != TAC_F32 && type != TAC_F16 && type != TAC_BF16) || k_tok < 0 || k_head < 0 || v_tok < 0 ||
      v_head < 0)
    return TAC_E_ARGUMENT;
  a.x[0] = K, a.x[1] = V;
  a.tok[0] = k_tok, a.tok[1] = v_tok;
  a.head[0] = k_head, a.head[1] = v_head;
  a.type = type;
  a.vec = aligned(K, 16) && aligned(V, 16) && (k_tok | k_head | v_tok | v_head) % 8 == 0;
  const int grid = rows_grid(a, cache->head_dim);
  if (grid <= 0) return TAC_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->head_dim == 64) kv4_append_kernel<64><<<grid, kRowThreads, 0, st>>>(a);
  else kv4_append_kernel<128><<<grid, kRowThreads, 0, st>>>(a);
  return status();
}

extern "C" int tac_kv4_read(const tac_kv4_cache* cache, const int32_t* page_table, const int32_t* lens,
                            const int32_t* indptr, int batch, int width, int total, float* K, float* V, void* stream) {
  RowArgs a{};
  if (int s = take_cache(cache, a.c)) return s;
  if (int s = take_seqs(page_table, lens, indptr, batch, width, total, a.c, a.s)) return s;
  if (!K || !V || !aligned(K, 16) || !aligned(V, 16)) return TAC_E_ARGUMENT;
  a.out[0] = K, a.out[1] = V;
  const int grid = rows_grid(a, cache->head_dim);
  if (grid <= 0) return TAC_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (cache->head_dim == 64) kv4_read_kernel<64><<<grid, kRowThreads, 0, st>>>(a);
  else kv4_read_kernel<128><<<grid, kRowThreads, 0, st>>>(a);
  return status();
}

extern "C" uint64_t tac_kv4_attention_workspace_bytes(int batch, int total, int q_heads, int kv_heads, int head_dim) {
  if (batch <= 0 || total <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  const int nt = rows_tiles(batch, total, q_heads / kv_heads);
  return rows_workspace(head_dim, nt);
}

extern "C" int tac_kv4_attention(const tac_kv4_cache* cache, const int32_t* page_table, const int32_t* lens,
                                 const int32_t* indptr, int batch, int width, int total, const void* Q, int64_t q_tok,
                                 int64_t q_head, int q_heads, int type, float scale, int causal, void* O, float* lse,
                                 void* workspace, uint64_t workspace_bytes, void* stream) {
  Kv4RowsParams p{};
  if (int s = take_cache(cache, p.c)) return s;
  if (int s = take_seqs(page_table, lens, indptr, batch, width, total, p.c, p.s)) return s;
  if (!Q || !O || (type != TAC_F16 && type != TAC_BF16) || q_tok < 0 || q_head < 0 || q_heads <= 0 ||
      q_heads % p.c.heads || q_heads > 65536 || int64_t(total) * q_heads > (int64_t(1) << 31) - 1)
    return TAC_E_ARGUMENT;
  if (!aligned(Q, 2) || !aligned(O, 2) || (lse && !aligned(lse, 4))) return TAC_E_ARGUMENT;
  if (!workspace || !aligned(workspace, 256) ||
      workspace_bytes < tac_kv4_attention_workspace_bytes(batch, total, q_heads, p.c.heads, cache->head_dim))
    return TAC_E_ARGUMENT;
  p.q = static_cast<const uint16_t*>(Q);
  p.o = static_cast<uint16_t*>(O);
  p.lse = lse;
  p.q_tok = q_tok;
  p.q_head = q_head;
  p.hq = q_heads;
  p.group = q_heads / p.c.heads;
  p.div = make_divider(p.group);
  p.bf16 = type == TAC_BF16;
  p.causal = causal != 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.o_vec = aligned(O, 16);
  p.q_vec = aligned(Q, 16) && (q_tok | q_head) % 8 == 0;
  if (sm_count() <= 0) return TAC_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (use_tc(batch, total, p.group)) {
    if (cache->head_dim == 64) return p.bf16 ? launch_tc<64, true>(p, st) : launch_tc<64, false>(p, st);
    return p.bf16 ? launch_tc<128, true>(p, st) : launch_tc<128, false>(p, st);
  }
  const int nt = rows_tiles(batch, total, p.group);
  if (cache->head_dim == 64) return nt == 1 ? launch_rows<64, 1>(p, workspace, st) : launch_rows<64, 2>(p, workspace, st);
  return nt == 1 ? launch_rows<128, 1>(p, workspace, st) : launch_rows<128, 2>(p, workspace, st);
}
