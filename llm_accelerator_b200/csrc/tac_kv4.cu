// 4-bit paged key / value cache: append, read back, attention (tac_kv4.cuh).
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "../../include/taccel_b200.h"
#include "tac_kv4.cuh"
#include "tac_kv4_rows.cuh"
#include "tac_kv4_tc.cuh"
#include "tac_launch.cuh"

namespace tac {
int* gemm_fault_word();
}

namespace {

using namespace tac;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

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
// A CTA takes a run of tokens.  Each lane of a warp finds the place of one of
// them (a search in indptr, the length, the page), all at once; then the
// tokens' 2 * heads rows go by, a few lanes a row, two tokens' loads in
// flight.  Bound by the bytes: D values in and D / 2 + 4 bytes out a row
// (append), D / 2 + 4 in and 4 D out (read).  Ragged prompts of 19,000 tokens,
// 8 heads of 128: append 32 us, bound by instructions (2.6 a clock) where its
// bytes take 15; read 32 us, 5.6 TB/s.
constexpr int kRowThreads = 256;

struct RowArgs {
  Kv4Cache c;
  Kv4Seqs s;
  const void* x[2];
  int64_t tok[2], head[2];
  float* out[2];
  int type, vec;
  int run;                // tokens of a CTA, at most 32
};

constexpr uint32_t kNoRow = 0xffffffffu;        // there are fewer than 2^32 rows

// Cache row of head 0 of new token `tok`, kNoRow where it has no place.
__device__ __forceinline__ uint32_t token_row(const Kv4Cache& c, const Kv4Seqs& s, int tok) {
  if (tok >= s.total) return kNoRow;
  int b = tok;
  if (s.indptr) {
    int lo = 0, hi = s.batch;                    // the last b with indptr[b] <= tok
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(s.indptr + mid) <= tok) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
  }
  if (b >= s.batch) return kNoRow;
  const int64_t cap = int64_t(s.width) * c.page_size;
  const Kv4Seq q = kv4_seq(s, b, cap);
  if (tok < q.q0 || tok >= q.q0 + q.n) return kNoRow;
  const int64_t pos = int64_t(q.p0) + (tok - q.q0);
  if (pos < 0 || pos >= cap) return kNoRow;
  const int page = __ldg(s.table + int64_t(b) * s.width + (pos >> c.page_shift));
  if (uint32_t(page) >= uint32_t(c.num_pages)) return kNoRow;
  return uint32_t(page) * c.heads * c.page_size + (uint32_t(pos) & (c.page_size - 1));
}

__device__ __forceinline__ float elem(const void* p, int type, int64_t i) {
  if (type == TAC_F32) return __ldg(static_cast<const float*>(p) + i);
  const uint16_t u = __ldg(static_cast<const uint16_t*>(p) + i);
  return type == TAC_F16 ? __half2float(__ushort_as_half(u)) : __uint_as_float(uint32_t(u) << 16);
}

// Codes of 16 values of a lane and the row's parameter word, from the row's
// extremes.  SHORT: the values have 11 significant bits at most (FP16, BF16).
template <bool SHORT>
__device__ __forceinline__ uint2 codes16(const float (&v)[16], float lo, float hi, uint32_t& word) {
  const float s = __bfloat162float(__float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f)));
  uint2 out = make_uint2(0, 0);
  if (!(s <= 3.3e38f)) {                         // an infinity, a NaN or a range beyond float32: the row reads as NaN
    word = 0x7fc00000u;
  } else if (s == 0.f) {
    word = 0;
  } else if (SHORT && s >= 0x1p-100f) {
    // x / s by one residual correction of x * (1 / s) (Markstein's): x has 11 bits at most and s 8, so x - q s is exact
    // and the corrected q within 2^-47 of the quotient, relative; a quotient halfway between two whole numbers is
    // representable and comes out exactly, and no other lies within 2^-13 of one.  Adding 1.5 * 2^23 rounds it to a
    // whole number, half to even; z and the clamp are exact there.  No code is below 0: z is lo's rounding.
    constexpr float kMagic = 12582912.f;
    const float r = __frcp_rn(s);
    auto quotient = [&](float x) {
      const float q = __fmul_rn(x, r);
      return __fmaf_rn(__fmaf_rn(-q, s, x), r, q);
    };
    const float z = -__fsub_rn(__fadd_rn(quotient(lo), kMagic), kMagic);
    uint32_t acc[2] = {0, 0};                    // sum of 16^j (bits of kMagic + code)
#pragma unroll
    for (int j = 15; j >= 0; --j) {
      const float c = fminf(__fadd_rn(__fadd_rn(quotient(v[j]), kMagic), z), kMagic + 15.f);
      acc[j / 8] = acc[j / 8] * 16u + __float_as_uint(c);
    }
    const uint32_t off = __float_as_uint(kMagic) * 0x11111111u;
    out = make_uint2(acc[0] - off, acc[1] - off);
    word = __float_as_uint(s) | uint32_t(z);
  } else {
    const float z = fminf(rintf(__fdiv_rn(-lo, s)), 15.f);   // a subnormal s may be far from (hi - lo) / 15
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float c = fminf(fmaxf(rintf(__fdiv_rn(v[j], s)) + z, 0.f), 15.f);
      (j < 8 ? out.x : out.y) |= uint32_t(c) << (4 * (j & 7));
    }
    word = __float_as_uint(s) | uint32_t(z);
  }
  return out;
}

// Extremes of packed 16-bit values; a NaN stays.
__device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b, bool f16) {
  uint32_t r;
  if (f16) asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, bool f16) {
  uint32_t r;
  if (f16) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// TYPE: TAC_F16 or TAC_BF16 with 16-byte aligned rows; -1: any type and alignment.
template <int D, int TYPE>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(RowArgs a) {
  constexpr int L = D / 16, kPair = 2;
  const int rows = blockDim.x / L;
  const int sub = threadIdx.x % L, lane = threadIdx.x & 31;
  const int64_t t0 = int64_t(blockIdx.x) * a.run;
  const uint32_t mine = lane < a.run && t0 + lane < a.s.total ? token_row(a.c, a.s, int(t0 + lane)) : kNoRow;
  // whole warps take part in every pass: its shuffles name every lane
  for (int r0 = 0; r0 < 2 * a.c.heads; r0 += rows) {
    const int r = r0 + int(threadIdx.x) / L;
    const bool in = r < 2 * a.c.heads;
    const int which = r >= a.c.heads, head = in ? r - (which ? a.c.heads : 0) : 0;
    const void* src = which ? a.x[1] : a.x[0];
    const int64_t tok = which ? a.tok[1] : a.tok[0];
    const int64_t e0 = t0 * tok + head * (which ? a.head[1] : a.head[0]) + sub * 16;
    uint8_t* const codes = (which ? a.c.vc : a.c.kc) + sub * 8;
    uint32_t* const words = which ? a.c.vp : a.c.kp;
    for (int k0 = 0; k0 < a.run; k0 += kPair) {
      uint32_t base[kPair];
      uint4 raw[kPair][2];
#pragma unroll
      for (int k = 0; k < kPair; ++k) {
        base[k] = k0 + k < a.run ? __shfl_sync(0xffffffffu, mine, k0 + k) : kNoRow;
        raw[k][0] = raw[k][1] = make_uint4(0, 0, 0, 0);
        if (TYPE >= 0 && in && base[k] != kNoRow) {
          const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(src) + e0 + (k0 + k) * tok);
          raw[k][0] = __ldg(q);
          raw[k][1] = __ldg(q + 1);
        }
      }
#pragma unroll
      for (int k = 0; k < kPair; ++k) {
        if (base[k] == kNoRow) continue;         // the whole CTA
        float v[16] = {}, lo, hi;
        if (TYPE >= 0) {
          constexpr bool kF16 = TYPE == TAC_F16;
          const uint32_t w[8] = {raw[k][0].x, raw[k][0].y, raw[k][0].z, raw[k][0].w, raw[k][1].x, raw[k][1].y, raw[k][1].z, raw[k][1].w};
          uint32_t mn = 0, mx = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) mn = min2(mn, w[j], kF16), mx = max2(mx, w[j], kF16);
#pragma unroll
          for (int o = 1; o < L; o <<= 1) {
            mn = min2(mn, __shfl_xor_sync(0xffffffffu, mn, o), kF16);
            mx = max2(mx, __shfl_xor_sync(0xffffffffu, mx, o), kF16);
          }
          mn = min2(mn, mn >> 16, kF16);
          mx = max2(mx, mx >> 16, kF16);
          auto f32 = [](uint32_t h) { return kF16 ? __half2float(__ushort_as_half(uint16_t(h))) : __uint_as_float(h << 16); };
          lo = f32(mn & 0xffffu);
          hi = f32(mx & 0xffffu);
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = f32((w[j / 2] >> (16 * (j & 1))) & 0xffffu);
        } else {
          bool nan = false;
          lo = hi = 0.f;
          if (in) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = elem(src, a.type, e0 + (k0 + k) * tok + j);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            lo = fminf(lo, v[j]);
            hi = fmaxf(hi, v[j]);
            nan |= v[j] != v[j];
          }
          if (nan) hi = __uint_as_float(0x7f800000u);
#pragma unroll
          for (int o = 1; o < L; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
          }
        }
        uint32_t word;
        const uint2 c = codes16<TYPE >= 0>(v, lo, hi, word);
        if (in) {
          const uint64_t row = base[k] + uint32_t(head) * a.c.page_size;
          *reinterpret_cast<uint2*>(codes + row * (D / 2)) = c;
          if (sub == 0) words[row] = word;
        }
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(RowArgs a) {
  constexpr int L = D / 4, kRows = kRowThreads / L, kQuad = 4;   // four values a lane: a warp writes 512 bytes in one run
  const int sub = threadIdx.x % L, lane = threadIdx.x & 31;
  const int64_t t0 = int64_t(blockIdx.x) * a.run;
  const uint32_t mine = lane < a.run && t0 + lane < a.s.total ? token_row(a.c, a.s, int(t0 + lane)) : kNoRow;
  for (int r0 = 0; r0 < 2 * a.c.heads; r0 += kRows) {
    const int r = r0 + int(threadIdx.x) / L;
    const bool in = r < 2 * a.c.heads;
    const int which = r >= a.c.heads, head = in ? r - (which ? a.c.heads : 0) : 0;
    const uint8_t* const codes = (which ? a.c.vc : a.c.kc) + sub * 2;
    const uint32_t* const words = which ? a.c.vp : a.c.kp;
    float* const dst = (which ? a.out[1] : a.out[0]) + (t0 * a.c.heads + head) * D + sub * 4;
    for (int k0 = 0; k0 < a.run; k0 += kQuad) {
      uint32_t code[kQuad], word[kQuad];
#pragma unroll
      for (int k = 0; k < kQuad; ++k) {
        code[k] = word[k] = 0;                   // a row without a place reads as zeros
        const uint32_t base = k0 + k < a.run ? __shfl_sync(0xffffffffu, mine, k0 + k) : kNoRow;
        if (in && base != kNoRow) {
          const uint64_t row = base + uint32_t(head) * a.c.page_size;
          code[k] = __ldg(reinterpret_cast<const uint16_t*>(codes + row * (D / 2)));
          word[k] = __ldg(words + row);
        }
      }
#pragma unroll
      for (int k = 0; k < kQuad; ++k) {
        if (!in || k0 + k >= a.run || t0 + k0 + k >= a.s.total) break;
        const float s = kv4_scale(word[k]), z = float(word[k] & 0xffffu);
        float4 o;
        o.x = __fmul_rn(s, float(code[k] & 15u) - z);
        o.y = __fmul_rn(s, float((code[k] >> 4) & 15u) - z);
        o.z = __fmul_rn(s, float((code[k] >> 8) & 15u) - z);
        o.w = __fmul_rn(s, float(code[k] >> 12) - z);
        *reinterpret_cast<float4*>(dst + int64_t(k0 + k) * a.c.heads * D) = o;
      }
    }
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

// Tokens of a CTA: one while every token finds an SM to itself, then as many as keep twelve CTAs an SM, to the lanes' 32.
void set_run(RowArgs& a, int* grid) {
  const int64_t ctas = int64_t(sm_count()) * 12;
  a.run = ctas > 0 ? int(std::max<int64_t>(1, std::min<int64_t>(32, (a.s.total + ctas - 1) / ctas))) : 0;
  *grid = a.run ? int((int64_t(a.s.total) + a.run - 1) / a.run) : 0;
}

template <int D>
int launch_append(const RowArgs& a, int grid, cudaStream_t st) {
  // no more threads than a token's rows keep busy
  const int threads = std::min(kRowThreads, (2 * a.c.heads * (D / 16) + 31) / 32 * 32);
  if (a.vec && a.type == TAC_F16) return launch(kv4_append_kernel<D, TAC_F16>, grid, threads, 0, st, a);
  if (a.vec && a.type == TAC_BF16) return launch(kv4_append_kernel<D, TAC_BF16>, grid, threads, 0, st, a);
  return launch(kv4_append_kernel<D, -1>, grid, threads, 0, st, a);
}

// ---- attention ------------------------------------------------------------------------------------------------------
// Rows of a unit: 8 while they hold the query rows of one key-value head of an average sequence, else 16.
int rows_tiles(int batch, int total, int group) { return int64_t(total) * group <= int64_t(8) * batch ? 1 : 2; }

// The workspace is sized for the most CTAs that a launch can have, on any device.
constexpr int kMaxSms = 160;
static_assert(kMaxSms * 2 <= 1024, "kv4_join_kernel holds a weight for each CTA");

// Whether CTAs share the units of long sequences.  Contexts of up to four tiles are not worth the second launch that
// joining pieces takes.  Tiles are counted in 31 bits; a batch that could have more goes by units.
bool rows_split(int batch, int width, int page_size, int total, int q_heads, int kv_heads, int nt) {
  const double capacity = double(width) * page_size;
  const double most = (double(total) * q_heads / (8 * nt) + double(batch) * kv_heads) * (capacity / kRowsTile + 1);
  return capacity > 4 * kRowsTile && most < 2147483648.0;
}

uint64_t rows_workspace(int D, int nt) {
  const uint64_t grid = uint64_t(kMaxSms) * rows_ctas(D, nt);
  return grid * 2 * (8 * nt) * (D + 2) * sizeof(float) + grid * sizeof(int4);
}

template <int D, int NT>
int launch_rows(Kv4RowsParams p, void* workspace, cudaStream_t st) {
  const int grid = std::min(sm_count(), kMaxSms) * rows_ctas(D, NT);
  p.split = rows_split(p.s.batch, p.s.width, p.c.page_size, p.s.total, p.hq, p.c.heads, NT);
  p.cuts = static_cast<int4*>(workspace);
  p.part = reinterpret_cast<float*>(p.cuts + grid);
  static bool smem_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (int e = status(cudaFuncSetAttribute(kv4_rows_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, rows_smem(D, NT)))) return e;
    smem_set[dev] = true;
  }
  if (int s = launch(kv4_rows_kernel<D, NT>, grid, kRowsThreads, rows_smem(D, NT), st, p)) return s;
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
  return status(cudaLaunchKernelEx(&cfg, kv4_join_kernel<D, NT>, p));
}

// The prompt kernel (256 rows a CTA, one CTA an SM) where it is faster than the row kernel, whose time goes with all
// rows: measured per key, 3.6e-6 us a row and key-value head against 0.025 us a round of CTAs over the SMs at D = 128,
// 2.3e-6 against 0.021 at D = 64 (64 rows for each of 64 heads: 63 us by rows, 136 by the prompt kernel; 512 rows for
// each of 16: 113 and 103).  The rows of a sequence are taken at their mean, and only batches of like sequences have been
// measured: one with a long chunk beside decode rows goes whole to one kernel, which is not the best for either part.
bool use_tc(int batch, int total, int group, int kv_heads, int head_dim) {
  const double rows = double(total) * group / batch, units = double(batch) * kv_heads;
  const double rounds = std::max(1.0, units * std::ceil(rows / kTcRows) / 148);
  return units * rows > (head_dim == 128 ? 8000 : 10500) * rounds;
}

template <int D, bool BF16>
int launch_tc(const Kv4RowsParams& r, cudaStream_t st) {
  static bool smem_set[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return TAC_E_CUDA;
  if (!smem_set[dev]) {
    if (int e = status(cudaFuncSetAttribute(kv4_tc_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, tc_smem(D)))) return e;
    smem_set[dev] = true;
  }
  Kv4TcParams p{};
  p.r = r;
  p.fault = gemm_fault_word();
  if (!p.fault) return TAC_E_CUDA;
  p.blocks = int((int64_t(r.s.total) * r.group + kTcRows - 1) / kTcRows) + r.s.batch;
  if (int64_t(p.blocks) * r.c.heads > (int64_t(1) << 31) - 1) return TAC_E_ARGUMENT;
  return launch(kv4_tc_kernel<D, BF16>, p.blocks * r.c.heads, kTcThreads, tc_smem(D), st, p);
}

}  // namespace

extern "C" int tac_kv4_append(const tac_kv4_cache* cache, const int32_t* page_table, const int32_t* lens,
                              const int32_t* indptr, int batch, int width, int total, const void* K, int64_t k_tok,
                              int64_t k_head, const void* V, int64_t v_tok, int64_t v_head, int type, void* stream) {
  RowArgs a{};
  if (int s = take_cache(cache, a.c)) return s;
  if (int s = take_seqs(page_table, lens, indptr, batch, width, total, a.c, a.s)) return s;
  if (!K || !V || (type != TAC_F32 && type != TAC_F16 && type != TAC_BF16) || k_tok < 0 || k_head < 0 || v_tok < 0 ||
      v_head < 0 || !aligned(K, type == TAC_F32 ? 4 : 2) || !aligned(V, type == TAC_F32 ? 4 : 2))
    return TAC_E_ARGUMENT;
  a.x[0] = K, a.x[1] = V;
  a.tok[0] = k_tok, a.tok[1] = v_tok;
  a.head[0] = k_head, a.head[1] = v_head;
  a.type = type;
  a.vec = aligned(K, 16) && aligned(V, 16) && (k_tok | k_head | v_tok | v_head) % 8 == 0;
  int grid;
  set_run(a, &grid);
  if (grid <= 0) return TAC_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return cache->head_dim == 64 ? launch_append<64>(a, grid, st) : launch_append<128>(a, grid, st);
}

extern "C" int tac_kv4_read(const tac_kv4_cache* cache, const int32_t* page_table, const int32_t* lens,
                            const int32_t* indptr, int batch, int width, int total, float* K, float* V, void* stream) {
  RowArgs a{};
  if (int s = take_cache(cache, a.c)) return s;
  if (int s = take_seqs(page_table, lens, indptr, batch, width, total, a.c, a.s)) return s;
  if (!K || !V || !aligned(K, 16) || !aligned(V, 16)) return TAC_E_ARGUMENT;
  a.out[0] = K, a.out[1] = V;
  int grid;
  set_run(a, &grid);
  if (grid <= 0) return TAC_E_CUDA;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return launch(cache->head_dim == 64 ? kv4_read_kernel<64> : kv4_read_kernel<128>, grid, kRowThreads, 0, st, a);
}

extern "C" uint64_t tac_kv4_attention_workspace_bytes(int batch, int width, int page_size, int total, int q_heads,
                                                      int kv_heads, int head_dim) {
  if (batch <= 0 || width <= 0 || page_size <= 0 || total <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  const int group = q_heads / kv_heads, nt = rows_tiles(batch, total, group);
  if (use_tc(batch, total, group, kv_heads, head_dim) || !rows_split(batch, width, page_size, total, q_heads, kv_heads, nt)) return 0;
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
  const uint64_t need =
      tac_kv4_attention_workspace_bytes(batch, width, cache->page_size, total, q_heads, p.c.heads, cache->head_dim);
  if (need && (!workspace || !aligned(workspace, 256) || workspace_bytes < need)) return TAC_E_ARGUMENT;
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
  if (use_tc(batch, total, p.group, p.c.heads, cache->head_dim)) {
    if (cache->head_dim == 64) return p.bf16 ? launch_tc<64, true>(p, st) : launch_tc<64, false>(p, st);
    return p.bf16 ? launch_tc<128, true>(p, st) : launch_tc<128, false>(p, st);
  }
  const int nt = rows_tiles(batch, total, p.group);
  if (cache->head_dim == 64) return nt == 1 ? launch_rows<64, 1>(p, workspace, st) : launch_rows<64, 2>(p, workspace, st);
  return nt == 1 ? launch_rows<128, 1>(p, workspace, st) : launch_rows<128, 2>(p, workspace, st);
}
