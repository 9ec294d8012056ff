// Attention of a few query rows over a 4-bit paged cache: a decode step, a
// group of drafted tokens.  See tac_kv4.cuh for the cache and the factored
// products.
//
// Both products run transposed on mma.sync m16n8k16, the keys (then the
// channels) on its 16 rows and the query rows of one key-value head on its 8
// columns: S^T = C q^T, O^T = C'^T (p s')^T.  A thread's fragment of C is the
// 16 or 8 contiguous bytes of one key that it loads, its fragment of C'^T the
// bytes of the same channels of two keys, interleaved by two PRMTs: the cache
// goes from global memory to registers to the tensor cores, with no shared
// memory and no shuffle.  P^T changes from accumulator to operand layout by
// movmatrix.  Bound by the cache's bytes: 4.5 bits a value at D = 128.
//
// Work is cut into equal shares over all (sequence, head, row block) units
// laid end to end in tiles of 128 keys, whatever the lengths: a unit that one
// CTA covers is finished there, the pieces of one that several cover go to
// the workspace and kv4_join_kernel adds them in order.  The cuts depend on
// the lengths and the grid only, so results do not change from run to run.
#pragma once
#include <type_traits>

#include "tac_kv4.cuh"

namespace tac {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr float kSlack = 8.f;
constexpr uint32_t kSlackV = 6;
constexpr int kRowsTile = kRowsWarps * 32;   // keys of a tile, 32 a warp

struct Kv4RowsParams {
  Kv4Cache c;
  Kv4Seqs s;
  const uint16_t* q;
  uint16_t* o;
  float* lse;            // or null
  int64_t q_tok, q_head; // strides in elements
  int hq, group;         // query heads, query heads of one key-value head
  int bf16, causal;
  float scale_log2;      // softmax scale * log2(e)
  int q_vec;             // q's rows are 16-byte aligned
  float* part;           // [2 * grid][rows * (D + 2)]
  int4* cuts;            // [grid]: the unit that CTA j's share begins inside of, if it is the first cut of that unit
};

__device__ __forceinline__ uint32_t h2_u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 u_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// Codes 0 and 4 (N = 0), 1 and 5, 2 and 6, 3 and 7 of a word as FP16 64 + c:
// a code in bits 4..7 of a half with the exponent of 64 is 64 + c, one in bits
// 0..3 with that of 1024 is 1024 + c, and 960 less is exact.  The common 64
// (and the zero point with it) is taken off the sums, once a score and once an
// output, where it costs 2^-24 * 64 of the operand's sum, not once a code.
// Of the two instructions that a pair takes, the masks run on the integer
// pipe, which bounds this kernel once the loads overlap, the additions beside
// them on the other.
// The mask and the exponent go in by one three-input instruction, written out
// because the compiler makes two of them.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}

template <int N>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t x) {
  const uint32_t y = N >= 2 ? x >> 8 : x;
  if (N & 1) return and_or(y, 0x00f000f0u, 0x54005400u);
  return h2_u(__hadd2(u_h2(and_or(y, 0x000f000fu, 0x64006400u)), __float2half2_rn(-960.f)));
}

// 64 + z of a parameter word as a float: z in the bits worth 1 .. 8 at 64.
__device__ __forceinline__ float kv4_zero64(uint32_t word) { return __uint_as_float(word * (1u << 17) + 0x42800000u); }

__device__ __forceinline__ float exp2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The shares: `total` tiles over `parts` CTAs, CTA j from total * j / parts on.
struct Shares {
  int64_t total;
  int parts;
  __device__ int64_t at(int64_t j) const { return total * j / parts; }
};

template <int D, int NT>
struct RowsCfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kPart = kRows * (D + 2);   // floats of a piece: O, then m and l of each row
};

// Tiles of one unit of sequence b, and its units.
__device__ __forceinline__ void seq_cost(const Kv4Seq& s, int group, int heads, int rows, int& tiles, int64_t& units) {
  tiles = max(1, (s.len + kRowsTile - 1) / kRowsTile);
  units = (int64_t(s.n) * group + rows - 1) / rows * heads;
}

// Every thread of the CTA: total tiles, then the sequence that tile `x` of all
// lies in and its first tile.
__device__ inline int64_t block_sum(int64_t v, int64_t* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kRowsWarps; ++w) v += red[w];
  return v;
}

__device__ inline int64_t seq_cost_of(const Kv4RowsParams& p, int b, int rows) {
  if (b >= p.s.batch) return 0;
  const Kv4Seq s = kv4_seq(p.s, b, int64_t(p.s.width) * p.c.page_size);
  int tiles;
  int64_t units;
  seq_cost(s, p.group, p.c.heads, rows, tiles, units);
  return units * tiles;
}

__device__ inline Shares make_shares(const Kv4RowsParams& p, int rows, int grid, int64_t* red) {
  int64_t v = 0;
  for (int b = threadIdx.x; b < p.s.batch; b += kRowsThreads) v += seq_cost_of(p, b, rows);
  Shares sh;
  sh.total = block_sum(v, red);
  sh.parts = sh.total < grid ? int(max(sh.total, int64_t(1))) : grid;
  return sh;
}

__device__ inline void find_seq(const Kv4RowsParams& p, int rows, int64_t x, int64_t* red, int* found, int& b, int64_t& first) {
  int64_t base = 0;
  for (int b0 = 0; b0 < p.s.batch; b0 += kRowsThreads) {
    const int64_t c = seq_cost_of(p, b0 + threadIdx.x, rows);
    int64_t inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, inc, o);
      if (int(threadIdx.x & 31) >= o) inc += u;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 31) red[threadIdx.x >> 5] = inc;
    __syncthreads();
    int64_t all = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      if (w < int(threadIdx.x >> 5)) before += red[w];
      all += red[w];
    }
    if (x < base + all) {
      const int64_t start = base + before + inc - c;
      if (x >= start && x < start + c) {
        found[0] = b0 + threadIdx.x;
        *reinterpret_cast<int64_t*>(found + 2) = start;
      }
      __syncthreads();
      b = found[0];
      first = *reinterpret_cast<int64_t*>(found + 2);
      __syncthreads();
      return;
    }
    base += all;
  }
  b = p.s.batch;
  first = base;
}

__device__ __forceinline__ float ld_q(const Kv4RowsParams& p, int64_t i) {
  const uint16_t u = __ldg(p.q + i);
  return p.bf16 ? __uint_as_float(uint32_t(u) << 16) : __half2float(__ushort_as_half(u));
}

__device__ __forceinline__ void st_o(const Kv4RowsParams& p, int64_t i, float v) {
  p.o[i] = p.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// Resident CTAs that the registers are cut for (kv4_rows_kernel).
__host__ __device__ constexpr int rows_ctas(int D, int NT) { return NT == 1 ? (D == 64 ? 4 : 3) : (D == 64 ? 3 : 2); }

template <int D, int NT>
__global__ void __launch_bounds__(kRowsThreads, rows_ctas(D, NT)) kv4_rows_kernel(Kv4RowsParams p) {
  using Cfg = RowsCfg<D, NT>;
  constexpr int R = Cfg::kRows;
  constexpr int W = D / 32;         // words of one key that a thread converts for S
  constexpr int VW = D / 64;        // words of one key that it converts for O
  __shared__ int64_t red[kRowsWarps];
  __shared__ __align__(8) int found[4];
  __shared__ float sm_o[kRowsWarps][R][D + 4];
  __shared__ float sm_m[kRowsWarps][R], sm_l[kRowsWarps][R];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const Shares sh = make_shares(p, R, gridDim.x, red);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (threadIdx.x == 0) p.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if (int(blockIdx.x) >= sh.parts || sh.total == 0) return;
  const int64_t x0 = sh.at(blockIdx.x), x1 = sh.at(blockIdx.x + 1);
  int b;
  int64_t off;
  find_seq(p, R, x0, red, found, b, off);
  off = x0 - off;

  for (int64_t x = x0; x < x1 && b < p.s.batch;) {
    const Kv4Seq s = kv4_seq(p.s, b, int64_t(p.s.width) * p.c.page_size);
    int tiles;
    int64_t units;
    seq_cost(s, p.group, p.c.heads, R, tiles, units);
    if (off >= units * tiles) {
      ++b;
      off = 0;
      continue;
    }
    const int64_t unit = off / tiles;
    const int t0 = int(off - unit * tiles);
    const int t1 = int(min(int64_t(tiles), t0 + (x1 - x)));
    const int h = int(unit % p.c.heads), r0 = int(unit / p.c.heads) * R;
    const int rows_all = s.n * p.group;
    const int32_t* table = p.s.table + int64_t(b) * p.s.width;
    if (x == x0 && threadIdx.x == 0) {
      // For kv4_join_kernel: this share's first unit, when the cut before it is the first one inside that unit, with
      // the last CTA that has a piece of it and the place of its first piece
      int4 cut = make_int4(-1, 0, 0, 0);
      const int64_t u0 = x0 - t0, prev = blockIdx.x ? sh.at(blockIdx.x - 1) : 0;
      if (t0 > 0 && u0 >= prev) {
        int last = blockIdx.x;
        while (last + 1 < sh.parts && sh.at(last + 1) < u0 + tiles) ++last;
        cut = make_int4(b, r0, last, (u0 == prev ? 0 : 1) | h << 1);
      }
      p.cuts[blockIdx.x] = cut;
    }

    // ---- the cache's words of one tile, held in registers a tile ahead ----
    uint32_t kw[2][2][W] = {}, kpw[2][2] = {}, vw[2][4][VW] = {}, vpw[2][2] = {};
    int page[2], page1[2];          // of the tile in kw / vw, of the one after it; -1: no keys
    auto get_page = [&](int tile, int u) -> int {
      const int k0 = tile * kRowsTile + warp * 32 + 16 * u;
      if (tile >= t1 || k0 >= s.len) return -1;
      const int id = __ldg(table + (k0 >> p.c.page_shift));
      return uint32_t(id) < uint32_t(p.c.num_pages) ? id : -1;
    };
    // Cache row of the first of the 16 keys; the number of rows fits 32 bits (checked on the host).
    auto row_of = [&](int tile, int u, int pg) -> uint32_t {
      const uint32_t k0 = tile * kRowsTile + warp * 32 + 16 * u;
      return (uint32_t(pg) * p.c.heads + h) * p.c.page_size + (k0 & (p.c.page_size - 1));
    };
    const uint8_t* const kc = p.c.kc + g * (D / 2) + t * (D / 8);
    const uint8_t* const vc = p.c.vc + 2 * t * (D / 2) + g * (D / 16);
    auto load_k = [&](const int (&pg)[2], const uint32_t (&row)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (pg[u] < 0) continue;
        const uint8_t* src = kc + uint64_t(row[u]) * (D / 2);
        const uint32_t* words = p.c.kp + g + uint64_t(row[u]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (W == 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + j * 8 * (D / 2)));
            kw[u][j][0] = v.x, kw[u][j][1] = v.y, kw[u][j][2] = v.z, kw[u][j][3] = v.w;
          } else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(src + j * 8 * (D / 2)));
            kw[u][j][0] = v.x, kw[u][j][1] = v.y;
          }
          kpw[u][j] = __ldg(words + 8 * j);
        }
      }
    };
    auto load_v = [&](const int (&pg)[2], const uint32_t (&row)[2]) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (pg[u] < 0) continue;
        const uint8_t* src = vc + uint64_t(row[u]) * (D / 2);
        const uint32_t* words = p.c.vp + g + uint64_t(row[u]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {        // keys 2t, 2t + 1, 2t + 8, 2t + 9
          const uint8_t* sj = src + ((j & 1) + 8 * (j >> 1)) * (D / 2);
          if constexpr (VW == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(sj));
            vw[u][j][0] = v.x, vw[u][j][1] = v.y;
          } else {
            vw[u][j][0] = __ldg(reinterpret_cast<const uint32_t*>(sj));
          }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) vpw[u][j] = __ldg(words + 8 * j);
      }
    };
    uint32_t row1[2];               // cache rows of the tile that the next loads take
#pragma unroll
    for (int u = 0; u < 2; ++u) page[u] = get_page(t0, u), page1[u] = get_page(t0 + 1, u);
#pragma unroll
    for (int u = 0; u < 2; ++u) row1[u] = row_of(t0, u, page[u]);
    load_k(page, row1);
    load_v(page, row1);
#pragma unroll
    for (int u = 0; u < 2; ++u) row1[u] = row_of(t0 + 1, u, page1[u]);

    // ---- query rows: FP16, each scaled by the power of two that brings its largest magnitude into [1, 2) ----
    uint32_t qf[NT][2 * W][2];
    float qs[NT][2], qsum[NT][2];
    int lim[NT][2];
    int lim_min = s.len;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 8 + g;
      const bool ok = r < rows_all;
      const int64_t qi = ok ? (s.q0 + r / p.group) * p.q_tok + (h * p.group + r % p.group) * p.q_head + (D / 4) * t : 0;
      float v[D / 4];
      uint32_t mx = 0;
      if (ok && p.q_vec) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 w = __ldg(reinterpret_cast<const uint4*>(p.q + qi) + i);
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint16_t e = uint16_t(ww[j / 2] >> (16 * (j & 1)));
            v[8 * i + j] = p.bf16 ? __uint_as_float(uint32_t(e) << 16) : __half2float(__ushort_as_half(e));
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 4; ++i) v[i] = ok ? ld_q(p, qi + i) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < D / 4; ++i) mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = int(mx >> 23);                        // biased exponent; infinities and NaN stay what they are
      e = e == 255 ? 127 : e < 1 ? 1 : e > 253 ? 253 : e;
      const float down = __uint_as_float(uint32_t(254 - e) << 23);
      float sum = 0.f;                              // of the FP16 values
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const __half2 q2 = __floats2half2_rn(v[8 * w + 2 * hf + j] * down, v[8 * w + 2 * hf + j + 4] * down);
            qf[n][2 * w + hf][j] = h2_u(q2);
            sum += __low2float(q2) + __high2float(q2);
          }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float up = __uint_as_float(uint32_t(e) << 23) * p.scale_log2;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qs[n][i] = __shfl_sync(0xffffffffu, up, (2 * t + i) * 4);
        qsum[n][i] = __shfl_sync(0xffffffffu, sum, (2 * t + i) * 4);
        const int rr = r0 + n * 8 + 2 * t + i;
        lim[n][i] = rr >= rows_all ? 0 : p.causal ? min(s.len, s.p0 + rr / p.group + 1) : s.len;   // keys below it are seen
        if (rr < rows_all) lim_min = min(lim_min, lim[n][i]);
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);   // every row sees the keys below

    // Softmax state of a row, per warp.  Weights are exp2(s - mu): mu follows the largest score only when one is more
    // than kSlack above it, so that most tiles need neither the maximum over the warp nor a rescaling.
    float o[NT][D / 16][4] = {};
    float mu[NT][2] = {}, l[NT][2] = {}, zo[NT][2] = {};   // zo: sum of weights * (64 + z), to be taken off o
    // A row's O is held in units of 2^(ve - 127), ve following the exponent of the largest s' among the keys that it
    // has seen (a NaN aside) in the same manner, so that its weights p s' fit FP16 whatever the values' magnitude, and
    // whatever it does not see: they stay below 2^kSlack 2^(kSlackV + 1).
    uint32_t ve[NT][2], vlim = 0;                     // vlim: a word from which on s' is 2^kSlackV such units or more
    uint32_t begun = 0;                               // bit 2n + i: the row has seen a key
#pragma unroll
    for (int n = 0; n < NT; ++n) ve[n][0] = ve[n][1] = 1;

    auto step = [&](int tile, auto masked_c) {
      constexpr bool kMasked = decltype(masked_c)::value;
      const int key0 = tile * kRowsTile + warp * 32;
      const bool have[2] = {page[0] >= 0, page[1] >= 0};
      auto seen = [&](int u, int j, int n, int i) { return key0 + 16 * u + 8 * j + g < lim[n][i] && have[u]; };
      // ---- S^T ----
      float sc[2][NT][4] = {};
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t a = kw[u][0][w], c = kw[u][1][w];
          const uint32_t p00 = kv4_pair<0>(a), p01 = kv4_pair<0>(c), p10 = kv4_pair<1>(a), p11 = kv4_pair<1>(c);
          const uint32_t p20 = kv4_pair<2>(a), p21 = kv4_pair<2>(c), p30 = kv4_pair<3>(a), p31 = kv4_pair<3>(c);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(sc[u][n], p00, p01, p10, p11, qf[n][2 * w][0], qf[n][2 * w][1]);
            mma_16816(sc[u][n], p20, p21, p30, p31, qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
          }
        }
      // scores less mu (0 for a row that has seen no key yet)
      float hot = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float ks = kv4_scale(kpw[u][j]), kz = kv4_zero64(kpw[u][j]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float v = fmaf(sc[u][n][2 * j + i] - kz * qsum[n][i], ks * qs[n][i], -mu[n][i]);
              if (kMasked && !seen(u, j, n, i)) v = -INFINITY;
              hot = fmaxf(hot, v);
              sc[u][n][2 * j + i] = v;
            }
        }
      load_k(page1, row1);                          // lands during the rest of this tile
      // ---- softmax over the keys of this warp ----
      const uint32_t vtop = max(max(vpw[0][0], vpw[0][1]), max(vpw[1][0], vpw[1][1]));
      if (__any_sync(0xffffffffu, kMasked || hot > kSlack || vtop >= vlim)) {
        vlim = 0xffffffffu;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float corr[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t vx = 0;
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                mx = fmaxf(mx, sc[u][n][2 * j + i]);
                const uint32_t e = (vpw[u][j] >> 23) & 0xffu;
                if ((!kMasked || seen(u, j, n, i)) && e != 255u) vx = max(vx, e);
              }
#pragma unroll
            for (int f = 4; f < 32; f <<= 1) {
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, f));
              vx = max(vx, __shfl_xor_sync(0xffffffffu, vx, f));
            }
            float shift = 0.f;
            if (mx != -INFINITY) {
              const float to = mu[n][i] + (begun >> (2 * n + i) & 1 ? fmaxf(mx, 0.f) : mx);
              shift = to - mu[n][i];
              mu[n][i] = to;
              begun |= 1u << (2 * n + i);
            }
            corr[i] = exp2_(-shift);                // a row's first keys find its sums zero: any finite factor does
            if (!(corr[i] < INFINITY)) corr[i] = 0.f;
            l[n][i] *= corr[i];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < 2; ++j) sc[u][n][2 * j + i] -= shift;
            vx = max(ve[n][i], min(vx, 253u));
            corr[i] *= __uint_as_float((127u - min(vx - ve[n][i], 126u)) << 23);   // 2^(ve - vx)
            ve[n][i] = vx;
            vlim = min(vlim, (vx + kSlackV) << 23);
          }
          zo[n][0] *= corr[0];
          zo[n][1] *= corr[1];
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][d][i] *= corr[i & 1];
        }
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float down[2] = {__uint_as_float((254u - ve[n][0]) << 23), __uint_as_float((254u - ve[n][1]) << 23)};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float vs = kv4_scale(vpw[u][j]), vz = kv4_zero64(vpw[u][j]);
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float e = exp2_(sc[u][n][2 * j + i]);
              l[n][i] += e;
              w[i] = e * (vs * down[i]);
              if (kMasked && !seen(u, j, n, i)) w[i] = 0.f;   // a key that this row does not see may hold a NaN scale
            }
            const __half2 w2 = __floats2half2_rn(w[0], w[1]);
            zo[n][0] += __low2float(w2) * vz;
            zo[n][1] += __high2float(w2) * vz;
            pb[u][n][j] = movmatrix(h2_u(w2));
          }
      }
      // ---- O^T ----
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7632 : 0x5410;
            const uint32_t a = __byte_perm(vw[u][0][w], vw[u][1][w], sel), c = __byte_perm(vw[u][2][w], vw[u][3][w], sel);
            const uint32_t p00 = kv4_pair<0>(a), p01 = kv4_pair<0>(c), p10 = kv4_pair<1>(a), p11 = kv4_pair<1>(c);
            const uint32_t p20 = kv4_pair<2>(a), p21 = kv4_pair<2>(c), p30 = kv4_pair<3>(a), p31 = kv4_pair<3>(c);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16816(o[n][4 * w + 2 * half], p00, p10, p01, p11, pb[u][n][0], pb[u][n][1]);
              mma_16816(o[n][4 * w + 2 * half + 1], p20, p30, p21, p31, pb[u][n][0], pb[u][n][1]);
            }
          }
      load_v(page1, row1);                          // lands during the next tile's scores
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        page[u] = page1[u];
        page1[u] = get_page(tile + 2, u);
        row1[u] = row_of(tile + 2, u, page1[u]);
      }
    };
    for (int tile = t0; tile < t1; ++tile) {
      const int key0 = tile * kRowsTile + warp * 32;
      if (key0 >= s.len) break;
      if (key0 + 32 > lim_min || page[0] < 0 || page[1] < 0) step(tile, std::true_type{});
      else step(tile, std::false_type{});
    }

    // ---- the warps' pieces of the unit, then the unit's result or this CTA's piece of it ----
    __syncthreads();                               // the last unit's reads of sm_* are done
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = l[n][i], z = zo[n][i];
#pragma unroll
        for (int f = 4; f < 32; f <<= 1) {
          v += __shfl_xor_sync(0xffffffffu, v, f);
          z += __shfl_xor_sync(0xffffffffu, z, f);
        }
        zo[n][i] = z;
        if (g == 0) {
          sm_m[warp][n * 8 + 2 * t + i] = v == 0.f ? -INFINITY : mu[n][i];
          sm_l[warp][n * 8 + 2 * t + i] = v;
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            sm_o[warp][n * 8 + 2 * t + (i & 1)][(D / 8) * g + 8 * w + 2 * j + (i >> 1)] =
                (o[n][4 * w + j][i] - zo[n][i & 1]) * __uint_as_float(ve[n][i & 1] << 23);
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    float* part = p.part + (2 * int64_t(blockIdx.x) + (x == x0 ? 0 : 1)) * Cfg::kPart;
    for (int i = threadIdx.x; i < R * D; i += kRowsThreads) {
      const int r = i / D, d = i % D;
      float mx = sm_m[0][r];
#pragma unroll
      for (int w = 1; w < kRowsWarps; ++w) mx = fmaxf(mx, sm_m[w][r]);
      const float mu = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float e = exp2_(sm_m[w][r] - mu);
        sum += sm_l[w][r] * e;
        acc += sm_o[w][r][d] * e;
      }
      if (whole) {
        const int rr = r0 + r;
        if (rr < rows_all) {
          const int64_t oi = int64_t(s.q0 + rr / p.group) * p.hq + h * p.group + rr % p.group;
          st_o(p, oi * D + d, sum == 0.f ? 0.f : acc / sum);
          if (p.lse && d == 0) p.lse[oi] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
        }
      } else {
        part[i] = acc;
        if (d == 0) part[R * D + r] = mx, part[R * D + R + r] = sum;
      }
    }
    x += t1 - t0;
    off += t1 - t0;
  }
}

// Joins the pieces of the units that several CTAs covered: CTA (j, r) row r of
// the unit whose first cut is the one before share j.  The pieces' weights
// first, so that their sums are independent loads.
template <int D, int NT>
__global__ void __launch_bounds__(D) kv4_join_kernel(Kv4RowsParams p) {
  using Cfg = RowsCfg<D, NT>;
  constexpr int R = Cfg::kRows, kMost = 1024;
  __shared__ float wt[kMost], wmax[D / 32], wsum[D / 32];
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const int j = blockIdx.x + 1, r = blockIdx.y;
  const int4 cut = p.cuts[j];
  if (cut.x < 0) return;
  const Kv4Seq s = kv4_seq(p.s, cut.x, int64_t(p.s.width) * p.c.page_size);
  const int rr = cut.y + r, h = cut.w >> 1;
  if (rr >= s.n * p.group) return;
  const int pieces = cut.z - j + 2;                // of CTAs j - 1 .. cut.z; at most the grid, which kMost bounds
  auto piece = [&](int i) { return p.part + (2 * int64_t(j - 1 + i) + (i == 0 ? cut.w & 1 : 0)) * Cfg::kPart; };
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < pieces; i += D) mx = fmaxf(mx, wt[i] = piece(i)[R * D + r]);
#pragma unroll
  for (int f = 16; f; f >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, f));
  if ((threadIdx.x & 31) == 0) wmax[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < D / 32; ++w) mx = fmaxf(mx, wmax[w]);
  const float mu = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  for (int i = threadIdx.x; i < pieces; i += D) {
    const float e = exp2_(wt[i] - mu);
    wt[i] = e;
    sum += piece(i)[R * D + R + r] * e;
  }
#pragma unroll
  for (int f = 16; f; f >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, f);
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < D / 32; ++w) sum += wsum[w];
  float acc = 0.f;
#pragma unroll 8
  for (int i = 0; i < pieces; ++i) acc += piece(i)[r * D + threadIdx.x] * wt[i];
  const int64_t oi = int64_t(s.q0 + rr / p.group) * p.hq + h * p.group + rr % p.group;
  st_o(p, oi * D + threadIdx.x, sum == 0.f ? 0.f : acc / sum);
  if (p.lse && threadIdx.x == 0) p.lse[oi] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace tac
