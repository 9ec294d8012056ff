// Attention of a few query rows over a 4-bit paged cache: a decode step, a
// group of drafted tokens.  See tac_kv4.cuh for the cache and the factored
// products.
//
// Both products run transposed on mma.sync m16n8k16, the keys (then the
// channels) on its 16 rows and the query rows of one key-value head on its 8
// columns: S^T = C q^T, O^T = C'^T (p s')^T.  A thread's fragment of C is the
// 16 or 8 contiguous bytes of one key that it loads, its fragment of C'^T the
// bytes of the same channels of two keys, interleaved by two PRMTs: no shuffle
// and no second pass through shared memory.  P^T changes from accumulator to
// operand layout by movmatrix.
//
// Each of eight warps takes 32 keys of a tile of 256 and has a ring of stages
// of its own, which it fills two or three tiles ahead by 16-byte asynchronous
// copies; nothing waits for another warp before the unit's end.  (Bulk copies,
// one for the 512 bytes that a head has of 16 keys, need an instruction for
// each, lane by lane: 132 us instead of 114 for 64 ragged sequences.)
//
// Bound by instructions and their latency, not by the cache's bytes: unpacking
// a code takes as many instructions as the products with it, 2.2 are issued a
// clock with 16 warps an SM (125 registers a thread).  64 sequences of
// 1000..8192 tokens, 32 query heads over 8 of 128 values: 96 us (3.1 TB/s; 91
// with the loads left out, 72 with loads alone).  Two of 100,001..131,072 over
// 4 heads: 40 us, of which 14 do not go with the length, and 6 for the join.
//
// Work is laid end to end over all (sequence, head, row block) units.  Where a
// sequence can be long (p.split), the CTAs take equal shares of its tiles
// whatever the lengths: a unit that one CTA covers is finished there, the
// pieces of one that several cover go to the workspace and kv4_join_kernel
// adds them in order.  Else they take whole units, and there is nothing to
// join.  The cuts depend on the lengths and the grid only, so results do not
// change from run to run.
#pragma once
#include <type_traits>

#include "tac_kv4.cuh"
#include "tac_sm100.cuh"

namespace tac {

constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = kRowsWarps * 32;
constexpr float kSlack = 8.f;
constexpr uint32_t kSlackV = 6;
constexpr int kRowsTile = kRowsWarps * 32;         // keys of a tile, 32 a warp

// n / d and n % d for n below 2^31: with 2^(s - 1) < d <= 2^s, m = ceil(2^(31 + s) / d) is less than one above the
// quotient, so n m / 2^(31 + s) exceeds n / d by less than 1 / d.
struct Divider {
  uint32_t d, m, s;
  __host__ __device__ int of(int n) const { return int((uint64_t(uint32_t(n)) * m) >> (31 + s)); }
  __host__ __device__ int rest(int n) const { return n - of(n) * int(d); }
};
inline Divider make_divider(uint32_t d) {
  uint32_t s = 0;
  while ((uint32_t(1) << s) < d) ++s;
  return {d, uint32_t(((uint64_t(1) << (31 + s)) + d - 1) / d), s};
}

struct Kv4RowsParams {
  Kv4Cache c;
  Kv4Seqs s;
  const uint16_t* q;
  uint16_t* o;
  float* lse;            // or null
  int64_t q_tok, q_head; // strides in elements
  int hq, group;         // query heads, query heads of one key-value head
  Divider div;           // by group
  int bf16, causal, split;
  int q_vec, o_vec;      // q's, o's rows are 16-byte aligned
  float scale_log2;      // softmax scale * log2(e)
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

// Codes 0 and 4 (N = 0), 1 and 5, 2 and 6, 3 and 7 of a word as FP16 numbers:
// a code in bits 4..7 of a half with the exponent of 64 is 64 + c, one in bits
// 0..3 with that of 1024 is 1024 + c.  Of the instructions that a pair takes,
// the masks run on the integer pipe, which bounds this kernel once the loads
// overlap, the additions beside them on the other.
//
// For the scores all become 64 + c (960 less is exact): the common 64, and the
// zero point with it, is taken off the sum of a score, where it costs 2^-24 *
// 64 times the query's sum, far below what the weight's rounding to FP16 does.
// For the outputs that would not do: thousands of weights cancel there (64 in
// the sums of 131,072 flat weights cost ten times the output's rounding).
// They get c - 8, and the sum of weights * (z - 8), small as well, is taken off.
// The mask and the exponent go in by one three-input instruction, written out
// because the compiler makes two of them.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(y) : "r"(x), "r"(mask), "r"(bits));
  return y;
}

template <int N>
__device__ __forceinline__ uint32_t kv4_pair64(uint32_t x) {
  const uint32_t y = N >= 2 ? x >> 8 : x;
  if (N & 1) return and_or(y, 0x00f000f0u, 0x54005400u);
  return h2_u(__hadd2(u_h2(and_or(y, 0x000f000fu, 0x64006400u)), __float2half2_rn(-960.f)));
}

template <int N>
__device__ __forceinline__ uint32_t kv4_pair8(uint32_t x) {
  const uint32_t y = N >= 2 ? x >> 8 : x;
  if (N & 1) return h2_u(__hadd2(u_h2(and_or(y, 0x00f000f0u, 0x54005400u)), __float2half2_rn(-72.f)));
  return h2_u(__hadd2(u_h2(and_or(y, 0x000f000fu, 0x64006400u)), __float2half2_rn(-1032.f)));
}

// 64 + z of a parameter word as a float: z in the bits worth 1 .. 8 at 64.
__device__ __forceinline__ float kv4_zero64(uint32_t word) { return __uint_as_float(word * (1u << 17) + 0x42800000u); }

// Two float32 operations an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float exp2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D, int NT>
struct RowsCfg {
  static constexpr int kRows = 8 * NT;
  static constexpr int kPart = kRows * (D + 2);   // floats of a piece: O, then m and l of each row
};

// Tiles of one unit of sequence b, its units, and its cost in what shares are cut in (units if !p.split, else tiles;
// the host sees to it that the sum over the sequences fits 31 bits).
struct SeqCost {
  uint32_t tiles, units, cost;
};

__device__ __forceinline__ SeqCost seq_cost(const Kv4RowsParams& p, const Kv4Seq& s, int rows) {
  SeqCost c;
  c.tiles = max(1, (s.len + kRowsTile - 1) / kRowsTile);
  c.units = (uint32_t(s.n) * p.group + rows - 1) / rows * p.c.heads;
  c.cost = p.split ? c.units * c.tiles : c.units;
  return c;
}

// `total` cut into `parts` shares, the first `rem` of them one larger.
struct Cuts {
  uint32_t total, parts, base, rem;
  Cuts() = default;
  __device__ Cuts(uint32_t total, uint32_t grid) : total(total), parts(min(total, grid)) {
    base = parts ? total / parts : 0;
    rem = total - base * parts;
  }
  __device__ uint32_t at(uint32_t i) const { return i < parts ? i * base + min(i, rem) : total; }
  // the share that tile x lies in
  __device__ uint32_t share(uint32_t x) const {
    const uint32_t big = rem * (base + 1);
    return min(x < big ? x / (base + 1) : rem + (x - big) / base, parts - 1);
  }
};

// All threads of the CTA: the cuts, and the sequence that share `me` begins in (none for an empty share) with the
// place where that sequence begins.
struct Start {
  Cuts cuts;
  uint32_t x0, x1, first;
  int b;
};

__device__ inline Start find_start(const Kv4RowsParams& p, int rows, uint32_t grid, uint32_t me, uint32_t* red, Start* found) {
  const int64_t cap = int64_t(p.s.width) * p.c.page_size;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool one = p.s.batch <= kRowsThreads;    // a thread for each sequence: one pass does
  Start st;
  st.x0 = st.x1 = st.first = 0;
  st.b = p.s.batch;
  // sequences that share rows (offsets that go back) can have more tiles than 32 bits count: then nothing may be found
  if (threadIdx.x == 0) *found = st;
  uint32_t base = 0;
  for (int pass = one ? 1 : 0; pass < 2; ++pass) {
    base = 0;
    for (int b0 = 0; b0 < p.s.batch; b0 += kRowsThreads) {
      const int b = b0 + threadIdx.x;
      const uint32_t c = b < p.s.batch ? seq_cost(p, kv4_seq(p.s, b, cap), rows).cost : 0;
      uint32_t inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += u;
      }
      __syncthreads();
      if (lane == 31) red[warp] = inc;
      __syncthreads();
      uint32_t all = 0, before = base;
#pragma unroll
      for (int w = 0; w < kRowsThreads / 32; ++w) {
        if (w < warp) before += red[w];
        all += red[w];
      }
      if (one) st.cuts = Cuts(all, grid);
      if (pass) {
        if (b0 == 0) st.x0 = st.cuts.at(me), st.x1 = st.cuts.at(me + 1);
        if (st.x0 >= st.x1) return st;           // an empty share
        if (st.x0 < base + all) {                // it begins in this chunk
          const uint32_t start = before + inc - c;
          if (st.x0 >= start && st.x0 < start + c) {
            st.first = start;
            st.b = b;
            *found = st;
          }
          __syncthreads();
          return *found;
        }
      }
      base += all;
    }
    if (!pass) st.cuts = Cuts(base, grid);
  }
  return st;                                     // not reached: a share that is not empty begins somewhere
}

__device__ __forceinline__ float ld_q(const Kv4RowsParams& p, int64_t i) {
  const uint16_t u = __ldg(p.q + i);
  return p.bf16 ? __uint_as_float(uint32_t(u) << 16) : __half2float(__ushort_as_half(u));
}

__device__ __forceinline__ void st_o(const Kv4RowsParams& p, int64_t i, float v) {
  p.o[i] = p.bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// Resident CTAs that the registers and the ring are cut for (kv4_rows_kernel).
__host__ __device__ constexpr int rows_ctas(int D, int NT) { return D == 128 && NT == 2 ? 1 : 2; }
// A stage: 32 keys' codes of K, then of V, then their words.
__host__ __device__ constexpr int rows_stage(int D) { return 2 * 32 * (D / 2) + 2 * 32 * 4; }
__host__ __device__ constexpr int rows_stages(int D, int NT) { return D == 128 && NT == 1 ? 3 : 4; }
// What one warp hands another: O, mu and l of its rows, a float4 of each lane at a time.  The slots take the rings'
// place once every warp has done its tiles.
__host__ __device__ constexpr int rows_slot(int D, int NT) { return 32 * 4 * (NT * D / 4 + 4 * NT); }
__host__ __device__ constexpr int rows_smem(int D, int NT) { return kRowsWarps * rows_stages(D, NT) * rows_stage(D); }

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(sm100::smem_u32(dst)), "l"(src) : "memory");
}

template <int D, int NT>
__global__ void __launch_bounds__(kRowsThreads, rows_ctas(D, NT)) kv4_rows_kernel(Kv4RowsParams p) {
  using Cfg = RowsCfg<D, NT>;
  constexpr int R = Cfg::kRows;
  constexpr int W = D / 32;         // words of one key that a thread converts for S
  constexpr int VW = D / 64;        // words of one key that it converts for O
  constexpr int ST = rows_stages(D, NT), kStage = rows_stage(D);
  static_assert(rows_smem(D, NT) >= 5 * rows_slot(D, NT), "the slots take the rings' place");
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint32_t red[kRowsThreads / 32];
  __shared__ Start found;

  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* const ring = ring_all + warp * ST * kStage;
  if (p.split && threadIdx.x == 0) p.cuts[blockIdx.x] = make_int4(-1, 0, 0, 0);
  const Start sh = find_start(p, R, gridDim.x, blockIdx.x, red, &found);
  // Key of a slab's row r and of row r + 8 (less 8): this order keeps both operands' reads of the ring free of bank
  // conflicts (V's at D = 128 aside: two rows of four share banks in any order).
  const int key_g = g & 1 ? 7 - (g >> 1) : g >> 1;

  int b = sh.b;
  uint32_t off = sh.x0 - sh.first;
  for (uint32_t x = sh.x0; x < sh.x1 && b < p.s.batch;) {
    const Kv4Seq s = kv4_seq(p.s, b, int64_t(p.s.width) * p.c.page_size);
    const SeqCost sc_b = seq_cost(p, s, R);
    if (off >= sc_b.cost) {
      ++b;
      off = 0;
      continue;
    }
    const uint32_t tiles = sc_b.tiles, unit = p.split ? off / tiles : off;
    const int t0 = p.split ? off - unit * tiles : 0;
    const int t1 = p.split ? min(tiles, t0 + (sh.x1 - x)) : tiles;
    const int step_x = p.split ? t1 - t0 : 1;
    const bool first_piece = x == sh.x0;
    const int h = unit % p.c.heads, r0 = unit / p.c.heads * R;
    const int rows_all = s.n * p.group;
    const int t_end = min(t1, (s.len + kRowsTile - 1) / kRowsTile);   // none for an empty sequence
    x += step_x;
    off += step_x;

    const int32_t* table = p.s.table + int64_t(b) * p.s.width;
    if (p.split && first_piece && threadIdx.x == 0) {
      // For kv4_join_kernel: this share's first unit, when the cut before it is the first one inside that unit, with
      // the last CTA that has a piece of it and the place of its first piece
      const uint32_t u0 = sh.x0 - t0, prev = blockIdx.x ? sh.cuts.at(blockIdx.x - 1) : 0;
      if (t0 > 0 && u0 >= prev)
        p.cuts[blockIdx.x] = make_int4(b, r0, sh.cuts.share(u0 + tiles - 1), (u0 == prev ? 0 : 1) | h << 1);
    }

    // ---- copies of this warp's 32 keys of a tile, two slabs of 16 keys that each lie in one page ----
    auto get_page = [&](int tile, int u) -> int {
      const int k0 = tile * kRowsTile + warp * 32 + 16 * u;
      if (tile >= t_end || k0 >= s.len) return -1;
      const int id = __ldg(table + (k0 >> p.c.page_shift));
      return uint32_t(id) < uint32_t(p.c.num_pages) ? id : -1;
    };
    uint32_t have_bits = 0;         // two bits a stage: which of its slabs hold keys
    auto fetch = [&](int tile, int st, const int (&pg)[2]) {
      uint8_t* dst = ring + st * kStage + lane * 16;
      uint32_t bits = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (pg[u] < 0) continue;
        bits |= 1u << u;
        const uint32_t k0 = tile * kRowsTile + warp * 32 + 16 * u;
        const uint64_t row = (uint32_t(pg[u]) * p.c.heads + h) * p.c.page_size + (k0 & (p.c.page_size - 1));   // fits 32 bits
        const uint8_t *ks = p.c.kc + row * (D / 2) + lane * 16, *vs = p.c.vc + row * (D / 2) + lane * 16;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) {
          copy16(dst + u * 16 * (D / 2) + i * 512, ks + i * 512);
          copy16(dst + (32 + u * 16) * (D / 2) + i * 512, vs + i * 512);
        }
        if (lane < 8) {               // the words: 64 bytes of K's, 64 of V's
          const uint32_t* ws = (lane < 4 ? p.c.kp : p.c.vp) + row + (lane & 3) * 4;
          copy16(ring + st * kStage + 32 * D + (lane >> 2) * 128 + u * 64 + (lane & 3) * 16, ws);
        }
      }
      asm volatile("cp.async.commit_group;\n" ::: "memory");
      have_bits = (have_bits & ~(3u << (2 * st))) | bits << (2 * st);
    };
    {
      int pg[ST][2];
#pragma unroll
      for (int i = 0; i < ST; ++i) pg[i][0] = get_page(t0 + i, 0), pg[i][1] = get_page(t0 + i, 1);
#pragma unroll
      for (int i = 0; i < ST; ++i) fetch(t0 + i, i, pg[i]);
    }

    // ---- query rows: FP16, each scaled by the power of two that brings its largest magnitude into [1, 2) ----
    uint32_t qf[NT][2 * W][2];
    float qs[NT][2], qsum[NT][2];
    int lim[NT][2];
    int lim_min = s.len;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 8 + g;
      const bool ok = r < rows_all;
      const int64_t qi = ok ? (s.q0 + p.div.of(r)) * p.q_tok + (h * p.group + p.div.rest(r)) * p.q_head + (D / 4) * t : 0;
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
        lim[n][i] = rr >= rows_all ? 0 : p.causal ? min(s.len, s.p0 + p.div.of(rr) + 1) : s.len;   // keys below it are seen
        if (rr < rows_all) lim_min = min(lim_min, lim[n][i]);
      }
    }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);   // every row sees the keys below

    // Softmax state of a row, per warp.  Weights are exp2(s - mu): mu follows the largest score only when one is more
    // than kSlack above it, so that most tiles need neither the maximum over the warp nor a rescaling.
    float o[NT][D / 16][4] = {};
    float mu[NT][2] = {}, l[NT][2] = {}, zo[NT][2] = {};   // zo: sum of weights * (z - 8), to be taken off o
    // A row's O is held in units of 2^(ve - 127), ve following the exponent of the largest s' among the keys that it
    // has seen (a NaN aside) in the same manner, so that its weights p s' fit FP16 whatever the values' magnitude, and
    // whatever it does not see: they stay below 2^kSlack 2^(kSlackV + 1).
    uint32_t ve[NT][2], vlim = 0;                     // vlim: a word from which on s' is 2^kSlackV such units or more
    uint32_t begun = 0;                               // bit 2n + i: the row has seen a key
#pragma unroll
    for (int n = 0; n < NT; ++n) ve[n][0] = ve[n][1] = 1;

    auto step = [&](int tile, int st, auto masked_c) {
      constexpr bool kMasked = decltype(masked_c)::value;
      const int key0 = tile * kRowsTile + warp * 32;
      const uint32_t have = have_bits >> (2 * st);
      auto seen = [&](int u, int j, int n, int i) { return key0 + 16 * u + 8 * j + key_g < lim[n][i] && (have >> u & 1); };
      const uint8_t* stage = ring + st * kStage;
      uint32_t kpw[2][2], vpw[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t* words = reinterpret_cast<const uint32_t*>(stage + 32 * D) + 16 * u + 8 * j + key_g;
          kpw[u][j] = words[0];
          vpw[u][j] = words[32];
          // a slot without a token may hold any bits
          if (kMasked && !(key0 + 16 * u + 8 * j + key_g < s.len && (have >> u & 1))) kpw[u][j] = vpw[u][j] = 0;
        }
      // ---- S^T ----
      float sc[2][NT][4] = {};
      uint32_t kw[2][2][W];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint8_t* src = stage + (16 * u + 8 * j + key_g) * (D / 2) + t * (D / 8);
          if constexpr (W == 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(src);
            kw[u][j][0] = v.x, kw[u][j][1] = v.y, kw[u][j][2] = v.z, kw[u][j][3] = v.w;
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            kw[u][j][0] = v.x, kw[u][j][1] = v.y;
          }
        }
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t a = kw[u][0][w], c = kw[u][1][w];
          const uint32_t p00 = kv4_pair64<0>(a), p01 = kv4_pair64<0>(c), p10 = kv4_pair64<1>(a), p11 = kv4_pair64<1>(c);
          const uint32_t p20 = kv4_pair64<2>(a), p21 = kv4_pair64<2>(c), p30 = kv4_pair64<3>(a), p31 = kv4_pair64<3>(c);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(sc[u][n], p00, p01, p10, p11, qf[n][2 * w][0], qf[n][2 * w][1]);
            mma_16816(sc[u][n], p20, p21, p30, p31, qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
          }
        }
      // scores less mu (0 for a row that has seen no key yet), two rows at a time
      float hot = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint64_t qs2 = pack2(qs[n][0], qs[n][1]), qsum2 = pack2(qsum[n][0], qsum[n][1]), mu2 = pack2(-mu[n][0], -mu[n][1]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float ks = kv4_scale(kpw[u][j]), kz = -kv4_zero64(kpw[u][j]);
            float v[2];
            unpack2(fma2(fma2(pack2(kz, kz), qsum2, pack2(sc[u][n][2 * j], sc[u][n][2 * j + 1])), mul2(pack2(ks, ks), qs2), mu2), v[0], v[1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (kMasked && !seen(u, j, n, i)) v[i] = -INFINITY;
              sc[u][n][2 * j + i] = v[i];
            }
            hot = max3(hot, v[0], v[1]);
          }
      }
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
            // a row that has seen no key has no mu yet: the next tile comes here whatever its values' scales are
            vlim = min(vlim, begun >> (2 * n + i) & 1 ? (vx + kSlackV) << 23 : 0u);
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
        const uint64_t down2 = pack2(__uint_as_float((254u - ve[n][0]) << 23), __uint_as_float((254u - ve[n][1]) << 23));
        uint64_t l2 = pack2(l[n][0], l[n][1]), zo2 = pack2(zo[n][0], zo[n][1]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float vs = kv4_scale(vpw[u][j]), vz = kv4_zero64(vpw[u][j]) - 72.f;
            const uint64_t e2 = pack2(exp2_(sc[u][n][2 * j]), exp2_(sc[u][n][2 * j + 1]));
            l2 = add2(l2, e2);
            float w[2];
            unpack2(mul2(e2, mul2(pack2(vs, vs), down2)), w[0], w[1]);
            if (kMasked) {                          // a key that this row does not see may hold a NaN scale
              if (!seen(u, j, n, 0)) w[0] = 0.f;
              if (!seen(u, j, n, 1)) w[1] = 0.f;
            }
            const __half2 w2 = __floats2half2_rn(w[0], w[1]);
            zo2 = fma2(pack2(__low2float(w2), __high2float(w2)), pack2(vz, vz), zo2);
            pb[u][n][j] = movmatrix(h2_u(w2));
          }
        unpack2(l2, l[n][0], l[n][1]);
        unpack2(zo2, zo[n][0], zo[n][1]);
      }
      // ---- O^T ----
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t vw[4][VW];
#pragma unroll
        for (int j = 0; j < 4; ++j) {          // rows 2t, 2t + 1, 2t + 8, 2t + 9 of the slab
          const uint8_t* src = stage + (32 + 16 * u + 8 * (j >> 1) + (j & 1 ? 7 - t : t)) * (D / 2) + g * (D / 16);
          if constexpr (VW == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(src);
            vw[j][0] = v.x, vw[j][1] = v.y;
          } else {
            vw[j][0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7632 : 0x5410;
            const uint32_t a = __byte_perm(vw[0][w], vw[1][w], sel), c = __byte_perm(vw[2][w], vw[3][w], sel);
            const uint32_t p00 = kv4_pair8<0>(a), p01 = kv4_pair8<0>(c), p10 = kv4_pair8<1>(a), p11 = kv4_pair8<1>(c);
            const uint32_t p20 = kv4_pair8<2>(a), p21 = kv4_pair8<2>(c), p30 = kv4_pair8<3>(a), p31 = kv4_pair8<3>(c);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16816(o[n][4 * w + 2 * half], p00, p10, p01, p11, pb[u][n][0], pb[u][n][1]);
              mma_16816(o[n][4 * w + 2 * half + 1], p20, p30, p21, p31, pb[u][n][0], pb[u][n][1]);
            }
          }
      }
    };
    int st = 0;
    for (int tile = t0; tile < t_end; ++tile) {
      const int key0 = tile * kRowsTile + warp * 32;
      if (key0 >= s.len) break;
      const int pg[2] = {get_page(tile + ST, 0), get_page(tile + ST, 1)};
      asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 1) : "memory");
      __syncwarp();                 // every lane's copies of this stage have landed
      if (key0 + 32 > lim_min || (have_bits >> (2 * st) & 3u) != 3u) step(tile, st, std::true_type{});
      else step(tile, st, std::false_type{});
      __syncwarp();                 // every lane has read the stage
      fetch(tile + ST, st, pg);
      if (++st == ST) st = 0;
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();                // every ring is at rest: the slots take their place

    // ---- the warps' shares of the unit join pairwise: warp w hands its rows to warp w - half ----
    float mx[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int f = 4; f < 32; f <<= 1) {
          l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], f);
          zo[n][i] += __shfl_xor_sync(0xffffffffu, zo[n][i], f);
        }
        mx[n][i] = l[n][i] == 0.f ? -INFINITY : mu[n][i];
        const float up = __uint_as_float(ve[n][i] << 23);
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          o[n][d][i] = (o[n][d][i] - zo[n][i]) * up;
          o[n][d][2 + i] = (o[n][d][2 + i] - zo[n][i]) * up;
        }
      }
    uint8_t* const slots = ring_all;
#pragma unroll
    for (int half = 4; half; half >>= 1) {
      // a slot is written by the warp that has read it last, or after a barrier that its last reader has joined
      const int slot = half == 4 ? (warp & 3) : half == 2 ? 2 + (warp & 1) : 4;
      float4* hand = reinterpret_cast<float4*>(slots + slot * rows_slot(D, NT)) + lane;
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int d = 0; d < D / 16; ++d) hand[(n * (D / 16 + 1) + d) * 32] = make_float4(o[n][d][0], o[n][d][1], o[n][d][2], o[n][d][3]);
          hand[(n * (D / 16 + 1) + D / 16) * 32] = make_float4(mx[n][0], mx[n][1], l[n][0], l[n][1]);
        }
      }
      __syncthreads();
      if (warp < half && warp + half < kRowsWarps) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 ml = hand[(n * (D / 16 + 1) + D / 16) * 32];
          const float m2[2] = {ml.x, ml.y}, l2[2] = {ml.z, ml.w};
          float ea[2], eb[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float top = fmaxf(mx[n][i], m2[i]), base = top == -INFINITY ? 0.f : top;
            ea[i] = exp2_(mx[n][i] - base);
            eb[i] = exp2_(m2[i] - base);
            mx[n][i] = top;
            l[n][i] = l[n][i] * ea[i] + l2[i] * eb[i];
          }
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const float4 v = hand[(n * (D / 16 + 1) + d) * 32];
            o[n][d][0] = o[n][d][0] * ea[0] + v.x * eb[0];
            o[n][d][1] = o[n][d][1] * ea[1] + v.y * eb[1];
            o[n][d][2] = o[n][d][2] * ea[0] + v.z * eb[0];
            o[n][d][3] = o[n][d][3] * ea[1] + v.w * eb[1];
          }
        }
      }
    }
    __syncthreads();                // the slots have been read: the next unit's copies may start
    if (warp != 0) continue;
    // ---- the unit's result, or this CTA's piece of it: a lane has D / 8 channels in a row of two rows each ----
    const bool whole = t0 == 0 && t1 == int(tiles);
    float* part = p.part + (2 * int64_t(blockIdx.x) + (first_piece ? 0 : 1)) * Cfg::kPart;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = n * 8 + 2 * t + i, rr = r0 + r;
        if (!whole) {
          float4* dst = reinterpret_cast<float4*>(part + r * D + (D / 8) * g);
#pragma unroll
          for (int d = 0; d < D / 16; d += 2) dst[d / 2] = make_float4(o[n][d][i], o[n][d][2 + i], o[n][d + 1][i], o[n][d + 1][2 + i]);
          if (g == 0) part[R * D + r] = mx[n][i], part[R * D + R + r] = l[n][i];
        } else if (rr < rows_all) {
          const int64_t oi = int64_t(s.q0 + p.div.of(rr)) * p.hq + h * p.group + p.div.rest(rr);
          const float inv = l[n][i] == 0.f ? 0.f : 1.f / l[n][i];
          uint16_t* dst = p.o + oi * D + (D / 8) * g;
          uint32_t w[D / 16];
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const float a = o[n][d][i] * inv, c = o[n][d][2 + i] * inv;
            w[d] = p.bf16 ? uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(a))) | uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(c))) << 16
                          : h2_u(__floats2half2_rn(a, c));
          }
          if (p.o_vec) {
#pragma unroll
            for (int d = 0; d < D / 16; d += 4) reinterpret_cast<uint4*>(dst)[d / 4] = make_uint4(w[d], w[d + 1], w[d + 2], w[d + 3]);
          } else {
#pragma unroll
            for (int d = 0; d < D / 16; ++d) dst[2 * d] = uint16_t(w[d]), dst[2 * d + 1] = uint16_t(w[d] >> 16);
          }
          if (p.lse && g == 0) p.lse[oi] = l[n][i] == 0.f ? -INFINITY : (mx[n][i] + log2f(l[n][i])) * 0.69314718055994531f;
        }
      }
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
  const int64_t oi = int64_t(s.q0 + p.div.of(rr)) * p.hq + h * p.group + p.div.rest(rr);
  st_o(p, oi * D + threadIdx.x, sum == 0.f ? 0.f : acc / sum);
  if (p.lse && threadIdx.x == 0) p.lse[oi] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
}

}  // namespace tac
