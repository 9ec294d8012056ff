// Attention of many query rows (prompt chunks) over a 4-bit paged cache, on
// tcgen05.  See tac_kv4.cuh for the cache.
//
// A CTA takes 256 query rows of one key-value head (token-major, the group's
// query heads of a token side by side, so one unpacking of a key serves them
// all) and walks the keys up to its last row's position in tiles of 128:
//   warps 0..3, 4..7  two row groups of 128, a thread a row: Q to shared
//                     memory, softmax of S out of TMEM, P into TMEM, O out
//   warps 8..11       unpack the tile's keys, a thread a key, into the
//                     swizzled layout that the MMAs read
//   warp 12           issues the MMAs: S = Q C^T (FP16), O += P V
//   warps 16..23      unpack its values, a thread half a key (13..15 idle)
// S, P and the MMAs go in steps of 64 keys, two steps in flight for each
// group: while a group's threads are at one step's softmax the tensor core
// does P V of the step before and S of the step after it.  (Whole tiles of 128
// keys, one S a group, left a group's threads and the tensor core waiting for
// each other: 353 us for ragged chunks of 5,596 rows of 32 heads, of
// which this took 335.)  Per
// tile and group D = 128 needs 1024 tensor clocks, and 1024 clocks of the
// exponential unit.
//
// Both products have whole numbers (codes less zero point, exact in FP16) for
// the cache's side.  The keys' scales multiply S in float32, the values' scales
// the weights before these are rounded to FP16, once; the query is FP16, scaled
// by a power of two for each row.  So nothing is rounded to BF16 but the result.
// Bound by the chain S, softmax, P, O of a group's step and the issue of its
// MMAs: 630 TFLOP/s at those chunks (342 us), tensor pipe 31 % and exponential
// unit 33 % busy, an eighth of the time in the CTAs' prologues.  One S product
// of 128 keys for two steps (366 us) and softmax steps pipelined within a
// thread at 192 registers (387 us) were slower.
// TMEM: two S of each group (64 columns; P takes the first half of its S), then
// O of both.
#pragma once
#include "tac_kv4_rows.cuh"

namespace tac {

enum Kv4TcFault : int { KV4_TIMEOUT_TILE = 21, KV4_TIMEOUT_S = 22, KV4_TIMEOUT_P = 23, KV4_TIMEOUT_DRAIN = 24 };

constexpr int kTcKeys = 128;
constexpr int kTcRows = 256;
constexpr int kTcThreads = 24 * 32;
// Registers a thread: 80 at launch, then shared out by warpgroup (two of rows, four others: 2 * 144 + 4 * 48 = 6 * 80).
constexpr int kTcRegsRows = 144, kTcRegsRest = 48;

__host__ __device__ constexpr int tc_tile_bytes(int D) { return kTcKeys * D * 2; }
// Q of two groups, two K tiles, two V tiles
__host__ __device__ constexpr int tc_smem(int D) { return 6 * tc_tile_bytes(D) + 1024; }

// kind::f16, FP16 operands, float32 accumulation; b_mn: B is MN-major (one row a K step).
__host__ __device__ constexpr uint32_t tc_idesc(uint32_t N, bool b_mn) {
  return (1u << 4) | (uint32_t(b_mn) << 16) | ((N >> 3) << 17) | ((128u >> 4) << 24);
}

__device__ __forceinline__ void mma_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  const uint32_t no_mask = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(no_mask));
}

// A out of TMEM: two 16-bit values of a row in each column.
__device__ __forceinline__ void mma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  const uint32_t no_mask = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(no_mask));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};\n" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// 32 columns of this thread's lane; the registers may be used after tmem_landed.
__device__ __forceinline__ void tmem_ld32_start(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Names the registers, so that no use of them moves ahead of the wait.
__device__ __forceinline__ void tmem_landed(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
  asm volatile(""
               : "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}

template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(N)); }

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

struct Kv4TcParams {
  Kv4RowsParams r;
  int blocks;            // row blocks of all sequences at most: the grid is blocks * heads
  int* fault;
};

// Place in a [128 rows][64 values] block of 16-bit values with 128-byte swizzle: 16-byte chunk c of row r.
__device__ __forceinline__ uint32_t sw128(uint32_t r, uint32_t c) {
  return (r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4);
}

// Codes of a key to shared memory as c - z in FP16, chunks from `first` on.  A chunk of eight values is stored in the
// order 0 4 1 5 2 6 3 7.
template <int W>
__device__ __forceinline__ void tc_unpack(uint8_t* dst, uint32_t key, int first, const uint4 (&words)[W / 4], uint32_t z) {
  const __half2 zlo = u_h2(0x64006400u + z * 0x10001u), zhi = u_h2(0x54005400u + z * 0x100010u);   // 1024 + z, 64 + z
#pragma unroll
  for (int q = 0; q < W / 4; ++q) {
    const uint32_t x4[4] = {words[q].x, words[q].y, words[q].z, words[q].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int w = first + 4 * q + j;
      const uint32_t x = x4[j], y = x >> 8;
      *reinterpret_cast<uint4*>(dst + (w >> 3) * (kTcKeys * 128) + sw128(key, w & 7)) =
          make_uint4(h2_u(__hsub2(u_h2(and_or(x, 0x000f000fu, 0x64006400u)), zlo)), h2_u(__hsub2(u_h2(and_or(x, 0x00f000f0u, 0x54005400u)), zhi)),
                     h2_u(__hsub2(u_h2(and_or(y, 0x000f000fu, 0x64006400u)), zlo)), h2_u(__hsub2(u_h2(and_or(y, 0x00f000f0u, 0x54005400u)), zhi)));
    }
  }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kTcThreads, 1) kv4_tc_kernel(Kv4TcParams pp) {
  const Kv4RowsParams& p = pp.r;
  constexpr int W = D / 8;                       // words of codes a key
  constexpr int kTile = tc_tile_bytes(D);
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t q_full, k_full[2], k_empty[2], ks_full[4], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], pv_done[2], o_full;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  // scales and presence of a tile's keys, and the largest exponent of the values' scales (a NaN aside) for each 32 of
  // them; a slot is written again when both groups are past the tile after it
  __shared__ __align__(16) float ks_s[4][kTcKeys], vs_s[4][kTcKeys];
  __shared__ uint32_t present_s[4][4], vexp_s[4][4];
  __shared__ float rf_s[kTcRows];

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // ---- this CTA's rows: later row blocks, which see more keys, come first (sequences by length instead of by number
  // made no difference) ----
  const int h = blockIdx.x % p.c.heads;
  int blk = pp.blocks - 1 - int(blockIdx.x / p.c.heads), b = 0;
  const int64_t cap = int64_t(p.s.width) * p.c.page_size;
  for (int b0 = 0;; b0 += 32) {                  // every warp for itself: the sequence that holds block blk
    if (b0 >= p.s.batch) return;                 // a block of no sequence
    const int mine = b0 + lane < p.s.batch ? (kv4_seq(p.s, b0 + lane, cap).n * p.group + kTcRows - 1) / kTcRows : 0;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    const int all = __shfl_sync(0xffffffffu, inc, 31);
    if (blk < all) {
      const int who = __ffs(__ballot_sync(0xffffffffu, blk < inc)) - 1;
      b = b0 + who;
      blk -= __shfl_sync(0xffffffffu, inc - mine, who);
      break;
    }
    blk -= all;
  }
  const Kv4Seq s = kv4_seq(p.s, b, cap);
  const int rows_all = s.n * p.group, r0 = blk * kTcRows;
  const int r_last = min(rows_all, r0 + kTcRows) - 1;
  const int groups = rows_all - r0 > 128 ? 2 : 1;
  const int key_end = max(0, p.causal ? min(s.len, s.p0 + p.div.of(r_last) + 1) : s.len);
  const int tiles = (key_end + kTcKeys - 1) / kTcKeys;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  uint8_t *const q_sm = smem, *const k_sm = smem + 2 * kTile, *const v_sm = smem + 4 * kTile;
  if (threadIdx.x == 0) {
    sm100::mbar_init(&q_full, 4 * groups);   // a warp each of those that write
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&k_full[i], 4);
      sm100::mbar_init(&v_full[i], 8);
      for (int j = 0; j < 2; ++j) {
        sm100::mbar_init(&p_full[i][j], 4);
        sm100::mbar_init(&s_full[i][j], 1);
      }
      sm100::mbar_init(&pv_done[i], 1);
      sm100::mbar_init(&k_empty[i], 1);
      sm100::mbar_init(&v_empty[i], 1);
    }
    sm100::mbar_init(&o_full, 1);
    for (int i = 0; i < 4; ++i) sm100::mbar_init(&ks_full[i], 4);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  if (warp == 8) sm100::tmem_alloc(&tmem_base, 512);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;
  // After a wait that ran out nothing waits any more (and no MMA is issued): the CTA runs to its end.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (sm100::mbar_try_wait(bar, parity)) return;
    if (!*abort_v && !sm100::mbar_wait(bar, parity, pp.fault, code)) *abort_v = 1;
  };

  const int32_t* table = p.s.table + int64_t(b) * p.s.width;
  // row of the cache that holds key `key` of tile i, kNone where none does
  constexpr uint32_t kNone = 0xffffffffu;        // no row: there are fewer than 2^32
  auto row_of = [&](int i, int key) -> uint32_t {
    const int pos = i * kTcKeys + key;
    if (i >= tiles || pos >= s.len) return kNone;
    const int pg = __ldg(table + (pos >> p.c.page_shift));
    if (uint32_t(pg) >= uint32_t(p.c.num_pages)) return kNone;
    return (uint32_t(pg) * p.c.heads + h) * p.c.page_size + (pos & (p.c.page_size - 1));
  };
  if (warp >= 12 && warp < 16) {
    // ---- MMA issue: the whole warp runs these loops and one elected lane issues, so that descriptors stay in uniform
    // registers ----
    regs_down<kTcRegsRest>();
    if (warp == 12 && tiles) {
      constexpr uint32_t kIdS = tc_idesc(64, false), kIdO = tc_idesc(D, true);
      // K-major rows of 128 bytes (64 values), blocks of 64 values 16 KB apart
      const uint64_t qd = sm100::smem_desc_sw128(sm100::smem_u32(q_sm), 16, 1024), kd = sm100::smem_desc_sw128(sm100::smem_u32(k_sm), 16, 1024);
      // MN-major: a key's 64 values a row of 128 bytes, 8 keys 1024 bytes, blocks of 64 values 16 KB apart
      const uint64_t vd = sm100::smem_desc_sw128(sm100::smem_u32(v_sm), kTcKeys * 128, 1024);
      const int steps = 2 * tiles;
      // the warp's own waits have one verdict: elect.sync needs every lane
      bool go = true;
      auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) {
        go = go && sm100::mbar_wait_warp(bar, parity, abort_v, pp.fault, code);
      };
      auto qk = [&](int j, int g) {              // S of step j: 64 keys are 8 KB of each block
        const uint64_t qg = qd + g * (kTile >> 4), ki = kd + ((j >> 1) & 1) * (kTile >> 4) + (j & 1) * (8192 >> 4);
        if (go && sm100::elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t o = ((k >> 2) * (kTcKeys * 128) + (k & 3) * 32) >> 4;
            mma_f16_ss(tmem + g * 128 + (j & 1) * 64, qg + o, ki + o, kIdS, k != 0);
          }
          sm100::mma_commit(&s_full[g][j & 1]);
          if ((j & 1) && g == groups - 1) sm100::mma_commit(&k_empty[(j >> 1) & 1]);
        }
        __syncwarp();
      };
      wait_all(&q_full, 0, KV4_TIMEOUT_TILE);
      wait_all(&k_full[0], 0, KV4_TIMEOUT_TILE);
      sm100::tc_fence_after();
      for (int j = 0; j < 2; ++j)
        for (int g = 0; g < groups; ++g) qk(j, g);
      for (int j = 0; j < steps; ++j) {
        if (!(j & 1)) {
          const int i = j >> 1;
          wait_all(&v_full[i & 1], (i >> 1) & 1, KV4_TIMEOUT_TILE);
          if (i + 1 < tiles) wait_all(&k_full[(i + 1) & 1], ((i + 1) >> 1) & 1, KV4_TIMEOUT_TILE);
        }
        const uint64_t vi = vd + ((j >> 1) & 1) * (kTile >> 4) + (j & 1) * (4 * 2048 >> 4);
        for (int g = 0; g < groups; ++g) {
          wait_all(&p_full[g][j & 1], (j >> 1) & 1, KV4_TIMEOUT_P);
          sm100::tc_fence_after();
          if (go && sm100::elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_f16_ts(tmem + 256 + g * 128, tmem + g * 128 + (j & 1) * 64 + k * 8, vi + k * (2048 >> 4), kIdO, j || k);
            sm100::mma_commit(&pv_done[g]);
            if ((j & 1) && g == groups - 1) sm100::mma_commit(&v_empty[(j >> 1) & 1]);
          }
          __syncwarp();
          if (j + 2 < steps) qk(j + 2, g);
        }
      }
      if (sm100::elect_one()) sm100::mma_commit(&o_full);
      __syncwarp();
      // every MMA has ended before TMEM is freed, also after a failed wait
      sm100::mbar_wait(&o_full, 0, pp.fault, KV4_TIMEOUT_DRAIN);
    }
  } else if (warp >= 16) {
    // ---- values: c - z; thread = half of a key's ----
    regs_down<kTcRegsRest>();
    constexpr int H = W / 2;
    const int key = threadIdx.x & 127, half = (threadIdx.x >> 7) & 1;
    uint4 cw[H / 4];
    uint32_t vp = 0;
    auto load = [&](uint32_t row) {
      if (row == kNone) return;
      const uint4* src = reinterpret_cast<const uint4*>(p.c.vc + uint64_t(row) * (D / 2) + half * (D / 4));
#pragma unroll
      for (int w = 0; w < H / 4; ++w) cw[w] = __ldg(src + w);
      vp = __ldg(p.c.vp + row);
    };
    uint32_t row = row_of(0, key), row1 = row_of(1, key);
    load(row);
    for (int i = 0; i < tiles; ++i) {
      uint8_t* const dst = v_sm + (i & 1) * kTile;
      wait(&v_empty[i & 1], ((i >> 1) & 1) ^ 1, KV4_TIMEOUT_TILE);
      if (row == kNone) {
#pragma unroll
        for (int w = half * H; w < half * H + H; ++w)
          *reinterpret_cast<uint4*>(dst + (w >> 3) * (kTcKeys * 128) + sw128(key, w & 7)) = make_uint4(0, 0, 0, 0);
      } else {
        tc_unpack<H>(dst, key, half * H, cw, vp & 15u);
      }
      sm100::fence_proxy_async();
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(&v_full[i & 1]);
      load(row1);                                // after the fence, which would wait for it
      row = row1;
      row1 = row_of(i + 2, key);
    }
  } else if (warp >= 8) {
    // ---- keys: c - z; thread = key of the tile ----
    regs_down<kTcRegsRest>();
    const int key = threadIdx.x & 127;
    uint4 cw[W / 4];
    uint32_t kp = 0, vp = 0;
    auto load = [&](uint32_t row) {
      if (row == kNone) return;
      const uint4* src = reinterpret_cast<const uint4*>(p.c.kc + uint64_t(row) * (D / 2));
#pragma unroll
      for (int w = 0; w < W / 4; ++w) cw[w] = __ldg(src + w);
      kp = __ldg(p.c.kp + row);
      vp = __ldg(p.c.vp + row);
    };
    uint32_t row = row_of(0, key), row1 = row_of(1, key);
    load(row);
    for (int i = 0; i < tiles; ++i) {
      wait(&k_empty[i & 1], ((i >> 1) & 1) ^ 1, KV4_TIMEOUT_TILE);
      const bool here = row != kNone;
      const int slot = i & 3;
      ks_s[slot][key] = here ? kv4_scale(kp) : 0.f;
      vs_s[slot][key] = here ? kv4_scale(vp) : 0.f;
      const uint32_t there = __ballot_sync(0xffffffffu, here), ve = here ? (vp >> 23) & 0xffu : 0u;
      const uint32_t top = __reduce_max_sync(0xffffffffu, ve == 255u ? 0u : ve);
      if (lane == 0) present_s[slot][warp - 8] = there, vexp_s[slot][warp - 8] = top;
      tc_unpack<W>(k_sm + (i & 1) * kTile, key, 0, cw, kp & 15u);
      sm100::fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        sm100::mbar_arrive(&k_full[i & 1]);
        sm100::mbar_arrive(&ks_full[i & 3]);
      }
      load(row1);
      row = row1;
      row1 = row_of(i + 2, key);
    }
  } else {
    // ---- rows ----
    regs_up<kTcRegsRows>();
    const int g = warp >> 2, row = threadIdx.x & 127;
    const int rr = r0 + g * 128 + row;
    const bool ok = rr < rows_all;
    if (g < groups) {
      uint8_t* const q_mine = q_sm + g * kTile;
      // ---- Q: D / 8 lanes a row; each row scaled by the power of two that brings its largest magnitude into [1, 2),
      // with the softmax scale's sign ----
      {
        constexpr int L = D / 8, R = 32 / L;     // lanes a row, rows at a time
        const int c = lane % L;
        uint4 qw[32 / R];
#pragma unroll
        for (int j = 0; j < 32 / R; ++j) {
          const int r = r0 + warp * 32 + j * R + lane / L;
          qw[j] = make_uint4(0, 0, 0, 0);
          if (r < rows_all) {
            const uint16_t* src = p.q + (s.q0 + p.div.of(r)) * p.q_tok + (h * p.group + p.div.rest(r)) * p.q_head + c * 8;
            if (p.q_vec) {
              qw[j] = __ldg(reinterpret_cast<const uint4*>(src));
            } else {
              uint32_t e[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) e[k] = uint32_t(__ldg(src + 2 * k)) | uint32_t(__ldg(src + 2 * k + 1)) << 16;
              qw[j] = make_uint4(e[0], e[1], e[2], e[3]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 32 / R; ++j) {
          const uint32_t ww[4] = {qw[j].x, qw[j].y, qw[j].z, qw[j].w};
          float v[8];
          uint32_t mx = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint16_t e = uint16_t(ww[k / 2] >> (16 * (k & 1)));
            v[k] = BF16 ? __uint_as_float(uint32_t(e) << 16) : __half2float(__ushort_as_half(e));
            mx = max(mx, __float_as_uint(v[k]) & 0x7fffffffu);
          }
#pragma unroll
          for (int o = 1; o < L; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
          int e = int(mx >> 23);                 // infinities and NaN stay what they are
          e = e == 255 ? 127 : e < 1 ? 1 : e > 253 ? 253 : e;
          const float down = copysignf(__uint_as_float(uint32_t(254 - e) << 23), p.scale_log2);
          const int q_row = (warp & 3) * 32 + j * R + lane / L;
          if (c == 0) rf_s[g * 128 + q_row] = __uint_as_float(uint32_t(e) << 23) * fabsf(p.scale_log2);
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = h2_u(__floats2half2_rn(v[k] * down, v[k + 4] * down));
          *reinterpret_cast<uint4*>(q_mine + (c >> 3) * (kTcKeys * 128) + sw128(q_row, c & 7)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      sm100::fence_proxy_async();
      __syncwarp();                              // rf_s: a warp reads what it wrote
      if (lane == 0) sm100::mbar_arrive(&q_full);
      const float rf = rf_s[g * 128 + row];
      // keys below it are seen; a row past the last one is a row of zeros that nothing stores, and needs no mask
      const int lim = ok && p.causal ? min(s.len, s.p0 + p.div.of(rr) + 1) : s.len;
      const uint32_t lanes = uint32_t((warp & 3) * 32) << 16, t_s = tmem + lanes + g * 128, t_o = tmem + lanes + 256 + g * 128;
      // Weights are exp2(s - mu) times the value's scale, l their sum without it, all in units of 2^(127 - ve): ve follows
      // the exponent of the largest scale among the keys that the row has seen, so that the products fit FP16 whatever
      // the values' magnitude.  mu and ve move only when a score or a scale passes them by kSlack or kSlackV.
      float mu = 0.f, l = 0.f;
      int ve = 127;
      bool begun = false;

      int vtop = 0;                              // largest exponent of the values' scales in the tile
      auto step = [&](int j, auto masked_c) {
        constexpr bool kMasked = decltype(masked_c)::value;
        const int slot = (j >> 1) & 3, key0 = j * 64;
        const uint32_t t_sj = t_s + (j & 1) * 64;
        const ulonglong2* ks = reinterpret_cast<const ulonglong2*>(ks_s[slot] + (j & 1) * 64);
        uint32_t v[64];
        tmem_ld32_start(t_sj, v);
        tmem_ld32_start(t_sj + 32, v + 32);
        tmem_landed(v);
        tmem_landed(v + 32);
        // scores, but for the row's factor
        uint64_t y[32];
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const ulonglong2 k4 = ks[q];
          y[2 * q] = mul2(pack2(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1])), k4.x);
          y[2 * q + 1] = mul2(pack2(__uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3])), k4.y);
          float f[4];
          unpack2(y[2 * q], f[0], f[1]);
          unpack2(y[2 * q + 1], f[2], f[3]);
          if (kMasked) {
            const uint32_t present = present_s[slot][(j & 1) * 2 + q / 8];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (!(key0 + 4 * q + e < lim && (present >> (4 * (q % 8) + e) & 1))) f[e] = -INFINITY;
            y[2 * q] = pack2(f[0], f[1]);
            y[2 * q + 1] = pack2(f[2], f[3]);
          }
          top4[(2 * q) & 3] = max3(top4[(2 * q) & 3], f[0], f[1]);
          top4[(2 * q + 1) & 3] = max3(top4[(2 * q + 1) & 3], f[2], f[3]);
        }
        const float mx = fmaxf(max3(top4[0], top4[1], top4[2]), top4[3]);
        const float top = mx == -INFINITY ? -INFINITY : mx * rf;
        const bool up = begun ? top > mu + kSlack || vtop >= ve + int(kSlackV) : mx != -INFINITY;
        if (__any_sync(0xffffffffu, up)) {
          float corr = 1.f;
          if (mx != -INFINITY) {
            int v_new = vtop;
            if (kMasked) {                       // of the keys that this row sees
              v_new = 0;
              for (int k = 0; k < 64; ++k) {
                const int e = (__float_as_uint(vs_s[slot][(j & 1) * 64 + k]) >> 23) & 0xff;
                if (key0 + k < lim && (present_s[slot][(j & 1) * 2 + k / 32] >> (k & 31) & 1) && e != 255) v_new = max(v_new, e);
              }
            }
            v_new = min(max(v_new, 27), 227);
            if (begun) v_new = max(v_new, ve);
            const float to = begun ? fmaxf(mu, top) : top;
            if (begun) corr = exp2_((mu - to) + float(ve - v_new));
            mu = to;
            ve = v_new;
            begun = true;
          }
          l *= corr;
          if (j) {
            wait(&pv_done[g], (j - 1) & 1, KV4_TIMEOUT_S);   // P V of the step before; the next one waits for this step's P
            __syncwarp();
            sm100::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t u[16];
              tmem_ld16(t_o + c * 16, u);
#pragma unroll
              for (int k = 0; k < 16; ++k) u[k] = __float_as_uint(__uint_as_float(u[k]) * corr);
              tmem_st16(t_o + c * 16, u);
            }
          }
        }
        const float shift = -(mu + float(ve - 127));
        const uint64_t rf2 = pack2(rf, rf), mu2 = pack2(shift, shift);
        const ulonglong2* vs = reinterpret_cast<const ulonglong2*>(vs_s[slot] + (j & 1) * 64);
        uint64_t sum2[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
          float x[32];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            unpack2(fma2(y[16 * c + k], rf2, mu2), x[2 * k], x[2 * k + 1]);
            if (kMasked) {                       // a row of factor 0 must not turn -inf into a NaN
              float ya, ye;
              unpack2(y[16 * c + k], ya, ye);
              x[2 * k] = ya == -INFINITY ? -INFINITY : x[2 * k];
              x[2 * k + 1] = ye == -INFINITY ? -INFINITY : x[2 * k + 1];
            }
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) x[k] = exp2_(x[k]);
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const ulonglong2 v4 = vs[8 * c + k / 2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const uint64_t e2 = pack2(x[2 * (k + q)], x[2 * (k + q) + 1]);
              sum2[q] = add2(sum2[q], e2);
              float a, e;
              unpack2(mul2(e2, q ? v4.y : v4.x), a, e);
              if (kMasked) {                     // a hidden key may hold a NaN scale
                a = x[2 * (k + q)] == 0.f ? 0.f : a;
                e = x[2 * (k + q) + 1] == 0.f ? 0.f : e;
              }
              w[k + q] = h2_u(__floats2half2_rn(a, e));
            }
          }
          tmem_st16(t_sj + c * 16, w);           // over S columns that have been read
        }
        float a, e;
        unpack2(add2(sum2[0], sum2[1]), a, e);
        l += a + e;
        tmem_wait_st();
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) sm100::mbar_arrive(&p_full[g][j & 1]);
      };
      for (int i = 0; i < tiles; ++i) {
        // ks_s, present_s: their slot is not filled again before this group is past the tile, so its barrier cannot
        // run a phase ahead
        wait(&ks_full[i & 3], (i >> 2) & 1, KV4_TIMEOUT_TILE);
        const uint32_t all = present_s[i & 3][0] & present_s[i & 3][1] & present_s[i & 3][2] & present_s[i & 3][3];
        const bool masked = __any_sync(0xffffffffu, (i + 1) * kTcKeys > lim || all != 0xffffffffu);
        vtop = max(max(vexp_s[i & 3][0], vexp_s[i & 3][1]), max(vexp_s[i & 3][2], vexp_s[i & 3][3]));
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {
          wait(&s_full[g][hh], i & 1, KV4_TIMEOUT_S);
          __syncwarp();
          sm100::tc_fence_after();
          if (masked) step(2 * i + hh, std::true_type{});
          else step(2 * i + hh, std::false_type{});
        }
      }
      // ---- the rows' results, through the group's Q buffer so that a row leaves in one run ----
      if (tiles) wait(&o_full, 0, KV4_TIMEOUT_S);
      __syncwarp();
      sm100::tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (tiles) sm100::tmem_ld32(t_o + c * 32, v);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {          // values 2j, 2j + 1 of the chunk, out of the order 0 4 1 5 2 6 3 7
            const int a = (2 * j) % 4 * 2 + (2 * j) / 4, e2 = (2 * j + 1) % 4 * 2 + (2 * j + 1) / 4;
            const float x = l == 0.f ? 0.f : __uint_as_float(v[8 * q + a]) * inv, z = l == 0.f ? 0.f : __uint_as_float(v[8 * q + e2]) * inv;
            w[j] = BF16 ? uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(x))) | uint32_t(__bfloat16_as_ushort(__float2bfloat16_rn(z))) << 16
                        : h2_u(__floats2half2_rn(x, z));
          }
          const int ch = c * 4 + q;
          *reinterpret_cast<uint4*>(q_mine + (ch >> 3) * (kTcKeys * 128) + sw128(row, ch & 7)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      if (ok && p.lse)
        p.lse[int64_t(s.q0 + p.div.of(rr)) * p.hq + h * p.group + p.div.rest(rr)] =
            l == 0.f ? -INFINITY : (mu + float(ve - 127) + log2f(l)) * 0.69314718055994531f;
      __syncwarp();                              // a warp stores its own rows
      {
        constexpr int L = D / 8, R = 32 / L;
        const int ch = lane % L;
#pragma unroll 4
        for (int j = 0; j < 32 / R; ++j) {
          const int q_row = (warp & 3) * 32 + j * R + lane / L, r = r0 + g * 128 + q_row;
          if (r >= rows_all) continue;
          const uint4 w = *reinterpret_cast<const uint4*>(q_mine + (ch >> 3) * (kTcKeys * 128) + sw128(q_row, ch & 7));
          uint16_t* dst = p.o + (int64_t(s.q0 + p.div.of(r)) * p.hq + h * p.group + p.div.rest(r)) * D + ch * 8;
          if (p.o_vec) {
            *reinterpret_cast<uint4*>(dst) = w;
          } else {
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) dst[k] = uint16_t(ww[k / 2] >> (16 * (k & 1)));
          }
        }
      }
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 512);
  }
}

}  // namespace tac
