// Attention of many query rows (prompt chunks) over a 4-bit paged cache, on
// tcgen05.  See tac_kv4.cuh for the cache.
//
// A CTA takes 256 query rows of one key-value head (token-major, the group's
// query heads of a token side by side, so one unpacking of a key serves them
// all) and walks the keys up to its last row's position in tiles of 128:
//   warps 0..3, 4..7  two row groups of 128, a thread a row: Q to shared
//                     memory, softmax of S out of TMEM, P into TMEM, O out
//   warps 8..11       unpack the tile's keys and values, a thread a key,
//                     into the swizzled layouts that the MMAs read
//   warp 12           issues the MMAs: S = Q C^T (FP16), O += P V
// While one group does its softmax the tensor core works for the other: per
// tile and group D = 128 needs 1024 tensor clocks, and 1024 clocks of the
// exponential unit.
//
// S comes from whole numbers (codes less zero point, exact in FP16) and the
// FP16 query scaled by a power of two for each row; the keys' scales multiply
// it in float32.  V is rounded once to the query's type, P as well.
// TMEM: S of both groups (128 columns each; P takes the first half of its S),
// then O of both.
#pragma once
#include "tac_kv4_rows.cuh"

namespace tac {

enum Kv4TcFault : int { KV4_TIMEOUT_TILE = 21, KV4_TIMEOUT_S = 22, KV4_TIMEOUT_P = 23, KV4_TIMEOUT_DRAIN = 24 };

constexpr int kTcKeys = 128;
constexpr int kTcRows = 256;
constexpr int kTcThreads = 13 * 32;

__host__ __device__ constexpr int tc_tile_bytes(int D) { return kTcKeys * D * 2; }
// Q of two groups, two K tiles, two V tiles
__host__ __device__ constexpr int tc_smem(int D) { return 6 * tc_tile_bytes(D) + 1024; }

// kind::f16 with float32 accumulation; b_mn: B is MN-major (one row a K step).
__host__ __device__ constexpr uint32_t tc_idesc(uint32_t N, bool bf16, bool b_mn) {
  return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(b_mn) << 16) | ((N >> 3) << 17) |
         ((128u >> 4) << 24);
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

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};\n" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
      "r"(taddr)
      : "memory");
}

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

// Codes of a key to shared memory as c - z (FP16), or s (c - z) rounded once: to BF16, to FP16 by an FP16 product (the
// eight bits of a scale down to 2^-17 are exact in FP16), to FP16 by a float32 product (any scale).  A chunk of eight
// values is stored in the order 0 4 1 5 2 6 3 7.
enum TcUnpack { UNPACK_CODES, UNPACK_BF16, UNPACK_F16, UNPACK_F32 };

template <int MODE>
__device__ __forceinline__ uint32_t tc_finish(__half2 v, float s) {
  if (MODE == UNPACK_BF16) {
    const __nv_bfloat162 r = __hmul2(__floats2bfloat162_rn(__low2float(v), __high2float(v)), __float2bfloat162_rn(s));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  if (MODE == UNPACK_F16) return h2_u(__hmul2(v, __float2half2_rn(s)));
  if (MODE == UNPACK_F32) return h2_u(__floats2half2_rn(__low2float(v) * s, __high2float(v) * s));
  return h2_u(v);
}

template <int W, int MODE>
__device__ __forceinline__ void tc_unpack(uint8_t* dst, uint32_t key, const uint4 (&words)[W / 4], uint32_t z, float s) {
  const __half2 zlo = u_h2(0x64006400u + z * 0x10001u), zhi = u_h2(0x54005400u + z * 0x100010u);   // 1024 + z, 64 + z
#pragma unroll
  for (int q = 0; q < W / 4; ++q) {
    const uint32_t x4[4] = {words[q].x, words[q].y, words[q].z, words[q].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int w = 4 * q + j;
      const uint32_t x = x4[j], y = x >> 8;
      uint4 o;
      o.x = tc_finish<MODE>(__hsub2(u_h2(and_or(x, 0x000f000fu, 0x64006400u)), zlo), s);
      o.y = tc_finish<MODE>(__hsub2(u_h2(and_or(x, 0x00f000f0u, 0x54005400u)), zhi), s);
      o.z = tc_finish<MODE>(__hsub2(u_h2(and_or(y, 0x000f000fu, 0x64006400u)), zlo), s);
      o.w = tc_finish<MODE>(__hsub2(u_h2(and_or(y, 0x00f000f0u, 0x54005400u)), zhi), s);
      *reinterpret_cast<uint4*>(dst + (w >> 3) * (kTcKeys * 128) + sw128(key, w & 7)) = o;
    }
  }
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kTcThreads, 1) kv4_tc_kernel(Kv4TcParams pp) {
  const Kv4RowsParams& p = pp.r;
  constexpr int W = D / 8;                       // words of codes a key
  constexpr int kTile = tc_tile_bytes(D);
  extern __shared__ uint8_t dyn_smem[];
  __shared__ __align__(8) uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full;
  __shared__ uint32_t tmem_base;
  __shared__ int abort_flag;
  // scale and presence of a tile's keys; a slot is written again when both groups are past the tile after it
  __shared__ __align__(16) float ks_s[4][kTcKeys];
  __shared__ uint32_t present_s[4][4];

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  // ---- this CTA's rows: later row blocks, which see more keys, come first ----
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
  const int key_end = max(0, p.causal ? min(s.len, s.p0 + r_last / p.group + 1) : s.len);
  const int tiles = (key_end + kTcKeys - 1) / kTcKeys;

  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_smem) + 1023) & ~uintptr_t(1023));
  uint8_t *const q_sm = smem, *const k_sm = smem + 2 * kTile, *const v_sm = smem + 4 * kTile;
  if (threadIdx.x == 0) {
    sm100::mbar_init(&q_full, groups * 128);
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(&k_full[i], 128);
      sm100::mbar_init(&v_full[i], 128);
      sm100::mbar_init(&k_empty[i], 1);
      sm100::mbar_init(&v_empty[i], 1);
      sm100::mbar_init(&s_full[i], 1);
      sm100::mbar_init(&p_full[i], 128);
    }
    sm100::mbar_init(&o_full, 1);
    abort_flag = 0;
    sm100::mbar_fence_init();
  }
  if (warp == 12) sm100::tmem_alloc(&tmem_base, 512);
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = tmem_base;
  volatile int* abort_v = &abort_flag;
  // After a wait that ran out nothing waits any more (and no MMA is issued): the CTA runs to its end.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (!*abort_v && !sm100::mbar_wait(bar, parity, pp.fault, code)) *abort_v = 1;
  };

  if (warp == 12) {
    // ---- MMA issue ----
    // The whole warp runs these loops and one elected lane issues, so that descriptors stay in uniform registers.
    if (tiles) {
      constexpr uint32_t kIdS = tc_idesc(kTcKeys, false, false), kIdO = tc_idesc(D, BF16, true);
      // K-major rows of 128 bytes (64 values), blocks of 64 values 16 KB apart
      const uint64_t qd = sm100::smem_desc_sw128(sm100::smem_u32(q_sm), 16, 1024), kd = sm100::smem_desc_sw128(sm100::smem_u32(k_sm), 16, 1024);
      // MN-major: a key's 64 values a row of 128 bytes, 8 keys 1024 bytes, blocks of 64 values 16 KB apart
      const uint64_t vd = sm100::smem_desc_sw128(sm100::smem_u32(v_sm), kTcKeys * 128, 1024);
      auto qk = [&](int i, int g) {
        const uint64_t qg = qd + g * (kTile >> 4), ki = kd + (i & 1) * (kTile >> 4);
        if (!*abort_v && sm100::elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t o = ((k >> 2) * (kTcKeys * 128) + (k & 3) * 32) >> 4;
            mma_f16_ss(tmem + g * 128, qg + o, ki + o, kIdS, k != 0);
          }
          sm100::mma_commit(&s_full[g]);
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (sm100::elect_one()) sm100::mma_commit(bar);
        __syncwarp();
      };
      wait(&q_full, 0, KV4_TIMEOUT_TILE);
      wait(&k_full[0], 0, KV4_TIMEOUT_TILE);
      sm100::tc_fence_after();
      for (int g = 0; g < groups; ++g) qk(0, g);
      commit(&k_empty[0]);
      for (int i = 0; i < tiles; ++i) {
        wait(&v_full[i & 1], (i >> 1) & 1, KV4_TIMEOUT_TILE);
        if (i + 1 < tiles) wait(&k_full[(i + 1) & 1], ((i + 1) >> 1) & 1, KV4_TIMEOUT_TILE);
        const uint64_t vi = vd + (i & 1) * (kTile >> 4);
        for (int g = 0; g < groups; ++g) {
          wait(&p_full[g], i & 1, KV4_TIMEOUT_P);
          sm100::tc_fence_after();
          if (!*abort_v && sm100::elect_one()) {
#pragma unroll
            for (int k = 0; k < kTcKeys / 16; ++k)
              mma_f16_ts(tmem + 256 + g * 128, tmem + g * 128 + k * 8, vi + k * (2048 >> 4), kIdO, i || k);
          }
          __syncwarp();
          if (i + 1 < tiles) qk(i + 1, g);
        }
        commit(&v_empty[i & 1]);
        if (i + 1 < tiles) commit(&k_empty[(i + 1) & 1]);
      }
      commit(&o_full);                           // every MMA has completed, before TMEM is read for the last time and freed
      sm100::mbar_wait(&o_full, 0, pp.fault, KV4_TIMEOUT_DRAIN);
    }
  } else if (warp >= 8) {
    // ---- unpacking: thread = key of the tile; the next tile's codes are on their way meanwhile ----
    const int key = threadIdx.x - 256;
    const int32_t* table = p.s.table + int64_t(b) * p.s.width;
    uint4 kw[W / 4], vw[W / 4], kn[W / 4], vn[W / 4];
    uint32_t kp = 0, vp = 0, kpn = 0, vpn = 0;
    bool here = false, here_n = false;
    auto load = [&](int i) {
      const int pos = i * kTcKeys + key;
      here_n = false;
      if (i < tiles && pos < s.len) {
        const int pg = __ldg(table + (pos >> p.c.page_shift));
        if (uint32_t(pg) < uint32_t(p.c.num_pages)) {
          here_n = true;
          const uint64_t row = (uint32_t(pg) * p.c.heads + h) * p.c.page_size + (pos & (p.c.page_size - 1));   // fits 32 bits
          const uint4* ks = reinterpret_cast<const uint4*>(p.c.kc + row * (D / 2));
          const uint4* vs = reinterpret_cast<const uint4*>(p.c.vc + row * (D / 2));
#pragma unroll
          for (int w = 0; w < W / 4; ++w) kn[w] = __ldg(ks + w), vn[w] = __ldg(vs + w);
          kpn = __ldg(p.c.kp + row);
          vpn = __ldg(p.c.vp + row);
        }
      }
    };
    load(0);
    for (int i = 0; i < tiles; ++i) {
#pragma unroll
      for (int w = 0; w < W / 4; ++w) kw[w] = kn[w], vw[w] = vn[w];
      kp = kpn, vp = vpn, here = here_n;
      load(i + 1);
      const uint32_t par = ((i >> 1) & 1) ^ 1;
      // K: c - z
      wait(&k_empty[i & 1], par, KV4_TIMEOUT_TILE);
      const float vs = here ? kv4_scale(vp) : 0.f;
      // a row of NaN, of K or of V, reaches the rows that see it through their scores
      const bool v_nan = vs != vs;
      ks_s[i & 3][key] = !here ? 0.f : v_nan ? vs : kv4_scale(kp);
      const uint32_t there = __ballot_sync(0xffffffffu, here);
      if (lane == 0) present_s[i & 3][warp - 8] = there;
      uint8_t* dst = k_sm + (i & 1) * kTile;
      tc_unpack<W, UNPACK_CODES>(dst, key, kw, kp & 15u, 0.f);
      sm100::fence_proxy_async();
      sm100::mbar_arrive(&k_full[i & 1]);
      // V: s (c - z), rounded once
      wait(&v_empty[i & 1], par, KV4_TIMEOUT_TILE);
      dst = v_sm + (i & 1) * kTile;
      if (!here || v_nan) {
#pragma unroll
        for (int w = 0; w < W; ++w)
          *reinterpret_cast<uint4*>(dst + (w >> 3) * (kTcKeys * 128) + sw128(key, w & 7)) = make_uint4(0, 0, 0, 0);
      } else if (BF16) {
        tc_unpack<W, UNPACK_BF16>(dst, key, vw, vp & 15u, vs);
      } else if (vs >= 0x1p-17f && vs < 65504.f) {
        tc_unpack<W, UNPACK_F16>(dst, key, vw, vp & 15u, vs);
      } else {
        tc_unpack<W, UNPACK_F32>(dst, key, vw, vp & 15u, vs);
      }
      sm100::fence_proxy_async();
      sm100::mbar_arrive(&v_full[i & 1]);
    }
  } else {
    // ---- rows ----
    const int g = warp >> 2, row = threadIdx.x & 127;
    const int rr = r0 + g * 128 + row;
    const bool ok = rr < rows_all;
    const int64_t oi = ok ? int64_t(s.q0 + rr / p.group) * p.hq + h * p.group + rr % p.group : 0;
    float rf = 0.f;
    if (g < groups) {
      const int64_t qi = ok ? (s.q0 + rr / p.group) * p.q_tok + (h * p.group + rr % p.group) * p.q_head : 0;
      uint32_t mx = 0;
      auto chunk = [&](int c, float (&v)[8]) {
        if (ok && p.q_vec) {
          const uint4 w = __ldg(reinterpret_cast<const uint4*>(p.q + qi) + c);
          const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint16_t e = uint16_t(ww[j / 2] >> (16 * (j & 1)));
            v[j] = BF16 ? __uint_as_float(uint32_t(e) << 16) : __half2float(__ushort_as_half(e));
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = ok ? ld_q(p, qi + 8 * c + j) : 0.f;
        }
      };
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        float v[8];
        chunk(c, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = max(mx, __float_as_uint(v[j]) & 0x7fffffffu);
      }
      int e = int(mx >> 23);
      e = e == 255 ? 127 : e < 1 ? 1 : e > 253 ? 253 : e;
      // the power of two that brings the row's largest magnitude into [1, 2), with the softmax scale's sign
      const float down = copysignf(__uint_as_float(uint32_t(254 - e) << 23), p.scale_log2);
      rf = __uint_as_float(uint32_t(e) << 23) * fabsf(p.scale_log2);
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        float v[8];
        chunk(c, v);
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = h2_u(__floats2half2_rn(v[j] * down, v[j + 4] * down));
        *reinterpret_cast<uint4*>(q_sm + g * kTile + (c >> 3) * (kTcKeys * 128) + sw128(row, c & 7)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      sm100::fence_proxy_async();
      sm100::mbar_arrive(&q_full);
      const int lim = ok ? (p.causal ? min(s.len, s.p0 + rr / p.group + 1) : s.len) : 0;
      const uint32_t lanes = uint32_t((warp & 3) * 32) << 16, t_s = tmem + lanes + g * 128, t_o = tmem + lanes + 256 + g * 128;
      float mu = 0.f, l = 0.f;
      bool begun = false;

      auto tile = [&](int i, auto masked_c) {
        constexpr bool kMasked = decltype(masked_c)::value;
        const float4* ks = reinterpret_cast<const float4*>(ks_s[i & 3]);
        auto score = [&](const uint32_t (&v)[32], int c, float (&y)[32]) {
          const uint32_t present = kMasked ? present_s[i & 3][c] : 0u;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 k4 = ks[c * 8 + j];
            y[4 * j] = __uint_as_float(v[4 * j]) * k4.x;
            y[4 * j + 1] = __uint_as_float(v[4 * j + 1]) * k4.y;
            y[4 * j + 2] = __uint_as_float(v[4 * j + 2]) * k4.z;
            y[4 * j + 3] = __uint_as_float(v[4 * j + 3]) * k4.w;
          }
          if (kMasked) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (!(i * kTcKeys + c * 32 + j < lim && (present >> j & 1))) y[j] = -INFINITY;
          }
        };
        float mx = -INFINITY;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          float y[32];
          sm100::tmem_ld32(t_s + c * 32, v);
          score(v, c, y);
#pragma unroll
          for (int j = 0; j < 32; ++j) mx = fmaxf(mx, y[j]);
        }
        const float top = mx == -INFINITY ? -INFINITY : mx * rf;
        const bool up = begun ? top > mu + kSlack : mx != -INFINITY;
        if (__any_sync(0xffffffffu, up)) {
          float corr = 1.f;
          if (mx != -INFINITY) {
            const float to = begun ? fmaxf(mu, top) : top;
            if (begun) corr = exp2_(mu - to);
            mu = to;
            begun = true;
          }
          l *= corr;
          if (i) {                               // P V of the tiles before has ended: it was issued before this S
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t v[32];
              sm100::tmem_ld32(t_o + c * 32, v);
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * corr);
              tmem_st32(t_o + c * 32, v);
            }
          }
        }
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32], w[16];
          float y[32];
          sm100::tmem_ld32(t_s + c * 32, v);
          score(v, c, y);
          float sum[4] = {};
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            y[j] = kMasked && y[j] == -INFINITY ? 0.f : exp2_(fmaf(y[j], rf, -mu));
            sum[j & 3] += y[j];
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            if (BF16) {
              const __nv_bfloat162 r = __floats2bfloat162_rn(y[2 * j], y[2 * j + 1]);
              w[j] = *reinterpret_cast<const uint32_t*>(&r);
            } else {
              w[j] = h2_u(__floats2half2_rn(y[2 * j], y[2 * j + 1]));
            }
          }
          tmem_st16(t_s + c * 16, w);            // over S columns that have been read
        }
        tmem_wait_st();
        sm100::tc_fence_before();
        sm100::mbar_arrive(&p_full[g]);
      };
      for (int i = 0; i < tiles; ++i) {
        wait(&k_full[i & 1], (i >> 1) & 1, KV4_TIMEOUT_TILE);   // ks_s, present_s
        wait(&s_full[g], i & 1, KV4_TIMEOUT_S);
        __syncwarp();
        sm100::tc_fence_after();
        const uint32_t all = present_s[i & 3][0] & present_s[i & 3][1] & present_s[i & 3][2] & present_s[i & 3][3];
        if (__any_sync(0xffffffffu, (i + 1) * kTcKeys > lim || all != 0xffffffffu)) tile(i, std::true_type{});
        else tile(i, std::false_type{});
      }
      // ---- the rows' results ----
      if (tiles) wait(&o_full, 0, KV4_TIMEOUT_S);
      __syncwarp();
      sm100::tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t v[32];
        if (tiles) sm100::tmem_ld32(t_o + c * 32, v);
        if (!ok) continue;
        uint16_t* dst = p.o + oi * D + c * 32;
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
          if (p.o_vec) {
            reinterpret_cast<uint4*>(dst)[q] = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) dst[8 * q + 2 * j] = uint16_t(w[j]), dst[8 * q + 2 * j + 1] = uint16_t(w[j] >> 16);
          }
        }
      }
      if (ok && p.lse) p.lse[oi] = l == 0.f ? -INFINITY : (mu + log2f(l)) * 0.69314718055994531f;
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    __syncwarp();
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 512);
  }
}

}  // namespace tac
