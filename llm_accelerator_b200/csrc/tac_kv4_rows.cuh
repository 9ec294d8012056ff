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
#include "tac_kv4.cuh"

namespace tac {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32;
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
  float* part;           // [2 * grid][rows * (D + 2)]
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

// Zero point as the two FP16 constants of kv4_pair: 1024 + z and -(64 + z), for the codes of one half each.
struct ZeroPair {
  __half2 lo, hi;
};
__device__ __forceinline__ ZeroPair zero_pair(uint32_t z0, uint32_t z1) {
  // FP16 integers 1024 + z have the bits 0x6400 + z; -(64 + z) follows exactly
  ZeroPair r;
  r.lo = u_h2(0x64006400u + z0 + (z1 << 16));
  r.hi = __hsub2(__float2half2_rn(960.f), r.lo);
  return r;
}

// Codes 0 and 4 (N = 0), 1 and 5, 2 and 6, 3 and 7 of a word as FP16 c - z:
// a code in the low bits of 0x6400 is 1024 + c, four bits up 1024 + 16 c.
template <int N>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t x, const ZeroPair& z) {
  const uint32_t y = N >= 2 ? x >> 8 : x;
  if (N & 1) return h2_u(__hfma2(u_h2((y & 0x00f000f0u) | 0x64006400u), __float2half2_rn(0.0625f), z.hi));
  return h2_u(__hsub2(u_h2((y & 0x000f000fu) | 0x64006400u), z.lo));
}

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

template <int D, int NT>
__global__ void __launch_bounds__(kRowsThreads, NT == 1 ? 3 : 2) kv4_rows_kernel(Kv4RowsParams p) {
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

    // ---- query rows: FP16, each scaled by the power of two that brings its largest magnitude into [1, 2) ----
    uint32_t qf[NT][2 * W][2];
    float qs[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 8 + g;
      const bool ok = r < rows_all;
      const int64_t qi = ok ? (s.q0 + r / p.group) * p.q_tok + (h * p.group + r % p.group) * p.q_head + (D / 4) * t : 0;
      float v[D / 4];
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < D / 4; ++i) {
        v[i] = ok ? ld_q(p, qi + i) : 0.f;
        mx = max(mx, __float_as_uint(v[i]) & 0x7fffffffu);
      }
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      int e = int(mx >> 23);                        // biased exponent; infinities and NaN stay what they are
      e = e == 255 ? 127 : e < 1 ? 1 : e > 253 ? 253 : e;
      const float down = __uint_as_float(uint32_t(254 - e) << 23);
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            qf[n][2 * w + hf][j] = h2_u(__floats2half2_rn(v[8 * w + 2 * hf + j] * down, v[8 * w + 2 * hf + j + 4] * down));
      const float up = __uint_as_float(uint32_t(e) << 23) * p.scale_log2;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        qs[n][j] = __shfl_sync(0xffffffffu, up, (2 * t + j) * 4);
        const int rr = r0 + n * 8 + 2 * t + j;
        lim[n][j] = rr >= rows_all ? 0 : p.causal ? min(s.len, s.p0 + rr / p.group + 1) : s.len;   // keys below it are seen
      }
    }
    int lim_min = s.len;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) lim_min = min(lim_min, r0 + n * 8 + 2 * t + j < rows_all ? lim[n][j] : lim_min);
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);   // every row sees the keys below

    float o[NT][D / 16][4] = {};
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
    // A row's O is held in units of 2^(ve - 127), ve the exponent of the largest s' among the keys that it has seen
    // (a NaN aside), so that its weights p s' fit FP16 whatever the values' magnitude, and whatever it does not see.
    uint32_t ve[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) ve[n][0] = ve[n][1] = 1;

    for (int tile = t0; tile < t1; ++tile) {
      const int key0 = tile * kRowsTile + warp * 32;
      if (key0 >= s.len) break;
      // ---- loads ----
      uint32_t kw[2][2][W], kpw[2][2], vw[2][4][VW], vpw[2][2], vz[2][4];
      bool have[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int k0 = key0 + 16 * u;
        int page = -1;
        if (k0 < s.len) page = __ldg(p.s.table + int64_t(b) * p.s.width + (k0 >> p.c.page_shift));
        have[u] = page >= 0 && page < p.c.num_pages;
        if (have[u]) {
          const int64_t row = (int64_t(page) * p.c.heads + h) * p.c.page_size + (k0 & (p.c.page_size - 1));
          const uint8_t* kr = p.c.kc + row * (D / 2);
          const uint8_t* vr = p.c.vc + row * (D / 2);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t* src = reinterpret_cast<const uint32_t*>(kr + (g + 8 * j) * (D / 2) + t * (D / 8));
            if constexpr (W == 4) {
              const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
              kw[u][j][0] = v.x, kw[u][j][1] = v.y, kw[u][j][2] = v.z, kw[u][j][3] = v.w;
            } else {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
              kw[u][j][0] = v.x, kw[u][j][1] = v.y;
            }
            kpw[u][j] = __ldg(p.c.kp + row + g + 8 * j);
            vpw[u][j] = __ldg(p.c.vp + row + g + 8 * j);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = 2 * t + (j & 1) + 8 * (j >> 1);
            const uint32_t* src = reinterpret_cast<const uint32_t*>(vr + key * (D / 2) + g * (D / 16));
            if constexpr (VW == 2) {
              const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
              vw[u][j][0] = v.x, vw[u][j][1] = v.y;
            } else {
              vw[u][j][0] = __ldg(src);
            }
            vz[u][j] = __ldg(p.c.vp + row + key) & 0xffffu;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            kpw[u][j] = vpw[u][j] = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) kw[u][j][w] = 0;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            vz[u][j] = 0;
#pragma unroll
            for (int w = 0; w < VW; ++w) vw[u][j][w] = 0;
          }
        }
      }
      // ---- S^T ----
      float sc[2][NT][4] = {};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t za = kpw[u][0] & 0xffffu, zb = kpw[u][1] & 0xffffu;
        const ZeroPair z0 = zero_pair(za, za), z1 = zero_pair(zb, zb);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const uint32_t a = kw[u][0][w], c = kw[u][1][w];
          const uint32_t p00 = kv4_pair<0>(a, z0), p01 = kv4_pair<0>(c, z1), p10 = kv4_pair<1>(a, z0), p11 = kv4_pair<1>(c, z1);
          const uint32_t p20 = kv4_pair<2>(a, z0), p21 = kv4_pair<2>(c, z1), p30 = kv4_pair<3>(a, z0), p31 = kv4_pair<3>(c, z1);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(sc[u][n], p00, p01, p10, p11, qf[n][2 * w][0], qf[n][2 * w][1]);
            mma_16816(sc[u][n], p20, p21, p30, p31, qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
          }
        }
      }
      // ---- softmax over the keys of this warp ----
      const bool masked = key0 + 32 > lim_min || !have[0] || !have[1];
      uint32_t vm[2][2], vm_all = 0;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float ks = kv4_scale(kpw[u][j]);
          const int key = key0 + 16 * u + 8 * j + g;
          vm[u][j] = (vpw[u][j] >> 23) & 0xffu;
          if (vm[u][j] == 255u) vm[u][j] = 0;
          vm_all = max(vm_all, vm[u][j]);
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float v = sc[u][n][2 * j + i] * (ks * qs[n][i]);
              if (masked && (key >= lim[n][i] || !have[u])) v = -INFINITY;
              sc[u][n][2 * j + i] = v;
            }
        }
      vm_all = __reduce_max_sync(0xffffffffu, vm_all);
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float corr[2], mu[2], down[2];
        bool moved = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t vx = vm_all;
          if (masked) {
            vx = 0;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (key0 + 16 * u + 8 * j + g < lim[n][i] && have[u]) vx = max(vx, vm[u][j]);
            vx = max(vx, __shfl_xor_sync(0xffffffffu, vx, 4));
            vx = max(vx, __shfl_xor_sync(0xffffffffu, vx, 8));
            vx = max(vx, __shfl_xor_sync(0xffffffffu, vx, 16));
          }
          vx = max(ve[n][i], min(vx, 253u));
          down[i] = __uint_as_float((254u - vx) << 23);
          float mx = fmaxf(fmaxf(sc[0][n][i], sc[0][n][2 + i]), fmaxf(sc[1][n][i], sc[1][n][2 + i]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = fmaxf(mx, m[n][i]);
          mu[i] = mx == -INFINITY ? 0.f : mx;
          corr[i] = exp2_(m[n][i] - mu[i]);
          moved |= mx != m[n][i] || vx != ve[n][i];
          m[n][i] = mx;
          l[n][i] *= corr[i];
          corr[i] *= __uint_as_float((127u - min(vx - ve[n][i], 126u)) << 23);   // 2^(ve - vx)
          ve[n][i] = vx;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][d][i] *= corr[i & 1];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float vs = kv4_scale(vpw[u][j]);
            float w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float e = exp2_(sc[u][n][2 * j + i] - mu[i]);
              l[n][i] += e;
              w[i] = e * (vs * down[i]);
              // a key that this row does not see may hold a NaN scale
              if (masked && (key0 + 16 * u + 8 * j + g >= lim[n][i] || !have[u])) w[i] = 0.f;
            }
            pb[u][n][j] = movmatrix(h2_u(__floats2half2_rn(w[0], w[1])));
          }
      }
      // ---- O^T ----
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const ZeroPair z0 = zero_pair(vz[u][0], vz[u][1]), z1 = zero_pair(vz[u][2], vz[u][3]);
#pragma unroll
        for (int w = 0; w < VW; ++w) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7632 : 0x5410;
            const uint32_t a = __byte_perm(vw[u][0][w], vw[u][1][w], sel), c = __byte_perm(vw[u][2][w], vw[u][3][w], sel);
            const uint32_t p00 = kv4_pair<0>(a, z0), p01 = kv4_pair<0>(c, z1), p10 = kv4_pair<1>(a, z0), p11 = kv4_pair<1>(c, z1);
            const uint32_t p20 = kv4_pair<2>(a, z0), p21 = kv4_pair<2>(c, z1), p30 = kv4_pair<3>(a, z0), p31 = kv4_pair<3>(c, z1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16816(o[n][4 * w + 2 * half], p00, p10, p01, p11, pb[u][n][0], pb[u][n][1]);
              mma_16816(o[n][4 * w + 2 * half + 1], p20, p30, p21, p31, pb[u][n][0], pb[u][n][1]);
            }
          }
        }
      }
    }

    // ---- the warps' pieces of the unit, then the unit's result or this CTA's piece of it ----
    __syncthreads();                               // the last unit's reads of sm_* are done
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = l[n][i];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) {
          sm_m[warp][n * 8 + 2 * t + i] = m[n][i];
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
                o[n][4 * w + j][i] * __uint_as_float(ve[n][i & 1] << 23);
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

// Joins the pieces of the units that several CTAs covered.  CTA j - 1 of this
// grid looks at the cut before CTA j of the other: it joins the unit there if
// that cut is the first inside it.
template <int D, int NT>
__global__ void __launch_bounds__(kRowsThreads) kv4_join_kernel(Kv4RowsParams p, int grid) {
  using Cfg = RowsCfg<D, NT>;
  constexpr int R = Cfg::kRows;
  __shared__ int64_t red[kRowsWarps];
  __shared__ __align__(8) int found[4];
  const Shares sh = make_shares(p, R, grid, red);
  const int j = blockIdx.x + 1;
  if (j >= sh.parts) return;
  const int64_t x = sh.at(j);
  int b;
  int64_t first;
  find_seq(p, R, x, red, found, b, first);
  if (b >= p.s.batch) return;
  const Kv4Seq s = kv4_seq(p.s, b, int64_t(p.s.width) * p.c.page_size);
  int tiles;
  int64_t units;
  seq_cost(s, p.group, p.c.heads, R, tiles, units);
  const int64_t unit = (x - first) / tiles, u0 = first + unit * tiles, u1 = u0 + tiles;
  if (u0 == x || u0 < sh.at(j - 1)) return;        // no unit is cut here, or an earlier cut's CTA joins it
  const int h = int(unit % p.c.heads), r0 = int(unit / p.c.heads) * R, rows_all = s.n * p.group;
  int last = j;                                    // the pieces are those of CTAs j - 1 .. last
  while (last + 1 < sh.parts && sh.at(last + 1) < u1) ++last;
  const float* p0 = p.part + (2 * int64_t(j - 1) + (u0 == sh.at(j - 1) ? 0 : 1)) * Cfg::kPart;
  for (int i = threadIdx.x; i < R * D; i += kRowsThreads) {
    const int r = i / D, d = i % D, rr = r0 + r;
    if (rr >= rows_all) break;
    float mx = p0[R * D + r];
    for (int c = j; c <= last; ++c) mx = fmaxf(mx, p.part[2 * int64_t(c) * Cfg::kPart + R * D + r]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float e = exp2_(p0[R * D + r] - mu);
    float sum = p0[R * D + R + r] * e, acc = p0[i] * e;
    for (int c = j; c <= last; ++c) {
      const float* pc = p.part + 2 * int64_t(c) * Cfg::kPart;
      e = exp2_(pc[R * D + r] - mu);
      sum += pc[R * D + R + r] * e;
      acc += pc[i] * e;
    }
    const int64_t oi = int64_t(s.q0 + rr / p.group) * p.hq + h * p.group + rr % p.group;
    st_o(p, oi * D + d, sum == 0.f ? 0.f : acc / sum);
    if (p.lse && d == 0) p.lse[oi] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * 0.69314718055994531f;
  }
}

}  // namespace tac
