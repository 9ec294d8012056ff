// Paged key / value cache held in 4 bits, and attention over it.
//
// A row x[0..D) (one token, one head) is stored as
//   lo = min(0, min x), hi = max(0, max x), s = bf16((hi - lo) / 15),
//   z = rint(-lo / s), c = clip(rint(x / s) + z, 0, 15),   value s (c - z),
// codes in a byte pairwise (2j low, 2j + 1 high), one parameter word a row:
// the bits of s above those of z.  Codes [page][head][slot][D / 2], words
// [page][head][slot]: the rows that one head needs of a page are contiguous.
//
// The factors s stay out of the matrix instructions:
//   q . k_j = s_j (q . (c_j - z_j)),   sum_j p_j v_j = sum_j (p_j s'_j)(c'_j - z'_j),
// so their operands are whole numbers in [-15, 15], exact in FP16, whatever
// the cache's values are; q (scaled by a power of two for each row, exactly)
// and p s' are the only rounded FP16 operands, and sums run in float32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace tac {

struct Kv4Cache {
  uint8_t *kc, *vc;
  uint32_t *kp, *vp;
  int num_pages, page_size, heads;   // page_size: 16, 32, 64 or 128
  int page_shift;
};

// Which token of which sequence: sequence b has rows [q0, q0 + n) of the new
// tokens, the last n of its len positions.
struct Kv4Seqs {
  const int32_t* table;   // [batch][width] page numbers; one outside [0, num_pages) holds no keys
  const int32_t* lens;    // [batch]
  const int32_t* indptr;  // [batch + 1], or null: one row a sequence
  int batch, width, total;
};

struct Kv4Seq {
  int len, q0, n;
  int p0;     // position of row q0; negative rows have none
};

// Lengths and offsets are clamped to the table's and the rows' extent, so no
// contents of these arrays lead outside the tensors.
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Seqs& s, int b, int64_t cap) {
  Kv4Seq r;
  const int len = __ldg(s.lens + b);
  r.len = len < 0 ? 0 : int64_t(len) > cap ? int(cap) : len;
  if (s.indptr) {
    int a = __ldg(s.indptr + b), e = __ldg(s.indptr + b + 1);
    a = a < 0 ? 0 : a > s.total ? s.total : a;
    e = e < a ? a : e > s.total ? s.total : e;
    r.q0 = a;
    r.n = e - a;
  } else {
    r.q0 = b;
    r.n = b < s.total ? 1 : 0;
  }
  r.p0 = max(len, 0) - r.n;
  return r;
}

__device__ __forceinline__ float kv4_scale(uint32_t word) { return __uint_as_float(word & 0xffff0000u); }

}  // namespace tac
