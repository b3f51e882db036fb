// What the paged-cache kernels share: exact division by a runtime constant and the page of a position.
#pragma once
#include "common.h"

typedef _Float16 f16;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 in one multiply: with L = ceil(log2 d) and
// m = floor(2^32 (2^L - d) / d) + 1, n / d = (mulhi(n, m) + n) >> L (the sum stays below 2^32).
struct FDiv {
  uint32_t d, m, s;
};
static inline FDiv make_fdiv(uint32_t d) {
  uint32_t L = 0;
  while ((1ull << L) < d) ++L;
  FDiv f;
  f.d = d;
  f.m = (uint32_t)((((1ull << 32) * ((1ull << L) - d)) / d) + 1);
  f.s = L;
  return f;
}
__device__ __forceinline__ int fdiv(int n, const FDiv& f) {
  return (int)((__umulhi((uint32_t)n, f.m) + (uint32_t)n) >> f.s);
}

// One sequence of a ragged batch as the device sees it: q_start, kv_len and start come from the caller's tensors
// and are clamped to what the buffers hold, so that no value of theirs reaches an address unchecked.
struct Seq {
  int q0, n;   // first row, rows
  int kv, st;  // keys (positions 0 .. kv - 1), first visible key
};
__device__ __forceinline__ Seq load_seq(const int* qs, const int* kl, const int* st, int s, int rows, int most) {
  Seq r;
  const int a = qs[s], b = qs[s + 1];
  r.q0 = min(max(a, 0), rows);
  r.n = min(max(b, r.q0), rows) - r.q0;
  r.kv = min(max(kl[s], 0), most);
  r.st = st ? min(max(st[s], 0), most) : 0;
  return r;
}

// dtype codes of the C ABI
enum { DT_BF16 = 0, DT_F16 = 1, DT_F32 = 2 };
