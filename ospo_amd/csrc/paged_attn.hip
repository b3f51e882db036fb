// Attention of new tokens over a paged key/value cache.
//
//   o[r] = sum_j p_rj v_j / sum_j p_rj,  p_rj = exp(scale q_r . k_j),  start <= j <= position of r
//
// One pass over the keys with the running maximum and sum of the softmax.  The query heads that share a
// key/value head are rows of one tile (row = token * group + head in group), so a key is read once for all of
// them.  S^T = K Q^T puts a query on a lane: its scores are the lane's registers, and those registers are the
// operand of O^T += V^T P^T.
//
// Work is cut into items (sequence, row tile, key/value head, key chunk).  The grid is sized from shapes alone;
// a workgroup finds its item from the lengths on the device, which also choose the chunk size, so that a captured
// call follows the lengths at its replay.  An item whose keys are one chunk writes its rows; others write
// (maximum, sum, O) in fp32 and a second launch joins them in chunk order: no atomics, the same bits each time.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace {

typedef __attribute__((ext_vector_type(16))) float f32x16;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float NONE = -3e38f;  // running maximum before any key: finite, so that exp2(m - m) is 1

struct PagedArgs {
  const void* q;
  const void* kc;
  const void* vc;
  void* o;
  float* lse;
  const int* bt;
  const int* qs;
  const int* kl;
  const int* st;
  long q_ts, q_hs, o_ts, o_hs, l_ts, l_hs;
  long c_ps, c_hs, c_ts;
  int rows, S, Hk, n_pages, max_pages, most;
  FDiv g, ps;      // query heads per key/value head, page size
  float cs;        // scale * log2 e
  int causal;
  int qvec, ovec;  // q rows and o rows allow 16-byte access
  int slots;       // workgroups that run at once: what a split aims for
  int split;       // 0: every item is one chunk
  int bar;         // keys are not cut where no sequence sees more of them than this
  long items, pairs;  // workgroups of the two launches: upper bounds
  int* plan;       // number of (tile, head) pairs, then from PLAN_HEAD on their records for the joining launch
  float* ws;       // partial O [row of a cut item][D]
  float* ml;       // (m, l) [row of a cut item][2]
  int cap;         // rows that both hold
};

// ---------------------------------------------------------------- items
// Wave-wide sums by data-parallel moves: rows of 16 lanes, then across the rows (a lane without a source adds 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp0(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int scan_add(int x) {  // inclusive
  x += dpp0<0x111, 0xf>(x);
  x += dpp0<0x112, 0xf>(x);
  x += dpp0<0x114, 0xf>(x);
  x += dpp0<0x118, 0xf>(x);
  x += dpp0<0x142, 0xa>(x);
  x += dpp0<0x143, 0xc>(x);
  return x;
}
__device__ __forceinline__ int lane_of(int x, int l) { return __builtin_amdgcn_readlane(x, l); }
__device__ __forceinline__ int sum_i(int x) { return lane_of(scan_add(x), 63); }
__device__ __forceinline__ float sum_f(float x) {
#define OSPO_STEP(C, R) x += __int_as_float(dpp0<C, R>(__float_as_int(x)))
  OSPO_STEP(0x111, 0xf);
  OSPO_STEP(0x112, 0xf);
  OSPO_STEP(0x114, 0xf);
  OSPO_STEP(0x118, 0xf);
  OSPO_STEP(0x142, 0xa);
  OSPO_STEP(0x143, 0xc);
#undef OSPO_STEP
  return __int_as_float(lane_of(__float_as_int(x), 63));
}
__device__ __forceinline__ int max_i(int x) {  // of values >= 0
  x = max(x, dpp0<0x111, 0xf>(x));
  x = max(x, dpp0<0x112, 0xf>(x));
  x = max(x, dpp0<0x114, 0xf>(x));
  x = max(x, dpp0<0x118, 0xf>(x));
  x = max(x, dpp0<0x142, 0xa>(x));
  x = max(x, dpp0<0x143, 0xc>(x));
  return lane_of(x, 63);
}

struct LaneSeq {  // the sequence of this lane: its rows in tiles of BM, its keys in units of KU
  Seq q;
  int tiles, units;
};
// units: key blocks of KU that the sequence's longest row sees (every tile of it is cut at the same places)
template <int BM, int KU>
__device__ __forceinline__ LaneSeq lane_seq(const PagedArgs& a, int s) {
  LaneSeq r{{0, 0, 0, 0}, 0, 1};
  if (s < a.S) {
    r.q = load_seq(a.qs, a.kl, a.st, s, a.rows, a.most);
    r.tiles = (r.q.n * (int)a.g.d + BM - 1) / BM;
    r.units = r.q.kv > r.q.st ? (r.q.kv + KU - 1) / KU - r.q.st / KU : 1;
  }
  return r;
}
// Key blocks of a chunk.  With L = all work / slots: where the tiles alone fill the slots, chunks of at most L / 4, but
// four blocks at least, even out the last round (with many tiles, only sequences longer than L are cut).  Where they do not, one round:
// of L, the smallest chunk that might do, and of the smaller of two that do (every tile cut as the longest may be;
// the work over the slots that the tiles leave), the first of four steps from one to the other that fits.
template <int BM, int KU>
__device__ __forceinline__ unsigned even_chunk(const PagedArgs& a, int lane, const LaneSeq& first) {
  float total = 0.f;
  int base = 0, most = 1, longest = 0;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const LaneSeq q = s0 ? lane_seq<BM, KU>(a, s0 + lane) : first;
    total += sum_f((float)q.tiles * (float)q.units);
    base += sum_i(q.tiles);
    most = max(most, max_i(q.tiles ? q.units : 0));
    longest = max(longest, max_i(q.tiles ? max(q.q.kv - q.q.st, 0) : 0));
  }
  if (longest <= a.bar) return 0x7fffffff;
  base = max(1, base * a.Hk);
  total *= (float)a.Hk;
  const float L = total / (float)a.slots;
  if (base > a.slots) return (unsigned)fmaxf(4.f, fminf((float)most, ceilf(base >= 4 * a.slots ? L : 0.25f * L)));
  const float lo = fmaxf(1.f, ceilf(L));
  const unsigned times = (unsigned)a.slots / (unsigned)base;
  float hi = (float)(((unsigned)most + times - 1) / times);
  if (a.slots > base) hi = fminf(hi, ceilf(1.00001f * total / (float)(a.slots - base)) + 1.f);
  hi = fmaxf(lo, hi) + (most > 1 << 22 ? 4.f : 0.f);  // (sums and counts of that size are rounded)
  for (int i = 0; i < 4; ++i) {
    const unsigned C = (unsigned)(lo + (hi - lo) * 0.25f * (float)i);
    int n = 0;
    for (int s0 = 0; s0 < a.S; s0 += 64) {
      const LaneSeq q = s0 ? lane_seq<BM, KU>(a, s0 + lane) : first;
      n += sum_i(q.tiles * (int)(((unsigned)q.units - 1) / C + 1));
    }
    if (n * a.Hk <= a.slots) return C;
    if (hi - lo < 1.f) break;
  }
  return (unsigned)hi;
}
__device__ __forceinline__ int chunks_of(const LaneSeq& q, unsigned C) { return (int)(((unsigned)q.units - 1) / C) + 1; }
// That chunk, larger where the partial results of the sequences that it cuts would not fit the workspace.  (One that cuts
// nothing needs none.)
template <int BM, int KU>
__device__ __forceinline__ unsigned pick_chunk(const PagedArgs& a, int lane, const LaneSeq& first) {
  if (!a.split) return 0x7fffffff;
  unsigned C = even_chunk<BM, KU>(a, lane, first);
  for (;;) {
    float need = 0.f;  // (the sum is exact up to 2^24, more than the workspace holds)
    for (int s0 = 0; s0 < a.S; s0 += 64) {
      const LaneSeq q = s0 ? lane_seq<BM, KU>(a, s0 + lane) : first;
      const int nch = chunks_of(q, C);
      need += sum_f(nch > 1 ? (float)q.q.n * (float)a.g.d * (float)nch : 0.f);
    }
    need *= (float)a.Hk;
    if (need <= (float)a.cap) return C;
    C = (unsigned)fminf(ceilf((float)C * fmaxf(need / (float)a.cap, 1.125f)), 2e9f);
  }
}

struct Item {
  Seq q;
  int seq, tile, head, chunk, nch, cs, u0, units;
  int slot;  // partial results: of the tile's first row
  int pair;  // number of the (tile, head)
};
// Order of a sequence's items: heads fastest over the XCDs (hb = largest power of two <= 8 that divides Hk, so a
// key/value head stays in its XCDs' L2), then chunks, then tiles from the last (the longest rows first), then the
// remaining heads.  Item 0's workgroup also notes how many (tile, head) pairs there are.
template <int BM, int KU>
__device__ __forceinline__ bool find_item(const PagedArgs& a, int id, int lane, Item& it) {
  const LaneSeq lead = lane_seq<BM, KU>(a, lane);
  const unsigned C = pick_chunk<BM, KU>(a, lane, lead);
  int before = 0, pairs = 0, slots = 0;
  bool got = false;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const LaneSeq q = s0 ? lane_seq<BM, KU>(a, s0 + lane) : lead;
    const int nch = chunks_of(q, C);
    const int own = q.tiles * a.Hk, mine = own * nch;
    const int cut = nch > 1 ? q.q.n * (int)a.g.d * nch * a.Hk : 0;
    const int upto = scan_add(mine), pupto = scan_add(own), cupto = scan_add(cut);
    const unsigned long long b = __ballot(id - before < upto);
    if (b && !got) {
      const int w = __ffsll(b) - 1;
      it.seq = s0 + w;
      it.q.q0 = lane_of(q.q.q0, w), it.q.n = lane_of(q.q.n, w);
      it.q.kv = lane_of(q.q.kv, w), it.q.st = lane_of(q.q.st, w);
      it.units = lane_of(q.units, w), it.nch = lane_of(nch, w);
      const unsigned tiles = (unsigned)lane_of(q.tiles, w);
      const unsigned at = (unsigned)(id - before - lane_of(upto - mine, w));
      const int hb = min(8, a.Hk & -a.Hk), sh = __ffs(hb) - 1;
      const unsigned z = at >> sh, per = tiles * it.nch;
      const unsigned hh = z / per, x = z - hh * per, tx = x / it.nch;
      it.head = (int)((hh << sh) + (at & (hb - 1)));
      it.tile = (int)(tiles - 1 - tx);
      it.chunk = (int)(x - tx * it.nch);
      it.cs = (int)(((unsigned)it.units + it.nch - 1) / it.nch);
      it.u0 = it.q.st / KU;
      it.slot = slots + lane_of(cupto - cut, w) + (it.head * it.nch + it.chunk) * it.q.n * (int)a.g.d + it.tile * BM;
      it.pair = pairs + lane_of(pupto - own, w) + (int)(((hh * tiles + tx) << sh) + (at & (hb - 1)));
      got = true;
      if (id > 0) return true;
    }
    before += lane_of(upto, 63);
    pairs += lane_of(pupto, 63);
    slots += lane_of(cupto, 63);
  }
  // (more than the launches' bounds only where q_start descends: nothing is joined then)
  if (id == 0 && a.split && threadIdx.x == 0) a.plan[0] = before <= a.items && pairs <= a.pairs ? pairs : 0;
  return got;
}
// one past the last key that any row of the tile sees
__device__ __forceinline__ int tile_end(const PagedArgs& a, const Item& it, int BM) {
  if (!a.causal) return it.q.kv;
  const int last = min((it.tile + 1) * BM, it.q.n * (int)a.g.d) - 1;
  return max(0, it.q.kv - it.q.n + fdiv(last, a.g) + 1);
}

// What the joining launch needs to know of a (tile, head): how many chunks to join (0: none), where the first row's partial
// results lie, and how far on those of the next chunk.
struct Record {
  int chunks, first, step, q0, head, row0, rows;
};
constexpr int PLAN_HEAD = 8, RECORD = 8;  // ints
template <int BM, int KU>
__device__ __forceinline__ void note(const PagedArgs& a, const Item& it, int end) {
  if (!a.split || it.chunk > 0 || threadIdx.x) return;
  const int left = min(end, (it.u0 + it.units) * KU) - it.u0 * KU;
  const int n = left > 0 ? ((left + KU - 1) / KU + it.cs - 1) / it.cs : 1;  // chunks that have keys (one writes if none has)
  Record r{it.nch > 1 ? n : 0, it.slot, it.q.n * (int)a.g.d, it.q.q0, it.head, it.tile * BM,
           min(BM, it.q.n * (int)a.g.d - it.tile * BM)};
  if (it.pair < a.pairs) *reinterpret_cast<Record*>(a.plan + PLAN_HEAD + (long)it.pair * RECORD) = r;
}

// ---------------------------------------------------------------- types
// mma: a product as the compiler sees it.  acc: one into accumulators that stay in the matrix unit's own registers (the
// compiler moves some of O to vector registers and back around its products).  It knows nothing of the waits that
// such a product needs: two states behind the vector unit's last write to an operand, which the block brings along,
// and the kernel's settle before anything but another product reads the accumulators.
//
// A probability is held as exp2(x - m) in the cache's type, m = the row's largest x less FEW or MANY (few and many rows).
// bf16 has fp32's exponents and needs no such offset.  fp16's last normal number is 2^-14 and its largest is 65504:
// from 2^15 at the largest score down, probabilities keep their 11 bits to 2^-29 of the row's largest and end at 2^-40
// (many rows, which leave a maximum as it is until it grew by 2^7: 2^-22 and 2^-33).  Without an offset they end at 2^-25,
// and a key that takes a row to itself with a value near zero would leave out what all others add up to.
template <typename T>
struct Frag;
template <>
struct Frag<bf16> {
  typedef bf16x8 v8;
  static constexpr unsigned EXP = 0x7f80, MAN = 0x007f;
  static constexpr float GROW = 24.f, FEW = 0.f, MANY = 0.f;
  __device__ static void acc(f32x16& c, const bf16x8& x, const bf16x8& y) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(x), "v"(y));
  }
  __device__ static void clear(f32x16& c, const bf16x8& zero) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %1, 0" : "=a"(c) : "v"(zero));
  }
  __device__ static f32x16 mma(const v8& x, const v8& y, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  }
};
template <>
struct Frag<f16> {
  typedef f16x8 v8;
  static constexpr unsigned EXP = 0x7c00, MAN = 0x03ff;
  static constexpr float GROW = 15.f, FEW = 15.f, MANY = 8.f;
  __device__ static void acc(f32x16& c, const f16x8& x, const f16x8& y) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(x), "v"(y));
  }
  __device__ static void clear(f32x16& c, const f16x8& zero) {
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %1, 0" : "=a"(c) : "v"(zero));
  }
  __device__ static f32x16 mma(const v8& x, const v8& y, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
  }
};

// 8 values with zeros for those that are not finite
template <typename T>
__device__ __forceinline__ i16x8 finite(i16x8 v) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (((unsigned short)v[i] & Frag<T>::EXP) == Frag<T>::EXP) v[i] = 0;
  return v;
}

// 16 bytes a lane from global memory to LDS (wave-uniform destination + 16 lane), without registers
__device__ __forceinline__ void dma16(const void* src, char* dst) {
  __builtin_amdgcn_global_load_lds(src, (LDS_AS void*)dst, 16, 0, 0);
}
// The same from a uniform base by a 32-bit byte offset a lane and a uniform one more.  (While pieces of the form above are
// in flight the compiler lets every LDS read wait for all that went before it.)
__device__ __forceinline__ void dma16_from(const void* base, char* dst, int voff, int soff) {
  const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, 0x7fffffff, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (LDS_AS void*)dst, 16, voff, soff, 0, 0);
}
// transposed read: a group of 16 lanes reads 4 rows x 16 columns, lane i gets column i
__device__ __forceinline__ i16x4 read_tr(const char* src) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS i16x4*)src);
}

// all loads and LDS-DMA but the last N done (a wait that the compiler sees: what it believes to be in flight, it waits
// for again, and then for all of it)
template <int N = 0>
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x0f70);  // vmcnt(N)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);  // (products on what was loaded stay behind it)
}
// barrier of the workgroup behind this wave's LDS accesses (loads and LDS-DMA from memory stay in flight)
__device__ __forceinline__ void sync_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ float other_half(float x) {  // the value of lane ^ 32
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// N finished values of a row from column d0 on: divided by the sum (a row that saw no key: zeros), rounded once
template <typename T, int N>
__device__ __forceinline__ void store_row(const PagedArgs& a, int tok, int hd, int d0, const float* x, float M, float L) {
  const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
  T* p = (T*)a.o + (long)tok * a.o_ts + (long)hd * a.o_hs + d0;
  struct alignas(2 * N) { T v[N]; } y;
#pragma unroll
  for (int i = 0; i < N; ++i) y.v[i] = (T)(L == 0.f ? 0.f : x[i] * inv);
  if (a.ovec) {
    *reinterpret_cast<decltype(y)*>(p) = y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = y.v[i];
  }
  if (a.lse && d0 == 0)
    a.lse[(long)tok * a.l_ts + (long)hd * a.l_hs] = L == 0.f ? -INFINITY : (M + __log2f(L)) * LN2;
}

constexpr int pitch_of(int D) { return D + 4; }  // floats of a staged output row

// ---------------------------------------------------------------- many rows
// Chunks and prompts: the matrix unit bounds it.  Four waves of 32 RB rows share tiles of 64 keys; a wave's 64 rows
// (RB = 2) feed two products from each fragment that it reads, so that LDS is read at half its rate (32 rows would
// need all of it).  One wave a SIMD, so its own instruction stream has to keep the matrix unit fed, in steps of 32
// keys: while scores of tile j become probabilities (vector unit), those of tile j + 1 are formed (matrix unit);
// while O takes tile j, sums of tile j and maxima of tile j + 1 are taken.  (64 keys at a time need more vector
// registers than there are.)  K(j + 2) and V(j + 1) come by LDS-DMA with the whole tile's time to arrive: one barrier
// a tile.
// The running maximum is raised (and O scaled) only when a score would reach more than 2^GROW (24 in bf16, 15 in fp16),
// which both types hold; sums stay in fp32.  (O is scaled where it is: put aside in memory and added up at the end, fp16's
// chunks of up to 257 tokens over up to 5000 keys, a few of whose rows grow by 2^7, took 42 us instead of 21.)
//
// Measured: whole prompts of 3.5k to 4k tokens, 32 heads over 8 of 128, at 945 TFLOP/s (500 us for four).  A tile of 64
// keys takes 3600 cycles, 2048 of them products; the matrix unit is busy for 54 % of all cycles.  32 instructions less a
// tile (of 580) change nothing, no exponentials at all would gain 7 %, fragments read 2 or 4 slots ahead the same time.
// The start of an item (lengths, page numbers, first keys: three round trips to memory, one behind the other) and its end
// take 7 us.
//
// LDS images: blocks of 16 keys x 32 columns, 1 KiB each, [16-byte chunk q of the columns][key, for V key ^ 4 q]: every
// fragment is one address and a constant, and the reads of K (16 keys of a chunk) and the transposed reads of V (4
// keys x 4 chunks by half a wave) meet every bank once.
template <typename T, int D, int RB, bool P16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1, 1))) void paged_many_kernel(const PagedArgs a) {
  using F = Frag<T>;
  using v8 = typename F::v8;
  constexpr int NW = 4, BM = 32 * RB * NW, KU = 64;
  constexpr int ROWB = D * 2, TILE = KU * ROWB;
  constexpr int KS = D / 16, DC = D / 32;
  constexpr int NL = D / 32;    // column blocks: LDS-DMA pieces of a wave's 16 keys
  // objects of their own, so that the compiler sees that a read of one does not wait for what is on its way to another
  __shared__ __attribute__((aligned(1024))) char K0[TILE], K1[TILE], V0[TILE], V1[TILE];
  __shared__ int inf[NW][RB * DC][64];  // where a sum is +infinity (bit r) and -infinity (bit 16 + r), see mend
  __shared__ int found;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hi = lane >> 5, l32 = lane & 31;

  Item it;
  if (!find_item<BM, KU>(a, blockIdx.x, lane, it)) return;
  const int R = it.q.n * (int)a.g.d;
  const int ub = it.u0 + it.chunk * it.cs;
  const int kb = ub * KU;
  const int end = tile_end(a, it, BM);
  const int ke = min(min(ub + it.cs, it.u0 + it.units) * KU, end);
  const bool part = it.nch > 1;
  note<BM, KU>(a, it, end);
  if (part && it.chunk > 0 && kb >= ke) return;
  const int R0 = it.tile * BM, row0 = R0 + wave * 32 * RB;

  // rows of this lane: row0 + 32 b + l32 (rows behind the last repeat it and are not stored)
  v8 qf[RB][KS];
  int lim[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int tok = fdiv(min(row0 + 32 * b + l32, R - 1), a.g);
    lim[b] = a.causal ? it.q.kv - it.q.n + tok : it.q.kv - 1;
  }
  auto load_q = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const int r = min(row0 + 32 * b + l32, R - 1);
      const int tok = fdiv(r, a.g), hd = it.head * (int)a.g.d + r - tok * (int)a.g.d;
      const T* p = (const T*)a.q + (long)(it.q.q0 + tok) * a.q_ts + (long)hd * a.q_hs + 8 * hi;
      if (a.qvec) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[b][ks] = *reinterpret_cast<const v8*>(p + 16 * ks);
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int i = 0; i < 8; ++i) qf[b][ks][i] = p[16 * ks + i];
      }
    }
  };
  // smallest limit of the wave's rows: tiles that end at or before it need no mask
  const int low = a.causal ? it.q.kv - it.q.n + fdiv(min(row0, R - 1), a.g) : it.q.kv - 1;

  f32x16 o[RB][DC], s[2][2][RB];  // scores: [tile parity][half]
  float m[RB], l[RB], mx[2][RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    m[b] = NONE, l[b] = 0.f, mx[0][b] = mx[1][b] = -INFINITY;
  }
  auto settle = [&]() __attribute__((always_inline)) {  // (a product takes 16 passes at most: 18 states)
    asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int c = 0; c < DC; ++c) asm volatile("" : "+a"(o[b][c]));
  };
  auto clear_o = [&]() __attribute__((always_inline)) {
    v8 zero;
#pragma unroll
    for (int i = 0; i < 8; ++i) zero[i] = (T)0.f;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int c = 0; c < DC; ++c) F::clear(o[b][c], zero);
  };
  clear_o();
  const int n = ke > kb ? (ke - kb + KU - 1) / KU : 0;  // tiles

  // ---- memory to LDS: this wave's 16 keys of a tile
  const T* kc = (const T*)a.kc + (long)it.head * a.c_hs;
  const T* vc = (const T*)a.vc + (long)it.head * a.c_hs;
  const int* bt = a.bt + (long)it.seq * a.max_pages;
  const int lastp = ke > 0 ? fdiv(ke - 1, a.ps) : 0;
  const int wrow = 16 * wave, q4 = lane >> 4;
  const int lkey[2] = {lane & 15, (lane & 15) ^ (q4 << 2)};  // key of this lane in a piece of K, of V
  struct At {  // element offsets: of the wave's first key (uniform; 16 keys lie in one page), or of this lane's two keys
    long u;
    long v[2];
  };
  int pbase = 0, pn = 0, pg[2];
  long pv = 0;  // offset of this lane's page
  auto clampp = [&](int p) __attribute__((always_inline)) { return min(max(p, 0), a.n_pages - 1); };
  auto lookup = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) pg[i] = bt[fdiv(min(k0 + wrow + lkey[i], ke - 1), a.ps)];
  };
  auto place = [&](int t, At& at) __attribute__((always_inline)) {
    const int k0 = kb + t * KU;
    if constexpr (P16) {
      const int pi = fdiv(k0 + wrow, a.ps), pc = min(pi, lastp);
      if (pc - pbase >= 64) {  // 64 page numbers sit on the lanes, the next 64 are on their way
        pbase += 64;
        pv = clampp(pn) * a.c_ps;
        pn = bt[min(pbase + 64 + lane, lastp)];
      }
      const unsigned lo = lane_of((int)pv, pc - pbase), up = lane_of((int)(pv >> 32), pc - pbase);
      at.u = (long)((unsigned long)up << 32 | lo) + (long)(k0 + wrow - pi * (int)a.ps.d) * (int)a.c_ts;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = min(k0 + wrow + lkey[i], ke - 1);
        at.v[i] = (long)clampp(pg[i]) * a.c_ps + (long)(key - fdiv(key, a.ps) * (int)a.ps.d) * a.c_ts + 8 * q4;
      }
      lookup(k0 + KU);
    }
  };
  const int loff[2] = {lkey[0] * (int)a.c_ts + 8 * q4, lkey[1] * (int)a.c_ts + 8 * q4};
  auto piece = [&](const T* base, const At& at, int i, char* buf, int p) __attribute__((always_inline)) {
    if constexpr (P16)
      dma16_from(base + at.u, buf + (4 * p + wave) * 1024, 2 * loff[i], 64 * p);
    else
      dma16(base + at.v[i] + 32 * p, buf + (4 * p + wave) * 1024);
  };
  auto fetch = [&](const T* base, const At& at, int i, char* buf) __attribute__((always_inline)) {
#pragma unroll
    for (int p = 0; p < NL; ++p) piece(base, at, i, buf, p);
  };

  // ---- fragments: read PF slots of RB products ahead of their use
  constexpr int PF = 3;
  const int kat = (l32 >> 4) * 1024 + hi * 256 + (l32 & 15) * 16;
  auto kfrag = [&](const char* kl, int h, int ks) __attribute__((always_inline)) {
    return *reinterpret_cast<const v8*>(kl + kat + (ks >> 1) * 4096 + (ks & 1) * 512 + h * 2048);
  };
  const int vq = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vr = 4 * hi + ((lane & 15) >> 2);
  const int vat0 = vq * 256 + (vr ^ (vq << 2)) * 16 + (lane & 1) * 8;
  const int vat1 = vq * 256 + ((vr + 8) ^ (vq << 2)) * 16 + (lane & 1) * 8;
  auto vfrag = [&](const char* vl, int c, int u) __attribute__((always_inline)) {
    const i16x4 x = read_tr(vl + vat0 + (4 * c + u) * 1024), y = read_tr(vl + vat1 + (4 * c + u) * 1024);
    return i16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };

  // ---- the parts of a step (t: tile, h: its 32-key half)
  auto scores = [&](const char* kl, int h, f32x16 (&x)[RB]) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const v8 kf = kfrag(kl, h, ks);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        if (ks == 0) {
          f32x16 z;
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] = 0.f;
          x[b] = F::mma(kf, qf[b][ks], z);
        } else {
          x[b] = F::mma(kf, qf[b][ks], x[b]);
        }
      }
    }
  };
  auto hidden = [&](int b, int key) __attribute__((always_inline)) { return key > lim[b] || key < it.q.st; };
  auto apply_mask = [&](int t, int h, f32x16 (&x)[RB]) __attribute__((always_inline)) {
    const int k0 = kb + t * KU + 32 * h;
    if (k0 >= it.q.st && k0 + 31 <= low) return;
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        x[b][r] = hidden(b, k0 + (r & 3) + 8 * (r >> 2) + 4 * hi) ? -INFINITY : x[b][r];
  };
  auto maxima = [&](int h, const f32x16 (&x)[RB]) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      float y = x[b][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) y = fmaxf(y, x[b][r]);
      mx[h][b] = y;
    }
  };
  // tiles that some row of the workgroup sees in part; whether one holds values that are not finite
  const int low0 = a.causal ? it.q.kv - it.q.n + fdiv(R0, a.g) : it.q.kv - 1;
  const int clear0 = it.q.st > kb ? (it.q.st - kb + KU - 1) / KU : 0, clear1 = low0 >= kb ? (low0 + 1 - kb) / KU : 0;
  auto edge = [&](int t) __attribute__((always_inline)) { return t < clear0 || t >= clear1; };
  auto look = [&](int t, const char* vl) __attribute__((always_inline)) {
    if (threadIdx.x == 0) found = 0;
    sync_lds();
    const int key = kb + t * KU + wrow + lkey[1];
    bool odd = false;
#pragma unroll
    for (int p = 0; p < NL; ++p) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(vl + (4 * p + wave) * 1024 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) odd = odd || (x[e] & F::EXP) == F::EXP || (x[e] >> 16 & F::EXP) == F::EXP;
    }
    if (odd) atomicOr(&found, key < ke && key >= it.q.st ? 3 : 1);  // 2: at a key that some row may see
    sync_lds();
    return found;
  };
  // A masked key has p = 0, but 0 times an infinity or NaN in its value would reach the row all the same.  Where a tile
  // that some row sees in part holds such values, they become zeros in LDS.  Where rows see them (rare, and slow:
  // key by key), which of their sums get +infinity or -infinity (NaN: both) is kept until the end.
  bool anyinf = false;
  auto mend = [&](int j, char* vl, bool seen) __attribute__((always_inline)) {
    if (seen) {
      if (!anyinf)
        for (int i = 0; i < RB * DC; ++i) inf[wave][i][lane] = 0;
      anyinf = true;
#pragma nounroll
      for (int key = 0; key < KU; ++key)
#pragma unroll
        for (int b = 0; b < RB; ++b)
          if (!hidden(b, kb + j * KU + key)) {
#pragma nounroll
            for (int r = 0; r < DC * 16; ++r) {  // column of O's register r
              const int d = 32 * (r >> 4) + (r & 3) + 8 * (r >> 2 & 3) + 4 * hi, q = d >> 3 & 3, k16 = key & 15;
              const unsigned v = *reinterpret_cast<const unsigned short*>(vl + (4 * (d >> 5) + (key >> 4)) * 1024 + q * 256 +
                                                                          (k16 ^ (q << 2)) * 16 + (d & 7) * 2);
              if ((v & F::EXP) == F::EXP) {
                const int up = (v & F::MAN) || !(v & 0x8000), dn = (v & F::MAN) || (v & 0x8000);
                inf[wave][(r >> 4) * RB + b][lane] |= (up | dn << 16) << (r & 15);
              }
            }
          }
      sync_lds();
    }
#pragma nounroll
    for (int p = 0; p < NL; ++p) {
      i16x8* x = reinterpret_cast<i16x8*>(vl + (4 * p + wave) * 1024 + lane * 16);
      *x = finite<T>(*x);
    }
    sync_lds();
  };
  // The maxima raised, O and the sums scaled to them: in the matrix unit's registers, one value at a time (rare; the vector
  // registers have no room for O).
  auto raise = [&]() __attribute__((always_inline)) {
    settle();
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const float most = fmaxf(mx[0][b], mx[1][b]);  // of this lane's keys
      const float mn = fmaxf(m[b], fmaf(fmaxf(most, other_half(most)), a.cs, -F::MANY));
      const float alpha = __builtin_amdgcn_exp2f(m[b] - mn);
      m[b] = mn;
      l[b] *= alpha;
#pragma unroll
      for (int c = 0; c < DC; ++c)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float x = o[b][c][r], t;
          asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1"
                       : "+a"(x), "=&v"(t)
                       : "v"(alpha));
          o[b][c][r] = x;
        }
    }
  };

  At ak{}, av{};  // of K(j + 1) / V(j + 1) at the start of step j
  if (n > 0) {
    if constexpr (P16) {
      pbase = min(fdiv(kb + wrow, a.ps), lastp);
      pv = clampp(bt[min(pbase + lane, lastp)]) * a.c_ps;
      pn = bt[min(pbase + 64 + lane, lastp)];
    } else {
      lookup(kb);
    }
    At a0{};
    place(0, a0);
    fetch(kc, a0, 0, K0);
    load_q();
    fetch(vc, a0, 1, V0);
    place(min(1, n - 1), ak);
    fetch(kc, ak, 0, K1);
    wait_loads<2 * NL>();  // K(0)
    sync_lds();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      scores(K0, h, s[0][h]);
      if (edge(0)) apply_mask(0, h, s[0][h]);
      maxima(h, s[0][h]);
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const float y = fmaxf(mx[0][b], mx[1][b]);
      m[b] = fmaxf(NONE, fmaf(fmaxf(y, other_half(y)), a.cs, -F::MANY));
    }
    wait_loads();  // V(0) and K(1)
    sync_lds();    // every wave has read K(0): K(2) takes its place
  }
  wait_loads();  // (nothing is in flight: the compiler sees a way around the wait above, and would wait in the loop)

  // half H of tile j: x its scores; y those of the same half of tile j + 1, from the K image kl.  Written in the order
  // in which it is to run, fenced slot by slot: a product, then what the vector unit does while it runs, with
  // fragments read PF slots ahead (kf: the first are on their way).  Left to itself the compiler puts all products first.
  auto half = [&](int j, auto hc, const char* kl, const char* vl, f32x16 (&x)[RB], f32x16 (&y)[RB], v8 (&kf)[PF + 1],
                  auto&& ahead) __attribute__((always_inline)) {
    constexpr int H = decltype(hc)::value;
    constexpr int PE = 16 / KS > 0 ? 16 / KS : 1;  // scores of a slot
    v8 pt[RB][2];
    i16x8 vf[PF + 1];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (ks + PF < KS) kf[(ks + PF) % (PF + 1)] = kfrag(kl, H, ks + PF);
      const int v = ks - (KS - PF);
      if (v >= 0) vf[v] = vfrag(vl, v >> 1, 2 * H + (v & 1));
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        if (ks == 0) {
          f32x16 z;
#pragma unroll
          for (int r = 0; r < 16; ++r) z[r] = 0.f;
          y[b] = F::mma(kf[0], qf[b][0], z);
        } else {
          y[b] = F::mma(kf[ks % (PF + 1)], qf[b][ks], y[b]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < PE; ++i) {
          const int e = (ks * RB + b) * PE + i, eb = e / 16, r = e % 16;
          const float p = __builtin_amdgcn_exp2f(fmaf(x[eb][r], a.cs, -m[eb]));
          x[eb][r] = p;
          pt[eb][r >> 3][r & 7] = (T)p;  // (rounded to nearest: the matrix unit's operand; the sums keep fp32)
        }
        if (ks % 2 && b == RB - 1) ahead(ks / 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // (behind the last tile y is what was there, and not used)
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
      for (int u = 0; u < 2; ++u) asm volatile("" : "+v"(pt[b][u]));
    __builtin_amdgcn_sched_barrier(0);
    if (j + 1 < n && edge(j + 1)) apply_mask(j + 1, H, y);
    constexpr int SL = 2 * DC, SE = RB * 16 / (SL * RB) > 0 ? 16 / SL : 1;  // slots; sums and maxima of one
    float t[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) t[b] = y[b][0];
#pragma unroll
    for (int i = 0; i < SL; ++i) {
      if (i + PF < SL) vf[(i + PF) % (PF + 1)] = vfrag(vl, (i + PF) >> 1, 2 * H + ((i + PF) & 1));
      if (H == 0 && i >= SL - PF) kf[i - (SL - PF)] = kfrag(kl, 1, i - (SL - PF));
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        F::acc(o[b][i >> 1], __builtin_bit_cast(v8, vf[i % (PF + 1)]), pt[b][i & 1]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < SE; ++k) {
          const int e = (i * RB + b) * SE + k, eb = e / 16, r = e % 16;
          if (e < RB * 16) {
            l[eb] += x[eb][r];
            t[eb] = fmaxf(t[eb], y[eb][r]);
          }
        }
        const int pb = (i * RB + b) * SE / 16 % RB;
        asm volatile("" : "+v"(l[pb]), "+v"(t[pb]));  // (here, not where they are used)
        if (i % 2 && b == RB - 1) ahead(NL + i / 2);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
#pragma unroll
    for (int b = 0; b < RB; ++b) mx[H][b] = t[b];
  };
  using H0 = std::integral_constant<int, 0>;
  using H1 = std::integral_constant<int, 1>;
  auto step = [&](int j, char* k0, char* k1, char* v0, char* v1, f32x16 (&x)[2][RB], f32x16 (&y)[2][RB])
                  __attribute__((always_inline)) {
    // V(j + 1) lies where K(j + 1) did and takes the place of V(j - 1); K(j + 2) that of K(j)
    // (behind the last tile: the last again), a piece every other slot of the first half, as a row of them would hold
    // up the wave
    v8 kf[PF + 1];
#pragma unroll
    for (int ks = 0; ks < PF; ++ks) kf[ks] = kfrag(k1, 0, ks);
    av = ak;
    place(min(j + 2, n - 1), ak);
    auto ahead = [&](int p) __attribute__((always_inline)) {
      if (p < NL)
        piece(vc, av, 1, v1, p);
      else
        piece(kc, ak, 0, k0, p - NL);
    };
    auto none = [](int) {};
    // raise the maxima where they grew too much
    float rise = fmaf(fmaxf(mx[0][0], mx[1][0]), a.cs, -m[0]);
#pragma unroll
    for (int b = 1; b < RB; ++b) rise = fmaxf(rise, fmaf(fmaxf(mx[0][b], mx[1][b]), a.cs, -m[b]));
    if (__ballot(rise > F::GROW)) raise();
    if (edge(j)) {
      const int odd = look(j, v0);
      if (odd) mend(j, v0, odd & 2);
    }
    half(j, H0{}, k1, v0, x[0], y[0], kf, ahead);
    half(j, H1{}, k1, v0, x[1], y[1], kf, none);
    wait_loads();
    sync_lds();
  };
  int j = 0;
  for (; j + 1 < n; j += 2) {  // (a condition on the second step would cost a move of all of O a turn)
    step(j, K0, K1, V0, V1, s[0], s[1]);
    step(j + 1, K1, K0, V1, V0, s[1], s[0]);
  }
  if (j < n) step(j, K0, K1, V0, V1, s[0], s[1]);

  settle();
  // A lane stores its own row: 8 values at a time, after an exchange with the lane that holds the other half of its keys'
  // columns.  (32 bytes of 32 rows a store, which L2 puts together: through LDS, in whole rows, an item took 2 us more.)
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const float L = l[b] + other_half(l[b]);
    const int r = row0 + 32 * b + l32, tok = fdiv(min(r, R - 1), a.g), hd = it.head * (int)a.g.d + r - tok * (int)a.g.d;
    float x[DC][16];
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) x[c][i] = o[b][c][i];
    if (anyinf) {
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const int bits = inf[wave][c * RB + b][lane];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (bits >> i & 1) x[c][i] += INFINITY;
          if (bits >> i & 65536) x[c][i] -= INFINITY;
        }
      }
    }
    if (part) {
      const long slot = it.slot + (r - R0);
      if (r < R) {
        if (hi == 0) *reinterpret_cast<f32x2*>(a.ml + slot * 2) = f32x2{m[b], L};
        float* to = a.ws + slot * D + 4 * hi;
#pragma unroll
        for (int c = 0; c < DC; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            *reinterpret_cast<f32x4*>(to + 32 * c + 8 * k) = f32x4{x[c][4 * k], x[c][4 * k + 1], x[c][4 * k + 2], x[c][4 * k + 3]};
      }
      continue;
    }
    const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;  // (a row that saw no key: zeros)
    if (a.lse && hi == 0 && r < R)
      a.lse[(long)(it.q.q0 + tok) * a.l_ts + (long)hd * a.l_hs] = L == 0.f ? -INFINITY : (m[b] + __log2f(L)) * LN2;
    T* to = (T*)a.o + (long)(it.q.q0 + tok) * a.o_ts + (long)hd * a.o_hs + 8 * hi;
#pragma unroll
    for (int c = 0; c < DC; ++c)
#pragma unroll
      for (int k = 0; k < 4; k += 2) {  // columns 32 c + 8 (k + hi) ..
        typedef T t4 __attribute__((ext_vector_type(4)));
        typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
        t4 y[2];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[0][e] = (T)(x[c][4 * k + e] * inv), y[1][e] = (T)(x[c][4 * k + 4 + e] * inv);  // rounded once
        const u32x2 lo = __builtin_bit_cast(u32x2, y[0]), up = __builtin_bit_cast(u32x2, y[1]);
        const auto s0 = __builtin_amdgcn_permlane32_swap(lo[0], up[0], false, false);
        const auto s1 = __builtin_amdgcn_permlane32_swap(lo[1], up[1], false, false);
        const u32x4 w = {s0[0], s1[0], s0[1], s1[1]};
        if (r >= R) continue;
        if (a.ovec)
          *reinterpret_cast<u32x4*>(to + 32 * c + 8 * k) = w;
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const unsigned short u = (unsigned short)(w[e >> 1] >> (16 * (e & 1)));
            to[32 * c + 8 * k + e] = __builtin_bit_cast(T, u);
          }
      }
  }
}

// ---------------------------------------------------------------- few rows
// Few rows for each sequence and key/value head (single tokens), in tiles of 16: the keys' bytes bound it.  Four waves share out
// the key tiles (32 keys each); a wave streams on its own, with no barrier until the end.  A tile's keys come into
// registers (as they lie in memory they are the A operand of S^T = K Q^T), its values into LDS, from where the
// transposed reads of O^T += V^T P^T take them.  16 x 16 x 32 products: a 32-row form would spend twice the
// exponentials and registers on rows that are not there.  One buffer a wave and three workgroups a CU start
// sooner than two buffers and two workgroups: 32 sequences of 24 to 640 keys, 32 heads of 128, in 28.9 us instead of 34.3;
// contexts of 4k to 32k are read at the same 5.1 TB/s.  Four workgroups a CU spill registers (4.4 TB/s).
//
// The V image of 16 keys x 32 columns is 1 KiB: [16-byte chunk q][key ^ 8 (q & 1)], so that the transposed reads of
// half a wave (8 keys x 2 chunks) meet every bank once.
template <typename T>
struct Mma16;
template <>
struct Mma16<bf16> {
  __device__ static f32x4 mma(const bf16x8& x, const bf16x8& y, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, c, 0, 0, 0);
  }
};
template <>
struct Mma16<f16> {
  __device__ static f32x4 mma(const f16x8& x, const f16x8& y, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, c, 0, 0, 0);
  }
};

// value of every lane combined with those 16, 32 and 48 lanes on
__device__ __forceinline__ float max_groups(float x) {
  unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __float_as_uint(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto q = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
  unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// 4 chains (64 columns) of V^T fragments: 8 transposed reads and their wait in one block, so that no read is in
// flight outside it (the compiler would also drain the LDS-DMA of the next tile in front of reads that it sees)
template <int OFF, int HI>
__device__ __forceinline__ void read_v4(unsigned at, i16x4 (&lo)[4], i16x4 (&hi)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%9\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %5, %8 offset:%14\n\t"
      "ds_read_b64_tr_b16 %6, %8 offset:%15\n\t"
      "ds_read_b64_tr_b16 %7, %8 offset:%16\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
      : "v"(at), "n"(OFF), "n"(OFF + 512), "n"(OFF + 1024), "n"(OFF + 1536), "n"(OFF + HI), "n"(OFF + HI + 512),
        "n"(OFF + HI + 1024), "n"(OFF + HI + 1536)
      : "memory");
}

// workgroups of a CU: what the registers allow without spills
constexpr int few_per_cu(int D) { return D <= 64 ? 4 : D <= 128 ? 3 : 2; }

template <typename T, int D, bool P16>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(few_per_cu(D)))) void paged_few_kernel(
    const PagedArgs a) {
  using v8 = typename Frag<T>::v8;
  constexpr int BM = 16, KT = 32, NW = 4, KU = KT * NW;
  constexpr int KS = D / 32;   // d steps of S; also 64-byte column blocks of a row
  constexpr int DC = D / 16;   // d chains of O
  constexpr int VB = KT * D * 2;  // bytes of a V tile
  constexpr int PITCH = pitch_of(D);
  constexpr int OUT = NW * BM * PITCH * 4 + NW * BM * 8;
  __shared__ __attribute__((aligned(16))) char smem[NW * VB > OUT ? NW * VB : OUT];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = lane >> 4, l16 = lane & 15;

  Item it;
  if (!find_item<BM, KU>(a, blockIdx.x, lane, it)) return;
  const int R = it.q.n * (int)a.g.d;
  const int ub = it.u0 + it.chunk * it.cs;
  const int kb = ub * KU;
  const int end = tile_end(a, it, BM);
  const int ke = min(min(ub + it.cs, it.u0 + it.units) * KU, end);
  const bool part = it.nch > 1;
  note<BM, KU>(a, it, end);
  if (part && it.chunk > 0 && kb >= ke) return;
  const int row0 = it.tile * BM;

  // this lane's row (rows behind the last repeat it and are not stored)
  v8 qf[KS];
  const int r = min(row0 + l16, R - 1);
  const int tok = fdiv(r, a.g), hd = it.head * (int)a.g.d + r - tok * (int)a.g.d;
  const int lim = a.causal ? it.q.kv - it.q.n + tok : it.q.kv - 1;
  {
    const T* p = (const T*)a.q + (long)(it.q.q0 + tok) * a.q_ts + (long)hd * a.q_hs + 8 * G;
    if (a.qvec) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const v8*>(p + 32 * ks);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[ks][i] = p[32 * ks + i];
    }
  }
  // smallest limit of the tile's rows: its first row's
  const int low = a.causal ? it.q.kv - it.q.n + fdiv(row0, a.g) : it.q.kv - 1;

  f32x4 o[DC];
#pragma unroll
  for (int c = 0; c < DC; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = NONE, l = 0.f;

  // addresses: pages are read ahead of their keys
  const T* kc = (const T*)a.kc + (long)it.head * a.c_hs;
  const T* vc = (const T*)a.vc + (long)it.head * a.c_hs;
  const int* bt = a.bt + (long)it.seq * a.max_pages;
  const int n = ke > kb + wave * KT ? (ke - kb - wave * KT + KU - 1) / KU : 0;  // this wave's tiles
  const int kw = kb + wave * KT;  // its first key
  const int lastp = ke > 0 ? fdiv(ke - 1, a.ps) : 0;
  const int vrow = l16 ^ ((G & 1) << 3);  // key of this lane in a V piece
  char* vbuf = smem + wave * VB;
  auto clampp = [&](int p) __attribute__((always_inline)) { return min(max(p, 0), a.n_pages - 1); };

  // P16 (the page size is a multiple of 16): 16 keys lie in one page; 64 page numbers at a time sit on the lanes.
  // Slots behind a sequence's end are read (they are inside its last page) and masked.
  int pbase = 0, pv = 0, pn = 0;
  // otherwise every lane looks up its own rows, one tile ahead: K rows l16 and 16 + l16, V rows vrow and 16 + vrow
  int pg[4];
  auto lookup = [&](int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = min(k0 + (i & 1) * 16 + (i < 2 ? l16 : vrow), ke - 1);
      pg[i] = bt[fdiv(key, a.ps)];
    }
  };
  if (n > 0) {
    if constexpr (P16) {
      pbase = fdiv(kw, a.ps);
      pv = clampp(bt[min(pbase + lane, lastp)]);
      pn = bt[min(pbase + 64 + lane, lastp)];
    } else {
      lookup(kw);
    }
  }

  // where tile i's keys and values lie (K by its own lanes' rows; V: the address is kept until its turn)
  const T *kp[2], *vp[2];
  auto place = [&](int i) __attribute__((always_inline)) {
    const int k0 = kw + i * KU;
    if constexpr (P16) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int k1 = k0 + 16 * t;
        const int pi = fdiv(k1, a.ps), slot = k1 - pi * (int)a.ps.d;
        const int pc = min(pi, lastp);
        if (pc - pbase >= 64) {
          pbase += 64;
          pv = clampp(pn);
          pn = bt[min(pbase + 64 + lane, lastp)];
        }
        const long off = (long)lane_of(pv, pc - pbase) * a.c_ps + (long)slot * a.c_ts;
        kp[t] = kc + off + l16 * a.c_ts + 8 * G;
        vp[t] = vc + off + vrow * a.c_ts + 8 * G;
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int kk = min(k0 + 16 * t + l16, ke - 1), kv = min(k0 + 16 * t + vrow, ke - 1);
        kp[t] = kc + (long)clampp(pg[t]) * a.c_ps + (long)(kk - fdiv(kk, a.ps) * (int)a.ps.d) * a.c_ts + 8 * G;
        vp[t] = vc + (long)clampp(pg[2 + t]) * a.c_ps + (long)(kv - fdiv(kv, a.ps) * (int)a.ps.d) * a.c_ts + 8 * G;
      }
      lookup(k0 + KU);
    }
  };
  v8 kf[2][KS];
  auto issue_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) kf[t][ks] = *reinterpret_cast<const v8*>(kp[t] + 32 * ks);
  };
  auto issue_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int p = 0; p < KS; ++p) dma16(vp[t] + 32 * p, vbuf + (t * KS + p) * 1024);
  };

  const int li = lane & 15, vq = (li & 3) >> 1;
  const unsigned va = (unsigned)(uintptr_t)((LDS_AS const char*)vbuf) +
                      (vq * 16 + ((4 * G + (li >> 2)) ^ (vq << 3))) * 16 + (li & 1) * 8;
  // A masked key has p = 0, but 0 times an infinity or NaN in its value would reach the row all the same: in a tile that
  // some row sees in part such values become zeros in LDS.  Where rows see them (rare, and slow: key by key), which of
  // their sums get +infinity or -infinity (NaN: both) is kept until the end: 8 bits for each chain of O.
  unsigned inf[DC / 4];
#pragma unroll
  for (int c = 0; c < DC / 4; ++c) inf[c] = 0;
  auto mend = [&](int k0) __attribute__((always_inline)) {
    char* vl = vbuf;
    bool odd = false, seen = false;
#pragma nounroll
    for (int p = 0; p < 2 * KS; ++p) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(vl + p * 1024 + lane * 16);
      bool here = false;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        here = here || (x[e] & Frag<T>::EXP) == Frag<T>::EXP || (x[e] >> 16 & Frag<T>::EXP) == Frag<T>::EXP;
      const int key = k0 + 16 * (p / KS) + vrow;
      odd = odd || here;
      seen = seen || (here && key < ke && key >= it.q.st);
    }
    if (!__ballot(odd)) return;
    if (__ballot(seen)) {
#pragma nounroll
      for (int key = 0; key < KT; ++key) {
        const bool hid = k0 + key > lim || k0 + key < it.q.st;
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          const int q = 2 * (c & 1) + (G >> 1), kk = (key & 15) ^ ((q & 1) << 3);
          const i16x4 x = *reinterpret_cast<const i16x4*>(vl + ((key >> 4) * KS + (c >> 1)) * 1024 + (q * 16 + kk) * 16 +
                                                          (G & 1) * 8);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned v = (unsigned short)x[e];
            const bool odd1 = !hid && (v & Frag<T>::EXP) == Frag<T>::EXP, nan = v & Frag<T>::MAN;
            if (odd1 && (nan || !(v & 0x8000))) inf[c >> 2] |= 1u << (8 * (c & 3) + e);
            if (odd1 && (nan || (v & 0x8000))) inf[c >> 2] |= 16u << (8 * (c & 3) + e);
          }
        }
      }
    }
#pragma nounroll
    for (int p = 0; p < 2 * KS; ++p) {
      i16x8* x = reinterpret_cast<i16x8*>(vl + p * 1024 + lane * 16);
      *x = finite<T>(*x);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  // A tile: its scores as soon as its keys are there; then the next tile's keys are sent for (`more`), then its values
  // are waited for; the next tile's follow behind their last use.
  constexpr int OPS = 2 * KS;  // loads of a tile's keys, and of its values
  auto work = [&](int i, auto more) __attribute__((always_inline)) {
    constexpr bool MORE = decltype(more)::value;
    const int k0 = kw + i * KU;
    wait_loads<OPS>();
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[t] = Mma16<T>::mma(kf[t][ks], qf[ks], s[t]);
    }
    if constexpr (MORE) {
      place(i + 1);
      issue_k();
    }
    const bool mask = k0 < it.q.st || k0 + KT - 1 > low;
    if (mask) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = k0 + 16 * t + 4 * G + e;
          s[t][e] = key > lim || key < it.q.st ? -INFINITY : s[t][e];
        }
    }
    float mx = s[0][0];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[t][e]);
    mx = max_groups(mx);
    const float mn = fmaxf(m, fmaf(mx, a.cs, -Frag<T>::FEW));
    const float alpha = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    float sum = 0.f;
    v8 pt;  // P in the cache's type (rounded to nearest: the matrix unit's operand; the sum keeps fp32)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[t][e], a.cs, -mn));
        sum += p;
        pt[4 * t + e] = (T)p;
      }
    l = l * alpha + sum;  // this lane's keys; the lanes of a row are added up at the end
    wait_loads<MORE ? OPS : 0>();
    if (mask) mend(k0);
#pragma unroll
    for (int c4 = 0; c4 < DC; c4 += 4) {
      i16x4 lo[4], hi[4];
      // (a column block's 64 columns are 2 KiB; key group 1 lies KS KiB behind group 0)
      if (c4 == 0) read_v4<0, KS * 1024>(va, lo, hi);
      if (c4 == 4) read_v4<2048, KS * 1024>(va, lo, hi);
      if (c4 == 8) read_v4<4096, KS * 1024>(va, lo, hi);
      if (c4 == 12) read_v4<6144, KS * 1024>(va, lo, hi);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const i16x8 vv = {lo[c][0], lo[c][1], lo[c][2], lo[c][3], hi[c][0], hi[c][1], hi[c][2], hi[c][3]};
        o[c4 + c] = Mma16<T>::mma(__builtin_bit_cast(v8, vv), pt, o[c4 + c] * alpha);
      }
    }
  };
  if (n > 0) {
    place(0);
    issue_k();
    issue_v();
    for (int i = 0; i + 1 < n; ++i) {
      work(i, std::true_type{});
      issue_v();
    }
    work(n - 1, std::false_type{});
  }
#pragma unroll
  for (int c = 0; c < DC; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (inf[c >> 2] >> (8 * (c & 3)) & 1u << e) o[c][e] += INFINITY;
      if (inf[c >> 2] >> (8 * (c & 3)) & 16u << e) o[c][e] -= INFINITY;
    }
  l = sum_groups(l);

  // join the waves and store
  const int rows = min(BM, R - row0);
  float* ml = reinterpret_cast<float*>(smem + NW * BM * PITCH * 4);
  __syncthreads();
  if (G == 0) ml[(wave * BM + l16) * 2] = m, ml[(wave * BM + l16) * 2 + 1] = l;
  if (l16 < rows) {
    float* mine = reinterpret_cast<float*>(smem) + (wave * BM + l16) * PITCH + 4 * G;
#pragma unroll
    for (int c = 0; c < DC; ++c) *reinterpret_cast<f32x4*>(mine + 16 * c) = o[c];
  }
  __syncthreads();
  constexpr int TPR = D / 4;
  for (int idx = threadIdx.x; idx < rows * TPR; idx += 64 * NW) {
    const int lr = idx / TPR, d0 = (idx % TPR) * 4;
    float M = NONE, L = 0.f;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < NW; ++k) M = fmaxf(M, ml[(k * BM + lr) * 2]);
#pragma unroll
    for (int k = 0; k < NW; ++k) {
      const float w = __builtin_amdgcn_exp2f(ml[(k * BM + lr) * 2] - M);
      L += ml[(k * BM + lr) * 2 + 1] * w;
      const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(smem) + (k * BM + lr) * PITCH + d0);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += y[e] * w;
    }
    if (part) {
      const long slot = it.slot + lr;
      *reinterpret_cast<f32x4*>(a.ws + slot * D + d0) = f32x4{x[0], x[1], x[2], x[3]};
      if (d0 == 0) *reinterpret_cast<f32x2*>(a.ml + slot * 2) = f32x2{M, L};
    } else {
      const int rr = row0 + lr, t = fdiv(rr, a.g);
      store_row<T, 4>(a, it.q.q0 + t, it.head * (int)a.g.d + rr - t * (int)a.g.d, d0, x, M, L);
    }
  }
}

// Joins the chunks of a (tile, head), in their order: D / 4 threads a row, ROWS rows a workgroup.
template <typename T, int D, int BM, int ROWS>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a) {
  if ((int)blockIdx.x >= a.plan[0]) return;
  const Record it = *reinterpret_cast<const Record*>(a.plan + PLAN_HEAD + (long)blockIdx.x * RECORD);
  const int r0 = blockIdx.y * ROWS;
  if (it.chunks <= 0 || r0 >= it.rows) return;
  constexpr int TPR = D / 4, RPB = 256 / TPR, AT = 8;  // chunks on their way at once
  const int d0 = (threadIdx.x % TPR) * 4;
  const long ds = it.step;
  for (int lr = r0 + threadIdx.x / TPR; lr < min(r0 + ROWS, it.rows); lr += RPB) {
    const long s0 = it.first + lr;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    float M = NONE, L = 0.f;
    for (int c0 = 0; c0 < it.chunks; c0 += AT) {
      f32x2 p[AT];
      f32x4 y[AT];
#pragma unroll
      for (int c = 0; c < AT; ++c) {
        const long slot = s0 + min(c0 + c, it.chunks - 1) * ds;
        p[c] = *reinterpret_cast<const f32x2*>(a.ml + slot * 2);
        y[c] = *reinterpret_cast<const f32x4*>(a.ws + slot * D + d0);
      }
      float mn = M;
#pragma unroll
      for (int c = 0; c < AT; ++c) mn = fmaxf(mn, p[c][0]);
      const float old = __builtin_amdgcn_exp2f(M - mn);
      M = mn;
      L *= old;
      x *= old;
#pragma unroll
      for (int c = 0; c < AT; ++c) {
        const float w = c0 + c < it.chunks ? __builtin_amdgcn_exp2f(p[c][0] - M) : 0.f;
        if (c0 + c < it.chunks) L += p[c][1] * w, x += y[c] * w;
      }
    }
    const int r = it.row0 + lr, tok = fdiv(r, a.g);
    const float y[4] = {x[0], x[1], x[2], x[3]};
    store_row<T, 4>(a, it.q0 + tok, it.head * (int)a.g.d + r - tok * (int)a.g.d, d0, y, M, L);
  }
}

// ---------------------------------------------------------------- host
struct Plan {
  int BM, KU;
  long pairs, items;  // upper bounds: (tile, head) pairs and items
  long cap;           // rows of partial results
  int slots, split;
  long bar;   // keys that one sequence has to see before any are cut (on the device)
  bool sums;  // 64 sequences' (tile, head) pairs, counted with all rows each, fit 32 bits
  size_t o_off, ml_off, bytes;
};

int device_cus() {
  static int cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  if (!cus[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1) n = 256;
    cus[dev] = n;
  }
  return cus[dev];
}

// At most 32 rows for each sequence and key/value head on average: the kernel for few rows.  Otherwise the one for many
// (256-row tiles; 128 with 256-wide heads, whose O fills the registers at 32 rows a wave).  Few against many, captured:
// 32 heads over 8 of 128, 8 sequences of 4000 keys with 16, 32, 64 rows 33 / 42, 44 / 42, 68 / 44 us; 64 of 1000 keys 47 / 72,
// 66 / 73, 124 / 77; 32 over 32, 8 of 4000 103 / 146, 128 / 153, 249 / 157; 16 over 4 of 64, 64 of 1000 20 / 27, 26 / 27,
// 35 / 28.  It is one choice for the whole batch: a prompt beside enough single tokens, or in a batch whose other places are
// empty, takes the kernel for few rows (4096 tokens of 32 heads in 256 places: 945 us, 206 alone).
Plan make_plan(long rows, int S, int Hq, int Hk, int D, long most) {
  Plan p;
  const long g = Hq / Hk;
  const bool few = rows * g <= 32l * S;
  p.BM = few ? 16 : D > 128 ? 128 : 256;
  p.KU = few ? 128 : 64;
  const long a = rows * g / p.BM + S, b = rows * ((g + p.BM - 1) / p.BM);
  p.pairs = (a < b ? a : b) * Hk;
  p.slots = device_cus() * (few ? few_per_cu(D) : 1);
  const long least = (rows * g + p.BM - 1) / p.BM * Hk;
  // Splitting costs the partial results' way through memory and a second launch.  It pays from more keys on the less room
  // the tiles leave for chunks, and not where there are tiles enough for four rounds.  Whole against cut: one token, 32
  // heads over 8 of 128, 400, 700, 1000, 4000 keys 12 / 17, 16 / 17, 20 / 17, 59 / 17 us; 8 times one token, 32 over 32,
  // 400, 1000, 2000: 15 / 19, 26 / 30, 46 / 49; 64 tokens over 200, 1000, 4000: 19 / 19, 36 / 22, 105 / 28; four chunks of
  // 256 tokens (half of the slots) over 200, 1000, 1500, 4000: 25 / 36, 42 / 46, 54 / 53, 111 / 87; four of 512 (all slots)
  // over 0, 512, 1000, 4000: 24 / 33, 38 / 46, 54 / 62, 139 / 147 (equal lengths, where there is nothing to even out).
  // Those are calls, two launches against one.  The host knows only the table's width, and a captured step's table is as
  // wide as its sequences may ever get: whether keys are cut then follows on the device from the longest sequence, by a bar
  // of the kernels' times alone.  Whole against cut, captured, a table of 200,000 keys: one token, 32 heads over 8, 256,
  // 512, 1000 keys 12.1 / 11.8, 15.0 / 12.1, 22.8 / 12.4 us; 8 times one token, 32 over 32, 13.3 / 15.7, 19.0 / 20.8,
  // 29.3 / 30.7; 64 tokens over 0, 256, 1000: 14.4 / 15.1, 20.8 / 18.6, 39.5 / 22.0; four chunks of 256 over 0, 512, 1000:
  // 21 / 32, 34 / 40, 48 / 48.
  const long bar = few ? 640 + 384 * p.pairs / p.slots : 256 + 2048 * p.pairs / p.slots;
  p.bar = few ? std::min(bar, 256 + 1536 * p.pairs / p.slots) : 96 + 1900 * p.pairs / p.slots;
  // (a q_start that descends may give every sequence all rows: not split where the device's sums of that could wrap)
  p.split = most > bar && least < 4l * p.slots && least * S < (1l << 30);
  p.sums = least < (1l << 25);
  p.items = !p.split ? p.pairs : p.pairs <= p.slots ? p.slots : p.pairs + 4l * p.slots;
  p.o_off = (size_t)(PLAN_HEAD + p.pairs * RECORD) * 4;  // bytes, a multiple of 16
  // Partial results: a tile's rows for every place of the launch, or all rows over all key blocks, where that is less.
  // Filling the places once takes no more.  Evening out several rounds may: four tiles' then of few rows, and beyond that
  // larger chunks (pick_chunk).  34 MB at most.
  p.cap = (long)std::min((double)p.slots * p.BM * (few && p.pairs > p.slots ? 4 : 1),
                         (double)rows * g * Hk * ((most + p.KU - 1) / p.KU));
  p.ml_off = p.o_off + (size_t)p.cap * D * 4;
  p.bytes = p.split ? p.ml_off + (size_t)p.cap * 2 * 4 : 0;
  return p;
}

template <typename T, int D, int BM>
int join(PagedArgs& a, const Plan& p, hipStream_t st) {
  OSPO_CHECK_LAUNCH();
  if (!p.split) return OSPO_OK;
  constexpr int ROWS = 1024 / D;  // rows of one pass
  paged_join_kernel<T, D, BM, ROWS><<<dim3((unsigned)p.pairs, BM / ROWS), 256, 0, st>>>(a);
  OSPO_CHECK_LAUNCH();
  return OSPO_OK;
}

template <typename T, int D>
int launch(PagedArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)p.items);
  if (p.BM == 16) {
    if (a.ps.d % 16 == 0)
      paged_few_kernel<T, D, true><<<grid, 256, 0, st>>>(a);
    else
      paged_few_kernel<T, D, false><<<grid, 256, 0, st>>>(a);
    return join<T, D, 16>(a, p, st);
  }
  constexpr int RB = D > 128 ? 1 : 2;
  // (16 keys in one page, and near enough to each other for 32-bit byte offsets)
  if (a.ps.d % 16 == 0 && a.c_ts >= 0 && a.c_ts < (1l << 26))
    paged_many_kernel<T, D, RB, true><<<grid, 256, 0, st>>>(a);
  else
    paged_many_kernel<T, D, RB, false><<<grid, 256, 0, st>>>(a);
  return join<T, D, 128 * RB>(a, p, st);
}

bool shapes_ok(int n, int S, int Hq, int Hk, int D, int n_pages, int page_size, int max_pages) {
  return n >= 0 && S >= 0 && Hk >= 1 && Hq >= Hk && Hq % Hk == 0 && Hq <= 4096 && n_pages >= 0 && page_size >= 1 &&
         max_pages >= 0 && (long)max_pages * page_size <= 0x7fff0000L && (long)n * (Hq / Hk) <= 0x7fffff00L;
}

}  // namespace

extern "C" size_t ospo_paged_attn_ws_bytes(int n, int n_seqs, int n_q_heads, int n_kv_heads, int head_dim,
                                           int page_size, int max_pages) {
  if (!shapes_ok(n, n_seqs, n_q_heads, n_kv_heads, head_dim, 0, page_size, max_pages) || !n || !n_seqs) return 0;
  return make_plan(n, n_seqs, n_q_heads, n_kv_heads, head_dim, (long)page_size * max_pages).bytes;
}

extern "C" int ospo_paged_attn(const void* q, long q_ts, long q_hs, const void* k_cache, const void* v_cache,
                               long page_stride, long head_stride, long slot_stride, int n_pages, int page_size,
                               const int* block_table, int max_pages, const int* q_start, const int* kv_len,
                               const int* start, int n_seqs, int n, int n_q_heads, int n_kv_heads, int head_dim,
                               float scale, int causal, void* out, long o_ts, long o_hs, float* lse, long l_ts,
                               long l_hs, int dtype, void* ws, size_t ws_bytes, hipStream_t stream) {
  if (!shapes_ok(n, n_seqs, n_q_heads, n_kv_heads, head_dim, n_pages, page_size, max_pages)) return OSPO_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return OSPO_ERR_UNSUPPORTED;
  if (dtype != DT_BF16 && dtype != DT_F16) return OSPO_ERR_UNSUPPORTED;
  if (!(scale > 0.f) || !(scale < INFINITY) || (causal != 0 && causal != 1)) return OSPO_ERR_ARG;
  if (n == 0 || n_seqs == 0) return OSPO_OK;
  if (!q || !out || !q_start || !kv_len) return OSPO_ERR_ARG;
  const bool keys = max_pages > 0 && n_pages > 0;  // a cache without pages: every row sees nothing
  if (keys && (!k_cache || !v_cache || !block_table)) return OSPO_ERR_ARG;
  if (keys && (!aligned16(k_cache) || !aligned16(v_cache))) return OSPO_ERR_ALIGN;
  if (page_stride % 8 || head_stride % 8 || slot_stride % 8) return OSPO_ERR_ALIGN;
  const Plan p = make_plan(n, n_seqs, n_q_heads, n_kv_heads, head_dim, (long)page_size * max_pages);
  if (p.items > 0x7fffffffL || p.pairs > 0x7fffffffL || !p.sums) return OSPO_ERR_SHAPE;
  if (p.split && (!ws || ws_bytes < p.bytes)) return OSPO_ERR_ARG;
  if (p.split && !aligned16(ws)) return OSPO_ERR_ALIGN;
  PagedArgs a{};
  a.q = q, a.kc = k_cache, a.vc = v_cache, a.o = out, a.lse = lse;
  a.bt = block_table, a.qs = q_start, a.kl = kv_len, a.st = start;
  a.q_ts = q_ts, a.q_hs = q_hs, a.o_ts = o_ts, a.o_hs = o_hs, a.l_ts = l_ts, a.l_hs = l_hs;
  a.c_ps = page_stride, a.c_hs = head_stride, a.c_ts = slot_stride;
  a.rows = n, a.S = n_seqs, a.Hk = n_kv_heads, a.n_pages = n_pages, a.max_pages = max_pages;
  a.most = keys ? max_pages * page_size : 0;
  a.g = make_fdiv((uint32_t)(n_q_heads / n_kv_heads));
  a.ps = make_fdiv((uint32_t)page_size);
  a.cs = scale * LOG2E;
  a.causal = causal;
  a.qvec = aligned16(q) && q_ts % 8 == 0 && q_hs % 8 == 0;
  a.ovec = aligned16(out) && o_ts % 8 == 0 && o_hs % 8 == 0;
  a.slots = p.slots, a.split = p.split, a.bar = (int)std::min(p.bar, 0x7fffffffL), a.items = p.items, a.pairs = p.pairs;
  a.cap = (int)p.cap;
  a.plan = (int*)ws, a.ws = (float*)((char*)ws + p.o_off), a.ml = (float*)((char*)ws + p.ml_off);
  if (dtype == DT_BF16) {
    switch (head_dim) {
      case 64: return launch<bf16, 64>(a, p, stream);
      case 128: return launch<bf16, 128>(a, p, stream);
      default: return launch<bf16, 256>(a, p, stream);
    }
  }
  switch (head_dim) {
    case 64: return launch<f16, 64>(a, p, stream);
    case 128: return launch<f16, 128>(a, p, stream);
    default: return launch<f16, 256>(a, p, stream);
  }
}
