// Rotary positions on queries and keys, and the append of keys and values to a paged cache with the rotation on
// the way.
//
// A pair (x1, x2) of a head at position p turns by the angle a = p f_i of the caller's fp32 tables:
//   y1 = x1 cos a - x2 sin a,  y2 = x2 cos a + x1 sin a        (gradient: the transpose, sin a negated)
// computed in fp32 and rounded once.  Pairs are (i, i + rot/2) or (2i, 2i + 1); elements behind rot pass through.
//
// Memory bound: every element is read once and written once.  A thread owns one unit (W elements and their
// partners) of one token and walks the heads, so a token's cos / sin are read once per unit and not per head.
// Measured: 32 + 32 heads of 128 for 4800 tokens (158 MB) in 26.9 us, 5.9 TB/s; the append of 8192 tokens with 32 + 8 heads
// of 128 (206 MB) in 41.9 us, 4.9 TB/s.  A copy of 4 GiB reaches 4.8 TB/s; these sizes sit partly in the Infinity Cache.
#include "paged.h"

namespace {

constexpr int RT = 256;  // threads per workgroup

template <typename T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {
  return (T)x;
}

template <typename T, int W>
struct alignas(sizeof(T) * W) Vec {
  T v[W];
};

struct Part {  // one tensor's heads: [token][head][dim] by strides
  const void* x;
  void* y;
  long x_ts, x_hs, y_ts, y_hs;
};

struct RotArgs {
  Part q, k, v;         // v: the append only
  int hq, hk, hv;       // heads of each (0: none)
  int n, D, rot;
  const int* positions;  // [n] (rotary only)
  const float* cos_t;    // [n_pos][rot / 2]
  const float* sin_t;
  int n_pos;
  float sgn;             // -1: the gradient
  int U, Ur;             // units per head, of which turn
  int hs, tpb;           // head slots and tokens per workgroup
  int copy;              // q and k out of place: pass-through units are copied
  // append
  const int* bt;
  const int* qs;
  const int* kl;
  int S, n_pages, max_pages;
  FDiv ps;
  long c_ps, c_hs, c_ts;  // cache strides: page, head, slot
};

// W elements per load; IL: pairs are neighbours; AP: the append
template <typename T, int W, bool IL, bool AP>
__global__ __launch_bounds__(RT) void rotary_kernel(const RotArgs a) {
  using V = Vec<T, W>;
  constexpr int P = IL ? (W > 1 ? W / 2 : 1) : W;  // pairs per unit
  const int tid = threadIdx.x;
  const int unit = tid % a.U, slot = tid / a.U;
  const int tl = slot / a.hs, h0 = slot - tl * a.hs;
  const long tok = (long)blockIdx.x * a.tpb + tl;
  const bool live = tl < a.tpb && tok < a.n;

  int pos = 0;
  long crow = 0;  // append: element offset of the token's cache row
  bool put = false;
  if constexpr (AP) {
    // sequence of a row: the number of q_start[1 ..] at or below it, counted by a wave at a time (rows of one
    // workgroup are few); a row outside every sequence, a negative position and a page outside the cache are
    // left out
    __shared__ int s_seq[RT];
    const int lane = tid & 63;
    for (int i = tid >> 6; i < a.tpb; i += RT / 64) {
      const long row = (long)blockIdx.x * a.tpb + i;
      int cnt = 0;
      for (int s0 = 0; s0 < a.S; s0 += 64) {
        const int s = s0 + lane;
        cnt += __popcll(__ballot(s < a.S && a.qs[min(s, a.S - 1) + 1] <= row));
      }
      if (lane == 0) s_seq[i] = cnt;
    }
    __syncthreads();
    if (!live) return;
    const int s = s_seq[tl];
    if (s >= a.S) return;
    const int row = (int)tok;
    if (row < a.qs[s]) return;
    pos = a.kl[s] - a.qs[s + 1] + row;
    if (pos >= 0) {
      const int pi = fdiv(pos, a.ps);
      if (pi < a.max_pages) {
        const int page = a.bt[(long)s * a.max_pages + pi];
        put = page >= 0 && page < a.n_pages;
        crow = (long)page * a.c_ps + (long)(pos - pi * (int)a.ps.d) * a.c_ts;
      }
    }
  } else {
    if (!live) return;
    pos = a.positions[tok];
  }

  const bool turn = unit < a.Ur;
  float c[P], s[P];
  if (turn && a.rot > 0) {
    const long t = (long)min(max(pos, 0), a.n_pos - 1) * (a.rot >> 1) + unit * P;
    if constexpr (P % 4 == 0) {
#pragma unroll
      for (int i = 0; i < P; i += 4) {
        *reinterpret_cast<f32x4*>(c + i) = *reinterpret_cast<const f32x4*>(a.cos_t + t + i);
        *reinterpret_cast<f32x4*>(s + i) = *reinterpret_cast<const f32x4*>(a.sin_t + t + i);
      }
    } else if constexpr (P == 2) {
      *reinterpret_cast<f32x2*>(c) = *reinterpret_cast<const f32x2*>(a.cos_t + t);
      *reinterpret_cast<f32x2*>(s) = *reinterpret_cast<const f32x2*>(a.sin_t + t);
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) c[i] = a.cos_t[t + i], s[i] = a.sin_t[t + i];
    }
#pragma unroll
    for (int i = 0; i < P; ++i) s[i] *= a.sgn;
  }
  // element offsets of the unit in a head: the first load, and the second of a turning unit
  int e0, e1;
  if (turn) {
    e0 = IL ? 2 * unit * P : unit * P;
    e1 = IL ? e0 + 1 : e0 + (a.rot >> 1);
  } else {
    e0 = a.rot + (unit - a.Ur) * W;
    e1 = e0;
  }
  const int H = a.hq + a.hk + a.hv;
  for (int h = h0; h < H; h += a.hs) {
    const T* src;
    T* dst;
    bool rotate = turn;
    if (h < a.hq) {
      src = (const T*)a.q.x + tok * a.q.x_ts + (long)h * a.q.x_hs;
      dst = (T*)a.q.y + tok * a.q.y_ts + (long)h * a.q.y_hs;
      if (!turn && !a.copy) continue;
    } else if (h < a.hq + a.hk) {
      const int i = h - a.hq;
      src = (const T*)a.k.x + tok * a.k.x_ts + (long)i * a.k.x_hs;
      if constexpr (AP) {
        if (!put) continue;
        dst = (T*)a.k.y + crow + (long)i * a.c_hs;
      } else {
        dst = (T*)a.k.y + tok * a.k.y_ts + (long)i * a.k.y_hs;
        if (!turn && !a.copy) continue;
      }
    } else {
      if (!put) continue;
      const int i = h - a.hq - a.hk;
      src = (const T*)a.v.x + tok * a.v.x_ts + (long)i * a.v.x_hs;
      dst = (T*)a.v.y + crow + (long)i * a.c_hs;
      rotate = false;
    }
    if constexpr (IL) {
      if constexpr (W == 1) {
        const float x1 = to_f(src[e0]), x2 = turn ? to_f(src[e1]) : 0.f;
        if (rotate) {
          dst[e0] = from_f<T>(x1 * c[0] - x2 * s[0]);
          dst[e1] = from_f<T>(x2 * c[0] + x1 * s[0]);
        } else {
          dst[e0] = src[e0];
          if (turn) dst[e1] = src[e1];
        }
      } else {
        V x = *reinterpret_cast<const V*>(src + e0);
        if (rotate) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float x1 = to_f(x.v[2 * i]), x2 = to_f(x.v[2 * i + 1]);
            x.v[2 * i] = from_f<T>(x1 * c[i] - x2 * s[i]);
            x.v[2 * i + 1] = from_f<T>(x2 * c[i] + x1 * s[i]);
          }
        }
        *reinterpret_cast<V*>(dst + e0) = x;
      }
    } else {
      V x = *reinterpret_cast<const V*>(src + e0);
      if (turn) {
        V z = *reinterpret_cast<const V*>(src + e1);
        if (rotate) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            const float x1 = to_f(x.v[i]), x2 = to_f(z.v[i]);
            x.v[i] = from_f<T>(x1 * c[i] - x2 * s[i]);
            z.v[i] = from_f<T>(x2 * c[i] + x1 * s[i]);
          }
        }
        *reinterpret_cast<V*>(dst + e1) = z;
      }
      *reinterpret_cast<V*>(dst + e0) = x;
    }
  }
}

template <typename T, bool AP>
int launch_w(RotArgs& a, int W, int il, hipStream_t st) {
  const int P = il ? (W > 1 ? W / 2 : 1) : W;
  a.Ur = a.rot / 2 / P;
  a.U = a.Ur + (a.D - a.rot) / W;
  if (a.U > RT) return OSPO_ERR_UNSUPPORTED;
  const int slots = RT / a.U, H = a.hq + a.hk + a.hv;
  a.hs = H < slots ? H : slots;
  a.tpb = slots / a.hs;
  const dim3 grid((unsigned)(((long)a.n + a.tpb - 1) / a.tpb)), block(RT);
#define OSPO_ROT(WW)                                                               \
  case WW:                                                                         \
    if (il)                                                                        \
      rotary_kernel<T, WW, true, AP><<<grid, block, 0, st>>>(a);                   \
    else                                                                           \
      rotary_kernel<T, WW, false, AP><<<grid, block, 0, st>>>(a);                  \
    break;
  switch (W) {
    OSPO_ROT(1)
    OSPO_ROT(2)
    OSPO_ROT(4)
    case 8:
      if constexpr (sizeof(T) == 2) {
        if (il)
          rotary_kernel<T, 8, true, AP><<<grid, block, 0, st>>>(a);
        else
          rotary_kernel<T, 8, false, AP><<<grid, block, 0, st>>>(a);
        break;
      }
    default:
      return OSPO_ERR_UNSUPPORTED;
  }
#undef OSPO_ROT
  OSPO_CHECK_LAUNCH();
  return OSPO_OK;
}

template <bool AP>
int launch(RotArgs& a, int W, int il, int dtype, hipStream_t st) {
  switch (dtype) {
    case DT_BF16: return launch_w<bf16, AP>(a, W, il, st);
    case DT_F16: return launch_w<f16, AP>(a, W, il, st);
    case DT_F32: return launch_w<float, AP>(a, W, il, st);
  }
  return OSPO_ERR_UNSUPPORTED;
}

// Widest load (elements) that every row, head and unit of the call allows: a power of two up to 16 bytes that
// divides the sizes and strides and to which the pointers are aligned.  (The append of 8192 tokens at 16, 8 and 2 bytes
// a load: 45, 49 and 83 us.)
struct Width {
  int es;
  int w;
  explicit Width(int es_) : es(es_), w(16 / es_) {}
  void elems(long v) {
    while (w > 1 && v % w) w >>= 1;
  }
  void ptr(const void* p, int bytes_per_elem) {
    while (w > 1 && ((uintptr_t)p) % (uintptr_t)(w * bytes_per_elem < 16 ? w * bytes_per_elem : 16)) w >>= 1;
  }
  void part(const Part& p, int heads, bool y) {
    if (!heads) return;
    ptr(p.x, es);
    elems(p.x_ts), elems(p.x_hs);
    ptr(p.y, es);
    if (y) elems(p.y_ts), elems(p.y_hs);
  }
};

int common_checks(const RotArgs& a, int il, int dtype) {
  if (dtype != DT_BF16 && dtype != DT_F16 && dtype != DT_F32) return OSPO_ERR_UNSUPPORTED;
  if (il != 0 && il != 1) return OSPO_ERR_ARG;
  if (a.n < 0 || a.D < 1 || a.D > 256 || a.rot < 0 || a.rot > a.D || a.rot % 2) return OSPO_ERR_SHAPE;
  if (a.hq < 0 || a.hk < 0 || a.hq > 4096 || a.hk > 4096) return OSPO_ERR_SHAPE;
  return OSPO_OK;
}

}  // namespace

extern "C" int ospo_rotary(const void* q, long q_ts, long q_hs, void* q_out, long qo_ts, long qo_hs, int n_q_heads,
                           const void* k, long k_ts, long k_hs, void* k_out, long ko_ts, long ko_hs, int n_k_heads,
                           int n, int head_dim, int rot_dim, int interleaved, const int* positions,
                           const float* cos_tab, const float* sin_tab, int n_pos, int backward, int dtype,
                           hipStream_t stream) {
  RotArgs a{};
  a.q = Part{q, q_out, q_ts, q_hs, qo_ts, qo_hs};
  a.k = Part{k, k_out, k_ts, k_hs, ko_ts, ko_hs};
  a.hq = n_q_heads, a.hk = n_k_heads, a.hv = 0;
  a.n = n, a.D = head_dim, a.rot = rot_dim;
  if (const int rc = common_checks(a, interleaved, dtype)) return rc;
  if (rot_dim < 2 || n_pos < 1 || n_q_heads < 1) return OSPO_ERR_SHAPE;
  if (backward != 0 && backward != 1) return OSPO_ERR_ARG;
  if (n == 0) return OSPO_OK;
  if (!q || !q_out || !positions || !cos_tab || !sin_tab) return OSPO_ERR_ARG;
  if (n_k_heads && (!k || !k_out)) return OSPO_ERR_ARG;
  a.positions = positions, a.cos_t = cos_tab, a.sin_t = sin_tab, a.n_pos = n_pos;
  a.sgn = backward ? -1.f : 1.f;
  // in place: the elements behind rot stay where they are
  a.copy = !(q == q_out && q_ts == qo_ts && q_hs == qo_hs &&
             (!n_k_heads || (k == k_out && k_ts == ko_ts && k_hs == ko_hs)));
  const int es = dtype == DT_F32 ? 4 : 2;
  Width w(es);
  w.part(a.q, a.hq, true);
  w.part(a.k, a.hk, true);
  w.elems(head_dim);
  w.elems(interleaved ? rot_dim : rot_dim / 2);
  w.ptr(cos_tab, 4), w.ptr(sin_tab, 4);
  return launch<false>(a, w.w, interleaved, dtype, stream);
}

extern "C" int ospo_paged_append(const void* k, long k_ts, long k_hs, const void* v, long v_ts, long v_hs,
                                 const void* q, long q_ts, long q_hs, void* q_out, long qo_ts, long qo_hs, int n,
                                 int n_q_heads, int n_kv_heads, int head_dim, void* k_cache, void* v_cache,
                                 long page_stride, long head_stride, long slot_stride, int n_pages, int page_size,
                                 const int* block_table, int max_pages, const int* q_start, const int* kv_len,
                                 int n_seqs, const float* cos_tab, const float* sin_tab, int n_pos, int rot_dim,
                                 int interleaved, int dtype, hipStream_t stream) {
  RotArgs a{};
  a.q = Part{q, q_out, q_ts, q_hs, qo_ts, qo_hs};
  a.k = Part{k, k_cache, k_ts, k_hs, 0, 0};
  a.v = Part{v, v_cache, v_ts, v_hs, 0, 0};
  a.hq = n_q_heads, a.hk = n_kv_heads, a.hv = n_kv_heads;
  a.n = n, a.D = head_dim, a.rot = rot_dim;
  if (const int rc = common_checks(a, interleaved, dtype)) return rc;
  if (n_kv_heads < 1 || n_seqs < 0 || n_pages < 0 || page_size < 1 || max_pages < 0) return OSPO_ERR_SHAPE;
  if ((long)max_pages * page_size > 0x7fff0000L) return OSPO_ERR_SHAPE;
  if (rot_dim > 0 && n_pos < 1) return OSPO_ERR_SHAPE;
  if (n == 0 || n_seqs == 0) return OSPO_OK;
  if (!k || !v || !q_start || !kv_len) return OSPO_ERR_ARG;
  // a cache without pages and a table without columns hold no address: no row is stored
  if ((n_pages > 0 && (!k_cache || !v_cache)) || (max_pages > 0 && !block_table)) return OSPO_ERR_ARG;
  if (rot_dim > 0 && (!cos_tab || !sin_tab)) return OSPO_ERR_ARG;
  if (n_q_heads && (!q || !q_out)) return OSPO_ERR_ARG;
  a.cos_t = cos_tab, a.sin_t = sin_tab, a.n_pos = n_pos, a.sgn = 1.f, a.copy = 1;
  a.bt = block_table, a.qs = q_start, a.kl = kv_len, a.S = n_seqs, a.n_pages = n_pages, a.max_pages = max_pages;
  a.ps = make_fdiv((uint32_t)page_size);
  a.c_ps = page_stride, a.c_hs = head_stride, a.c_ts = slot_stride;
  Width w(dtype == DT_F32 ? 4 : 2);
  w.part(a.q, a.hq, true);
  w.part(a.k, a.hk, false);
  w.part(a.v, a.hv, false);
  w.elems(page_stride), w.elems(head_stride), w.elems(slot_stride);
  w.elems(head_dim);
  if (rot_dim > 0) {
    w.elems(interleaved ? rot_dim : rot_dim / 2);
    w.ptr(cos_tab, 4), w.ptr(sin_tab, 4);
  }
  return launch<true>(a, w.w, interleaved, dtype, stream);
}
