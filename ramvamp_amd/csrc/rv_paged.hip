// rv_paged.hip — rotary positions of rows of heads, and rows into a paged cache
// (K normed and rotated on the way) and back.
//
// Rotation (primitives/rope.rs:31-45, for any part of a head, both pairings and
// scaled frequencies): a row's angles p * f_i, their cosines and sines are
// computed once per workgroup in f64, rounded to f32 and kept in LDS, and all of
// the workgroup's heads take them from there; the rotation's products and sums
// are f32 with one rounding each (contraction off). So a row's values do not
// depend on which call rotated it.
#include "rv_paged.hpp"

#include <algorithm>

namespace rv {

PagedView paged_view(const rv_paged* pg, size_t layer, const rv_page_table& t) {
  PagedView w{};
  const size_t codes = pg->n_layers * pg->layer_elems() * pg->elem_size();
  const size_t at = layer * pg->layer_elems() * pg->elem_size();
  w.k = (char*)pg->k + at;
  w.v = (char*)pg->v + at;
  if (pg->elem == RV_ELEM_Q8_0) {
    w.ks = (uint16_t*)((char*)pg->k + codes) + layer * (pg->layer_elems() / 32);
    w.vs = (uint16_t*)((char*)pg->v + codes) + layer * (pg->layer_elems() / 32);
  }
  w.hd = (int)pg->head_dim;
  w.n_kv = (int)pg->n_kv_heads;
  w.layer = (uint32_t)layer;
  w.status = pg->status;
  w.t = Pages{t.ids, (long)t.stride, (uint32_t)t.n_seqs, (uint32_t)t.pages, (uint32_t)pg->n_pages,
              __builtin_ctzll(pg->page_rows)};
  return w;
}

namespace {

template <int N>
struct Turns {
  // (A last piece of fewer than four pairs reads a few past them.)
  __attribute__((aligned(16))) float c[N + 4], s[N + 4];
};

// Cosines and sines of a row's pairs, by the threads of a workgroup.
template <int N>
__device__ __forceinline__ void fill_turns(const RopeArgs<N>& rope, int pos, Turns<N>& t) {
  for (int i = threadIdx.x; i < rope.pairs; i += blockDim.x) {
    double sd, cd;
    sincos((double)pos * rope.freq[i], &sd, &cd);
    t.c[i] = (float)(rope.gain * cd);
    t.s[i] = (float)(rope.gain * sd);
  }
}

// ---- rotary positions ---------------------------------------------------------

typedef Oct Piece;  // four pairs of one head, or eight of its values that pass through

struct RopeShape {
  int hd, pairs, pair_groups, groups;  // a head's pieces: those of pairs, all
  uint32_t pieces;                     // of a row
  // A piece of four pairs is two quads of values: of one half of the rotated part and
  // of the other (so that neighbouring threads' quads are neighbours), or, of
  // interleaved pairs that do not come in fours, eight values in a row.
  bool halves;
};

// The quads' places in a head.
template <bool INTER>
__device__ __forceinline__ int quad_a(const RopeShape& sh, int g) { return INTER && !sh.halves ? 8 * g : 4 * g; }
template <bool INTER>
__device__ __forceinline__ int quad_b(const RopeShape& sh, int g) {
  return INTER && !sh.halves ? 8 * g + 4 : sh.pairs + 4 * g;
}

template <bool INTER>
__device__ __forceinline__ Piece load_piece(const RopeShape& sh, const float* __restrict__ head, int g) {
  Piece p{};
  const bool turned = g < sh.pair_groups;
  const int at = 2 * sh.pairs + 8 * (g - sh.pair_groups);  // of eight that pass through
  const int n = turned ? 2 * (sh.pairs - 4 * g) : sh.hd - at;  // values left
  const int qa = turned ? quad_a<INTER>(sh, g) : at, qb = turned ? quad_b<INTER>(sh, g) : at + 4;
  if (n >= 8) {
    p.a = *reinterpret_cast<const f32x4u*>(head + qa);
    p.b = *reinterpret_cast<const f32x4u*>(head + qb);
  } else {
    const int na = turned && !INTER ? n / 2 : min(n, 4), nb = n - na;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < na) p.a[e] = head[qa + e];
      if (e < nb) p.b[e] = head[qb + e];
    }
  }
  return p;
}

template <bool INTER, int N>
__device__ __forceinline__ void store_piece(const RopeShape& sh, const Turns<N>& t, float* __restrict__ head, int g,
                                            const Piece& p) {
#pragma clang fp contract(off)
  const bool turned = g < sh.pair_groups;
  const int at = 2 * sh.pairs + 8 * (g - sh.pair_groups);
  const int n = turned ? 2 * (sh.pairs - 4 * g) : sh.hd - at;
  const int qa = turned ? quad_a<INTER>(sh, g) : at, qb = turned ? quad_b<INTER>(sh, g) : at + 4;
  f32x4 a = p.a, b = p.b;
  if (turned && INTER) {
    const int ia = qa / 2, ib = qb / 2;  // the quads' first pairs
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float ca = t.c[ia + e], sa = t.s[ia + e], cb = t.c[ib + e], sb = t.s[ib + e];
      a[2 * e] = p.a[2 * e] * ca - p.a[2 * e + 1] * sa;
      a[2 * e + 1] = p.a[2 * e] * sa + p.a[2 * e + 1] * ca;
      b[2 * e] = p.b[2 * e] * cb - p.b[2 * e + 1] * sb;
      b[2 * e + 1] = p.b[2 * e] * sb + p.b[2 * e + 1] * cb;
    }
  } else if (turned) {
    const f32x4 c = *reinterpret_cast<const f32x4*>(t.c + 4 * g), s = *reinterpret_cast<const f32x4*>(t.s + 4 * g);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = p.a[e] * c[e] - p.b[e] * s[e];
      b[e] = p.a[e] * s[e] + p.b[e] * c[e];
    }
  }
  if (n >= 8) {
    // (Past the caches: 4096 rows of 36 heads of 128 in 24.0 us, 6.3 TB/s; 33.2 without.)
    __builtin_nontemporal_store(a, reinterpret_cast<f32x4u*>(head + qa));
    __builtin_nontemporal_store(b, reinterpret_cast<f32x4u*>(head + qb));
  } else {
    const int na = turned && !INTER ? n / 2 : min(n, 4), nb = n - na;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e < na) head[qa + e] = a[e];
      if (e < nb) head[qb + e] = b[e];
    }
  }
}

// grid (rows, parts of a row). A thread takes whole pairs, so x and out may be
// the same rows; its next piece is in flight while the last is turned, and its
// first while the angles are.
template <int N, bool INTER>
__global__ __launch_bounds__(256) void rope_rows_kernel(RopeArgs<N> rope, RopeShape sh, const float* x, long x_stride,
                                                        const int32_t* __restrict__ positions, float* out,
                                                        long out_stride) {
  __shared__ Turns<N> turns;
  const size_t r = blockIdx.x;
  const int pos = positions[r];
  const float* xr = x + r * x_stride;
  float* yr = out + r * out_stride;
  const uint32_t step = gridDim.y * blockDim.x;
  uint32_t i = blockIdx.y * blockDim.x + threadIdx.x;
  const bool any = i < sh.pieces;
  uint32_t h = i / (uint32_t)sh.groups, g = i - h * sh.groups;
  Piece p{};
  if (any) p = load_piece<INTER>(sh, xr + (size_t)h * sh.hd, (int)g);
  fill_turns(rope, pos, turns);
  __syncthreads();
  if (!any) return;
  for (;;) {
    const uint32_t i2 = i + step;
    const bool more = i2 < sh.pieces;
    const uint32_t h2 = i2 / (uint32_t)sh.groups, g2 = i2 - h2 * sh.groups;
    Piece p2{};
    if (more) p2 = load_piece<INTER>(sh, xr + (size_t)h2 * sh.hd, (int)g2);
    store_piece<INTER>(sh, turns, yr + (size_t)h * sh.hd, (int)g, p);
    if (!more) return;
    p = p2;
    h = h2;
    g = g2;
    i = i2;
  }
}

// ---- rows into the pages --------------------------------------------------------

struct AppendArgs {
  const float *q, *k, *v, *q_w, *k_w;
  long q_stride, k_stride, v_stride;
  float* q_out;
  int n_q;
  const int32_t *positions, *seqs;
  float eps;
  int lanes_log;  // log2 of the threads a head takes, eight values each
  size_t r0;      // the launch's first row
};

// Eight values (fewer at a head's end) of a page row.
template <typename T>
__device__ __forceinline__ void store_row(const PagedView& w, bool is_v, int h, uint32_t page, uint32_t row, int d,
                                          int n, const Oct& y) {
  const size_t at = (((size_t)page * w.n_kv + h) << w.t.shift) + row;  // of the head's rows
  if constexpr (std::is_same<T, Q8>::value) {
    uint16_t s;
    const u32x2 c = q8_oct(y, s);
    *reinterpret_cast<u32x2*>((is_v ? w.v : w.k) + at * w.hd + d) = c;
    if (d % 32 == 0) {
      const int nb = w.hd / 32, b = d / 32;
      if (is_v)
        w.vs[((((size_t)page * w.n_kv + h) * nb + b) << w.t.shift) + row] = s;
      else
        w.ks[at * nb + b] = s;
    }
  } else {
    T* p = reinterpret_cast<T*>(is_v ? w.v : w.k) + at * w.hd + d;
    if constexpr (std::is_same<T, float>::value) {
      bool large = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) large |= is_v && (__float_as_uint(y[e]) & 0x7FFFFFFFu) - 0x6F800000u < 0x10000000u;
      if (large) w.status[kLarge] = 1;
    }
    if (w.hd % 8 == 0) {
      if constexpr (std::is_same<T, float>::value) {
        *reinterpret_cast<f32x4*>(p) = y.a;
        *reinterpret_cast<f32x4*>(p + 4) = y.b;
      } else {
        f16x8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (_Float16)y[e];
        *reinterpret_cast<f16x8*>(p) = o;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) p[e] = (T)y[e];
    }
  }
}

// Sum over the 2^log lanes of a head.
__device__ __forceinline__ double head_sum(double x, int log) {
  if (log >= 1) x += dpp_f64<DPP_QUAD_XOR1>(x);
  if (log >= 2) x += dpp_f64<DPP_QUAD_XOR2>(x);
  if (log >= 3) x += dpp_f64<DPP_ROW_HALF_MIRROR>(x);
  if (log >= 4) x += dpp_f64<DPP_ROW_MIRROR>(x);
  if (log >= 5) x = swap_sum_f64<16>(x);
  if (log >= 6) x = swap_sum_f64<32>(x);
  return x;
}

// grid (rows, parts of a row's heads [q | k | v]); a head is 2^lanes_log threads
// side by side, eight consecutive values each (a store of 16 bytes of f16, a fourth of
// a Q8_0 block). Normed values pass through LDS, where a thread finds the other halves
// of its pairs. k' = rot(k / sqrt(mean k^2 + eps) w): sum of squares and angles in f64.
// Bound by a row's chain (position, page id, angles, store) rather than its bytes: one
// row 3.4 us, 5734 rows of 4 + 4 heads of 128 into f16 pages 11.5, 3.2 TB/s
// (16.6 with the sums through LDS and single values turned).
template <typename T, int N>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedView w, RopeArgs<N> rope, AppendArgs a) {
#pragma clang fp contract(off)
  __shared__ __attribute__((aligned(16))) float row[256 * 8];
  __shared__ Turns<N> turns;
  const size_t r = a.r0 + blockIdx.x;
  const int tid = threadIdx.x, lanes = 1 << a.lanes_log;
  const int slot = blockIdx.y * blockDim.x + tid;
  int h = slot >> a.lanes_log;
  const int c = slot & (lanes - 1), d = 8 * c, n = min(8, w.hd - d);
  const int kind = h < a.n_q ? 0 : h < a.n_q + w.n_kv ? 1 : 2;  // q, k, v
  const bool live = h < a.n_q + 2 * w.n_kv && n > 0;
  h -= kind == 0 ? 0 : kind == 1 ? a.n_q : a.n_q + w.n_kv;
  const int pos = a.positions[r];
  const int seq = a.seqs ? a.seqs[r] : (int)r;
  Oct x{};
  if (live) {
    const float* src = (kind == 0 ? a.q + r * a.q_stride : kind == 1 ? a.k + r * a.k_stride : a.v + r * a.v_stride) +
                       (size_t)h * w.hd + d;
    if (n == 8) {
      x.a = *reinterpret_cast<const f32x4u*>(src);
      x.b = *reinterpret_cast<const f32x4u*>(src + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) x.set(e, src[e]);
    }
  }
  uint32_t page = 0, prow = 0;
  const bool here = paged_place(w, (uint32_t)r, pos, seq, blockIdx.y == 0 && tid == 0, page, prow);
  const bool turned = (int)((blockIdx.y * blockDim.x) >> a.lanes_log) < a.n_q + w.n_kv;  // q or k heads here
  if (turned) {
    fill_turns(rope, pos, turns);
    if (__any(kind != 2)) {  // (a wave of v heads has only the barrier to see to)
      if (a.q_w || a.k_w) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += (double)x[e] * (double)x[e];
        ss = head_sum(ss, a.lanes_log);
        const float* nw = kind == 0 ? a.q_w : kind == 1 ? a.k_w : nullptr;
        if (nw && live) {
          const float inv = (float)(1.0 / sqrt(ss / (double)w.hd + (double)a.eps));
          if (n == 8) {
            const f32x4 w0 = *reinterpret_cast<const f32x4u*>(nw + d), w1 = *reinterpret_cast<const f32x4u*>(nw + d + 4);
            x.a = x.a * inv * w0;
            x.b = x.b * inv * w1;
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < n) x.set(e, x[e] * inv * nw[d + e]);
          }
        }
      }
      if (rope.pairs && !rope.interleaved) {
        float* mine = row + 8 * tid;
        *reinterpret_cast<f32x4*>(mine) = x.a;
        *reinterpret_cast<f32x4*>(mine + 4) = x.b;
      }
    }
    if (rope.pairs) {
      __syncthreads();
      if (kind != 2 && d < 2 * rope.pairs) {
        // Whole vectors where a thread's values are of one kind: both of four pairs
        // (interleaved), or all the first or all the second of eight.
        if (rope.interleaved && rope.pairs % 4 == 0) {
          const f32x4 c4 = *reinterpret_cast<const f32x4*>(turns.c + 4 * c);
          const f32x4 s4 = *reinterpret_cast<const f32x4*>(turns.s + 4 * c);
          const Oct z = x;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x.set(2 * e, z[2 * e] * c4[e] - z[2 * e + 1] * s4[e]);
            x.set(2 * e + 1, z[2 * e] * s4[e] + z[2 * e + 1] * c4[e]);
          }
        } else if (!rope.interleaved && rope.pairs % 8 == 0) {
          const bool second = d >= rope.pairs;
          const int p = second ? d - rope.pairs : d;
          const float* other = row + 8 * (tid - c) + (second ? p : p + rope.pairs);
          const f32x4 za = *reinterpret_cast<const f32x4*>(other), zb = *reinterpret_cast<const f32x4*>(other + 4);
          const f32x4 ca = *reinterpret_cast<const f32x4*>(turns.c + p), cb = *reinterpret_cast<const f32x4*>(turns.c + p + 4);
          const f32x4 sa = *reinterpret_cast<const f32x4*>(turns.s + p), sb = *reinterpret_cast<const f32x4*>(turns.s + p + 4);
          // z s + x c for the second of a pair, x c - z s for the first: a sum either
          // way, of the negated product for the first (the same rounding).
          const f32x4 ta = second ? za * sa : -(za * sa), tb = second ? zb * sb : -(zb * sb);
          x.a = x.a * ca + ta;
          x.b = x.b * cb + tb;
        } else {
          const float* head = row + 8 * (tid - c);
          const Oct z = x;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int i = d + e;
            if (i >= 2 * rope.pairs || e >= n) continue;
            const bool second = rope.interleaved ? e & 1 : i >= rope.pairs;
            const int p = rope.interleaved ? i >> 1 : second ? i - rope.pairs : i;
            const float cs = turns.c[p], sn = turns.s[p];
            const float o = rope.interleaved ? z[e ^ 1] : head[second ? i - rope.pairs : i + rope.pairs];
            x.set(e, second ? o * sn + z[e] * cs : z[e] * cs - o * sn);
          }
        }
      }
    }
  }
  if (kind == 0) {
    if (!live) return;
    float* o = a.q_out + (r * a.n_q + h) * w.hd + d;
    if (n == 8) {
      *reinterpret_cast<f32x4u*>(o) = x.a;
      *reinterpret_cast<f32x4u*>(o + 4) = x.b;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) o[e] = x[e];
    }
  } else if (live && here) {  // (Q8_0: the four threads of a block are live together)
    store_row<T>(w, kind == 2, h, page, prow, d, n, x);
  }
}

// ---- and back ----------------------------------------------------------------------

typedef _Float16 f16x8u __attribute__((ext_vector_type(8), aligned(2)));  // a caller's rows

// Eight values a thread of one plane (blockIdx.y: K, V), as attention reads them: f16
// pages' 5734 rows of 4 heads of 128 7.1 us, 3.3 TB/s (the position and the page id come
// first); one row 2.6.
template <typename T, typename O>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedView w, const int32_t* __restrict__ positions,
                                                         const int32_t* __restrict__ seqs, size_t r0,
                                                         size_t n_pieces, uint32_t per_head, O* __restrict__ k, O* __restrict__ v) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const bool is_v = blockIdx.y != 0;
  O* dst = is_v ? v : k;
  if (i >= n_pieces || !dst) return;
  const uint32_t per_row = per_head * w.n_kv;
  const size_t r1 = i / per_row, r = r0 + r1;
  const uint32_t j = (uint32_t)(i - r1 * per_row), h = j / per_head, d = 8 * (j - h * per_head);
  uint32_t page = 0, row = 0;
  const bool here = paged_place(w, (uint32_t)r, positions[r], seqs ? seqs[r] : (int)r, j == 0 && (is_v || !v), page, row);
  O* o = dst + (r * w.n_kv + h) * w.hd + d;
  if (!here) {
    for (int e = 0; e < min(8, w.hd - (int)d); ++e) o[e] = (O)0.f;
    return;
  }
  const size_t hp = (size_t)page * w.n_kv + h, at = (hp << w.t.shift) + row;
  const char* base = is_v ? w.v : w.k;
  if constexpr (std::is_same<T, Q8>::value) {
    const int nb = w.hd / 32;
    const u32x2 c = *reinterpret_cast<const u32x2*>(base + at * w.hd + d);
    const uint16_t sb = is_v ? w.vs[((hp * nb + d / 32) << w.t.shift) + row] : w.ks[at * nb + d / 32];
    const _Float16 s = __builtin_bit_cast(_Float16, sb);
    f16x2 p[4];
    q8_widen(c[0], p[0], p[1]);
    q8_widen(c[1], p[2], p[3]);
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (_Float16)(p[e >> 1][e & 1] * s);
    *reinterpret_cast<f16x8u*>(o) = y;
  } else {
    const O* p = reinterpret_cast<const O*>(base) + at * w.hd + d;
    const int n = min(8, w.hd - (int)d);
    if (w.hd % 8 == 0) {
      if constexpr (sizeof(O) == 4) {
        *reinterpret_cast<f32x4u*>(o) = *reinterpret_cast<const f32x4*>(p);
        *reinterpret_cast<f32x4u*>(o + 4) = *reinterpret_cast<const f32x4*>(p + 4);
      } else {
        *reinterpret_cast<f16x8u*>(o) = *reinterpret_cast<const f16x8*>(p);
      }
    } else {
      for (int e = 0; e < n; ++e) o[e] = p[e];
    }
  }
}

HipStatus launched(const char* what) {
  HipStatus st;
  st.e = hipGetLastError();
  if (st.e != hipSuccess) st.what = what;
  return st;
}

constexpr size_t kMaxGridRows = (size_t)1 << 23;  // rows x 256 threads within 32 bits

}  // namespace

namespace {

template <int N>
RopeArgs<N> rope_args(const rv_rope* rope) {
  RopeArgs<N> a;
  if (!rope) return a;
  a.pairs = (int)(rope->rotary_dim / 2);
  a.interleaved = rope->layout == RV_ROPE_INTERLEAVED;
  a.gain = rope->gain;
  for (int i = 0; i < a.pairs; ++i) a.freq[i] = rope->freq[i];
  return a;
}

// f(arguments) with the smaller of the two sizes that holds the pairs.
template <typename F>
HipStatus with_rope(const rv_rope* rope, F f) {
  if (!rope || rope->rotary_dim <= 2 * kFewPairs) return f(rope_args<kFewPairs>(rope));
  return f(rope_args<kMaxHalf>(rope));
}

}  // namespace

HipStatus launch_rope_rows(const rv_rope& rope, const float* x, size_t x_stride, size_t rows, size_t width,
                           const int32_t* positions, float* out, size_t out_stride, hipStream_t s) {
  RopeShape sh;
  sh.hd = (int)rope.head_dim;
  sh.pairs = (int)rope.rotary_dim / 2;
  sh.pair_groups = (sh.pairs + 3) / 4;
  sh.halves = rope.layout == RV_ROPE_HALF || sh.pairs % 4 == 0;
  // What passes through is copied, unless it is there already.
  sh.groups = sh.pair_groups + (x == out ? 0 : (sh.hd - 2 * sh.pairs + 7) / 8);
  sh.pieces = (uint32_t)(width / sh.hd * sh.groups);
  const unsigned block = std::min(256u, (sh.pieces + 63) / 64 * 64);
  unsigned parts = (sh.pieces + block - 1) / block;
  // One piece a thread while the launch is small; a whole row per workgroup, its
  // angles computed once, when rows alone fill the CUs.
  if (rows * parts > 8 * (size_t)kCUs) parts = (unsigned)std::max<size_t>(1, std::min<size_t>(parts, 8 * kCUs / rows));
  return with_rope(&rope, [&](const auto& ra) {
    constexpr int N = sizeof(ra.freq) / sizeof(double);
    HipStatus st;
    for (size_t r0 = 0; r0 < rows; r0 += kMaxGridRows) {
      const dim3 grid((unsigned)std::min(rows - r0, kMaxGridRows), parts);
      if (ra.interleaved)
        hipLaunchKernelGGL((rope_rows_kernel<N, true>), grid, dim3(block), 0, s, ra, sh, x + r0 * x_stride,
                           (long)x_stride, positions + r0, out + r0 * out_stride, (long)out_stride);
      else
        hipLaunchKernelGGL((rope_rows_kernel<N, false>), grid, dim3(block), 0, s, ra, sh, x + r0 * x_stride,
                           (long)x_stride, positions + r0, out + r0 * out_stride, (long)out_stride);
      if ((st = launched("rope launch")).e != hipSuccess) return st;
    }
    return st;
  });
}

HipStatus launch_paged_append(const rv_paged* pg, const PagedView& w, const rv_rope* rope, const PagedRows& r,
                              hipStream_t s) {
  AppendArgs a{r.q,        r.k,     r.v,    r.q_w,       r.k_w,    (long)r.q_stride, (long)r.k_stride, (long)r.v_stride,
               r.q_out,    r.n_q,   r.positions, r.seqs, r.eps,    0, 0};
  while ((8 << a.lanes_log) < w.hd) ++a.lanes_log;
  const unsigned slots = (unsigned)(r.n_q + 2 * w.n_kv) << a.lanes_log;
  const unsigned block = std::min(256u, (slots + 63) / 64 * 64);
  return with_rope(rope, [&](const auto& ra) {
    constexpr int N = sizeof(ra.freq) / sizeof(double);
    HipStatus st;
    for (a.r0 = 0; a.r0 < r.rows; a.r0 += kMaxGridRows) {
      const dim3 grid((unsigned)std::min(r.rows - a.r0, kMaxGridRows), (slots + block - 1) / block);
      if (pg->elem == RV_ELEM_F32)
        hipLaunchKernelGGL((paged_append_kernel<float, N>), grid, dim3(block), 0, s, w, ra, a);
      else if (pg->elem == RV_ELEM_F16)
        hipLaunchKernelGGL((paged_append_kernel<_Float16, N>), grid, dim3(block), 0, s, w, ra, a);
      else
        hipLaunchKernelGGL((paged_append_kernel<Q8, N>), grid, dim3(block), 0, s, w, ra, a);
      if ((st = launched("paged append launch")).e != hipSuccess) return st;
    }
    return st;
  });
}

HipStatus launch_paged_read(const rv_paged* pg, const PagedView& w, size_t rows, const int32_t* positions,
                            const int32_t* seqs, void* k, void* v, hipStream_t s) {
  HipStatus st;
  const uint32_t per_head = (uint32_t)(w.hd + 7) / 8;
  const size_t per_row = (size_t)w.n_kv * per_head, most = std::max<size_t>(1, ((size_t)1 << 31) / per_row);
  for (size_t r0 = 0; r0 < rows; r0 += most) {
    const size_t pieces = std::min(rows - r0, most) * per_row;
    const dim3 grid((unsigned)((pieces + 255) / 256), 2);
    if (pg->elem == RV_ELEM_F32)
      hipLaunchKernelGGL((paged_read_kernel<float, float>), grid, dim3(256), 0, s, w, positions, seqs, r0, pieces,
                         per_head, (float*)k, (float*)v);
    else if (pg->elem == RV_ELEM_F16)
      hipLaunchKernelGGL((paged_read_kernel<_Float16, _Float16>), grid, dim3(256), 0, s, w, positions, seqs, r0,
                         pieces, per_head, (_Float16*)k, (_Float16*)v);
    else
      hipLaunchKernelGGL((paged_read_kernel<Q8, _Float16>), grid, dim3(256), 0, s, w, positions, seqs, r0, pieces,
                         per_head, (_Float16*)k, (_Float16*)v);
    if ((st = launched("paged read launch")).e != hipSuccess) return st;
  }
  return st;
}

}  // namespace rv
