// rv_q8.hip — rows into a cache and back: the Q8_0 quantization of appended
// rows, the QK-RMSNorm + RoPE prologue of a cache whose rows are not written by
// rv_prologue.hip (Q8_0 planes, and one row to each of many layers), and the
// row reads.
//
// A block is 32 consecutive values of one head's row (quantize_row_q8_0,
// kernels/quants/quantize.rs:37-55): d = amax / 127, code = round(x * (1 / d))
// half away from zero, d stored in f16; all in f32, so the bits are the
// reference's. Two cases it has no answer for: a block whose scale times 127
// would pass f16's range takes the largest scale that does not (515.5), its
// larger values saturating at code 127; a block that holds an infinity or a
// NaN gets a NaN scale, so that its 32 values all read as NaN (a code cannot
// carry one).
//
// Bound by bytes, 4 in and 34/32 out per value, as long as a thread's share of a
// block is large enough to spread the block's own work (two divisions, the
// scale's rounding) over it: eight values a thread, four lanes a block (the
// maximum over them is two DPP steps). 4096 rows of 512, both planes: 16.8 MB in
// and 4.5 out in 6.0 us (3.5 TB/s; vector instructions are 60 % of the cycles),
// where four values a thread and roundf took 8.8; the rows read back, 4.5 in and
// 16.8 out, in 6.9 (3.1 TB/s, mostly stores).
#include "rv_rows.hpp"

#include <algorithm>

namespace rv {
namespace {

struct NoLens {};
struct EachLens {
  uint32_t len[kMaxEach];
};

// RowDst as the kernels take it.
struct DstArgs {
  size_t layer_bytes, layer_scales;  // from one row's layer to the next (0 unless each)
  long row0, pos0;
  const uint32_t* d_pos;
  uint32_t max_pos;
  uint32_t* status;
  uint32_t layer;
};

// Quantizes eight values [d, d + 8) of kv head h and stores them at row t of the
// layer `w` (+ its offsets). The 4 lanes that hold a block call it together.
template <bool V>
__device__ __forceinline__ void store_oct(const KvView& w, size_t lb, size_t ls, int hd, int h, long t, int d,
                                          const Oct& x) {
  uint16_t s;
  const u32x2 c = q8_oct(x, s);
  const size_t row = (size_t)h * w.rows + t;
  *reinterpret_cast<u32x2*>(const_cast<char*>(V ? w.v : w.k) + lb + row * hd + d) = c;
  if (d % 32 == 0) {
    const int nb = hd / 32, b = d / 32;
    if (V)
      const_cast<uint16_t*>(w.vs)[ls + ((size_t)h * nb + b) * w.rows + t] = s;
    else
      const_cast<uint16_t*>(w.ks)[ls + row * nb + b] = s;
  }
}

// Eight consecutive values a thread, of one plane (blockIdx.y: K, V), into a Q8_0
// cache.
template <bool EACH>
__global__ __launch_bounds__(256) void append_q8_kernel(KvView w, DstArgs a, const float* __restrict__ k,
                                                        const float* __restrict__ v, uint32_t n_octs, int hd,
                                                        std::conditional_t<EACH, EachLens, NoLens> lens) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n_octs) return;  // (the four lanes of a block together)
  const bool is_v = blockIdx.y != 0;
  const f32x4u* src = reinterpret_cast<const f32x4u*>((is_v ? v : k) + 8 * (size_t)i);  // (rows are contiguous)
  const Oct x{__builtin_nontemporal_load(src), __builtin_nontemporal_load(src + 1)};
  const uint32_t per_row = (uint32_t)w.kv_dim / 8;
  const uint32_t r = i / per_row, j = 8 * (i - r * per_row), h = j / (uint32_t)hd, d = j - h * hd;
  long t;
  if constexpr (EACH)
    t = lens.len[r];
  else
    t = a.row0 + r;
  const size_t lb = (size_t)r * a.layer_bytes, ls = (size_t)r * a.layer_scales;
  if (is_v)
    store_oct<true>(w, lb, ls, hd, h, t, d, x);
  else
    store_oct<false>(w, lb, ls, hd, h, t, d, x);
}

// One row to each layer of an f16 or f32 cache: one thread per value.
template <typename T>
__global__ __launch_bounds__(256) void append_each_kernel(KvView w, DstArgs a, const float* __restrict__ k,
                                                          const float* __restrict__ v, int rows, EachLens lens) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  const int r = (int)(i / w.kv_dim), j = (int)(i % w.kv_dim);
  if (r >= rows) return;
  const bool is_v = blockIdx.y != 0;
  const float x = (is_v ? v : k)[(size_t)r * w.kv_dim + j];
  const long t = lens.len[r];
  T* p = reinterpret_cast<T*>(const_cast<char*>(is_v ? w.v : w.k) + (size_t)r * a.layer_bytes) + (size_t)t * w.kv_dim + j;
  if constexpr (std::is_same<T, float>::value)
    *p = x;
  else
    *p = f32_to_f16_bits(x);
}

constexpr int kMaxHd = 512;

// grid (rows, q heads + k heads + v heads), one wave each. Lane l owns the
// rotation's pairs (i, i + half), i = l + 64 p; the f32 operations are
// norm.rs:18-26 and rope.rs:31-45's, one rounding each, the mean of squares
// and the angles in f64 (as rv_prologue.hip's). k and v heads of a Q8_0 cache pass
// through LDS to the store's order, eight consecutive values a lane.
template <typename T, bool EACH>
__global__ __launch_bounds__(64) void prologue_dst_kernel(KvView w, DstArgs a, const float* __restrict__ q,
                                                          float* __restrict__ q_out, int n_q,
                                                          const float* __restrict__ k, const float* __restrict__ v,
                                                          int n_kv, int hd, const float* __restrict__ q_w,
                                                          const float* __restrict__ k_w, float eps, InvFreq inv,
                                                          std::conditional_t<EACH, EachLens, NoLens> lens) {
#pragma clang fp contract(off)
  __shared__ __attribute__((aligned(16))) float row[kMaxHd];
  constexpr int NP = kMaxHd / 2 / 64;
  const int r = blockIdx.x, lane = threadIdx.x, half = hd / 2;
  int s = blockIdx.y;
  long t = a.row0 + r, pos = a.pos0 + r;
  if constexpr (EACH) {
    t = lens.len[r];
    pos = a.pos0 + lens.len[r];
  } else if (a.d_pos) {
    const uint32_t p = *a.d_pos;
    if (p > a.max_pos) {
      if (s == 0 && lane == 0 && a.status[0] == 0) {
        a.status[1] = a.layer;
        a.status[2] = p;
        a.status[3] = a.max_pos + 1;
        a.status[0] = RV_KV_CAPACITY_EXCEEDED;
      }
      return;
    }
    t = pos = (long)p;
  }
  const bool is_q = s < n_q, is_v = s >= n_q + n_kv;
  const int h = is_q ? s : is_v ? s - n_q - n_kv : s - n_q;
  const float* x = is_q ? q + ((size_t)r * n_q + h) * hd : (is_v ? v : k) + ((size_t)r * n_kv + h) * hd;
  float x0[NP], x1[NP];
  double ss = 0.0;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int i = lane + 64 * p;
    x0[p] = i < half ? x[i] : 0.f;
    x1[p] = i < half ? x[i + half] : 0.f;
    ss += (double)x0[p] * (double)x0[p] + (double)x1[p] * (double)x1[p];
  }
  float y0[NP], y1[NP];
  if (!is_v) {
    ss = wave_sum_f64(ss);
    const float inv_rms = (float)(1.0 / sqrt(ss / (double)hd + (double)eps));
    const float* nw = is_q ? q_w : k_w;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int i = lane + 64 * p;
      y0[p] = y1[p] = 0.f;
      if (i >= half) continue;
      double sd, cd;
      sincos((double)pos * inv.f[i], &sd, &cd);
      const float sn = (float)sd, cs = (float)cd;
      const float a0 = x0[p] * inv_rms * nw[i], a1 = x1[p] * inv_rms * nw[i + half];
      y0[p] = a0 * cs - a1 * sn;
      y1[p] = a0 * sn + a1 * cs;
    }
  } else {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      y0[p] = x0[p];
      y1[p] = x1[p];
    }
  }
  if (is_q) {
    float* d = q_out + ((size_t)r * n_q + h) * hd;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int i = lane + 64 * p;
      if (i >= half) continue;
      d[i] = y0[p];
      d[i + half] = y1[p];
    }
    return;
  }
  const size_t lb = (size_t)r * a.layer_bytes, ls = (size_t)r * a.layer_scales;
  if constexpr (std::is_same<T, Q8>::value) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int i = lane + 64 * p;
      if (i >= half) continue;
      row[i] = y0[p];
      row[i + half] = y1[p];
    }
    __syncthreads();
    // Whole groups of 4 lanes are past the row's end together (hd % 32 == 0).
    const int d = 8 * lane;
    if (d < hd) {
      const f32x4* y = reinterpret_cast<const f32x4*>(row + d);
      const Oct x{y[0], y[1]};
      if (is_v)
        store_oct<true>(w, lb, ls, hd, h, t, d, x);
      else
        store_oct<false>(w, lb, ls, hd, h, t, d, x);
    }
  } else {
    T* dst = reinterpret_cast<T*>(const_cast<char*>(is_v ? w.v : w.k) + lb) + (size_t)t * w.kv_dim + (size_t)h * hd;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int i = lane + 64 * p;
      if (i >= half) continue;
      if constexpr (std::is_same<T, float>::value) {
        dst[i] = y0[p];
        dst[i + half] = y1[p];
      } else {
        dst[i] = f32_to_f16_bits(y0[p]);
        dst[i + half] = f32_to_f16_bits(y1[p]);
      }
    }
  }
}

// Rows [pos, pos + ..) of one plane (blockIdx.y: K, V) as f32, W values a thread.
template <typename T, int W>
__global__ __launch_bounds__(256) void read_rows_kernel(KvView w, int hd, long pos, uint32_t n_pieces,
                                                        float* __restrict__ k, float* __restrict__ v) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  const bool is_v = blockIdx.y != 0;
  float* dst = is_v ? v : k;
  if (i >= n_pieces || !dst) return;
  const uint32_t per_row = (uint32_t)w.kv_dim / W;
  const uint32_t r = i / per_row, j = (i - r * per_row) * W, h = j / (uint32_t)hd, d = j - h * hd;
  const long t = pos + r;
  float x[W];
  if constexpr (std::is_same<T, Q8>::value) {
    static_assert(W == 8, "pieces inside a block");
    const int nb = hd / 32;
    const size_t row = (size_t)h * w.rows + t;
    const u32x2 c = *reinterpret_cast<const u32x2*>((is_v ? w.v : w.k) + row * hd + d);
    const uint16_t sb = is_v ? w.vs[((size_t)h * nb + d / 32) * w.rows + t] : w.ks[row * nb + d / 32];
    const _Float16 s = __builtin_bit_cast(_Float16, sb);
    f16x2 p[4];
    q8_widen(c[0], p[0], p[1]);
    q8_widen(c[1], p[2], p[3]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)(_Float16)(p[e >> 1][e & 1] * s);
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e)
      x[e] = is_v ? kv_value<T, true>(w, hd, h, t, d + e) : kv_value<T, false>(w, hd, h, t, d + e);
  }
  float* o = dst + (size_t)i * W;
  if constexpr (W >= 4) {
#pragma unroll
    for (int e = 0; e < W; e += 4)
      *reinterpret_cast<f32x4u*>(o + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
  } else {
    *o = x[0];
  }
}

// One Q8_0 row in ggml's block_q8_0 order, 34 bytes a block.
__global__ __launch_bounds__(256) void read_blocks_kernel(KvView w, int hd, int plane_v, long pos,
                                                          uint8_t* __restrict__ dst) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= (int)w.kv_dim) return;
  const int h = i / hd, d = i % hd, nb = hd / 32;
  const size_t row = (size_t)h * w.rows + pos;
  const uint8_t c = (uint8_t)(plane_v ? w.v : w.k)[row * hd + d];
  uint8_t* blk = dst + (size_t)(i / 32) * 34;
  blk[2 + i % 32] = (uint8_t)(c - 128);
  if (i % 32 == 0) {
    const uint16_t s = plane_v ? w.vs[((size_t)h * nb + d / 32) * w.rows + pos] : w.ks[row * nb + d / 32];
    blk[0] = (uint8_t)s;
    blk[1] = (uint8_t)(s >> 8);
  }
}

DstArgs dst_args(const RowDst& d, const KvView& w) {
  DstArgs a{};
  if (d.each_n) {
    a.layer_bytes = w.layer_bytes;
    a.layer_scales = w.layer_scales;
  }
  a.row0 = d.row0;
  a.pos0 = d.pos0;
  a.d_pos = d.d_pos;
  a.max_pos = d.max_pos;
  a.status = d.status;
  a.layer = (uint32_t)d.layer;
  return a;
}

EachLens each_lens(const RowDst& d) {
  EachLens e;
  for (int i = 0; i < kMaxEach; ++i) e.len[i] = d.len[i];
  return e;
}

HipStatus launched(const char* what) {
  HipStatus st;
  st.e = hipGetLastError();
  if (st.e != hipSuccess) st.what = what;
  return st;
}

unsigned blocks_of(size_t threads) { return (unsigned)((threads + 255) / 256); }

// Rows a launch takes: the kernels count its pieces in 32 bits.
size_t rows_at_once(size_t kv_dim) { return std::max<size_t>(1, ((size_t)1 << 30) / kv_dim); }

}  // namespace

HipStatus launch_append_dst(const rv_kv* kv, const RowDst& dst, const float* k, const float* v, size_t rows,
                            hipStream_t s) {
  if (rows == 0) return HipStatus{};
  const KvView w = kv_view(kv, dst.layer);
  DstArgs a = dst_args(dst, w);
  const int hd = (int)kv->head_dim;
  const dim3 block(256);
  if (kv->elem == RV_ELEM_Q8_0 && !dst.each_n) {
    for (size_t r0 = 0, n; r0 < rows; r0 += n) {
      n = std::min(rows - r0, rows_at_once(kv->kv_dim));
      const size_t octs = n * kv->kv_dim / 8;
      hipLaunchKernelGGL(append_q8_kernel<false>, dim3(blocks_of(octs), 2), block, 0, s, w, a, k + r0 * kv->kv_dim,
                         v + r0 * kv->kv_dim, (uint32_t)octs, hd, NoLens{});
      a.row0 += (long)n;
    }
    return launched("append launch");
  }
  const size_t octs = rows * kv->kv_dim / 8;  // (at most kMaxEach rows)
  const dim3 vals(blocks_of(rows * kv->kv_dim), 2);
  if (kv->elem == RV_ELEM_Q8_0)
    hipLaunchKernelGGL(append_q8_kernel<true>, dim3(blocks_of(octs), 2), block, 0, s, w, a, k, v, (uint32_t)octs, hd,
                       each_lens(dst));
  else if (kv->elem == RV_ELEM_F32)
    hipLaunchKernelGGL(append_each_kernel<float>, vals, block, 0, s, w, a, k, v, (int)rows, each_lens(dst));
  else
    hipLaunchKernelGGL(append_each_kernel<uint16_t>, vals, block, 0, s, w, a, k, v, (int)rows, each_lens(dst));
  return launched("append launch");
}

HipStatus launch_prologue_dst(const rv_kv* kv, const RowDst& dst, const float* q, float* q_out, size_t n_q,
                              const float* k, const float* v, size_t rows, const float* q_w, const float* k_w,
                              float eps, const InvFreq& inv, hipStream_t s) {
  if (rows == 0) return HipStatus{};
  const KvView w = kv_view(kv, dst.layer);
  const DstArgs a = dst_args(dst, w);
  const int hd = (int)kv->head_dim, n_kv = (int)kv->n_kv_heads;
  const dim3 grid((unsigned)rows, (unsigned)(n_q + 2 * n_kv));
#define RV_DST(T, EACH, LENS)                                                                                      \
  hipLaunchKernelGGL((prologue_dst_kernel<T, EACH>), grid, dim3(64), 0, s, w, a, q, q_out, (int)n_q, k, v, n_kv, hd, \
                     q_w, k_w, eps, inv, LENS)
  if (kv->elem == RV_ELEM_Q8_0) {
    if (dst.each_n)
      RV_DST(Q8, true, each_lens(dst));
    else
      RV_DST(Q8, false, NoLens{});
  } else if (kv->elem == RV_ELEM_F32) {
    RV_DST(float, true, each_lens(dst));
  } else {
    RV_DST(uint16_t, true, each_lens(dst));
  }
#undef RV_DST
  return launched("prologue launch");
}

HipStatus launch_read_rows(const rv_kv* kv, size_t layer, size_t pos, size_t rows, float* k, float* v, hipStream_t s) {
  const KvView w = kv_view(kv, layer);
  const int hd = (int)kv->head_dim;
  const bool four = hd % 4 == 0;
  for (size_t r0 = 0, n; r0 < rows; r0 += n) {
    n = std::min(rows - r0, rows_at_once(kv->kv_dim));
    const size_t pieces = n * kv->kv_dim / (kv->elem == RV_ELEM_Q8_0 ? 8 : four ? 4 : 1);
    const dim3 grid(blocks_of(pieces), 2), block(256);
    float *dk = k ? k + r0 * kv->kv_dim : nullptr, *dv = v ? v + r0 * kv->kv_dim : nullptr;
#define RV_READ(T, W)                                                                                            \
  hipLaunchKernelGGL((read_rows_kernel<T, W>), grid, block, 0, s, w, hd, (long)(pos + r0), (uint32_t)pieces, dk, dv)
    if (kv->elem == RV_ELEM_Q8_0)
      RV_READ(Q8, 8);
    else if (kv->elem == RV_ELEM_F32 && four)
      RV_READ(float, 4);
    else if (kv->elem == RV_ELEM_F32)
      RV_READ(float, 1);
    else if (four)
      RV_READ(_Float16, 4);
    else
      RV_READ(_Float16, 1);
#undef RV_READ
  }
  return launched("read rows launch");
}

HipStatus launch_read_blocks(const rv_kv* kv, int plane_v, size_t layer, size_t pos, uint8_t* dst, hipStream_t s) {
  hipLaunchKernelGGL(read_blocks_kernel, dim3(blocks_of(kv->kv_dim)), dim3(256), 0, s, kv_view(kv, layer),
                     (int)kv->head_dim, plane_v, (long)pos, dst);
  return launched("read blocks launch");
}

}  // namespace rv
