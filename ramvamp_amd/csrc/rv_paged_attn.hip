// rv_paged_attn.hip — attention of one new token of each sequence of a batch
// over its pages.
//
// o = sum_t p_t v_t / sum_t p_t, p_t = exp(scale * (q . k_t) - m), in one pass over
// the rows with the running maximum m.
//
// The lengths are on the device and ragged, so the work is dealt there: a unit is
// kUnitRows positions of one item (a sequence's kv head, or a part of its query
// heads), the units of the batch in order are cut into equal ranges, one a
// workgroup, and every workgroup finds its own range by a prefix sum over the
// lengths. An item inside one range is finished there; one that is cut leaves a
// partial (maximum, sum, weighted sum of v) per range, at most two a workgroup
// (its first item and its last), and a second launch joins them in order, so
// that results do not depend on which workgroup ends first.
#include "rv_paged.hpp"

#include <algorithm>

namespace rv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const float* q;
  long q_stride;
  const int32_t* lens;
  uint32_t n;
  bool step;
  int group, cols, blocks;  // query heads per kv head, per item, items per kv head
  float scale;
  float* out;
  long out_stride;
  long* plan;   // [0] units a range, [1 + s] units before sequence s
  float* part;  // [workgroup][2][cols * (hd + 2)]: maxima, sums, rows
};

// Rows sequence s attends; negative: refused.
__device__ __forceinline__ long seq_rows(const PagedView& w, const AttnArgs& a, uint32_t s, bool say) {
  const int len = a.lens[s];
  const long rows = attended_rows(w.t, len, a.step);
  if (rows < 0 && say)
    paged_refuse(w, RV_PAGED_POSITION_OUT_OF_RANGE, s, (uint32_t)len, (uint32_t)min(table_rows(w.t), 0xFFFFFFFFl));
  return rows;
}

// Sum over the workgroup, and of the threads before this one.
__device__ __forceinline__ long block_scan(long x, long& before, long* sums) {
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  long inc = x;
  for (int o = 1; o < 64; o <<= 1) {
    const long y = __shfl_up(inc, o, 64);
    if (lane >= o) inc += y;
  }
  __syncthreads();
  if (lane == 63) sums[wv] = inc;
  __syncthreads();
  long total = 0, skip = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < wv) skip += sums[i];
    total += sums[i];
  }
  before = skip + inc - x;
  return total;
}

template <typename T>
__device__ __forceinline__ float paged_value(const PagedView& w, bool is_v, size_t hp, uint32_t row, int d) {
  const size_t at = (hp << w.t.shift) + row;
  const char* base = is_v ? w.v : w.k;
  if constexpr (std::is_same<T, Q8>::value) {
    const int nb = w.hd / 32;
    return q8_value((uint8_t)base[at * w.hd + d],
                    is_v ? w.vs[((hp * nb + d / 32) << w.t.shift) + row] : w.ks[at * nb + d / 32]);
  } else {
    return (float)reinterpret_cast<const T*>(base)[at * w.hd + d];
  }
}

// Any head width: one query head an item, a wave one position at a time, the
// head's values over its lanes.
template <typename T>
struct Plain {
  static constexpr int kPer = kMaxHalf * 2 / 64;
  struct Shared {
    float o[4][kMaxHalf * 2];
    float m[4], l[4];
  };
  // Positions [p0, p1) of sequence s, kv head h, query head qh (of the whole).
  static __device__ __forceinline__ void segment(const PagedView& w, const AttnArgs& a, Shared& sh, uint32_t s, int h,
                                                 int qh, int, long p0, long p1, bool whole, float* part) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const float* q = a.q + s * a.q_stride + (long)qh * w.hd;
    const float scale = a.scale * kLog2e;
    float x[kPer], o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int d = lane + 64 * j;
      x[j] = d < w.hd ? q[d] : 0.f;
      o[j] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (long p = p0 + wv; p < p1; p += 4) {
      uint32_t page = (uint32_t)w.t.ids[(long)s * w.t.stride + (p >> w.t.shift)];
      if (page >= w.t.n_pages) {
        if (lane == 0) paged_refuse(w, RV_PAGED_PAGE_OUT_OF_RANGE, s, page, w.t.n_pages);
        l = NAN;
        continue;
      }
      const size_t hp = (size_t)page * w.n_kv + h;
      const uint32_t row = (uint32_t)p & ((1u << w.t.shift) - 1);
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int d = lane + 64 * j;
        if (d < w.hd) dot += x[j] * paged_value<T>(w, false, hp, row, d);
      }
      dot = swap_sum<32>(swap_sum<16>(group_sum<16>(dot)));
      const float y = dot * scale, mn = fmaxf(m, y);
      const float c = mn == -INFINITY ? 1.f : exp2f(m - mn), e = mn == -INFINITY ? 0.f : exp2f(y - mn);
      m = mn;
      l = l * c + e;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int d = lane + 64 * j;
        if (d < w.hd) o[j] = o[j] * c + e * paged_value<T>(w, true, hp, row, d);
      }
    }
    __syncthreads();
    if (lane == 0) sh.m[wv] = m, sh.l[wv] = l;
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh.o[wv][lane + 64 * j] = o[j];
    __syncthreads();
    const float top = fmaxf(fmaxf(sh.m[0], sh.m[1]), fmaxf(sh.m[2], sh.m[3]));
    float f[4], sum = 0.f;
    for (int i = 0; i < 4; ++i) {
      f[i] = sh.m[i] == -INFINITY ? (sh.l[i] == 0.f ? 0.f : 1.f) : exp2f(sh.m[i] - top);
      sum += f[i] * sh.l[i];
    }
    for (int d = threadIdx.x; d < w.hd; d += 256) {
      float y = 0.f;
      for (int i = 0; i < 4; ++i)
        if (f[i] != 0.f) y += f[i] * sh.o[i][d];
      if (whole)
        a.out[s * a.out_stride + (long)qh * w.hd + d] = y / sum;
      else
        part[2 + d] = y;
    }
    if (!whole && threadIdx.x == 0) part[0] = top, part[1] = sum;
  }
};

template <typename Inner>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedView w, AttnArgs a) {
  __shared__ typename Inner::Shared sh;
  __shared__ long sums[4];
  __shared__ long found[2];
  const int tid = threadIdx.x;
  const bool planner = blockIdx.x == 0;
  const long items = (long)w.n_kv * a.blocks;
  long mine = 0, before;
  for (uint32_t s = tid; s < a.n; s += 256) mine += units_of(seq_rows(w, a, s, planner)) * items;
  const long total = block_scan(mine, before, sums);
  const long per = units_per_range(total, gridDim.x);
  const long start = blockIdx.x * per, end = min(total, start + per);
  if (tid == 0) found[0] = -1;
  long base = 0;
  for (uint32_t s0 = 0; s0 < a.n; s0 += 256) {
    const uint32_t s = s0 + tid;
    const long u = s < a.n ? units_of(seq_rows(w, a, s, false)) * items : 0;
    const long sum = block_scan(u, before, sums);
    if (planner && s < a.n) a.plan[1 + s] = base + before;
    if (start >= base + before && start < base + before + u) found[0] = s, found[1] = base + before;
    base += sum;
    if (!planner && start < base) break;
  }
  if (planner && tid == 0) a.plan[0] = per;
  if (start >= end) return;
  __syncthreads();
  walk_units(
      (uint32_t)found[0], start - found[1], start, end, items, [&](uint32_t s) { return seq_rows(w, a, s, false); },
      [&](uint32_t s, long rows, long item, long u0, long u1, long at) {
        const int h = (int)(item / a.blocks), c0 = (int)(item % a.blocks) * a.cols;
        float* part = a.part + ((long)blockIdx.x * 2 + partial_of(blockIdx.x, per, at)) * a.cols * (w.hd + 2);
        Inner::segment(w, a, sh, s, h, h * a.group + c0, min(a.cols, a.group - c0), u0 * kUnitRows,
                       min(rows, u1 * kUnitRows), u0 == 0 && u1 == units_of(rows), part);
      });
}

// grid (sequences, query heads): joins the partials of items that were cut; a
// sequence without rows gets zeros, a refused one NaN.
__global__ __launch_bounds__(128) void paged_join_kernel(PagedView w, AttnArgs a) {
  const uint32_t s = blockIdx.x, qh = blockIdx.y;
  float* out = a.out + s * a.out_stride + (long)qh * w.hd;
  const long rows = seq_rows(w, a, s, false), units = units_of(rows);
  if (rows <= 0) {
    for (int d = threadIdx.x; d < w.hd; d += 128) out[d] = rows < 0 ? NAN : 0.f;
    return;
  }
  const long per = a.plan[0], h = qh / a.group, g = qh % a.group;
  const long start = a.plan[1 + s] + (h * a.blocks + g / a.cols) * units, end = start + units;
  const long w0 = start / per, w1 = (end - 1) / per;
  if (w0 == w1) return;
  const int c = (int)(g % a.cols);
  const long step = (long)a.cols * (w.hd + 2);
  auto part = [&](long i) { return a.part + (i * 2 + partial_of(i, per, start)) * step; };
  float top = -INFINITY;
  for (long i = w0; i <= w1; ++i) top = fmaxf(top, part(i)[c]);
  float sum = 0.f;
  for (long i = w0; i <= w1; ++i) {
    const float m = part(i)[c], l = part(i)[a.cols + c];
    sum += m == -INFINITY ? l : exp2f(m - top) * l;
  }
  for (int d = threadIdx.x; d < w.hd; d += 128) {
    float y = 0.f;
    for (long i = w0; i <= w1; ++i) {
      const float m = part(i)[c];
      if (m != -INFINITY) y += exp2f(m - top) * part(i)[2 * a.cols + (long)c * w.hd + d];
    }
    out[d] = y / sum;
  }
}

// Workgroups that deal the work of any lengths.
unsigned ranges(const rv_paged*, size_t n, size_t n_q) {
  return (unsigned)std::min<size_t>(2048, std::max<size_t>(2 * kCUs, n * n_q));
}

size_t plan_bytes(size_t n) { return ((n + 1) * sizeof(long) + 255) / 256 * 256; }

}  // namespace

size_t paged_attn_ws(const rv_paged* pg, size_t n, size_t n_q) {
  return plan_bytes(n) + (size_t)ranges(pg, n, n_q) * 2 * (pg->head_dim + 2) * sizeof(float);
}

HipStatus launch_paged_attn(const rv_paged* pg, const PagedView& w, const PagedAttn& p, hipStream_t s) {
  AttnArgs a{};
  a.q = p.q;
  a.q_stride = (long)p.q_stride;
  a.lens = p.lens;
  a.n = (uint32_t)p.n;
  a.step = p.step;
  a.group = p.n_q / w.n_kv;
  a.cols = 1;
  a.blocks = (a.group + a.cols - 1) / a.cols;
  a.scale = p.scale;
  a.out = p.out;
  a.out_stride = (long)p.out_stride;
  a.plan = (long*)pg->ws;
  a.part = (float*)((char*)pg->ws + plan_bytes(p.n));
  const dim3 grid(ranges(pg, p.n, p.n_q));
  HipStatus st;
  if (pg->elem == RV_ELEM_F32)
    hipLaunchKernelGGL(paged_attn_kernel<Plain<float>>, grid, dim3(256), 0, s, w, a);
  else if (pg->elem == RV_ELEM_F16)
    hipLaunchKernelGGL(paged_attn_kernel<Plain<_Float16>>, grid, dim3(256), 0, s, w, a);
  else
    hipLaunchKernelGGL(paged_attn_kernel<Plain<Q8>>, grid, dim3(256), 0, s, w, a);
  st.e = hipGetLastError();
  if (st.e != hipSuccess) {
    st.what = "paged attention launch";
    return st;
  }
  hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)p.n, (unsigned)p.n_q), dim3(128), 0, s, w, a);
  st.e = hipGetLastError();
  if (st.e != hipSuccess) st.what = "paged join launch";
  return st;
}

}  // namespace rv
