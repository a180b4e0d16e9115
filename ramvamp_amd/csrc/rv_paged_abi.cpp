// rv_paged_abi.cpp — the C ABI of include/ramvamp_paged.h: the rotary
// frequencies, the paged cache's life, and the host's checks of its calls. What
// a call reads from device memory its kernels check (rv_paged.hip,
// rv_paged_attn.hip). Nothing is queued before a call's checks have passed.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <new>

#include "rv_paged.hpp"

namespace {

int32_t fail(rv_error* err, int32_t code, uint64_t a = 0, uint64_t b = 0, uint64_t c = 0, uint64_t d = 0,
             const char* what = nullptr) {
  if (err) *err = rv_error{code, a, b, c, d, what};
  return code;
}

int32_t ok(rv_error* err) { return fail(err, RV_OK); }

int32_t null_arg(rv_error* err, const char* what) { return fail(err, RV_ERR_NULL_ARG, 0, 0, 0, 0, what); }

int32_t unsupported(rv_error* err, uint64_t a, const char* what) {
  return fail(err, RV_ERR_UNSUPPORTED, a, 0, 0, 0, what);
}

int32_t hip_fail(rv_error* err, const rv::HipStatus& st) {
  return fail(err, rv::status_code(st.e), (uint64_t)st.e, 0, 0, 0, st.what);
}

int32_t hip_fail(rv_error* err, hipError_t e, const char* what) { return hip_fail(err, rv::HipStatus{e, what}); }

// Makes a device current for the scope of one call.
struct DeviceGuard {
  int prev = -1;
  explicit DeviceGuard(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    if (prev != dev) (void)hipSetDevice(dev);
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && hipGetDevice(&cur) == hipSuccess && cur != prev) (void)hipSetDevice(prev);
  }
};

// A call's scope: the cache's device current, and what it queues behind earlier calls.
struct Queued {
  DeviceGuard dg;
  const hipError_t e;
  explicit Queued(rv_paged* pg) : dg(pg->device), e(pg->order.settle()) {}
};

int32_t check_flags(uint32_t flags, rv_error* err) {
  if (flags & RV_HOST_PTRS) return unsupported(err, flags, "RV_HOST_PTRS (device pointers only)");
  return RV_OK;
}

int32_t check_stride(size_t rows, size_t width, size_t stride, const char* what, rv_error* err) {
  if (rows > 1 && stride < width) return fail(err, RV_PRIM_LENGTH_MISMATCH, width, stride, 0, 0, what);
  return RV_OK;
}

// Bytes from the first to the last value of strided rows of f32.
size_t extent(size_t rows, size_t width, size_t stride) { return ((rows - 1) * stride + width) * sizeof(float); }

// Whether two sets of rows share memory; rows side by side in one buffer (one
// stride) do not.
bool overlap(const float* x, size_t x_stride, const float* y, size_t y_stride, size_t rows, size_t width) {
  if (rows == 0 || width == 0) return false;
  const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
  if (a + extent(rows, width, x_stride) <= b || b + extent(rows, width, y_stride) <= a) return false;
  if (x_stride != y_stride || rows == 1) return true;
  const size_t step = x_stride * sizeof(float), need = width * sizeof(float);
  const size_t apart = (a > b ? a - b : b - a) % step;
  return apart < need || apart + need > step;
}

// Whether `bytes` at p share memory with rows of f32 (with them, not what is between).
bool meets(const void* p, size_t bytes, const float* y, size_t y_stride, size_t rows, size_t width) {
  if (bytes == 0 || rows == 0 || width == 0) return false;
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)y;
  if (a + bytes <= b || b + extent(rows, width, y_stride) <= a) return false;
  if (a < b || rows == 1) return true;
  const size_t step = y_stride * sizeof(float), i = (a - b) / step, in_row = (a - b) % step;
  return in_row < width * sizeof(float) || (i + 1 < rows && in_row + bytes > step);
}

// Bytes of a table from its first id to the last of n sequences.
size_t table_bytes(const rv_page_table& t, size_t n) {
  return n && t.pages ? ((n - 1) * t.stride + t.pages) * sizeof(int32_t) : 0;
}

// As rv_kv_new's geometry, for pages.
int32_t geometry(size_t n_layers, size_t n_kv_heads, size_t head_dim, size_t n_pages, size_t page_rows, int elem,
                 size_t* bytes, rv_error* err) {
  if (elem != RV_ELEM_F16 && elem != RV_ELEM_F32 && elem != RV_ELEM_Q8_0)
    return fail(err, RV_ERR_BAD_ELEM, (uint64_t)elem);
  auto invalid = [&](const char* why) {
    return fail(err, RV_KV_INVALID_DIMS, n_layers, n_kv_heads, head_dim, n_pages, why);
  };
  if (n_layers == 0 || n_kv_heads == 0 || head_dim == 0 || n_pages == 0) return invalid("all dims must be nonzero");
  if (page_rows < 8 || page_rows > 1024 || (page_rows & (page_rows - 1)))
    return invalid("page_rows must be a power of two from 8 to 1024");
  if (head_dim > 512) return unsupported(err, head_dim, "head_dim above 512");
  if (elem == RV_ELEM_Q8_0 && head_dim % 32) return invalid("Q8_0 rows need a head_dim that is a multiple of 32");
  if (n_pages > 0x7FFFFFFFu) return unsupported(err, n_pages, "pages past 2^31 - 1");
  if (n_kv_heads > 65535) return unsupported(err, n_kv_heads, "kv heads past 65535");
  size_t n = n_kv_heads * head_dim;
  if (__builtin_mul_overflow(n, page_rows * n_pages, &n) || __builtin_mul_overflow(n, n_layers, &n))
    return invalid("total size overflows usize");
  const bool q8 = elem == RV_ELEM_Q8_0;
  if (__builtin_mul_overflow(q8 ? n / 32 : n, (size_t)2 * (q8 ? 34 : elem == RV_ELEM_F32 ? 4 : 2), bytes))
    return invalid("total size in bytes overflows usize");
  return RV_OK;
}

rv::HipStatus grow(rv_paged* pg, void** buf, size_t* have, size_t bytes, const char* what) {
  rv::HipStatus st;
  if (bytes <= *have) return st;
  if (rv::capturing(pg->order.stream)) {
    st.e = hipErrorStreamCaptureUnsupported;
    st.what = "workspace growth under graph capture (run a call of this shape uncaptured first)";
    return st;
  }
  const size_t want = std::max(bytes, 2 * *have);
  void* p = nullptr;
  try {
    pg->retired.reserve(pg->retired.size() + 1);
  } catch (const std::bad_alloc&) {
    st.e = hipErrorOutOfMemory;
    st.what = what;
    return st;
  }
  st.e = hipMalloc(&p, want);
  if (st.e != hipSuccess) {
    (void)hipGetLastError();
    st.what = what;
    return st;
  }
  if (*buf) pg->retired.push_back(*buf);
  *buf = p;
  *have = want;
  return st;
}

// What attention needs of the cache; the units it deals are counted in 32 bits.
int32_t ready_attn(rv_paged* pg, const rv_page_table& t, size_t n, size_t n_q, rv::PagedAttnPlan* plan,
                   rv_error* err) {
  *plan = rv::paged_attn_plan(pg, t, n, n_q);
  if (plan->units > 0x7FFFFFFFu)
    return fail(err, RV_ERR_UNSUPPORTED, plan->units, 0, 0, 0, "rows of the tables (128 a unit, for each kv head)");
  rv::HipStatus st = grow(pg, &pg->ws, &pg->ws_bytes, plan->ws_bytes, "hipMalloc workspace");
  const size_t had = pg->ticket_bytes;
  if (st.e == hipSuccess)
    st = grow(pg, (void**)&pg->tickets, &pg->ticket_bytes, plan->ticket_bytes, "hipMalloc tickets");
  if (st.e == hipSuccess && pg->ticket_bytes != had) {
    st.e = hipMemset(pg->tickets, 0, pg->ticket_bytes);
    if (st.e == hipSuccess) st.e = hipDeviceSynchronize();
    if (st.e != hipSuccess) {
      st.what = "clear the tickets";
      pg->ticket_bytes = 0;  // (the next call makes them anew)
    }
  }
  return st.e == hipSuccess ? RV_OK : hip_fail(err, st);
}

int32_t check_layer(const rv_paged* pg, size_t layer, rv_error* err) {
  if (layer >= pg->n_layers) return fail(err, RV_KV_LAYER_OUT_OF_RANGE, layer, pg->n_layers);
  return RV_OK;
}

// The table's shape, for rows that name sequences of it (or are its sequences).
int32_t check_table(const rv_page_table* t, size_t rows, bool by_row, rv_error* err) {
  if (!t) return null_arg(err, "table");
  if (t->n_seqs > 0x7FFFFFFFu || t->pages > 0x7FFFFFFFu)
    return unsupported(err, std::max(t->n_seqs, t->pages), "table past 2^31 - 1");
  if (t->n_seqs > 1 && t->stride < t->pages)
    return fail(err, RV_PRIM_LENGTH_MISMATCH, t->pages, t->stride, 0, 0, "table rows vs their stride");
  size_t n;
  if (t->n_seqs > 1 && (__builtin_mul_overflow(t->stride, t->n_seqs, &n) || n > (SIZE_MAX >> 4)))
    return unsupported(err, t->stride, "table size");
  if (t->n_seqs && t->pages && !t->ids) return null_arg(err, "table ids");
  if (by_row && rows > t->n_seqs)
    return fail(err, RV_PRIM_LENGTH_MISMATCH, t->n_seqs, rows, 0, 0, "sequences of the table vs rows");
  if (rows > 0x7FFFFFFFu) return unsupported(err, rows, "rows past 2^31 - 1");
  return RV_OK;
}

int32_t check_norm(const float* w, size_t len, size_t hd, rv_error* err) {
  if (w && len != hd)
    return fail(err, RV_PRIM_LENGTH_MISMATCH, hd, len, 0, 0, "rmsnorm_in_place: x vs weight");
  return RV_OK;
}

int32_t check_rope(const rv_paged* pg, const rv_rope* rope, rv_error* err) {
  if (rope && rope->head_dim != pg->head_dim)
    return fail(err, RV_PRIM_LENGTH_MISMATCH, pg->head_dim, rope->head_dim, 0, 0, "the cache's head_dim vs the rope's");
  return RV_OK;
}

int32_t finish(hipStream_t s, uint32_t flags, const rv::HipStatus& st, rv_error* err) {
  if (st.e != hipSuccess) return hip_fail(err, st);
  if (flags & RV_SYNC) {
    const hipError_t e = hipStreamSynchronize(s);
    if (e != hipSuccess) return hip_fail(err, e, "hipStreamSynchronize");
  }
  return ok(err);
}

// q_dim's heads and their kv heads.
int32_t check_q(const rv_paged* pg, size_t q_dim, rv_error* err) {
  const size_t hd = pg->head_dim;
  if (q_dim == 0 || q_dim % hd) return fail(err, RV_ATTN_Q_LEN_INDIVISIBLE, q_dim, hd);
  if ((q_dim / hd) % pg->n_kv_heads) return fail(err, RV_ATTN_GQA_GROUP_MISMATCH, q_dim / hd, pg->n_kv_heads);
  if (q_dim / hd > 65535) return unsupported(err, q_dim / hd, "query heads past 65535");
  return RV_OK;
}

constexpr size_t kMaxSeqs = (size_t)1 << 23;

}  // namespace

extern "C" {

// ---- rotary positions ------------------------------------------------------------

int32_t rv_rope_new(size_t head_dim, size_t rotary_dim, uint32_t layout, double theta, uint32_t scaling,
                    double factor, size_t trained_positions, double beta_fast, double beta_slow, rv_rope** out,
                    rv_error* err) {
  if (!out) return null_arg(err, "out");
  if (head_dim == 0 || rotary_dim == 0 || rotary_dim % 2 || rotary_dim > head_dim)
    return fail(err, RV_PRIM_INVALID_HEAD_DIM, rotary_dim, head_dim);
  if (head_dim > 512) return unsupported(err, head_dim, "head_dim above 512");
  if (layout != RV_ROPE_HALF && layout != RV_ROPE_INTERLEAVED) return unsupported(err, layout, "rope layout");
  if (scaling > RV_ROPE_YARN) return unsupported(err, scaling, "rope scaling");
  const bool yarn = scaling == RV_ROPE_YARN;
  if (!std::isfinite(theta) || theta <= (yarn ? 1.0 : 0.0)) return unsupported(err, 0, "rope theta");
  if (scaling != RV_ROPE_UNSCALED && !(std::isfinite(factor) && factor >= 1.0))
    return unsupported(err, 0, "rope factor (finite, at least 1)");
  if (scaling == RV_ROPE_NTK && rotary_dim <= 2) return unsupported(err, rotary_dim, "NTK of a rotary_dim of 2");
  if (yarn && trained_positions == 0) return unsupported(err, 0, "trained_positions of 0");
  if (yarn && !(std::isfinite(beta_fast) && beta_slow > 0.0 && beta_fast > beta_slow))
    return unsupported(err, 0, "rope betas (finite, beta_fast > beta_slow > 0)");
  rv_rope* r = new (std::nothrow) rv_rope();
  if (!r) return fail(err, RV_ERR_HIP, (uint64_t)hipErrorOutOfMemory, 0, 0, 0, "host allocation");
  r->head_dim = head_dim;
  r->rotary_dim = rotary_dim;
  r->layout = layout;
  const double dim = (double)rotary_dim;
  const double base = scaling == RV_ROPE_NTK ? theta * pow(factor, dim / (dim - 2.0)) : theta;
  double lo = 0.0, hi = 0.0;
  if (yarn) {
    auto pair = [&](double turns) {
      return dim * log((double)trained_positions / (2.0 * M_PI * turns)) / (2.0 * log(theta));
    };
    lo = std::max(floor(pair(beta_fast)), 0.0);
    hi = std::min(ceil(pair(beta_slow)), dim - 1.0);
    r->gain = 0.1 * log(factor) + 1.0;
  }
  for (size_t i = 0; i < rotary_dim / 2; ++i) {
    double f = pow(base, -2.0 * (double)i / dim);
    if (scaling == RV_ROPE_LINEAR) f /= factor;
    if (yarn) {
      const double ramp = std::min(std::max(((double)i - lo) / std::max(hi - lo, 0.001), 0.0), 1.0);
      f = f * (1.0 - ramp) + f / factor * ramp;
    }
    if (!std::isfinite(base) || !std::isfinite(f * 0x1p31)) {
      delete r;
      return unsupported(err, 0, "rope theta (angles past the range of f64)");
    }
    r->freq[i] = f;
  }
  *out = r;
  return ok(err);
}

void rv_rope_free(rv_rope* rope) { delete rope; }

int32_t rv_rope_frequencies(const rv_rope* rope, double* freq, size_t n, double* gain, rv_error* err) {
  if (!rope || !freq) return null_arg(err, !rope ? "rope" : "freq");
  if (n != rope->rotary_dim / 2)
    return fail(err, RV_PRIM_LENGTH_MISMATCH, rope->rotary_dim / 2, n, 0, 0, "pairs vs freq");
  for (size_t i = 0; i < n; ++i) freq[i] = rope->freq[i];
  if (gain) *gain = rope->gain;
  return ok(err);
}

int32_t rv_rope_rows(const rv_rope* rope, const float* x, size_t x_stride, size_t rows, size_t width,
                     const int32_t* positions, float* out, size_t out_stride, void* stream, uint32_t flags,
                     rv_error* err) {
  if (!rope) return null_arg(err, "rope");
  int32_t rc = check_flags(flags, err);
  if (rc) return rc;
  const size_t hd = rope->head_dim;
  if (width == 0 || width % hd) return fail(err, RV_ATTN_Q_LEN_INDIVISIBLE, width, hd);
  if (width > 0x7FFFFFFFu) return unsupported(err, width, "row width past 2^31 - 1");
  if ((rc = check_stride(rows, width, x_stride, "x rows vs their stride", err))) return rc;
  if ((rc = check_stride(rows, width, out_stride, "out rows vs their stride", err))) return rc;
  if (rows == 0) return finish((hipStream_t)stream, flags, {}, err);
  if (!x || !positions || !out) return null_arg(err, !x ? "x" : !positions ? "positions" : "out");
  if (rows == 1) x_stride = out_stride = width;
  if (!(x == out && x_stride == out_stride) && overlap(x, x_stride, out, out_stride, rows, width))
    return unsupported(err, 0, "out overlaps x");
  if (meets(positions, rows * sizeof(int32_t), out, out_stride, rows, width))
    return unsupported(err, 0, "out overlaps positions");
  const rv::HipStatus st = rv::launch_rope_rows(*rope, x, x_stride, rows, width, positions, out,
                                                out_stride, (hipStream_t)stream);
  return finish((hipStream_t)stream, flags, st, err);
}

// ---- the cache ---------------------------------------------------------------------

int32_t rv_paged_projected_bytes(size_t n_layers, size_t n_kv_heads, size_t head_dim, size_t n_pages,
                                 size_t page_rows, rv_elem elem, uint64_t* bytes, rv_error* err) {
  if (!bytes) return null_arg(err, "bytes");
  size_t b;
  const int32_t rc = geometry(n_layers, n_kv_heads, head_dim, n_pages, page_rows, elem, &b, err);
  if (rc) return rc;
  *bytes = b;
  return ok(err);
}

int32_t rv_paged_new(size_t n_layers, size_t n_kv_heads, size_t head_dim, size_t n_pages, size_t page_rows,
                     rv_elem elem, int device, rv_paged** out, rv_error* err) {
  if (!out) return null_arg(err, "out");
  size_t bytes;
  int32_t rc = geometry(n_layers, n_kv_heads, head_dim, n_pages, page_rows, elem, &bytes, err);
  if (rc) return rc;
  int devices = 0;
  hipError_t e = hipGetDeviceCount(&devices);
  if (e == hipSuccess && (device < 0 || device >= devices)) e = hipErrorInvalidDevice;
  if (e != hipSuccess) return hip_fail(err, e, "device");
  rv_paged* pg = new (std::nothrow) rv_paged();
  if (!pg) return fail(err, RV_ERR_HIP, (uint64_t)hipErrorOutOfMemory, 0, 0, 0, "host allocation");
  pg->n_layers = n_layers;
  pg->n_kv_heads = n_kv_heads;
  pg->head_dim = head_dim;
  pg->n_pages = n_pages;
  pg->page_rows = page_rows;
  pg->kv_dim = n_kv_heads * head_dim;
  pg->elem = elem;
  pg->device = device;
  DeviceGuard dg(device);
  e = hipMalloc(&pg->k, pg->plane_bytes());
  if (e == hipSuccess) e = hipMalloc(&pg->v, pg->plane_bytes());
  if (e == hipSuccess) e = hipMemset(pg->k, 0, pg->plane_bytes());
  if (e == hipSuccess) e = hipMemset(pg->v, 0, pg->plane_bytes());
  if (e == hipSuccess) e = hipMalloc((void**)&pg->status, 256);
  if (e == hipSuccess) e = hipMemset(pg->status, 0, 256);
  if (e == hipSuccess) e = hipDeviceSynchronize();
  if (e == hipSuccess) pg->xcd_ok = rv::xcd_dealing_ok(device);
  if (e != hipSuccess) {
    rv_paged_free(pg);
    (void)hipGetLastError();  // (reported here, not by the next call to ask)
    return hip_fail(err, e, "hipMalloc pages");
  }
  *out = pg;
  return ok(err);
}

void rv_paged_free(rv_paged* pg) {
  if (!pg) return;
  {
    DeviceGuard dg(pg->device);
    (void)hipDeviceSynchronize();
    for (void* p : {pg->k, pg->v, (void*)pg->status, pg->ws, (void*)pg->tickets, (void*)pg->qbuf})
      if (p) (void)hipFree(p);
    for (void* p : pg->retired) (void)hipFree(p);
    if (pg->order.api.ev) (void)hipEventDestroy(pg->order.api.ev);
  }
  delete pg;
}

int32_t rv_paged_set_tuning(rv_paged* pg, int32_t knob, int64_t value, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  if (knob != RV_TUNE_PAGED_JOIN) return unsupported(err, (uint64_t)knob, "tuning knob");
  if (value != 0 && value != 2) return unsupported(err, (uint64_t)value, "RV_TUNE_PAGED_JOIN (0 or 2)");
  pg->tune_join = value;
  return ok(err);
}

int32_t rv_paged_set_stream(rv_paged* pg, void* hip_stream, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  const hipStream_t next = (hipStream_t)hip_stream;
  if (next == pg->order.stream) return ok(err);
  DeviceGuard dg(pg->device);
  const hipError_t e = pg->order.move_to(next);
  return e == hipSuccess ? ok(err) : hip_fail(err, e, "stream hand-over");
}

int32_t rv_paged_synchronize(rv_paged* pg, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  const Queued queued(pg);
  if (queued.e != hipSuccess) return hip_fail(err, queued.e, "stream hand-over");
  return finish(pg->order.stream, RV_SYNC, {}, err);
}

int32_t rv_paged_device_status(rv_paged* pg, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  const Queued queued(pg);
  if (queued.e != hipSuccess) return hip_fail(err, queued.e, "stream hand-over");
  if (rv::capturing(pg->order.stream)) return unsupported(err, 0, "device status under graph capture");
  uint32_t w[5] = {};
  hipError_t e = hipStreamSynchronize(pg->order.stream);
  if (e == hipSuccess) e = hipMemcpy(w, pg->status, sizeof(w), hipMemcpyDeviceToHost);
  if (e != hipSuccess) return hip_fail(err, e, "read the device status");
  if (w[0] == 0) return ok(err);
  e = hipMemset(pg->status, 0, sizeof(w));
  if (e == hipSuccess) e = hipDeviceSynchronize();
  if (e != hipSuccess) return hip_fail(err, e, "clear the device status");
  return fail(err, (int32_t)w[0], w[1], w[2], w[3], w[4], "refused on the device");
}

// ---- rows ----------------------------------------------------------------------------

int32_t rv_paged_append_rows(rv_paged* pg, size_t layer, const rv_rope* rope, const float* k, size_t k_stride,
                             const float* v, size_t v_stride, size_t rows, const int32_t* positions,
                             const int32_t* seqs, const rv_page_table* table, const float* k_norm_w,
                             size_t k_norm_len, float eps, uint32_t flags, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  int32_t rc = check_flags(flags, err);
  if (rc) return rc;
  if ((rc = check_layer(pg, layer, err))) return rc;
  if ((rc = check_rope(pg, rope, err))) return rc;
  if ((rc = check_norm(k_norm_w, k_norm_len, pg->head_dim, err))) return rc;
  if ((rc = check_stride(rows, pg->kv_dim, k_stride, "k rows vs their stride", err))) return rc;
  if ((rc = check_stride(rows, pg->kv_dim, v_stride, "v rows vs their stride", err))) return rc;
  if ((rc = check_table(table, rows, !seqs, err))) return rc;
  const Queued queued(pg);
  if (queued.e != hipSuccess) return hip_fail(err, queued.e, "stream hand-over");
  if (rows == 0) return finish(pg->order.stream, flags, {}, err);
  if (!k || !v || !positions) return null_arg(err, !k ? "k" : !v ? "v" : "positions");
  rv::PagedRows r{};
  r.k = k;
  r.k_stride = k_stride;
  r.v = v;
  r.v_stride = v_stride;
  r.rows = rows;
  r.positions = positions;
  r.seqs = seqs;
  r.k_w = k_norm_w;
  r.eps = eps;
  return finish(pg->order.stream, flags,
                rv::launch_paged_append(pg, rv::paged_view(pg, layer, *table), rope, r, pg->order.stream), err);
}

int32_t rv_paged_read_rows(rv_paged* pg, size_t layer, size_t rows, const int32_t* positions, const int32_t* seqs,
                           const rv_page_table* table, void* k, void* v, uint32_t flags, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  int32_t rc = check_flags(flags, err);
  if (rc) return rc;
  if ((rc = check_layer(pg, layer, err))) return rc;
  if ((rc = check_table(table, rows, !seqs, err))) return rc;
  const Queued queued(pg);
  if (queued.e != hipSuccess) return hip_fail(err, queued.e, "stream hand-over");
  if (rows == 0 || (!k && !v)) return finish(pg->order.stream, flags, {}, err);
  if (!positions) return null_arg(err, "positions");
  const size_t es = pg->elem == RV_ELEM_F32 ? 4 : 2, n = rows * pg->kv_dim * es;
  const auto apart = [&](const void* x, const void* y, size_t bytes) {
    return !x || !y || (uintptr_t)x + n <= (uintptr_t)y || (uintptr_t)y + bytes <= (uintptr_t)x;
  };
  if (!apart(k, v, n)) return unsupported(err, 0, "k overlaps v");
  const size_t ids = table_bytes(*table, seqs ? table->n_seqs : rows);
  for (const void* x : {k, v})
    if (!apart(x, positions, rows * sizeof(int32_t)) || !apart(x, seqs, rows * sizeof(int32_t)) || (ids && !apart(x, table->ids, ids)))
      return unsupported(err, 0, "k or v overlaps positions, seqs or the table");
  return finish(pg->order.stream, flags,
                rv::launch_paged_read(pg, rv::paged_view(pg, layer, *table), rows, positions, seqs, k, v, pg->order.stream),
                err);
}

// ---- attention -----------------------------------------------------------------------

int32_t rv_paged_attention(rv_paged* pg, size_t layer, const float* q, size_t q_stride, size_t n_seqs, size_t q_dim,
                           const rv_page_table* table, const int32_t* lens, float scale, float* out,
                           size_t out_stride, uint32_t flags, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  int32_t rc = check_flags(flags, err);
  if (rc) return rc;
  if ((rc = check_q(pg, q_dim, err))) return rc;
  if ((rc = check_layer(pg, layer, err))) return rc;
  if ((rc = check_stride(n_seqs, q_dim, q_stride, "q rows vs their stride", err))) return rc;
  if ((rc = check_stride(n_seqs, q_dim, out_stride, "out rows vs their stride", err))) return rc;
  if ((rc = check_table(table, n_seqs, true, err))) return rc;
  if (n_seqs > kMaxSeqs) return unsupported(err, n_seqs, "sequences past 2^23");
  const Queued queued(pg);
  if (queued.e != hipSuccess) return hip_fail(err, queued.e, "stream hand-over");
  if (n_seqs == 0) return finish(pg->order.stream, flags, {}, err);
  if (!q || !lens || !out) return null_arg(err, !q ? "q" : !lens ? "lens" : "out");
  if (n_seqs == 1) q_stride = out_stride = q_dim;
  if (overlap(q, q_stride, out, out_stride, n_seqs, q_dim)) return unsupported(err, 0, "out overlaps q");
  if (meets(lens, n_seqs * sizeof(int32_t), out, out_stride, n_seqs, q_dim) ||
      meets(table->ids, table_bytes(*table, n_seqs), out, out_stride, n_seqs, q_dim))
    return unsupported(err, 0, "out overlaps lens or the table");
  const size_t n_q = q_dim / pg->head_dim;
  rv::PagedAttnPlan plan;
  if ((rc = ready_attn(pg, *table, n_seqs, n_q, &plan, err))) return rc;
  const rv::PagedAttn a{q, q_stride, n_seqs, (int)n_q, lens, false, scale, out, out_stride};
  return finish(pg->order.stream, flags, rv::launch_paged_attn(pg, rv::paged_view(pg, layer, *table), a, plan, pg->order.stream),
                err);
}

int32_t rv_paged_decode_step(rv_paged* pg, size_t layer, const rv_rope* rope, const float* q, size_t q_stride,
                             const float* k, size_t k_stride, const float* v, size_t v_stride, size_t n_seqs,
                             size_t q_dim, const float* q_norm_w, size_t q_norm_len, const float* k_norm_w,
                             size_t k_norm_len, float eps, const rv_page_table* table, const int32_t* positions,
                             float scale, float* out, size_t out_stride, uint32_t flags, rv_error* err) {
  if (!pg) return null_arg(err, "pg");
  int32_t rc = check_flags(flags, err);
  if (rc) return rc;
  if ((rc = check_rope(pg, rope, err))) return rc;
  if ((rc = check_norm(q_norm_w, q_norm_len, pg->head_dim, err))) return rc;
  if ((rc = check_norm(k_norm_w, k_norm_len, pg->head_dim, err))) return rc;
  if ((rc = check_q(pg, q_dim, err))) return rc;
  if ((rc = check_layer(pg, layer, err))) return rc;
  if ((rc = check_stride(n_seqs, q_dim, q_stride, "q rows vs their stride", err))) return rc;
  if ((rc = check_stride(n_seqs, pg->kv_dim, k_stride, "k rows vs their stride", err))) return rc;
  if ((rc = check_stride(n_seqs, pg->kv_dim, v_stride, "v rows vs their stride", err))) return rc;
  if ((rc = check_stride(n_seqs, q_dim, out_stride, "out rows vs their stride", err))) return rc;
  if ((rc = check_table(table, n_seqs, true, err))) return rc;
  if (n_seqs > kMaxSeqs) return unsupported(err, n_seqs, "sequences past 2^23");
  const Queued queued(pg);
  if (queued.e != hipSuccess) return hip_fail(err, queued.e, "stream hand-over");
  if (n_seqs == 0) return finish(pg->order.stream, flags, {}, err);
  for (const auto& p : {std::pair<const void*, const char*>{q, "q"}, {k, "k"}, {v, "v"}, {positions, "positions"}, {out, "out"}})
    if (!p.first) return null_arg(err, p.second);
  // (q, k and v are read, and q copied, before the first output is written.)
  if (meets(positions, n_seqs * sizeof(int32_t), out, out_stride, n_seqs, q_dim) ||
      meets(table->ids, table_bytes(*table, n_seqs), out, out_stride, n_seqs, q_dim))
    return unsupported(err, 0, "out overlaps positions or the table");
  const size_t n_q = q_dim / pg->head_dim;
  rv::PagedAttnPlan plan;
  if ((rc = ready_attn(pg, *table, n_seqs, n_q, &plan, err))) return rc;
  rv::HipStatus st = grow(pg, (void**)&pg->qbuf, &pg->qbuf_bytes, n_seqs * q_dim * sizeof(float), "hipMalloc q buffer");
  if (st.e != hipSuccess) return hip_fail(err, st);
  rv::PagedRows r{};
  r.q = q;
  r.q_stride = q_stride;
  r.n_q = (int)n_q;
  r.q_out = pg->qbuf;
  r.q_w = q_norm_w;
  r.k = k;
  r.k_stride = k_stride;
  r.v = v;
  r.v_stride = v_stride;
  r.rows = n_seqs;
  r.positions = positions;
  r.k_w = k_norm_w;
  r.eps = eps;
  const rv::PagedView w = rv::paged_view(pg, layer, *table);
  st = rv::launch_paged_append(pg, w, rope, r, pg->order.stream);
  if (st.e == hipSuccess) {
    const rv::PagedAttn a{pg->qbuf, q_dim, n_seqs, (int)n_q, positions, true, scale, out, out_stride};
    st = rv::launch_paged_attn(pg, w, a, plan, pg->order.stream);
  }
  return finish(pg->order.stream, flags, st, err);
}

}  // extern "C"
