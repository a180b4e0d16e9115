// rv_paged.hpp — the paged cache's host state, what its kernels share
// (rv_paged.hip: rotation, rows in and out; rv_paged_attn.hip: attention), and
// their launchers. Not part of the public ABI.
//
// A plane of a layer is [n_pages][n_kv_heads][page_rows][head_dim]: a kv head's
// rows of a page are one contiguous range, so that a tile of its positions is
// read in whole lines. A Q8_0 plane holds codes (+ 128) so, and the f16 scales
// apart from them, K's [page][head][row][block], V's [page][head][block][row]
// (an MFMA operand of K holds one position a lane, one of V consecutive
// positions: each finds its scales side by side).
#pragma once

#include <math.h>

#include <vector>

#include "../../include/ramvamp_paged.h"
#include "rv_pages.hpp"
#include "rv_rows.hpp"

struct rv_rope {
  size_t head_dim = 0, rotary_dim = 0;
  uint32_t layout = 0;
  double gain = 1.0;
  double freq[rv::kMaxHalf] = {};
};

struct rv_paged {
  size_t n_layers = 0, n_kv_heads = 0, head_dim = 0, n_pages = 0, page_rows = 0, kv_dim = 0;
  int elem = RV_ELEM_F16;
  int device = 0;
  bool xcd_ok = false;  // xcd_dealing_ok of the device
  int64_t tune_join = 0;
  void* k = nullptr;
  void* v = nullptr;
  rv::StreamOrder<rv::HipStreams> order;  // order.stream: what calls are queued on
  unsigned* status = nullptr;  // [0] code, [1] layer, [2] row, [3] what it read, [4] the bound, [kLarge]
  // Grown on first need; a replaced buffer is kept until the cache is freed,
  // since a graph captured earlier may still address it.
  void* ws = nullptr;  // attention's partials
  size_t ws_bytes = 0;
  unsigned* tickets = nullptr;  // and their tickets, behind the words that say whose turn it is
  size_t ticket_bytes = 0;
  float* qbuf = nullptr;  // a step's normed and rotated q rows
  size_t qbuf_bytes = 0;
  std::vector<void*> retired;

  size_t elem_size() const { return elem == RV_ELEM_F32 ? 4 : elem == RV_ELEM_F16 ? 2 : 1; }
  size_t layer_elems() const { return n_pages * page_rows * kv_dim; }
  size_t plane_bytes() const {
    return n_layers * layer_elems() * elem_size() + (elem == RV_ELEM_Q8_0 ? n_layers * layer_elems() / 32 * 2 : 0);
  }
};

namespace rv {

// One layer's pages as the kernels take them.
struct PagedView {
  char* k;
  char* v;
  uint16_t* ks;  // Q8_0: scales
  uint16_t* vs;
  int hd, n_kv;
  uint32_t layer;
  unsigned* status;
  Pages t;
};
PagedView paged_view(const rv_paged* pg, size_t layer, const rv_page_table& t);

// The rotation as the kernels take it: frequencies by value, of up to N pairs (the
// most that a head has would make every launch's arguments 2 KiB).
template <int N>
struct RopeArgs {
  int pairs = 0;  // 0: none
  int interleaved = 0;
  double gain = 1.0;
  double freq[N];
};
constexpr int kFewPairs = 64;

// The word beside the status that says whether f32 pages have ever held a finite value of
// V of 2^96 or more: where none has, no sum of up to 2^31 of them passes the floats' range.
constexpr int kLarge = 16;

// Records a refusal: the first since the last read stays.
__device__ __forceinline__ void paged_refuse(const PagedView& w, uint32_t code, uint32_t row, uint32_t got,
                                             uint32_t bound) {
  if (atomicCAS(w.status, 0u, code) == 0u) {
    w.status[1] = w.layer;
    w.status[2] = row;
    w.status[3] = got;
    w.status[4] = bound;
  }
}

// Row r's place: its page and the row inside it; false for padding and for what
// is refused (`say`: this thread records it).
__device__ __forceinline__ bool paged_place(const PagedView& w, uint32_t r, int pos, int seq, bool say,
                                            uint32_t& page, uint32_t& row) {
  uint32_t got = 0;
  const Place p = place_of(w.t, pos, seq, page, row, got);
  if (p <= kPadding) return p == kHere;
  if (say) {
    if (p == kNoSequence)
      paged_refuse(w, RV_PAGED_SEQUENCE_OUT_OF_RANGE, r, got, w.t.n_seqs);
    else if (p == kNoPosition)
      paged_refuse(w, RV_PAGED_POSITION_OUT_OF_RANGE, r, got, (uint32_t)min(table_rows(w.t), 0xFFFFFFFFl));
    else
      paged_refuse(w, RV_PAGED_PAGE_OUT_OF_RANGE, r, got, w.t.n_pages);
  }
  return false;
}

HipStatus launch_rope_rows(const rv_rope& rope, const float* x, size_t x_stride, size_t rows, size_t width,
                           const int32_t* positions, float* out, size_t out_stride, hipStream_t s);
// k and v rows into the pages and, with n_q heads a row, q rows normed and
// rotated into q_out (contiguous).
struct PagedRows {
  const float* q = nullptr;
  size_t q_stride = 0;
  int n_q = 0;
  float* q_out = nullptr;
  const float* q_w = nullptr;
  const float* k;
  size_t k_stride;
  const float* v;
  size_t v_stride;
  size_t rows;
  const int32_t* positions;
  const int32_t* seqs;
  const float* k_w;
  float eps;
};
HipStatus launch_paged_append(const rv_paged* pg, const PagedView& w, const rv_rope* rope, const PagedRows& r,
                              hipStream_t s);
HipStatus launch_paged_read(const rv_paged* pg, const PagedView& w, size_t rows, const int32_t* positions,
                            const int32_t* seqs, void* k, void* v, hipStream_t s);

// Attention over rows 0 .. lens[i] of each sequence (a step: and row lens[i]).
struct PagedAttn {
  const float* q;
  size_t q_stride;
  size_t n;    // sequences
  int n_q;     // query heads
  const int32_t* lens;
  bool step;
  float scale;
  float* out;
  size_t out_stride;
};
struct PagedAttnPlan {
  size_t units;  // of work at most, by what the tables can hold
  size_t ws_bytes, tickets, ticket_bytes;
};
PagedAttnPlan paged_attn_plan(const rv_paged* pg, const rv_page_table& t, size_t n, size_t n_q);
HipStatus launch_paged_attn(const rv_paged* pg, const PagedView& w, const PagedAttn& a, const PagedAttnPlan& plan,
                            hipStream_t s);

}  // namespace rv
