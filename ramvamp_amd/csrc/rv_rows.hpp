// rv_rows.hpp — what the Q8_0 cache's kernels (rv_q8.hip) and the attention of
// many query columns over one range of rows (rv_rows.hip) share: where a
// layer's rows are, and how an element type's values are read.
//
// A Q8_0 plane keeps, per (layer, kv head), the rows' codes contiguous
// ([capacity, padded][head_dim], one byte each, code + 128), so a tile of
// positions is one contiguous range, and the scales (f16) apart from them: K's
// per row ([capacity][head_dim / 32]), V's per block ([head_dim / 32][capacity]).
// An MFMA operand of K holds one position per lane, one of V consecutive
// positions per lane, and so each finds its scales side by side. The capacity
// is padded to kQ8Pad rows, which makes every whole tile addressable.
//
// The value a reader sees is f16(scale * code): the product rounded once to
// f16, so that it is a matrix instruction's operand as it stands and all
// readers (the attention kernels, the row reads) agree on it bit for bit. The
// rounding is at most 2^-11 of the value where the code itself is up to
// 1/254 of the block's largest value off.
#pragma once

#include "rv_device.hpp"
#include "rv_internal.hpp"

namespace rv {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Q8 {};  // the element tag of a Q8_0 plane

// One layer's rows of one cache, and the step to the next layer.
struct KvView {
  const char* k = nullptr;
  const char* v = nullptr;
  const uint16_t* ks = nullptr;  // Q8_0: scales
  const uint16_t* vs = nullptr;
  size_t layer_bytes = 0;   // of one plane (Q8_0: its codes)
  size_t layer_scales = 0;  // Q8_0: scales of one plane
  long kv_dim = 0;
  long rows = 0;  // rows a layer has room for (Q8_0: padded)
};

inline KvView kv_view(const rv_kv* kv, size_t layer) {
  KvView w;
  w.k = kv->k_layer(layer);
  w.v = kv->v_layer(layer);
  w.layer_bytes = kv->layer_bytes();
  w.kv_dim = (long)kv->kv_dim;
  w.rows = (long)kv->row_cap();
  if (kv->elem == RV_ELEM_Q8_0) {
    w.layer_scales = kv->layer_scales();
    w.ks = kv->k_scales(layer);
    w.vs = kv->v_scales(layer);
  }
  return w;
}

// f16 codes - 128 of four code bytes of one row: 0x6400 | code is 1024 + code.
__device__ __forceinline__ void q8_widen(uint32_t w, f16x2& a, f16x2& b) {
  const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
  a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
  b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
}

__device__ __forceinline__ float q8_value(uint8_t code, uint16_t scale) {
  return (float)((_Float16)(float)((int)code - 128) * __builtin_bit_cast(_Float16, scale));
}

// Element `d` of kv head `h` at position `t`, as the readers see it.
template <typename T, bool V>
__device__ __forceinline__ float kv_value(const KvView& w, int hd, int h, long t, int d) {
  if constexpr (std::is_same<T, Q8>::value) {
    const size_t row = (size_t)h * w.rows + t;
    const int nb = hd / 32;
    const uint16_t s = V ? w.vs[((size_t)h * nb + d / 32) * w.rows + t] : w.ks[row * nb + d / 32];
    return q8_value((uint8_t)(V ? w.v : w.k)[row * hd + d], s);
  } else {
    return (float)reinterpret_cast<const T*>(V ? w.v : w.k)[(size_t)t * w.kv_dim + (size_t)h * hd + d];
  }
}

}  // namespace rv
