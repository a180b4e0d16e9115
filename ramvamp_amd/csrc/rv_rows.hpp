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

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kMaxScale = 515.5f;  // 127 * 515.5 rounds to 65472; the next f16, 516, to infinity

struct Oct {
  f32x4 a, b;
  __device__ __forceinline__ float operator[](int e) const { return e < 4 ? a[e] : b[e - 4]; }
  __device__ __forceinline__ void set(int e, float x) {
    if (e < 4)
      a[e] = x;
    else
      b[e - 4] = x;
  }
};

// Eight values of a block held by 4 lanes: their codes (+ 128) and the scale.
__device__ __forceinline__ u32x2 q8_oct(const Oct& x, uint16_t& scale) {
#pragma clang fp contract(off)
  // The largest magnitude's bits order as integers, and a NaN or an infinity has
  // larger bits than any finite value.
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR1, 0xF, 0xF, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR2, 0xF, 0xF, false));
  const bool finite = m < 0x7F800000u;
  float d = finite ? __uint_as_float(m) / 127.f : 0.f;
  if (d >= 515.75f) d = kMaxScale;  // (halfway to 516, the even one of the two)
  // Below the smallest normal float the reciprocal may overflow; the f16 scale
  // is zero there and the codes stand for nothing.
  const float id = d >= 1.17549435e-38f ? 1.f / d : 0.f;
  scale = finite ? __builtin_bit_cast(uint16_t, (_Float16)d) : (uint16_t)0x7E00;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    // Half away from zero: the conversion truncates, and adding the float below
    // one half rounds up to the next whole number from exactly one half on.
    const float y = __builtin_amdgcn_fmed3f(x[e] * id, -127.f, 127.f);
    const int c = finite ? (int)(y + __builtin_copysignf(0x1.fffffep-2f, y)) : 0;
    w[e >> 2] |= (uint32_t)(c + 128) << (8 * (e & 3));
  }
  return u32x2{w[0], w[1]};
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
