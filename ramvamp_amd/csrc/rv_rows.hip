// rv_rows.hip — attention of many query columns over one range of rows.
//
// A column is one query head of one query row; a kv head's columns all read
// the same K and V rows. That covers a Q8_0 cache's decode (the group's heads
// of one row), a chunk over it (each row sees start + r + 1 positions), and
// the decode of a batch of sequences that share a prefix (every sequence's
// heads over the prefix, then each sequence's over its own rows).
//
//   o[c] = sum_t p[c][t] v[t] / sum_t p[c][t],  p[c][t] = 2^(q'[c] . k[t] - m[c])
//
// with q' = q * scale * log2(e) and m a base that follows the running maximum. K and V are f16
// matrix operands as stored (Q8_0: f16(scale * code); f32 planes: hi + lo
// halves); q' and p are split into f16 hi + lo halves whose products are
// summed in f32, which keeps fp32-equivalent products: a column over a position
// of 128 dims is 1024 operations (f32 planes 1536), and K and V are read once for
// all columns of an item. One token is bound by those bytes or, up to some
// thousand positions, by the launch's own latencies; from about 100 columns a kv
// head on by the matrix and vector instructions.
#include "rv_rows.hpp"

#include <algorithm>
#include <cfloat>

namespace rv {
namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // as a caller's rows may be

constexpr int kD = 128;
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are taken relative to a base kUp below the running maximum (it
// cancels in o / l), which moves when a score passes it by more than kUp + kSlack:
// they stay at or below 2^15, inside f16, and the lo half of a small one, which
// shares f16's last bit of 2^-24, still holds 2^-36 of the largest.
constexpr float kSlack = 4.f, kUp = 11.f;
// An f32 sum drops the terms below 2^-24 of it, all of them where one row's weight
// towers over the others' (as the first token's often does): 2^-28 a row, 16 rows
// a term. So after this many rows a wave's sums of o and l join those that it has
// put aside and are begun again: what is dropped stays below 2^-15 (wide) and 2^-18
// (narrow) of the weight, however long the split. A wide item's sums go
// through memory (128 KiB out and in; 4096 rows at 131000 14.9 -> 15.1 ms), a narrow
// one's through the LDS that its waves meet in.
constexpr int kWalkWide = 8192, kWalkNarrow = 32 * 32;
constexpr int kFold = 16;  // splits of a kv head that the launch folds itself

struct NoLens {};
struct TailLens {
  uint32_t len[kMaxEach];
};

struct RowsArgs {
  KvView main, tail;      // at the call's layers
  const float* q;
  float* out;             // written when there is one slot in all
  // Partials, a 16-column block's (narrow and tail items) or a 32-column
  // block's (wide items) rows in the order of its wave's registers, so that
  // stores and the merge's loads are whole lines: [slot][block][16 bytes i][64
  // lanes]. ml: base and sum by [slot][column].
  float* part;
  float* ml;
  f32x4* aside;           // wide main items longer than kWalkWide: [item][wave][17 x 16 bytes][64 lanes]
  unsigned* tickets;      // narrow main items fold in the launch: one per kv head, 128 bytes apart
  size_t slot_floats;     // of part, from one main slot to the next
  size_t t_base, t_slot_floats;  // of part: the first tail slot, from one to the next
  const uint32_t* d_pos;  // positions from device memory
  int rows, n_q_heads, group, kv_lo, n_heads;
  int positions, start;   // limit of row r: causal ? start + r + 1 : positions
  int causal;
  int n_cb, n_splits, split_len;           // main items: column blocks x splits x kv heads
  int t_cb, t_splits, t_split_len;         // tail items per sequence and kv head
  int main_items;
  int single;             // one slot: write out
  float qscale;
};

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// ---- a tile of 32 positions in LDS ------------------------------------------------
// Fragments of the 32x32x16 product's A operand, 1 KiB each, lane l's 16 bytes
// side by side. K: fragment c (dims 16 c ..), lane (position, half h) holds
// dims 16 c + 8 h .. + 7. V: fragment (dt, s), lane (dim of 32 dt .., h) holds
// the positions whose scores the C layout gives lane half h for registers
// 8 s .. 8 s + 7: 16 s + 4 h + {0..3}, then + 8. Lane slots are permuted
// within eights so that a staging store's lanes fall on all banks.
constexpr int kFragB = 1024;
constexpr int kTileB = 8 * kFragB;  // one plane of 32 positions

__device__ __forceinline__ int k_slot(int pos, int h) { return (pos ^ (4 * h)) + 32 * h; }
__device__ __forceinline__ int v_slot(int dt, int dim, int h) { return (dim ^ (((dt & 1) << 2) | (dim >> 3))) + 32 * h; }

template <typename T>
struct Lo {
  static constexpr bool value = std::is_same<T, float>::value;  // planes with a lo half in LDS
};

template <typename T>
constexpr int stage_bytes(int positions) {
  return positions / 32 * 2 * kTileB * (Lo<T>::value ? 2 : 1);
}

// ---- the range of f32 planes ----------------------------------------------------------
// hi + lo f16 halves hold a value to 2^-22 of itself between 2^-3 and 2^15, and
// to 2^-25 below. Rows computed together are scaled by a power of two that keeps
// their largest magnitude in [2^9, 2^15), so that any finite values keep 2^-22 of
// themselves or 2^-34 of the largest: K's per tile, undone on the scores; V's by a
// running exponent that follows the largest value seen, the outputs so far scaled
// along.
__device__ __forceinline__ float wave_max(float x) { return swap_max<32>(swap_max<16>(group_max<16>(x))); }
__device__ __forceinline__ uint32_t uniform_bits(float x) {
  return (uint32_t)__builtin_amdgcn_readfirstlane(__float_as_int(x));
}
__device__ __forceinline__ float power(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// The largest magnitude of N values (NaN does not count).
template <int N, typename F>
__device__ __forceinline__ float largest(const F& at) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) m = fmaxf(fmaxf(m, fabsf(at(i))), fabsf(at(i + 1)));
  return m;
}

// The exponent for values whose largest magnitude has the bits `m` (wave-uniform),
// `e` if that still holds them (or they hold an infinity).
__device__ __forceinline__ int range_exponent(uint32_t m, int e) {
  if (m == 0 || m >= 0x7F800000u) return e;
  const int x = (int)(m >> 23) - 127;  // in [2^x, 2^(x + 1)); subnormal: -127
  return x >= e + 15 || x < e + 9 ? min(max(x - 13, -110), 114) : e;
}

struct VRange {  // wave-uniform
  int e = 0;
  uint32_t seen = 0;
  // Takes in values of largest magnitude m (its bits, which order as it does).
  // True: the outputs so far are to be scaled by `by`.
  __device__ __forceinline__ bool take(uint32_t m, float& by) {
    const bool outputs = seen != 0;
    if (m < 0x7F800000u) seen = max(seen, m);
    const int before = e;
    e = range_exponent(seen, e);
    by = power(max(before - e, -126));
    return outputs && e != before;
  }
  // The factor that unscales a partial's outputs. Past 2^60 it takes another form
  // of the same value, o, l and 2^m by 2^64, so that p v stays finite (m's sum is
  // exact up to scores of 2^30).
  __device__ __forceinline__ float undo(float& m, float& l) const {
    const int sh = e > 60 ? 64 : 0;
    m += (float)sh;
    l *= power(-sh);
    return power(e - sh);
  }
};

// x as computed here: addresses made from it are not kept from before a loop in
// registers that the loop has better use for.
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// x - hi, one instruction that reads the f16 half where it is. (A plain
// subtraction widens the half first; the constant is kept from the compiler,
// which would turn the product by it back into one.)
__device__ __forceinline__ float minus_f16(float x, _Float16 hi) {
  float minus_one = -1.f;
  asm("" : "+s"(minus_one));
  return __builtin_fmaf((float)hi, minus_one, x);
}

// The base for scores of maximum mx. A score minus its base is exact, whatever the
// scores' size; where their last bit weighs as much as kUp (from 2^25 on) mx - kUp
// may round further down than that, and the base is the maximum itself.
__device__ __forceinline__ float base_of(float mx) {
  const float b = mx - kUp;
  return mx - b > kUp ? mx : b;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight f32 values as f16 hi and lo halves.
__device__ __forceinline__ void split8(const float (&x)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const f32x2 v = {x[e], x[e + 1]};
    const f16x2 h = __builtin_convertvector(v, f16x2);
    const f32x2 r = {minus_f16(v[0], h[0]), minus_f16(v[1], h[1])};
    const f16x2 l = __builtin_convertvector(r, f16x2);
    hi[e] = h[0];
    hi[e + 1] = h[1];
    lo[e] = l[0];
    lo[e + 1] = l[1];
  }
}

// ---- few columns: a wave's tiles in registers --------------------------------------
// 32 rows a tile on 16x16x32 products, 16 NB columns. K's lane (row li, quarter
// lk) loads dims 32 lk .. + 31 of rows li and 16 + li (the dot product's order
// of dims is free as long as q follows it: a Q8_0 block is one lane's, with one
// scale); V's lane (li, lk) dims 8 li .. + 7 of the rows whose probabilities
// the scores' C layout gives quarter lk: 4 lk .. + 3 and 16 + 4 lk .. + 3, so
// that P needs no exchange. Output tile b holds dims 8 i + b.
//
// For one token's columns it is the bytes that count: 131000 Q8_0 positions, 143
// MB, 29 us (4.9 TB/s, a large copy's rate); 4097 positions 6.1 and the merge 4.3; of
// 100 positions' 5.4 us 1.6 are the tile, the rest the way to its loads and the
// waves' fold. With the tiles through LDS the whole calls took 166, 26 and 13.6
// where they now take 33, 10.3 and 6.1. With 32 columns, a tile is 64 products
// (1024 cycles of a SIMD) and about 360 vector instructions (1440), 208 of them the
// codes' conversion, and two workgroups a CU, which 256 registers a wave allow,
// run one's products beside the other's vector work: 32 sequences over 8192
// positions 31.4 us with one, 25.8 with two.
template <typename T>
struct Raw;
template <>
struct Raw<Q8> {
  u32x4 k[2][2];
  uint32_t ks[2];
  u32x2 v[8];
  u32x2 vs[2];
};
template <>
struct Raw<_Float16> {
  f16x8 k[2][4];
  f16x8 v[8];
};
template <>
struct Raw<float> {
  f32x4 k[2][8];
  f32x4 v[8][2];
};

template <typename T>
__device__ __forceinline__ void load_raw_k(Raw<T>& x, const KvView& w, int h, long p0, long last, int li, int lk) {
  if constexpr (std::is_same<T, Q8>::value) {
    const char* kb = w.k + ((size_t)h * w.rows + p0) * kD;
    const uint16_t* sb = w.ks + ((size_t)h * w.rows + p0) * 4;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const int r = 16 * a + li;
      x.k[a][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kb + r * kD + 32 * lk));
      x.k[a][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kb + r * kD + 32 * lk + 16));
      x.ks[a] = sb[4 * r + lk];
    }
  } else {
    const T* kb = reinterpret_cast<const T*>(w.k) + (size_t)p0 * w.kv_dim + (size_t)h * kD;
    const int left = (int)min(last - p0, 31L);
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const T* r = kb + ((uint32_t)min(16 * a + li, left) * (uint32_t)w.kv_dim + 32 * lk);
      constexpr int n = std::is_same<T, float>::value ? 8 : 4;
#pragma unroll
      for (int c = 0; c < n; ++c)
        x.k[a][c] = *reinterpret_cast<const std::remove_reference_t<decltype(x.k[0][0])>*>(r + 16 / sizeof(T) * c);
    }
  }
}

template <typename T>
__device__ __forceinline__ void load_raw_v(Raw<T>& x, const KvView& w, int h, long p0, long last, int li, int lk) {
  if constexpr (std::is_same<T, Q8>::value) {
    const char* vb = w.v + ((size_t)h * w.rows + p0) * kD + 8 * li;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x.v[i] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x2*>(vb + (16 * (i >> 2) + 4 * lk + (i & 3)) * kD));
    const uint16_t* vs = w.vs + ((size_t)h * 4 + (li >> 2)) * w.rows + p0 + 4 * lk;
    x.vs[0] = *reinterpret_cast<const u32x2*>(vs);
    x.vs[1] = *reinterpret_cast<const u32x2*>(vs + 16);
  } else {
    const T* vb = reinterpret_cast<const T*>(w.v) + (size_t)p0 * w.kv_dim + (size_t)h * kD;
    const int left = (int)min(last - p0, 31L);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T* r = vb + ((uint32_t)min(16 * (i >> 2) + 4 * lk + (i & 3), left) * (uint32_t)w.kv_dim + 8 * li);
      if constexpr (std::is_same<T, float>::value) {
        x.v[i][0] = reinterpret_cast<const f32x4*>(r)[0];
        x.v[i][1] = reinterpret_cast<const f32x4*>(r)[1];
      } else {
        x.v[i] = *reinterpret_cast<const f16x8*>(r);
      }
    }
  }
}

// K operand of row tile a, dims 32 lk + 8 c .. + 7 (f32: hi and lo).
template <typename T>
__device__ __forceinline__ void raw_k(const Raw<T>& x, int a, int c, f16x8& hi, f16x8& lo) {
  if constexpr (std::is_same<T, Q8>::value) {
    const uint32_t w0 = x.k[a][c >> 1][2 * (c & 1)], w1 = x.k[a][c >> 1][2 * (c & 1) + 1];
    f16x2 p[4];
    q8_widen(w0, p[0], p[1]);
    q8_widen(w1, p[2], p[3]);
    const uint16_t sb = (uint16_t)x.ks[a];
    const _Float16 s = __builtin_bit_cast(_Float16, sb);
    const f16x2 ss = {s, s};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 v = p[i] * ss;
      hi[2 * i] = v[0];
      hi[2 * i + 1] = v[1];
    }
  } else if constexpr (std::is_same<T, float>::value) {
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = x.k[a][2 * c + (e >> 2)][e & 3];
    split8(f, hi, lo);
  } else {
    hi = x.k[a][c];
  }
}

// Zeroes the rows past `last` (what a plane holds there may not be finite).
template <typename T>
__device__ __forceinline__ void mask_v(Raw<T>& x, long p0, long last, int lk) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (p0 + 16 * (i >> 2) + 4 * lk + (i & 3) <= last) continue;
    if constexpr (std::is_same<T, Q8>::value) {
      const uint32_t w = x.vs[i >> 2][(i & 3) >> 1];
      x.vs[i >> 2][(i & 3) >> 1] = w & ((i & 1) ? 0x0000FFFFu : 0xFFFF0000u);
    } else if constexpr (std::is_same<T, float>::value) {
      x.v[i][0] = f32x4{};
      x.v[i][1] = f32x4{};
    } else {
      x.v[i] = f16x8{};
    }
  }
}

// V operands of output tiles 2 u and 2 u + 1.
template <typename T>
__device__ __forceinline__ void raw_v2(const Raw<T>& x, int u, f16x8 (&hi)[2], f16x8 (&lo)[2]) {
  if constexpr (std::is_same<T, Q8>::value) {
    const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = x.v[2 * i][u >> 1], b = x.v[2 * i + 1][u >> 1], sw = x.vs[i >> 1][i & 1];
      const f16x2 s = __builtin_bit_cast(f16x2, sw);
      // (a's byte, b's byte) of both dims, then each pair widened.
      const uint32_t t = __builtin_amdgcn_perm(b, a, (u & 1) ? 0x07030602u : 0x05010400u);
      const uint32_t t0 = __builtin_amdgcn_perm(0x64646464u, t, 0x04010400u);
      const uint32_t t1 = __builtin_amdgcn_perm(0x64646464u, t, 0x04030402u);
      const f16x2 v0 = (__builtin_bit_cast(f16x2, t0) + off) * s, v1 = (__builtin_bit_cast(f16x2, t1) + off) * s;
      hi[0][2 * i] = v0[0];
      hi[0][2 * i + 1] = v0[1];
      hi[1][2 * i] = v1[0];
      hi[1][2 * i + 1] = v1[1];
    }
  } else if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = x.v[i][u >> 1][2 * (u & 1) + k];
      split8(f, hi[k], lo[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) hi[k][i] = x.v[i][2 * u + k];
  }
}

// The f16 hi and lo halves of a column's q' = q * qscale, scaled by a power of
// two that brings its largest value to [2^13, 2^14); N values a lane, the
// column's lanes 16 and 32 apart (or 32 apart only). Returns the power back.
template <int N, bool QUARTERS, bool HL>
__device__ __forceinline__ float split_q(const f32x4 (&q)[N / 4], float qscale, f16x8 (&hi)[N / 8],
                                         f16x8 (&lo)[HL ? N / 8 : 1]) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) amax = fmaxf(fmaxf(amax, fabsf(q[i / 4][i % 4])), fabsf(q[i / 4][i % 4 + 1]));
  if constexpr (QUARTERS) amax = swap_max<16>(amax);
  amax = swap_max<32>(amax) * fabsf(qscale);
  int ex = 14;
  if (amax > 0.f && amax < INFINITY) (void)frexpf(amax, &ex);
  const int k = max(ex - 14, -100);
  const float c = ldexpf(qscale, -k);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const f32x2 v = {q[i / 4][i % 4] * c, q[i / 4][i % 4 + 1] * c};
    const f16x2 h = __builtin_convertvector(v, f16x2);
    hi[i / 8][i % 8] = h[0];
    hi[i / 8][i % 8 + 1] = h[1];
    if constexpr (HL) {
      const f32x2 r = {minus_f16(v[0], h[0]), minus_f16(v[1], h[1])};
      const f16x2 t = __builtin_convertvector(r, f16x2);
      lo[i / 8][i % 8] = t[0];
      lo[i / 8][i % 8 + 1] = t[1];
    }
  }
  return ldexpf(1.f, k);
}

// N probabilities as f16 hi (and lo) operand halves, and their sum added to l:
// p = 2^(s * up - base), up a power of two.
template <int N, bool HL>
__device__ __forceinline__ void probabilities(const float (&s)[N], float up, float base, f16x8 (&hi)[N / 8],
                                              f16x8 (&lo)[N / 8], float& l) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const f32x2 p = {__builtin_amdgcn_exp2f(__builtin_fmaf(s[i], up, -base)),
                     __builtin_amdgcn_exp2f(__builtin_fmaf(s[i + 1], up, -base))};
    sum += p[0];
    sum += p[1];
    const f16x2 h = __builtin_convertvector(p, f16x2);
    hi[i / 8][i % 8] = h[0];
    hi[i / 8][i % 8 + 1] = h[1];
    if constexpr (HL) {
      const f32x2 r = {minus_f16(p[0], h[0]), minus_f16(p[1], h[1])};
      const f16x2 t = __builtin_convertvector(r, f16x2);
      lo[i / 8][i % 8] = t[0];
      lo[i / 8][i % 8 + 1] = t[1];
    }
  }
  l += sum;
}

__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Where an item's partials go, and how they are folded.
struct PartDst {
  float* part;  // of the item's slot, kv head and (a tail's) sequence
  float* ml;
  // Folded by the last of the unit's items to finish (ticket != null), one for
  // each split of `positions`: `part` and `ml` are then the first slot's, this
  // item's `slot`.
  unsigned* ticket = nullptr;
  int positions = 0, slot = 0;
  size_t slot_floats = 0, ml_slot = 0;
};

// A store and a load that another XCD's L2 sees: the store goes through this
// one's, the load past it.
constexpr int kDeviceScope = 16;  // the sc1 bit of a buffer instruction's cache policy
__device__ __forceinline__ __amdgpu_buffer_rsrc_t device_rsrc(const float* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), (short)0, 0x7FFFFFFF, 0x00020000);
}

constexpr int kRegB = 34 * 64 * 4;  // a wave's block: 32 output values, maximum and sum by lane
constexpr int NW = 4;
constexpr int narrow_lds(int nb) { return NW * nb * kRegB; }

// Columns [col0, col0 + 16 NB) of kv head h over rows [t_begin, t_end) of `w`,
// by four waves of the workgroup (wave wv of them takes tiles wv, wv + 4, ...).
// All waves of the workgroup call it together; `run` false: nothing to do but
// the barriers. causal: column c sees start + row + 1 rows. WALK: longer than
// kWalkNarrow rows a wave.
template <typename T, int NB, bool CAUSAL, bool WALK>
__device__ void run_narrow(const RowsArgs& a, const KvView& w, int h, int col0, int n_cols, int row0, long t_begin,
                           long t_end, const PartDst& to, int wv, bool run, char* lds) {
  constexpr bool LO = Lo<T>::value, Q = std::is_same<T, Q8>::value;
  const int hk = a.kv_lo + h;
  const long last = t_end - 1;
  float m_run[NB], l_run[NB];
  uint32_t taint = 0;  // bit n: column block n saw a NaN row of this lane's dims (Q8_0, causal)
  f32x4 o[NB][8];
  VRange range;  // (f32)
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = 0.f;
#pragma unroll
    for (int b = 0; b < 8; ++b) o[n][b] = f32x4{};
  }
  const int n_tiles = run ? (int)((t_end - t_begin + 31) >> 5) : 0;
  f32x4* om = reinterpret_cast<f32x4*>(lds);  // [wave][NB][8][64]
  float* sums = reinterpret_cast<float*>(lds + NW * NB * 32 * 64 * 4);  // [wave][NB][2][64]
  // The wave's own part of both holds the sums that it has put aside.
  bool aside = false;
  // The running sums and those put aside, joined: piece(n, b, value) for each.
  const auto join = [&](int lane, const auto& piece) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int at = wv * NB + n;
      const float unscale = LO ? range.undo(m_run[n], l_run[n]) : 1.f;
      float f1 = 1.f, f2 = 0.f;
      if (WALK && aside) {
        const float m2 = sums[2 * at * 64 + lane], l2 = sums[(2 * at + 1) * 64 + lane];
        const float mn = fmaxf(m_run[n], m2), ms = mn == -INFINITY ? 0.f : mn;
        f1 = __builtin_amdgcn_exp2f(m_run[n] - ms);
        f2 = __builtin_amdgcn_exp2f(m2 - ms);
        m_run[n] = mn;
        l_run[n] = l_run[n] * f1 + l2 * f2;
      }
#pragma unroll
      for (int b = 0; b < 8; ++b) {
        f32x4 v = o[n][b];
        if constexpr (LO) v *= unscale;
        if (WALK && aside) v = v * f1 + om[(at * 8 + b) * 64 + lane] * f2;
        piece(n, b, v);
      }
    }
  };
  if (wv < n_tiles) {
    const int lane = threadIdx.x & 63, li = lane & 15, lk = lane >> 4;
    float q_up[NB], m_sub[NB];
    long limit[NB];
    f32x4 qv[NB][8];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m_sub[n] = 0.f;
      const int cc = min(col0 + 16 * n + li, n_cols - 1);
      const int r = a.rows == 1 ? 0 : row0 + cc / a.group;
      limit[n] = CAUSAL ? min((long)a.start + r + 1, t_end) : t_end;
      const float* qp = a.q + ((size_t)r * a.n_q_heads + (size_t)hk * a.group + (cc - (r - row0) * a.group)) * kD + 32 * lk;
#pragma unroll
      for (int i = 0; i < 8; ++i) qv[n][i] = *reinterpret_cast<const f32x4u*>(qp + 4 * i);
    }
    // A wave's loads run ahead of its products: K of the next tile is loaded into
    // the registers that this one's scores have read, V into those that its
    // output has.
    Raw<T> x;
    load_raw_k<T>(x, w, hk, t_begin + 32L * wv, last, li, lk);
    load_raw_v<T>(x, w, hk, t_begin + 32L * wv, last, li, lk);
    // What every column sees at least.
    const long w_first = CAUSAL ? min((long)a.start + row0 + min(col0, n_cols - 1) / a.group + 1, t_end) : t_end;
    f16x8 qh[NB][4], ql[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) q_up[n] = split_q<32, true, true>(qv[n], a.qscale, qh[n], ql[n]);
    for (int tile = wv; tile < n_tiles; tile += NW) {
      const long p0 = t_begin + 32L * tile;
      float k_up = 1.f;
      if constexpr (LO) {
        const int e = range_exponent(uniform_bits(wave_max(largest<64>([&](int i) { return x.k[i >> 5][(i >> 2) & 7][i & 3]; }))), 0);
        if (e != 0) {
          k_up = power(e);
#pragma unroll
          for (int i = 0; i < 16; ++i) x.k[i >> 3][i & 7] *= power(-e);
        }
      }
      // Products of one sum follow each other at a distance: with one block of
      // columns hi and lo are summed apart, with two in turn.
      constexpr int SA = NB == 1 ? 2 : 1;
      f32x4 s[NB][2][SA];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[n][t][0] = s[n][t][SA - 1] = f32x4{};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        f16x8 kh[2], kl[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) raw_k<T>(x, t, c, kh[t], kl[t]);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int t = 0; t < 2; ++t) s[n][t][0] = mfma16(kh[t], qh[n][c], s[n][t][0]);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int t = 0; t < 2; ++t) s[n][t][SA - 1] = mfma16(kh[t], ql[n][c], s[n][t][SA - 1]);
        if constexpr (LO) {
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int t = 0; t < 2; ++t) s[n][t][SA - 1] = mfma16(kl[t], qh[n][c], s[n][t][SA - 1]);
        }
      }
      // (f16 and f32 by 32 columns have the registers for it one product later)
      constexpr bool K_LATE = !Q && NB == 2;
      if (!K_LATE && tile + NW < n_tiles) load_raw_k<T>(x, w, hk, p0 + 32 * NW, last, li, lk);
      f16x8 ph[NB], pl[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        float y[8], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = SA == 1 ? s[n][i >> 2][0][i & 3] : s[n][i >> 2][0][i & 3] + s[n][i >> 2][SA - 1][i & 3];
        if (p0 + 32 > w_first) {
          const int seen = (int)max(limit[n] - p0, 0L) - 4 * lk;  // of this quarter's rows 16 t + r
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (16 * (i >> 2) + (i & 3) >= seen) y[i] = -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, y[i]);
        const float up = LO ? fmaxf(q_up[n] * k_up, FLT_MIN) : q_up[n];  // (above zero: a masked score is -inf)
        mx = swap_max<16>(mx);
        mx = swap_max<32>(mx) * up;
        if (__builtin_amdgcn_ballot_w64(mx - m_run[n] > kUp + kSlack) != 0) {
          const float mn = fmaxf(m_run[n], base_of(mx)), ms = mn == -INFINITY ? 0.f : mn;
          const float alpha = __builtin_amdgcn_exp2f(m_run[n] - ms);
          m_run[n] = mn;
          m_sub[n] = ms;
          l_run[n] *= alpha;
#pragma unroll
          for (int b = 0; b < 8; ++b) o[n][b] *= alpha;
        }
        f16x8 h1[1], l1[1];
        probabilities<8, true>(y, up, m_sub[n], h1, l1, l_run[n]);
        ph[n] = h1[0];
        pl[n] = l1[0];
      }
      if (p0 + 32 > t_end) mask_v<T>(x, p0, last, lk);
      if constexpr (LO) {
        float f;
        if (range.take(uniform_bits(wave_max(largest<64>([&](int i) { return x.v[i >> 3][(i >> 2) & 1][i & 3]; }))), f)) {
#pragma unroll
          for (int i = 0; i < 8 * NB; ++i) o[i >> 3][i & 7] *= f;
        }
        if (range.e != 0) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x.v[i >> 1][i & 1] *= power(-range.e);
        }
      }
      if constexpr (Q && CAUSAL) {
        // A row's NaN scale makes its block NaN; it must not reach columns that do
        // not see the row (0 * NaN): it goes in as zero and the columns that see it
        // are marked. (NaN: all exponent bits set, no scale is infinite, so adding
        // one to the exponent reaches the sign, which is clear.)
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= (x.vs[i >> 1][i & 1] & 0x7C007C00u) + 0x04000400u;
        if (__builtin_amdgcn_ballot_w64((bad & 0x80008000u) != 0) != 0) {
          uint32_t rows = 0;  // of the tile, NaN in this lane's output dims (block lk)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t half = (i & 1) ? 0xFFFF0000u : 0x0000FFFFu, sw = x.vs[i >> 2][(i & 3) >> 1];
            const bool nan = (sw & half & 0x7C007C00u) == (half & 0x7C007C00u);
            x.vs[i >> 2][(i & 3) >> 1] = nan ? sw & ~half : sw;
            const uint64_t who = __builtin_amdgcn_ballot_w64(nan);  // lane (4 block, quarter): its row
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (who >> (4 * lk + 16 * k) & 1) rows |= 1u << (16 * (i >> 2) + 4 * k + (i & 3));
          }
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            const long seen = limit[n] - p0;
            const uint32_t mask = seen >= 32 ? 0xFFFFFFFFu : seen <= 0 ? 0u : (1u << seen) - 1;
            if (rows & mask) taint |= 1u << n;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f16x8 vh[2], vl[2];
        raw_v2<T>(x, u, vh, vl);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          o[n][2 * u] = mfma16(vh[0], ph[n], o[n][2 * u]);
          o[n][2 * u + 1] = mfma16(vh[1], ph[n], o[n][2 * u + 1]);
          o[n][2 * u] = mfma16(vh[0], pl[n], o[n][2 * u]);
          o[n][2 * u + 1] = mfma16(vh[1], pl[n], o[n][2 * u + 1]);
          if constexpr (LO) {
            o[n][2 * u] = mfma16(vl[0], ph[n], o[n][2 * u]);
            o[n][2 * u + 1] = mfma16(vl[1], ph[n], o[n][2 * u + 1]);
          }
        }
        if (K_LATE && u == 0 && tile + NW < n_tiles) load_raw_k<T>(x, w, hk, p0 + 32 * NW, last, li, lk);
      }
      if (tile + NW < n_tiles) load_raw_v<T>(x, w, hk, p0 + 32 * NW, last, li, lk);
      if (WALK && (tile / NW + 1) % (kWalkNarrow / 32) == 0 && tile + NW < n_tiles) {
        const int lane = here(threadIdx.x & 63);
        join(lane, [&](int n, int b, f32x4 v) { om[((wv * NB + n) * 8 + b) * 64 + lane] = v; });
        aside = true;
        range = VRange{};
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          sums[2 * (wv * NB + n) * 64 + lane] = m_run[n];
          sums[(2 * (wv * NB + n) + 1) * 64 + lane] = l_run[n];
          m_run[n] = -INFINITY;  // (the first maximum above it clears the outputs)
          l_run[n] = 0.f;
        }
      }
    }
  }
  const int lane = WALK ? here(threadIdx.x & 63) : threadIdx.x & 63, li = lane & 15, lk = lane >> 4;
  if (LO || WALK) join(lane, [&](int n, int b, f32x4 v) { o[n][b] = v; });
  // The waves' partials meet in LDS, and each wave folds its share of the values,
  // in wave order. A lane's 16 bytes i are dims 32 lk + 4 i .. + 3 of column li.
  const int used = min(NW, n_tiles);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    // Each lane summed its own rows: the other quarters of the column's.
    l_run[n] = swap_sum<16>(l_run[n]);
    l_run[n] = swap_sum<32>(l_run[n]);
    if (Q && CAUSAL && (taint & (1u << n))) {
#pragma unroll
      for (int b = 0; b < 8; ++b) o[n][b] *= __builtin_nanf("");
    }
    if (wv < used) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        om[((wv * NB + n) * 8 + i) * 64 + lane] = f32x4{o[n][4 * (i & 1)][i >> 1], o[n][4 * (i & 1) + 1][i >> 1],
                                                        o[n][4 * (i & 1) + 2][i >> 1], o[n][4 * (i & 1) + 3][i >> 1]};
      sums[((wv * NB + n) * 2) * 64 + lane] = m_run[n];
      sums[((wv * NB + n) * 2 + 1) * 64 + lane] = l_run[n];
    }
  }
  __syncthreads();
  constexpr int IW = 8 / NW;  // 16-byte pieces a wave folds
  if (run) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float f[NW], M = -INFINITY, L = 0.f;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        f[k] = k < used ? sums[((k * NB + n) * 2) * 64 + lane] : -INFINITY;
        M = fmaxf(M, f[k]);
      }
      const float ms = M == -INFINITY ? 0.f : M;
#pragma unroll
      for (int k = 0; k < NW; ++k) {
        f[k] = __builtin_amdgcn_exp2f(f[k] - ms);
        if (k < used) L += f[k] * sums[((k * NB + n) * 2 + 1) * 64 + lane];
      }
      const int col = col0 + 16 * n + li;
      if (col >= n_cols) continue;
#pragma unroll
      for (int j = 0; j < IW; ++j) {
        const int i = wv * IW + j;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NW; ++k)
          if (k < used) v += om[((k * NB + n) * 8 + i) * 64 + lane] * f[k];
        if (a.single) {
          const int row = a.rows == 1 ? 0 : row0 + col / a.group;
          float* dst = a.out + ((size_t)row * a.n_heads * a.group + (size_t)h * a.group + (col - (row - row0) * a.group)) * kD +
                       32 * lk + 4 * i;
          const f32x4 r = v / L;
#pragma unroll
          for (int e = 0; e < 4; ++e) dst[e] = r[e];
        } else if (to.ticket) {
          __builtin_amdgcn_raw_buffer_store_b128(
              v, device_rsrc(to.part + to.slot * to.slot_floats),
              (int)(((size_t)(col / 16) * (16 * kD) + 4 * lane + 256 * i) * sizeof(float)), 0, kDeviceScope);
        } else {
          *reinterpret_cast<f32x4*>(to.part + (size_t)(col / 16) * (16 * kD) + 4 * lane + 256 * i) = v;
        }
      }
      if (!a.single && wv == 0 && lk == 0) {
        if (to.ticket) {
          const __amdgpu_buffer_rsrc_t rs = device_rsrc(to.ml + to.slot * to.ml_slot);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(M), rs, 8 * col, 0, kDeviceScope);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_int(L), rs, 8 * col + 4, 0, kDeviceScope);
        } else {
          to.ml[2 * col] = M;
          to.ml[2 * col + 1] = L;
        }
      }
    }
  }
  if (!to.ticket) return;  // (workgroup-uniform)
  // The last item of the unit folds all of them, slots in order, so that the
  // result does not depend on which one it is; it resets the ticket.
  __shared__ unsigned drawn;
  const int n_items = a.d_pos ? (int)(((unsigned)to.positions + a.split_len - 1) / (unsigned)a.split_len) : a.n_splits;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's stores are where other XCDs see them
  __syncthreads();
  if (threadIdx.x == 0) {
    drawn = __hip_atomic_fetch_add(to.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (drawn == (unsigned)n_items - 1) __hip_atomic_store(to.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (drawn != (unsigned)n_items - 1) return;
  const __amdgpu_buffer_rsrc_t rp = device_rsrc(to.part), rm = device_rsrc(to.ml);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int col = col0 + 16 * n + li;
    if (col >= n_cols) continue;
    float M = -INFINITY, L = 0.f;
    f32x4 r[IW];
#pragma unroll
    for (int j = 0; j < IW; ++j) r[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    constexpr int C = 8;  // slots in flight
    for (int k0 = 0; k0 < n_items; k0 += C) {
      float f[C], s[C];
      f32x4 v[IW][C];
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const int slot = min(k0 + k, n_items - 1);
        const int mo = (int)((slot * to.ml_slot + 2 * col) * sizeof(float));
        f[k] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rm, mo, 0, kDeviceScope));
        s[k] = __int_as_float(__builtin_amdgcn_raw_buffer_load_b32(rm, mo + 4, 0, kDeviceScope));
#pragma unroll
        for (int j = 0; j < IW; ++j) {
          const auto raw = __builtin_amdgcn_raw_buffer_load_b128(
              rp,
              (int)((slot * to.slot_floats + (size_t)(col / 16) * (16 * kD) + 4 * lane + 256 * (wv * IW + j)) *
                    sizeof(float)),
              0, kDeviceScope);
          v[j][k] = __builtin_bit_cast(f32x4, raw);
        }
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k0 + k < n_items) mn = fmaxf(mn, f[k]);
      const float ms = mn == -INFINITY ? 0.f : mn, g = __builtin_amdgcn_exp2f(M - ms);
      M = mn;
      L *= g;
#pragma unroll
      for (int j = 0; j < IW; ++j) r[j] *= g;
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k0 + k < n_items) {
          const float e = __builtin_amdgcn_exp2f(f[k] - ms);
          L += s[k] * e;
#pragma unroll
          for (int j = 0; j < IW; ++j) r[j] += v[j][k] * e;
        }
    }
    const int row = a.rows == 1 ? 0 : row0 + col / a.group;
    float* dst = a.out + ((size_t)row * a.n_heads * a.group + (size_t)h * a.group + (col - (row - row0) * a.group)) * kD + 32 * lk;
#pragma unroll
    for (int j = 0; j < IW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[4 * (wv * IW + j) + e] = r[j][e] / L;
  }
}

// ---- many columns: tiles staged through LDS -----------------------------------------
// Eight waves; half of them stage K, half V. A thread's share of a step of S
// rows in its raw type: K, units of 8 dims of one row; V, units of 4 dims of
// the eight rows of one operand slot.
template <typename T, int S>
struct Share {
  static constexpr int KU = S / 16, VU = S / 64;  // units a thread
  static constexpr int kw = std::is_same<T, Q8>::value ? 2 : std::is_same<T, float>::value ? 8 : 4;
  static constexpr int N = std::is_same<T, Q8>::value ? (KU * 3 > VU * 12 ? KU * 3 : VU * 12) : KU * kw;
  uint32_t r[N];
};

template <typename T, int S>
__device__ __forceinline__ void load_share(Share<T, S>& x, const KvView& w, int h, long t0, long last, bool is_v,
                                           int tt) {
  constexpr bool Q = std::is_same<T, Q8>::value;
  if (!is_v) {
    const int j = tt & 15;
#pragma unroll
    for (int i = 0; i < Share<T, S>::KU; ++i) {
      const long t = t0 + (tt >> 4) + 16 * i;
      if constexpr (Q) {
        const size_t row = (size_t)h * w.rows + t;
        const u32x2 c = *reinterpret_cast<const u32x2*>(w.k + row * kD + 8 * j);
        x.r[3 * i] = c[0];
        x.r[3 * i + 1] = c[1];
        x.r[3 * i + 2] = w.ks[row * 4 + (j >> 2)];
      } else {
        const T* base = reinterpret_cast<const T*>(w.k) + (size_t)t0 * w.kv_dim + (size_t)h * kD;
        const uint32_t at = (uint32_t)min((tt >> 4) + 16 * i, (int)min(last - t0, S - 1L)) * (uint32_t)w.kv_dim + 8 * j;
        const u32x4* p = reinterpret_cast<const u32x4*>(base + at);
#pragma unroll
        for (int k = 0; k < Share<T, S>::kw / 4; ++k) {
          const u32x4 c = p[k];
#pragma unroll
          for (int e = 0; e < 4; ++e) x.r[Share<T, S>::kw * i + 4 * k + e] = c[e];
        }
      }
    }
  } else {
    const int j = tt & 31;
#pragma unroll
    for (int u = 0; u < Share<T, S>::VU; ++u) {
      const int pg = (tt >> 5) + 8 * u;
      const long b = t0 + 32 * (pg >> 2) + 16 * ((pg >> 1) & 1) + 4 * (pg & 1);
      if constexpr (Q) {
        const char* p = w.v + ((size_t)h * w.rows + b) * kD + 4 * j;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x.r[12 * u + i] = *reinterpret_cast<const uint32_t*>(p + ((i & 3) + 8 * (i >> 2)) * kD);
        const uint16_t* sp = w.vs + ((size_t)h * 4 + (j >> 3)) * w.rows + b;
        const u32x2 s0 = *reinterpret_cast<const u32x2*>(sp), s1 = *reinterpret_cast<const u32x2*>(sp + 8);
        x.r[12 * u + 8] = s0[0];
        x.r[12 * u + 9] = s0[1];
        x.r[12 * u + 10] = s1[0];
        x.r[12 * u + 11] = s1[1];
      } else {
        constexpr int n = std::is_same<T, float>::value ? 4 : 2;  // words of 4 dims
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const T* base = reinterpret_cast<const T*>(w.v) + (size_t)t0 * w.kv_dim + (size_t)h * kD;
          const int row = (int)(b - t0) + (i & 3) + 8 * (i >> 2);
          const T* p = base + ((uint32_t)min(row, (int)min(last - t0, S - 1L)) * (uint32_t)w.kv_dim + 4 * j);
          typedef uint32_t uw __attribute__((ext_vector_type(n)));
          const uw c = *reinterpret_cast<const uw*>(p);
#pragma unroll
          for (int e = 0; e < n; ++e) x.r[8 * n * u + n * i + e] = c[e];
        }
      }
    }
  }
}

// Converts a share and writes it to the tiles at `lds` (K of all subtiles, V,
// then their lo halves). Rows past `last` go in as zeros (V). A Q8_0 row's NaN
// scale makes its block NaN; it must not reach columns that do not see the row
// (0 * NaN), so the block goes in as zeros and nan_rows[subtile][block] marks
// the row.
template <typename T, int S>
__device__ __forceinline__ void store_share(const Share<T, S>& x, char* lds, long t0, long last, bool is_v, int tt,
                                            uint32_t (*nan_rows)[4]) {
  constexpr bool Q = std::is_same<T, Q8>::value, LO = Lo<T>::value;
  constexpr int kPlane = S / 32 * kTileB;
  if (!is_v) {
    const int j = tt & 15;
#pragma unroll
    for (int i = 0; i < Share<T, S>::KU; ++i) {
      const int p = (tt >> 4) + 16 * i;
      f16x8 hi, lo;
      if constexpr (Q) {
        f16x2 c[4];
        q8_widen(x.r[3 * i], c[0], c[1]);
        q8_widen(x.r[3 * i + 1], c[2], c[3]);
        const uint16_t sb = (uint16_t)x.r[3 * i + 2];
        const _Float16 s = __builtin_bit_cast(_Float16, sb);
        const f16x2 ss = {s, s};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const f16x2 v = c[k] * ss;
          hi[2 * k] = v[0];
          hi[2 * k + 1] = v[1];
        }
      } else if constexpr (LO) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(x.r[8 * i + e]);
        split8(f, hi, lo);
      } else {
        const u32x4 c = {x.r[4 * i], x.r[4 * i + 1], x.r[4 * i + 2], x.r[4 * i + 3]};
        hi = __builtin_bit_cast(f16x8, c);
      }
      char* dst = lds + ((p >> 5) * 8 + (j >> 1)) * kFragB + k_slot(p & 31, j & 1) * 16;
      *reinterpret_cast<f16x8*>(dst) = hi;
      if constexpr (LO) *reinterpret_cast<f16x8*>(dst + 2 * kPlane) = lo;
    }
  } else {
    const int j = tt & 31, dt = j >> 3;
#pragma unroll
    for (int u = 0; u < Share<T, S>::VU; ++u) {
      const int pg = (tt >> 5) + 8 * u, st = pg >> 2, s = (pg >> 1) & 1, hh = pg & 1;
      const long b = t0 + 32 * st + 16 * s + 4 * hh;
      const bool edge = t0 + S - 1 > last;  // (of the step)
      f16x8 hi[4], lo[4];
      if constexpr (Q) {
        uint32_t sw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sw[i] = x.r[12 * u + 8 + i];
        if (edge) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (b + (i & 3) + 8 * (i >> 2) > last) sw[i >> 1] &= (i & 1) ? 0x0000FFFFu : 0xFFFF0000u;
        }
        // A scale's NaN: all exponent bits set (no scale is infinite), so that
        // adding one to the exponent reaches the (clear) sign.
        uint32_t nan = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) nan |= ((sw[i] & 0x7C007C00u) + 0x04000400u);
        uint32_t bad = 0;
        if (nan & 0x80008000u) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t half = (i & 1) ? 0xFFFF0000u : 0x0000FFFFu;
            if ((sw[i >> 1] & half & 0x7C007C00u) == (half & 0x7C007C00u)) {
              sw[i >> 1] &= ~half;
              bad |= 1u << (16 * s + 4 * hh + (i & 3) + 8 * (i >> 2));
            }
          }
        }
        if (bad && (j & 7) == 0) atomicOr(&nan_rows[st][dt], bad);
        const f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a = x.r[12 * u + 2 * i], c = x.r[12 * u + 2 * i + 1];
          const f16x2 sc = __builtin_bit_cast(f16x2, sw[i]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t t = __builtin_amdgcn_perm(c, a, k ? 0x07030602u : 0x05010400u);
            const uint32_t p0 = __builtin_amdgcn_perm(0x64646464u, t, 0x04010400u);
            const uint32_t p1 = __builtin_amdgcn_perm(0x64646464u, t, 0x04030402u);
            const f16x2 v0 = (__builtin_bit_cast(f16x2, p0) + off) * sc;
            const f16x2 v1 = (__builtin_bit_cast(f16x2, p1) + off) * sc;
            hi[2 * k][2 * i] = v0[0];
            hi[2 * k][2 * i + 1] = v0[1];
            hi[2 * k + 1][2 * i] = v1[0];
            hi[2 * k + 1][2 * i + 1] = v1[1];
          }
        }
      } else if constexpr (LO) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            f[i] = edge && b + (i & 3) + 8 * (i >> 2) > last ? 0.f : __uint_as_float(x.r[32 * u + 4 * i + d]);
          split8(f, hi[d], lo[d]);
        }
      } else {
        uint32_t c[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          c[i] = edge && b + ((i >> 1) & 3) + 8 * (i >> 3) > last ? 0u : x.r[16 * u + i];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          u32x4 p;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            p[i] = __builtin_amdgcn_perm(c[4 * i + 2 + (d >> 1)], c[4 * i + (d >> 1)], (d & 1) ? 0x07060302u : 0x05040100u);
          hi[d] = __builtin_bit_cast(f16x8, p);
        }
      }
      char* base = lds + kPlane + (st * 8 + dt * 2 + s) * kFragB;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int at = v_slot(dt, (j & 7) * 4 + d, hh) * 16;
        *reinterpret_cast<f16x8*>(base + at) = hi[d];
        if constexpr (LO) *reinterpret_cast<f16x8*>(base + at + 2 * kPlane) = lo[d];
      }
    }
  }
}

// The columns [col0, col0 + 32 WC) of kv head h (column c: row c / group, head
// c % group) over rows [t_begin, t_end) of `w`, on 32x32x16 products; wave (wc,
// wp) takes columns 32 wc .. and the 32-row subtiles wp, wp + WP, ... of each
// step. The next step's rows are in flight while this one's are computed, and
// its tiles the other half of the LDS.
//
// Eight waves convert a tile once for up to 256 columns, where the narrow items
// would convert it eight times: a step of 64 rows by 256 columns takes 3.5 us, half
// of it matrix instructions, the softmax and the conversion the rest (1000 rows
// at 12000 positions: 57 % and 34 % of the SIMDs' cycles; 410 GFLOP in 380 us, 1.08
// PFLOP/s, as much as a large f16 product reaches on this card under its power
// limit). Two such workgroups a CU with half the columns each, the
// instruction priority moved with the phases, or K's staging between the
// subtiles measured the same or slower (512 rows at 3449: 79, 80 and 79 us).
template <int WC>
constexpr int wide_step() {
  return WC == 2 ? 128 : 64;
}
template <typename T, int WC>
constexpr int wide_lds() {
  const int stages = 2 * stage_bytes<T>(wide_step<WC>());
  const int merge = (8 / WC - 1) * WC * 66 * 64 * 4;
  return stages > merge ? stages : merge;
}

template <typename T, int WC, bool HL>
__device__ void run_wide(const RowsArgs& a, const KvView& w, int h, int col0, int n_cols, long t_begin, long t_end,
                         bool causal, int split, char* lds) {
  constexpr int WP = 8 / WC, S = wide_step<WC>(), SUB = S / 32 / WP;
  constexpr bool LO = Lo<T>::value, Q = std::is_same<T, Q8>::value;
  constexpr int kPlane = S / 32 * kTileB, kStage = stage_bytes<T>(S);
  __shared__ __attribute__((aligned(16))) uint32_t nan_rows[3][S / 32][4];  // by step mod 3: cleared two steps ahead of its reads
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wc = wave % WC, wp = wave / WC;
  const bool is_v = wave >= 4;
  const int tt = tid & 255;
  const int lc = lane & 31, lh = lane >> 5;
  const int col = col0 + 32 * wc + lc;
  const bool live = col < n_cols;
  const int crow = (live ? col : n_cols - 1) / a.group, chead = (live ? col : n_cols - 1) % a.group;
  const long limit = causal ? min((long)a.start + crow + 1, t_end) : t_end;
  // What the wave's first column sees, and its last.
  const int wcol0 = min(col0 + 32 * wc, n_cols - 1), wcol1 = min(col0 + 32 * wc + 31, n_cols - 1);
  const long w_first = causal ? min((long)a.start + wcol0 / a.group + 1, t_end) : t_end;
  const long w_last = causal ? min((long)a.start + wcol1 / a.group + 1, t_end) : t_end;
  const int hk = a.kv_lo + h;
  const long last = t_end - 1;

  Share<T, S> sh;
  load_share<T, S>(sh, w, hk, t_begin, last, is_v, tt);
  f16x8 qh[8], ql[HL ? 8 : 1];
  float q_up;
  {  // dims 16 c + 8 lh .. + 7 of each chunk c
    const float* qp = a.q + ((size_t)crow * a.n_q_heads + (size_t)hk * a.group + chead) * kD;
    f32x4 v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = *reinterpret_cast<const f32x4u*>(qp + 16 * (i >> 1) + 8 * lh + 4 * (i & 1));
    q_up = split_q<64, false, HL>(v, a.qscale, qh, ql);
  }
  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = f32x16{};
  // f32: the largest magnitudes of a step's K and V rows, by all waves that stage
  // them, before any converts its share.
  __shared__ uint32_t range_bits[2][2];
  VRange range;
  float k_up = 1.f;
  const auto scale_share = [&](int slot) {
    const float m = is_v ? largest<Share<T, S>::VU * 32>([&](int i) { return __uint_as_float(sh.r[i]); })
                         : largest<Share<T, S>::KU * 8>([&](int i) { return __uint_as_float(sh.r[i]); });
    const float w = wave_max(m);
    if (lane == 0) atomicMax(&range_bits[slot][is_v], __float_as_uint(w));
    __syncthreads();
    const int ke = range_exponent(__builtin_amdgcn_readfirstlane(range_bits[slot][0]), 0);
    k_up = power(ke);
    if (tid < 2) range_bits[slot ^ 1][tid] = 0;
    float f;
    if (range.take(__builtin_amdgcn_readfirstlane(range_bits[slot][1]), f)) {
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] *= f;
    }
    const int e = is_v ? range.e : ke;
    if (e != 0) {
#pragma unroll
      for (int i = 0; i < Share<T, S>::N; ++i) sh.r[i] = __float_as_uint(__uint_as_float(sh.r[i]) * power(-e));
    }
  };
  if constexpr (Q || LO) {
    if (Q && tid < 3 * (S / 32) * 4) (&nan_rows[0][0][0])[tid] = 0;
    if (LO && tid < 2) range_bits[0][tid] = 0;
    __syncthreads();
  }
  if constexpr (LO) scale_share(0);
  store_share<T, S>(sh, lds, t_begin, last, is_v, tt, Q ? nan_rows[0] : nullptr);
  __syncthreads();

  if (wave >= 4) __builtin_amdgcn_s_setprio(1);
  float m_run = -INFINITY, m_sub = 0.f, l_run = 0.f;
  uint32_t taint = 0;  // Q8_0: this lane's dims met a NaN block in a row its column sees
  int buf = 0, n3 = 0;
  // The sums put aside: o by lane, then (m, l).
  const auto place = [&] { return a.aside + (size_t)(blockIdx.x * 8 + wave) * (17 * 64) + here(threadIdx.x & 63); };
  bool aside = false;
  // The running sums and those put aside, joined: piece(i, registers 4 i ..) for each.
  const auto join = [&](f32x4* store, const auto& piece) {
    const float unscale = LO ? range.undo(m_run, l_run) : 1.f;
    float f1 = 1.f, f2 = 0.f;
    if (aside) {
      const f32x4 s2 = store[16 * 64];
      const float mn = fmaxf(m_run, s2[0]), ms = mn == -INFINITY ? 0.f : mn;
      f1 = __builtin_amdgcn_exp2f(m_run - ms);
      f2 = __builtin_amdgcn_exp2f(s2[0] - ms);
      m_run = mn;
      l_run = l_run * f1 + s2[1] * f2;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // (few registers are left for the loads in flight)
      f32x4 v = {o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2], o[i >> 2][4 * (i & 3) + 3]};
      if constexpr (LO) v *= unscale;
      if (aside) v = v * f1 + store[64 * i] * f2;
      piece(i, v);
    }
  };
  for (long t0 = t_begin; t0 < t_end; t0 += S) {
    const bool more = t0 + S < t_end;
    if (more && !LO) load_share<T, S>(sh, w, hk, t0 + S, last, is_v, tt);
    if constexpr (Q) {
      const int clear = n3 == 0 ? 2 : n3 - 1;  // (n3 + 2) mod 3
      if (tid < (S / 32) * 4) (&nan_rows[clear][0][0])[tid] = 0;
    }
    const char* tile = lds + buf * kStage;
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub) {
      const int st = wp + WP * sub;
      const long p0 = t0 + 32 * st;
      if (p0 >= w_last) continue;  // wave-uniform; barriers are outside
      const char* kt = tile + st * kTileB + k_slot(lc, lh) * 16;
      const char* vt = tile + kPlane + st * kTileB;
      f32x16 acc = {};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const f16x8 kf = *reinterpret_cast<const f16x8*>(kt + c * kFragB);
        acc = mfma(kf, qh[c], acc);
        if constexpr (HL) acc = mfma(kf, ql[c], acc);
        if constexpr (LO) acc = mfma(*reinterpret_cast<const f16x8*>(kt + 2 * kPlane + c * kFragB), qh[c], acc);
      }
      float x[16], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = acc[i];
      if (p0 + 32 > w_first) {  // some column does not see all of it
        const int seen = (int)max(limit - p0, 0L) - 4 * lh;  // of this half's rows 8 t + r
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i >> 2) + (i & 3) >= seen) x[i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, x[i]);
      const float up = LO ? fmaxf(q_up * k_up, FLT_MIN) : q_up;  // (above zero: a masked score is -inf)
      mx = swap_max<32>(mx) * up;
      if (__builtin_amdgcn_ballot_w64(mx - m_run > kUp + kSlack) != 0) {
        const float mn = fmaxf(m_run, base_of(mx)), ms = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m_run - ms);
        m_run = mn;
        m_sub = ms;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= alpha;
      }
      f16x8 ph[2], pl[2];
      probabilities<16, HL>(x, up, m_sub, ph, pl, l_run);
      if constexpr (Q) {
        // Lane (column, lh) holds dims of every block d.
        const u32x4 bad = *reinterpret_cast<const u32x4*>(nan_rows[n3][st]);
        if (__builtin_amdgcn_readfirstlane(bad[0] | bad[1] | bad[2] | bad[3])) {
          const long seen = limit - p0;  // rows of this subtile the column sees
          const uint32_t mask = seen >= 32 ? 0xFFFFFFFFu : seen <= 0 ? 0u : (1u << seen) - 1;
#pragma unroll
          for (int d = 0; d < 4; ++d)
            if (bad[d] & mask) taint |= 1u << d;
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f16x8 vf[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          vf[d] = *reinterpret_cast<const f16x8*>(vt + (d * 2 + s) * kFragB + v_slot(d, lc, lh) * 16);
          o[d] = mfma(vf[d], ph[s], o[d]);
        }
        if constexpr (HL) {
#pragma unroll
          for (int d = 0; d < 4; ++d) o[d] = mfma(vf[d], pl[s], o[d]);
        }
        if constexpr (LO) {
#pragma unroll
          for (int d = 0; d < 4; ++d)
            o[d] = mfma(*reinterpret_cast<const f16x8*>(vt + 2 * kPlane + (d * 2 + s) * kFragB + v_slot(d, lc, lh) * 16),
                        ph[s], o[d]);
        }
      }
    }
    if (more && (int)(t0 + S - t_begin) % kWalkWide == 0) {
      f32x4* const store = place();
      join(store, [&](int i, f32x4 v) { store[64 * i] = v; });
      store[16 * 64] = f32x4{m_run, l_run, 0.f, 0.f};
      aside = true;
      range = VRange{};
      m_run = -INFINITY;  // (the first maximum above it clears the outputs)
      l_run = 0.f;
    }
    buf ^= 1;
    n3 = n3 == 2 ? 0 : n3 + 1;
    if constexpr (LO) {
      if (more) {
        load_share<T, S>(sh, w, hk, t0 + S, last, is_v, tt);  // (no registers to hold it meanwhile)
        scale_share(buf);
      }
    }
    if (more) store_share<T, S>(sh, lds + buf * kStage, t0 + S, last, is_v, tt, Q ? nan_rows[n3] : nullptr);
    __syncthreads();
  }
  if (LO || aside)
    join(place(), [&](int i, f32x4 v) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i >> 2][4 * (i & 3) + e] = v[e];
    });
  // Each lane summed its own rows: the other half of the column's.
  l_run = swap_sum<32>(l_run);
  if constexpr (Q) {
    if (taint) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (taint & (1u << d)) o[d] = o[d] * __builtin_nanf("");
    }
  }
  // The row groups' partials meet in LDS, in wave order.
  if constexpr (WP > 1) {
    float* om = reinterpret_cast<float*>(lds);  // [wp - 1][wc][64 registers][64 lanes], then (m, l)
    constexpr int kWave = 66 * 64;
    if (wp > 0) {
      float* d = om + ((wp - 1) * WC + wc) * kWave + lane;
#pragma unroll
      for (int i = 0; i < 64; ++i) d[64 * i] = o[i >> 4][i & 15];
      d[64 * 64] = m_run;
      d[64 * 65] = l_run;
    }
    __syncthreads();
    if (wp == 0) {
      for (int p = 1; p < WP; ++p) {
        const float* d = om + ((p - 1) * WC + wc) * kWave + lane;
        const float m2 = d[64 * 64], l2 = d[64 * 65];
        const float mn = fmaxf(m_run, m2), ms = mn == -INFINITY ? 0.f : mn;
        const float f1 = __builtin_amdgcn_exp2f(m_run - ms), f2 = __builtin_amdgcn_exp2f(m2 - ms);
        m_run = mn;
        l_run = l_run * f1 + l2 * f2;
#pragma unroll
        for (int i = 0; i < 64; ++i) o[i >> 4][i & 15] = o[i >> 4][i & 15] * f1 + d[64 * i] * f2;
      }
    }
  }
  if (wp != 0 || !live) return;
  if (a.single) {
    const float inv = 1.f / l_run;
    float* dst = a.out + ((size_t)crow * a.n_heads * a.group + (size_t)h * a.group + chead) * kD;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dst[32 * d + 8 * (i >> 2) + 4 * lh + (i & 3)] = o[d][i] * inv;
    return;
  }
  float* dst = a.part + split * a.slot_floats + ((size_t)h * ((n_cols + 31) / 32) + col / 32) * (32 * kD) + 4 * lane;
#pragma unroll
  for (int i = 0; i < 16; ++i) {  // dims 8 i + 4 lh .. + 3
    const f32x4 v = {o[i >> 2][4 * (i & 3)], o[i >> 2][4 * (i & 3) + 1], o[i >> 2][4 * (i & 3) + 2],
                     o[i >> 2][4 * (i & 3) + 3]};
    *reinterpret_cast<f32x4*>(dst + 256 * i) = v;
  }
  if (lh == 0) {
    float* ml = a.ml + 2 * (((size_t)split * a.n_heads + h) * n_cols + col);
    ml[0] = m_run;
    ml[1] = l_run;
  }
}

// Positions of a call that takes them from device memory; false: refused.
__device__ __forceinline__ bool device_positions(const uint32_t* d_pos, int planned, int& positions) {
  if (!d_pos) return true;
  const uint32_t p = *d_pos;
  if (p >= (uint32_t)planned) return false;
  positions = (int)p + 1;
  return true;
}

// A tail item by the four waves `wv` counts: sequence, column block of 16,
// split (b past them: none, the waves only keep the barriers).
template <typename T, bool WALK>
__device__ void tail_item(const RowsArgs& a, const TailLens& lens, int b, int wv, char* lds) {
  const int split = b % a.t_splits;
  b /= a.t_splits;
  const int cb = b % a.t_cb;
  b /= a.t_cb;
  const int h = b % a.n_heads, seq = b / a.n_heads;
  const long len = seq < a.rows ? lens.len[seq] : 0, t_begin = (long)split * a.t_split_len;
  KvView w = a.tail;
  w.k += (size_t)seq * w.layer_bytes;
  w.v += (size_t)seq * w.layer_bytes;
  w.ks += (size_t)seq * w.layer_scales;
  w.vs += (size_t)seq * w.layer_scales;
  PartDst to;
  to.part = a.part + a.t_base + split * a.t_slot_floats + ((size_t)seq * a.n_heads + h) * a.t_cb * (16 * kD);
  to.ml = a.ml + 2 * (((size_t)(a.n_splits + split) * a.n_heads + h) * a.rows + seq) * a.group;
  run_narrow<T, 1, false, WALK>(a, w, h, cb * 16, a.group, seq, t_begin, min(len, t_begin + a.t_split_len), to, wv,
                                t_begin < len, lds);
}

// Workgroup b of the main items. Those of one XCD (b mod 8) are consecutive in
// the order (kv head, split, column block), so that the column blocks of a split
// meet in its L2, and every XCD has as many (600 rows at 3400, 19 blocks of 12
// splits: 169 us with whole splits to an XCD, 90 so).
__device__ __forceinline__ bool main_item(const RowsArgs& a, int b, int& h, int& split, int& cb) {
  const int n = a.n_heads * a.n_splits * a.n_cb, i = (b & 7) * (a.main_items >> 3) + (b >> 3);
  if (i >= n) return false;
  cb = i % a.n_cb;
  const int u = i / a.n_cb;
  split = u % a.n_splits;
  h = u / a.n_splits;
  return true;
}

// Workgroups of narrow items that a CU's registers are to hold.
template <typename T>
constexpr int narrow_waves(int nb, bool walk) {
  return nb == 2 && (Lo<T>::value || (walk && !std::is_same<T, Q8>::value)) ? 1 : 2;
}

template <typename T, int NB, bool TAILS, bool CAUSAL, bool WALK>
__global__ __launch_bounds__(256, narrow_waves<T>(NB, WALK)) void rows_narrow_kernel(RowsArgs a,
                                                              std::conditional_t<TAILS, TailLens, NoLens> lens) {
  __shared__ __attribute__((aligned(16))) char lds[narrow_lds(NB)];
  const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  // All of the arguments at once, in place of one trip to memory at each branch
  // that needs more of them (16 sequences over 4096 20.9 -> 20.6 us).
  asm volatile("" ::"s"(a.split_len), "s"(a.q), "s"(a.main.k), "s"(a.main.v), "s"(a.main.ks), "s"(a.main.vs),
               "s"(a.main.rows), "s"(a.rows), "s"(a.group), "s"(a.kv_lo), "s"(a.part), "s"(a.qscale));
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  int split, h, cb = 0;
  if constexpr (TAILS) {
    if ((int)blockIdx.x >= a.main_items) {
      tail_item<T, WALK>(a, lens, (int)blockIdx.x - a.main_items, wv, lds);
      return;
    }
    if (!main_item(a, blockIdx.x, h, split, cb)) return;
  } else {  // grid (splits, kv heads, column blocks)
    split = blockIdx.x;
    h = blockIdx.y;
    cb = blockIdx.z;
  }
  const int n_cols = a.rows * a.group, col0 = cb * 16 * NB;
  long t_end = positions;
  if constexpr (CAUSAL) t_end = min(t_end, (long)a.start + (min(col0 + 16 * NB, n_cols) - 1) / a.group + 1);
  const long t_begin = (long)split * a.split_len;
  t_end = min(t_end, t_begin + a.split_len);
  if (t_begin >= t_end) return;
  PartDst to;
  const size_t part = (size_t)h * ((n_cols + 15) / 16) * (16 * kD), ml_slot = 2 * (size_t)a.n_heads * n_cols;
  to.part = a.part + part;
  to.ml = a.ml + 2 * (size_t)h * n_cols;
  if (!TAILS && !CAUSAL && a.tickets) {
    to.ticket = a.tickets + 32 * h;
    to.positions = positions;
    to.slot = split;
    to.slot_floats = a.slot_floats;
    to.ml_slot = ml_slot;
  } else {
    to.part += split * a.slot_floats;
    to.ml += split * ml_slot;
  }
  run_narrow<T, NB, CAUSAL, WALK>(a, a.main, h, col0, n_cols, 0, t_begin, t_end, to, wv, true, lds);
}

template <typename T, int WC, bool HL, bool TAILS>
__global__ __launch_bounds__(512) void rows_wide_kernel(RowsArgs a, std::conditional_t<TAILS, TailLens, NoLens> lens) {
  constexpr int kMain = wide_lds<T, WC>(), kTail = TAILS ? 2 * narrow_lds(1) : 0;
  __shared__ __attribute__((aligned(1024))) char lds[kMain > kTail ? kMain : kTail];
  const int b = blockIdx.x;
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  if (!TAILS || b < a.main_items) {
    int h, split, cb;
    if (!main_item(a, b, h, split, cb)) return;
    if (a.causal) cb = a.n_cb - 1 - cb;  // the longest first
    const int n_cols = a.rows * a.group, col0 = cb * 32 * WC;
    long t_end = positions;
    if (a.causal) {  // the last column's limit
      const int r = (min(col0 + 32 * WC, n_cols) - 1) / a.group;
      t_end = min(t_end, (long)a.start + r + 1);
    }
    const long t_begin = (long)split * a.split_len;
    t_end = min(t_end, t_begin + a.split_len);
    if (t_begin >= t_end) return;
    run_wide<T, WC, HL>(a, a.main, h, col0, n_cols, t_begin, t_end, a.causal != 0, split, lds);
  } else if constexpr (TAILS) {  // two items, four waves each
    const int half = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8);
    tail_item<T, true>(a, lens, 2 * (b - a.main_items) + half, __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) & 3),
                 lds + half * narrow_lds(1));
  }
}

// Folds the columns' partials, slots in an order that depends on their number
// alone. A wave has 16 bytes (i = 0..15) of a block of 32 columns, lane (column,
// half) dims 8 i + 4 half .. + 3; G waves share the slots of one, four loads in
// flight each, and meet in LDS. Bound by the partials' bytes where there are many
// (1000 rows in two splits: 33 MB in, 16 out, 11.8 us, 4.2 TB/s), by a launch and two
// dependent loads, 4 us, where there are few. G by the slots: 33 slots by one
// wave of 4 loads at a time would be 9 trips to memory, by 16 waves it is one.
template <int G, bool TAILS>
__global__ __launch_bounds__(64 * (G < 4 ? 4 : G)) void rows_merge_kernel(
    RowsArgs a, int narrow, std::conditional_t<TAILS, TailLens, NoLens> lens) {
  constexpr int W = G < 4 ? 4 : G;
  __shared__ f32x4 sm_o[G > 1 ? W : 1][64];
  __shared__ float sm_m[G > 1 ? W : 1][64], sm_l[G > 1 ? W : 1][64];
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lc = lane & 31, lh = lane >> 5;
  const int n_cols = a.rows * a.group, blocks = (n_cols + 31) / 32;
  const int item = (int)blockIdx.x * (W / G) + wave / G, sub = wave % G;
  const int i = item % 16, block = item / 16 % blocks, h = item / 16 / blocks;
  const int col = 32 * block + lc;
  const bool live = h < a.n_heads && col < n_cols;
  if (G == 1 && !live) return;
  const int c = live ? col : 0, hh = live ? h : 0, row = c / a.group;
  long limit = positions;
  if (a.causal) limit = min(limit, (long)a.start + row + 1);
  const int n_main = (int)((limit + a.split_len - 1) / a.split_len);
  int n_all = n_main;
  const float* part = a.part + (narrow ? ((size_t)hh * ((n_cols + 15) / 16) + c / 16) * (16 * kD) +
                                             256 * (2 * (i & 3) + lh) + 4 * ((c & 15) + 16 * (i >> 2))
                                       : ((size_t)hh * blocks + block) * (32 * kD) + 256 * i + 4 * lane);
  const float* ml = a.ml + 2 * ((size_t)hh * n_cols + c);
  const size_t ml_slot = 2 * (size_t)a.n_heads * n_cols;
  const float* tail = nullptr;
  if constexpr (TAILS) {
    n_all += (int)((lens.len[row] + a.t_split_len - 1) / a.t_split_len);
    const int g = c % a.group;  // its block of 16, and dims 8 i + 4 lh = 32 lk + 4 j
    tail = a.part + a.t_base + (((size_t)row * a.n_heads + hh) * a.t_cb + g / 16) * (16 * kD) +
           256 * (2 * (i & 3) + lh) + 4 * ((g & 15) + 16 * (i >> 2));
  }
  float M = -INFINITY, L = 0.f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = sub; k0 < n_all; k0 += 4 * G) {
    float m[4], s[4];
    f32x4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int j = min(k0 + k * G, n_all - 1);
      const bool is_tail = TAILS && j >= n_main;
      const float* p = is_tail ? tail + (j - n_main) * a.t_slot_floats : part + j * a.slot_floats;
      const float* q = ml + (size_t)(is_tail ? a.n_splits + j - n_main : j) * ml_slot;
      m[k] = q[0];
      s[k] = q[1];
      v[k] = *reinterpret_cast<const f32x4*>(p);
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k0 + k * G < n_all) mn = fmaxf(mn, m[k]);
    const float ms = mn == -INFINITY ? 0.f : mn;
    const float f = __builtin_amdgcn_exp2f(M - ms);
    M = mn;
    L *= f;
    O *= f;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k0 + k * G < n_all) {
        const float e = __builtin_amdgcn_exp2f(m[k] - ms);
        L += s[k] * e;
        O += v[k] * e;
      }
  }
  if constexpr (G > 1) {
    sm_o[wave][lane] = O;
    sm_m[wave][lane] = M;
    sm_l[wave][lane] = L;
    __syncthreads();
    if (sub != 0) return;
#pragma unroll
    for (int k = 1; k < G; ++k) {
      const float m2 = sm_m[wave + k][lane], mn = fmaxf(M, m2), ms = mn == -INFINITY ? 0.f : mn;
      const float f1 = __builtin_amdgcn_exp2f(M - ms), f2 = __builtin_amdgcn_exp2f(m2 - ms);
      M = mn;
      L = L * f1 + sm_l[wave + k][lane] * f2;
      O = O * f1 + sm_o[wave + k][lane] * f2;
    }
  }
  if (!live) return;
  const f32x4 r = O / L;
  float* dst = a.out + ((size_t)row * a.n_heads * a.group + (size_t)h * a.group + c % a.group) * kD + 8 * i + 4 * lh;
#pragma unroll
  for (int e = 0; e < 4; ++e) dst[e] = r[e];  // out may be only 4-byte aligned
}

// ---- any head size up to 512 --------------------------------------------------------
// One workgroup a column; each wave walks every fourth row (one row at a time,
// the head's values over the lanes), f32 products, the sums over rows in f64 (one
// term a row: an f32 sum would drop those below 2^-24 of it), the waves' joined in
// LDS. For geometries no model of this library's path has; it is right, not fast.
template <typename T, bool TAILS>
__global__ __launch_bounds__(256) void rows_generic_kernel(RowsArgs a, int hd,
                                                           std::conditional_t<TAILS, TailLens, NoLens> lens) {
  constexpr int kPer = 8;
  __shared__ double sm_o[3][64 * kPer], sm_l[3];
  __shared__ float sm_m[3];
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n_q = a.n_heads * a.group;
  const int row = blockIdx.x / n_q, hq = blockIdx.x % n_q, h = a.kv_lo + hq / a.group;
  const float* qp = a.q + ((size_t)row * a.n_q_heads + (size_t)a.kv_lo * a.group + hq) * hd;
  float q[kPer];
  double o[kPer], l = 0.0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    q[i] = lane + 64 * i < hd ? qp[lane + 64 * i] * a.qscale : 0.f;
    o[i] = 0.0;
  }
  float m = -INFINITY;
  auto walk = [&](const KvView& w, long len) {
    for (long t = wave; t < len; t += 4) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 64 * i < hd) x += q[i] * kv_value<T, false>(w, hd, h, t, lane + 64 * i);
      x = group_sum<32>(x);
      x = swap_sum<32>(x);
      const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.f : mn;
      const double f = __builtin_amdgcn_exp2f(m - ms), p = __builtin_amdgcn_exp2f(x - ms);
      m = mn;
      l = l * f + p;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 64 * i < hd) o[i] = o[i] * f + p * (double)kv_value<T, true>(w, hd, h, t, lane + 64 * i);
    }
  };
  long limit = positions;
  if (a.causal) limit = min(limit, (long)a.start + row + 1);
  walk(a.main, limit);
  if constexpr (TAILS) {
    KvView w = a.tail;
    w.k += (size_t)row * w.layer_bytes;
    w.v += (size_t)row * w.layer_bytes;
    w.ks += (size_t)row * w.layer_scales;
    w.vs += (size_t)row * w.layer_scales;
    walk(w, lens.len[row]);
  }
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) sm_o[wave - 1][lane + 64 * i] = o[i];
    if (lane == 0) {
      sm_m[wave - 1] = m;
      sm_l[wave - 1] = l;
    }
  }
  __syncthreads();
  if (wave > 0) return;
  for (int p = 0; p < 3; ++p) {
    const float mn = fmaxf(m, sm_m[p]), ms = mn == -INFINITY ? 0.f : mn;
    const double f1 = __builtin_amdgcn_exp2f(m - ms), f2 = __builtin_amdgcn_exp2f(sm_m[p] - ms);
    m = mn;
    l = l * f1 + sm_l[p] * f2;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * f1 + sm_o[p][lane + 64 * i] * f2;
  }
  float* dst = a.out + ((size_t)row * n_q + hq) * hd;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 64 * i < hd) dst[lane + 64 * i] = (float)(o[i] / l);
}

// ---- plans ------------------------------------------------------------------------
struct RowsPlan {
  bool generic = false;
  int nb = 0, wc = 0;  // narrow: blocks of 16 columns; wide: waves of 32
  bool fold = false;           // narrow: in the launch
  int n_cb = 0, n_splits = 0, split_len = 128;
  int t_cb = 0, t_splits = 0, t_split_len = 128;
  size_t rows = 0;  // of one launch (sequences go in batches of kMaxEach)
  size_t slots() const { return (size_t)n_splits + t_splits; }
  int columns() const { return nb ? 16 * nb : 32 * wc; }  // of a main item
};

constexpr int kPosStep = 128;

// Splits of `positions` for `units` independent items so that the launch has
// about `want` of them: lengths in whole steps.
void split_positions(long positions, long units, long want, int* n_splits, int* split_len) {
  const long steps = (positions + kPosStep - 1) / kPosStep;
  const long n = std::max<long>(1, std::min<long>(steps, want / std::max<long>(units, 1)));
  const long per = (steps + n - 1) / n;
  *split_len = (int)(per * kPosStep);
  *n_splits = (int)((steps + per - 1) / per);
}

// A launch's shape by the time each choice would take: whether its main items
// are narrow (32 columns, 4 waves) or wide and of how many columns, and into how
// many splits they and the tails are cut. The times (us) are fitted on this card
// to 45 shapes, chunks of 5..1000 rows and batches of 8..100 sequences at 0..16000
// positions, each in every column count and its better split lengths, four caches
// in turn, as a model's layers are; what counts is that they rank the choices as
// those measure (the choice is 0.8 % off the best one on the average). Both sides,
// us, of one cache unless said:
// 77 rows at 901, narrow in 2, 3, 4 splits 16.3, 16.0, 18.6, wide with 2, 4, 8 waves
// of columns 21.2, 22.4, 23.8; 200 at 4000, four caches, narrow 60.9, wide with 4, 8
// waves 49.8, 47.1; 512 at 1000, narrow 35.6, wide 57.9, 46.2, 43.7; 1000
// at 12000, narrow 485, wide 539, 449, 386; 64 x 4000 Q8_0, narrow 26.8, wide 32.9,
// 31.9, 34.3; 64 x 16000 f16 56.4, and 66.3, 57.6, 53.6 (four caches in turn 62.3,
// and 70.9, 59.1, 55.1): there the model picks the narrow form, 13 % off.
// A wide item takes a CU for 7.4 (starting, loading its queries, storing) and `c`
// per 128 positions. A narrow one takes 5.4 and `n1` alone on its CU, 7.0 and `n2`
// beside another (f32's registers leave no room for one). What the card does not
// hold at once goes in rounds, which a chunk's items, the later ones longer, fill
// in part. A tail is four waves' work of 1 to 2 per 128 positions, beside the main
// items. A partial's floats are written and read once.
void plan_shape(RowsPlan& p, long positions, long cols, long heads, int elem, long tails, long longest, long columns,
                long chunk) {
  const long steps = (positions + kPosStep - 1) / kPosStep;
  const bool f32 = elem == RV_ELEM_F32, f16 = elem == RV_ELEM_F16;
  const double n1 = f32 ? 2.87 : f16 ? 1.3 : 1.42, n2 = f32 ? n1 : f16 ? 2.39 : 2.27;
  const double share = 1 - 0.5 * chunk / positions;  // of the positions, that a chunk's rows see on the average
  const long room = (f32 ? 1 : 2) * kCUs;  // narrow items at once
  double best = 1e300;
  for (long t_want : {kCUs / 2, kCUs, 2 * kCUs}) {
    int t_splits = 0, t_len = kPosStep;
    if (tails && longest)
      split_positions(longest, tails, t_want, &t_splits, &t_len);
    else if (t_want != kCUs)
      continue;
    const double t_steps = t_len / kPosStep;
    for (int wc : {0, 2, 4, 8}) {
      if (wc == 2 && f32) continue;  // (its LDS tiles are twice as large)
      if (columns && columns != (wc ? 32 * wc : 32)) continue;
      const double c = f32   ? (wc == 4 ? 7.86 : 10.1)
                       : f16 ? (wc == 2 ? 2.72 : wc == 4 ? 3.62 : 5.96)
                             : (wc == 2 ? 2.5 : wc == 4 ? 4.07 : 6.23);
      const double t_tail = !t_splits ? 1 : wc ? 10.9 + 2.0 * t_steps : 5.4 + 1.05 * t_steps;
      const long t_wgs = wc ? (tails * t_splits + 1) / 2 : tails * t_splits;
      const long units = heads * ((cols + (wc ? 32 * wc : 32) - 1) / (wc ? 32 * wc : 32));
      long n = 1;
      for (long prev = 0; n <= steps; n = n == steps ? n + 1 : std::min(steps, n < 4 ? n + 1 : n * 5 / 4 + 1)) {
        const long per = (steps + n - 1) / n, splits = (steps + per - 1) / per;
        if (splits == prev) continue;
        prev = splits;
        const long items = units * splits;
        if (items > 4 * kCUs && n > 1) break;
        double total;
        if (wc) {
          const double t = 7.4 + c * per, mean = 7.4 + c * per * share;
          // CUs the tails take meanwhile, one after the other on each.
          const long in_a_row = std::max(1L, (long)(t / t_tail)), t_cus = (t_wgs + in_a_row - 1) / in_a_row;
          if (items + t_cus <= kCUs) {
            total = std::max(t, t_tail);
          } else {
            total = t * ((items + kCUs - 1) / kCUs);
            if (chunk)
              total = std::max(t, std::min(total, items * mean / kCUs + 0.97 * t));
            else
              total = std::max(total, (items * t + t_wgs * t_tail) / kCUs + 0.12 * t);
          }
        } else {
          const double alone = 5.4 + n1 * per, beside = f32 ? alone : 7.0 + n2 * per;
          if (items + t_wgs <= kCUs) {
            total = std::max(alone, t_tail);
          } else if (items + t_wgs <= room) {
            total = std::max(items > kCUs ? beside : alone + 0.3 * (beside - alone) * std::min(1.0, t_tail / alone), t_tail);
          } else {
            const long rounds = (items + room - 1) / room;
            const long fit = (rounds * room - items) * (long)(beside / t_tail);
            total = rounds * beside;
            if (chunk) total = std::max(beside, std::min(total, items * (7.0 + n2 * per * share) / room + 0.32 * beside));
            total += 2.15 * t_tail * std::max(0L, t_wgs - fit) / room;
          }
        }
        const long slots = splits + t_splits;
        if (slots > 1) total += 4.6 + slots * cols * heads * (kD + 2) * 8 / 7.5e6;
        if (total < best) {
          best = total;
          p.nb = wc ? 0 : 2;
          p.wc = wc;
          p.n_splits = (int)splits;
          p.split_len = (int)(per * kPosStep);
          p.t_splits = t_splits;
          p.t_split_len = t_len;
        }
      }
    }
  }
}

RowsPlan plan_rows(const RowsCall& c, const rv_kv* owner) {
  RowsPlan p;
  const rv_kv* g = c.main ? c.main : c.tails;
  p.generic = g->head_dim != (size_t)kD;
  p.rows = c.tails ? std::min<size_t>(c.rows, kMaxEach) : c.rows;
  if (p.generic) return p;
  // Planned for all kv heads, so that a range of them takes the whole call's splits
  // and its outputs are that part of the whole call's, bit for bit.
  const long group = (long)(c.n_q_heads / g->n_kv_heads), heads = (long)g->n_kv_heads;
  const long cols = (long)p.rows * group;
  const long positions = c.main ? (long)c.positions : 0;
  const bool causal = c.causal && c.rows > 1;  // (one row: its limit is `positions`)
  long longest = 0;
  if (c.tails) {
    p.t_cb = (int)((group + 15) / 16);
    for (size_t i = 0; i < c.rows; ++i) longest = std::max(longest, (long)c.tails->lens[c.tail_layer + i]);
  }
  const long tails = heads * p.t_cb * (long)p.rows;
  if (positions && (cols > 32 || causal)) {
    const long k = (long)owner->tune_rows_columns;
    // (narrow column blocks are a grid's z, 65535 at most)
    const bool known = (k == 32 && cols <= 32 * 65535L) || (k == 64 && g->elem != RV_ELEM_F32) || k == 128 || k == 256;
    plan_shape(p, positions, cols, heads, g->elem, tails, longest, known ? k : 0, causal ? (long)c.rows : 0);
  } else {
    // One narrow block of columns a kv head. A decode's splits, 32 query heads over
    // 4 kv heads, us: 200 positions whole 6.3, in two 7.5; 400 in four 7.8, whole
    // 8.0; 1000 in eight 7.8, in four 8.6; 2000 in 16 8.7, in 8 9.6; 4096 in 16 9.7,
    // in 32 10.0; 16384 in 64 12.0, in 128 14.3; 131000 in 64 32.5, in 128 32.2.
    p.nb = cols <= 16 ? 1 : 2;
    if (positions && positions <= 2 * kPosStep) {
      p.n_splits = 1;
      p.split_len = 2 * kPosStep;
    } else if (positions) {
      split_positions(positions, heads, positions <= 2 * kFold * kPosStep ? kFold * heads : kCUs, &p.n_splits, &p.split_len);
    }
    if (longest) split_positions(longest, tails, 2 * kCUs, &p.t_splits, &p.t_split_len);
  }
  if (positions && owner->tune_decode_split_len > 0) {
    p.split_len = (int)((std::min<int64_t>(owner->tune_decode_split_len, 1 << 30) + kPosStep - 1) / kPosStep * kPosStep);
    p.n_splits = (int)((positions + p.split_len - 1) / p.split_len);
  }
  if (positions && causal && owner->tune_prefill_kv_split > 0) {
    const long n = std::min<long>(owner->tune_prefill_kv_split, (positions + kPosStep - 1) / kPosStep);
    p.split_len = (int)(((positions + n - 1) / n + kPosStep - 1) / kPosStep * kPosStep);
    p.n_splits = (int)((positions + p.split_len - 1) / p.split_len);
  }
  // Splits folded by the launch: 1.3 us of its own against 4.3 for a second one,
  // while they are few (and their offsets within 31 bits).
  p.fold = cols <= 32 && !c.tails && !causal && p.n_splits > 1 && p.n_splits <= kFold && heads < 4096;
  if (p.columns()) p.n_cb = (int)((cols + p.columns() - 1) / p.columns());
  return p;
}

// Floats of one main slot's and one tail slot's partials (whole blocks of
// columns), for `n` rows.
size_t main_floats(const RowsPlan& p, size_t n, size_t group, size_t heads) {
  const size_t b = p.nb ? 16 : 32;
  return heads * ((n * group + b - 1) / b) * b * kD;
}
size_t tail_floats(const RowsPlan& p, size_t n, size_t heads) { return n * heads * p.t_cb * 16 * kD; }

// A launch's workgroups of main items.
size_t main_items(const RowsPlan& p, size_t heads) { return (heads * p.n_splits * p.n_cb + 7) / 8 * 8; }

// Floats that its wide items' sums are put aside in.
size_t aside_floats(const RowsPlan& p, size_t heads) {
  return p.wc && p.split_len > kWalkWide ? main_items(p, heads) * 8 * 17 * 64 * 4 : 0;
}

size_t plan_floats(const RowsPlan& p, const RowsCall& c) {
  if (p.generic) return 0;
  const rv_kv* g = c.main ? c.main : c.tails;
  const size_t group = c.n_q_heads / g->n_kv_heads, heads = c.kv_hi - c.kv_lo;
  if (p.slots() <= 1) return aside_floats(p, heads);
  return aside_floats(p, heads) + p.n_splits * main_floats(p, p.rows, group, heads) + p.t_splits * tail_floats(p, p.rows, heads) +
         2 * p.slots() * p.rows * group * heads;
}

template <int G>
void launch_merge_g(const RowsArgs& a, int items, bool narrow, const TailLens* lens, hipStream_t s) {
  constexpr int W = G < 4 ? 4 : G;
  const dim3 grid((unsigned)((items + W / G - 1) / (W / G))), block(64 * W);
  if (lens)
    hipLaunchKernelGGL((rows_merge_kernel<G, true>), grid, block, 0, s, a, (int)narrow, *lens);
  else
    hipLaunchKernelGGL((rows_merge_kernel<G, false>), grid, block, 0, s, a, (int)narrow, NoLens{});
}

template <typename T, bool TAILS, bool WALK, typename L>
void launch_narrow(const RowsPlan& p, const TimedPair& tp, const RowsArgs& a, unsigned tail_items, hipStream_t s,
                   const L& lens) {
  if constexpr (TAILS) {
    const dim3 grid((unsigned)a.main_items + tail_items);
    if (p.nb == 1)
      launch_timed(tp, rows_narrow_kernel<T, 1, true, false, WALK>, grid, dim3(256), s, a, lens);
    else
      launch_timed(tp, rows_narrow_kernel<T, 2, true, false, WALK>, grid, dim3(256), s, a, lens);
  } else {
    const dim3 grid((unsigned)a.n_splits, (unsigned)a.n_heads, (unsigned)a.n_cb);
    if (a.causal)
      launch_timed(tp, rows_narrow_kernel<T, 2, false, true, WALK>, grid, dim3(256), s, a, lens);
    else if (p.nb == 2)
      launch_timed(tp, rows_narrow_kernel<T, 2, false, false, WALK>, grid, dim3(256), s, a, lens);
    else
      launch_timed(tp, rows_narrow_kernel<T, 1, false, false, WALK>, grid, dim3(256), s, a, lens);
  }
}

template <typename T, bool HL, bool TAILS, typename L>
void launch_plan(const RowsPlan& p, const TimedPair& tp, const RowsArgs& a, unsigned tail_items, hipStream_t s,
                 const L& lens) {
  if (p.nb) {
    // (the longer form costs short items 2 to 7 %, f16 ones of 32 columns 24 %)
    if (std::max(p.split_len, p.t_split_len) > NW * kWalkNarrow)
      launch_narrow<T, TAILS, true>(p, tp, a, tail_items, s, lens);
    else
      launch_narrow<T, TAILS, false>(p, tp, a, tail_items, s, lens);
    return;
  }
  const dim3 grid((unsigned)a.main_items + (tail_items + 1) / 2);
  if (p.wc == 8)
    launch_timed(tp, rows_wide_kernel<T, 8, HL, TAILS>, grid, dim3(512), s, a, lens);
  else if (p.wc == 4)
    launch_timed(tp, rows_wide_kernel<T, 4, HL, TAILS>, grid, dim3(512), s, a, lens);
  else if constexpr (!Lo<T>::value)
    launch_timed(tp, rows_wide_kernel<T, 2, HL, TAILS>, grid, dim3(512), s, a, lens);
}

}  // namespace

size_t rows_ws_need(const rv_kv* owner, const RowsCall& c) { return plan_floats(plan_rows(c, owner), c) * sizeof(float); }

size_t rows_ws_bound(const rv_kv* kv) {
  if (kv->head_dim != (size_t)kD) return 0;
  // A decode's items: kFold or fewer per kv head, or kCUs in all.
  return std::max<size_t>(kCUs, kFold * kv->n_kv_heads) * 16 * (kD + 2) * sizeof(float);
}

HipStatus launch_rows(rv_kv* owner, const RowsCall& c, hipStream_t s, const Workspace* ws) {
  HipStatus st;
  const rv_kv* g = c.main ? c.main : c.tails;
  const RowsPlan p = plan_rows(c, owner);
  const size_t need = plan_floats(p, c) * sizeof(float);
  float* base = nullptr;
  if (ws) {
    if (need > ws->bytes) {
      st.e = hipErrorInvalidValue;
      st.what = "decode scratch too small";
      return st;
    }
    base = (float*)ws->base;
  } else if (need) {
    // Doubled (up to a GiB more), so that what a growing context or batch has
    // outgrown, kept for the graphs captured over it, does not add up.
    st = ensure_workspace(owner, need, std::min(2 * owner->ws_bytes, need + ((size_t)1 << 30)));
    if (st.e != hipSuccess) return st;
    base = (float*)owner->ws;
  }
  const int group = (int)(c.n_q_heads / g->n_kv_heads);
  const size_t hd = g->head_dim;
  for (size_t r0 = 0; r0 < c.rows; r0 += p.rows) {
    const size_t n = std::min(p.rows, c.rows - r0);
    RowsArgs a{};
    if (c.main) a.main = kv_view(c.main, c.layer);
    TailLens lens{};
    if (c.tails) {
      a.tail = kv_view(c.tails, c.tail_layer + r0);
      for (size_t i = 0; i < n; ++i) lens.len[i] = (uint32_t)c.tails->lens[c.tail_layer + r0 + i];
    }
    a.q = c.q + r0 * c.n_q_heads * hd;
    a.out = c.out + r0 * (c.kv_hi - c.kv_lo) * group * hd;
    a.rows = (int)n;
    a.n_q_heads = (int)c.n_q_heads;
    a.group = group;
    a.kv_lo = (int)c.kv_lo;
    a.n_heads = (int)(c.kv_hi - c.kv_lo);
    a.positions = (int)c.positions;
    a.start = (int)c.start;
    a.causal = c.causal && c.rows > 1;  // (one row: its limit is `positions`)
    a.d_pos = c.d_pos;
    a.qscale = c.scale * kLog2e;
    if (p.generic) {
      const dim3 grid((unsigned)(n * a.n_heads * group)), block(256);
#define RV_GENERIC(T)                                                                                  \
  if (c.tails)                                                                                         \
    hipLaunchKernelGGL((rows_generic_kernel<T, true>), grid, block, 0, s, a, (int)hd, lens);           \
  else                                                                                                 \
    hipLaunchKernelGGL((rows_generic_kernel<T, false>), grid, block, 0, s, a, (int)hd, NoLens{})
      if (g->elem == RV_ELEM_Q8_0) {
        RV_GENERIC(Q8);
      } else if (g->elem == RV_ELEM_F32) {
        RV_GENERIC(float);
      } else {
        RV_GENERIC(_Float16);
      }
#undef RV_GENERIC
    } else {
      a.aside = (f32x4*)base;
      a.part = base ? base + aside_floats(p, a.n_heads) : nullptr;
      a.slot_floats = main_floats(p, n, group, a.n_heads);
      a.t_base = p.n_splits * a.slot_floats;
      a.t_slot_floats = tail_floats(p, n, a.n_heads);
      a.ml = base ? a.part + a.t_base + p.t_splits * a.t_slot_floats : nullptr;
      a.n_cb = (int)((n * group + p.columns() - 1) / p.columns());
      a.n_splits = p.n_splits;
      a.split_len = p.split_len;
      a.t_cb = p.t_cb;
      a.t_splits = p.t_splits;
      a.t_split_len = p.t_split_len;
      a.main_items = (int)((a.n_heads * a.n_splits * a.n_cb + 7) / 8 * 8);
      a.single = p.slots() == 1;
      a.tickets = p.fold ? xcd_tickets(owner) : nullptr;
      const unsigned tail_items = (unsigned)(n * a.n_heads * a.t_cb * a.t_splits);
      const TimedPair tp = ws ? TimedPair{} : timing_pair(owner, s);
      if (c.tails) {
        if (g->elem == RV_ELEM_Q8_0)
          launch_plan<Q8, true, true>(p, tp, a, tail_items, s, lens);
        else if (g->elem == RV_ELEM_F32)
          launch_plan<float, true, true>(p, tp, a, tail_items, s, lens);
        else
          launch_plan<_Float16, true, true>(p, tp, a, tail_items, s, lens);
      } else if (c.split) {
        launch_plan<Q8, true, false>(p, tp, a, 0, s, NoLens{});
      } else {
        launch_plan<Q8, false, false>(p, tp, a, 0, s, NoLens{});
      }
      if (!a.single && !p.fold) {
        const int merges = 16 * a.n_heads * (int)((n * group + 31) / 32);
        const TailLens* tl = c.tails ? &lens : nullptr;
        if (p.slots() <= 4)
          launch_merge_g<1>(a, merges, p.nb != 0, tl, s);
        else if (p.slots() <= 32)
          launch_merge_g<4>(a, merges, p.nb != 0, tl, s);
        else
          launch_merge_g<16>(a, merges, p.nb != 0, tl, s);
      }
    }
    st.e = hipGetLastError();
    if (st.e != hipSuccess) {
      st.what = "rows attention launch";
      return st;
    }
  }
  return st;
}

}  // namespace rv
