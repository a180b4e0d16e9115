// rv_paged_attn.hip — attention of one new token of each sequence of a batch
// over its pages.
//
// o = sum_t p_t v_t / sum_t p_t, p_t = exp(scale * (q . k_t) - m), in one pass over
// the rows with the running maximum m. Where f32 pages may hold values of V whose sum
// over the sequence's n rows passes the floats' range, p_t is times 2^-k < 1 / (2 n)
// in numerator and denominator alike.
//
// The lengths are on the device and ragged, so the work is dealt there: a unit is
// kUnitRows rows of one item (a sequence's kv head, or a part of its query
// heads), the units of the batch in order are cut into equal ranges, one a
// workgroup, and every wave finds its workgroup's range by a prefix sum over the
// lengths. An item inside one range is finished there; one that is cut leaves a
// partial (weighted sum of v, maximum, sum) per range, at most two a workgroup
// (its first item and its last). The workgroup that leaves an item's last partial
// joins them all, in order, so that results do not depend on which that is. Where
// they are all of a group (up to 16 workgroups of one XCD) they pass through its L2,
// where they are many first those of each group do (loads at device scope bring a CU
// some 12 bytes a cycle, loads from its L2 several times that), and else, and across
// groups, they are stored and loaded at device scope, since the XCDs' L2s do not see
// each other's lines. Partials are counted by tickets, two sets of them in turn by the
// launch, each cleared by the launch after its own.
//
// Bound by the pages' bytes where there are many: f16, 32 query heads over 4 of 128, 64
// sequences of up to 16000 rows 188 us, 6.6 TB/s (a streaming read's rate); one of 131000
// 46.5, 5.8 TB/s. Q8_0 by no one unit (32 of up to 8192 rows 38 us, 3.8 TB/s: vector
// instructions 56 % of the cycles, matrix instructions 12 %, waves waiting 24 %); few rows
// by one phase after the other: 100 rows 5.8, 4096 11.3 us, a third of it the joins.
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
  int slots;          // log2 of the XCDs that workgroups are known to be dealt to in turn
  int most, few;      // log2 of the ranges there may be (cut_units)
  Turn* turns;        // a word a workgroup (rv_pages.hpp)
  unsigned* tickets;  // two sets of [group][2], then one an item; from one set to the other:
  size_t set_words;
  uint32_t n_tickets;
  // [range][2], then [group][2]: rows [cols][hd], then (maximum, sum) of each column
  // (partial_floats).
  float* part;
  uint32_t part_bytes;
};

constexpr uint32_t kMaxRanges = 2 * kCUs, kGroups = kMaxRanges / kGroup;
static_assert(kTurns % kMaxRanges == 0, "a turn's word for every workgroup");
constexpr uint32_t kRefused = 0xFFFFFFFFu;

// Rows a sequence of this length attends, kRefused where the table has not so many.
__device__ __forceinline__ uint32_t rows_of_len(const PagedView& w, const AttnArgs& a, int len) {
  return (uint32_t)attended_rows(w.t, len, a.step);
}

__device__ __forceinline__ uint32_t units_of_rows(uint32_t rows) { return rows == kRefused ? 0 : units_of(rows); }

// Sum of the lanes up to and including this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
#define RV_SHIFTED(CTRL, ROWS) (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, false)
  x += RV_SHIFTED(0x111, 0xF);  // row_shr:1, 2, 4, 8: within 16 lanes
  x += RV_SHIFTED(0x112, 0xF);
  x += RV_SHIFTED(0x114, 0xF);
  x += RV_SHIFTED(0x118, 0xF);
  x += RV_SHIFTED(0x142, 0xA);  // row_bcast:15 into the odd rows
  x += RV_SHIFTED(0x143, 0xC);  // row_bcast:31 into the upper half
#undef RV_SHIFTED
  return x;
}

// A power of two that n weights of at most 1 each times it make less than one half of.
__device__ __forceinline__ float weight_unit(uint32_t n) { return ldexpf(1.f, __builtin_clz(n) - 33); }

// The average y that a sum o gives: of finite values finite, whatever its last rounding.
__device__ __forceinline__ float finite(float o, float y) {
  return __builtin_isinf(y) && !__builtin_isinf(o) ? __builtin_copysignf(0x1.fffffep127f, y) : y;
}

// ---- partials ---------------------------------------------------------------------

// Cache policies of the buffer instructions: the sc1 bit, device scope; the sc0 bit of a
// load, workgroup scope, which the CU's L1 may serve. That is enough for partials that
// this XCD wrote: a launch begins with an empty L1, a partial's lines are its own, and
// they are written once, before the first load of any of them.
constexpr int kDeviceScope = 16, kXcdScope = 1;

struct Partials {
  __amdgpu_buffer_rsrc_t rs;
  int cols, hd;
  uint32_t bytes;  // of one
  __device__ __forceinline__ Partials(const AttnArgs& a, int hd_)
      : rs(__builtin_amdgcn_make_buffer_rsrc(a.part, (short)0, (int)a.part_bytes, 0x00020000)),
        cols(a.cols),
        hd(hd_),
        bytes(partial_floats((uint32_t)a.cols, (uint32_t)hd_) * 4u) {}
  // Byte offset of a partial (2 * range + which; the groups' behind them); of column
  // c's (maximum, sum) in it.
  __device__ __forceinline__ uint32_t at(uint32_t i) const { return i * bytes; }
  __device__ __forceinline__ uint32_t stat(int c) const { return (uint32_t)(cols * hd + 2 * c) * 4u; }
  // Stores to be seen on this XCD, or on all.
  __device__ __forceinline__ void put(uint32_t o, float x, bool here) const {
    if (here)
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, x), rs, o, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(int, x), rs, o, 0, kDeviceScope);
  }
  __device__ __forceinline__ void put(uint32_t o, f32x4 x, bool here) const {
    if (here)
      __builtin_amdgcn_raw_buffer_store_b128(x, rs, o, 0, 0);
    else
      __builtin_amdgcn_raw_buffer_store_b128(x, rs, o, 0, kDeviceScope);
  }
  __device__ __forceinline__ void put_stat(uint32_t p, int c, float m, float l, bool here) const {
    put(p + stat(c), m, here);
    put(p + stat(c) + 4, l, here);
  }
  template <int POLICY>
  __device__ __forceinline__ float word(uint32_t o) const {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, o, 0, POLICY));
  }
};

constexpr uint32_t kMostPieces = 32;  // that are joined at once

// Joins `count` partials (at most kMostPieces), in order, partial `first` and then
// rest, rest + 2, ..: into `out` (ncols rows of hd), or into partial `to` for all
// XCDs. What a load costs the CU's address unit is by the instruction: LANES lanes
// have a column, VEC of its values each, load its partials' (maximum, sum) one a lane,
// and pass their factors on by lane permutes; 16 partials' values are in flight.
template <int VEC, int LANES, int POLICY>
__device__ __forceinline__ void join(const Partials& p, uint32_t first, uint32_t rest, uint32_t count, int ncols,
                                     float* out, uint32_t to, bool large) {
  typedef float Row __attribute__((ext_vector_type(VEC)));
  constexpr uint32_t kBatch = 16;
  constexpr int kStats = LANES < (int)kMostPieces ? (int)kMostPieces / LANES : 1, kColumns = 256 / LANES;  // a lane's; of the workgroup at once
  const int lane = threadIdx.x & 63, mine = lane & (LANES - 1);
  const uint32_t one = p.at(1);
  auto place = [&](uint32_t i) { return (i ? rest + 2 * (i - 1) : first) * one; };
  for (int c0 = 0; c0 < ncols; c0 += kColumns) {
    const int cc = c0 + (int)threadIdx.x / LANES, c = min(cc, ncols - 1);
    float m[kStats], l[kStats], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < kStats; ++i) {
      const uint32_t k = mine + LANES * i, at = place(min(k, count - 1)) + p.stat(c);
      m[i] = p.word<POLICY>(at);
      l[i] = p.word<POLICY>(at + 4);
    }
    for (int d = mine * VEC; d < (p.hd + LANES * VEC - 1) / (LANES * VEC) * (LANES * VEC); d += LANES * VEC) {
      const uint32_t row = (uint32_t)(c * p.hd + min(d, p.hd - VEC)) * 4u;
      Row o = (Row)0.f;
      for (uint32_t b0 = 0; b0 < count; b0 += kBatch) {
        Row x[kBatch];
        uint32_t at = place(b0) + row;
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
          if (i % 4 == 0 && b0 + i >= count) break;  // (past the last, up to three: it again, not counted)
          if constexpr (VEC == 4)
            x[i] = __builtin_bit_cast(Row, __builtin_amdgcn_raw_buffer_load_b128(p.rs, at, 0, POLICY));
          else
            x[i] = p.word<POLICY>(at);
          if (b0 + i + 1 < count) at = b0 + i ? at + 2 * one : rest * one + row;
        }
        if (b0 == 0 && d == mine * VEC) {
#pragma unroll
          for (int i = 0; i < kStats; ++i) {
            const bool in = mine + LANES * i < (int)count;
            m[i] = in ? m[i] : -INFINITY;
            l[i] = in ? l[i] : 0.f;
            top = fmaxf(top, m[i]);
          }
          top = group_max<16>(top);
          if (LANES >= 32) top = swap_max<16>(top);
          if (LANES >= 64) top = swap_max<32>(top);
          // (Where every score is minus infinity or NaN nothing is scaled, and the sums
          // carry what there is.)
#pragma unroll
          for (int i = 0; i < kStats; ++i) {
            m[i] = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[i] - top);
            sum += m[i] * l[i];
          }
          sum = group_sum<16>(sum);
          if (LANES >= 32) sum = swap_sum<16>(sum);
          if (LANES >= 64) sum = swap_sum<32>(sum);
        }
        float fs = m[0];  // (a batch's factors are all in one register)
#pragma unroll
        for (int s = 1; s < kStats; ++s) fs = b0 / LANES == (uint32_t)s ? m[s] : fs;
        const int from = (lane & ~(LANES - 1)) + (int)(b0 & (LANES - 1));
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
          if (i % 4 == 0 && b0 + i >= count) break;
          const float f = __shfl(fs, from + (int)i, 64);
          o += x[i] * (b0 + i < count ? f : 0.f);
        }
      }
      if (cc >= ncols || d >= p.hd) continue;
      if (out) {
        const float inv = 1.f / sum;
        Row y = o * inv;
        if (large) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = finite(o[e], y[e]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[(long)c * p.hd + d + e] = y[e];
      } else {
        if constexpr (VEC == 4)
          p.put(p.at(to) + row, o, false);
        else
          p.put(p.at(to) + row, o[0], false);
        if (d == 0) p.put_stat(p.at(to), c, top, sum, false);
      }
    }
  }
}

// Whether this workgroup is the last of `n` to come here, its stores of partials
// complete.
__device__ __forceinline__ bool last_of(unsigned* ticket, uint32_t n, unsigned& drawn) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) drawn = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const bool last = drawn == n - 1;
  __syncthreads();  // (the next draw writes it)
  return last;
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

// Any head width: one query head an item, a wave four rows at a time, the head's
// values over its lanes, so that a row is read again for every query head of its
// group: for the widths that tiles do not take. 16 sequences of 2000
// f16 rows, 4 kv heads of 8 query heads of 100: 232 us (791 a row at a time; 182 with
// sums of f32; 20 the tiles at 104).
template <typename T>
struct Plain {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int kPer = kMaxHalf * 2 / 64;
  static constexpr int kVec = 1, kLanes = 64;
  struct Shared {
    float o[4][kMaxHalf * 2];
    float m[4], l[4];
  };
  // Rows [p0, p1) of sequence s, kv head h, query head qh (of the whole): the
  // output where `whole`, else the partial that where() names.
  template <typename Where>
  static __device__ __forceinline__ void segment(const PagedView& w, const AttnArgs& a, Shared& sh, uint32_t s, int h,
                                                 int qh, int, uint32_t p0, uint32_t p1, float unit, bool whole,
                                                 const Partials& pt, Where where) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const float* q = a.q + s * a.q_stride + (long)qh * w.hd;
    const float scale = a.scale * kLog2e;
    float x[kPer];
    double o[kPer];  // (in f32 many small weights behind a large one would be dropped)
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int d = lane + 64 * j;
      x[j] = d < w.hd ? q[d] : 0.f;
      o[j] = 0.0;
    }
    float m = -INFINITY;
    double l = 0.0;
    // Four rows of one page at a time; past the last row it again, without weight.
    for (uint32_t b = p0 + 4 * wv; b < p1; b += 16) {
      const uint32_t page = (uint32_t)w.t.ids[(long)s * w.t.stride + (b >> w.t.shift)];
      if (page >= w.t.n_pages) {
        if (lane == 0) paged_refuse(w, RV_PAGED_PAGE_OUT_OF_RANGE, s, page, w.t.n_pages);
        l = NAN;
        continue;
      }
      const size_t hp = (size_t)page * w.n_kv + h;
      const uint32_t mask = (1u << w.t.shift) - 1;
      uint32_t row[4];
      float y[4] = {}, v[4][kPer];
#pragma unroll
      for (int r = 0; r < 4; ++r) row[r] = min(b + r, p1 - 1) & mask;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        if (64 * j >= w.hd) break;
        const int d = min(lane + 64 * j, w.hd - 1);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          y[r] += x[j] * paged_value<T>(w, false, hp, row[r], d);
          v[r][j] = paged_value<T>(w, true, hp, row[r], d);
        }
      }
      float mn = m;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[r] = b + r < p1 ? swap_sum<32>(swap_sum<16>(group_sum<16>(y[r]))) * scale : -INFINITY;
        mn = fmaxf(mn, y[r]);
      }
      const float c = mn == -INFINITY ? 1.f : exp2f(m - mn);
      m = mn;
      l *= c;
#pragma unroll
      for (int j = 0; j < kPer; ++j) o[j] *= c;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float e = y[r] == -INFINITY ? 0.f : exp2f(y[r] - mn);  // (NaN of a NaN)
        l += e;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (64 * j < w.hd) o[j] += (double)e * v[r][j];
      }
    }
    __syncthreads();
    if (lane == 0) sh.m[wv] = m, sh.l[wv] = (float)(l * unit);
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh.o[wv][lane + 64 * j] = (float)(o[j] * unit);
    __syncthreads();
    bool here = false;
    const uint32_t part = whole ? 0 : where(here);
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
        a.out[s * a.out_stride + (long)qh * w.hd + d] = unit != 1.f ? finite(y, y / sum) : y / sum;
      else
        pt.put(part + 4u * d, y, here);
    }
    if (!whole && threadIdx.x == 0) pt.put_stat(part, 0, top, sum, here);
  }
};

// Heads of whole 16-byte pieces, up to 256 wide (padded to HDP): up to 16 query
// heads of one kv head are the 16 columns of matrix instructions, a wave takes
// kRows rows at a time and every fourth such tile of its segment (16 rows of f32, and
// where 32 of 256 values would leave registers for one wave a SIMD only: f16, 128
// sequences of 300 45.4 -> 41.0 us; Q8_0, 32 of up to 4000 57.7 -> 53.5).
//
// Scores: S[row][column] = K (A operand: a row a lane, 16 bytes of it straight from
// memory) times q (B operand, in registers for the whole segment). f16 and Q8_0
// rows: 16x16x32 f16, q as hi + lo halves scaled by a power of two that puts its
// largest value in [2^14, 2^15); f32 rows: 16x16x4 f32. A lane then holds four
// rows of one column (of each 16 rows), which is the A operand of the second
// product as it stands when the rows are counted in that order: O[column][d] = P
// times V, for which a lane loads whole 16-byte pieces of those same rows of V and
// turns the 8 x 8 halves around in registers. P (times 2^15, so that weights down
// to 2^-38 of the largest count) is hi + lo halves as well.
//
// Bound by the rows' bytes: a tile of 32 f16 rows of 128 is 16 KiB and 32 matrix
// instructions of 16 cycles, and a SIMD's share of the memory rate brings it in
// some 8000 cycles. So the loads are what is arranged: the next tile's K is asked
// for as soon as this one's scores are done, its V after this one's product, each
// into the registers just freed, and page ids a tile ahead of that.
template <typename T, int HDP, bool FULL>
struct Tiled {
  static constexpr bool kF32 = std::is_same<T, float>::value, kQ8 = std::is_same<T, Q8>::value;
  static constexpr int kRows = kF32 || (HDP == 256 && FULL) ? 16 : 32, kSub = kRows / 16;
  static constexpr int kStep = 4 * kRows;  // from one of a wave's tiles to its next
  // A sum of f32 drops what is below 2^-24 of it, the many small weights behind a large
  // one whole: a wave's sums are put aside (in LDS) and begun again after so many tiles.
  // So at most 2^-18 of the largest value is lost in the tiles between: a product's rows
  // (32, 16, of f32 4) count down to 2^-25 together. They begin again with what the addition to
  // those put aside has rounded off (the sum s of a and b is off by (a - (s - (s - a))) +
  // (b - (s - a)) exactly), so that nothing is added to that however many tiles there are;
  // but with zero where whole heads of 256 leave no registers for it (f16 and Q8_0, two
  // waves a SIMD: 41 to 56 values spilled): there up to 2^-25 more a time.
  static constexpr uint32_t kAside = kF32 ? 32 : 64;
  static constexpr bool kKeepRest = HDP < 256 || !FULL || kF32;
  static constexpr int VD = kF32 || HDP == 64 ? 4 : 8;  // values of a row of V a lane loads together
  static constexpr int NH = HDP / (16 * VD);
  static constexpr int NK = kF32 ? HDP / 16 : kQ8 ? HDP / 64 : HDP / 32;  // 16-byte loads of a row of K a lane
  static constexpr int NQ = HDP / 32;
  static constexpr int kBytes = kF32 ? 4 : kQ8 ? 1 : 2;
  static constexpr int kVec = 4, kLanes = HDP / 4;
  static __device__ __forceinline__ int width(const PagedView& w) { return FULL ? HDP : w.hd; }
  typedef std::conditional_t<kF32, f32x4, u32x4> KReg;
  typedef std::conditional_t<kF32, f32x4,
                             std::conditional_t<kQ8, std::conditional_t<VD == 8, u32x2, uint32_t>,
                                                std::conditional_t<VD == 8, f16x8, f16x4>>> VReg;
  typedef std::conditional_t<kSub == 2, f16x8, f16x4> PReg;  // a lane's rows of one column of P, or of V
  static __device__ __forceinline__ f32x4 weigh(PReg p, PReg v, f32x4 c) {
    if constexpr (kSub == 2)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(p, v, c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x16f16(p, v, c, 0, 0, 0);
  }
  struct Shared {
    __attribute__((aligned(16))) float o[4][16][HDP + 4];
    float m[4][16], l[4][16];
  };
  struct Tile {
    KReg k[kSub][NK];
    uint16_t ks[kSub][NK];
    VReg v[4 * kSub][NH];
    f16x4 vs[kSub][NH];
  };

  // The first of the eight (f32: four) values of a head that lane group g holds in
  // operand i.
  static __device__ __forceinline__ int q_dim(int i, int g) {
    return kF32 ? 16 * i + 4 * g : kQ8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
  }

  // Loads past the caches (every row is read once): 64 sequences of up to 16000 f16
  // rows 229 -> 203 us. Not of rows below a line of 128 bytes, which would be brought
  // twice: 32 of up to 8000 Q8_0 rows of 64 23.0 us so, 25.2 past the caches. Nor where
  // a narrower head's first values are loaded twice, but for f16: 32 of up to 4000 rows
  // of 96, through the caches | past them: f32 65 | 69, Q8_0 28 | 30, f16 40 | 36.
  template <typename V>
  static __device__ __forceinline__ V stream(const char* p) {
    if constexpr (HDP * kBytes >= 128 && (FULL || (!kF32 && !kQ8 && HDP > 64)))
      return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    else
      return *reinterpret_cast<const V*>(p);
  }

  // Past a head's width its first values are loaded again: of K they meet a q of zero
  // (and are no less finite than their row), of V they make outputs that nobody takes.
  // Rows past the last one are rows of the last page, cleared before they count. So no
  // lane goes another way than the others while the operands are in registers, and
  // nothing waits for a load before its tile's turn (with masks at the loads 32 sequences
  // of up to 4000 f32 rows of 96 109 us, so 65; f16 47, so 36).
  template <typename V>
  static __device__ __forceinline__ V keep(V x, bool in) {
    static_assert(sizeof(V) % 4 == 0, "whole words");
    struct Words {
      uint32_t w[sizeof(V) / 4];
    };
    Words y = __builtin_bit_cast(Words, x);
#pragma unroll
    for (int i = 0; i < (int)sizeof(V) / 4; ++i) y.w[i] &= in ? 0xFFFFFFFFu : 0u;
    return __builtin_bit_cast(V, y);
  }

  static __device__ __forceinline__ void load_k(const PagedView& w, const size_t (&at)[kSub], int g, Tile& t) {
    const int hd = width(w);
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      const char* row = w.k + at[j] * hd * kBytes;
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int d = kF32 ? 16 * i + 4 * g : kQ8 ? 64 * i + 16 * g : 32 * i + 8 * g;
        const int dd = FULL || d < hd ? d : 0;
        t.k[j][i] = stream<KReg>(row + dd * kBytes);
        if constexpr (kQ8) t.ks[j][i] = w.ks[at[j] * (hd / 32) + dd / 32];
      }
    }
  }

  // hp: page * kv heads + head of the rows.
  static __device__ __forceinline__ void load_v(const PagedView& w, const size_t (&hp)[kSub],
                                                const uint32_t (&row)[kSub], int n, Tile& t) {
    const int hd = width(w);
#pragma unroll
    for (int j = 0; j < kSub; ++j) {
      const char* p = w.v + ((hp[j] << w.t.shift) + row[j]) * hd * kBytes;
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int d = 16 * VD * h + VD * n, dd = FULL || d < hd ? d : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) t.v[4 * j + i][h] = stream<VReg>(p + ((size_t)i * hd + dd) * kBytes);
        if constexpr (kQ8)
          t.vs[j][h] =
              *reinterpret_cast<const f16x4*>(w.vs + ((hp[j] * (hd / 32) + dd / 32) << w.t.shift) + row[j]);
      }
    }
  }

  static __device__ __forceinline__ f16x8 widen8(uint32_t a, uint32_t b, _Float16 s) {
    f16x2 p[4];
    q8_widen(a, p[0], p[1]);
    q8_widen(b, p[2], p[3]);
    f16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = p[e >> 1][e & 1] * s;
    return y;
  }

  template <typename Where>
  static __device__ __forceinline__ void segment(const PagedView& w, const AttnArgs& a, Shared& sh, uint32_t s, int h,
                                                 int qh, int ncols, uint32_t p0, uint32_t p1, float unit, bool whole,
                                                 const Partials& pt, Where where) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t mask = (1u << w.t.shift) - 1;
    const int32_t* ids = w.t.ids + (long)s * w.t.stride;
    uint32_t no_page = 0;  // a page id that names no page
    auto fetch = [&](uint32_t b, uint32_t (&id)[kSub]) {
#pragma unroll
      for (int j = 0; j < kSub; ++j) id[j] = (uint32_t)ids[min(b + 16 * j + n, p1 - 1) >> w.t.shift];
    };
    size_t k_at[kSub], v_hp[kSub];
    uint32_t v_row[kSub];
    auto locate = [&](uint32_t b, const uint32_t (&id)[kSub]) {
#pragma unroll
      for (int j = 0; j < kSub; ++j) {
        const bool is = id[j] < w.t.n_pages;
        no_page = is ? no_page : id[j];
        const uint32_t page = is ? id[j] : 0;
        k_at[j] = (((size_t)page * w.n_kv + h) << w.t.shift) + ((b + 16 * j + n) & mask);
        v_hp[j] = (size_t)(uint32_t)__shfl((int)page, 4 * g, 64) * w.n_kv + h;
        v_row[j] = (b + 16 * j + 4 * g) & mask;
      }
    };
    uint32_t b = p0 + wv * kRows;
    const bool any = b < p1;
    Tile t;
    uint32_t id[kSub];
    f32x4 acc[NH * VD];
#pragma unroll
    for (int i = 0; i < NH * VD; ++i) acc[i] = f32x4{};
    float m = -INFINITY, l = 0.f;
    float m_aside = -INFINITY, l_aside = 0.f;
    bool aside = false;
    auto place = [&](int r, int i) { return reinterpret_cast<f32x4*>(&sh.o[wv][4 * g + r][16 * VD * (i / VD) + VD * n + i % VD]); };
    auto put_aside = [&](auto is_last) {
#pragma clang fp contract(off)
      constexpr bool kRest = kKeepRest && !decltype(is_last)::value;
      auto add = [](auto a, auto b, auto& rest) {
        const auto sum = a + b, part = sum - a;
        rest = (a - (sum - part)) + (b - part);
        return sum;
      };
      const float c = m_aside == m ? 1.f : __builtin_amdgcn_exp2f(m_aside - m);
      l_aside = add(l_aside * c, l, l);
      m_aside = m;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = __shfl(c, 4 * g + r, 64);
#pragma unroll
        for (int i = 0; i < NH * VD; i += 4) {
          f32x4 x = {acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]}, rest{};
          if (aside) {
            if constexpr (kRest)
              x = add(*place(r, i) * f, x, rest);
            else
              x += *place(r, i) * f;
          }
          *place(r, i) = x;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i + e][r] = rest[e];
        }
      }
      aside = true;
    };
    if (p1 - p0 > kAside * kStep) __syncthreads();  // (the last segment's reads)
    if (any) {
      fetch(b, id);
      const float* q = a.q + s * a.q_stride + (long)(qh + min(n, ncols - 1)) * w.hd;
      f32x4 x[kF32 ? NK : 2 * NQ];
#pragma unroll
      for (int i = 0; i < (kF32 ? NK : 2 * NQ); ++i) {
        const int d = kF32 ? q_dim(i, g) : q_dim(i >> 1, g) + 4 * (i & 1);
        const bool in = n < ncols && (FULL || d < w.hd);
        x[i] = keep<f32x4>(*reinterpret_cast<const f32x4u*>(q + (FULL || d < w.hd ? d : 0)), in);
      }
      locate(b, id);
      load_k(w, k_at, g, t);
      fetch(b + kStep, id);
      __builtin_amdgcn_sched_barrier(0);  // (loads in the order in which they are waited for)
      load_v(w, v_hp, v_row, n, t);
      __builtin_amdgcn_sched_barrier(0);
      float mul = a.scale * kLog2e;
      f16x8 q_hi[NQ], q_lo[NQ];
      if constexpr (!kF32) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * NQ; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[i][e]));
        top = swap_max<32>(swap_max<16>(top));
        // 2^(14 - its exponent), in two steps where that passes the floats' range.
        const int ex = top > 0.f && top < INFINITY ? 14 - ilogbf(top) : 0;
        mul = ldexpf(mul, -ex);
#pragma unroll
        for (int i = 0; i < NQ; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = ldexpf(x[2 * i + (e >> 2)][e & 3], ex);
            q_hi[i][e] = (_Float16)y;
            q_lo[i][e] = (_Float16)(y - (float)q_hi[i][e]);
          }
      }
      // A tile: its scores, then the next one's K in the place of its own, its part of
      // the output, and the next one's V.
      // A wave's last tile is another instance of the step: in the others every load is
      // unconditional, so that the wait for one is not for those after it as well that
      // another path would not have, and no row is past the last (f16, 8 sequences of 7000
      // 28.5 -> 26.9 us; f32 45.8 -> 43.1; f16, 1000 of 100 74 -> 68).
      auto step = [&](auto is_last, bool first) {
        constexpr bool kLast = decltype(is_last)::value;
        // (Every chain of dependent matrix instructions is as short as it can be: hi and
        // lo apart, the two 16 rows in turn.)
        f32x4 sc[kSub], sl[kSub];
#pragma unroll
        for (int j = 0; j < kSub; ++j) sc[j] = sl[j] = f32x4{};
        if constexpr (kF32) {
#pragma unroll
          for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f32x4& c = i & 1 ? sl[0] : sc[0];
              c = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[0][i][e], x[i][e], c, 0, 0, 0);
            }
        } else {
#pragma unroll
          for (int i = 0; i < NQ; ++i)
#pragma unroll
            for (int j = 0; j < kSub; ++j) {
              f16x8 k;
              if constexpr (kQ8)
                k = widen8(t.k[j][i >> 1][2 * (i & 1)], t.k[j][i >> 1][2 * (i & 1) + 1],
                           __builtin_bit_cast(_Float16, t.ks[j][i >> 1]));
              else
                k = __builtin_bit_cast(f16x8, t.k[j][i]);
              sl[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q_lo[i], sl[j], 0, 0, 0);
              sc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q_hi[i], sc[j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int j = 0; j < kSub; ++j) sc[j] += sl[j];
        const uint32_t nb = b + kStep;
        const bool tail = kLast && b + kRows > p1;
        if constexpr (!kLast) {
          locate(nb, id);
          load_k(w, k_at, g, t);
          fetch(nb + kStep, id);
        }
        float y[4 * kSub], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4 * kSub; ++i) {
          y[i] = sc[i >> 2][i & 3] * mul;
          if (tail && b + 16 * (i >> 2) + 4 * g + (i & 3) >= p1) y[i] = -INFINITY;
          top = fmaxf(top, y[i]);
        }
        top = fmaxf(m, swap_max<32>(swap_max<16>(top)));
        if (__any(top > m)) {
          const float c = m == top ? 1.f : __builtin_amdgcn_exp2f(m - top);
          l *= c;
          m = top;
          if (!first)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float f = __shfl(c, 4 * g + r, 64);
#pragma unroll
            for (int i = 0; i < NH * VD; ++i) acc[i][r] *= f;
          }
        }
        float p[4 * kSub], lt[kSub];
#pragma unroll
        for (int i = 0; i < 4 * kSub; ++i) {
          p[i] = kF32 ? __builtin_amdgcn_exp2f(y[i] - m) * unit : __builtin_amdgcn_exp2f(y[i] - m + 15.f);
          lt[i >> 2] = i & 3 ? lt[i >> 2] + p[i] : p[i];
        }
        l += kSub == 2 ? lt[0] + lt[kSub - 1] : lt[0];
        if (tail) {  // (what lies behind the last row may be anything)
#pragma unroll
          for (int i = 0; i < 4 * kSub; ++i) {
            const bool in = b + 16 * (i >> 2) + 4 * g + (i & 3) < p1;
#pragma unroll
            for (int hh = 0; hh < NH; ++hh) {
              if constexpr (kQ8)
                t.vs[i >> 2][hh][i & 3] = in ? t.vs[i >> 2][hh][i & 3] : (_Float16)0.f;
              else
                t.v[i][hh] = keep(t.v[i][hh], in);
            }
          }
        }
        if constexpr (kF32) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int hh = 0; hh < NH; ++hh)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                acc[4 * hh + e] =
                    __builtin_amdgcn_mfma_f32_16x16x4f32(p[r], t.v[r][hh][e], acc[4 * hh + e], 0, 0, 0);
        } else {
          PReg p_hi, p_lo;
#pragma unroll
          for (int i = 0; i < 4 * kSub; ++i) {
            p_hi[i] = (_Float16)p[i];
            p_lo[i] = (_Float16)(p[i] - (float)p_hi[i]);
          }
#pragma unroll
          for (int hh = 0; hh < NH; ++hh) {
            _Float16 v[4 * kSub][VD];
#pragma unroll
            for (int i = 0; i < 4 * kSub; ++i) {
              if constexpr (kQ8) {
                const _Float16 vs = t.vs[i >> 2][hh][i & 3];
                f16x2 c[VD / 2];
                if constexpr (VD == 8) {
                  q8_widen(t.v[i][hh][0], c[0], c[1]);
                  q8_widen(t.v[i][hh][1], c[2], c[3]);
                } else {
                  q8_widen(t.v[i][hh], c[0], c[1]);
                }
#pragma unroll
                for (int e = 0; e < VD; ++e) v[i][e] = c[e >> 1][e & 1] * vs;
              } else {
#pragma unroll
                for (int e = 0; e < VD; ++e) v[i][e] = t.v[i][hh][e];
              }
            }
#pragma unroll
            for (int e = 0; e < VD; ++e) {
              PReg o;
#pragma unroll
              for (int i = 0; i < 4 * kSub; ++i) o[i] = v[i][e];
              f32x4& c = acc[VD * hh + e];
              c = weigh(p_lo, o, c);
              c = weigh(p_hi, o, c);
            }
          }
        }
        if constexpr (!kLast) load_v(w, v_hp, v_row, n, t);
      };
      const bool only = b + kStep >= p1;
      // (A loop of its own for what lies between: its sums stay in their registers.)
      while (b + kStep < p1) {
        uint32_t left = kAside;
        do {
          step(std::false_type{}, false);
          b += kStep;
        } while (--left && b + kStep < p1);
        if (left == 0) put_aside(std::false_type{});
      }
      step(std::true_type{}, only);
      if (aside) {
        put_aside(std::true_type{});
        l = l_aside;
      }
      l = swap_sum<32>(swap_sum<16>(l));
    }
    if (__any(no_page >= w.t.n_pages)) {
      l = NAN;
      if (no_page >= w.t.n_pages) paged_refuse(w, RV_PAGED_PAGE_OUT_OF_RANGE, s, no_page, w.t.n_pages);
    }
    __syncthreads();  // (the last segment's reads)
    if (lane < 16) sh.m[wv][n] = m, sh.l[wv][n] = l;
    if (!aside) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * g + r < ncols) {
#pragma unroll
          for (int i = 0; i < NH * VD; i += 4)
            *place(r, i) = f32x4{acc[i][r], acc[i + 1][r], acc[i + 2][r], acc[i + 3][r]};
        }
    }
    bool here = false;
    const uint32_t part = whole ? 0 : where(here);
    __syncthreads();
    for (int i = threadIdx.x; i < ncols * (HDP / 4); i += 256) {
      const int c = i / (HDP / 4), d = 4 * (i % (HDP / 4));
      if (!FULL && d >= w.hd) continue;
      const float top = fmaxf(fmaxf(sh.m[0][c], sh.m[1][c]), fmaxf(sh.m[2][c], sh.m[3][c]));
      f32x4 o{};
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // (A wave without rows has a sum of zero and a maximum of minus infinity.)
        const float lk = sh.l[k][c], f = lk != 0.f ? __builtin_amdgcn_exp2f(sh.m[k][c] - top) : 0.f;
        o += *reinterpret_cast<const f32x4*>(&sh.o[k][c][d]) * f;
        sum += f * lk;
      }
      if (whole) {
        const float inv = 1.f / sum;
        f32x4 y = o * inv;
        if (unit != 1.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) y[e] = finite(o[e], y[e]);
        }
        *reinterpret_cast<f32x4u*>(a.out + s * a.out_stride + (long)(qh + c) * w.hd + d) = y;
      } else {
        pt.put(part + (uint32_t)(c * w.hd + d) * 4u, o, here);
        if (d == 0) pt.put_stat(part, c, top, sum, here);
      }
    }
  }
};

template <typename Inner, int WAVES>
__global__ __launch_bounds__(256, WAVES) void paged_attn_kernel(PagedView w, AttnArgs a) {
  __shared__ typename Inner::Shared sh;
  __shared__ unsigned drawn;
  const int lane = threadIdx.x & 63;
  const uint32_t items = (uint32_t)(w.n_kv * a.blocks);
  const bool large = Inner::kF32 && w.status[kLarge] != 0;
  const Turn turn = a.turns[own_turn(blockIdx.x, gridDim.x)];
  unsigned* const tickets = a.tickets + (turn.set ? a.set_words : 0);
  // Sequence i's rows, for the 64 from s0 on a lane each.
  auto chunk = [&](uint32_t s0) {
    return s0 + lane < a.n ? rows_of_len(w, a, a.lens[s0 + lane]) : 0u;
  };
  uint32_t rows = chunk(0), sum = wave_scan(units_of_rows(rows) * items), base = 0;
  uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  if (a.n > 64) {
    uint32_t mine = 0;
#pragma unroll 8
    for (uint32_t s0 = 64; s0 < a.n; s0 += 64) mine += units_of_rows(chunk(s0));
    total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(mine * items), 63);
  }
  const auto divide = [](uint32_t x, uint32_t y) { return quotient(x, y, __builtin_amdgcn_rcpf((float)y)); };
  const Cut cut = cut_units(total, a.most, a.few, a.slots, divide);
  const uint32_t per = cut.per, in_slot = cut.in_slot, slot = slot_of(blockIdx.x, a.slots);
  const uint32_t ranges = in_slot << a.slots, r = range_of(blockIdx.x, a.slots, in_slot);
  const uint32_t start = r * per, end = blockIdx.x < ranges ? min(total, start + per) : 0;
  // By the wave that draws tickets, and here, where nothing waits for its stores: 100 rows
  // 5.7 us, 6.0 at the end.
  if (threadIdx.x < 64) {
    unsigned* const other = a.tickets + (turn.set ? 0 : a.set_words);
    end_turn(
        turn, blockIdx.x, gridDim.x, threadIdx.x, 64, a.n_tickets, [&](uint32_t c, Turn next) { a.turns[c] = next; },
        [&](size_t i) { other[i] = 0; });
  }
  if (start < end) {
    uint32_t s0 = 0;
    while (s0 < a.n) {  // the chunk that holds the range's first unit (none: the lengths have been changed)
      const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
      if (start < base + all) break;
      base += all;
      s0 += 64;
      rows = chunk(s0);
      sum = wave_scan(units_of_rows(rows) * items);
    }
    const int at0 = __builtin_ctzll(__ballot(start < base + sum) | 1ull << 63);
    const uint32_t before = base + (at0 ? (uint32_t)__builtin_amdgcn_readlane((int)sum, at0 - 1) : 0u);
    const Partials pt(a, w.hd);
    walk_units(
        s0 + at0, start - before, start, s0 < a.n ? end : start, items,
        [&](uint32_t s) -> uint32_t { return (uint32_t)__builtin_amdgcn_readlane((int)rows, (int)(s - s0)); },
        [&](uint32_t s) -> uint32_t {
          for (;;) {
            if (s >= a.n) return kNoMore;
            if (s - s0 >= 64) {
              s0 = s;
              rows = chunk(s0);
            }
            const uint64_t live = __ballot(units_of_rows(rows) != 0) >> (s - s0);
            if (live) return s + (uint32_t)__builtin_ctzll(live);
            s = s0 + 64;
          }
        },
        [&](uint32_t s, uint32_t n, uint32_t item, uint32_t u0, uint32_t u1, uint32_t at) {
          const uint32_t units = units_of(n), first = at - u0;
          const int h = a.blocks == 1 ? (int)item : (int)divide(item, (uint32_t)a.blocks);
          const int c0 = ((int)item - h * a.blocks) * a.cols;
          const int qh = h * a.group + c0, ncols = min(a.cols, a.group - c0);
          const bool whole = u0 == 0 && u1 == units;
          Pieces ps{};
          uint32_t of_group = 0;
          bool once = false;   // joined at once, at device scope
          bool alone = false;  // the group's only piece of many: its partial as it is
          Inner::segment(w, a, sh, s, h, qh, ncols, u0 * kUnitRows, min(n, u1 * kUnitRows), large ? weight_unit(n) : 1.f,
                         whole, pt, [&](bool& here) {
            const Group g = group_of(r, slot, in_slot);
            ps = pieces_of(g, divide(first, per), divide(first + units - 1, per), first, per, in_slot, divide);
            of_group = group_partial(g, first, per);
            once = a.slots == 0 || (ps.groups > 1 && ps.all <= kGroup);
            alone = !once && ps.groups > 1 && ps.count == 1;
            here = !once && !alone;
            return pt.at(alone ? 2 * ranges + of_group : 2 * r + partial_of(r, per, at));
          });
          if (whole) return;
          unsigned* const ticket = tickets + 2 * kGroups + s * items + item;
          float* const out = a.out + s * a.out_stride + (long)qh * w.hd;
          uint32_t piece0 = 2 * ps.first + partial_of(ps.first, per, first), rest = 2 * (ps.first + 1), count = ps.groups;
          if (once) {
            piece0 = 2 * ps.w0 + partial_of(ps.w0, per, first);
            rest = 2 * (ps.w0 + 1);
            count = ps.all;
          } else {
            const bool only = ps.groups == 1;
            if (!alone) {
              if (!last_of(only ? ticket : tickets + of_group, ps.count, drawn)) return;
              join<Inner::kVec, Inner::kLanes, kXcdScope>(pt, piece0, rest, ps.count, ncols, only ? out : nullptr,
                                                          2 * ranges + of_group, large);
            }
            if (only) return;
            piece0 = 2 * ranges + ps.group0;
            rest = (piece0 & ~1u) + 2;
          }
          if (last_of(ticket, count, drawn))
            join<Inner::kVec, Inner::kLanes, kDeviceScope>(pt, piece0, rest, count, ncols, out, 0, large);
        },
        divide);
  }
  // Sequences without rows: zeros; refused ones: NaN.
  for (uint32_t s = blockIdx.x; s < a.n; s += gridDim.x) {
    const int len = a.lens[s];
    const uint32_t n = rows_of_len(w, a, len);
    if (n != 0 && n != kRefused) continue;
    if (n == kRefused && threadIdx.x == 0)
      paged_refuse(w, RV_PAGED_POSITION_OUT_OF_RANGE, s, (uint32_t)len, (uint32_t)min(table_rows(w.t), 0xFFFFFFFFl));
    for (int d = threadIdx.x; d < w.n_kv * a.group * w.hd; d += 256) a.out[s * a.out_stride + d] = n ? NAN : 0.f;
  }
}

// The matrix-instruction kernel takes heads of whole 16-byte pieces (in any type)
// up to 256 wide; the others one position at a time.
bool tiled(int hd) { return hd % 8 == 0 && hd <= 256; }

int cols_of(int hd, int group) { return tiled(hd) ? std::min(group, 16) : 1; }

// log2 of the ranges the work is cut into: two a CU (what is resident), or one where
// the registers hold one (f32 256 wide, and widths between 128 and 256). f16 and f32
// above 64 wide take one a CU from two units a range on, where the items are no more
// than the CUs (f32: half the CUs): with more, some wait for others to end. us at 256 |
// 512 ranges: f16, 128 wide, 64 sequences of up to 16000 rows 191 | 198, 8 of 4000 17.8 |
// 18.4, but 128 of 300 22.7 | 20.1; f16, 256 wide, 32 of up to 4000 81.6 | 87.4; not of
// f16 64 wide, 64 of up to 8000 127 | 124; f32, 128 wide, 8 of 7000 44.7 | 47.4, but 64 of
// up to 4000 112 | 105; Q8_0, 128 wide, 32 of up to 8192 51 | 39. Where the XCDs are not
// known apart, an item has at most kMostPieces.
void set_ranges(const rv_paged* pg, size_t items, size_t units, AttnArgs& a) {
  const bool wide = pg->head_dim > 128 && (pg->head_dim != 256 || pg->elem == RV_ELEM_F32);
  a.slots = pg->xcd_ok && pg->tune_join != 2 ? 3 : 0;
  a.most = a.slots == 0 ? 5 : wide ? 8 : 9;
  while (a.most > 3 && units <= ((size_t)1 << a.most) / 2) --a.most;  // (never so many units)
  const size_t even = pg->elem == RV_ELEM_F16 ? kCUs : pg->elem == RV_ELEM_F32 ? kCUs / 2 : 0;
  a.few = a.most == 9 && pg->head_dim > 64 && items <= even ? 8 : a.most;
}

size_t items_per_seq(const rv_paged* pg, size_t n_q) {
  const size_t group = n_q / pg->n_kv_heads, cols = cols_of((int)pg->head_dim, (int)group);
  return pg->n_kv_heads * ((group + cols - 1) / cols);
}

template <typename T>
void launch_attn(const PagedView& w, const AttnArgs& a, dim3 grid, hipStream_t s) {
#define RV_TILED(HDP, FULL, WAVES) \
  hipLaunchKernelGGL((paged_attn_kernel<Tiled<T, HDP, FULL>, WAVES>), grid, dim3(256), 0, s, w, a)
  if (!tiled(w.hd))
    hipLaunchKernelGGL((paged_attn_kernel<Plain<T>, 1>), grid, dim3(256), 0, s, w, a);
  else if (w.hd == 64)
    RV_TILED(64, true, 2);
  else if (w.hd < 64)
    RV_TILED(64, false, 2);
  else if (w.hd == 128)
    RV_TILED(128, true, 2);
  else if (w.hd < 128)
    RV_TILED(128, false, 2);
  else if (w.hd == 256)
    RV_TILED(256, true, (std::is_same<T, float>::value ? 1 : 2));
  else
    RV_TILED(256, false, 1);
#undef RV_TILED
}

}  // namespace

PagedAttnPlan paged_attn_plan(const rv_paged* pg, const rv_page_table& t, size_t n, size_t n_q) {
  PagedAttnPlan p;
  const size_t items = n * items_per_seq(pg, n_q), rows = t.pages * pg->page_rows;
  const size_t cols = cols_of((int)pg->head_dim, (int)(n_q / pg->n_kv_heads));
  if (__builtin_mul_overflow(items, (rows + kUnitRows - 1) / kUnitRows, &p.units)) p.units = SIZE_MAX;
  p.ws_bytes = (size_t)2 * (kMaxRanges + kGroups) * partial_floats((uint32_t)cols, (uint32_t)pg->head_dim) * sizeof(float);
  p.tickets = 2 * kGroups + items;
  if (p.tickets > 0x7FFFFFFFu) p.units = SIZE_MAX;  // (tables without pages)
  p.ticket_bytes = kTurns * sizeof(Turn) + 2 * set_words(p.tickets) * sizeof(unsigned);
  return p;
}

HipStatus launch_paged_attn(const rv_paged* pg, const PagedView& w, const PagedAttn& p, const PagedAttnPlan& plan,
                            hipStream_t s) {
  AttnArgs a{};
  a.q = p.q;
  a.q_stride = (long)p.q_stride;
  a.lens = p.lens;
  a.n = (uint32_t)p.n;
  a.step = p.step;
  a.group = p.n_q / w.n_kv;
  a.cols = cols_of(w.hd, a.group);
  a.blocks = (a.group + a.cols - 1) / a.cols;
  a.scale = p.scale;
  a.out = p.out;
  a.out_stride = (long)p.out_stride;
  a.turns = (Turn*)pg->tickets;
  a.tickets = (unsigned*)(a.turns + kTurns);
  a.set_words = (pg->ticket_bytes - kTurns * sizeof(Turn)) / sizeof(unsigned) / 2 / kLineFloats * kLineFloats;
  a.n_tickets = (uint32_t)plan.tickets;
  a.part = (float*)pg->ws;
  a.part_bytes = (uint32_t)plan.ws_bytes;
  set_ranges(pg, p.n * w.n_kv * a.blocks, plan.units, a);
  const dim3 grid(1u << a.most);
  HipStatus st;
  if (pg->elem == RV_ELEM_F32)
    launch_attn<float>(w, a, grid, s);
  else if (pg->elem == RV_ELEM_F16)
    launch_attn<_Float16>(w, a, grid, s);
  else
    launch_attn<Q8>(w, a, grid, s);
  st.e = hipGetLastError();
  if (st.e != hipSuccess) st.what = "paged attention launch";
  return st;
}

}  // namespace rv
