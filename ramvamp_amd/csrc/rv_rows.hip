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
// with q' = q * scale * log2(e) and m the running maximum. K and V are f16
// matrix operands as stored (Q8_0: f16(scale * code); f32 planes: hi + lo
// halves); q' and p are split into f16 hi + lo halves whose products are
// summed in f32, which keeps fp32-equivalent products.
#include "rv_rows.hpp"

#include <algorithm>

namespace rv {
namespace {

constexpr int kD = 128;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;    // p may reach 2^kSlack before the maximum moves
constexpr float kPScale = 64.f;  // p * kPScale <= 2^14, inside f16

struct NoLens {};
struct TailLens {
  uint32_t len[kMaxEach];
};

struct RowsArgs {
  KvView main, tail;      // at the call's layers
  const float* q;
  float* out;             // written when there is one slot in all
  float* part;            // [slot][column][kD]
  float* ml;              // [slot][column][2]: maximum, sum
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

// Eight f32 values as f16 hi and lo halves.
__device__ __forceinline__ void split8(const float (&x)[8], f16x8& hi, f16x8& lo) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const _Float16 h = (_Float16)x[e];
    hi[e] = h;
    lo[e] = (_Float16)(x[e] - (float)h);
  }
}

// Dims 8 j .. + 7 of kv head h's K row t as f16 (f32: hi and lo).
template <typename T>
__device__ __forceinline__ void load_k8(const KvView& w, int h, long t, int j, f16x8& hi, f16x8& lo) {
  if constexpr (std::is_same<T, Q8>::value) {
    const size_t row = (size_t)h * w.rows + t;
    const u32x2 c = *reinterpret_cast<const u32x2*>(w.k + row * kD + 8 * j);
    const _Float16 s = __builtin_bit_cast(_Float16, w.ks[row * 4 + (j >> 2)]);
    f16x2 p[4];
    q8_widen(c[0], p[0], p[1]);
    q8_widen(c[1], p[2], p[3]);
    const f16x2 ss = {s, s};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f16x2 v = p[i] * ss;
      hi[2 * i] = v[0];
      hi[2 * i + 1] = v[1];
    }
  } else {
    const T* p = reinterpret_cast<const T*>(w.k) + (size_t)t * w.kv_dim + (size_t)h * kD + 8 * j;
    if constexpr (std::is_same<T, float>::value) {
      float x[8];
      load8(p, x);
      split8(x, hi, lo);
    } else {
      hi = *reinterpret_cast<const f16x8*>(p);
    }
  }
}

// Dims 8 j .. + 7 of eight V rows t0 + {0..3}, t0 + 8 + {0..3}, one f16x8 of
// the rows per dim; rows past `last` are zeros (their probabilities are zero,
// and what the plane holds there may not be finite).
template <typename T>
__device__ __forceinline__ void load_v8x8(const KvView& w, int h, long t0, long last, int j, f16x8 (&hi)[8],
                                          f16x8 (&lo)[8]) {
  if constexpr (std::is_same<T, Q8>::value) {
    const uint16_t* sp = w.vs + ((size_t)h * 4 + (j >> 2)) * w.rows + t0;
    const u32x2 sa = *reinterpret_cast<const u32x2*>(sp), sb = *reinterpret_cast<const u32x2*>(sp + 8);
    const char* base = w.v + ((size_t)h * w.rows + t0) * kD + 8 * j;
    u32x2 c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = *reinterpret_cast<const u32x2*>(base + (size_t)((i & 3) + 8 * (i >> 2)) * kD);
    // (Through scalars: a bit cast of a vector's element reads its element 0.)
    const uint32_t sw[4] = {sa[0], sa[1], sb[0], sb[1]};
    f16x2 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = __builtin_bit_cast(f16x2, sw[i]);
    if (t0 + 11 > last) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t0 + (i & 3) + 8 * (i >> 2) > last) s[i >> 1][i & 1] = (_Float16)0.f;
    }
#define RV_DIM(W, D)                                                            \
  {                                                                             \
    _Pragma("unroll") for (int i = 0; i < 4; ++i) {                             \
      const f16x2 v = q8_widen_pair<D>(c[2 * i][W], c[2 * i + 1][W]) * s[i];    \
      hi[4 * W + D][2 * i] = v[0];                                              \
      hi[4 * W + D][2 * i + 1] = v[1];                                          \
    }                                                                           \
  }
    RV_DIM(0, 0) RV_DIM(0, 1) RV_DIM(0, 2) RV_DIM(0, 3) RV_DIM(1, 0) RV_DIM(1, 1) RV_DIM(1, 2) RV_DIM(1, 3)
#undef RV_DIM
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long t = t0 + (i & 3) + 8 * (i >> 2);
      const T* p = reinterpret_cast<const T*>(w.v) + (size_t)min(t, last) * w.kv_dim + (size_t)h * kD + 8 * j;
      if constexpr (std::is_same<T, float>::value) {
        float x[8];
        load8(p, x);
        if (t > last) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.f;
        }
        f16x8 a, b;
        split8(x, a, b);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          hi[d][i] = a[d];
          lo[d][i] = b[d];
        }
      } else {
        f16x8 x = *reinterpret_cast<const f16x8*>(p);
        if (t > last) x = f16x8{};
#pragma unroll
        for (int d = 0; d < 8; ++d) hi[d][i] = x[d];
      }
    }
  }
}

// ---- one work item ----------------------------------------------------------------
// The columns [col0, col0 + 32 WC) of kv head h (column c: row c / group, head
// c % group) over rows [t_begin, t_end) of `w`; wave (wc, wp) takes columns
// 32 wc .. and the 32-position subtiles wp, wp + WP, ... of each step of the
// workgroup. Every wave runs the same number of steps.
template <typename T, int WC, bool HL>
__device__ void run_item(const RowsArgs& a, const KvView& w, int h, int col0, int n_cols, int row0, long t_begin,
                         long t_end, bool causal, int slot, char* lds) {
  constexpr int WP = 4 / WC;
  constexpr int S = WC == 1 ? 128 : 64;     // positions per step
  constexpr int SUB = S / 32 / WP;          // subtiles of a wave per step
  constexpr bool LO = Lo<T>::value;
  constexpr int kPlane = S / 32 * kTileB;   // K hi, V hi, then K lo, V lo
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wc = wave % WC, wp = wave / WC;
  const int lc = lane & 31, lh = lane >> 5;
  const int col = col0 + 32 * wc + lc;
  const bool live = col < n_cols;
  const int crow = (live ? col : n_cols - 1) / a.group, chead = (live ? col : n_cols - 1) % a.group;
  const int q_row = row0 + crow;
  const long limit = causal ? min((long)a.start + q_row + 1, t_end) : t_end;
  // What the wave's first column sees, and its last.
  const int wcol0 = min(col0 + 32 * wc, n_cols - 1), wcol1 = min(col0 + 32 * wc + 31, n_cols - 1);
  const long w_first = causal ? min((long)a.start + row0 + wcol0 / a.group + 1, t_end) : t_end;
  const long w_last = causal ? min((long)a.start + row0 + wcol1 / a.group + 1, t_end) : t_end;

  // q' of the column, dims 16 c + 8 lh .. + 7 of each chunk c, scaled by a
  // power of two that brings its largest value to [2^13, 2^14).
  f16x8 qh[8], ql[HL ? 8 : 1];
  float q_up;
  {
    const float* qp = a.q + ((size_t)q_row * a.n_q_heads + (size_t)(a.kv_lo + h) * a.group + chead) * kD;
    float x[8][8];
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[c][e] = live ? qp[16 * c + 8 * lh + e] * a.qscale : 0.f;
        amax = fmaxf(amax, fabsf(x[c][e]));
      }
    amax = swap_max<32>(amax);
    int ex = 14;
    if (amax > 0.f && amax < INFINITY) (void)frexpf(amax, &ex);
    const int k = max(ex - 14, -100);
    const float down = ldexpf(1.f, -k);
    q_up = ldexpf(1.f, k);
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = x[c][e] * down;
        const _Float16 hi = (_Float16)v;
        qh[c][e] = hi;
        if constexpr (HL) ql[c][e] = (_Float16)(v - (float)hi);
      }
  }
  f32x16 o[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) o[d] = f32x16{};
  float m_run = -INFINITY, m_sub = 0.f, l_run = 0.f;
  uint32_t taint = 0;  // Q8_0: this lane's dims met a NaN block in a row its column sees

  __shared__ uint32_t nan_rows[4][4];  // [subtile of 32][block of 32 dims]: rows whose V scale is NaN

  const int hk = a.kv_lo + h;
  const long last = t_end - 1;
  for (long t0 = t_begin; t0 < t_end; t0 += S) {
    __syncthreads();  // the previous step's reads are done
    if constexpr (std::is_same<T, Q8>::value) {
      if (tid < 4 * (S / 32)) nan_rows[tid >> 2][tid & 3] = 0;
      __syncthreads();
    }
    // K: thread -> (16-byte chunk j of a row, row); V: thread -> (8 dims, 8 rows).
    for (int u = tid; u < S * 16; u += 256) {
      const int j = u & 15, p = u >> 4;
      f16x8 hi, lo;
      load_k8<T>(w, hk, std::is_same<T, Q8>::value ? t0 + p : min(t0 + p, last), j, hi, lo);
      char* dst = lds + ((p >> 5) * 8 + (j >> 1)) * kFragB + k_slot(p & 31, j & 1) * 16;
      *reinterpret_cast<f16x8*>(dst) = hi;
      if constexpr (LO) *reinterpret_cast<f16x8*>(dst + 2 * kPlane) = lo;
    }
    for (int u = tid; u < S * 2; u += 256) {
      const int j = u & 15, pg = u >> 4, st = pg >> 2, s = (pg >> 1) & 1, hh = pg & 1;
      f16x8 hi[8], lo[8];
      load_v8x8<T>(w, hk, t0 + 32 * st + 16 * s + 4 * hh, last, j, hi, lo);
      if constexpr (std::is_same<T, Q8>::value) {
        // A NaN scale makes a row's whole block NaN; it must not reach columns
        // that do not see the row (0 * NaN), so the block goes in as zeros and
        // the columns that see it are marked.
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (hi[0][i] != hi[0][i]) bad |= 1u << (16 * s + 4 * hh + (i & 3) + 8 * (i >> 2));
        if (bad) {
          atomicOr(&nan_rows[st][j >> 2], bad);
#pragma unroll
          for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (hi[d][i] != hi[d][i]) hi[d][i] = (_Float16)0.f;
        }
      }
      const int dt = j >> 2;
      char* base = lds + kPlane + (st * 8 + dt * 2 + s) * kFragB;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const int at = v_slot(dt, (j & 3) * 8 + d, hh) * 16;
        *reinterpret_cast<f16x8*>(base + at) = hi[d];
        if constexpr (LO) *reinterpret_cast<f16x8*>(base + at + 2 * kPlane) = lo[d];
      }
    }
    __syncthreads();
#pragma unroll
    for (int sub = 0; sub < SUB; ++sub) {
      const int st = wp + WP * sub;
      const long p0 = t0 + 32 * st;
      if (p0 >= w_last) continue;  // wave-uniform; barriers are outside
      const char* kt = lds + st * kTileB;
      const char* vt = lds + kPlane + st * kTileB;
      f32x16 s0 = {}, s1 = {};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const f16x8 kf = *reinterpret_cast<const f16x8*>(kt + c * kFragB + k_slot(lc, lh) * 16);
        s0 = mfma(kf, qh[c], s0);
        if constexpr (HL) s1 = mfma(kf, ql[c], s1);
        if constexpr (LO) {
          const f16x8 kl = *reinterpret_cast<const f16x8*>(kt + 2 * kPlane + c * kFragB + k_slot(lc, lh) * 16);
          s1 = mfma(kl, qh[c], s1);
        }
      }
      float x[16], mx = -INFINITY;
      const bool edge = p0 + 32 > w_first;  // some column does not see all of it
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = (HL || LO ? s0[i] + s1[i] : s0[i]) * q_up;
        if (edge && p0 + 8 * (i >> 2) + (i & 3) + 4 * lh >= limit) x[i] = -INFINITY;
        mx = fmaxf(mx, x[i]);
      }
      mx = swap_max<32>(mx);
      if (__builtin_amdgcn_ballot_w64(mx > m_run + kSlack) != 0) {
        const float mn = fmaxf(m_run, mx);
        const float ms = mn == -INFINITY ? 0.f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m_run - ms);
        m_run = mn;
        m_sub = ms;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] *= alpha;
      }
      f16x8 ph[2], pl[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float p = __builtin_amdgcn_exp2f(x[i] - m_sub);
        l_run += p;
        const float pp = p * kPScale;
        const _Float16 hi = (_Float16)pp;
        ph[i >> 3][i & 7] = hi;
        if constexpr (HL) pl[i >> 3][i & 7] = (_Float16)(pp - (float)hi);
      }
      if constexpr (std::is_same<T, Q8>::value) {
        const long seen = limit - p0;  // rows of this subtile the column sees
        const uint32_t mask = seen >= 32 ? 0xFFFFFFFFu : seen <= 0 ? 0u : (1u << seen) - 1;
        // Lane (column, lh) holds dims 32 dt + 8 a + 4 lh + r of every dt.
#pragma unroll
        for (int d = 0; d < 4; ++d)
          if (nan_rows[st][d] & mask) taint |= 1u << d;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const f16x8 vf = *reinterpret_cast<const f16x8*>(vt + (d * 2 + s) * kFragB + v_slot(d, lc, lh) * 16);
          o[d] = mfma(vf, ph[s], o[d]);
          if constexpr (HL) o[d] = mfma(vf, pl[s], o[d]);
          if constexpr (LO) {
            const f16x8 vl =
                *reinterpret_cast<const f16x8*>(vt + 2 * kPlane + (d * 2 + s) * kFragB + v_slot(d, lc, lh) * 16);
            o[d] = mfma(vl, ph[s], o[d]);
          }
        }
    }
  }
  // Each lane summed its own rows: the other half of the column's.
  l_run = swap_sum<32>(l_run);
  if constexpr (std::is_same<T, Q8>::value) {
    if (taint) {
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (taint & (1u << d)) o[d] = o[d] * __builtin_nanf("");
    }
  }
  // The position groups' partials meet in LDS, in wave order.
  if constexpr (WP > 1) {
    float* om = reinterpret_cast<float*>(lds);  // [wp - 1][wc][64 registers][64 lanes], then (m, l)
    constexpr int kWave = 66 * 64;
    __syncthreads();
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
  constexpr float kDown = 1.f / kPScale;
  if (a.single) {
    const float inv = kDown / l_run;
    float* dst = a.out + ((size_t)q_row * a.n_heads * a.group + (size_t)h * a.group + chead) * kD;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dst[32 * d + 8 * (i >> 2) + 4 * lh + (i & 3)] = o[d][i] * inv;
    return;
  }
  const size_t column = (size_t)h * a.rows * a.group + (size_t)row0 * a.group + col;
  const size_t at = (size_t)slot * a.n_heads * a.rows * a.group + column;
  float* dst = a.part + at * kD;
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const f32x4 v = {o[d][4 * g] * kDown, o[d][4 * g + 1] * kDown, o[d][4 * g + 2] * kDown, o[d][4 * g + 3] * kDown};
      *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * g + 4 * lh) = v;
    }
  if (lh == 0) {
    a.ml[2 * at] = m_run;
    a.ml[2 * at + 1] = l_run;
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

template <typename T, int WC, bool HL, bool TAILS>
__global__ __launch_bounds__(256) void rows_kernel(RowsArgs a, std::conditional_t<TAILS, TailLens, NoLens> lens) {
  constexpr int kMain = stage_bytes<T>(WC == 1 ? 128 : 64), kTail = TAILS ? stage_bytes<T>(128) : 0;
  constexpr int kMerge = (TAILS || WC == 1 ? 3 : WC == 2 ? 2 : 0) * 66 * 64 * 4;
  constexpr int kBytes = kMain > kTail ? (kMain > kMerge ? kMain : kMerge) : (kTail > kMerge ? kTail : kMerge);
  __shared__ __attribute__((aligned(1024))) char lds[kBytes];
  int b = blockIdx.x;
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  if (!TAILS || b < a.main_items) {
    const int split = b % a.n_splits;
    b /= a.n_splits;
    const int cb = b % a.n_cb, h = b / a.n_cb;
    const int n_cols = a.rows * a.group, col0 = cb * 32 * WC;
    long t_end = positions;
    if (a.causal) {  // the last column's limit
      const int r = (min(col0 + 32 * WC, n_cols) - 1) / a.group;
      t_end = min(t_end, (long)a.start + r + 1);
    }
    const long t_begin = (long)split * a.split_len;
    t_end = min(t_end, t_begin + a.split_len);
    if (t_begin >= t_end) return;
    run_item<T, WC, HL>(a, a.main, h, col0, n_cols, 0, t_begin, t_end, a.causal != 0, split, lds);
  } else if constexpr (TAILS) {
    b -= a.main_items;
    const int split = b % a.t_splits;
    b /= a.t_splits;
    const int cb = b % a.t_cb;
    b /= a.t_cb;
    const int h = b % a.n_heads, seq = b / a.n_heads;
    const long len = lens.len[seq], t_begin = (long)split * a.t_split_len;
    if (t_begin >= len) return;
    KvView w = a.tail;
    w.k += (size_t)seq * w.layer_bytes;
    w.v += (size_t)seq * w.layer_bytes;
    w.ks += (size_t)seq * w.layer_scales;
    w.vs += (size_t)seq * w.layer_scales;
    run_item<T, 1, HL>(a, w, h, cb * 32, a.group, seq, t_begin, min(len, t_begin + a.t_split_len), false,
                       a.n_splits + split, lds);
  }
}

// Folds a column's partials: 32 lanes a column, 4 dims each, slots in order.
template <bool TAILS>
__global__ __launch_bounds__(256) void rows_merge_kernel(RowsArgs a, std::conditional_t<TAILS, TailLens, NoLens> lens) {
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  const int n = a.n_heads * a.rows * a.group;
  const int column = blockIdx.x * 8 + (threadIdx.x >> 5), l = threadIdx.x & 31;
  if (column >= n) return;
  const int h = column / (a.rows * a.group), c = column % (a.rows * a.group), row = c / a.group;
  long limit = positions;
  if (a.causal) limit = min(limit, (long)a.start + row + 1);
  const int n_main = (int)((limit + a.split_len - 1) / a.split_len);
  int n_all = n_main;
  if constexpr (TAILS) n_all += (int)((lens.len[row] + a.t_split_len - 1) / a.t_split_len);
  float M = -INFINITY, L = 0.f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  for (int i = 0; i < n_all; ++i) {
    const int slot = i < n_main ? i : a.n_splits + i - n_main;
    const size_t at = (size_t)slot * n + column;
    const float m = a.ml[2 * at], s = a.ml[2 * at + 1];
    const f32x4 v = *reinterpret_cast<const f32x4*>(a.part + at * kD + 4 * l);
    const float mn = fmaxf(M, m), ms = mn == -INFINITY ? 0.f : mn;
    const float f1 = __builtin_amdgcn_exp2f(M - ms), f2 = __builtin_amdgcn_exp2f(m - ms);
    M = mn;
    L = L * f1 + s * f2;
    O = O * f1 + v * f2;
  }
  const f32x4 r = O / L;
  float* dst = a.out + ((size_t)row * a.n_heads * a.group + (size_t)h * a.group + c % a.group) * kD + 4 * l;
#pragma unroll
  for (int e = 0; e < 4; ++e) dst[e] = r[e];  // out may be only 4-byte aligned
}

// ---- any head size up to 512 --------------------------------------------------------
// One workgroup a column; each wave walks every fourth row (one row at a time,
// the head's values over the lanes), f32 arithmetic, the waves' sums joined in
// LDS. For geometries no model of this library's path has; it is right, not fast.
template <typename T, bool TAILS>
__global__ __launch_bounds__(256) void rows_generic_kernel(RowsArgs a, int hd,
                                                           std::conditional_t<TAILS, TailLens, NoLens> lens) {
  constexpr int kPer = 8;
  __shared__ float sm_o[3][64 * kPer], sm_m[3], sm_l[3];
  int positions = a.positions;
  if (!device_positions(a.d_pos, a.positions, positions)) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int n_q = a.n_heads * a.group;
  const int row = blockIdx.x / n_q, hq = blockIdx.x % n_q, h = a.kv_lo + hq / a.group;
  const float* qp = a.q + ((size_t)row * a.n_q_heads + (size_t)a.kv_lo * a.group + hq) * hd;
  float q[kPer], o[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    q[i] = lane + 64 * i < hd ? qp[lane + 64 * i] * a.qscale : 0.f;
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  auto walk = [&](const KvView& w, long len) {
    for (long t = wave; t < len; t += 4) {
      float x = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 64 * i < hd) x += q[i] * kv_value<T, false>(w, hd, h, t, lane + 64 * i);
      x = group_sum<32>(x);
      x = swap_sum<32>(x);
      const float mn = fmaxf(m, x), ms = mn == -INFINITY ? 0.f : mn;
      const float f = __builtin_amdgcn_exp2f(m - ms), p = __builtin_amdgcn_exp2f(x - ms);
      m = mn;
      l = l * f + p;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + 64 * i < hd) o[i] = o[i] * f + p * kv_value<T, true>(w, hd, h, t, lane + 64 * i);
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
    const float f1 = __builtin_amdgcn_exp2f(m - ms), f2 = __builtin_amdgcn_exp2f(sm_m[p] - ms);
    m = mn;
    l = l * f1 + sm_l[p] * f2;
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = o[i] * f1 + sm_o[p][lane + 64 * i] * f2;
  }
  float* dst = a.out + ((size_t)row * n_q + hq) * hd;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 64 * i < hd) dst[lane + 64 * i] = o[i] / l;
}

// ---- plans ------------------------------------------------------------------------
struct RowsPlan {
  bool generic = false;
  int wc = 1, n_cb = 0, n_splits = 0, split_len = 128;
  int t_cb = 0, t_splits = 0, t_split_len = 128;
  size_t rows = 0;  // of one launch (sequences go in batches of kMaxEach)
  size_t slots() const { return (size_t)n_splits + t_splits; }
};

constexpr long kWantItems = 2 * kCUs;
constexpr int kPosStep = 128;

// Splits of `positions` for `units` independent items so that the launch has
// about kWantItems of them: lengths in whole steps.
void split_positions(long positions, long units, int* n_splits, int* split_len) {
  const long steps = (positions + kPosStep - 1) / kPosStep;
  const long want = std::max<long>(1, std::min<long>(steps, kWantItems / std::max<long>(units, 1)));
  const long per = (steps + want - 1) / want;
  *split_len = (int)(per * kPosStep);
  *n_splits = (int)((steps + per - 1) / per);
}

RowsPlan plan_rows(const RowsCall& c, const rv_kv* owner) {
  RowsPlan p;
  const rv_kv* g = c.main ? c.main : c.tails;
  p.generic = g->head_dim != (size_t)kD;
  p.rows = c.tails ? std::min<size_t>(c.rows, kMaxEach) : c.rows;
  if (p.generic) return p;
  const long group = (long)(c.n_q_heads / g->n_kv_heads), heads = (long)(c.kv_hi - c.kv_lo);
  if (c.main && c.positions) {
    const long cols = (long)p.rows * group;
    p.wc = cols <= 32 ? 1 : cols <= 64 ? 2 : 4;
    p.n_cb = (int)((cols + 32 * p.wc - 1) / (32 * p.wc));
    split_positions((long)c.positions, heads * p.n_cb, &p.n_splits, &p.split_len);
    if (owner->tune_decode_split_len > 0) {
      p.split_len = (int)((std::min<int64_t>(owner->tune_decode_split_len, 1 << 30) + kPosStep - 1) / kPosStep * kPosStep);
      p.n_splits = (int)((c.positions + p.split_len - 1) / p.split_len);
    }
  }
  if (c.tails) {
    size_t longest = 0;
    for (size_t i = 0; i < c.rows; ++i) longest = std::max(longest, c.tails->lens[c.tail_layer + i]);
    p.t_cb = (int)((group + 31) / 32);
    if (longest) split_positions((long)longest, heads * p.t_cb * (long)p.rows, &p.t_splits, &p.t_split_len);
  }
  return p;
}

size_t plan_floats(const RowsPlan& p, const RowsCall& c) {
  const rv_kv* g = c.main ? c.main : c.tails;
  const size_t cols = p.rows * (c.n_q_heads / g->n_kv_heads) * (c.kv_hi - c.kv_lo);
  return p.generic || p.slots() <= 1 ? 0 : p.slots() * cols * (kD + 2);
}

template <typename T, int WC, bool HL, bool TAILS, typename L>
void launch_rows_kernel(const TimedPair& tp, const RowsArgs& a, unsigned items, hipStream_t s, const L& lens) {
  launch_timed(tp, rows_kernel<T, WC, HL, TAILS>, dim3(items), dim3(256), s, a, lens);
}

template <typename T, bool HL, bool TAILS, typename L>
void launch_wc(int wc, const TimedPair& tp, const RowsArgs& a, unsigned items, hipStream_t s, const L& lens) {
  if (wc == 1)
    launch_rows_kernel<T, 1, HL, TAILS>(tp, a, items, s, lens);
  else if (wc == 2)
    launch_rows_kernel<T, 2, HL, TAILS>(tp, a, items, s, lens);
  else
    launch_rows_kernel<T, 4, HL, TAILS>(tp, a, items, s, lens);
}

}  // namespace

size_t rows_ws_need(const rv_kv* owner, const RowsCall& c) { return plan_floats(plan_rows(c, owner), c) * sizeof(float); }

size_t rows_ws_bound(const rv_kv* kv) {
  if (kv->head_dim != (size_t)kD) return 0;
  // At most kWantItems items of 32 columns (one wave's), and one per kv head.
  return (size_t)std::max<long>(kWantItems, (long)kv->n_kv_heads) * 32 * (kD + 2) * sizeof(float);
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
    st = ensure_workspace(owner, need);
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
    a.causal = c.causal;
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
      const size_t cols = n * group * a.n_heads;
      a.part = base;
      a.ml = base ? base + p.slots() * cols * kD : nullptr;
      a.n_cb = (int)((n * group + 32 * p.wc - 1) / (32 * p.wc));
      a.n_splits = p.n_splits;
      a.split_len = p.split_len;
      a.t_cb = p.t_cb;
      a.t_splits = p.t_splits;
      a.t_split_len = p.t_split_len;
      a.main_items = a.n_heads * a.n_cb * a.n_splits;
      a.single = p.slots() == 1;
      const unsigned items = (unsigned)(a.main_items + n * a.n_heads * a.t_cb * a.t_splits);
      const TimedPair tp = ws ? TimedPair{} : timing_pair(owner, s);
      if (c.tails) {
        if (g->elem == RV_ELEM_Q8_0)
          launch_wc<Q8, true, true>(p.wc, tp, a, items, s, lens);
        else if (g->elem == RV_ELEM_F32)
          launch_wc<float, true, true>(p.wc, tp, a, items, s, lens);
        else
          launch_wc<_Float16, true, true>(p.wc, tp, a, items, s, lens);
      } else if (c.split) {
        launch_wc<Q8, true, false>(p.wc, tp, a, items, s, NoLens{});
      } else {
        launch_wc<Q8, false, false>(p.wc, tp, a, items, s, NoLens{});
      }
      if (!a.single) {
        const dim3 grid((unsigned)((cols + 7) / 8)), block(256);
        if (c.tails)
          hipLaunchKernelGGL(rows_merge_kernel<true>, grid, block, 0, s, a, lens);
        else
          hipLaunchKernelGGL(rows_merge_kernel<false>, grid, block, 0, s, a, NoLens{});
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
