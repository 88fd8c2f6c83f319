// Log-probabilities of given labels with the entropy and the most probable classes of every row.
//
//   m = max x,  s = Σ e^(x−m),  t = Σ (x−m) e^(x−m)
//   log p_j = x_j − m − log s        H = log s − t / s
//   ∂/∂x_j (g·log p_y + h·H + Σ_i g_i·log p_{k_i}) =
//       g·[j=y] + Σ_i g_i·[j=k_i] − p_j (g + Σ_i g_i + h (log p_j + H))
//
// One read of the logits forward: maximum, sum and entropy term are carried together (a running
// maximum rescales the two sums), the k best classes come from the same pass.  The backward pass
// reads the logits once more and recomputes the probabilities from (m, log s, H).
//
// Rows of at most 2048 classes belong to a group of 1..64 lanes (one 8-element vector per lane and
// step), so a wave works on 64 / LPR rows and nothing leaves its registers.  Longer rows belong to
// a workgroup, or to several where there are too few rows to fill the chip: the parts' sums and
// candidates meet in a second small launch.
//
// Special rows: a label equal to ignore_index gives log p = 0 and no gradient; a label outside
// [0, C) gives NaN (nothing is read out of range); a row of −∞ only has log p = −∞, H = 0,
// alternatives −∞ in index order and a zero gradient; a row that holds NaN or +∞ gives NaN in every
// float and the indices 0..k−1.  Sums are 32-bit floats; only the gradient is rounded to its type.
#include "common.h"
#include "kernels.h"

#include <float.h>

namespace tdl {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float FLOOR = -1e4f;  // finite stand-in for −∞ where it is multiplied by an exact 0

// 8 elements at any element alignment: rows of odd length start anywhere, and the hardware takes
// 16-byte accesses at 2-byte alignment, so there is no peeling
typedef uint32_t u4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4_a4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void ld8(const bf16_t* p, float* f) {
  const u4_a2 v = *(const u4_a2*)p;
  unpack8(make_uint4(v.x, v.y, v.z, v.w), f);
}
__device__ __forceinline__ void ld8(const float* p, float* f) {
  const f4_a4 a = ((const f4_a4*)p)[0], b = ((const f4_a4*)p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void st8(bf16_t* p, const float* f) {
  const uint4 v = pack8(f);
  *(u4_a2*)p = u4_a2{v.x, v.y, v.z, v.w};
}
__device__ __forceinline__ void st8(float* p, const float* f) {
  ((f4_a4*)p)[0] = f4_a4{f[0], f[1], f[2], f[3]};
  ((f4_a4*)p)[1] = f4_a4{f[4], f[5], f[6], f[7]};
}

// All-lanes reductions over groups of W adjacent lanes without LDS: within 16 lanes by DPP (quad
// swaps, then mirrors: after a step all lanes of a half hold the same value, so its mirror is its
// partner), across them by row and half swaps.  Both partners combine the same two values.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int STEP>
__device__ __forceinline__ void partners(uint32_t v, uint32_t* a, uint32_t* b) {
  *a = v;
  if constexpr (STEP == 1) *b = dpp<0xB1>(v);
  else if constexpr (STEP == 2) *b = dpp<0x4E>(v);
  else if constexpr (STEP == 4) *b = dpp<0x141>(v);
  else if constexpr (STEP == 8) *b = dpp<0x140>(v);
  else if constexpr (STEP == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    *a = r[0];
    *b = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    *a = r[0];
    *b = r[1];
  }
}
template <int W, int STEP = 1, typename F>
__device__ __forceinline__ uint32_t reduce_bits(uint32_t v, F op) {
  if constexpr (STEP < W) {
    uint32_t a, b;
    partners<STEP>(v, &a, &b);
    return reduce_bits<W, 2 * STEP>(op(a, b), op);
  }
  return v;
}
template <int W>
__device__ __forceinline__ float gmax(float v) {
  return __uint_as_float(reduce_bits<W>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
template <int W>
__device__ __forceinline__ float gsum(float v) {
  return __uint_as_float(reduce_bits<W>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
template <int W>
__device__ __forceinline__ uint32_t gmin(uint32_t v) {
  return reduce_bits<W>(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
// 64-bit keys: both halves move together
template <int W, int STEP = 1>
__device__ __forceinline__ unsigned long long gmax_key(unsigned long long k) {
  if constexpr (STEP < W) {
    uint32_t ah, bh, al, bl;
    partners<STEP>((uint32_t)(k >> 32), &ah, &bh);
    partners<STEP>((uint32_t)k, &al, &bl);
    return gmax_key<W, 2 * STEP>(max((unsigned long long)ah << 32 | al, (unsigned long long)bh << 32 | bl));
  }
  return k;
}

// (m, s, t) of a set of elements; t in units of log 2
struct Stat {
  float m, s, t;
};

__device__ __forceinline__ Stat stat_empty() { return Stat{-FLT_MAX, 0.f, 0.f}; }

__device__ __forceinline__ void stat_rescale(Stat& a, float m) {
  const float w = fmaxf((a.m - m) * LOG2E, FLOOR);
  const float f = __builtin_amdgcn_exp2f(w);
  a.t = f * (a.t + w * a.s);
  a.s = f * a.s;
  a.m = m;
}

__device__ __forceinline__ Stat stat_join(Stat a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  stat_rescale(a, m);
  stat_rescale(b, m);
  return Stat{m, a.s + b.s, a.t + b.t};
}

// one element: NaN and +∞ (x − m = NaN) reach the sum, −∞ adds exact zeros to both
__device__ __forceinline__ void stat_add(Stat& a, float x) {
  const float w = (x - a.m) * LOG2E;
  const float e = __builtin_amdgcn_exp2f(w);
  a.s += e;
  a.t = fmaf(fmaxf(w, FLOOR), e, a.t);
}

// over a whole wave: one common maximum, then plain sums
__device__ __forceinline__ Stat stat_wave(Stat a) {
  stat_rescale(a, gmax<64>(a.m));
  a.s = gsum<64>(a.s);
  a.t = gsum<64>(a.t);
  return a;
}

// what a row's outputs are made of
struct RowEnd {
  float m, logs, ent;
  bool empty, bad;
  __device__ __forceinline__ float lp(float x) const {
    return bad ? NAN : empty ? -INFINITY : (x - m) - logs;
  }
};

__device__ __forceinline__ RowEnd row_end(const Stat& a) {
  RowEnd r;
  r.bad = !(a.s == a.s);
  r.empty = a.s == 0.f;
  r.m = a.m;
  r.logs = r.empty ? 0.f : logf(a.s);
  r.ent = r.bad ? NAN : r.empty ? 0.f : r.logs - LN2 * (a.t / a.s);
  return r;
}

// the row's label and its logit, loaded ahead of the row (two dependent loads: behind it they would
// end every row with their latency)
struct RowLabel {
  long y = 0;
  float x = 0.f;
  template <typename T>
  __device__ __forceinline__ void load(const LogProbArgs& a, long row, const T* xr) {
    if (!a.labels) return;
    y = a.labels[row];
    const bool in = y >= 0 && y < a.C;
    x = load1(xr + (in ? y : 0));
    if (!in) x = NAN;
  }
};

__device__ __forceinline__ void write_row(const LogProbArgs& a, long row, const RowLabel& l,
                                          const RowEnd& r) {
  if (a.labels) a.logp[row] = l.y == a.ignore ? 0.f : l.x != l.x ? NAN : r.lp(l.x);
  a.ent[row] = r.ent;
  if (a.stat) {
    a.stat[3 * row] = r.m;
    // a row with nothing left: log s = +∞ makes every recomputed probability an exact 0
    a.stat[3 * row + 1] = r.bad ? NAN : r.empty ? INFINITY : r.logs;
    a.stat[3 * row + 2] = r.ent;
  }
}

// order-preserving (value, lowest index first) key; 0 = none
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t idx) {
  const uint32_t u = __float_as_uint(x + 0.f);  // −0 and +0 tie
  const uint32_t o = u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
  return (unsigned long long)o << 32 | (0xffffffffu - idx);
}
__device__ __forceinline__ float key_val(unsigned long long k) {
  const uint32_t o = (uint32_t)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint32_t key_idx(unsigned long long k) { return 0xffffffffu - (uint32_t)k; }

// ----------------------------------------------------------------------------- short rows
// Lane l of a row's LPR lanes holds vectors l, l + LPR, ….  The row's last, partial vector is read
// at C − 8 instead (inside the row); its elements that belong to the vector before are masked out.
template <typename T, int LPR, int V>
struct RowVec {
  float x[V][8];
  int base[V];   // index of x[v][0]
  int first[V];  // elements below this index are not this lane's
  __device__ __forceinline__ void load(const T* row, int C, int lane, bool live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int start = (lane + v * LPR) * 8;
      base[v] = start;
      first[v] = C;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[v][e] = -INFINITY;
      if (!live || start >= C) continue;
      first[v] = start;
      if (C < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < C) x[v][e] = load1(row + e);
      } else {
        base[v] = min(start, C - 8);
        ld8(row + base[v], x[v]);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (base[v] + e < start) x[v][e] = -INFINITY;
      }
    }
  }
  __device__ __forceinline__ bool owns(int v, int e, int C) const {
    return base[v] + e >= first[v] && base[v] + e < C;
  }
};

// alternative j of a row: kept by lane j where the group has a lane for each (written once, at the
// end), else written at once
template <int LPR>
struct TopOut {
  const LogProbArgs& a;
  const RowEnd& r;
  long row;
  bool live;
  float x = 0.f;
  uint32_t idx = 0;
  __device__ __forceinline__ void put(int j, float v, uint32_t i) const {
    a.top_lp[row * a.k + j] = r.lp(v);
    a.top_idx[row * a.k + j] = r.bad ? j : i;
  }
  __device__ __forceinline__ void take(int j, int lane, float v, uint32_t i) {
    if (LPR < LOGPROB_MAX_K) {
      if (live && lane == 0) put(j, v, i);
    } else if (lane == j) {
      x = v;
      idx = i;
    }
  }
  __device__ __forceinline__ void done(int lane) const {
    if (LPR >= LOGPROB_MAX_K && live && lane < a.k) put(lane, x, idx);
  }
};

template <typename T, int LPR, int V, bool TOPK>
__global__ void __launch_bounds__(256) logprob_rows_kernel(LogProbArgs a) {
  const int lane = threadIdx.x % LPR;
  const long rows_per_grid = (long)gridDim.x * (256 / LPR);
  // whole waves leave the loop together: a group without a row takes part in the shuffles
  for (long r0 = (long)blockIdx.x * (256 / LPR); r0 < a.N; r0 += rows_per_grid) {
    const long row = r0 + threadIdx.x / LPR;
    const bool live = row < a.N;
    const T* x = (const T*)a.x + (live ? row : 0) * a.ld;
    const int C = (int)a.C;
    RowLabel lab;
    if (live) lab.load(a, row, x);
    RowVec<T, LPR, V> d;
    d.load(x, C, lane, live);
    Stat st = stat_empty();
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) st.m = fmaxf(st.m, d.x[v][e]);
    st.m = gmax<LPR>(st.m);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) stat_add(st, d.x[v][e]);
    st.s = gsum<LPR>(st.s);
    st.t = gsum<LPR>(st.t);
    const RowEnd r = row_end(st);
    if (live && lane == 0) write_row(a, row, lab, r);
    TopOut<LPR> out{a, r, row, live};
    if constexpr (TOPK && sizeof(T) == 2) {
      // bf16: value and index of an element fit one ordered 32-bit key, different for every element,
      // so a maximum is its own place and its removal one comparison (k passes over the registers;
      // 8192 × 1000, k = 5: 12.8 us, with a search for the place as below 15.4)
      uint32_t key[V * 8];
#pragma unroll
      for (int i = 0; i < V * 8; ++i) {
        const uint32_t o = (uint32_t)(key_of(d.x[i / 8][i % 8], 0) >> 32) & 0xffff0000u;
        key[i] = d.owns(i / 8, i % 8, C) ? o | (0xffffu - (uint32_t)(d.base[i / 8] + i % 8)) : 0u;
      }
      for (int j = 0; j < a.k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < V * 8; ++i) best = max(best, key[i]);
        best = reduce_bits<LPR>(best, [](uint32_t p, uint32_t q) { return max(p, q); });
#pragma unroll
        for (int i = 0; i < V * 8; ++i) key[i] = key[i] == best ? 0u : key[i];
        const uint32_t v = (best & 0x80000000u ? best ^ 0x80000000u : ~best) & 0xffff0000u;
        out.take(j, lane, __uint_as_float(v), 0xffffu - (best & 0xffffu));
      }
    } else if constexpr (TOPK) {
      // k times the group's maximum; NaN marks what is taken or not this lane's (maxima pass over it,
      // nothing equals it)
#pragma unroll
      for (int i = 0; i < V * 8; ++i)
        if (!d.owns(i / 8, i % 8, C)) d.x[i / 8][i % 8] = NAN;
      for (int j = 0; j < a.k; ++j) {
        float best = d.x[0][0];
#pragma unroll
        for (int i = 1; i < V * 8; ++i) best = fmaxf(best, d.x[i / 8][i % 8]);
        best = gmax<LPR>(best);
        uint32_t mine = ~0u;
#pragma unroll
        for (int i = V * 8 - 1; i >= 0; --i)
          if (d.x[i / 8][i % 8] == best) mine = d.base[i / 8] + i % 8;
        const uint32_t idx = gmin<LPR>(mine);
#pragma unroll
        for (int i = 0; i < V * 8; ++i)
          if (idx == (uint32_t)(d.base[i / 8] + i % 8)) d.x[i / 8][i % 8] = NAN;
        out.take(j, lane, best, idx);
      }
    }
    if (TOPK) out.done(lane);
  }
}

// the gradient of one element from the row's recomputed probability
struct RowGrad {
  float m, logs, ent, g, gall, h;
  long y;
  __device__ __forceinline__ float of(float x) const {
    const float lp = (x - m) - logs;
    const float p = __builtin_amdgcn_exp2f(lp * LOG2E);
    return -p * fmaf(h, fmaxf(lp, FLOOR) + ent, gall);
  }
};

__device__ __forceinline__ RowGrad row_grad(const LogProbGradArgs& a, long row) {
  RowGrad r;
  r.m = a.stat[3 * row];
  r.logs = a.stat[3 * row + 1];
  r.ent = a.stat[3 * row + 2];
  const bool lab = a.labels && (a.g_logp || a.dloss);
  r.y = lab ? a.labels[row] : -1;
  const bool counts = !lab || r.y != a.ignore;
  float g;
  if (a.dloss) {  // the mean loss: every row that counts has the same factors
    g = -a.dloss[0] * a.inv_rows[0];
    r.h = counts ? a.ent_weight * g : 0.f;
  } else {
    g = a.g_logp ? a.g_logp[row] : 0.f;
    r.h = a.g_ent ? a.g_ent[row] : 0.f;
  }
  // a label out of range had log p = NaN: so is a gradient through it
  r.g = !lab || !counts ? 0.f : g != 0.f && (r.y < 0 || r.y >= a.C) ? NAN : g;
  if (!counts) r.y = -1;
  const bool empty = r.logs == INFINITY;
  if (empty) r.g = r.h = 0.f;  // nothing depends on the logits
  r.gall = r.g;
  if (a.g_top && !empty)
    for (int j = 0; j < a.k; ++j) r.gall += a.g_top[row * a.k + j];
  return r;
}

// adds of a label / alternative that lies in the 8 elements from base
__device__ __forceinline__ void add_at(float* v, int base, int idx, float g) {
  // a branch of the whole wave around selects: with 8 alternatives (4096 × 131072 bf16) the gradient
  // takes 567 us, with an indexed add 626, with a branch per element 751 (the label alone: no difference)
  const uint32_t d = (uint32_t)(idx - base);
  if (__builtin_amdgcn_ballot_w64(d < 8)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += d == e ? g : 0.f;
  }
}

__device__ __forceinline__ void grad8(const LogProbGradArgs& a, const RowGrad& r, long row,
                                      int base, float* v) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = r.of(v[e]);
  if (r.y >= 0) add_at(v, base, (int)r.y, r.g);
  if (a.g_top && r.logs != INFINITY)
    for (int j = 0; j < a.k; ++j) add_at(v, base, (int)a.top_idx[row * a.k + j], a.g_top[row * a.k + j]);
}

template <typename T>
__device__ __forceinline__ void grad_vec(const LogProbGradArgs& a, const RowGrad& r, long row,
                                         const T* x, T* dx, int start) {
  const int C = (int)a.C;
  float v[8];
  if (C < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < C ? load1(x + e) : 0.f;
    grad8(a, r, row, 0, v);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < C) store1(dx + e, v[e]);
    return;
  }
  // the last vector overlaps the one before: both write the same values to the shared elements
  const int base = min(start, C - 8);
  ld8(x + base, v);
  grad8(a, r, row, base, v);
  st8(dx + base, v);
}

template <typename T, int LPR, int V>
__global__ void __launch_bounds__(256) logprob_rows_bwd_kernel(LogProbGradArgs a) {
  const int lane = threadIdx.x % LPR;
  const long rows_per_grid = (long)gridDim.x * (256 / LPR);
  for (long row = (long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR; row < a.N;
       row += rows_per_grid) {
    const RowGrad r = row_grad(a, row);
    const T* x = (const T*)a.x + row * a.ld;
    T* dx = (T*)a.dx + row * a.C;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int start = (lane + v * LPR) * 8;
      if (start < a.C) grad_vec(a, r, row, x, dx, start);
    }
  }
}

// ----------------------------------------------------------------------------- longer rows
// Elements per workgroup: two rounds of two vectors per thread (2047 × 50021 fp32: 171 us, 8 rounds
// of one 215, one round of four 165; 4096 × 131072 bf16: 367, 390, 359; 4096 × 4096 bf16: 13.3, 13.2,
// 16.5; inputs that change from call to call)
constexpr int BWD_U = 2, BWD_CHUNK = 256 * 8 * BWD_U * 2;

template <typename T>
__global__ void __launch_bounds__(256) logprob_long_bwd_kernel(LogProbGradArgs a, uint32_t chunks) {
  const uint32_t total = (uint32_t)a.N * chunks;  // < 2^32: the card's memory holds fewer chunks
  const int C = (int)a.C;
  for (uint32_t b = blockIdx.x; b < total; b += gridDim.x) {
    const uint32_t r0 = b / chunks;
    const long row = r0;
    const int c0 = (int)(b - r0 * chunks) * BWD_CHUNK, c1 = min(C, c0 + BWD_CHUNK);
    const RowGrad r = row_grad(a, row);
    const T* x = (const T*)a.x + row * a.ld;
    T* dx = (T*)a.dx + row * a.C;
    // C > 2048: every vector lies in the row, the last one moved back as in grad_vec.  The loads
    // come before the stores (the compiler cannot know that dx is not x)
    for (int s = c0 + (int)threadIdx.x * 8; s < c1; s += 256 * 8 * BWD_U) {
      float f[BWD_U][8];
#pragma unroll
      for (int u = 0; u < BWD_U; ++u) ld8(x + min(s + u * 2048, C - 8), f[u]);
#pragma unroll
      for (int u = 0; u < BWD_U; ++u) {
        const int base = min(s + u * 2048, C - 8);
        grad8(a, r, row, base, f[u]);
        if (s + u * 2048 < c1) st8(dx + base, f[u]);
      }
    }
  }
}

constexpr int MAX_K = 32, CAND = 2048;

// the k largest of n distinct keys in LDS by counting, dst[0..k) (0 where there are fewer)
template <int NTH>
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int n, int k,
                                          unsigned long long* dst) {
  if ((int)threadIdx.x < k && (int)threadIdx.x >= n) dst[threadIdx.x] = 0;
  for (int i = threadIdx.x; i < n; i += NTH) {
    const unsigned long long me = keys[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keys[j] > me;
    if (rank < k) dst[rank] = me;
  }
}

// One workgroup: elements [c0, c1) of a row.  Thread i owns vectors i, i + NTH, … and tracks its
// maximum and the vector it is in.  Groups of GL lanes offer a lower bound of their best key; the
// k-th largest of these bounds τ is below at least k elements, so only vectors of threads whose
// maximum reaches τ can hold one of the k best.  The whole workgroup reads those again (about
// 2 k / NTH of the row; one thread alone would wait for each of its vectors: 130 us of 325 at
// 4096 × 131072, k = 8) and hands in the elements ≥ τ.  More than CAND of them (a row sorted
// against the grain) takes k passes instead.
template <typename T, int NTH, bool TOPK>
__global__ void __launch_bounds__(NTH) logprob_long_kernel(LogProbArgs a, int parts, int part_len) {
  constexpr int GL = NTH / 32, G = 32, U = 4;
  static_assert(G >= MAX_K, "");
  __shared__ Stat sh_st[NTH / 64];
  __shared__ unsigned long long gkey[TOPK ? G : 1], cand[TOPK ? CAND : 1], best[TOPK ? MAX_K : 1];
  __shared__ unsigned long long tau;
  __shared__ int count, nsel;
  __shared__ uint16_t sel[TOPK ? NTH : 1];
  const int tid = threadIdx.x;
  const long total = a.N * parts;
  for (long b = blockIdx.x; b < total; b += gridDim.x) {
    const long row = b / parts;
    const int part = (int)(b - row * parts);
    const T* x = (const T*)a.x + row * a.ld;
    const int c0 = part * part_len, c1 = (int)min((long)c0 + part_len, a.C);
    const int nvec = (c1 - c0) / 8, tail = (c1 - c0) % 8;  // the tail's elements: one per thread
    RowLabel lab;
    if (parts == 1) lab.load(a, row, x);
    Stat st = stat_empty();
    float vb = -INFINITY;
    int vi = tid;
    auto look = [&](const float* f, int vec) {
      float m = f[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) m = fmaxf(m, f[e]);
      if (TOPK && m > vb) {
        vb = m;
        vi = vec;
      }
      return m;
    };
    int v = tid;
    for (; v + (U - 1) * NTH < nvec; v += U * NTH) {
      float f[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) ld8(x + c0 + (v + u * NTH) * 8, f[u]);
      float m = st.m;
#pragma unroll
      for (int u = 0; u < U; ++u) m = fmaxf(m, look(f[u], v + u * NTH));
      if (m > st.m) stat_rescale(st, m);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) stat_add(st, f[u][e]);
    }
    for (; v < nvec; v += NTH) {
      float f[8];
      ld8(x + c0 + v * 8, f);
      const float m = fmaxf(st.m, look(f, v));
      if (m > st.m) stat_rescale(st, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) stat_add(st, f[e]);
    }
    float xt = -INFINITY;  // thread tid < tail holds element nvec·8 + tid
    if (tid < tail) {
      xt = load1(x + c0 + nvec * 8 + tid);
      if (xt > st.m) stat_rescale(st, xt);
      stat_add(st, xt);
    }
    // ---- the part's sums
    st = stat_wave(st);
    __syncthreads();  // the row before has been read out of LDS
    if ((tid & 63) == 0) sh_st[tid >> 6] = st;
    if (TOPK) {
      // lower bound of the thread's best key: the last index of its vector
      unsigned long long lo = tid < nvec ? key_of(vb, c0 + vi * 8 + 7) : 0;
      if (tid < tail) lo = max(lo, key_of(xt, c0 + nvec * 8 + tid));
      lo = gmax_key<GL>(lo);
      if (tid % GL == 0) gkey[tid / GL] = lo;
      if (tid == 0) {
        tau = 0;
        count = 0;
        nsel = 0;
      }
    }
    __syncthreads();
    st = sh_st[0];
#pragma unroll
    for (int w = 1; w < NTH / 64; ++w) st = stat_join(st, sh_st[w]);
    const bool bad = !(st.s == st.s);
    if (TOPK && !bad) {
      if (tid < G) {
        const unsigned long long me = gkey[tid];
        int rank = 0;
        for (int j = 0; j < G; ++j) rank += gkey[j] > me;
        if (me && rank == a.k - 1) tau = me;
      }
      __syncthreads();
      const unsigned long long t = tau;
      auto offer = [&](float f, int idx) {
        const unsigned long long key = key_of(f, idx);
        if (key >= t) {
          const int at = atomicAdd(&count, 1);
          if (at < CAND) cand[at] = key;
        }
      };
      if (tid < nvec && key_of(vb, c0 + vi * 8) >= t) sel[atomicAdd(&nsel, 1)] = (uint16_t)tid;
      __syncthreads();
      const int ns = nsel, per = (nvec + NTH - 1) / NTH;
      const float tv = t ? key_val(t) : -INFINITY;
      for (int i = tid; i < ns * per; i += NTH) {
        const int u = sel[i % ns] + i / ns * NTH;
        if (u >= nvec) continue;
        float f[8];
        ld8(x + c0 + u * 8, f);
        float m = f[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) m = fmaxf(m, f[e]);
        if (m < tv) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) offer(f[e], c0 + u * 8 + e);
      }
      if (tid < tail) offer(xt, c0 + nvec * 8 + tid);
      __syncthreads();
      const int n = count;
      if (n <= CAND) {
        rank_keys<NTH>(cand, n, a.k, best);
      } else {
        unsigned long long last = ~0ull;
        for (int j = 0; j < a.k; ++j) {
          unsigned long long mine = 0;
          for (int i = c0 + tid; i < c1; i += NTH) {
            const unsigned long long key = key_of(load1(x + i), i);
            if (key < last && key > mine) mine = key;
          }
          mine = gmax_key<64>(mine);
          __syncthreads();
          if ((tid & 63) == 0) gkey[tid >> 6] = mine;
          __syncthreads();
          last = gkey[0];
#pragma unroll
          for (int w = 1; w < NTH / 64; ++w) last = max(last, gkey[w]);
          if (tid == 0) best[j] = last;
        }
      }
      __syncthreads();
    }
    if (parts == 1) {
      const RowEnd r = row_end(st);
      if (tid == 0) write_row(a, row, lab, r);
      if (TOPK && tid < a.k) {
        a.top_lp[row * a.k + tid] = bad ? NAN : r.lp(key_val(best[tid]));
        a.top_idx[row * a.k + tid] = bad ? tid : (long)key_idx(best[tid]);
      }
    } else {
      if (tid == 0) ((Stat*)a.part_stat)[b] = st;
      if (TOPK && tid < a.k) a.part_key[b * a.k + tid] = bad ? 0 : best[tid];
    }
  }
}

// The parts of a row, one wave: lane p holds part p's sums and walks down its sorted candidates; k
// times the best head is taken.
template <typename T, bool TOPK>
__global__ void __launch_bounds__(64) logprob_join_kernel(LogProbArgs a, int parts) {
  __shared__ unsigned long long keys[TOPK ? LOGPROB_MAX_PARTS * MAX_K : 1];
  const int lane = threadIdx.x;
  for (long row = blockIdx.x; row < a.N; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.ld;
    RowLabel lab;
    lab.load(a, row, x);
    Stat st = stat_empty();
    if (lane < parts) st = ((const Stat*)a.part_stat)[row * parts + lane];
    if (TOPK) {
      __syncthreads();
      // 8 loads in flight: one after the other their latency was most of the launch
      const unsigned long long* from = a.part_key + row * parts * a.k;
      for (int i = lane; i < parts * a.k; i += 8 * 64) {
        unsigned long long v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = i + u * 64 < parts * a.k ? from[i + u * 64] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if (i + u * 64 < parts * a.k) keys[i + u * 64] = v[u];
      }
    }
    const RowEnd r = row_end(stat_wave(st));
    if (lane == 0) write_row(a, row, lab, r);
    if (TOPK) {
      __syncthreads();
      int at = 0;
      unsigned long long head = lane < parts ? keys[lane * a.k] : 0, mine = 0;
      for (int j = 0; j < a.k; ++j) {
        const unsigned long long best = gmax_key<64>(head);
        if (lane == j) mine = best;
        if (head == best && best) head = ++at < a.k ? keys[lane * a.k + at] : 0;
      }
      if (lane < a.k) {
        a.top_lp[row * a.k + lane] = r.bad ? NAN : r.lp(key_val(mine));
        a.top_idx[row * a.k + lane] = r.bad ? lane : (long)key_idx(mine);
      }
    }
  }
}

// Mean over the rows that count of −(log p + weight · H), and 1 / max(1, rows).  Several workgroups
// leave sums in part, one workgroup adds them in order (a captured step must not clear
// memory, and the order of float atomics would change the result).
constexpr int LOSS_ROWS = 4096;  // rows per workgroup

__global__ void __launch_bounds__(256) logprob_loss_kernel(const float* __restrict__ logp,
                                                           const float* __restrict__ ent,
                                                           const int64_t* __restrict__ labels,
                                                           long ignore, float weight, long N,
                                                           double* __restrict__ part,
                                                           float* __restrict__ loss,
                                                           float* __restrict__ inv) {
  __shared__ double sh[2][256];
  const int tid = threadIdx.x;
  double sum = 0, rows = 0;
  if (part && loss) {  // the join: part holds N pairs
    for (long i = tid; i < N; i += 256) {
      sum += part[2 * i];
      rows += part[2 * i + 1];
    }
  } else {
    const long first = (long)blockIdx.x * LOSS_ROWS, last = min(N, first + LOSS_ROWS);
    for (long i = first + tid; i < last; i += 256)
      if (labels[i] != ignore) {
        sum += (double)(weight != 0.f ? fmaf(weight, ent[i], logp[i]) : logp[i]);
        rows += 1;
      }
  }
  sh[0][tid] = sum;
  sh[1][tid] = rows;
  for (int o = 128; o > 0; o >>= 1) {
    __syncthreads();
    if (tid < o) {
      sh[0][tid] += sh[0][tid + o];
      sh[1][tid] += sh[1][tid + o];
    }
  }
  if (tid) return;
  if (loss) {
    const double i = 1.0 / (sh[1][0] > 1 ? sh[1][0] : 1.0);
    *loss = (float)(-sh[0][0] * i);
    *inv = (float)i;
  } else {
    part[2 * blockIdx.x] = sh[0][0];
    part[2 * blockIdx.x + 1] = sh[1][0];
  }
}

inline unsigned grid_for(long blocks) { return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)); }

// lanes per row and vectors per lane of the short-row kernels: the fewest lanes that hold the row
#define ROWS_DISPATCH(RUN)      \
  if (a.C <= 8) RUN(1, 1);      \
  else if (a.C <= 16) RUN(2, 1);   \
  else if (a.C <= 32) RUN(4, 1);   \
  else if (a.C <= 64) RUN(8, 1);   \
  else if (a.C <= 128) RUN(16, 1); \
  else if (a.C <= 256) RUN(32, 1); \
  else if (a.C <= 512) RUN(64, 1); \
  else if (a.C <= 1024) RUN(64, 2); \
  else RUN(64, 4)

template <typename T>
void fwd(const LogProbArgs& a, int parts, int part_len, hipStream_t st) {
  if (a.C <= LOGPROB_SHORT) {
#define RUN(L, V)                                                                       \
  do {                                                                                  \
    const unsigned g = grid_for((a.N + 256 / L - 1) / (256 / L));                       \
    if (a.k) logprob_rows_kernel<T, L, V, true><<<g, 256, 0, st>>>(a);                  \
    else logprob_rows_kernel<T, L, V, false><<<g, 256, 0, st>>>(a);                     \
  } while (0)
    ROWS_DISPATCH(RUN);
#undef RUN
    return;
  }
  const unsigned g = grid_for(a.N * parts);
  // 512 threads where every one of them gets four vectors (4096 × 131072 without alternatives:
  // 192 us; 256 threads 198, 1024 threads 222)
  if (part_len >= 512 * 32) {
    if (a.k) logprob_long_kernel<T, 512, true><<<g, 512, 0, st>>>(a, parts, part_len);
    else logprob_long_kernel<T, 512, false><<<g, 512, 0, st>>>(a, parts, part_len);
  } else {
    if (a.k) logprob_long_kernel<T, 256, true><<<g, 256, 0, st>>>(a, parts, part_len);
    else logprob_long_kernel<T, 256, false><<<g, 256, 0, st>>>(a, parts, part_len);
  }
  if (parts > 1) {
    const unsigned gj = grid_for(a.N);
    if (a.k) logprob_join_kernel<T, true><<<gj, 64, 0, st>>>(a, parts);
    else logprob_join_kernel<T, false><<<gj, 64, 0, st>>>(a, parts);
  }
}

template <typename T>
void bwd(const LogProbGradArgs& a, hipStream_t st) {
  if (a.C <= LOGPROB_SHORT) {
#define RUN(L, V)                                                        \
  logprob_rows_bwd_kernel<T, L, V>                                       \
      <<<grid_for((a.N + 256 / L - 1) / (256 / L)), 256, 0, st>>>(a)
    ROWS_DISPATCH(RUN);
#undef RUN
    return;
  }
  const uint32_t chunks = (uint32_t)cdiv(a.C, BWD_CHUNK);
  logprob_long_bwd_kernel<T><<<grid_for(a.N * chunks), 256, 0, st>>>(a, chunks);
}

}  // namespace

// parts of 2048 classes or more while there are fewer than 512 workgroups
int logprob_parts(long N, long C) {
  if (C <= LOGPROB_SHORT) return 1;
  long p = (512 + N - 1) / N;
  p = p < C / 2048 ? p : C / 2048;
  p = p < LOGPROB_MAX_PARTS ? p : LOGPROB_MAX_PARTS;
  return p < 1 ? 1 : (int)p;
}

void logprob_launch(const LogProbArgs& a, bool bf16, int parts, hipStream_t st) {
  // parts of whole vectors; the last one is the shortest, never empty
  const int part_len = (int)(((a.C + parts - 1) / parts + 7) / 8 * 8);
  parts = cdiv(a.C, part_len);
  if (bf16) fwd<bf16_t>(a, parts, part_len, st);
  else fwd<float>(a, parts, part_len, st);
}

long logprob_loss_parts(long N) { return N <= LOSS_ROWS ? 0 : (N + LOSS_ROWS - 1) / LOSS_ROWS; }

void logprob_loss_launch(const float* logp, const float* ent, const int64_t* labels, long ignore,
                         float weight, long N, double* part, float* loss, float* inv, hipStream_t st) {
  const long parts = logprob_loss_parts(N);
  if (!parts) {
    logprob_loss_kernel<<<1, 256, 0, st>>>(logp, ent, labels, ignore, weight, N, nullptr, loss, inv);
    return;
  }
  logprob_loss_kernel<<<(unsigned)parts, 256, 0, st>>>(logp, ent, labels, ignore, weight, N, part, nullptr, nullptr);
  logprob_loss_kernel<<<1, 256, 0, st>>>(logp, ent, labels, ignore, weight, parts, part, loss, inv);
}

void logprob_bwd_launch(const LogProbGradArgs& a, bool bf16, hipStream_t st) {
  if (bf16) bwd<bf16_t>(a, st);
  else bwd<float>(a, st);
}

}  // namespace tdl
