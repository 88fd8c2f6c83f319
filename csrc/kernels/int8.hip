// Linear layer / 1×1 convolution in 8-bit integers: one scale per row of the activations (token,
// pixel), one per output channel of the weights.
//
//   s_m = max_k |x_mk| / 127      q_mk = rint(127 x_mk / max)
//   y_mn = act( s_m · w_n · Σ_k q_mk W_nk + bias_n [+ res_mn] )
//
// The sum is exact (32-bit integers, K ≤ 131071); each output is rounded to its type once, from
// three 32-bit float operations.  Operand order in memory: int8.h.
#include "conv_common.h"
#include "int8.h"

#include <atomic>
#include <type_traits>

namespace tdl {
namespace {

using convk::make_rsrc;
using convk::rsrc_t;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void_t;

// ------------------------------------------------------------------------------- quantiser
// the smallest row maximum a scale is made from: rows below it quantise towards 0, not to NaN
constexpr float TINY = 0x1p-40f;

struct __attribute__((packed, aligned(2))) q4_a2 { uint32_t x, y, z, w; };
struct __attribute__((packed, aligned(4))) q4_a4 { float x, y, z, w; };

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
constexpr uint32_t INF_BITS = 0x7f800000u;

// 16 elements of a row as stored (any element alignment), the row's end filled with zeros
template <typename T>
struct Raw16;
template <>
struct Raw16<bf16_t> {
  uint4 v[2];
  __device__ __forceinline__ void load(const bf16_t* p, long left) {
    if (left >= 16) {
      const q4_a2 a = ((const q4_a2*)p)[0], b = ((const q4_a2*)p)[1];
      v[0] = make_uint4(a.x, a.y, a.z, a.w);
      v[1] = make_uint4(b.x, b.y, b.z, b.w);
    } else {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = (2 * i < left ? (uint32_t)p[2 * i] : 0u) |
               (2 * i + 1 < left ? (uint32_t)p[2 * i + 1] << 16 : 0u);
      v[0] = make_uint4(w[0], w[1], w[2], w[3]);
      v[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
  }
  __device__ __forceinline__ void get(float* f) const {
    unpack8(v[0], f);
    unpack8(v[1], f + 8);
  }
  // max |x| as the bits of a float: in integer order NaN is above infinity above every number
  __device__ __forceinline__ uint32_t top() const {
    const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu));
    return (uint32_t)max(m[0], m[1]) << 16;
  }
};
template <>
struct Raw16<float> {
  float v[16];
  __device__ __forceinline__ void load(const float* p, long left) {
    if (left >= 16) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const q4_a4 a = ((const q4_a4*)p)[i];
        v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = i < left ? p[i] : 0.f;
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = v[i];
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
};

// q = rint(127 x / top), exactly rounded (ties to even) in both types.  c127 = 127·2^-64 and top is
// scaled alike for rows that reach 2^64, so that the product cannot overflow.
// bf16: 127 x is exact in 32 bits and, with 8-bit mantissas, the quotient is at least 2^-16 of
// itself away from the middle of two steps unless it is the middle.  Corrected once by its
// remainder it has an error of 2^-23 of itself and returns a representable quotient, which a middle
// is, exactly: every case is decided.
// fp32: a quotient that is not within 2^-13 of a middle has the right nearest integer (its error is
// below 127·2^-22); else the remainder 127 x − q top, 31 bits, exact in 64, tells.
struct RowScale {
  float top, rtop, c127;
};
__device__ __forceinline__ RowScale row_scale(float top) {
  const float s = top >= 0x1p64f ? 0x1p-64f : 1.f;
  return RowScale{top * s, 1.f / (top * s), 127.f * s};
}
// the result's low byte is q: adding 1.5·2^23 rounds to the nearest integer, ties to even, and
// leaves it in the low bits
template <typename T>
__device__ __forceinline__ uint32_t quant1(float x, const RowScale& r);
template <>
__device__ __forceinline__ uint32_t quant1<bf16_t>(float x, const RowScale& r) {
  const float n = r.c127 * x;
  float q = n * r.rtop;
  q = fmaf(fmaf(-q, r.top, n), r.rtop, q);
  return __float_as_uint(q + 12582912.f);
}
template <>
__device__ __forceinline__ uint32_t quant1<float>(float x, const RowScale& s) {
  const float t = (s.c127 * x) * s.rtop;
  float q = rintf(t);
  if (!(fabsf(t - q) < 0.5f - 0x1p-13f)) {
    const double top = s.top, half = 0.5 * top, r = fma(-(double)q, top, (double)s.c127 * (double)x);
    const bool odd = (int)q & 1;
    if (r > half || (r == half && odd)) q += 1.f;
    if (r < -half || (r == -half && odd)) q -= 1.f;
  }
  return __float_as_uint(q + 12582912.f);
}
template <typename T>
__device__ __forceinline__ uint32_t quant4(const float* f, const RowScale& r) {
  const uint32_t a = quant1<T>(f[0], r), b = quant1<T>(f[1], r), c = quant1<T>(f[2], r), d = quant1<T>(f[3], r);
  // bytes: 0–3 of the second operand, 4–7 of the first
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                               0x05040100u);
}

// A workgroup of NW waves quantises RG rows (16 or 4).  Lane l of a wave holds 16 elements of row
// l % RG at k = (1024 / RG) u + 16 (l / RG).  RG = 16: reads are 16 segments of 64 elements, the write
// is one block of 1 KiB; RG = 4: 4 segments of 256 elements and 16 pieces of 64 bytes of 4 blocks.
// Wave w takes steps u = w, w + NW, …; V of them stay in registers, longer rows are read twice.
template <typename T, int RG, int NW, int V, bool LONG>
__global__ void __launch_bounds__(64 * NW) quantize_kernel(const T* __restrict__ x, long ld, long M,
                                                           long K, int nb, int8_t* __restrict__ q,
                                                           float* __restrict__ scale) {
  constexpr int BW = 16 / RG;  // blocks of 64 k a wave covers at once
  __shared__ uint32_t sh[NW][RG];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane % RG, c = lane / RG;
  const int nu = (nb + BW - 1) / BW;
  const long groups = (M + 15) / 16 * BW;
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const long row = g * RG + r;
    const bool live = row < M;
    const T* xr = x + (live ? row : 0) * ld;
    Raw16<T> d[V];
    uint32_t bits = 0;
    auto fetch = [&](Raw16<T>& raw, int u) {
      const long k = ((long)u * (64 / RG) + c) * 16;
      raw.load(xr + k, live ? K - k : 0);
    };
    for (int u0 = w; u0 < nu; u0 += NW * V) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (u0 + v * NW < nu) fetch(d[v], u0 + v * NW);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (u0 + v * NW < nu) bits = max(bits, d[v].top());
      if (!LONG) break;
    }
#pragma unroll
    for (int o = RG; o < 64; o *= 2) bits = max(bits, __shfl_xor(bits, o, 64));
    __syncthreads();
    if (lane < RG) sh[w][lane] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) bits = max(bits, sh[i][r]);
    // a NaN or an infinity makes the row's scale NaN: it cannot be held in 8 bits
    const bool bad = bits >= INF_BITS;
    const float top = fmaxf(__uint_as_float(bits), TINY);
    if (threadIdx.x < RG && live) scale[row] = bad ? NAN : top / 127.f;
    const RowScale rs = row_scale(top);
    auto emit = [&](const Raw16<T>& raw, int u) {
      float f[16];
      raw.get(f);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = bad ? 0u : quant4<T>(f + 4 * i, rs);
      const int b = u * BW + c / 4;
      if (BW == 1 || b < nb)
        *(uint4*)(q + (row / 16 * nb + b) * 1024 + (c % 4 * 16 + row % 16) * 16) =
            make_uint4(o[0], o[1], o[2], o[3]);
    };
    for (int u0 = w; u0 < nu; u0 += NW * V) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (LONG && u0 + v * NW < nu) fetch(d[v], u0 + v * NW);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (u0 + v * NW < nu) emit(d[v], u0 + v * NW);
      if (!LONG) break;
    }
  }
}

// ------------------------------------------------------------------------------- product
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void raw_barrier() { asm volatile("s_barrier" ::: "memory"); }

// One wave copies a block of 1 KiB into LDS at the wave-uniform address dst.  Written as assembly
// so that the compiler does not wait for every copy in flight before each LDS read; the waits are
// explicit (vmcnt, then a barrier).  No register is written.
__device__ __forceinline__ void dma_block(rsrc_t r, uint32_t dst, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(dst), "v"(off), "s"(r)
               : "memory", "m0");
}

typedef __attribute__((address_space(3))) const i32x4 lds_i32x4;
__device__ __forceinline__ i32x4 lds_frag(uint32_t at) { return *(lds_i32x4*)(uintptr_t)at; }

// 8 elements of a row at any element alignment, as stored; the first `left` of them are the row's
template <typename T>
struct Raw8;
template <>
struct Raw8<bf16_t> {
  uint4 v;
  __device__ __forceinline__ void load(const bf16_t* p, int left) {
    if (left >= 8) {
      const q4_a2 a = *(const q4_a2*)p;
      v = make_uint4(a.x, a.y, a.z, a.w);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = (2 * i < left ? (uint32_t)p[2 * i] : 0u) |
               (2 * i + 1 < left ? (uint32_t)p[2 * i + 1] << 16 : 0u);
      v = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ void get(float* f) const { unpack8(v, f); }
};
template <>
struct Raw8<float> {
  float v[8];
  __device__ __forceinline__ void load(const float* p, int left) {
    if (left >= 8) {
      const q4_a4 a = ((const q4_a4*)p)[0], b = ((const q4_a4*)p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : 0.f;
    }
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = v[i];
  }
};
__device__ __forceinline__ void ld8u(const float* p, float* f) {
  const q4_a4 a = ((const q4_a4*)p)[0], b = ((const q4_a4*)p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
// two values per conversion instruction
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void st8u(bf16_t* p, const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bf16x2 h = __builtin_convertvector((f32x2{f[2 * i], f[2 * i + 1]}), bf16x2);
    w[i] = __builtin_bit_cast(uint32_t, h);
  }
  *(q4_a2*)p = q4_a2{w[0], w[1], w[2], w[3]};
}
__device__ __forceinline__ void st8u(float* p, const float* f) {
  ((q4_a4*)p)[0] = q4_a4{f[0], f[1], f[2], f[3]};
  ((q4_a4*)p)[1] = q4_a4{f[4], f[5], f[6], f[7]};
}

// 16-row tiles to workgroups: XCD x takes a contiguous run (its L2 keeps what neighbours share),
// ordered in groups of 8 row tiles, down the rows first
__device__ __forceinline__ void tile_of(int id, int tm, int tn, int* m, int* n) {
  constexpr int GM = 8;
  id = xcd_remap(id, tm * tn);
  const int per = GM * tn, g = id / per, gm = min(GM, tm - g * GM), r = id - g * per;
  *n = r / gm;
  *m = g * GM + r - *n * gm;
}

typedef int i32x16 __attribute__((ext_vector_type(16)));

// A wave's products on MF × MF tiles of the matrix unit (16×16×64 or 32×32×32; the weights are the
// first operand, so a lane holds 4 consecutive columns of one row).  R rows × C columns of 16.
template <int MF, int R, int C>
struct Tile;
template <int R, int C>
struct Tile<16, R, C> {
  i32x4 acc[R][C] = {};
  // lane l: row l % 16, k = 16 (l / 16)
  static __device__ __forceinline__ uint32_t lane_off(int l) { return l * 16; }
  static __device__ __forceinline__ constexpr uint32_t frag_off(int i) { return i * 1024; }
  __device__ __forceinline__ void products(const i32x4 (&a)[R], const i32x4 (&b)[C]) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[j], a[i], acc[i][j], 0, 0, 0);
  }
  // row tile i to LDS: put(row in the tile, column, 4 values)
  template <typename F>
  __device__ __forceinline__ void each(int i, int l, F put) {
#pragma unroll
    for (int j = 0; j < C; ++j) put(l & 15, j * 16 + (l >> 4) * 4, acc[i][j]);
  }
};
template <int R, int C>
struct Tile<32, R, C> {
  i32x16 acc[R / 2][C / 2] = {};
  // lane l: row l % 32, k = 16 (l / 32) of the 32 of a fragment; fragment i: rows 32 (i / 2), k half i % 2
  static __device__ __forceinline__ uint32_t lane_off(int l) {
    return ((l >> 4) & 1) * 1024 + (l >> 5) * 256 + (l & 15) * 16;
  }
  static __device__ __forceinline__ constexpr uint32_t frag_off(int i) { return (i >> 1) * 2048 + (i & 1) * 512; }
  __device__ __forceinline__ void products(const i32x4 (&a)[R], const i32x4 (&b)[C]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < R / 2; ++i)
#pragma unroll
        for (int j = 0; j < C / 2; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[2 * j + h], a[2 * i + h], acc[i][j], 0, 0, 0);
  }
  template <typename F>
  __device__ __forceinline__ void each(int i, int l, F put) {
#pragma unroll
    for (int j = 0; j < C / 2; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        put(l & 31, j * 32 + g * 8 + (l >> 5) * 4,
            i32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]});
  }
};

// FM × FN blocks of 16 × 16 per wave, WM × WN waves, ST stages of 64 KB k in LDS.
//
// Step kt: the copies of stage kt + 1 have landed (vmcnt, barrier); stage kt + ST − 1 is copied into
// the slot of stage kt − 1, whose fragments went into products before the barrier; the fragments of
// kt + 1 are read while the products of kt run.  Copies past the end read zeros, which keeps the
// count of copies in flight the same in every step.
// (16 waves per CU, two workgroups, where the accumulators leave registers for it)
template <typename T, int MF, int FM, int FN, int WM, int WN, int KB, int ST>
__global__ void __launch_bounds__(64 * WM * WN, FM * FN <= 8 ? 4 : 2) gemm_kernel(Int8GemmArgs a) {
  constexpr int NW = WM * WN, BM = FM * 16 * WM, BN = FN * 16 * WN;
  constexpr int BLK = (BM + BN) / 16, PER = BLK * KB / NW, STAGE = BLK * KB * 1024;
  static_assert(BLK * KB % NW == 0, "every wave moves the same number of blocks");
  static_assert(ST >= 3, "");
  extern __shared__ char smem[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int nb = a.Kp / 64;
  const int tn = (a.N + BN - 1) / BN, tm = (int)((a.M + BM - 1) / BM);
  int im, in;
  tile_of(blockIdx.x, tm, tn, &im, &in);
  const long m0 = (long)im * BM;
  const int n0 = in * BN;
  // rows past the end read as zeros: the descriptors end with the last whole block row
  const long mrows = min((long)BM, (a.M + 15) / 16 * 16 - m0);
  const int nrows = min(BN, (a.N + 15) / 16 * 16 - n0);
  const rsrc_t ra = make_rsrc(a.q + m0 * a.Kp, (uint32_t)(mrows * a.Kp));
  const rsrc_t rb = make_rsrc(a.w + (long)n0 * a.Kp, (uint32_t)((long)nrows * a.Kp));
  const uint32_t base = (uint32_t)(uintptr_t)(lds_void_t*)smem;
  uint32_t off[PER];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const int i = p * NW + w, b = i % BLK;  // [k block][BM/16 of activations, BN/16 of weights]
    off[p] = (uint32_t)((b < BM / 16 ? b : b - BM / 16) * nb + i / BLK) * 1024u + lane * 16u;
  }
  auto issue = [&](int kt, int slot) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int i = p * NW + w, b = i % BLK;
      const uint32_t o = kt * KB + i / BLK < nb ? off[p] + (uint32_t)(kt * KB) * 1024u : convk::OOB;
      const uint32_t dst = base + slot * STAGE + i * 1024;
      // (which operand: known at compile time where a round of the waves does not straddle them)
      if (p * NW % BLK + NW <= BM / 16) dma_block(ra, dst, o);
      else if (p * NW % BLK >= BM / 16 && p * NW % BLK + NW <= BLK) dma_block(rb, dst, o);
      else dma_block(b < BM / 16 ? ra : rb, dst, o);
    }
  };
  using Acc = Tile<MF, FM, FN>;
  Acc t;
  const int wm = w / WN, wn = w % WN;
  const uint32_t fa0 = base + wm * FM * 1024 + Acc::lane_off(lane);
  const uint32_t fb0 = base + (BM / 16) * 1024 + wn * FN * 1024 + Acc::lane_off(lane);
  auto frags = [&](i32x4(&fa)[KB][FM], i32x4(&fb)[KB][FN], int slot) {
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const uint32_t at = slot * STAGE + k * BLK * 1024;
#pragma unroll
      for (int j = 0; j < FN; ++j) fb[k][j] = lds_frag(fb0 + at + Acc::frag_off(j));
#pragma unroll
      for (int i = 0; i < FM; ++i) fa[k][i] = lds_frag(fa0 + at + Acc::frag_off(i));
    }
  };
  i32x4 xa[KB][FM], xb[KB][FN], ya[KB][FM], yb[KB][FN];
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) issue(s, s);
  // Epilogue layout (below): lane l finishes 8 columns of row l / CPR of each pass.  Its scales and
  // biases are loaded behind the first copies (one after the other behind the products they cost
  // more than a short sum), and the residual where it leaves registers for two workgroups per CU
  // (50176 × 256 → 1024 fp32: 94 us, loaded ahead there too 105).
  constexpr int CPR = FN * 2, RPI = 64 / CPR, PASSES = FM * 16 / RPI;
  constexpr bool PRE = PASSES * 8 * sizeof(T) <= 64;
  const bool inside = m0 + BM <= a.M && n0 + BN <= a.N;
  const int col = n0 + wn * FN * 16 + lane % CPR * 8;
  const int left = a.N - col;
  const long row0 = m0 + wm * FM * 16 + lane / CPR;
  const T* res0 = (const T*)a.res + row0 * a.N + col;
  float ws[8], bias[8] = {}, qs[PASSES];
  Raw8<T> res[PRE ? PASSES : 1];
  if (inside) {
    ld8u(a.ws + col, ws);
    if (a.bias) ld8u(a.bias + col, bias);
#pragma unroll
    for (int p = 0; p < PASSES; ++p) qs[p] = a.qs[row0 + p * RPI];
    if (PRE && a.res) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p) res[p].load(res0 + (long)p * RPI * a.N, 8);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = min(col + e, a.N - 1);
      ws[e] = a.ws[c];
      if (a.bias) bias[e] = a.bias[c];
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) qs[p] = a.qs[min(row0 + p * RPI, a.M - 1)];
    if (PRE && a.res) {
#pragma unroll
      for (int p = 0; p < PASSES; ++p)
        res[p].load(res0 + (long)p * RPI * a.N, row0 + p * RPI < a.M ? left : 0);
    }
  }
  wait_vmcnt<PER*(ST - 2)>();
  raw_barrier();
  frags(xa, xb, 0);
  int slot = 0;  // of stage kt
  auto next = [](int s) { return s + 1 == ST ? 0 : s + 1; };
  auto step = [&](int kt, const i32x4(&fa)[KB][FM], const i32x4(&fb)[KB][FN], i32x4(&ga)[KB][FM],
                  i32x4(&gb)[KB][FN]) {
    // no product of the step before moves below the barrier: its fragments' slot is refilled here
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<PER*(ST - 3)>();
    raw_barrier();
    issue(kt + ST - 1, slot == 0 ? ST - 1 : slot - 1);
    slot = next(slot);
    frags(ga, gb, slot);
#pragma unroll
    for (int k = 0; k < KB; ++k) t.products(fa[k], fb[k]);
  };
  // two steps at a time; a step past the end multiplies the zeros its copies brought
  for (int kt = 0; kt * KB < nb; kt += 2) {
    step(kt, xa, xb, ya, yb);
    step(kt + 1, ya, yb, xa, xb);
  }
  __builtin_amdgcn_sched_barrier(0);
  wait_vmcnt<0>();  // no copy into LDS outlives the loop
  raw_barrier();

  // Epilogue, MF rows at a time through the wave's own part of LDS: the matrix unit leaves 4 columns
  // of one row in a lane, memory wants whole rows.
  constexpr int PITCH = FN * 64 + 16;
  const uint32_t ep = base + w * MF * PITCH;
  T* y0 = (T*)a.y + row0 * a.N + col;
  auto finish = [&](auto whole) {  // whole: the tile lies inside y
    constexpr bool W = decltype(whole)::value;
#pragma unroll
    for (int i = 0; i < FM * 16 / MF; ++i) {
      t.each(i, lane, [&](int r, int c, const i32x4& v) {
        *(__attribute__((address_space(3))) i32x4*)(uintptr_t)(ep + r * PITCH + c * 4) = v;
      });
      // lanes read what others wrote: one wave's LDS accesses run in order, and stay in it here
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int r = 0; r < MF; r += RPI) {
        const uint32_t at = ep + (r + lane / CPR) * PITCH + lane % CPR * 32;
        const i32x4 lo = lds_frag(at), hi = lds_frag(at + 16);
        const int pass = (i * MF + r) / RPI;
        if (!W && (row0 + i * MF + r >= a.M || left <= 0)) continue;
        const long d = (long)(i * MF + r) * a.N;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)(e < 4 ? lo[e] : hi[e - 4]) * (qs[pass] * ws[e]) + bias[e];
        if (a.res) {
          float add[8];
          if (!PRE) res[0].load(res0 + d, W ? 8 : left);
          res[PRE ? pass : 0].get(add);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += add[e];
        }
        if (a.relu) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __builtin_elementwise_maximum(v[e], 0.f);  // NaN stays NaN
        }
        if (W || left >= 8) {
          st8u(y0 + d, v);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < left) store1(y0 + d + e, v[e]);
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  if (inside) finish(std::true_type());
  else finish(std::false_type());
}

template <typename T, int RG>
void quantize_groups(const T* x, long ld, long M, long K, int8_t* q, float* scale, hipStream_t st) {
  const int nb = (int)(int8_kp(K) / 64), nu = (nb * RG + 15) / 16;
  const long groups = (M + 15) / 16 * (16 / RG);
  const unsigned grid = (unsigned)(groups < (1 << 20) ? groups : (1 << 20));
  // waves enough that each holds few blocks: 16 rows alone are little work for a workgroup
#define QUANT(NW, V, LONG)                                                                      \
  return quantize_kernel<T, RG, NW, V, LONG><<<grid, 64 * NW, 0, st>>>(x, ld, M, K, nb, q, scale)
  if (nu <= 4) QUANT(4, 1, false);
  if (nu <= 8) QUANT(8, 1, false);
  if (nu <= 16) QUANT(16, 1, false);
  if (nu <= 32) QUANT(16, 2, false);
  if (nu <= 64) QUANT(16, 4, false);
  if constexpr (sizeof(T) == 2)  // (fp32: more registers than there are)
    if (nu <= 128) QUANT(16, 8, false);
  QUANT(16, 4, true);
#undef QUANT
}
template <typename T>
void quantize(const T* x, long ld, long M, long K, int8_t* q, float* scale, hipStream_t st) {
  // 4 rows per workgroup where 16 would leave CUs idle (256 × 4096 bf16: 4.4 us against 8.3; 4096 ×
  // 4096: 12.2 against 10.7, whose 64-byte pieces of the blocks cost more) or hold too much of a row
  // per wave (8192 × 8192: 34.8 against 41.2 on one input, 42 against 47 on inputs that the last-level
  // cache does not hold; 1024 × 8192 fp32 9.5 against 36.9)
  const long few = sizeof(T) == 2 ? 160 * 16 : 96 * 16;
  if (K > 4096 || (K > 512 && M < few)) quantize_groups<T, 4>(x, ld, M, K, q, scale, st);
  else quantize_groups<T, 16>(x, ld, M, K, q, scale, st);
}

// ------------------------------------------------------------------------------- few rows
// Up to 16 MB rows: the weights are read once, straight into registers in the order the matrix unit
// takes them, so the kernel is a stream over them.  A workgroup owns 16 output channels; its NW
// waves take the blocks of 64 k in turn, U loads of 1 KiB in flight each, and add their sums in LDS.
//
// FUSED (x in its own type instead of quantised blocks): every workgroup quantises the rows itself,
// under the latency of its first weight loads; a launch of its own costs 3 us more while that is
// little work (1 × 2048 → 1000: 3.7 us against 7.5; int8_linear_fused below).
constexpr int FUSED_ROWS = 16, FUSED_ITEMS = 4;

template <typename T, int MB, int NW, bool FUSED>
__global__ void __launch_bounds__(64 * NW) stream_kernel(Int8GemmArgs a, const T* __restrict__ x,
                                                         long ld, long K) {
  constexpr int U = 8;
  static_assert(!FUSED || MB == 1, "");
  extern __shared__ char smem[];  // FUSED: quantised rows, [Kp / 16][M][16 bytes]
  __shared__ i32x4 part[NW][MB][64];
  __shared__ uint32_t tops[FUSED_ROWS];
  __shared__ float scales[FUSED_ROWS];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int nb = a.Kp / 64, M = (int)a.M;
  const int n0 = blockIdx.x * 16;
  const i32x4* wp = (const i32x4*)(a.w + (long)blockIdx.x * 16 * a.Kp) + lane;
  i32x4 wr[U];
  auto fetch = [&](int kb0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (kb0 + u * NW < nb) wr[u] = wp[(long)(kb0 + u * NW) * 64];
  };
  fetch(w);
  if (FUSED) {
    const int kc = a.Kp / 16, items = M * kc;
    if (tid < FUSED_ROWS) tops[tid] = 0;
    __syncthreads();
    // items past the end hold zeros of the last row: every lane stays in the wave's reductions
    Raw16<T> d[FUSED_ITEMS];
    int row[FUSED_ITEMS], ck[FUSED_ITEMS];
#pragma unroll
    for (int i = 0; i < FUSED_ITEMS; ++i) {
      if (i * 64 * NW >= items) break;
      const int item = tid + i * 64 * NW;
      row[i] = item < items ? item / kc : M - 1;
      ck[i] = item < items ? item - row[i] * kc : kc;
      d[i].load(x + row[i] * ld + ck[i] * 16, K - ck[i] * 16);
    }
#pragma unroll
    for (int i = 0; i < FUSED_ITEMS; ++i) {
      if (i * 64 * NW >= items) break;
      uint32_t bits = d[i].top();
      // one atomic per wave where the wave is within a row
      const int row0 = __builtin_amdgcn_readfirstlane(row[i]);
      if (__all(row[i] == row0)) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) bits = max(bits, __shfl_xor(bits, o, 64));
        if (lane == 0) atomicMax(&tops[row0], bits);
      } else {
        atomicMax(&tops[row[i]], bits);
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < FUSED_ITEMS; ++i) {
      if (i * 64 * NW >= items) break;
      if (ck[i] >= kc) continue;
      const bool bad = tops[row[i]] >= INF_BITS;
      const float top = fmaxf(__uint_as_float(tops[row[i]]), TINY);
      if (ck[i] == 0) scales[row[i]] = bad ? NAN : top / 127.f;
      const RowScale rs = row_scale(top);
      float f[16];
      d[i].get(f);
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = bad ? 0u : quant4<T>(f + 4 * j, rs);
      ((uint4*)smem)[ck[i] * M + row[i]] = make_uint4(o[0], o[1], o[2], o[3]);
    }
    __syncthreads();
  }
  i32x4 acc[MB] = {};
  const int r = lane & 15, c = lane >> 4;
  const i32x4* qp = (const i32x4*)a.q + lane;
  for (int kb0 = w; kb0 < nb; kb0 += NW * U) {
    if (kb0 != w) fetch(kb0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * NW;
      if (kb >= nb) break;
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        // rows past the last one repeat it: their sums are not stored
        const i32x4 q = FUSED ? ((const i32x4*)smem)[(kb * 4 + c) * M + min(r, M - 1)]
                              : m * 16 < M ? qp[((long)m * nb + kb) * 64] : i32x4{};
        acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wr[u], q, acc[m], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MB; ++m) part[w][m][lane] = acc[m];
  __syncthreads();
  // lane l of a sum holds channels 4 (l / 16) … + 3 of row l % 16
  for (int o = tid; o < MB * 256; o += 64 * NW) {
    const int row = o >> 4, ch = o & 15, n = n0 + ch;
    if (row >= M || n >= a.N) continue;
    int sum = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) sum += part[i][row >> 4][(ch >> 2) * 16 + (row & 15)][ch & 3];
    const float qs = FUSED ? scales[row] : a.qs[row];
    const long at = (long)row * a.N + n;
    float v = (float)sum * (qs * a.ws[n]) + (a.bias ? a.bias[n] : 0.f) +
              (a.res ? load1((const T*)a.res + at) : 0.f);
    if (a.relu && v < 0.f) v = 0.f;
    store1((T*)a.y + at, v);
  }
}

// true at the first call on each device (a kernel's LDS limit is set per device)
struct DeviceOnce {
  std::atomic<bool> done[64] = {};
  bool first() {
    int d = 0;
    if (hipGetDevice(&d) != hipSuccess || d < 0 || d >= 64) return true;
    return !done[d].exchange(true);
  }
};

template <typename T, int MF, int FM, int FN, int WM, int WN, int KB, int ST>
void run_gemm(const Int8GemmArgs& a, hipStream_t st) {
  constexpr int BM = FM * 16 * WM, BN = FN * 16 * WN, ring = ST * KB * (BM + BN) * 64,
                epi = WM * WN * MF * (FN * 64 + 16), lds = ring > epi ? ring : epi;
  static DeviceOnce once;
  if (lds > 64 * 1024 && once.first())
    (void)hipFuncSetAttribute((const void*)gemm_kernel<T, MF, FM, FN, WM, WN, KB, ST>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  const long tiles = ((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  gemm_kernel<T, MF, FM, FN, WM, WN, KB, ST><<<(unsigned)tiles, 64 * WM * WN, lds, st>>>(a);
}

template <typename T, int MB, int NW, bool FUSED>
void run_stream(const Int8GemmArgs& a, const T* x, long ld, long K, hipStream_t st) {
  const int lds = FUSED ? (int)(a.M * a.Kp) : 0;
  if (FUSED) {
    static DeviceOnce once;
    if (once.first())
      (void)hipFuncSetAttribute((const void*)stream_kernel<T, MB, NW, FUSED>,
                                hipFuncAttributeMaxDynamicSharedMemorySize, FUSED_ITEMS * 1024 * 16);
  }
  stream_kernel<T, MB, NW, FUSED><<<(unsigned)((a.N + 15) / 16), 64 * NW, lds, st>>>(a, x, ld, K);
}

template <typename T>
void gemm(const Int8GemmArgs& a, hipStream_t st) {
  // few rows: 32 × 2048 → 1000 3.5 us on the stream, 6.5 on tiles; 64 × 2048 → 1000 4.9 and 6.3; 64 ×
  // 4096 → 4096 10.6 and 9.1 (each workgroup reads all the rows again: tiles share them)
  if (a.M <= 32 || (a.M <= 64 && a.Kp <= 2048)) {
    const bool wide = a.Kp > 64 * 64;  // waves enough to keep 4 loads or more in flight in each
    if (a.M <= 16) wide ? run_stream<T, 1, 16, false>(a, nullptr, 0, 0, st) : run_stream<T, 1, 8, false>(a, nullptr, 0, 0, st);
    else if (a.M <= 32) wide ? run_stream<T, 2, 16, false>(a, nullptr, 0, 0, st) : run_stream<T, 2, 8, false>(a, nullptr, 0, 0, st);
    else run_stream<T, 4, 8, false>(a, nullptr, 0, 0, st);
    return;
  }
  auto tiles = [&](long bm, long bn) { return ((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn); };
  // 256 × 256 reads LDS and L2 least (8192³, 200 calls in a row: 407 us on uniform random bytes, 384 on
  // rectified activations, 128 × 128 510 and 458; 16384 × 4096 → 1024 56 and 66) but
  // leaves one workgroup per CU, which short sums do not hide (50176 × 256 → 1024: 73 us against 55).
  // 64 × 64, 128 k per step, while 128 × 128 gives no more than a tile to every other CU (512 × 4096 →
  // 4096, 128 tiles: 15.3 us against 17.7; 1024 × 4096 → 4096, 256 tiles: 28 against 21).  The
  // 32×32×32 form of the matrix unit wins on the smaller tiles (2049 × 1999 → 1003 on 128 × 128: 14.3
  // us against 19.5), the 16×16×64 form on the large one (8192³: 407 against 433 us, 384 against 389).
  if (tiles(256, 256) >= 180 && a.Kp >= 1024) run_gemm<T, 16, 8, 4, 2, 4, 1, 4>(a, st);
  else if (tiles(128, 128) > 128) run_gemm<T, 32, 4, 2, 2, 4, 1, 4>(a, st);
  else run_gemm<T, 32, 2, 2, 2, 2, 2, 4>(a, st);
}

}  // namespace

// Few rows, few enough 16-element items for the registers (fp32: half as many), and less than 2^20
// (fp32: 2^19) of them over all workgroups, which all quantise the same rows: 16 × 4096 → 4096 in
// bf16, 2^20 items, 10.2 us against 12.8 with a launch for them; 8 × 4096 → 16384, 2^21, 22.0
// against 20.0; in fp32 8 × 4096 → 4096, 2^19, 10.6 against 14.7 and 4 × 4096 → 16384, 2^20, 26.5
// against 22.1.
bool int8_linear_fused(long M, long N, long Kp, bool bf16) {
  const long items = M * (Kp / 16), all = items * ((N + 15) / 16);
  return M <= FUSED_ROWS && items <= FUSED_ITEMS * (bf16 ? 1024 : 512) && all <= 1l << (bf16 ? 20 : 19);
}

namespace {

template <typename T>
void linear(const T* x, long ld, long K, Int8GemmArgs a, int8_t* q, float* qs, hipStream_t st) {
  if (int8_linear_fused(a.M, a.N, a.Kp, sizeof(T) == 2)) {
    if (a.M * (a.Kp / 16) <= FUSED_ITEMS * 512 && (a.Kp <= 64 * 64 || sizeof(T) == 4))
      return run_stream<T, 1, 8, true>(a, x, ld, K, st);
    if constexpr (sizeof(T) == 2) return run_stream<T, 1, 16, true>(a, x, ld, K, st);
  }
  quantize(x, ld, a.M, K, q, qs, st);
  a.q = q;
  a.qs = qs;
  gemm<T>(a, st);
}

}  // namespace

void int8_linear_launch(const void* x, long ld, long K, const Int8GemmArgs& a, int8_t* q, float* qs,
                        bool bf16, hipStream_t st) {
  if (bf16) linear((const bf16_t*)x, ld, K, a, q, qs, st);
  else linear((const float*)x, ld, K, a, q, qs, st);
}

void int8_quantize_launch(const void* x, long ld, bool bf16, long M, long K, int8_t* q,
                          float* scale, hipStream_t st) {
  if (bf16) quantize((const bf16_t*)x, ld, M, K, q, scale, st);
  else quantize((const float*)x, ld, M, K, q, scale, st);
}

void int8_gemm_launch(const Int8GemmArgs& a, bool bf16, hipStream_t st) {
  if (bf16) gemm<bf16_t>(a, st);
  else gemm<float>(a, st);
}

}  // namespace tdl
