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
};

// q = rint(127 x / top), exactly rounded (ties to even) in both types.  c127 = 127·2^-64 and top is
// scaled alike for rows that reach 2^64, so that the product cannot overflow.
// bf16: 127 x is exact in 32 bits and, with 8-bit mantissas, the quotient is at least 2^-16 of
// itself away from the middle of two steps unless it is the middle.  Corrected once by its
// remainder it has an error of 2^-23 of itself and returns a representable quotient, which a middle
// is, exactly: every case is decided.
// fp32: the remainder 127 x − q top has 31 bits, exact in 64; it tells whether q is the nearest.
struct RowScale {
  float top, rtop, c127;
};
__device__ __forceinline__ RowScale row_scale(float top) {
  const float s = top >= 0x1p64f ? 0x1p-64f : 1.f;
  return RowScale{top * s, 1.f / (top * s), 127.f * s};
}
template <typename T>
__device__ __forceinline__ int quant1(float x, const RowScale& r);
template <>
__device__ __forceinline__ int quant1<bf16_t>(float x, const RowScale& r) {
  const float n = r.c127 * x;
  float q = n * r.rtop;
  q = fmaf(fmaf(-q, r.top, n), r.rtop, q);
  return (int)rintf(q);
}
template <>
__device__ __forceinline__ int quant1<float>(float x, const RowScale& s) {
  float q = rintf((s.c127 * x) * s.rtop);
  const double top = s.top, half = 0.5 * top, r = fma(-(double)q, top, (double)s.c127 * (double)x);
  const bool odd = (int)q & 1;
  if (r > half || (r == half && odd)) q += 1.f;
  if (r < -half || (r == -half && odd)) q -= 1.f;
  return (int)q;
}

// A workgroup of NW waves quantises 16 rows.  Lane l of a wave holds 16 elements of row l % 16 at
// k = 64 b + 16 (l / 16): reads are 16 segments of 128 bytes, the write is one block of 1 KiB.
// Wave w takes blocks w, w + NW, …; V of them stay in registers, longer rows are read twice.
template <typename T, int NW, int V, bool LONG>
__global__ void __launch_bounds__(64 * NW) quantize_kernel(const T* __restrict__ x, long ld, long M,
                                                           long K, int nb, int8_t* __restrict__ q,
                                                           float* __restrict__ scale) {
  __shared__ float sh[NW][16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r = lane & 15, c = lane >> 4;
  const long groups = (M + 15) / 16;
  for (long g = blockIdx.x; g < groups; g += gridDim.x) {
    const long row = g * 16 + r;
    const bool live = row < M;
    const T* xr = x + (live ? row : 0) * ld;
    Raw16<T> d[V];
    float top = 0.f;
    bool fin = true;
    auto fetch = [&](Raw16<T>& raw, int b) {
      const long k = (long)b * 64 + c * 16;
      raw.load(xr + k, live ? K - k : 0);
    };
    auto scan = [&](const Raw16<T>& raw) {
      float f[16];
      raw.get(f);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        top = fmaxf(top, fabsf(f[i]));
        fin = fin && fabsf(f[i]) < INFINITY;
      }
    };
    for (int b0 = w; b0 < nb; b0 += NW * V) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (b0 + v * NW < nb) fetch(d[v], b0 + v * NW);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (b0 + v * NW < nb) scan(d[v]);
      if (!LONG) break;
    }
    // a NaN or an infinity makes the row's scale NaN: it cannot be held in 8 bits
    if (!fin) top = INFINITY;
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    __syncthreads();
    if (lane < 16) sh[w][lane] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) top = fmaxf(top, sh[i][r]);
    top = fmaxf(top, TINY);
    const bool bad = top == INFINITY;
    if (threadIdx.x < 16 && live) scale[row] = bad ? NAN : top / 127.f;
    const RowScale rs = row_scale(top);
    auto emit = [&](const Raw16<T>& raw, int b) {
      float f[16];
      raw.get(f);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[i] |= (uint32_t)(uint8_t)(bad ? 0 : quant1<T>(f[4 * i + j], rs)) << (8 * j);
      }
      *(uint4*)(q + (g * nb + b) * 1024 + lane * 16) = make_uint4(o[0], o[1], o[2], o[3]);
    };
    for (int b0 = w; b0 < nb; b0 += NW * V) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (LONG && b0 + v * NW < nb) fetch(d[v], b0 + v * NW);
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (b0 + v * NW < nb) emit(d[v], b0 + v * NW);
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

// N fragments of 1 KiB each, consecutive in LDS; the wait is in the same block, so the registers
// hold the data when the compiler may use them
template <int N>
__device__ __forceinline__ void lds_frags(i32x4 (&f)[N], uint32_t at);
template <>
__device__ __forceinline__ void lds_frags<4>(i32x4 (&f)[4], uint32_t at) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %4 offset:1024\n\t"
      "ds_read_b128 %2, %4 offset:2048\n\tds_read_b128 %3, %4 offset:3072\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(f[0]), "=&v"(f[1]), "=&v"(f[2]), "=&v"(f[3])
      : "v"(at)
      : "memory");
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v, int left, bool vec);
template <>
__device__ __forceinline__ void store4<bf16_t>(bf16_t* p, const float* v, int left, bool vec) {
  if (vec && left >= 4) {
    *(uint2*)p = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) store1(p + i, v[i]);
  }
}
template <>
__device__ __forceinline__ void store4<float>(float* p, const float* v, int left, bool vec) {
  if (vec && left >= 4) {
    *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = v[i];
  }
}

// four outputs of one row from column n on
template <typename T>
__device__ __forceinline__ void finish4(const Int8GemmArgs& a, const i32x4& acc, long m, int n,
                                        float qs, bool vec) {
  if (m >= a.M || n >= a.N) return;
  const int left = a.N - n;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = i < left ? n + i : n;
    v[i] = (float)acc[i] * (qs * a.ws[j]);
    if (a.bias) v[i] += a.bias[j];
  }
  T* y = (T*)a.y + m * a.N + n;
  if (a.res) {
    const T* r = (const T*)a.res + m * a.N + n;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) v[i] += load1(r + i);
  }
  if (a.relu) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // NaN stays NaN
  }
  store4<T>(y, v, left, vec);
}

// BM × BN outputs per workgroup, 64 × 64 per wave; ST stages of 64 k in LDS, filled by LDS-DMA
// while the matrix unit works on the oldest.
template <typename T, int BM, int BN, int ST>
__global__ void __launch_bounds__(BM * BN / 64) gemm_kernel(Int8GemmArgs a) {
  constexpr int NW = BM / 64 * (BN / 64), WN = BN / 64;
  constexpr int BLK = (BM + BN) / 16, PER = BLK / NW;  // blocks of a stage, per wave
  static_assert(BLK % NW == 0, "every wave moves the same number of blocks");
  extern __shared__ char smem[];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nb = a.Kp / 64;
  const int tn = (a.N + BN - 1) / BN;
  const long m0 = (long)(blockIdx.x / tn) * BM;
  const int n0 = (int)(blockIdx.x % tn) * BN;
  // rows past the end read as zeros: the descriptors end with the last whole block row
  const long mrows = min((long)BM, (a.M + 15) / 16 * 16 - m0);
  const int nrows = min(BN, (a.N + 15) / 16 * 16 - n0);
  const rsrc_t ra = make_rsrc(a.q + m0 * a.Kp, (uint32_t)(mrows * a.Kp));
  const rsrc_t rb = make_rsrc(a.w + (long)n0 * a.Kp, (uint32_t)((long)nrows * a.Kp));
  auto issue = [&](int kt) {
    char* stage = smem + (kt % ST) * (BLK * 1024);
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int b = p * NW + w;  // 0 .. BM/16 − 1: activations, then weights
      const bool isa = b < BM / 16;
      const int rb16 = isa ? b : b - BM / 16;
      const uint32_t off = kt < nb ? (uint32_t)(rb16 * nb + kt) * 1024u + lane * 16u : 0xffffff00u;
      lds_void_t* dst = (lds_void_t*)(stage + b * 1024);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(isa ? ra : rb, dst, 16, off, 0, 0, 0);
    }
  };
  i32x4 acc[4][4] = {};
  const int wm = w / WN, wn = w % WN;
  for (int s = 0; s < ST - 1; ++s) issue(s);
  const uint32_t base = (uint32_t)(uintptr_t)(lds_void_t*)smem;
  for (int kt = 0; kt < nb; ++kt) {
    wait_vmcnt<PER*(ST - 2)>();
    raw_barrier();
    issue(kt + ST - 1);  // past the end: zeros into a slot nobody reads, and the count stays even
    const uint32_t st = base + (kt % ST) * (BLK * 1024) + lane * 16;
    i32x4 fa[4], fb[4];
    lds_frags<4>(fa, st + wm * 4096);
    lds_frags<4>(fb, st + (BM / 16) * 1024 + wn * 4096);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
  }
  wait_vmcnt<0>();  // no copy into LDS outlives the workgroup
  const bool vec = a.N % 4 == 0 && (uintptr_t)a.y % 16 == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long m = m0 + wm * 64 + i * 16 + (lane & 15);
    const float qs = m < a.M ? a.qs[m] : 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      finish4<T>(a, acc[i][j], m, n0 + wn * 64 + j * 16 + (lane >> 4) * 4, qs, vec);
  }
}

template <typename T>
void quantize(const T* x, long ld, long M, long K, int8_t* q, float* scale, hipStream_t st) {
  const int nb = (int)(int8_kp(K) / 64);
  const long groups = (M + 15) / 16;
  const unsigned grid = (unsigned)(groups < (1 << 20) ? groups : (1 << 20));
  if (nb <= 4 * 8) quantize_kernel<T, 4, 8, false><<<grid, 256, 0, st>>>(x, ld, M, K, nb, q, scale);
  else if (nb <= 8 * 8) quantize_kernel<T, 8, 8, false><<<grid, 512, 0, st>>>(x, ld, M, K, nb, q, scale);
  else quantize_kernel<T, 16, 4, true><<<grid, 1024, 0, st>>>(x, ld, M, K, nb, q, scale);
}

template <typename T>
void gemm(const Int8GemmArgs& a, hipStream_t st) {
  const long tiles = ((a.M + 127) / 128) * ((a.N + 127) / 128);
  constexpr int lds = 4 * 16 * 1024;
  gemm_kernel<T, 128, 128, 4><<<(unsigned)tiles, 256, lds, st>>>(a);
}

}  // namespace

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
