// Inverted dropout whose mask is a function of a counter and is never stored:
//
//   y_i = keep_i ? x_i / (1 − p') : 0,     keep_i = (16 random bits of element i) ≥ 65536·p'
//
// with p' = round(65536 p) / 65536.  Element i takes half i % 8 of the four 32-bit words of
// Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter
// (i / 8, call number) under the 64-bit seed, so any kernel — the backward pass above all — makes
// the same mask from the two numbers of the key, whatever its grid.
//
// One generator call (10 rounds of two 32×32→64-bit products) covers the 8 elements of one 16-byte
// bf16 access: with 16 bits per element the arithmetic stays below the time the bytes take; with
// 32 bits it would not.  The price is the step of p', 2^-16.  A dropped element is an exact 0 also
// where x is NaN or infinite.
#include "common.h"
#include "kernels.h"

namespace tdl {
namespace {

struct u4v { uint32_t x, y, z, w; };

__device__ __forceinline__ u4v philox10(uint64_t block, uint64_t call, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)call, c3 = (uint32_t)(call >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return u4v{c0, c1, c2, c3};
}

// E elements of a group from element `first` on: their 16 bits are in E / 2 of its words
template <int E>
__device__ __forceinline__ void apply(float* f, const u4v& r, int first, uint32_t cut, float scale) {
  uint32_t w[4] = {r.x, r.y, r.z, r.w};
  if (E == 4 && first) {
    w[0] = w[2];
    w[1] = w[3];
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const uint32_t h = e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
    f[e] = h >= cut ? f[e] * scale : 0.f;
  }
}

// A thread's E elements are one 16-byte access: a whole group in bf16, half of one in fp32 (whose
// other half's thread makes the same numbers again; 8 bytes per element leave time for that, and
// 32-byte pieces per lane cost more: 22.6 M elements 41 us).
// VEC: both pointers are 16-byte aligned; else (a view that starts inside a vector) element by element
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(const T* __restrict__ x, T* __restrict__ y,
                                                      long n, const int64_t* __restrict__ key,
                                                      uint32_t cut, float scale) {
  constexpr int E = 16 / sizeof(T);
  const uint64_t seed = (uint64_t)key[0], call = (uint64_t)key[1];
  const long pieces = (n + E - 1) / E;
  for (long g = (long)blockIdx.x * 256 + threadIdx.x; g < pieces; g += (long)gridDim.x * 256) {
    const long i = g * E;
    const bool whole = i + E <= n;
    float f[E];
    if (VEC && whole) {
      if constexpr (E == 8) {
        load8(x + i, f);
      } else {
        const float4 v = *(const float4*)(x + i);
        f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = i + e < n ? load1(x + i + e) : 0.f;
    }
    apply<E>(f, philox10((uint64_t)(i / 8), call, seed), (int)(i % 8), cut, scale);
    if (VEC && whole) {
      if constexpr (E == 8) store8(y + i, f);
      else *(float4*)(y + i) = make_float4(f[0], f[1], f[2], f[3]);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < n) store1(y + i + e, f[e]);
    }
  }
}

// two calls on two streams draw different numbers: the call number is taken atomically
__global__ void dropout_next_key_kernel(int64_t* state, int64_t* out) {
  out[0] = state[0];
  out[1] = (int64_t)atomicAdd((unsigned long long*)(state + 1), 1ull);
}

}  // namespace

void dropout_launch(const void* x, void* y, long n, bool bf16, const int64_t* key, uint32_t cut,
                    float scale, hipStream_t st) {
  const long e = bf16 ? 8 : 4, blocks = ((n + e - 1) / e + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 256 * 16 ? blocks : 256 * 16);
  const bool vec = ((uintptr_t)x | (uintptr_t)y) % 16 == 0;
  if (bf16) {
    if (vec) dropout_kernel<bf16_t, true><<<grid, 256, 0, st>>>((const bf16_t*)x, (bf16_t*)y, n, key, cut, scale);
    else dropout_kernel<bf16_t, false><<<grid, 256, 0, st>>>((const bf16_t*)x, (bf16_t*)y, n, key, cut, scale);
  } else {
    if (vec) dropout_kernel<float, true><<<grid, 256, 0, st>>>((const float*)x, (float*)y, n, key, cut, scale);
    else dropout_kernel<float, false><<<grid, 256, 0, st>>>((const float*)x, (float*)y, n, key, cut, scale);
  }
}

void dropout_next_key_launch(int64_t* state, int64_t* out, hipStream_t st) {
  dropout_next_key_kernel<<<1, 1, 0, st>>>(state, out);
}

}  // namespace tdl
