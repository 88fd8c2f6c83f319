// 8-bit linear layer (int8.hip).  Operands of the product are kept in the order the matrix unit
// takes them: a block is 16 rows × 64 bytes of k as [4 chunks of 16 k][16 rows][16 bytes], 1 KiB,
// and a matrix is [rows / 16][Kp / 64] blocks, zero-padded to whole blocks and to Kp = a multiple
// of 128.  One wave load, one LDS-DMA and one fragment read are each 64 consecutive 16-byte pieces.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tdl {

constexpr int INT8_MAX_K = 131071;  // K·127·128 stays below 2^31

inline long int8_kp(long K) { return (K + 127) / 128 * 128; }
inline long int8_rows(long M) { return (M + 15) / 16 * 16; }

// rows of x (bf16 / fp32, row stride ld) -> q in block order + scale[M] = max|x| / 127
void int8_quantize_launch(const void* x, long ld, bool bf16, long M, long K, int8_t* q,
                          float* scale, hipStream_t st);

struct Int8GemmArgs {
  const int8_t* q;      // activations, blocks
  const float* qs;      // [M]
  const int8_t* w;      // weights, blocks
  const float* ws;      // [N]
  const float* bias;    // [N] or null
  const void* res;      // [M][N] of y's type, or null
  void* y;              // [M][N]
  long M;
  int N, Kp;
  bool relu;
};
// quantise x's rows and multiply; q / qs: room for the blocks and scales, not touched when the
// rows are few enough to be quantised where they are used (int8_linear_fused)
bool int8_linear_fused(long M, long N, long Kp, bool bf16);
void int8_linear_launch(const void* x, long ld, long K, const Int8GemmArgs& a, int8_t* q, float* qs,
                        bool bf16, hipStream_t st);
void int8_gemm_launch(const Int8GemmArgs& a, bool bf16, hipStream_t st);

}  // namespace tdl
