// Launchers of the fp8 quantisers (fp8_quant.cuh), in a translation unit of their own.
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace b200dq {

enum : int { FP8_E4M3 = 0, FP8_E5M2 = 1 };
enum : int { FP8_IN_F16 = 0, FP8_IN_BF16 = 1, FP8_IN_F32 = 2 };
// What is quantised: the rows themselves, silu(gate) * up, or the gradient of that.
enum : int { FP8_OF_ROWS = 0, FP8_OF_SILU_MUL = 1, FP8_OF_SILU_MUL_GRAD = 2 };

struct Fp8QuantParams {
  const void* x;          // rows (M, K); or h = [gate | up], (M, 2 F)
  const void* d;          // SILU_MUL_GRAD: gradient of silu(gate) * up, (M, F); else null
  uint8_t* codes;         // (M, cols) bytes, row pitch ld_codes
  float* scales;          // (M, ceil(cols / 128)), contiguous
  long long ld_x, ld_d, ld_codes;   // row pitches in elements
  long long rows;
  int cols;               // columns of the result: K, F or 2 F
  int half;               // F (0 for plain rows)
  int in_type, out_type;
  bool vec;               // pointers and pitches allow the 16-elements-a-thread kernel
};

cudaError_t launch_fp8_quant(int mode, const Fp8QuantParams& p, cudaStream_t stream);

// 128 x 128 blocks of (batch, N, K) -> codes and (batch, ceil(N / 128), ceil(K / 128)) scales; codes have the row
// pitch ld_codes, the rest is contiguous.
cudaError_t launch_fp8_quant_blocks(const void* x, uint8_t* codes, float* scales, long long batch, int N, int K,
                                    long long ld_codes, int in_type, int out_type, cudaStream_t stream);

}  // namespace b200dq
