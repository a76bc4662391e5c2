// Host side of the fp8 quantisers.
#include "fp8_quant_launch.h"

#include "fp8_quant.cuh"

namespace b200dq {

namespace {

template <typename T, int OUT, int MODE>
cudaError_t launch(const Fp8QuantParams& p, cudaStream_t stream) {
  const long long row_blocks = ((MODE == FP8_OF_SILU_MUL_GRAD && p.vec ? p.half : p.cols) + 127) / 128;
  const long long grid = p.vec ? (p.rows * row_blocks * 8 + 255) / 256 : (p.rows * row_blocks + 7) / 8;
  if (grid > 0x7fffffffll) return cudaErrorInvalidValue;
  return chain_launch(p.vec ? fp8_quant_vec_kernel<T, OUT, MODE> : fp8_quant_any_kernel<T, OUT, MODE>,
                      static_cast<unsigned>(grid), 256, 0, stream, 0, p);
}

template <typename T, int OUT>
cudaError_t launch_mode(int mode, const Fp8QuantParams& p, cudaStream_t stream) {
  if (mode == FP8_OF_ROWS) return launch<T, OUT, FP8_OF_ROWS>(p, stream);
  if (mode == FP8_OF_SILU_MUL) return launch<T, OUT, FP8_OF_SILU_MUL>(p, stream);
  return launch<T, OUT, FP8_OF_SILU_MUL_GRAD>(p, stream);
}

template <typename T>
cudaError_t launch_out(int mode, const Fp8QuantParams& p, cudaStream_t stream) {
  return p.out_type == FP8_E4M3 ? launch_mode<T, FP8_E4M3>(mode, p, stream) : launch_mode<T, FP8_E5M2>(mode, p, stream);
}

template <typename T>
cudaError_t launch_blocks(const void* x, uint8_t* codes, float* scales, long long batch, int N, int K,
                          long long ld_codes, int out_type, cudaStream_t stream) {
  const dim3 grid((K + 127) / 128, (N + 127) / 128, static_cast<unsigned>(batch));
  if (out_type == FP8_E4M3)
    fp8_quant_blocks_kernel<T, FP8_E4M3><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), codes, scales, N, K, ld_codes);
  else
    fp8_quant_blocks_kernel<T, FP8_E5M2><<<grid, 256, 0, stream>>>(static_cast<const T*>(x), codes, scales, N, K, ld_codes);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_fp8_quant(int mode, const Fp8QuantParams& p, cudaStream_t stream) {
  if (p.in_type == FP8_IN_F16) return launch_out<__half>(mode, p, stream);
  if (p.in_type == FP8_IN_BF16) return launch_out<__nv_bfloat16>(mode, p, stream);
  return launch_out<float>(mode, p, stream);
}

cudaError_t launch_fp8_quant_blocks(const void* x, uint8_t* codes, float* scales, long long batch, int N, int K,
                                    long long ld_codes, int in_type, int out_type, cudaStream_t stream) {
  if (in_type == FP8_IN_F16) return launch_blocks<__half>(x, codes, scales, batch, N, K, ld_codes, out_type, stream);
  if (in_type == FP8_IN_BF16) return launch_blocks<__nv_bfloat16>(x, codes, scales, batch, N, K, ld_codes, out_type, stream);
  return launch_blocks<float>(x, codes, scales, batch, N, K, ld_codes, out_type, stream);
}

}  // namespace b200dq
