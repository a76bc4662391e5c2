// Quantisers to 8-bit floating point with one fp32 scale for each block of 128 (rows: 1 x 128,
// weights: 128 x 128).
//
//   scale = max |x| over the block / largest finite code (448 for e4m3, 57344 for e5m2), at least
//           2^-126 so that its reciprocal is finite; code = rn(x * (1 / scale)), ties to even.
//
// The maximum is NaN where any value is (bit patterns of magnitudes order like the magnitudes, NaN above
// infinity; max.NaN does the same on values): a block that holds a NaN gets the scale NaN, one that holds an infinity the
// scale infinity, so neither turns into a finite number on its way through a product. All
// arithmetic is fp32; the one rounding to 8 bits is the result. Products are not left to contraction into
// fmas, so that codes do not depend on which kernel computed them.
//
// Bound: HBM, one read of the input and one byte written per element. The silu forms read gate and
// up once and never write the 16-bit activation (or its gradient) that would otherwise go out and
// come back.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "chain_launch.cuh"
#include "fp8_quant_launch.h"

namespace b200dq {

template <typename T> struct Fp8In;
template <> struct Fp8In<__half> {
  static __device__ __forceinline__ float get(const __half v) { return __half2float(v); }
};
template <> struct Fp8In<__nv_bfloat16> {
  static __device__ __forceinline__ float get(const __nv_bfloat16 v) { return __bfloat162float(v); }
};
template <> struct Fp8In<float> {
  static __device__ __forceinline__ float get(const float v) { return v; }
};

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// max(m, |v|), NaN if either is: one instruction, where the bit patterns take two
__device__ __forceinline__ float max_magnitude(float m, float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
  return r;
}

template <int OUT>
__device__ __forceinline__ float fp8_scale_of(uint32_t amax_bits) {
  const float s = __fmul_rn(__uint_as_float(amax_bits), OUT == FP8_E4M3 ? 1.0f / 448.0f : 1.0f / 57344.0f);
  return s < 1.17549435e-38f ? 1.17549435e-38f : s;      // a comparison with NaN is false: NaN stays
}

// Two codes, `lo` in the low byte. satfinite: rounding of 1 / scale may carry the largest value past 448.
template <int OUT>
__device__ __forceinline__ uint32_t fp8_pair(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, OUT == FP8_E4M3 ? __NV_E4M3 : __NV_E5M2);
}

// 1 / (1 + e^-g) from the hardware's base-2 exponential and reciprocal, a relative error of at most
// |g| 2^-24 + 2^-21 (the rounded exponent, then 2 and 1 units in the last place): far below the codes' half
// step. Below g = -87.3, where it would be less than 2^-126, the result is 0. (The library's expf and an IEEE division made
// the gradient's quantiser bound by instructions: 72 us for 24576 x 1408, of which the bytes need 42.)
__device__ __forceinline__ float sigmoid_of(float g) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-1.4426950408889634f * g));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}
__device__ __forceinline__ float silu_mul_of(float g, float u) { return __fmul_rn(__fmul_rn(g, sigmoid_of(g)), u); }
// d/dg and d/du of silu(g) u, times the incoming d: with p = sigmoid(g), d u p (1 + g (1 - p)) and d g p.
__device__ __forceinline__ void silu_mul_grad(float g, float u, float d, float* dgate, float* dup) {
  const float p = sigmoid_of(g);
  *dgate = __fmul_rn(__fmul_rn(d, u), __fmul_rn(p, __fmaf_rn(g, __fadd_rn(1.0f, -p), 1.0f)));
  *dup = __fmul_rn(d, __fmul_rn(g, p));
}

template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]) {
  constexpr int kPerVec = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 16 / kPerVec; ++i) {
    const uint4 raw = reinterpret_cast<const uint4*>(p)[i];
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int j = 0; j < kPerVec; ++j) v[i * kPerVec + j] = Fp8In<T>::get(e[j]);
  }
}

// The eight lanes of a block of 128 agree on its maximum, then write 16 codes each.
template <int OUT>
__device__ __forceinline__ uint4 quant16(const float (&v)[16], float* scale) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max_magnitude(m, v[i]);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max_magnitude(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float s = fp8_scale_of<OUT>(__float_as_uint(m));
  const float inv = __frcp_rn(s);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = fp8_pair<OUT>(__fmul_rn(v[4 * i], inv), __fmul_rn(v[4 * i + 1], inv)) |
           (fp8_pair<OUT>(__fmul_rn(v[4 * i + 2], inv), __fmul_rn(v[4 * i + 3], inv)) << 16);
  *scale = s;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 columns a thread, eight threads a block of 128: two 16-byte loads in flight per thread for
// 16-bit inputs and one 16-byte store. Needs columns (and half) to be multiples of 16, for the
// gradient half a multiple of 128, and 16-byte aligned rows; the other kernel takes the rest.
template <typename T, int OUT, int MODE>
__global__ void __launch_bounds__(256) fp8_quant_vec_kernel(const Fp8QuantParams p) {
  chain_next();
  chain_wait();
  const int cols = MODE == FP8_OF_SILU_MUL_GRAD ? p.half : p.cols;
  const unsigned blocks = (cols + 127) / 128;            // blocks of a row (of one half of it for the gradient)
  const long long idx = blockIdx.x * 256ll + threadIdx.x;
  const long long total = p.rows * blocks * 8;
  const bool in_range = idx < total;
  const long long row = in_range ? idx / (blocks * 8) : 0;
  const int part = in_range ? static_cast<int>(idx - row * (blocks * 8)) : 0;
  const int c = part * 16;
  const bool active = in_range && c < cols;
  const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
  const int all_blocks = (p.cols + 127) / 128;
  float v[16], w[16], s;
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = w[i] = 0.f;
  if (active) {
    if (MODE == FP8_OF_ROWS) {
      load16(x + c, v);
    } else {
      float g[16], u[16], d[16];
      load16(x + c, g);
      load16(x + p.half + c, u);
      if (MODE == FP8_OF_SILU_MUL_GRAD) load16(static_cast<const T*>(p.d) + row * p.ld_d + c, d);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (MODE == FP8_OF_SILU_MUL) {
          v[i] = silu_mul_of(g[i], u[i]);
        } else {
          silu_mul_grad(g[i], u[i], d[i], &v[i], &w[i]);
        }
      }
    }
  }
  // whole warps meet here: the shuffles of quant16 see every lane
  uint4 codes = quant16<OUT>(v, &s);
  if (active) {
    *reinterpret_cast<uint4*>(p.codes + row * p.ld_codes + c) = codes;
    if ((part & 7) == 0) p.scales[row * all_blocks + part / 8] = s;
  }
  if (MODE == FP8_OF_SILU_MUL_GRAD) {
    // half is a multiple of 128 here: the up half's blocks start where a block of the row starts
    codes = quant16<OUT>(w, &s);
    if (active) {
      *reinterpret_cast<uint4*>(p.codes + row * p.ld_codes + p.half + c) = codes;
      if ((part & 7) == 0) p.scales[row * all_blocks + blocks + part / 8] = s;
    }
  }
}

// One element of what is quantised, for the kernel without alignment rules.
template <typename T, int MODE>
__device__ __forceinline__ float fp8_source(const Fp8QuantParams& p, long long row, int c) {
  const T* x = static_cast<const T*>(p.x) + row * p.ld_x;
  if (MODE == FP8_OF_ROWS) return Fp8In<T>::get(x[c]);
  if (MODE == FP8_OF_SILU_MUL) return silu_mul_of(Fp8In<T>::get(x[c]), Fp8In<T>::get(x[p.half + c]));
  const bool gate = c < p.half;
  const int i = gate ? c : c - p.half;
  float dgate, dup;
  silu_mul_grad(Fp8In<T>::get(x[i]), Fp8In<T>::get(x[p.half + i]), Fp8In<T>::get(static_cast<const T*>(p.d)[row * p.ld_d + i]),
                &dgate, &dup);
  return gate ? dgate : dup;
}

// Any width, pitch and alignment: a warp takes a block of 128, a lane four columns 32 apart, so
// that loads and byte stores of a warp are contiguous.
template <typename T, int OUT, int MODE>
__global__ void __launch_bounds__(256) fp8_quant_any_kernel(const Fp8QuantParams p) {
  chain_next();
  chain_wait();
  const int lane = threadIdx.x & 31;
  const int blocks = (p.cols + 127) / 128;
  const long long idx = blockIdx.x * 8ll + (threadIdx.x >> 5);
  if (idx >= p.rows * blocks) return;
  const long long row = idx / blocks;
  const int b = static_cast<int>(idx - row * blocks);
  float v[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = b * 128 + i * 32 + lane;
    v[i] = c < p.cols ? fp8_source<T, MODE>(p, row, c) : 0.f;
    m = max(m, magnitude_bits(v[i]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  const float s = fp8_scale_of<OUT>(m);
  const float inv = __frcp_rn(s);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = b * 128 + i * 32 + lane;
    if (c < p.cols) p.codes[row * p.ld_codes + c] = static_cast<uint8_t>(fp8_pair<OUT>(__fmul_rn(v[i], inv), 0.f));
  }
  if (lane == 0) p.scales[idx] = s;
}

// A CTA of eight warps takes a block of 128 x 128: a warp 16 rows, a lane four columns 32 apart. The
// block is read twice, the second time from L1 / L2 (weights are quantised once, at load).
template <typename T, int OUT>
__global__ void __launch_bounds__(256) fp8_quant_blocks_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                               float* __restrict__ scales, int N, int K,
                                                               long long ld_codes) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kb = blockIdx.x, nb = blockIdx.y;
  const long long batch = blockIdx.z;
  const size_t base = static_cast<size_t>(batch) * N * K;
  uint32_t m = 0;
  for (int r = nb * 128 + warp; r < min(N, nb * 128 + 128); r += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = kb * 128 + i * 32 + lane;
      if (c < K) m = max(m, magnitude_bits(Fp8In<T>::get(x[base + static_cast<size_t>(r) * K + c])));
    }
  m = __reduce_max_sync(0xffffffffu, m);
  __shared__ uint32_t warp_max[8];
  if (lane == 0) warp_max[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = max(m, warp_max[w]);
  const float s = fp8_scale_of<OUT>(m);
  const float inv = __frcp_rn(s);
  for (int r = nb * 128 + warp; r < min(N, nb * 128 + 128); r += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = kb * 128 + i * 32 + lane;
      if (c < K)
        codes[(batch * N + r) * ld_codes + c] = static_cast<uint8_t>(
            fp8_pair<OUT>(__fmul_rn(Fp8In<T>::get(x[base + static_cast<size_t>(r) * K + c]), inv), 0.f));
    }
  if (threadIdx.x == 0) scales[(batch * gridDim.y + nb) * gridDim.x + kb] = s;
}

}  // namespace b200dq
