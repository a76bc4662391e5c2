// Token exchange of a mixture-of-experts layer: every (token, slot) pair becomes a row, rows are
// sorted by expert (equal ones in pair order), and come back as weighted sums; with gradients.
//
//   row_of[t, s]   = rows of smaller experts + pairs of the same expert before (t, s)
//   dispatch       : rows[row_of[t, s]] = x[t]                 gradient: dx[t] = sum_s drows[row_of[t, s]]
//   combine        : out[t] = sum_s w[t, s] y[row_of[t, s]]    gradient: dy[row_of[t, s]] = w[t, s] dout[t],
//                                                                        dw[t, s] = <dout[t], y[row_of[t, s]]>
//
// A pair whose expert id lies outside [0, num_experts) takes part in nothing: it sorts behind the
// last expert, its row holds zeros, row_of is -1 - row, and sums skip it.
//
// All of it walks tokens, not rows: a token is read once and written to its top_k rows (the row-wise
// gather reads it top_k times), and a sum has its terms in slot order, in fp32, rounded once. There
// are no floating-point atomics, so results do not depend on the order in which CTAs run. Counting
// uses integer atomics in shared memory, whose sum has no order.
//
// Bound: HBM for many tokens, launch latency for few.
#pragma once
#include <cstdint>

#include "exchange_launch.h"
#include "fp8_quant.cuh"

namespace b200dq {

__device__ __forceinline__ int expert_of(const ExchangeSortParams& p, long long pair) {
  const long long e = p.experts_int64 ? static_cast<const long long*>(p.experts)[pair]
                                      : static_cast<long long>(static_cast<const int*>(p.experts)[pair]);
  return e < 0 || e >= p.num_experts ? p.num_experts : static_cast<int>(e);
}

// Exclusive prefix of bins[0 .. n) in place, by one warp.
__device__ __forceinline__ void warp_exclusive_scan(int* bins, int n, int lane) {
  int before = 0;
  for (int base = 0; base < n; base += 32) {
    const int i = base + lane;
    const int own = i < n ? bins[i] : 0;
    int v = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, d);
      if (lane >= d) v += u;
    }
    if (i < n) bins[i] = before + v - own;
    before += __shfl_sync(0xffffffffu, v, 31);
  }
}

// Rows of the pairs [first, last) in pair order, by one warp: next[e] is the next free row of expert e.
__device__ __forceinline__ void warp_place(const ExchangeSortParams& p, long long first, long long last, int* next,
                                           int lane) {
  for (long long base = first; base < last; base += 128) {
    int ids[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = base + 32 * j + lane;
      ids[j] = i < last ? expert_of(p, i) : p.num_experts + 1;       // a bin of its own, never placed
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long long i = base + 32 * j + lane;
      const bool in = i < last;
      const int e = ids[j];
      const unsigned peers = __match_any_sync(0xffffffffu, e);
      const int rank = __popc(peers & ((1u << lane) - 1u));
      int row = 0;
      if (in) row = next[e] + rank;
      __syncwarp();
      if (in && rank == 0) next[e] += __popc(peers);
      __syncwarp();
      if (in) p.row_of[i] = e == p.num_experts ? -1ll - row : static_cast<long long>(row);
    }
  }
}

// ---- moving rows ---------------------------------------------------------------------------------

// Threads [0, threads) of a CTA move the rows of one token. `rows` holds its top_k row_of values.
__device__ __forceinline__ void copy_token(const ExchangeRowsParams& r, long long t, const long long* rows, int top_k,
                                           int tid, int threads) {
  const int size = r.type == EXCHANGE_F32 ? 4 : 2;
  const uint8_t* src = static_cast<const uint8_t*>(r.x) + t * r.ld_x * size;
  uint8_t* out = static_cast<uint8_t*>(r.out);
  const long long pitch = static_cast<long long>(r.width) * size;
  if (r.vec) {
    for (int i = tid; i < r.width * size / 16; i += threads) {
      const uint4 v = reinterpret_cast<const uint4*>(src)[i];
      for (int s = 0; s < top_k; ++s) {
        const long long row = rows[s];
        if (row >= 0) __stcs(reinterpret_cast<uint4*>(out + row * pitch) + i, v);
        else reinterpret_cast<uint4*>(out + (-1 - row) * pitch)[i] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  for (int i = tid; i < r.width; i += threads) {
    const uint32_t v = size == 4 ? reinterpret_cast<const uint32_t*>(src)[i] : reinterpret_cast<const uint16_t*>(src)[i];
    for (int s = 0; s < top_k; ++s) {
      const long long row = rows[s];
      const uint32_t o = row >= 0 ? v : 0u;
      uint8_t* dst = out + (row >= 0 ? row : -1 - row) * pitch;
      if (size == 4) reinterpret_cast<uint32_t*>(dst)[i] = o;
      else reinterpret_cast<uint16_t*>(dst)[i] = static_cast<uint16_t>(o);
    }
  }
}

// The same with the token quantised on its way: once, however many rows it goes to. Zero rows get
// scale 2^-126, what the quantiser gives a block of zeros. All threads of the CTA call it together.
template <typename T, int OUT>
__device__ __forceinline__ void quant_token(const ExchangeRowsParams& r, long long t, const long long* rows, int top_k,
                                            int tid, int threads) {
  const T* src = static_cast<const T*>(r.x) + t * r.ld_x;
  const int blocks = (r.width + 127) / 128;
  uint8_t* out = static_cast<uint8_t*>(r.out);
  if (r.vec) {
    for (int base = 0; base < blocks * 8; base += threads) {           // threads is a multiple of 32: whole warps
      const int part = base + tid;
      const int c = part * 16;
      const bool active = c < r.width;
      float v[16], s;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
      if (active) load16(src + c, v);
      const uint4 codes = quant16<OUT>(v, &s);
      if (!active) continue;
      for (int k = 0; k < top_k; ++k) {
        const bool kept = rows[k] >= 0;
        const long long row = kept ? rows[k] : -1 - rows[k];
        *reinterpret_cast<uint4*>(out + row * r.ld_out + c) = kept ? codes : make_uint4(0, 0, 0, 0);
        if ((part & 7) == 0) r.scales[row * blocks + part / 8] = kept ? s : 1.17549435e-38f;
      }
    }
    return;
  }
  const int lane = tid & 31;
  for (int b = tid >> 5; b < blocks; b += threads >> 5) {
    float v[4];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = b * 128 + i * 32 + lane;
      v[i] = c < r.width ? Fp8In<T>::get(src[c]) : 0.f;
      m = max(m, magnitude_bits(v[i]));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    const float s = fp8_scale_of<OUT>(m);
    const float inv = __frcp_rn(s);
    for (int k = 0; k < top_k; ++k) {
      const bool kept = rows[k] >= 0;
      const long long row = kept ? rows[k] : -1 - rows[k];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = b * 128 + i * 32 + lane;
        if (c < r.width)
          out[row * r.ld_out + c] = kept ? static_cast<uint8_t>(fp8_pair<OUT>(__fmul_rn(v[i], inv), 0.f)) : uint8_t(0);
      }
      if (lane == 0) r.scales[row * blocks + b] = kept ? s : 1.17549435e-38f;
    }
  }
}

// How a kernel moves a token: MOVE_COPY, or quantise from one of the input types.
template <typename T, int OUT> struct QuantMove {
  static __device__ __forceinline__ void run(const ExchangeRowsParams& r, long long t, const long long* rows, int k) {
    quant_token<T, OUT>(r, t, rows, k, threadIdx.x, blockDim.x);
  }
};
struct CopyMove {
  static __device__ __forceinline__ void run(const ExchangeRowsParams& r, long long t, const long long* rows, int k) {
    copy_token(r, t, rows, k, threadIdx.x, blockDim.x);
  }
};

// ---- few pairs: everything in one launch -----------------------------------------------------------
// CTA b owns tokens [b * per, (b + 1) * per). It counts all pairs, and those before its own, in shared
// memory (at most 4096 ids from L2: about 16 loads a thread), so no CTA waits for another.
template <typename MOVE>
__global__ void __launch_bounds__(256) exchange_dispatch_small_kernel(const ExchangeSortParams p,
                                                                      const ExchangeRowsParams r, int per) {
  chain_next();
  chain_wait();
  extern __shared__ int exchange_smem[];
  int* all = exchange_smem;                       // [E + 1] pairs of each expert, then their first rows
  int* next = exchange_smem + p.num_experts + 1;  // [E + 1] those before this CTA's pairs, then the next free row
  const int bins = p.num_experts + 1;
  const long long pairs = p.tokens * p.top_k;
  const long long t0 = static_cast<long long>(blockIdx.x) * per;
  const long long t1 = min(p.tokens, t0 + per);
  for (int i = threadIdx.x; i < 2 * bins; i += 256) exchange_smem[i] = 0;
  __syncthreads();
  for (long long i = threadIdx.x; i < pairs; i += 256) {
    const int e = expert_of(p, i);
    atomicAdd(&all[e], 1);
    if (i < t0 * p.top_k) atomicAdd(&next[e], 1);
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e < p.num_experts; e += 256) p.counts[e] = all[e];
  __syncthreads();
  if (threadIdx.x < 32) warp_exclusive_scan(all, bins, threadIdx.x);
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += 256) next[e] += all[e];
  __syncthreads();
  if (threadIdx.x < 32) warp_place(p, t0 * p.top_k, t1 * p.top_k, next, threadIdx.x);
  __syncthreads();                                // row_of of this CTA's pairs, written by its first warp
  for (long long t = t0; t < t1; ++t) MOVE::run(r, t, p.row_of + t * p.top_k, p.top_k);
}

// ---- many pairs: count, place, move ---------------------------------------------------------------
__global__ void __launch_bounds__(256) exchange_count_kernel(const ExchangeSortParams p, long long per) {
  chain_next();
  chain_wait();
  extern __shared__ int exchange_smem[];
  const int bins = p.num_experts + 1;
  const long long first = blockIdx.x * per, last = min(p.tokens * p.top_k, first + per);
  for (int i = threadIdx.x; i < bins; i += 256) exchange_smem[i] = 0;
  __syncthreads();
  for (long long i = first + threadIdx.x; i < last; i += 256) atomicAdd(&exchange_smem[expert_of(p, i)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += 256) p.scratch[blockIdx.x * bins + i] = exchange_smem[i];
}

// A chunk's CTA adds up the counts of all chunks and of those before it (at most 128 rows from L2),
// cuts its chunk into one piece per warp, counts the pieces and lets every warp place its own.
constexpr int kPlaceWarps = 8;
__global__ void __launch_bounds__(kPlaceWarps * 32) exchange_place_kernel(const ExchangeSortParams p, long long per) {
  chain_next();
  chain_wait();
  extern __shared__ int exchange_smem[];
  const int bins = p.num_experts + 1;
  int* all = exchange_smem;                // [bins]
  int* before = exchange_smem + bins;      // [bins]
  int* next = exchange_smem + 2 * bins;    // [warps][bins]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long first = blockIdx.x * per, last = min(p.tokens * p.top_k, first + per);
  const long long piece = ((per + kPlaceWarps - 1) / kPlaceWarps + 31) / 32 * 32;
  const long long w0 = min(last, first + warp * piece), w1 = min(last, w0 + piece);
  for (int i = threadIdx.x; i < (kPlaceWarps + 2) * bins; i += kPlaceWarps * 32) exchange_smem[i] = 0;
  __syncthreads();
  for (long long i = w0 + lane; i < w1; i += 32) atomicAdd(&next[warp * bins + expert_of(p, i)], 1);
  // a warp adds up every eighth chunk's counts, its lanes neighbouring experts
  for (int e = lane; e < bins; e += 32) {
    int total = 0, below = 0;
#pragma unroll
    for (int j = 0; j < kExchangeMaxChunks / kPlaceWarps; ++j) {
      const int c = warp + j * kPlaceWarps;
      const int n = c < static_cast<int>(gridDim.x) ? p.scratch[c * bins + e] : 0;
      total += n;
      if (c < static_cast<int>(blockIdx.x)) below += n;
    }
    atomicAdd(&all[e], total);
    atomicAdd(&before[e], below);
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = threadIdx.x; e < p.num_experts; e += kPlaceWarps * 32) p.counts[e] = all[e];
  __syncthreads();                         // the scan turns the counts into first rows
  if (warp == 0) warp_exclusive_scan(all, bins, lane);
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += kPlaceWarps * 32) {
    int at = all[e] + before[e];
    for (int w = 0; w < kPlaceWarps; ++w) {
      const int n = next[w * bins + e];
      next[w * bins + e] = at;
      at += n;
    }
  }
  __syncthreads();
  warp_place(p, w0, w1, next + warp * bins, lane);
}

template <typename MOVE>
__global__ void __launch_bounds__(256) exchange_move_kernel(const ExchangeSortParams p, const ExchangeRowsParams r) {
  chain_next();
  chain_wait();
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) MOVE::run(r, t, p.row_of + t * p.top_k, p.top_k);
}

// ---- back, and the gradients ----------------------------------------------------------------------

template <typename T> __device__ __forceinline__ T exchange_round(float v);
template <> __device__ __forceinline__ __half exchange_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 exchange_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ float exchange_round<float>(float v) { return v; }

// out[t] = sum_s w[t, s] y[row_of[t, s]] (w null: one): a CTA takes a token, a thread 16 bytes of the row;
// the terms' loads are started four at a time (eight take the registers that keep other warps
// resident: 128 against 86 us for 16384 x 6 rows of 2048). Rows pass through the caches once and are marked so
// (78 us).
template <typename T>
__global__ void __launch_bounds__(256) exchange_sum_kernel(const ExchangeSumParams p) {
  chain_next();
  chain_wait();
  constexpr int V = 16 / sizeof(T);
  const T* y = static_cast<const T*>(p.y);
  const long long all_rows = p.tokens * p.top_k;          // indices outside add nothing and are not followed
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const long long* rows = p.row_of + t * p.top_k;
    const float* w = p.weights != nullptr ? p.weights + t * p.top_k : nullptr;
    T* out = static_cast<T*>(p.out) + t * p.width;
    if (p.vec) {
      for (int c = threadIdx.x; c < p.width / V; c += blockDim.x) {
        float acc[V];
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.f;
        for (int s0 = 0; s0 < p.top_k; s0 += 4) {
          uint4 v[4];
          float f[4];
          bool kept[4];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const long long row = s0 + s < p.top_k ? rows[s0 + s] : -1;
            kept[s] = row >= 0 && row < all_rows;
            f[s] = kept[s] && w != nullptr ? w[s0 + s] : 1.f;
            if (kept[s]) v[s] = __ldcs(reinterpret_cast<const uint4*>(y + row * p.width) + c);
          }
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            if (!kept[s]) continue;
            const T* e = reinterpret_cast<const T*>(&v[s]);
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j] = fmaf(f[s], Fp8In<T>::get(e[j]), acc[j]);
          }
        }
        uint4 o;
        T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int j = 0; j < V; ++j) oe[j] = exchange_round<T>(acc[j]);
        __stcs(reinterpret_cast<uint4*>(out) + c, o);
      }
    } else {
      for (int c = threadIdx.x; c < p.width; c += blockDim.x) {
        float acc = 0.f;
        for (int s = 0; s < p.top_k; ++s)
          if (rows[s] >= 0 && rows[s] < all_rows)
            acc = fmaf(w != nullptr ? w[s] : 1.f, Fp8In<T>::get(y[rows[s] * p.width + c]), acc);
        out[c] = exchange_round<T>(acc);
      }
    }
  }
}

// dy[row_of[t, s]] = w[t, s] dout[t] and dw[t, s] = <dout[t], y[row_of[t, s]]>: a warp takes a pair, the
// warps of a CTA neighbouring pairs, so that a token's dout is read from memory once and from L1 after
// that. No barrier: lanes' partial dot products are added by shuffles (a CTA per token, its
// threads across the row and two barriers for every four slots, took 205 us for 16384 x 6 rows of 2048, this
// takes 133: the copy bandwidth).
template <typename T>
__global__ void __launch_bounds__(256) exchange_sum_grad_kernel(const ExchangeSumGradParams p) {
  chain_next();
  chain_wait();
  constexpr int V = 16 / sizeof(T);
  constexpr int kUnroll = 4;
  const int lane = threadIdx.x & 31;
  const long long pairs = p.tokens * p.top_k;
  for (long long i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < pairs; i += gridDim.x * 8ll) {
    const long long row = p.row_of[i];
    const bool kept = row >= 0 && row < pairs;
    const long long at = row >= 0 ? row : -1 - row;
    const float w = kept ? p.weights[i] : 0.f;
    const T* d = static_cast<const T*>(p.d_out) + i / p.top_k * p.width;
    const T* y = p.d_weights != nullptr && kept ? static_cast<const T*>(p.y) + row * p.width : nullptr;
    T* d_y = p.d_y != nullptr && at < pairs ? static_cast<T*>(p.d_y) + at * p.width : nullptr;
    float dot = 0.f;
    if (p.vec) {
      const int vecs = p.width / V;
      for (int c0 = lane; c0 < vecs; c0 += 32 * kUnroll) {
        uint4 dv[kUnroll], yv[kUnroll];
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
          const int c = c0 + 32 * j;
          dv[j] = kept && c < vecs ? reinterpret_cast<const uint4*>(d)[c] : make_uint4(0, 0, 0, 0);
          yv[j] = y != nullptr && c < vecs ? reinterpret_cast<const uint4*>(y)[c] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < kUnroll; ++j) {
          const int c = c0 + 32 * j;
          if (c >= vecs) continue;
          const T* de = reinterpret_cast<const T*>(&dv[j]);
          const T* ye = reinterpret_cast<const T*>(&yv[j]);
          uint4 o;
          T* oe = reinterpret_cast<T*>(&o);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float dd = Fp8In<T>::get(de[e]);
            if (y != nullptr) dot = fmaf(dd, Fp8In<T>::get(ye[e]), dot);
            oe[e] = exchange_round<T>(kept ? w * dd : 0.f);
          }
          if (d_y != nullptr) reinterpret_cast<uint4*>(d_y)[c] = o;
        }
      }
    } else {
      for (int c = lane; c < p.width; c += 32) {
        const float dd = kept ? Fp8In<T>::get(d[c]) : 0.f;
        if (y != nullptr) dot = fmaf(dd, Fp8In<T>::get(y[c]), dot);
        if (d_y != nullptr) d_y[c] = exchange_round<T>(kept ? w * dd : 0.f);
      }
    }
    if (p.d_weights == nullptr) continue;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (lane == 0) p.d_weights[i] = dot;                              // a dropped pair's dot is zero
  }
}

}  // namespace b200dq
