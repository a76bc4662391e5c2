// Launchers of the token exchange of a mixture-of-experts layer (exchange.cuh).
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace b200dq {

enum : int { EXCHANGE_F16 = 0, EXCHANGE_BF16 = 1, EXCHANGE_F32 = 2 };

constexpr int kExchangeMaxExperts = 1024;
constexpr int kExchangeMaxWidth = 1 << 28;       // bytes of a row are counted in 32 bits
// Up to this many (token, slot) pairs every CTA counts all of them itself and sorting, copying and
// quantising are one launch; above it two launches count and place, a third one moves the rows.
constexpr int kExchangeOneLaunchPairs = 4096;
constexpr int kExchangeMaxChunks = 128;      // chunks of the counting launch: one row of the scratch each

struct ExchangeSortParams {
  const void* experts;      // (tokens, top_k) int32 or int64, contiguous
  int experts_int64;
  long long tokens;
  int top_k, num_experts;
  long long* row_of;        // (tokens, top_k)
  long long* counts;        // (num_experts)
  int* scratch;             // kExchangeMaxChunks x (num_experts + 1) ints, more than kExchangeOneLaunchPairs pairs only
};

struct ExchangeRowsParams {
  const void* x;            // (tokens, width) rows, pitch ld_x elements
  long long ld_x;
  int width, type;          // type: EXCHANGE_*
  void* out;                // (tokens * top_k, width) rows of the same type, contiguous; or codes, pitch ld_out
  long long ld_out;
  float* scales;            // quantising: (tokens * top_k, ceil(width / 128)); null: rows are copied
  int fp8_type;
  bool vec;                 // 16-byte accesses are allowed
};

struct ExchangeSumParams {
  const void* y;            // (tokens * top_k, width)
  const long long* row_of;
  const float* weights;     // (tokens, top_k) or null (all one)
  void* out;                // (tokens, width)
  long long tokens;
  int top_k, width, type;
  bool vec;
};

struct ExchangeSumGradParams {
  const void* d_out;        // (tokens, width)
  const void* y;            // (tokens * top_k, width)
  const long long* row_of;
  const float* weights;     // (tokens, top_k)
  void* d_y;                // (tokens * top_k, width) or null
  float* d_weights;         // (tokens, top_k) or null
  long long tokens;
  int top_k, width, type;
  bool vec;
};

cudaError_t launch_exchange_dispatch(const ExchangeSortParams& s, const ExchangeRowsParams& r, cudaStream_t stream);
cudaError_t launch_exchange_sum(const ExchangeSumParams& p, cudaStream_t stream);
cudaError_t launch_exchange_sum_grad(const ExchangeSumGradParams& p, cudaStream_t stream);

}  // namespace b200dq
