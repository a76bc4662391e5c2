// Launchers of the block-scaled fp8 products (fp8_gemm.cuh), in a translation unit of their own.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace b200dq {

struct DeviceStatus;

// C[m, p] = sum_b sa[m, b] sum_{q in block b} a[m, q] w(p, q) sw(p / 128, b), with w stored (P, Q), or (Q, P) when
// transposed. P: columns of the output, Q: contraction.
struct Fp8GemmParams {
  const float* a_scale;      // (M, q_blocks), row pitch ld_a_scale
  long long ld_a_scale;
  const float* w_scale;      // element (p block, q block) at p_block * ws_p + q_block * ws_q, + group * ws_group
  long long ws_p, ws_q, ws_group;
  void* c;                   // (M, P) row-major
  long long ldc;             // P
  int M, P, q_blocks;
  int p_tiles;
  int out_type;              // OUT_BF16, OUT_F16, OUT_F32
  int a_fmt, w_fmt;          // FP8_E4M3 / FP8_E5M2
  int trans_w;
  int c_vec;                 // four columns may be stored at once
  int c_vec16;               // 16 bytes may be stored at once
  const void* counts;        // grouped: rows of each group, on the device; null: one group of M rows
  int counts_int64, num_groups;
  // CTA pairs only
  int tile_cols;             // columns of C that a tile advances by: 256, gated 128
  uint8_t* gate_codes;       // gated: codes of silu(g) u, (M, P / 2), row pitch ld_gate; else null
  float* gate_scales;        // (M, P / 256), contiguous
  long long ld_gate;
  int gate_fp8;
  int split;                 // CTAs of a cluster that share a tile's contraction
  DeviceStatus* status;
};

constexpr int kFp8BoxBytes = 128;   // columns of every box: one swizzle atom
constexpr int kFp8BoxRows = 128;    // rows of a weight box, and of a token box whose tokens own lanes

// Tokens own the accumulator's 128 lanes (tokens_on_lanes) or its columns, `tile_tokens` (16, 32, 128) of them.
cudaError_t launch_fp8_tile_gemm(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const Fp8GemmParams& p,
                                 bool tokens_on_lanes, int tile_tokens, long long tiles, cudaStream_t stream);

// Clusters of `split` CTAs that the current device holds at once with this tile.
cudaError_t fp8_resident_clusters(int tile_tokens, int split, int* clusters);

// CTA pairs, 256 tokens x 256 columns (p.p_tiles counts tiles of p.tile_cols); `pairs` clusters of two. With
// gate_codes the columns of a tile are 128 of the gate's and 128 of the up half's, and c (bf16) may be null.
// tmap_c: C with boxes of 128 rows x 128 bytes and the 128-byte swizzle, used where p.c_vec16 is set.
cudaError_t launch_fp8_pair_gemm(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w, const CUtensorMap& tmap_c,
                                 const Fp8GemmParams& p, int pairs, cudaStream_t stream);
constexpr int kFp8PairMaxGroups = 256;

}  // namespace b200dq
