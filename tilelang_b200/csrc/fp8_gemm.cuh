// Products of 8-bit floats with one fp32 scale per block of 128 along the contraction:
//
//   C[m, p] = sum_b sa[m, b] * sw[p / 128, b] * ( sum_{q in block b} a[m, q] * w(p, q) )
//
// The inner sums run on the tensor cores (tcgen05.mma kind::f8f6f4, exact products, fp32 sums); the
// scales differ from block to block, so every block of 128 gets an accumulator of its own in tensor
// memory, and warps that read it back add it, scaled, to fp32 sums in registers. That costs one
// fma per element and block on the fp32 pipe (128 lanes) against 128 multiply-adds on the tensor
// pipe (8192 a cycle): half the tensor time, hidden behind it by several accumulators and packed fmas.
//
// Weights are stored (P, Q), along the contraction, or for the gradient of the input (Q, P): the
// same bytes, read through the other operand layout of the instruction, so no transposed copy.
// Grouped (mixture of experts): rows of `a` are sorted by group, the rows of each group counted on
// the device; every CTA finds its own tile from the counts, so nothing is planned on the host.
#pragma once
#include "chain_launch.cuh"
#include "fp8_launch.h"
#include "fp8_ptx.cuh"
#include "umma_gemm.cuh"   // OutType, packed-float bit casts

namespace b200dq {

struct Fp8Tile {
  int group, m0, m_end, p0;     // rows [m0, m_end) of a and C (at most one tile of them), columns from p0
};

// Tile `t` of the grouped (or dense) problem, p tiles fastest; false behind the last one. One warp.
template <int TOKENS>
__device__ __forceinline__ bool fp8_find_tile(const Fp8GemmParams& p, long long t, int lane, Fp8Tile* out) {
  const long long token_tile = t / p.p_tiles;
  const int p0 = static_cast<int>(t - token_tile * p.p_tiles) * 128;
  if (p.counts == nullptr) {
    const long long m0 = token_tile * TOKENS;
    *out = Fp8Tile{0, static_cast<int>(m0), p.M, p0};
    return m0 < p.M;
  }
  long long rows = 0, tiles = 0;
  for (int base = 0; base < p.num_groups; base += 32) {
    const int g = base + lane;
    long long c = 0;
    if (g < p.num_groups)
      c = p.counts_int64 ? static_cast<const long long*>(p.counts)[g] : static_cast<const int*>(p.counts)[g];
    c = min(max(c, 0ll), static_cast<long long>(p.M));        // wrong counts read and write no other row than a's
    long long r = c, n = (c + TOKENS - 1) / TOKENS;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long ru = __shfl_up_sync(0xffffffffu, r, d), nu = __shfl_up_sync(0xffffffffu, n, d);
      if (lane >= d) { r += ru; n += nu; }
    }
    const unsigned here = __ballot_sync(0xffffffffu, tiles + n > token_tile);
    if (here != 0) {
      const int src = __ffs(here) - 1;
      const long long r_end = rows + __shfl_sync(0xffffffffu, r, src), cnt = __shfl_sync(0xffffffffu, c, src);
      const long long n_end = tiles + __shfl_sync(0xffffffffu, n, src), own = (cnt + TOKENS - 1) / TOKENS;
      const long long m0 = r_end - cnt + (token_tile - (n_end - own)) * TOKENS;
      const long long m_end = min(r_end, static_cast<long long>(p.M));
      *out = Fp8Tile{base + src, static_cast<int>(min(m0, static_cast<long long>(p.M))), static_cast<int>(m_end), p0};
      return m0 < m_end;
    }
    rows += __shfl_sync(0xffffffffu, r, 31);
    tiles += __shfl_sync(0xffffffffu, n, 31);
  }
  return false;
}

// Four neighbouring columns of one row of C, rounded once to the output type.
__device__ __forceinline__ void fp8_store4(const Fp8GemmParams& p, long long m, int col, float4 v) {
  const size_t at = static_cast<size_t>(m) * p.ldc + col;
  if (p.c_vec) {                                        // P % 4 == 0 and an aligned base: col is a multiple of 4
    if (col >= p.P) return;
    if (p.out_type == OUT_F32) {
      *reinterpret_cast<float4*>(static_cast<float*>(p.c) + at) = v;
    } else {
      uint2 h;
      if (p.out_type == OUT_BF16)
        h = make_uint2(bf162_as_u32(__floats2bfloat162_rn(v.x, v.y)), bf162_as_u32(__floats2bfloat162_rn(v.z, v.w)));
      else
        h = make_uint2(h2_as_u32(__floats2half2_rn(v.x, v.y)), h2_as_u32(__floats2half2_rn(v.z, v.w)));
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.c) + at) = h;
    }
    return;
  }
  const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (col + i >= p.P) break;
    if (p.out_type == OUT_F32) static_cast<float*>(p.c)[at + i] = f[i];
    else if (p.out_type == OUT_BF16) static_cast<__nv_bfloat16*>(p.c)[at + i] = __float2bfloat16_rn(f[i]);
    else static_cast<__half*>(p.c)[at + i] = __float2half_rn(f[i]);
  }
}

// ---- one tile per cluster, its contraction split over the cluster's CTAs ---------------------------
//
// For few tokens and for problems of fewer tiles than the GPU has SMs. TN tokens x 128 weight rows:
//   TOK_LANE = false, TN = 16 or 32: weights own the 128 lanes (the instruction's M), tokens its N = TN
//     columns, so a token costs a column and not a lane; token scales reach the reading warps through a ring of TN
//     floats per block in shared memory, filled by 4-byte asynchronous copies.
//   TOK_LANE = true, TN = 128: tokens own the lanes, 128 weight rows the columns; a reading thread then
//     has one token and one scale per block (no vector of scales, half the fp32 work). Faster from 33
//     tokens on, half empty as it is then (48 tokens, 14336 x 4096: 17 us, in columns of 32 20; columns of 64
//     measure the same 17 and would be one more kernel).
// A cluster of up to 8 CTAs cuts the contraction, leaves its partial sums in shared memory, and every
// CTA adds up a share of the tile from all of them in rank order: no scratch, one launch, and the
// same bits every time.
//
// warp 0: TMA producer; warp 1: MMA issuer; warp 2: token scales; warp 3: tensor memory; then 4 or 8
// reading warps. Waits are bounded.
template <int TN> struct Fp8TileConfig {
  static constexpr int kReadWarps = TN == 128 ? 8 : 4;
  static constexpr int kThreads = 128 + 32 * kReadWarps;
  static constexpr int kCols = TN / (kReadWarps / 4);              // columns a reading thread adds up
  static constexpr int kAcc = 4;                                   // accumulators: the way round is longer than a block
  static constexpr int kTmemCols = TN * kAcc;                      // 64, 128, 512
  static constexpr int kTokenBytes = TN * 128;
  static constexpr int kStageBytes = 128 * 128 + kTokenBytes;
  // Up to 32 tokens two CTAs share an SM (bytes in flight, and one's start under the other's end); at 128
  // the reading threads need the registers and the four accumulators all of tensor memory.
  static constexpr int kStages = TN == 32 ? 5 : 6;
  static constexpr int kCtasPerSm = TN == 128 ? 1 : 2;
  static constexpr int kScaleSlots = 8;
  static constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kScaleSlots * TN * 4 + 512;
};

template <int TN>
struct Fp8TileCtl {
  using C = Fp8TileConfig<TN>;
  uint64_t full[C::kStages], empty[C::kStages];
  uint64_t acc_full[C::kAcc], acc_empty[C::kAcc];
  uint64_t sc_full[C::kScaleSlots], sc_empty[C::kScaleSlots];
  uint32_t tmem_base;
  int abort_flag;
  int valid;
  Fp8Tile tile;
};

template <bool TOK_LANE, int TN>
__global__ void __launch_bounds__(Fp8TileConfig<TN>::kThreads, Fp8TileConfig<TN>::kCtasPerSm)
fp8_tile_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                     const Fp8GemmParams p) {
  using C = Fp8TileConfig<TN>;
  static_assert(!TOK_LANE || TN == 128, "tokens on the lanes: 128 of them");
  static_assert(sizeof(Fp8TileCtl<TN>) <= 512, "control block");
  extern __shared__ uint8_t fp8_smem_raw[];
  // The offset to the 1 KiB boundary is the same in every CTA of the cluster: peers map each other's addresses.
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(fp8_smem_raw) + 1023) & ~uintptr_t(1023));
  float* scale_ring = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
  auto* ctl = reinterpret_cast<Fp8TileCtl<TN>*>(smem + C::kStages * C::kStageBytes + C::kScaleSlots * TN * 4);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* abort_flag = &ctl->abort_flag;
  DeviceStatus* st = p.status;
  const int rank = static_cast<int>(cluster_rank());

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kStages; ++i) { mbar_init(&ctl->full[i], 1); mbar_init(&ctl->empty[i], 1); }
    for (int i = 0; i < C::kAcc; ++i) { mbar_init(&ctl->acc_full[i], 1); mbar_init(&ctl->acc_empty[i], C::kReadWarps); }
    for (int i = 0; i < C::kScaleSlots; ++i) { mbar_init(&ctl->sc_full[i], 32); mbar_init(&ctl->sc_empty[i], C::kReadWarps); }
    ctl->abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 3) {
    tmem_alloc(&ctl->tmem_base, C::kTmemCols);
    tmem_relinquish();
  }
  chain_wait();
  if (warp == 2) {
    Fp8Tile tile;
    const bool valid = fp8_find_tile<TN>(p, blockIdx.x / p.split, lane, &tile);
    if (lane == 0) { ctl->tile = tile; ctl->valid = valid; }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  chain_next();
  const uint32_t tmem_base = ctl->tmem_base;
  const Fp8Tile tile = ctl->tile;
  // A tile behind the last one: every CTA of the cluster finds the same and does nothing but the
  // barriers below.
  const bool valid = ctl->valid;
  const int kb0 = static_cast<int>(static_cast<long long>(p.q_blocks) * rank / p.split);
  const int kb1 = valid ? static_cast<int>(static_cast<long long>(p.q_blocks) * (rank + 1) / p.split) : kb0;

  if (warp == 0) {
    if (lane == 0) {
      uint32_t s = 0, phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&ctl->empty[s], phase ^ 1u, abort_flag, st, 1)) break;
        uint8_t* stage = smem + s * C::kStageBytes;
        mbar_arrive_expect_tx(&ctl->full[s], C::kStageBytes);
        if (p.trans_w) tma_load_3d(stage, &tmap_w, tile.p0, kb * 128, tile.group, &ctl->full[s]);
        else tma_load_3d(stage, &tmap_w, kb * 128, tile.p0, tile.group, &ctl->full[s]);
        tma_load_2d(stage + 128 * 128, &tmap_a, kb * 128, tile.m0, &ctl->full[s]);
        if (++s == C::kStages) { s = 0; phase ^= 1u; }
      }
    }
  } else if (warp == 1) {
    // the whole warp runs this loop, so that operands sit in uniform registers; one lane issues
    const uint32_t idesc = TOK_LANE ? make_idesc_f8(p.a_fmt, p.w_fmt, 0, p.trans_w, 128, 128)
                                    : make_idesc_f8(p.w_fmt, p.a_fmt, p.trans_w, 0, 128, TN);
    // the next 32 of the contraction: 32 bytes on in a row, or 32 rows on where rows run along it
    const uint64_t w_step = p.trans_w ? 32 * 128 / 16 : 2;
    uint32_t s = 0, phase = 0, i = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb, ++i) {
      const uint32_t buf = i % C::kAcc;
      const uint32_t stage = smem_u32(smem + s * C::kStageBytes);
      const uint64_t w_desc = make_smem_desc_sw128(stage), t_desc = make_smem_desc_sw128(stage + 128 * 128);
      ok = ok && mbar_wait(&ctl->full[s], phase, abort_flag, st, 3);
      ok = ok && mbar_wait(&ctl->acc_empty[buf], ((i / C::kAcc) & 1u) ^ 1u, abort_flag, st, 2);
      tc_fence_after_sync();
      if (ok && elect_one()) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t w = w_desc + j * w_step, t = t_desc + 2 * j;
          umma_ss_f8(tmem_base + buf * TN, TOK_LANE ? t : w, TOK_LANE ? w : t, idesc, j != 0);
        }
        tc_commit(&ctl->acc_full[buf]);
        // The last stages are not handed back: nobody would wait for them, and an arrival that nobody waits for may come
        // when the CTA has left and its shared memory is someone else's.
        if (kb + C::kStages < kb1) tc_commit(&ctl->empty[s]);
      }
      __syncwarp();
      if (++s == C::kStages) { s = 0; phase ^= 1u; }
    }
  } else if (warp == 2) {
    if (!TOK_LANE) {
      uint32_t s = 0, phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait_warp(&ctl->sc_empty[s], phase ^ 1u, abort_flag, st, 4, lane)) break;
        for (int j = lane; j < TN; j += 32) {
          const long long m = min(tile.m0 + j, p.M - 1);                // rows behind the tile's: any valid address
          cp_async4(smem_u32(scale_ring + s * TN + j), p.a_scale + m * p.ld_a_scale + kb);
        }
        cp_async_arrive(&ctl->sc_full[s]);
        if (++s == C::kScaleSlots) { s = 0; phase ^= 1u; }
      }
      cp_async_wait_all();
    }
  } else if (warp >= 4) {
    const int quarter = warp & 3;
    const int col0 = ((warp - 4) >> 2) * C::kCols;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int row = quarter * 32 + lane;                                // this thread's lane of the accumulator
    constexpr int kChunk = C::kCols < 32 ? C::kCols : 32;
    uint64_t acc[C::kCols / 2];
#pragma unroll
    for (int i = 0; i < C::kCols / 2; ++i) acc[i] = 0;
    const float* ws = p.w_scale + tile.group * p.ws_group + (tile.p0 / 128) * p.ws_p;
    const float* as = p.a_scale + static_cast<long long>(min(tile.m0 + row, p.M - 1)) * p.ld_a_scale;
    uint32_t i = 0, s = 0, phase = 0;
    bool ok = true;
    // the scales two blocks ahead: their latency is longer than a block's multiplication
    float w0 = 0.f, w1 = 0.f, a0 = 1.f, a1 = 1.f;
    if (kb0 < kb1) { w0 = ws[kb0 * p.ws_q]; if (TOK_LANE) a0 = as[kb0]; }
    if (kb0 + 1 < kb1) { w1 = ws[(kb0 + 1) * p.ws_q]; if (TOK_LANE) a1 = as[kb0 + 1]; }
    for (int kb = kb0; kb < kb1; ++kb, ++i) {
      const uint32_t buf = i % C::kAcc;
      float w2 = 0.f, a2 = 1.f;
      if (kb + 2 < kb1) { w2 = ws[(kb + 2) * p.ws_q]; if (TOK_LANE) a2 = as[kb + 2]; }
      const float lane_scale = TOK_LANE ? a0 * w0 : w0;
      const uint64_t ls = pack2f(lane_scale, lane_scale);
      if (!TOK_LANE) ok &= mbar_wait(&ctl->sc_full[s], phase, abort_flag, st, 5);
      ok &= mbar_wait(&ctl->acc_full[buf], (i / C::kAcc) & 1u, abort_flag, st, 6);
      __syncwarp();
      tc_fence_after_sync();
      // all of this thread's columns at once: one latency of tensor memory a block, not one per piece
      uint32_t v[C::kCols / kChunk][kChunk];
#pragma unroll
      for (int c = 0; c < C::kCols / kChunk; ++c) tmem_ld_cols(tmem_base + lane_addr + buf * TN + col0 + c * kChunk, v[c]);
      uint64_t sc[TOK_LANE ? 1 : C::kCols / 2];
      if (TOK_LANE) {
        sc[0] = ls;
      } else {
        const float4* f = reinterpret_cast<const float4*>(scale_ring + s * TN + col0);
#pragma unroll
        for (int j = 0; j < C::kCols / 4; ++j) {
          const float4 q = f[j];
          sc[(2 * j) % (TOK_LANE ? 1 : C::kCols / 2)] = fmul2(pack2f(q.x, q.y), ls);
          sc[(2 * j + 1) % (TOK_LANE ? 1 : C::kCols / 2)] = fmul2(pack2f(q.z, q.w), ls);
        }
      }
#pragma unroll
      for (int c = 0; c < C::kCols / kChunk; ++c) tc_wait_ld(v[c]);
      // the accumulator and the scales go back before the additions
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&ctl->acc_empty[buf]);
        if (!TOK_LANE) mbar_arrive(&ctl->sc_empty[s]);
      }
#pragma unroll
      for (int c = 0; c < C::kCols / kChunk; ++c)
#pragma unroll
        for (int j = 0; j < kChunk / 2; ++j) {
          const int at = c * (kChunk / 2) + j;
          acc[at] = ffma2(pack2(v[c][2 * j], v[c][2 * j + 1]), sc[TOK_LANE ? 0 : at], acc[at]);
        }
      if (!TOK_LANE && ++s == C::kScaleSlots) { s = 0; phase ^= 1u; }
      w0 = w1; w1 = w2; a0 = a1; a1 = a2;
    }
    // Partial sums to shared memory. The ring is free: the last accumulator was full, so every MMA
    // has read its operands and every copy has landed. (After a wait that gave up nothing is written.)
    float* part = reinterpret_cast<float*>(smem);
    if (ok && valid) {
#pragma unroll
      for (int j = 0; j < C::kCols / 2; ++j) {
        const float2 f = unpack2(acc[j]);
        if (TOK_LANE) {
          // [token][132]: the four words of padding keep the 16-byte rows of a warp apart
          *reinterpret_cast<float2*>(part + row * 132 + col0 + 2 * j) = f;
        } else {
          part[(col0 + 2 * j) * 128 + row] = f.x;
          part[(col0 + 2 * j + 1) * 128 + row] = f.y;
        }
      }
    }
  }

  if (*abort_flag) {
    // copies in flight land before the shared memory goes away
    const uint64_t t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
  }
  __syncwarp();
  tc_fence_before_sync();
  if (p.split > 1) cluster_sync_all(); else __syncthreads();
  tc_fence_after_sync();

  // Every CTA adds up its share of the tile's tokens: work item = (token, four columns).
  if (valid && !*abort_flag) {
    const int tokens = min(TN, tile.m_end - tile.m0);
    const uint32_t part = smem_u32(smem);
    for (int w = warp; w * p.split + rank < tokens; w += C::kThreads / 32) {
      const int t = w * p.split + rank;
      const uint32_t at = part + 4u * static_cast<uint32_t>(TOK_LANE ? t * 132 + lane * 4 : t * 128 + lane * 4);
      float4 v;
      if (p.split == 1) {
        v = *reinterpret_cast<const float4*>(smem + (at - part));
      } else {
        v = cluster_load4(cluster_map(at, 0));
        for (int r = 1; r < p.split; ++r) {
          const float4 u = cluster_load4(cluster_map(at, r));
          v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
      }
      fp8_store4(p, static_cast<long long>(tile.m0) + t, tile.p0 + lane * 4, v);
    }
  }
  __syncwarp();
  // peers may still be reading this CTA's sums
  if (p.split > 1) cluster_sync_all(); else __syncthreads();
  if (warp == 3) tmem_dealloc(tmem_base, C::kTmemCols);
}

}  // namespace b200dq
