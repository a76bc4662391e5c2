// The product of fp8_gemm.cuh for many tokens: CTA pairs, tiles of 256 tokens x 256 weight rows.
//
// A pair of CTAs on two SMs works on one tile with tcgen05.mma.cta_group::2 (M = N = 256): each CTA
// loads 128 tokens and 128 weight rows per block of 128, 32 KB for its 4.2 million multiply-adds, two thirds
// of what a 128 x 256 tile of its own would pull through L2 for the same work. Its 128 x 256 sums per block go to
// one of two accumulators that fill tensor memory, and eight warps move them, scaled, to fp32
// registers: thread = one token, 128 columns, one scale per block; 64 packed fmas.
//
// What bounds it (4096 x 28672 x 8192, 760 us in a burst, 2530 TFLOP/s, the GPU at its power limit near 1.5 GHz): the
// way round of an accumulator. Timestamps of one buffer, in cycles: hand-back seen to accumulator full 910
// (four instructions of 128, issue, commit), first columns in registers 300, the rest read and added
// 270, hand-back to the issuing warp 90; two buffers in turn make 780 a block, where the multiplication alone
// needs 512 (590 at the rate it reaches with nobody waiting: 618 us). Tensor memory holds no third
// accumulator of this width; four of 128 columns (twice the instructions, each half as wide) measured
// 932 us, sixteen summing warps 957, three pieces in flight (registers spill) 839. So everything on the way
// is short: the issuing warp runs uniformly (operands in uniform registers; a single issuing thread took
// 920 us) and commits the accumulator before the stage. Strips of 16 token tiles, not 8: 826 against 840 us.
//
// Persistent: one pair per two SMs, tiles in strips of 16 token tiles so that the tiles in flight
// share their operands in L2. warp 0: TMA producer (both CTAs); warp 1: MMA issuer (first CTA);
// warp 2: tensor memory, output copies; warp 3: where tiles lie; warps 4-11: sums and output, which leaves through
// shared memory by TMA.
//
// GATED: weights are [gate; up], F rows each; the first CTA loads 128 gate rows, the second the 128 up
// rows that belong to them, so that a tile's columns 0-127 and 128-255 are g and u of the same 128
// features: exactly one quantiser block. The two warps that hold a token's g and u swap a half each
// through shared memory, compute silu(g) u on 64 columns each, agree on the maximum and write codes: h
// (4 bytes per value out, 4 back in, or 2 and 2) never goes to memory unless the caller wants it.
#pragma once
#include "fp8_gemm.cuh"
#include "fp8_quant.cuh"

namespace b200dq {

constexpr int kPairThreads = 384;
constexpr int kPairStages = 5;
constexpr int kPairHalf = 128 * 128;                          // one operand's half tile: 128 rows x 128 bytes
constexpr int kPairStageBytes = 2 * kPairHalf;
constexpr int kPairBoxBytes = 128 * 128;                      // 128 output rows of 128 bytes: one copy's box
constexpr int kPairSlabBytes = 32 * 128;                      // a summing warp's rows of it
constexpr int kPairOutBytes = 4 * kPairBoxBytes;              // two boxes for each half of the tile's columns
constexpr int kPairStrip = 16;
constexpr int kPairMaxGroups = 256;                           // groups whose tile table fits the control block
// setmaxnreg moves registers from warps 0-3 to the eight summing warps: 128 * 40 + 256 * 232 = 384 * 168
constexpr int kPairOtherRegs = 40, kPairSumRegs = 232;

struct Fp8PairCtl {
  uint64_t full[kPairStages], empty[kPairStages];
  uint64_t acc_full[2], acc_empty[2];
  uint64_t out_full[2], out_empty[2];                         // boxes of a half of the columns: written, and copied
  uint64_t place_full[2], place_empty[2];                     // where the tile two, or one, ahead lies
  Fp8Tile place[2];
  uint32_t tmem_base;
  int abort_flag;
  int row_prefix[kPairMaxGroups + 1];
  int tile_prefix[kPairMaxGroups + 1];                        // token tiles before each group
};
constexpr int kPairSmemBytes = kPairStages * kPairStageBytes + kPairOutBytes +
                               static_cast<int>((sizeof(Fp8PairCtl) + 15) / 16 * 16);
static_assert(kPairSmemBytes <= 232448, "shared memory of a CTA");

// Row and token-tile prefixes of the groups, by one warp. Counts are cut off at M rows in all.
__device__ __forceinline__ void fp8_pair_prefixes(const Fp8GemmParams& p, Fp8PairCtl* ctl, int lane) {
  long long rows = 0;
  int tiles = 0;
  for (int base = 0; base < p.num_groups; base += 32) {
    const int g = base + lane;
    long long c = 0;
    if (g < p.num_groups)
      c = p.counts_int64 ? static_cast<const long long*>(p.counts)[g] : static_cast<const int*>(p.counts)[g];
    long long r = min(max(c, 0ll), static_cast<long long>(p.M));
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, r, d);
      if (lane >= d) r += u;
    }
    const long long end = min(rows + r, static_cast<long long>(p.M));
    long long begin = __shfl_up_sync(0xffffffffu, end, 1);
    if (lane == 0) begin = min(rows, static_cast<long long>(p.M));
    int n = static_cast<int>((end - begin + 255) / 256);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, n, d);
      if (lane >= d) n += u;
    }
    if (g < p.num_groups) {
      ctl->row_prefix[g + 1] = static_cast<int>(end);
      ctl->tile_prefix[g + 1] = tiles + n;
    }
    rows += __shfl_sync(0xffffffffu, r, 31);
    tiles += __shfl_sync(0xffffffffu, n, 31);
  }
  if (lane == 0) ctl->row_prefix[0] = ctl->tile_prefix[0] = 0;
}

// n / d (inv = 1 / d to 2 units in the last place): the rounded quotient is off by one at most below 2^21, and by three
// for the most column tiles that an output can have, 2^23; the remainder, exact in 32 bits, puts it right. An
// integer division takes some 200 cycles, three of them in a row between two tiles.
__device__ __forceinline__ int div_small(int n, int d, float inv) {
  int q = static_cast<int>(static_cast<float>(n) * inv);
  int r = static_cast<int>(static_cast<unsigned>(n) - static_cast<unsigned>(q) * static_cast<unsigned>(d));
  for (; r < 0; r += d) --q;
  for (; r >= d; r -= d) ++q;
  return q;
}

// Where tile t lies: strips of kPairStrip token tiles, within a strip token tiles fastest.
__device__ __forceinline__ Fp8Tile fp8_pair_tile(const Fp8GemmParams& p, const Fp8PairCtl* ctl, int token_tiles, int t) {
  const int strip_tiles = kPairStrip * p.p_tiles;
  const int strip = token_tiles <= kPairStrip ? 0 : div_small(t, strip_tiles, __fdividef(1.0f, static_cast<float>(strip_tiles)));
  const int in_strip = t - strip * strip_tiles;
  const int high = min(kPairStrip, token_tiles - strip * kPairStrip);
  const int column = high == kPairStrip ? in_strip / kPairStrip
                                        : div_small(in_strip, high, __fdividef(1.0f, static_cast<float>(high)));
  const int tt = strip * kPairStrip + in_strip - column * high;
  const int p0 = column * p.tile_cols;
  if (p.counts == nullptr) return Fp8Tile{0, tt * 256, p.M, p0};
  int lo = 0, hi = p.num_groups;                              // tile_prefix[lo] <= tt < tile_prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ctl->tile_prefix[mid] <= tt) lo = mid; else hi = mid;
  }
  return Fp8Tile{lo, ctl->row_prefix[lo] + (tt - ctl->tile_prefix[lo]) * 256, ctl->row_prefix[lo + 1], p0};
}

__device__ __forceinline__ void st_shared4(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ uint4 ld_shared4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

// Whether this CTA's 128 rows leave by TMA, `rows` of them in C or in the group: a box may hang over the last row
// of C, which the hardware cuts off, but not over the last row of a group.
__device__ __forceinline__ bool pair_box_is_whole(const Fp8GemmParams& p, int rows) {
  return p.c_vec16 && (rows >= 128 || (rows > 0 && p.counts == nullptr));
}

// A warp's 32 rows x 128 columns of fp32 sums (thread = row) to C, through its slab of the two boxes of its half
// of the columns (128 bytes of each row, 16-byte chunks rotated by the row, as the tensor map's
// 128-byte swizzle has them: no bank conflicts). Whole boxes leave by TMA, issued by a thread of another warp:
// issuing keeps a thread for hundreds of cycles, which the next tile's sums would wait for. Where a group
// ends inside the box, or C's rows do not start on 16 bytes, the warps write the rows. `rows`: of the CTA's
// 128. `swap` = 64: the thread's first 64 columns are the tile's second 64 (gated u). `used`: rounds of the
// boxes so far, counted by every summing warp and by the issuing one alike.
template <int OUT_TYPE>
__device__ __forceinline__ bool fp8_pair_store(const Fp8GemmParams& p, Fp8PairCtl* ctl, int half, int quarter, uint32_t slab,
                                               const uint64_t (&acc)[64], int m0, int rows, int col0, int swap, int lane,
                                               uint32_t& used) {
  constexpr int kSize = OUT_TYPE == OUT_F32 ? 4 : 2;
  constexpr int kCols = 128 / kSize;                          // columns of a box
  const uint32_t out_rot = (lane & 7) << 4;
  const bool whole = pair_box_is_whole(p, rows);
  bool ok = true;
#pragma unroll
  for (int round = 0; round < 64 / kCols; ++round, ++used) {
    ok &= mbar_wait(&ctl->out_empty[half], (used & 1u) ^ 1u, &ctl->abort_flag, p.status, 17);
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 16; ++j) {                            // 16-byte chunks of this thread's row
      uint32_t h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (OUT_TYPE == OUT_F32) {
          const float2 f = unpack2(acc[round * 32 + 2 * j + (i >> 1)]);
          h[i] = __float_as_uint(i & 1 ? f.y : f.x);
        } else {
          const float2 f = unpack2(acc[round * 64 + 4 * j + i]);
          h[i] = OUT_TYPE == OUT_BF16 ? bf162_as_u32(__floats2bfloat162_rn(f.x, f.y)) : h2_as_u32(__floats2half2_rn(f.x, f.y));
        }
      }
      st_shared4(slab + (j >> 3) * kPairBoxBytes + lane * 128 + (((j & 7) << 4) ^ out_rot), h);
    }
    if (whole) {
      fence_proxy_async_smem();
      __syncwarp();
    } else {
      __syncwarp();
      const int chunk = lane & 7;
#pragma unroll 1
      for (int k = 0; k < 2; ++k) {
        const int c = col0 + (((round * 2 + k) * kCols) ^ swap) + chunk * (16 / kSize);
#pragma unroll 1
        for (int row = lane >> 3; row < 32 && quarter * 32 + row < rows; row += 4) {
          const uint4 v = ld_shared4(slab + k * kPairBoxBytes + row * 128 + ((chunk ^ (row & 7)) << 4));
          uint8_t* dst = static_cast<uint8_t*>(p.c) + (static_cast<size_t>(m0 + quarter * 32 + row) * p.ldc + c) * kSize;
          if (p.c_vec16 && c < p.P) {
            *reinterpret_cast<uint4*>(dst) = v;
          } else {
            const uint32_t e4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 16 / kSize; ++e) {
              if (c + e >= p.P) break;
              if (kSize == 4) reinterpret_cast<uint32_t*>(dst)[e] = e4[e];
              else reinterpret_cast<uint16_t*>(dst)[e] = static_cast<uint16_t>(e4[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
      }
      __syncwarp();
    }
    if (lane == 0) mbar_arrive(&ctl->out_full[half]);
  }
  return ok;
}

// The issuing thread's side of one tile: each half's boxes as its four warps have filled them.
template <int OUT_TYPE, bool GATED>
__device__ __forceinline__ bool fp8_pair_copy_out(const Fp8GemmParams& p, const CUtensorMap* tmap_c, Fp8PairCtl* ctl,
                                                  uint32_t boxes, const Fp8Tile& tile, int rank, uint32_t& used) {
  constexpr int kCols = OUT_TYPE == OUT_F32 ? 32 : 64;
  const int m0 = tile.m0 + rank * 128;
  const bool whole = pair_box_is_whole(p, tile.m_end - m0);
#pragma unroll 1
  for (int round = 0; round < 64 / kCols; ++round, ++used) {
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
      if (!mbar_wait(&ctl->out_full[half], used & 1u, &ctl->abort_flag, p.status, 18)) return false;
      if (!whole) continue;
      const int swap = GATED && half == 1 ? 64 : 0;
      const int col0 = tile.p0 + half * (GATED ? p.P / 2 : 128);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int col = col0 + (((round * 2 + k) * kCols) ^ swap);
        if (col < p.P) tma_store_2d_at(tmap_c, boxes + (half * 2 + k) * kPairBoxBytes, col, m0);
      }
    }
    tma_store_commit();
    tma_store_wait_read<0>();
    mbar_arrive(&ctl->out_empty[0]);
    mbar_arrive(&ctl->out_empty[1]);
  }
  return true;
}

// acc[at ..] += scale * 32 columns, in pairs.
__device__ __forceinline__ void fp8_pair_add(uint64_t (&acc)[64], const int at, const uint32_t (&v)[32], uint64_t scale) {
#pragma unroll
  for (int j = 0; j < 16; ++j) acc[at + j] = ffma2(pack2(v[2 * j], v[2 * j + 1]), scale, acc[at + j]);
}

__device__ __forceinline__ void pair_barrier(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// silu(g) u on two values at a time, as sigmoid_of and silu_mul_of round it.
__device__ __forceinline__ uint64_t silu_mul2(uint64_t g, uint64_t u) {
  const float2 t = unpack2(fmul2(g, pack2f(-1.4426950408889634f, -1.4426950408889634f)));
  float2 e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
  const float2 d = unpack2(fadd2(pack2f(e.x, e.y), pack2f(1.0f, 1.0f)));
  float2 r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  return fmul2(fmul2(g, pack2f(r.x, r.y)), u);
}

// This warp's 64 features, in place of the first half of `acc`; returns the largest magnitude.
template <bool GATE>
__device__ __forceinline__ float fp8_pair_act(uint64_t (&acc)[64], uint32_t partner, int lane) {
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const uint4 o = ld_shared4(partner + (j >> 3) * kPairBoxBytes + lane * 128 + (((j & 7) ^ (lane & 7)) << 4));
    const uint64_t got[2] = {pack2(o.x, o.y), pack2(o.z, o.w)};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint64_t own = acc[2 * j + e];
      const uint64_t v = GATE ? silu_mul2(own, got[e]) : silu_mul2(got[e], own);
      const float2 f = unpack2(v);
      amax = max_magnitude(max_magnitude(amax, f.x), f.y);
      acc[2 * j + e] = v;
    }
  }
  return amax;
}

// The two warps of a lane quarter hold g and u of 32 tokens x 128 features, each its own 64 features in the
// first half of `acc`. They swap the second halves, compute silu(g) u on 64 features each, agree
// on the rows' maxima and write codes. `mine`, `partner`: the two warps' slabs of their pairs of boxes.
template <int FP8>
__device__ __forceinline__ void fp8_pair_gate(const Fp8GemmParams& p, uint32_t mine, uint32_t partner, uint64_t (&acc)[64],
                                              int half, int quarter, int m_first, int rows, int f0, int lane) {
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const float2 a = unpack2(acc[32 + 2 * j]), b = unpack2(acc[32 + 2 * j + 1]);
    const uint32_t w[4] = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y)};
    st_shared4(mine + (j >> 3) * kPairBoxBytes + lane * 128 + (((j & 7) ^ (lane & 7)) << 4), w);
  }
  pair_barrier(1 + quarter);
  float amax = half == 0 ? fp8_pair_act<true>(acc, partner, lane) : fp8_pair_act<false>(acc, partner, lane);
  pair_barrier(1 + quarter);                                  // both have read
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(mine + kPairBoxBytes + lane * 4), "f"(amax) : "memory");
  pair_barrier(1 + quarter);
  float other;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(other) : "r"(partner + kPairBoxBytes + lane * 4) : "memory");
  amax = max_magnitude(amax, other);
  const float s = fp8_scale_of<FP8>(__float_as_uint(amax));
  const float inv = __frcp_rn(s);
  const uint64_t inv2 = pack2f(inv, inv);
  // codes: 64 bytes of each row through the first box, so that a store instruction writes 8 rows' 64 bytes
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 a = unpack2(fmul2(acc[j * 8 + 2 * i], inv2)), b = unpack2(fmul2(acc[j * 8 + 2 * i + 1], inv2));
      w[i] = fp8_pair<FP8>(a.x, a.y) | (fp8_pair<FP8>(b.x, b.y) << 16);
    }
    st_shared4(mine + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), w);
  }
  if (half == 0 && lane < rows) p.gate_scales[static_cast<long long>(m_first + lane) * p.p_tiles + f0 / 128] = s;
  __syncwarp();
  uint8_t* dst = p.gate_codes + static_cast<long long>(m_first) * p.ld_gate + f0 + half * 64 + (lane & 3) * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = i * 8 + (lane >> 2);
    const uint4 v = ld_shared4(mine + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
    if (row < rows) *reinterpret_cast<uint4*>(dst + row * p.ld_gate) = v;
  }
  pair_barrier(1 + quarter);                                  // the partner has read the maxima; the boxes are free
}

template <bool GATED>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_pair_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                     const __grid_constant__ CUtensorMap tmap_c, const Fp8GemmParams p) {
  extern __shared__ __align__(1024) uint8_t fp8_pair_smem[];     // swizzle atoms start on 1 KiB boundaries
  uint8_t* smem = fp8_pair_smem;
  uint8_t* stage_out = smem + kPairStages * kPairStageBytes;
  auto* ctl = reinterpret_cast<Fp8PairCtl*>(stage_out + kPairOutBytes);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  volatile int* abort_flag = &ctl->abort_flag;
  DeviceStatus* st = p.status;
  const int rank = static_cast<int>(cluster_rank());

  if (threadIdx.x == 0) {
    for (int i = 0; i < kPairStages; ++i) { mbar_init(&ctl->full[i], 1); mbar_init(&ctl->empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&ctl->acc_full[i], 1); mbar_init(&ctl->acc_empty[i], 16); }
    for (int i = 0; i < 2; ++i) { mbar_init(&ctl->out_full[i], 4); mbar_init(&ctl->out_empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&ctl->place_full[i], 1); mbar_init(&ctl->place_empty[i], 8); }
    ctl->place[0] = ctl->place[1] = Fp8Tile{0, 0, 0, 0};      // a valid place also after a wait that gave up
    ctl->abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
  }
  if (warp == 2) {
    tmem_alloc_pair(&ctl->tmem_base, 512);
    tmem_relinquish_pair();
  }
  chain_wait();
  if (warp == 3 && p.counts != nullptr) fp8_pair_prefixes(p, ctl, lane);
  __syncwarp();
  tc_fence_before_sync();
  cluster_sync_all();                                         // the peer's barriers exist
  tc_fence_after_sync();
  chain_next();
  const uint32_t tmem_base = ctl->tmem_base;
  const int token_tiles = p.counts != nullptr ? ctl->tile_prefix[p.num_groups] : (p.M + 255) / 256;
  const int tiles = token_tiles * p.p_tiles;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairOtherRegs));
    if (warp == 0 && lane == 0) {
      // ---------------- producer: this CTA's halves, completing on the first CTA's barriers ----------------
      uint32_t s = 0, phase = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        const Fp8Tile tile = fp8_pair_tile(p, ctl, token_tiles, t);
        const int m0 = tile.m0 + rank * 128, p0 = tile.p0 + rank * (GATED ? p.P / 2 : 128);
        for (int kb = 0; kb < p.q_blocks; ++kb) {
          ok = mbar_wait(&ctl->empty[s], phase ^ 1u, abort_flag, st, 11);
          if (!ok) break;
          uint8_t* stage = smem + s * kPairStageBytes;
          const uint32_t bar = cluster_map(smem_u32(&ctl->full[s]), 0);
          if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], 2 * kPairStageBytes);
          tma_load_2d_pair(stage, &tmap_a, kb * 128, m0, bar);
          if (p.trans_w) tma_load_3d_pair(stage + kPairHalf, &tmap_w, p0, kb * 128, tile.group, bar);
          else tma_load_3d_pair(stage + kPairHalf, &tmap_w, kb * 128, p0, tile.group, bar);
          if (++s == kPairStages) { s = 0; phase ^= 1u; }
        }
      }
    } else if (warp == 1 && rank == 0) {
      // ---------------- MMA issuer for both CTAs ----------------
      const uint32_t idesc = make_idesc_f8(p.a_fmt, p.w_fmt, 0, p.trans_w, 256, 256);
      const uint64_t w_step = p.trans_w ? 32 * 128 / 16 : 2;
      uint32_t s = 0, phase = 0, i = 0;
      // Blocks of all of this pair's tiles. The last stages are not handed back: nobody would wait for them, and an
      // arrival that nobody waits for may come when a CTA has left and its shared memory is someone else's.
      const uint32_t blocks = pair < tiles ? static_cast<uint32_t>((tiles - pair - 1) / pairs + 1) * p.q_blocks : 0;
      bool ok = true;
      for (int t = pair; t < tiles; t += pairs) {
        for (int kb = 0; kb < p.q_blocks; ++kb, ++i) {
          const uint32_t buf = i & 1u, acc = tmem_base + buf * 256;
          const uint32_t stage = smem_u32(smem + s * kPairStageBytes);
          const uint64_t a_desc = make_smem_desc_sw128(stage), w_desc = make_smem_desc_sw128(stage + kPairHalf);
          ok = ok && mbar_wait(&ctl->full[s], phase, abort_flag, st, 13);
          ok = ok && mbar_wait(&ctl->acc_empty[buf], ((i >> 1) & 1u) ^ 1u, abort_flag, st, 12);
          tc_fence_after_sync();
          if (ok && elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              umma_pair_ss_f8(acc, a_desc + 2 * j, w_desc + j * w_step, idesc, j != 0);
            tc_commit_pair(&ctl->acc_full[buf]);
            if (i + kPairStages < blocks) tc_commit_pair(&ctl->empty[s]);
          }
          __syncwarp();
          if (++s == kPairStages) { s = 0; phase ^= 1u; }
        }
      }
    } else if (warp == 2 && lane == 0 && (!GATED || p.c != nullptr)) {
      // ---------------- output copies of this CTA's rows ----------------
      uint32_t used = 0;
      bool ok = true;
      for (int t = pair; ok && t < tiles; t += pairs) {
        const Fp8Tile tile = fp8_pair_tile(p, ctl, token_tiles, t);
        if (GATED || p.out_type != OUT_F32)
          ok = fp8_pair_copy_out<OUT_BF16, GATED>(p, &tmap_c, ctl, smem_u32(stage_out), tile, rank, used);
        else
          ok = fp8_pair_copy_out<OUT_F32, GATED>(p, &tmap_c, ctl, smem_u32(stage_out), tile, rank, used);
      }
      tma_store_wait_read<0>();                               // copies have read their boxes before the memory goes away
    } else if (warp == 3) {
      // ---------------- the summing warps' tiles, ahead of them, and the first sectors of their scales into L1 ----------------
      uint32_t n = 0;
      for (int t = pair; t < tiles; t += pairs, ++n) {
        if (!mbar_wait_warp(&ctl->place_empty[n & 1u], ((n >> 1) & 1u) ^ 1u, abort_flag, st, 19, lane)) break;
        const Fp8Tile tile = fp8_pair_tile(p, ctl, token_tiles, t);
        if (lane == 0) {
          ctl->place[n & 1u] = tile;
          mbar_arrive(&ctl->place_full[n & 1u]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          prefetch_l1(p.a_scale + static_cast<long long>(min(tile.m0 + rank * 128 + 32 * j + lane, p.M - 1)) * p.ld_a_scale);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairSumRegs));
    // ---------------- sums: thread = one token of this CTA, 128 of the tile's columns ----------------
    const int quarter = warp & 3, half = (warp - 4) >> 2;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t slab = smem_u32(stage_out + half * 2 * kPairBoxBytes + quarter * kPairSlabBytes);
    const uint32_t other = smem_u32(stage_out + (half ^ 1) * 2 * kPairBoxBytes + quarter * kPairSlabBytes);
    const uint32_t empty_bar = cluster_map(smem_u32(&ctl->acc_empty[0]), 0);
    // gated, the warps of u take their columns in the order 64-127, 0-63: every warp then keeps its first 64
    const uint32_t swap = GATED && half == 1 ? 64 : 0;
    const uint32_t acc_addr = tmem_base + lane_addr + half * 128;
    uint32_t i = 0, used = 0;
    bool ok = true;
    // Where a tile lies comes from warp 3 (divisions and, grouped, a search: some 400 cycles between two tiles). Its
    // scales are fetched two blocks ahead (their latency is longer than a block's multiplication), the next
    // tile's first two before this one's rows are written.
    Fp8Tile tile;
    const float *as = nullptr, *ws = nullptr;
    float a0 = 0.f, w0 = 0.f, a1 = 0.f, w1 = 0.f;
    const auto begin = [&](uint32_t n) {
      ok &= mbar_wait(&ctl->place_full[n & 1u], (n >> 1) & 1u, abort_flag, st, 20);
      tile = ctl->place[n & 1u];
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->place_empty[n & 1u]);
      // a tile may end before its second half; gated, the second half is the up half of the weight
      const int p_block = GATED ? (tile.p0 + half * (p.P / 2)) / 128 : min(tile.p0 / 128 + half, (p.P - 1) / 128);
      as = p.a_scale + static_cast<long long>(min(tile.m0 + rank * 128 + quarter * 32 + lane, p.M - 1)) * p.ld_a_scale;
      ws = p.w_scale + tile.group * p.ws_group + p_block * p.ws_p;
      a0 = as[0]; w0 = ws[0];
      if (p.q_blocks > 1) { a1 = as[1]; w1 = ws[p.ws_q]; }
      as += 2; ws += 2 * p.ws_q;
    };
    uint32_t n = 0;
    if (pair < tiles) begin(0);
    for (int t = pair; t < tiles; t += pairs) {
      uint64_t acc[64];
#pragma unroll
      for (int j = 0; j < 64; ++j) acc[j] = 0;
      // Pieces of 32 columns, one being added while the next is read: under the multiplication a piece takes
      // about 90 cycles to read and 64 to add (two warps share the pipes). The accumulator goes back with the
      // last piece in registers.
      uint32_t v[2][32];
      ok &= mbar_wait(&ctl->acc_full[i & 1u], (i >> 1) & 1u, abort_flag, st, 14);
      __syncwarp();
      tc_fence_after_sync();
      tmem_ld_32x32b_x32(acc_addr + (i & 1u) * 256 + swap, v[0]);
#pragma unroll 1
      for (int kb = 0; kb < p.q_blocks; ++kb, ++i) {
        const uint32_t buf = i & 1u, addr = acc_addr + buf * 256, next = acc_addr + (buf ^ 1u) * 256;
        const bool more = kb + 1 < p.q_blocks;
        float a2 = 0.f, w2 = 0.f;
        if (kb + 2 < p.q_blocks) {
          a2 = *as; w2 = *ws;
          ++as; ws += p.ws_q;
        }
        const float s0 = a0 * w0;
        const uint64_t scale = pack2f(s0, s0);
        tc_wait_ld(v[0]);
        tmem_ld_32x32b_x32(addr + swap + 32, v[1]);
        fp8_pair_add(acc, 0, v[0], scale);
        tc_wait_ld(v[1]);
        tmem_ld_32x32b_x32(addr + (64 - swap), v[0]);
        fp8_pair_add(acc, 16, v[1], scale);
        tc_wait_ld(v[0]);
        tmem_ld_32x32b_x32(addr + (96 - swap), v[1]);
        fp8_pair_add(acc, 32, v[0], scale);
        tc_wait_ld(v[1]);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(empty_bar + 8 * buf);
        fp8_pair_add(acc, 48, v[1], scale);
        if (more) {
          ok &= mbar_wait(&ctl->acc_full[buf ^ 1u], ((i + 1) >> 1) & 1u, abort_flag, st, 14);
          __syncwarp();
          tc_fence_after_sync();
          tmem_ld_32x32b_x32(next + swap, v[0]);
        }
        a0 = a1; w0 = w1; a1 = a2; w1 = w2;
      }
      const Fp8Tile done = tile;
      if (t + pairs < tiles) begin(++n);
      const int m0 = done.m0 + rank * 128;
      ok = __all_sync(0xffffffffu, ok);                        // a wait that gave up: no lane writes
      const int rows = ok ? done.m_end - m0 : 0;               // of this CTA's 128; may be none or more
      if (GATED) {
        if (p.c != nullptr) {
          ok &= fp8_pair_store<OUT_BF16>(p, ctl, half, quarter, slab, acc, m0, rows, done.p0 + half * (p.P / 2), swap, lane, used);
          // h has left both halves' boxes
          ok &= mbar_wait(&ctl->out_empty[0], (used & 1u) ^ 1u, abort_flag, st, 17);
          ok &= mbar_wait(&ctl->out_empty[1], (used & 1u) ^ 1u, abort_flag, st, 17);
          __syncwarp();
        }
        // both warps of a quarter meet in here, whatever happened to either
        const int m_first = m0 + quarter * 32, mine = min(32, rows - quarter * 32);
        if (p.gate_fp8 == FP8_E4M3) fp8_pair_gate<FP8_E4M3>(p, slab, other, acc, half, quarter, m_first, mine, done.p0, lane);
        else fp8_pair_gate<FP8_E5M2>(p, slab, other, acc, half, quarter, m_first, mine, done.p0, lane);
      } else {
        const int col0 = done.p0 + half * 128;
        if (p.out_type == OUT_BF16) ok &= fp8_pair_store<OUT_BF16>(p, ctl, half, quarter, slab, acc, m0, rows, col0, 0, lane, used);
        else if (p.out_type == OUT_F16) ok &= fp8_pair_store<OUT_F16>(p, ctl, half, quarter, slab, acc, m0, rows, col0, 0, lane, used);
        else ok &= fp8_pair_store<OUT_F32>(p, ctl, half, quarter, slab, acc, m0, rows, col0, 0, lane, used);
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
  cluster_sync_all();                                         // neither CTA leaves while the other may use its memory
  tc_fence_after_sync();
  if (warp == 2) tmem_dealloc_pair(tmem_base, 512);
}

}  // namespace b200dq
