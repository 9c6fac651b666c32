// Low-rank adapters of many requests beside a shared projection: out[m] = y[m] + scale_a (x[m] A_a^T) B_a^T, a the
// adapter of row m, or out[m] = y[m] where it has none.
//
// HBM-bound with many rows (x once, y once, out once; the adapters' weights stay in the L2s), latency-bound with few.
// 32768 rows x 5120 -> 15360, rank 32: 82 us (4.1 TB/s) and 384 (5.2 TB/s; a copy: 5.2); 64 single rows of 16 adapters,
// 5120 -> 5120, rank 16: 8 us and 5.
//
// The plan holds the rows sorted by adapter and cut into tiles of 32 or 64 rows of one adapter, so requests in any order
// and rows of one adapter that lie apart share a tile; rows are read and written where they lie.
//   adapter_down_kernel  u = x A^T in fp32: a workgroup a tile, its waves on every NW-th step of 64 k.
//   adapter_join_kernel  only where few tiles over a deep K are cut along K, or an fp16 rank is over 128: adds the shares.
//   adapter_up_kernel    out = y + scale (u B^T): a workgroup 32 rows of a tile and a range of columns.
// No atomics: every sum has a fixed order.
//
// u is handed on as two 16-bit values, a leading and a trailing one, in the operand order of the second product (x A^T is
// not rounded to 16 bits: the doubled rank costs nothing where memory is the bound). For fp16 each row of u first gets a
// power-of-two scale that keeps it in range, so a workgroup needs all of its ranks; bfloat16 has float32's range, and its
// ranks may be shared out among workgroups.
#pragma once

#include "block_types.h"

namespace hf {

constexpr int kAdChunk = 64;  // k of one step

struct AdapterTile {
  int32_t adapter, start, count, pad;
};

struct AdapterArgs {
  const uint16_t *x, *y, *down, *up;
  const float* scale;
  uint16_t* out;
  v4u* frags;       // [tiles][r32 / 16][row blocks][leading, trailing][64]
  float* factors;   // [tiles][tile rows]
  float* planes;    // [splits][tiles][tile rows][r32], where the sums are joined
  const AdapterTile* tiles;
  const int32_t* rows;
  int64_t ldx, ldy, ldo, K, N;
  int live_tiles, tile_rows, r, r32, splits, blocks_per_wg, col_groups, in_place, stream_y;
};

// Row `row` of a tile's u, fp32 in LDS at p, ranks lo to hi, into operand order, and the row's factor: four neighbouring
// lanes a row, `part` of 0 to 3. For fp16 lo is 0 and hi the whole rank.
template <class T>
__device__ __forceinline__ void adapter_operands(const AdapterArgs& a, const AdapterTile& tile, int tile_index,
                                                 const float* p, int row, int part, int blocks, int lo, int hi) {
  p -= lo;
  float grow = 1.0f;
  if constexpr (T::kNarrow) {
    float most = 0.0f;
    for (int j = part; j < hi / 8; j += 4)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * j + e < a.r) most = fmaxf(most, fabsf(p[8 * j + e]));
    most = fmaxf(most, __shfl_xor(most, 1, 64));
    most = fmaxf(most, __shfl_xor(most, 2, 64));
    // 2^(6 - exponent): the row's largest lands in [2^6, 2^7), where fp16 holds it and its trailing part is normal. Rows
    // of infinities and of values near the ends of fp32 stay as they are.
    const bool fine = most >= 0x1p-100f && most <= 0x1p100f;
    grow = fine ? __uint_as_float((260u - (__float_as_uint(most) >> 23)) << 23) : 1.0f;
  }
  const float scale = a.scale ? a.scale[tile.adapter] : 1.0f;
  if (part == 0 && lo == 0) a.factors[(int64_t)tile_index * a.tile_rows + row] = scale / grow;  // exact: a power of two
  v4u* frags = a.frags + (int64_t)tile_index * (a.r32 / 16) * blocks * 128;
  for (int j = lo / 8 + part; j < hi / 8; j += 4) {
    v4u lead, trail;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int rank = 8 * j + 2 * e;
      const float v = rank < a.r ? p[rank] * grow : 0.0f, w = rank + 1 < a.r ? p[rank + 1] * grow : 0.0f;
      lead[e] = T::pack(v, w);
      const float v1 = T::lo(lead[e]), w1 = T::hi(lead[e]);
      // An infinity or NaN has no trailing part.
      trail[e] = T::pack(fabsf(v1) < __builtin_inff() ? v - v1 : 0.0f, fabsf(w1) < __builtin_inff() ? w - w1 : 0.0f);
    }
    v4u* to = frags + ((j >> 1) * blocks + (row >> 5)) * 128 + (j & 1) * 32 + (row & 31);
    to[0] = lead;
    to[64] = trail;
  }
}

// Stages of a wave's ring and bytes of one: RB rank blocks and NB row blocks of 32 rows x 64 k.
__host__ __device__ constexpr int ad_stage_bytes(int rb, int nb) { return 4096 * (rb + nb); }
__host__ __device__ constexpr int ad_stages(int rb, int nb, int nw) {
  return 147456 / (ad_stage_bytes(rb, nb) * nw) < 4 ? 147456 / (ad_stage_bytes(rb, nb) * nw) : 4;
}
__host__ __device__ constexpr int ad_down_lds(int rb, int nb, int nw) {
  return ad_stages(rb, nb, nw) * ad_stage_bytes(rb, nb) * nw;
}

// Waits until at most n of the wave's loads are on their way (n from 2 to 24, any other: none).
__device__ __forceinline__ void ad_wait(int n) {
  switch (n) {
#define HF_WAIT(N) case N: asm volatile("s_waitcnt vmcnt(" #N ")" ::: "memory"); break;
    HF_WAIT(2) HF_WAIT(3) HF_WAIT(4) HF_WAIT(5) HF_WAIT(6) HF_WAIT(7) HF_WAIT(8) HF_WAIT(9) HF_WAIT(10) HF_WAIT(11)
    HF_WAIT(12) HF_WAIT(13) HF_WAIT(14) HF_WAIT(15) HF_WAIT(16) HF_WAIT(17) HF_WAIT(18) HF_WAIT(19) HF_WAIT(20)
    HF_WAIT(21) HF_WAIT(22) HF_WAIT(23) HF_WAIT(24)
#undef HF_WAIT
    default: asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); break;
  }
}

// Tile blockIdx.x, K share blockIdx.y, ranks from 32 RB blockIdx.z on.
//
// Each wave streams its own steps of 64 k through a ring of its own in LDS (16 bytes a lane, whole 128-byte lines, past
// the registers), so the loop has no barrier; the waves' sums are added at the end. Rows lie 128 bytes apart in LDS,
// swizzled so that fragment reads are conflict-free.
template <class T, int RB, int NB, int NW>
__global__ __launch_bounds__(64 * NW, 1) void adapter_down_kernel(AdapterArgs a) {
  constexpr int S = ad_stages(RB, NB, NW), kStage = ad_stage_bytes(RB, NB), kLoads = 4 * (RB + NB);
  static_assert(S >= 2, "the next step is loaded while one is computed");
  extern __shared__ __attribute__((aligned(1024))) unsigned char ad_lds[];
  const AdapterTile tile = a.tiles[blockIdx.x];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int sub = lane & 31, half = lane >> 5;
  const int rank0 = blockIdx.z * 32 * RB;
  unsigned char HF_LDS* ring = (unsigned char HF_LDS*)ad_lds + wave * S * kStage;

  // Load i of a step fills rows 8i .. 8i + 7 of the step's NB x 32 rows of x and RB x 32 of A; lane l row l / 8, from
  // chunk swizzle128(row, l % 8). Groups of 8 rows past the tile or the rank are not loaded, and rows past them within a
  // group repeat the last one: what comes of them is not used.
  const uint16_t* from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = 8 * i + (lane >> 3), c = swizzle128(r & 31, lane & 7);
    from[i] = i < 4 * NB ? a.x + (int64_t)a.rows[tile.start + min(r, tile.count - 1)] * a.ldx + 8 * c
                         : a.down + ((int64_t)tile.adapter * a.r + min(rank0 + r - 32 * NB, a.r - 1)) * a.K + 8 * c;
  }
  const int64_t full = a.K / kAdChunk;  // whole steps; what is left of K comes after the loop
  const int64_t share = (full + a.splits - 1) / a.splits;
  const int64_t c_lo = min(share * blockIdx.y, full), c_hi = min(c_lo + share, full);
  const int steps = c_hi - c_lo > wave ? (int)((c_hi - c_lo - wave + NW - 1) / NW) : 0;
  const int x_loads = min(4 * NB, (tile.count + 7) / 8);
  const int loads = x_loads + min(4 * RB, (a.r - rank0) / 8);
  auto load = [&](int step, int slot) __attribute__((always_inline)) {
    const int64_t k0 = (c_lo + wave + (int64_t)step * NW) * kAdChunk;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (i < 4 * NB ? i >= x_loads : i - 4 * NB >= loads - x_loads) continue;
      __builtin_amdgcn_global_load_lds((const void __attribute__((address_space(1)))*)(from[i] + k0),
                                       (void HF_LDS*)(ring + slot * kStage + i * 1024), 16, 0, 0);
    }
  };

  v16f acc[RB][NB];
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int n = 0; n < NB; ++n) acc[b][n] = (v16f){0};
#pragma unroll
  for (int s = 0; s < S; ++s)
    if (s < steps) load(s, s);
  int slot = 0;
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    // The step's loads have landed; those of the S - 1 steps after it may be on their way.
    static_assert((S - 1) * kLoads <= 24, "a wait for this ring");
    ad_wait(step + S > steps ? 0 : (S - 1) * loads);
    const unsigned char HF_LDS* at = ring + slot * kStage;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int chunk = swizzle128(sub, 2 * s + half) * 16 + sub * 128;
      v4u xf[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) xf[n] = *(const v4u HF_LDS*)(at + n * 4096 + chunk);
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const v4u df = *(const v4u HF_LDS*)(at + (NB + b) * 4096 + chunk);
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[b][n] = T::mfma(df, xf[n], acc[b][n]);
      }
    }
    // Every read of the slot has returned: it takes the step S further on. Filled after the products rather than before
    // them, the whole ring is on its way whenever the wave waits, and latency is what the loop would wait for.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (step + S < steps) load(step + S, slot);
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  if (a.K % kAdChunk && wave == 0 && blockIdx.y + 1 == gridDim.y) {
    const v4u zero = {0, 0, 0, 0};
    for (int64_t k0 = full * kAdChunk; k0 < a.K; k0 += 16) {
      const int64_t k = k0 + 8 * half;
      v4u xf[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n)
        xf[n] = k < a.K ? *(const v4u*)(a.x + (int64_t)a.rows[tile.start + min(32 * n + sub, tile.count - 1)] * a.ldx + k)
                        : zero;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const v4u df = k < a.K ? *(const v4u*)(a.down + ((int64_t)tile.adapter * a.r +
                                                         min(rank0 + 32 * b + sub, a.r - 1)) * a.K + k)
                               : zero;
#pragma unroll
        for (int n = 0; n < NB; ++n) acc[b][n] = T::mfma(df, xf[n], acc[b][n]);
      }
    }
  }

  // The waves' sums, added in wave order. A lane (row sub, half h) holds ranks 8g + 4h + i of a block.
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  v4f* part = (v4f*)ad_lds;  // [wave][block][g][lane]
#pragma unroll
  for (int b = 0; b < RB; ++b)
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        part[((wave * RB * NB + b * NB + n) * 4 + g) * 64 + lane] =
            (v4f){acc[b][n][4 * g], acc[b][n][4 * g + 1], acc[b][n][4 * g + 2], acc[b][n][4 * g + 3]};
  __syncthreads();
  constexpr int kSums = RB * NB * 256, kPer = (kSums + 64 * NW - 1) / (64 * NW);
  v4f sums[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = tid + i * 64 * NW;
    if (at < kSums) {
      sums[i] = part[at];
#pragma unroll
      for (int w = 1; w < NW; ++w) sums[i] += part[w * kSums + at];
    }
  }
  const bool join = a.splits > 1 || (T::kNarrow && gridDim.z > 1);
  constexpr int kPitch = 32 * RB + 4;
  float* u = (float*)ad_lds;
  float* plane = a.planes + ((int64_t)blockIdx.y * a.live_tiles + blockIdx.x) * a.tile_rows * a.r32;
  if (!join) __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int at = tid + i * 64 * NW;
    const int l = at & 63, g = (at >> 6) & 3, n = (at >> 8) % NB, b = (at >> 8) / NB;
    const int row = 32 * n + (l & 31), rank = 32 * b + 8 * g + 4 * (l >> 5);
    if (at >= kSums || rank0 + rank >= a.r32) continue;
    if (join) *(v4f*)(plane + row * a.r32 + rank0 + rank) = sums[i];
    else *(v4f*)(u + row * kPitch + rank) = sums[i];
  }
  if (join) return;
  __syncthreads();
  for (int row = tid >> 2; row < 32 * NB; row += 16 * NW)
    adapter_operands<T>(a, tile, blockIdx.x, u + row * kPitch, row, tid & 3, NB, rank0, min(rank0 + 32 * RB, a.r32));
}

// The K shares of a tile's u added in order, then into operand order. 256 threads.
template <class T>
__global__ __launch_bounds__(256) void adapter_join_kernel(AdapterArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char ad_lds[];
  float* u = (float*)ad_lds;
  const AdapterTile tile = a.tiles[blockIdx.x];
  const int per_row = a.r32 / 4;
  const int64_t plane = (int64_t)a.live_tiles * a.tile_rows * a.r32;
  const float* from = a.planes + (int64_t)blockIdx.x * a.tile_rows * a.r32;
  for (int i = threadIdx.x; i < a.tile_rows * per_row; i += 256) {
    v4f sum = *(const v4f*)(from + 4 * i);
    for (int s = 1; s < a.splits; ++s) sum += *(const v4f*)(from + s * plane + 4 * i);
    *(v4f*)(u + i / per_row * (a.r32 + 4) + i % per_row * 4) = sum;
  }
  __syncthreads();
  for (int row = threadIdx.x >> 2; row < a.tile_rows; row += 64)
    adapter_operands<T>(a, tile, blockIdx.x, u + row * (a.r32 + 4), row, threadIdx.x & 3, a.tile_rows / 32, 0,
                        a.r32);
}

constexpr int kAdUpThreads = 256;
constexpr int kAdUpPitch = 68;  // floats of a row of 64 columns in LDS: 16-byte accesses of 16 rows meet every bank once
constexpr int kAdSteps = 4;
constexpr int kAdUpStage = 16 * kAdUpPitch * 4;

// Row block blockIdx.x / col_groups (of a tile) and a group of its columns, neighbours in memory side by side in the
// launch; VEC: y and out take 16-byte accesses.
//
// A wave computes 32 rows x 64 columns transposed (the weight is the first operand), turns them in LDS, in fp32, and adds
// them to y in whole 128-byte lines of a row. y of the next 64 columns is on its way meanwhile. kAdSteps steps of 16 ranks
// have their weights in registers at once (two of them at rank 32: 380 -> 408 us). out is stored past the caches, y read past
// them where they do not hold it (58 MB: through them, 51 us against 55; 1 GB: past them, 526 against 537).
template <class T, bool VEC>
__global__ __launch_bounds__(kAdUpThreads, 3) void adapter_up_kernel(AdapterArgs a) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char ad_lds[];
  const int blocks = a.tile_rows / 32;
  const int row_block = blockIdx.x / a.col_groups, group = blockIdx.x - row_block * a.col_groups;
  const int tile_index = row_block / blocks, block = row_block - tile_index * blocks;
  const AdapterTile tile = a.tiles[tile_index];
  const int count = min(tile.count - 32 * block, 32);
  if (count <= 0 || (tile.adapter < 0 && a.in_place)) return;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, sub = lane & 31, half = lane >> 5;
  const int64_t n_blocks = (a.N + 63) / 64;
  const int64_t b_lo = (int64_t)group * a.blocks_per_wg;
  const int64_t b_hi = min(b_lo + a.blocks_per_wg, n_blocks);

  // This lane's rows of y and out: 8i + lane / 8, columns 8 (lane % 8) .. of 64.
  int64_t at[4];
  bool live[4];
  float factor[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 3);
    live[i] = r < count;
    at[i] = a.rows[tile.start + 32 * block + min(r, count - 1)];
    factor[i] = tile.adapter < 0 ? 0.0f : a.factors[(int64_t)tile_index * a.tile_rows + 32 * block + r];
  }
  const int col8 = 8 * (lane & 7);
  auto load_y = [&](int64_t blk, v4u* v) {
    const int64_t col = blk * 64 + col8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = (v4u){0, 0, 0, 0};
      if (VEC) {
        if (live[i] && blk < b_hi && col < a.N) {
          const v4u* from = (const v4u*)(a.y + at[i] * a.ldy + col);
          v[i] = a.stream_y ? __builtin_nontemporal_load(from) : *from;
        }
      } else if (live[i] && blk < b_hi) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < a.N) v[i][e >> 1] |= (uint32_t)a.y[at[i] * a.ldy + col + e] << (16 * (e & 1));
      }
    }
  };
  auto store = [&](int64_t blk, int i, v4u v) {
    const int64_t col = blk * 64 + col8;
    if (VEC) {
      if (live[i] && col < a.N) store_stream((v4i*)(a.out + at[i] * a.ldo + col), __builtin_bit_cast(v4i, v));
    } else if (live[i]) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < a.N) a.out[at[i] * a.ldo + col + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
    }
  };
  if (tile.adapter < 0) {
    for (int64_t blk = b_lo + wave; blk < b_hi; blk += 4) {
      v4u v[4];
      load_y(blk, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) store(blk, i, v[i]);
    }
    return;
  }
  v4u yv[4], yn[4];
  load_y(b_lo + wave, yn);
  const int steps = a.r32 / 16;
  v4u* operands = (v4u*)ad_lds;  // [step][leading, trailing][lane]
  {
    const v4u* from = a.frags + (int64_t)tile_index * steps * blocks * 128 + block * 128;
    for (int i = tid; i < steps * 128; i += kAdUpThreads) operands[i] = from[(int64_t)(i >> 7) * blocks * 128 + (i & 127)];
  }
  __syncthreads();
  float* turn = (float*)(ad_lds + steps * 2048 + wave * kAdUpStage);
  const uint16_t* up = a.up + (int64_t)tile.adapter * a.N * a.r;
#pragma unroll 1
  for (int64_t blk = b_lo + wave; blk < b_hi; blk += 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) yv[i] = yn[i];
    load_y(blk + 4, yn);
    v16f acc[2];
    acc[0] = acc[1] = (v16f){0};
#pragma unroll 1
    for (int s0 = 0; s0 < steps; s0 += kAdSteps) {
      v4u w[kAdSteps][2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const uint16_t* row = up + min(blk * 64 + 32 * b + sub, a.N - 1) * a.r + 8 * half + 16 * s0;
#pragma unroll
        for (int s = 0; s < kAdSteps; ++s)  // r is a multiple of 8: ranks past it are not read
          w[s][b] = 16 * (s0 + s) + 8 * half < a.r ? *(const v4u*)(row + 16 * s) : (v4u){0, 0, 0, 0};
      }
#pragma unroll
      for (int s = 0; s < kAdSteps; ++s) {
        if (s0 + s >= steps) break;
        const v4u lead = operands[(s0 + s) * 128 + lane], trail = operands[(s0 + s) * 128 + 64 + lane];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          acc[b] = T::mfma(w[s][b], lead, acc[b]);
          acc[b] = T::mfma(w[s][b], trail, acc[b]);
        }
      }
    }
    // Lane (row sub, half h) holds columns 32b + 8g + 4h + i; 16 rows at a time go through LDS.
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      if ((sub >> 4) == p) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *(v4f*)(turn + (sub & 15) * kAdUpPitch + 32 * b + 8 * g + 4 * half) =
                (v4f){acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]};
      }
      wave_lds_sync();
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int i = 2 * p + x;
        const v4f lo = *(const v4f*)(turn + (8 * x + (lane >> 3)) * kAdUpPitch + col8);
        const v4f hi = *(const v4f*)(turn + (8 * x + (lane >> 3)) * kAdUpPitch + col8 + 4);
        v4u o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d0 = e < 2 ? lo[2 * e] : hi[2 * e - 4], d1 = e < 2 ? lo[2 * e + 1] : hi[2 * e - 3];
          o[e] = T::pack(fmaf(d0, factor[i], T::lo(yv[i][e])), fmaf(d1, factor[i], T::hi(yv[i][e])));
        }
        store(blk, i, o);
      }
      wave_lds_sync();
    }
  }
}

}  // namespace hf
