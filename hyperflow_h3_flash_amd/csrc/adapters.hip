// Low-rank adapters of many requests beside a shared projection: out[m] = y[m] + scale_a (x[m] A_a^T) B_a^T, a the
// adapter of row m, or out[m] = y[m] where it has none.
//
// HBM-bound with many rows (x once, y once, out once; the adapters' weights stay in the L2s), latency-bound with few.
//
// The plan holds the rows sorted by adapter and cut into tiles of at most 64 rows of one adapter, so requests in any
// order and rows of one adapter that lie apart share a tile; rows are read and written where they lie.
//   adapter_down_kernel  u = x A^T, fp32: a workgroup a tile and a share of K, its four waves on every fourth 64 k.
//   adapter_up_kernel    out = y + scale (u B^T): a workgroup a tile and a range of columns.
// u goes through a fp32 workspace, one plane per share of K (joined in a fixed order, no atomics). For the second
// product each u is split into a leading and a trailing 16-bit value (x A^T is not rounded to 16 bits: the doubled
// rank costs nothing where memory is the bound), after a power-of-two scale of its row that keeps fp16 in range.
#pragma once

#include "block_types.h"

namespace hf {

constexpr int kAdThreads = 256;
constexpr int kAdRows = 64;  // rows of a tile
constexpr int kAdChunk = 64;  // K of one step

struct AdapterTile {
  int32_t adapter, start, count, pad;
};

struct AdapterArgs {
  const uint16_t *x, *y, *down, *up;
  const float* scale;
  uint16_t* out;
  float* u;  // [splits][rows][r32]
  const AdapterTile* tiles;
  const int32_t* rows;
  int64_t ldx, ldy, ldo, K, N, n_rows;
  int r, r32, splits, chunks_per_split, blocks_per_wg, in_place;
};

// RB rank blocks of 32 from blockIdx.z * 32 RB on, rows blockIdx.x's tile, K share blockIdx.y.
template <class T, int RB>
__global__ __launch_bounds__(kAdThreads) void adapter_down_kernel(AdapterArgs a) {
  __shared__ v4f part[4][4][64];  // one 32 x 32 block of each wave
  const AdapterTile tile = a.tiles[blockIdx.x];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, sub = lane & 31, half = lane >> 5;
  const int rank0 = blockIdx.z * 32 * RB;
  const bool two = tile.count > 32;
  const uint16_t* xr[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int i = min(n * 32 + sub, tile.count - 1);  // a row past the tile repeats its last one: not stored
    xr[n] = a.x + (int64_t)a.rows[tile.start + i] * a.ldx + 32 * half;
  }
  const uint16_t* dr[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int j = min(rank0 + 32 * b + sub, a.r - 1);  // likewise
    dr[b] = a.down + ((int64_t)tile.adapter * a.r + j) * a.K + 32 * half;
  }
  v16f acc[RB][2];
#pragma unroll
  for (int b = 0; b < RB; ++b) acc[b][0] = acc[b][1] = (v16f){0};
  const int64_t chunks = (a.K + kAdChunk - 1) / kAdChunk;
  const int64_t c_lo = (int64_t)blockIdx.y * a.chunks_per_split;
  const int64_t c_hi = min(c_lo + a.chunks_per_split, chunks);
  const v4u zero = {0, 0, 0, 0};
  // Lane half h holds k 32h .. 32h + 31 of the chunk in both operands: 64 contiguous bytes a lane, a whole line a row.
  for (int64_t c = c_lo + wave; c < c_hi; c += 4) {
    const int64_t k0 = c * kAdChunk;
    v4u xv[2][4], dv[RB][4];
    if (k0 + kAdChunk <= a.K) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        xv[0][s] = *(const v4u*)(xr[0] + k0 + 8 * s);
        xv[1][s] = two ? *(const v4u*)(xr[1] + k0 + 8 * s) : zero;
      }
#pragma unroll
      for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int s = 0; s < 4; ++s) dv[b][s] = *(const v4u*)(dr[b] + k0 + 8 * s);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bool in = k0 + 32 * half + 8 * s < a.K;
        xv[0][s] = in ? *(const v4u*)(xr[0] + k0 + 8 * s) : zero;
        xv[1][s] = in && two ? *(const v4u*)(xr[1] + k0 + 8 * s) : zero;
#pragma unroll
        for (int b = 0; b < RB; ++b) dv[b][s] = in ? *(const v4u*)(dr[b] + k0 + 8 * s) : zero;
      }
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        acc[b][0] = T::mfma(dv[b][s], xv[0][s], acc[b][0]);
        if (two) acc[b][1] = T::mfma(dv[b][s], xv[1][s], acc[b][1]);
      }
  }
  // Lane (row sub, half h) of a block holds ranks 8g + 4h + i. The waves' blocks are added in wave order; thread
  // (g = wave, lane) adds and stores value group g.
  float* u = a.u + (int64_t)blockIdx.y * a.n_rows * a.r32;
#pragma unroll
  for (int b = 0; b < RB; ++b) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (n && !two) break;
      __syncthreads();
#pragma unroll
      for (int g = 0; g < 4; ++g)
        part[wave][g][lane] = (v4f){acc[b][n][4 * g], acc[b][n][4 * g + 1], acc[b][n][4 * g + 2], acc[b][n][4 * g + 3]};
      __syncthreads();
      const v4f sum = ((part[0][wave][lane] + part[1][wave][lane]) + part[2][wave][lane]) + part[3][wave][lane];
      const int i = n * 32 + sub, rank = rank0 + 32 * b + 8 * wave + 4 * half;
      if (i < tile.count && rank < a.r32) *(v4f*)(u + (int64_t)(tile.start + i) * a.r32 + rank) = sum;
    }
  }
}

// Sum over the K shares of 8 ranks of u.
__device__ __forceinline__ void adapter_u8(const AdapterArgs& a, int64_t row, int rank, float out[8]) {
  const float* p = a.u + row * a.r32 + rank;
  v4f s0 = *(const v4f*)p, s1 = *(const v4f*)(p + 4);
  for (int i = 1; i < a.splits; ++i) {
    p += a.n_rows * a.r32;
    s0 += *(const v4f*)p;
    s1 += *(const v4f*)(p + 4);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    out[e] = rank + e < a.r ? s0[e] : 0.0f;
    out[4 + e] = rank + 4 + e < a.r ? s1[e] : 0.0f;
  }
}

// VEC: y and out take 16-byte accesses.
template <class T, bool VEC>
__global__ __launch_bounds__(kAdThreads) void adapter_up_kernel(AdapterArgs a) {
  extern __shared__ v4u ad_lds[];  // u in operand order: [k step][row block][leading, trailing][lane]
  __shared__ float row_scale[kAdRows];
  const AdapterTile tile = a.tiles[blockIdx.x];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, sub = lane & 31, half = lane >> 5;
  const int64_t n_blocks = (a.N + 63) / 64;
  const int64_t b_lo = (int64_t)blockIdx.y * a.blocks_per_wg;
  const int64_t b_hi = min(b_lo + a.blocks_per_wg, n_blocks);
  if (tile.adapter < 0) {
    if (a.in_place) return;
    const int64_t n0 = b_lo * 64, n1 = min(b_hi * 64, a.N);
    constexpr int E = VEC ? 8 : 1;
    const int64_t per_row = (n1 - n0) / E;
    for (int64_t i = tid; i < per_row * tile.count; i += kAdThreads) {
      const int64_t row = a.rows[tile.start + i / per_row], n = n0 + i % per_row * E;
      if (VEC) {
        *(v4u*)(a.out + row * a.ldo + n) = *(const v4u*)(a.y + row * a.ldy + n);
      } else {
        a.out[row * a.ldo + n] = a.y[row * a.ldy + n];
      }
    }
    return;
  }
  const float scale = a.scale ? a.scale[tile.adapter] : 1.0f;
  const int steps = a.r32 / 16;
  {
    // Thread (row tid / 4, part tid % 4): the row's largest |u|, then its ranks 8 at a time into operand order.
    const int row = tid >> 2, part = tid & 3;
    const bool live = row < tile.count;
    float most = 0.0f;
    for (int j = part; j < a.r32 / 8; j += 4) {
      float v[8];
      if (live) {
        adapter_u8(a, tile.start + row, 8 * j, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
      }
    }
    most = fmaxf(most, __shfl_xor(most, 1, 64));
    most = fmaxf(most, __shfl_xor(most, 2, 64));
    // 2^(6 - exponent): the row's largest lands in [2^6, 2^7), where fp16 holds it and its trailing part is normal.
    const bool fine = most >= 0x1p-100f && most <= 0x1p100f;
    const float grow = fine ? __uint_as_float((uint32_t)(127 + 6 + 127 - (int)(__float_as_uint(most) >> 23)) << 23) : 1.0f;
    if (part == 0) row_scale[row] = scale / grow;  // exact up to scale's own rounding: a power of two
    for (int j = part; j < a.r32 / 8; j += 4) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.0f;
      if (live) adapter_u8(a, tile.start + row, 8 * j, v);
      v4u lead, trail;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = v[2 * e] * grow, q = v[2 * e + 1] * grow;
        lead[e] = T::pack(p, q);
        const float p1 = T::lo(lead[e]), q1 = T::hi(lead[e]);
        // An infinity or NaN has no trailing part.
        trail[e] = T::pack(fabsf(p1) < __builtin_inff() ? p - p1 : 0.0f, fabsf(q1) < __builtin_inff() ? q - q1 : 0.0f);
      }
      v4u* to = ad_lds + ((j >> 1) * 2 + (row >> 5)) * 128 + (j & 1) * 32 + (row & 31);
      to[0] = lead;
      to[64] = trail;
    }
  }
  __syncthreads();
  const bool two = tile.count > 32;
  // Output column of operand row m = 8g + 4h + i of column block b: 64 * block + 32h + 16b + 4g + i, so that a lane
  // (row sub, half h) ends with 32 neighbouring columns: 64 bytes, and a row's two lanes a whole line.
  const int col_of_sub = ((sub >> 2) & 1) * 32 + (sub >> 3) * 4 + (sub & 3);
  int64_t at[2];
  bool live[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    live[n] = n * 32 + sub < tile.count;
    at[n] = a.rows[tile.start + min(n * 32 + sub, tile.count - 1)];
  }
  const float f[2] = {row_scale[sub], row_scale[32 + sub]};
  const uint16_t* up = a.up + (int64_t)tile.adapter * a.N * a.r;
  for (int64_t blk = b_lo + wave; blk < b_hi; blk += 4) {
    const int64_t n0 = blk * 64;
    const int64_t col = n0 + 32 * half;  // this lane's first output column
    v4u yv[2][4];
    if (VEC) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          yv[n][c] = live[n] && col + 8 * c < a.N ? *(const v4u*)(a.y + at[n] * a.ldy + col + 8 * c) : (v4u){0, 0, 0, 0};
    }
    v16f acc[2][2];
#pragma unroll
    for (int b = 0; b < 2; ++b) acc[b][0] = acc[b][1] = (v16f){0};
    const uint16_t* ur[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) ur[b] = up + min(n0 + 16 * b + col_of_sub, a.N - 1) * a.r + 8 * half;
    for (int s = 0; s < steps; ++s) {
      v4u w[2];
      const bool in = 16 * s + 8 * half < a.r;  // r is a multiple of 8: ranks past it are not read
#pragma unroll
      for (int b = 0; b < 2; ++b) w[b] = in ? *(const v4u*)(ur[b] + 16 * s) : (v4u){0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        if (n && !two) break;
        const v4u lead = ad_lds[(s * 2 + n) * 128 + lane], trail = ad_lds[(s * 2 + n) * 128 + 64 + lane];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          acc[b][n] = T::mfma(w[b], lead, acc[b][n]);
          acc[b][n] = T::mfma(w[b], trail, acc[b][n]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (!live[n]) continue;
      if (VEC) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          v4u o;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int v = 8 * (c & 1) + 2 * e;
            o[e] = T::pack(fmaf(acc[c >> 1][n][v], f[n], T::lo(yv[n][c][e])),
                           fmaf(acc[c >> 1][n][v + 1], f[n], T::hi(yv[n][c][e])));
          }
          if (col + 8 * c < a.N) *(v4u*)(a.out + at[n] * a.ldo + col + 8 * c) = o;
        }
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const int64_t j = col + c;
          if (j < a.N)
            a.out[at[n] * a.ldo + j] =
                (uint16_t)T::pack(fmaf(acc[c >> 4][n][c & 15], f[n], T::lo(a.y[at[n] * a.ldy + j])), 0.0f);
        }
      }
    }
  }
}

}  // namespace hf
