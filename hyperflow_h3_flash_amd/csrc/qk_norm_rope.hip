// The norm of each query and key head and the rotation of its channels by the token's position, in one pass.
//
//   n = x * rsqrt(mean(x^2) + eps) * w;   (a, b) -> (a c - b s, a s + b c) for each pair of channels
//
// HBM-bound: each element is read once and written once, ~10 operations each. 37710 tokens x (56 + 56) heads of 128,
// three axes: 400 us for 2.16 GB, 5.4 TB/s (a copy of 1 GiB: 5.2).
//
// A row is one head of one token. LPR lanes share it (D / 16 of them at work), each with two chunks of 8 channels that
// lie half the rotary width apart, so that with either pair layout both channels of a pair are in one lane: halves pair
// chunk with chunk, interleaved pairs lie inside a chunk. Channels after the rotary width are taken two neighbouring
// chunks a lane. The sum of squares goes over LPR lanes by lane exchanges.
//
// A workgroup takes all query heads or all key heads (or a share of them, when there are few tokens) of a few tokens:
// their sines and cosines are computed once into LDS and serve every head. The angle is reduced in fp64 to less than
// half a turn before the sine: one fp64 product a token, side and pair. The rounding of that product and of the rate grows
// with the position: at 2^31 the angle of a pair that turns by 1 errs by 1e-7 (an ulp or two of the fp32 sine), at 2^40 by
// 7e-5, and int64 positions past 2^53 are rounded.
#pragma once

#include "block_types.h"

namespace hf {

constexpr int kRopeThreads = 256;

struct RopeSide {
  const uint16_t* x;
  uint16_t* out;
  const void* w;
  int64_t x_token, x_head, o_token, o_head;
  int heads, tokens, heads_per_wg, parts;  // tokens and heads of a workgroup, workgroups of a token
};

struct RopeArgs {
  RopeSide side[2];  // q, k
  const void* pos;
  int64_t ld_pos;
  const double* turns;
  const int32_t* axis;
  int64_t T;
  int pos_type, pairs, D, q_blocks, weight_f32;
  float eps;
};

__device__ __forceinline__ double rope_position(const RopeArgs& a, int64_t at) {
  if (a.pos_type == 0) return (double)((const int32_t*)a.pos)[at];
  if (a.pos_type == 1) return (double)((const int64_t*)a.pos)[at];
  return (double)((const float*)a.pos)[at];
}

// 8 weights from d on, in fp32.
template <class T>
__device__ __forceinline__ void rope_weights(const void* w, int d, bool f32, float* out) {
  if (f32) {
    const v4f a = *(const v4f*)((const float*)w + d), b = *(const v4f*)((const float*)w + d + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = a[e], out[4 + e] = b[e];
  } else {
    const v4u a = *(const v4u*)((const uint16_t*)w + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[2 * e] = T::lo(a[e]), out[2 * e + 1] = T::hi(a[e]);
  }
}

// The first q_blocks workgroups take the queries, the others the keys.
template <class T, int LPR, bool INTERLEAVED, bool NORM>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(RopeArgs a) {
  extern __shared__ v2f rope_table[];  // [tokens][pairs] of (cos, sin)
  const bool key = (int)blockIdx.x >= a.q_blocks;
  const RopeSide s = a.side[key];
  const int block = (int)blockIdx.x - (key ? a.q_blocks : 0), group = block / s.parts;
  const int h_lo = (block - group * s.parts) * s.heads_per_wg, nh = min(h_lo + s.heads_per_wg, s.heads) - h_lo;
  const int tid = threadIdx.x;
  const int64_t t0 = (int64_t)group * s.tokens;
  const int nt = (int)min((int64_t)s.tokens, a.T - t0);

  constexpr int kRows = kRopeThreads / LPR;
  const int lane = tid % LPR, row = tid / LPR;
  const int rotary_lanes = a.pairs / 8;
  const bool rotary = lane < rotary_lanes, active = lane < a.D / 16;
  // First channels of the lane's two chunks.
  const int c0 = rotary ? 8 * lane : 2 * a.pairs + 16 * (lane - rotary_lanes);
  const int c1 = rotary ? a.pairs + 8 * lane : c0 + 8;

  // Rows (t, h) of this side in order, kRows of them at a time; U of those rounds are on their way before the first is
  // used, the first ones before the table is made.
  constexpr int U = 4;
  const int rows = nt * nh;
  v4u in[U][2];
  int tt[U], hh[U];
  auto load = [&](int r0) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * kRows;
      tt[u] = r / nh;
      hh[u] = h_lo + (r - tt[u] * nh);
      in[u][0] = in[u][1] = (v4u){0, 0, 0, 0};
      if (r < rows && active) {
        const uint16_t* x = s.x + (t0 + tt[u]) * s.x_token + hh[u] * s.x_head;
        in[u][0] = *(const v4u*)(x + c0);
        in[u][1] = *(const v4u*)(x + c1);
      }
    }
  };
  load(row);
  float w[16];
  if (NORM) {
#pragma unroll
    for (int e = 0; e < 16; ++e) w[e] = 1.0f;
    if (active && s.w) {
      rope_weights<T>(s.w, c0, a.weight_f32, w);
      rope_weights<T>(s.w, c1, a.weight_f32, w + 8);
    }
  }
  for (int i = tid; i < nt * a.pairs; i += kRopeThreads) {
    const int t = i / a.pairs, p = i - t * a.pairs;
    const double turn = rope_position(a, (t0 + t) * a.ld_pos + a.axis[p]) * a.turns[p];
    const float part = (float)(turn - rint(turn));
    float sin, cos;
    sincospif(2.0f * part, &sin, &cos);
    rope_table[i] = (v2f){cos, sin};
  }
  __syncthreads();

  for (int r0 = row; r0 < rows; r0 += kRows * U) {
    if (r0 != row) load(r0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[2 * e] = T::lo(in[u][e / 4][e % 4]);
        x[2 * e + 1] = T::hi(in[u][e / 4][e % 4]);
      }
      if (NORM) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sum = fmaf(x[e], x[e], sum);
#pragma unroll
        for (int off = LPR / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
        const float r = 1.0f / sqrtf(sum / (float)a.D + a.eps);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = (x[e] * r) * w[e];
      }
      if (r0 + u * kRows >= rows || !active) continue;
      if (rotary) {
        const v2f* table = rope_table + tt[u] * a.pairs;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // Interleaved: pair e % 4 of chunk e / 4; halves: channel e of both chunks.
          const int p = INTERLEAVED ? (e < 4 ? c0 / 2 : c1 / 2 - 4) + e : c0 + e;
          const int i = INTERLEAVED ? 2 * e : e, j = INTERLEAVED ? 2 * e + 1 : e + 8;
          const v2f cs = table[p];
          const float x0 = x[i], x1 = x[j];
          x[i] = fmaf(x0, cs[0], -(x1 * cs[1]));
          x[j] = fmaf(x0, cs[1], x1 * cs[0]);
        }
      }
      uint16_t* o = s.out + (t0 + tt[u]) * s.o_token + hh[u] * s.o_head;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        v4u v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = T::pack(x[8 * c + 2 * e], x[8 * c + 2 * e + 1]);
        *(v4u*)(o + (c ? c1 : c0)) = v;
      }
    }
  }
}

}  // namespace hf
