// The norms after and before a block with its gate and residual, in one pass:
//
//   r = residual x + gate P(y),   n = N(r) w (1 + scale) + shift
//
// HBM-bound: each element of x and y is read once, of r and n written once. A row stays in the registers of its waves from
// the first read to the last write, up to NV chunks of 8 channels a lane; the sums of its norms go over the lanes by
// exchanges and over the waves through LDS. Variances are sums of squared differences from the mean, not differences of
// sums: a row far from zero keeps its digits.
#pragma once

#include "block_types.h"

namespace hf {

struct NormArgs {
  const void* x;
  const uint16_t* y;
  void* r;
  uint16_t* n;
  const void *gate, *scale, *shift, *post_weight, *weight;
  const int32_t* group;
  int64_t ldx, ldy, ldr, ldn, ld_gate, ld_scale, ld_shift;
  int64_t T;
  int C, post, norm, per_row, vectors_f32;
  float residual, eps;
};

// 8 values from `at` on, of the type or in fp32.
template <class T>
__device__ __forceinline__ void norm_load(const void* p, int64_t at, bool f32, float* out) {
  if (f32) {
    const v4f a = *(const v4f*)((const float*)p + at), b = *(const v4f*)((const float*)p + at + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = a[e], out[4 + e] = b[e];
  } else {
    const v4u a = *(const v4u*)((const uint16_t*)p + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) out[2 * e] = T::lo(a[e]), out[2 * e + 1] = T::hi(a[e]);
  }
}

template <class T>
__device__ __forceinline__ void norm_store(void* p, int64_t at, bool f32, const float* v) {
  if (f32) {
    *(v4f*)((float*)p + at) = (v4f){v[0], v[1], v[2], v[3]};
    *(v4f*)((float*)p + at + 4) = (v4f){v[4], v[5], v[6], v[7]};
  } else {
    *(v4u*)((uint16_t*)p + at) =
        (v4u){T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]), T::pack(v[6], v[7])};
  }
}

// W waves a row; a workgroup has max(4, W) waves.
template <class T, bool WIDE, int W, int NV>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256) void residual_norm_kernel(NormArgs a) {
  constexpr int kRows = W > 4 ? 1 : 4 / W;
  __shared__ float partial[2][8];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * kRows + wave / W;
  if (W == 1 && t >= a.T) return;  // with more waves a row there is one row a workgroup
  const int first = (wave % W) * 64 + lane;
  int turn = 0;
  // A sum over the row, in a fixed order.
  auto sum = [&](float v) __attribute__((always_inline)) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    if constexpr (W > 1) {
      if (lane == 0) partial[turn][wave] = v;
      __syncthreads();
      v = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) v += partial[turn][w];
      turn ^= 1;  // the next sum writes the other half: a wave may be ahead by one
    }
    return v;
  };
  const float size = (float)a.C;
  auto normed = [&](float (&h)[NV][8], int kind) __attribute__((always_inline)) {
    if (kind == 0) return;
    if (kind == 2) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += h[i][e];
      const float mean = sum(s) / size;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (8 * (first + 64 * W * i) < a.C)
#pragma unroll
          for (int e = 0; e < 8; ++e) h[i][e] -= mean;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(h[i][e], h[i][e], s);
    const float f = 1.0f / sqrtf(sum(s) / size + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] *= f;
  };

  const int64_t g = a.group ? a.group[t] : a.per_row ? t : 0;
  float h[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (first + 64 * W * i);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[i][e] = 0.0f;
    if (c < a.C) norm_load<T>(a.x, t * a.ldx + c, WIDE, h[i]);
  }
  if (a.y) {
    float b[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (first + 64 * W * i);
#pragma unroll
      for (int e = 0; e < 8; ++e) b[i][e] = 0.0f;
      if (c < a.C) norm_load<T>(a.y, t * a.ldy + c, false, b[i]);
    }
    normed(b, a.post);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = 8 * (first + 64 * W * i);
      if (c >= a.C) continue;
      float w[8];
      if (a.post_weight) {
        norm_load<T>(a.post_weight, c, a.vectors_f32, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) b[i][e] *= w[e];
      }
      if (a.gate) {
        norm_load<T>(a.gate, g * a.ld_gate + c, a.vectors_f32, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) b[i][e] *= w[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] = fmaf(a.residual, h[i][e], b[i][e]);
      norm_store<T>(a.r, t * a.ldr + c, WIDE, h[i]);
    }
  }
  if (!a.n) return;
  normed(h, a.norm);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = 8 * (first + 64 * W * i);
    if (c >= a.C) continue;
    float w[8];
    if (a.weight) {
      norm_load<T>(a.weight, c, a.vectors_f32, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] *= w[e];
    }
    if (a.scale) {
      norm_load<T>(a.scale, g * a.ld_scale + c, a.vectors_f32, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] *= 1.0f + w[e];
    }
    if (a.shift) {
      norm_load<T>(a.shift, g * a.ld_shift + c, a.vectors_f32, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[i][e] += w[e];
    }
    norm_store<T>(a.n, t * a.ldn + c, false, h[i]);
  }
}

}  // namespace hf
