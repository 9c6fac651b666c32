// The norms after and before a block with its gate and residual, in one pass:
//
//   r = residual x + gate P(y),   n = N(r) w (1 + scale) + shift
//
// HBM-bound: each element of x and y is read once, of r and n written once. A row stays in the registers of its waves from
// the first read to the last write, up to NV chunks of 8 channels a lane (rows above 12288 channels with fp32 vectors nearly:
// their sixteen waves have 128 registers each, and 4 of a lane's, 12 with x in fp32, go through scratch memory). The sums of its
// norms go over the lanes by exchanges between registers and over the waves through LDS. Variances are sums of squared
// differences from the mean, not differences of sums: a row far from zero keeps its digits.
//
// Every load of a row is on its way before the first sum, the vectors' among them (from the caches), through descriptors of
// the row: past its end loads give zero and stores nothing, and what is absent has a descriptor of no bytes, so there is no
// condition to wait at. What hides the rest of a row's way is other rows on the same compute unit. 37710 rows of 5376, a
// layer norm with gate, scale and shift, us: this 278, with the vectors loaded where they are used 432; teams of waves that
// take rows one behind the other with the next row's loads on their way 377 (fewer waves for more registers), the same with
// the vectors held in registers no better; sums by exchanges through LDS 380 against 377. Six waves of two chunks 343, three
// of four 310, two of six 389.
// Norms before and after with weights and modulation, by width and the vectors' type, 1.6 GB of bfloat16 x, y, r and n, TB/s:
// 5376 5.2 and 4.6 (fp32 vectors: more loads from the L2 for the same rows), 8192 4.8 and 3.7, 12288 5.1 and 4.1, 16384 4.2 and
// 3.3; with x and r in fp32 5.3 and 4.7, 5.5 and 4.3, 5.1 and 4.5, 5.2 and 3.3.
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
  int64_t t0, T;  // rows of this launch: t0 .. T - 1
  int C, post, norm, per_row, stream;
  float residual, eps;
};

// A row's descriptor: C values from `row` on of the type or in fp32; nothing where p is NULL.
template <bool F32>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t norm_row(const void* p, int64_t row, int C) {
  return make_rsrc((const unsigned char*)p + row * (F32 ? 4 : 2), p ? (uint32_t)C * (F32 ? 4u : 2u) : 0u);
}

// 8 values as they lie in memory: of the type, or in fp32.
template <bool F32>
struct NormRaw {
  v4u v[F32 ? 2 : 1];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t row, uint32_t c) {
    v[0] = __builtin_amdgcn_raw_buffer_load_b128(row, c * (F32 ? 4u : 2u), 0, 0);
    if constexpr (F32) v[1] = __builtin_amdgcn_raw_buffer_load_b128(row, c * 4u + 16u, 0, 0);
  }
  template <class T>
  __device__ __forceinline__ void values(float* out) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (F32) out[e] = __uint_as_float(v[0][e]), out[4 + e] = __uint_as_float(v[1][e]);
      else out[2 * e] = T::lo(v[0][e]), out[2 * e + 1] = T::hi(v[0][e]);
    }
  }
};

// 8 results; those that the Infinity Cache would not hold until they are read go past it.
template <class T, bool F32>
__device__ __forceinline__ void norm_store(__amdgpu_buffer_rsrc_t row, uint32_t c, const float* v, bool stream) {
  constexpr int kStream = 2;  // non-temporal
  if constexpr (F32) {
    const v4u a = __builtin_bit_cast(v4u, (v4f){v[0], v[1], v[2], v[3]});
    const v4u b = __builtin_bit_cast(v4u, (v4f){v[4], v[5], v[6], v[7]});
    if (stream) {
      __builtin_amdgcn_raw_buffer_store_b128(a, row, c * 4u, 0, kStream);
      __builtin_amdgcn_raw_buffer_store_b128(b, row, c * 4u + 16u, 0, kStream);
    } else {
      __builtin_amdgcn_raw_buffer_store_b128(a, row, c * 4u, 0, 0);
      __builtin_amdgcn_raw_buffer_store_b128(b, row, c * 4u + 16u, 0, 0);
    }
  } else {
    const v4u a = {T::pack(v[0], v[1]), T::pack(v[2], v[3]), T::pack(v[4], v[5]), T::pack(v[6], v[7])};
    if (stream) __builtin_amdgcn_raw_buffer_store_b128(a, row, c * 2u, 0, kStream);
    else __builtin_amdgcn_raw_buffer_store_b128(a, row, c * 2u, 0, 0);
  }
}

// The sum over a wave: within rows of 16 lanes by lane permutations of the additions' operands, then over the four rows.
template <int CTRL>
__device__ __forceinline__ float norm_add(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float norm_wave_sum(float v) {
  v = norm_add<0xb1>(v);   // lane ^ 1
  v = norm_add<0x4e>(v);   // lane ^ 2
  v = norm_add<0x141>(v);  // mirrored in 8: the other four
  v = norm_add<0x140>(v);  // mirrored in 16: the other eight
  return quad_sum(v);
}

// Waves of a workgroup: rows of one wave each share one.
__host__ __device__ constexpr int norm_waves(int w) { return w == 1 ? 4 : w; }

// W waves a row, NV chunks of 8 channels a lane. WIDE: x and r in fp32; VF32: the vectors; Y: there is a branch to add.
template <class T, bool WIDE, bool VF32, bool Y, int W, int NV>
__global__ __launch_bounds__(64 * norm_waves(W)) void residual_norm_kernel(NormArgs a) {
  constexpr int kRows = norm_waves(W) / W;
  __shared__ float partial[2][W];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t t = a.t0 + (int64_t)blockIdx.x * kRows + wave / W;
  if (t >= a.T) return;  // a whole workgroup where rows have several waves
  const uint32_t first = (wave % W) * 64 + lane;
  auto channel = [&](int i) __attribute__((always_inline)) { return 8 * (first + 64 * W * i); };
  int turn = 0;
  // A sum over the row, in a fixed order.
  auto sum = [&](float v) __attribute__((always_inline)) {
    v = norm_wave_sum(v);
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
  // h minus its mean (kind 2); returns the factor of the norm.
  auto norm_of = [&](float (&h)[NV][8], int kind) __attribute__((always_inline)) {
    if (kind == 0) return 1.0f;
    if (kind == 2) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += h[i][e];
      const float mean = sum(s) / size;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] = channel(i) < (uint32_t)a.C ? h[i][e] - mean : 0.0f;
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(h[i][e], h[i][e], s);
    return 1.0f / sqrtf(sum(s) / size + a.eps);
  };

  NormRaw<WIDE> x[NV];
  NormRaw<false> y[NV];
  NormRaw<VF32> gate[NV], post_weight[NV], weight[NV], scale[NV], shift[NV];
  const int64_t g = a.group ? a.group[t] : a.per_row ? t : 0;
  {
    const auto xr = norm_row<WIDE>(a.x, t * a.ldx, a.C);
    const auto yr = norm_row<false>(a.y, t * a.ldy, a.C);
    const auto gr = norm_row<VF32>(a.gate, g * a.ld_gate, a.C), pr = norm_row<VF32>(a.post_weight, 0, a.C);
    const auto wr = norm_row<VF32>(a.weight, 0, a.C), sr = norm_row<VF32>(a.scale, g * a.ld_scale, a.C);
    const auto hr = norm_row<VF32>(a.shift, g * a.ld_shift, a.C);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i].load(xr, channel(i));
      if constexpr (Y) y[i].load(yr, channel(i));
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if constexpr (Y) {
        gate[i].load(gr, channel(i));
        post_weight[i].load(pr, channel(i));
      }
      weight[i].load(wr, channel(i));
      scale[i].load(sr, channel(i));
      shift[i].load(hr, channel(i));
    }
  }
  float h[NV][8];
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i].template values<T>(h[i]);
  if constexpr (Y) {
    float b[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) y[i].template values<T>(b[i]);
    const float f = norm_of(b, a.post);
    const auto rr = norm_row<WIDE>(a.r, t * a.ldr, a.C);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float p[8], q[8];
      post_weight[i].template values<T>(p);
      gate[i].template values<T>(q);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v = b[i][e] * f;
        if (a.post_weight) v *= p[e];
        if (a.gate) v *= q[e];
        h[i][e] = fmaf(a.residual, h[i][e], v);
      }
      norm_store<T, WIDE>(rr, channel(i), h[i], a.stream);
    }
  }
  const float f = norm_of(h, a.norm);
  const auto nr = norm_row<false>(a.n, t * a.ldn, a.C);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float w[8], s[8], d[8];
    weight[i].template values<T>(w);
    scale[i].template values<T>(s);
    shift[i].template values<T>(d);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = h[i][e] * f;
      if (a.weight) v *= w[e];
      h[i][e] = fmaf(v, 1.0f + s[e], d[e]);
    }
    norm_store<T, false>(nr, channel(i), h[i], a.stream);
  }
}

}  // namespace hf
