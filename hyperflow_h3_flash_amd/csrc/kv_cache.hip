// Keys and values in pages of 4-bit codes: written, read back, and pages copied. The layout is hf_cache.h's.
#pragma once

#include "block_types.h"

namespace hf {

// Rows of one page: tokens first .. first + rows - 1 of the page are rows row0 .. of the packed tensors.
struct CacheSegment {
  int32_t page, first, rows, row0;
};

__host__ __device__ constexpr int kv_scale_bytes(int groups) { return groups == 3 ? 4 : groups; }
// Bytes of a page's tokens of one head.
__host__ __device__ constexpr int64_t kv_slab(int groups, int page) {
  return (int64_t)page * 2 * (16 * groups + kv_scale_bytes(groups));
}

struct CacheTypeBf16 {
  typedef Bf16 Type;
  static constexpr int kLeast = -125, kMost = 125;
};
struct CacheTypeFp16 {
  typedef Fp16 Type;
  static constexpr int kLeast = -23, kMost = 13;
};

// Two codes of byte `I` of a dword as a pair of the type, times 2^(exponent of scale): exact (all bytes and the exponents
// that are written were compared).
template <class T, int I>
__device__ __forceinline__ uint32_t kv_pair(uint32_t codes, float scale) {
  if constexpr (T::kNarrow) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, I));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, I));
}
template <class T>
__device__ __forceinline__ v4u kv_values(uint32_t codes, float scale) {
  return (v4u){kv_pair<T, 0>(codes, scale), kv_pair<T, 1>(codes, scale), kv_pair<T, 2>(codes, scale),
               kv_pair<T, 3>(codes, scale)};
}

struct CacheWriteArgs {
  const uint16_t* x[2];  // k, v
  int64_t token[2], head[2], page_bytes;
  unsigned char* cache;
  const CacheSegment* segments;
  int D, page;
};

constexpr int kCacheThreads = 256;

// Groups that a workgroup takes side by side, and the tokens of one round of it (fours of lanes over both).
constexpr int kv_side(int groups) { return groups == 3 ? 4 : groups; }
constexpr int kv_round(int groups) { return kCacheThreads / 4 / kv_side(groups); }

// HBM-bound, and short (8045 tokens, 8 heads of 128: written in 10.9 us, read back in 6.8, 3.9 and 6.2 TB/s from the caches and
// memory; with each load waited for by itself 13.8 and 11.2): a workgroup takes up to kCacheRounds rounds of a segment's tokens of one head, and every load of them
// is on its way before the first is used. Four lanes share a group of a token (16 bytes of input and 4 of codes each);
// neighbouring fours take neighbouring tokens, so that codes and scales go out side by side.
constexpr int kCacheRounds = 4;
template <class CT, int G>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(CacheWriteArgs a) {
  typedef typename CT::Type T;
  constexpr int S = kv_scale_bytes(G), kTokens = kv_round(G);
  const CacheSegment seg = a.segments[blockIdx.x];
  const int head = blockIdx.y, part = threadIdx.x & 3, four = threadIdx.x >> 2;
  const int g = four / kTokens, c = 32 * g + 8 * part;
  unsigned char* slab = a.cache + (int64_t)seg.page * a.page_bytes + head * kv_slab(G, a.page);
  for (int row0 = 0; row0 < seg.rows; row0 += kTokens * kCacheRounds) {
    v4u in[kCacheRounds][2];
#pragma unroll
    for (int i = 0; i < kCacheRounds; ++i) {
      const int row = row0 + i * kTokens + four % kTokens;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        in[i][which] = (v4u){0, 0, 0, 0};
        if (row < seg.rows && c < a.D)
          in[i][which] = *(const v4u*)(a.x[which] + (seg.row0 + (int64_t)row) * a.token[which] + head * a.head[which] + c);
      }
    }
#pragma unroll
    for (int i = 0; i < kCacheRounds; ++i) {
      const int row = row0 + i * kTokens + four % kTokens, at = seg.first + row;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        float h[8], top = 0.0f;
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          h[2 * e] = T::lo(in[i][which][e]);
          h[2 * e + 1] = T::hi(in[i][which][e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          top = fmaxf(top, __builtin_fabsf(h[e]));
          finite &= __builtin_fabsf(h[e]) < __builtin_inff();
        }
        top = finite ? top : __builtin_inff();
#pragma unroll
        for (int off = 1; off <= 2; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
        finite = top < __builtin_inff();
        // top = m 2^x with m in [0.5, 1): top <= 7 2^e from e = x - 3 on for m <= 7 / 8, else from x - 2.
        int x2;
        const float m = frexpf(finite ? top : 1.0f, &x2);
        const int e2 = min(max(x2 - (m <= 0.875f ? 3 : 2), CT::kLeast), CT::kMost);
        const float scale = __uint_as_float((uint32_t)(e2 + 127) << 23);
        // Nearest, ties to even, saturating: compared for every 16-bit float.
        uint32_t codes = 0;
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, h[0], h[1], scale, 0);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, h[2], h[3], scale, 1);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, h[4], h[5], scale, 2);
        codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, h[6], h[7], scale, 3);
        if (row >= seg.rows || g >= G) continue;
        *(uint32_t*)(slab + ((which * G + g) * a.page + at) * 16 + 4 * part) = finite ? codes : 0u;
        if (part == 0)
          slab[2 * G * a.page * 16 + (2 * at + which) * S + g] = finite ? (unsigned char)(e2 + 127) : 255;
      }
    }
  }
}

struct CacheReadArgs {
  const unsigned char* cache;
  uint16_t* out[2];  // k, v: [rows, heads, D]
  const CacheSegment* segments;
  int64_t page_bytes;
  int D, page, heads;
};

// As the writing, with lanes side by side over the channels of a token.
template <class CT, int G>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(CacheReadArgs a) {
  typedef typename CT::Type T;
  constexpr int S = kv_scale_bytes(G), kTokens = kv_round(G), kLanes = 4 * kv_side(G);
  const CacheSegment seg = a.segments[blockIdx.x];
  const int head = blockIdx.y, lane = threadIdx.x % kLanes, token = threadIdx.x / kLanes;
  const int g = lane >> 2, c = 8 * lane;
  if (c >= a.D) return;
  const unsigned char* slab = a.cache + (int64_t)seg.page * a.page_bytes + head * kv_slab(G, a.page);
  for (int row0 = 0; row0 < seg.rows; row0 += kTokens * kCacheRounds) {
    uint32_t codes[kCacheRounds][2], e[kCacheRounds][2];
#pragma unroll
    for (int i = 0; i < kCacheRounds; ++i) {
      const int row = row0 + i * kTokens + token, at = seg.first + min(row, seg.rows - 1);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        codes[i][which] = *(const uint32_t*)(slab + ((which * G + g) * a.page + at) * 16 + 4 * (lane & 3));
        e[i][which] = slab[2 * G * a.page * 16 + (2 * at + which) * S + g];
      }
    }
#pragma unroll
    for (int i = 0; i < kCacheRounds; ++i) {
      const int row = row0 + i * kTokens + token;
      if (row >= seg.rows) return;
#pragma unroll
      for (int which = 0; which < 2; ++which)  // a scale byte of 255 gives NaN
        *(v4u*)(a.out[which] + ((seg.row0 + (int64_t)row) * a.heads + head) * a.D + c) =
            kv_values<T>(codes[i][which], __uint_as_float(e[i][which] << 23));
    }
  }
}

// Copies are bound by memory (128 pages of 47 layers, 69 KB each: 166 us, 5.05 TB/s; 16 KB a workgroup). Pages of a launch, with
// their numbers among its parameters: nothing to upload, and nothing that a captured graph would
// have to keep.
constexpr int kCopyPairs = 256;
struct CopyArgs {
  unsigned char* pool;
  int64_t layer_bytes, page_bytes;
  int32_t src[kCopyPairs], dst[kCopyPairs];
};
constexpr int kCopyBytes = kCacheThreads * 16 * 4;  // of a workgroup

__global__ __launch_bounds__(kCacheThreads) void copy_pages_kernel(CopyArgs a) {
  const int64_t at = (int64_t)blockIdx.x * kCopyBytes;
  unsigned char* layer = a.pool + (int64_t)blockIdx.z * a.layer_bytes;
  const unsigned char* from = layer + (int64_t)a.src[blockIdx.y] * a.page_bytes;
  unsigned char* to = layer + (int64_t)a.dst[blockIdx.y] * a.page_bytes;
  v4u v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = at + (i * kCacheThreads + threadIdx.x) * 16;
    if (o < a.page_bytes) v[i] = *(const v4u*)(from + o);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t o = at + (i * kCacheThreads + threadIdx.x) * 16;
    if (o < a.page_bytes) *(v4u*)(to + o) = v[i];
  }
}

}  // namespace hf
