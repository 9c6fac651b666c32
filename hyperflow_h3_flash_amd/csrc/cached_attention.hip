// Attention of few rows over keys and values in pages of 4-bit codes (kv_cache.hip).
//
// Rows, items and the running maximum and sum are those of attention.hip: a row is a (token, head of the group) pair, here
// up to 32 of them a workgroup, and scores are computed transposed. The four waves of a workgroup take the item's blocks of
// 32 keys in turn, each with sums of its own, and join them at the end through LDS.
//
// Operands. Codes go from memory to registers, 16 bytes (a group of 32 channels of a key) a lane: for the scores that is
// already the order of the first product's operand, four steps of 8 channels a lane, when the queries' channels are taken in
// the same order; codes become values of the type two at a time with the group's scale (exact). Values are turned
// into the second product's operand through LDS, by wave: written by key, read transposed, as in attention.hip.
#pragma once

#include "attention.hip"
#include "kv_cache.hip"

namespace hf {

constexpr int kCaRows = 32, kCaWaves = 4, kCaKeys = 32;

struct CachedItem {
  int32_t q0, nq, nk, row0, key_lo, key_hi, head, slot, table0, pad[3];
};
struct CachedJoin {
  int32_t q0, nq, nk, row0, head, slot0, slots, rows;
};

struct CachedArgs {
  const uint16_t* q;
  uint16_t* out;
  const unsigned char* cache;
  float* ws;
  const CachedItem* items;
  const CachedJoin* joins;
  const int32_t* tables;
  int64_t q_token, q_head, o_token, o_head, page_bytes;
  int group, D, causal, page;
  float scale_log2, lift;
};

// Floats of a workspace tile: O [kCaRows][32 G], then m and l per row.
__host__ __device__ constexpr int ca_slot_floats(int groups) { return kCaRows * (32 * groups + 2); }
__host__ __device__ constexpr int ca_pitch(int groups) { return groups > 2 ? 256 : 128; }
// LDS: a wave's values of a block; two waves' sums at the end; each row's maximum and sum by wave.
__host__ __device__ constexpr int ca_lds(int groups) {
  return kCaWaves * kCaKeys * ca_pitch(groups) > 2 * 4096 * groups ? kCaWaves * kCaKeys * ca_pitch(groups)
                                                                   : 2 * 4096 * groups;
}

template <class T, int G>
__global__ __launch_bounds__(64 * kCaWaves) void cached_rows_kernel(CachedArgs a) {
  constexpr int G2 = (G + 1) / 2, S = kv_scale_bytes(G), PITCH = ca_pitch(G);
  __shared__ __attribute__((aligned(1024))) unsigned char ca_mem[ca_lds(G)];
  __shared__ v2f ca_stat[kCaWaves][kCaRows];
  const CachedItem it = a.items[blockIdx.x];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int sub = lane & 31, half = lane >> 5;

  const int64_t row = (int64_t)it.row0 + sub;
  const bool live = row < (int64_t)it.nq * a.group;
  const int token = live ? (int)((uint32_t)row / (uint32_t)a.group) : 0;
  const int head = it.head * a.group + (live ? (int)(row - (int64_t)token * a.group) : 0);
  const int last = live ? (a.causal ? min(token + it.nk - it.nq, it.nk - 1) : it.nk - 1) : -1;
  const int first_last = __builtin_amdgcn_readfirstlane(last);  // the first row sees the fewest keys

  // Queries in the order of the codes: step (i, w) takes channels 32 (2 i + half) + 8 w ..
  v4u qf[G2][4];
  {
    const uint16_t* q = a.q + (it.q0 + (int64_t)token) * a.q_token + head * a.q_head;
#pragma unroll
    for (int i = 0; i < G2; ++i)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int c = 32 * (2 * i + half) + 8 * w;
        qf[i][w] = live && c < a.D ? *(const v4u*)(q + c) : (v4u){0, 0, 0, 0};
      }
  }

  struct Block {
    v4u k[G2], v[G2];
    uint32_t ks, vs;
  };
  const int page_shift = 31 - __builtin_clz(a.page);
  const int64_t slab_bytes = kv_slab(G, a.page);
  auto load = [&](int key0, Block& b) __attribute__((always_inline)) {
    const int page = a.tables[it.table0 + (key0 >> page_shift)];
    const unsigned char* slab = a.cache + (int64_t)page * a.page_bytes + it.head * slab_bytes;
    const int at = (key0 & (a.page - 1)) + sub;
#pragma unroll
    for (int i = 0; i < G2; ++i) {
      const int g = min(2 * i + half, G - 1);
      b.k[i] = *(const v4u*)(slab + ((int64_t)g * a.page + at) * 16);
      b.v[i] = *(const v4u*)(slab + ((int64_t)(G + g) * a.page + at) * 16);
    }
    const unsigned char* scales = slab + (int64_t)2 * G * a.page * 16 + at * S;
    if constexpr (S == 4) {
      b.ks = *(const uint32_t*)scales;
      b.vs = *(const uint32_t*)(scales + (int64_t)a.page * S);
    } else if constexpr (S == 2) {
      b.ks = *(const uint16_t*)scales;
      b.vs = *(const uint16_t*)(scales + (int64_t)a.page * S);
    } else {
      b.ks = *scales;
      b.vs = *(scales + (int64_t)a.page * S);
    }
  };
  auto scale_of = [&](uint32_t scales, int i) __attribute__((always_inline)) {
    const int g = min(2 * i + half, G - 1);
    return __uint_as_float(((scales >> (8 * g)) & 255u) << 23);
  };
  auto any_nan = [&](uint32_t scales) __attribute__((always_inline)) {
    bool bad = false;
#pragma unroll
    for (int g = 0; g < G; ++g) bad |= ((scales >> (8 * g)) & 255u) == 255u;
    return bad;
  };

  unsigned char HF_LDS* tile = (unsigned char HF_LDS*)ca_mem + wave * kCaKeys * PITCH;
  uint32_t vaddr;
  {
    const int r = 4 * half + ((lane & 15) >> 2), ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    vaddr = (uint32_t)(r * PITCH + ((ch ^ at_swizzle<PITCH>(r)) * 16) + (lane & 1) * 8);
  }
  auto vfrag = [&](int ks, int d) __attribute__((always_inline)) {
    typedef short v8s __attribute__((ext_vector_type(8)));
    const unsigned char HF_LDS* at = tile + ks * 16 * PITCH;
    const v4s f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(at + (vaddr ^ (uint32_t)(64 * d))));
    const v4s f1 =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(at + 8 * PITCH + (vaddr ^ (uint32_t)(64 * d + 32))));
    return __builtin_bit_cast(v4u, (v8s)__builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  const float c = a.scale_log2;
  v16f o[G];
#pragma unroll
  for (int d = 0; d < G; ++d) o[d] = (v16f){0};
  float m = -__builtin_inff(), l = 0.0f;

  auto step = [&](int key0, Block& b) __attribute__((always_inline)) {
    // What lies past the sequence in its last page counts nothing, whatever it is.
    if (key0 + sub >= it.nk) b.ks = b.vs = 0;
    uint32_t knan = 0, vnan[G];
    const bool odd = __any(any_nan(b.ks) || any_nan(b.vs));
    if (odd) {
      knan = (uint32_t)__ballot(any_nan(b.ks));
#pragma unroll
      for (int g = 0; g < G; ++g) vnan[g] = (uint32_t)__ballot(((b.vs >> (8 * g)) & 255u) == 255u);
      if (any_nan(b.ks)) b.ks = 0;
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (((b.vs >> (8 * g)) & 255u) == 255u) b.vs &= ~(255u << (8 * g));
    }
    v16f s = (v16f){0};
#pragma unroll
    for (int i = 0; i < G2; ++i) {
      const float scale = scale_of(b.ks, i);
#pragma unroll
      for (int w = 0; w < 4; ++w) s = T::mfma(kv_values<T>(b.k[i][w], scale), qf[i][w], s);
    }
    // Value v is key 8 (v / 4) + 4 half + v % 4 of the block.
    if (odd && knan) {
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if ((knan >> (8 * (v >> 2) + 4 * half + (v & 3))) & 1u) s[v] = __builtin_nanf("");
    }
    if (key0 + kCaKeys - 1 > first_last) {
      const int left = last - key0 - 4 * half;
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (8 * (v >> 2) + (v & 3) > left) s[v] = -__builtin_inff();
    }
    // A lane's values of its key to LDS.
#pragma unroll
    for (int i = 0; i < G2; ++i) {
      const float scale = scale_of(b.vs, i);
      const int g = 2 * i + half;
      if (g < G) {
#pragma unroll
        for (int w = 0; w < 4; ++w)
          *(v4u HF_LDS*)(tile + sub * PITCH + (((4 * g + w) ^ at_swizzle<PITCH>(sub)) * 16)) =
              kv_values<T>(b.v[i][w], scale);
      }
    }
    float top = s[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) top = fmaxf(top, s[v]);
    top = half_max(top);
    // The maximum is taken anew where a weight would pass 2^8 (see attention.hip on at_lift); each row goes by its own
    // scores, so that its bits do not depend on the rows that share its wave.
    const bool move = (top - m) * c > 8.0f + at_lift<T>();
    if (__any(move)) {
      const float next = move ? top - a.lift : m;
      const float alpha = move ? __builtin_amdgcn_exp2f((m - next) * c) : 1.0f;
      m = next;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < G; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
    }
    const float mc = m == -__builtin_inff() ? 0.0f : m * c;
    v4u pf[2];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      // Rounded to the type for the second product (attention.hip); the sum is of the unrounded ones.
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * p], c, -mc)), p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * p + 1], c, -mc));
      l += p0 + p1;
      pf[p >> 2][p & 3] = T::pack(p0, p1);
    }
    wave_lds_sync();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int d = 0; d < G; ++d) o[d] = T::mfma(vfrag(ks, d), pf[ks], o[d]);
    if (odd) {
#pragma unroll
      for (int g = 0; g < G; ++g)
        if (vnan[g] && key0 + __builtin_ctz(vnan[g]) <= last)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[g][v] = __builtin_nanf("");
    }
    wave_lds_sync();
  };

  constexpr int kStride = kCaWaves * kCaKeys;
  int key0 = it.key_lo + wave * kCaKeys;
  if (key0 < it.key_hi) {
    Block b;
    load(key0, b);
#pragma unroll 1
    for (;;) {
      const int next = key0 + kStride;
      Block ahead;
      if (next < it.key_hi) load(next, ahead);
      step(key0, b);
      if (next >= it.key_hi) break;
      b = ahead;
      key0 = next;
    }
  }
  l = half_sum(l);
  if (l != l && m == -__builtin_inff()) m = 0.0f;  // only scores that are NaN: seen, so not to be left out below

  // The waves' sums joined: each row's maximum over the waves, every wave's sums to that, then added two by two.
  if (half == 0) ca_stat[wave][sub] = (v2f){m, l};
  __syncthreads();
  float top = -__builtin_inff(), total = 0.0f;
#pragma unroll
  for (int w = 0; w < kCaWaves; ++w) top = fmaxf(top, ca_stat[w][sub][0]);
#pragma unroll
  for (int w = 0; w < kCaWaves; ++w) {
    const v2f ml = ca_stat[w][sub];
    total += ml[0] == -__builtin_inff() ? 0.0f : ml[1] * __builtin_amdgcn_exp2f((ml[0] - top) * c);
  }
  const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - top) * c);
  auto hand = [&](int place) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < G; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(v4f*)(ca_mem + place * 4096 * G + ((4 * d + g) * 64 + lane) * 16) =
            (v4f){o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
  };
  auto take = [&](int place) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < G; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const v4f x = *(const v4f*)(ca_mem + place * 4096 * G + ((4 * d + g) * 64 + lane) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][4 * g + e] += x[e];
      }
  };
#pragma unroll
  for (int d = 0; d < G; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = m == -__builtin_inff() ? 0.0f : o[d][v] * f;
  if (wave >= 2) hand(wave - 2);
  __syncthreads();
  if (wave < 2) take(wave);
  __syncthreads();
  if (wave == 1) hand(0);
  __syncthreads();
  if (wave > 0) return;
  take(0);

  if (it.slot >= 0) {
    float* part = a.ws + (int64_t)it.slot * ca_slot_floats(G);
    if (!live) return;
#pragma unroll
    for (int d = 0; d < G; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(v4f*)(part + sub * 32 * G + 32 * d + 8 * g + 4 * half) =
            (v4f){o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) *(v2f*)(part + kCaRows * 32 * G + 2 * sub) = (v2f){top, total};
    return;
  }
  const float inv = 1.0f / total;
  uint16_t* out = a.out + (it.q0 + (int64_t)token) * a.o_token + head * a.o_head;
#pragma unroll
  for (int d = 0; d < G; ++d)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      uint32_t w[2][2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int v = 4 * (g + x) + 2 * e;
          w[x][e] = last < 0 ? 0u : T::pack(o[d][v] * inv, o[d][v + 1] * inv);
        }
      v4u line;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const auto r = __builtin_amdgcn_permlane32_swap(w[0][e], w[1][e], false, false);
        line[e] = r[0];
        line[2 + e] = r[1];
      }
      const int channel = 32 * d + 8 * (g + half);
      if (live && channel < a.D) *(v4u*)(out + channel) = line;
    }
}

// The shares of a tile joined, as attention_join_kernel does. blockIdx.y takes kJoinRows rows of the tile.
template <class T, int G>
__global__ __launch_bounds__(64 * kJoinRows) void cached_join_kernel(CachedArgs a) {
  const CachedJoin j = a.joins[blockIdx.x];
  const int lane = threadIdx.x & 63, group = lane >> 4;
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 6), d = 8 * (lane & 15);
  if (r >= j.rows) return;
  const int64_t row = (int64_t)j.row0 + r;
  const int token = (int)((uint32_t)row / (uint32_t)a.group);
  const int head = j.head * a.group + (int)(row - (int64_t)token * a.group);
  const int64_t step = ca_slot_floats(G);
  const float* part = a.ws + (int64_t)j.slot0 * step;
  const float* stat = part + kCaRows * 32 * G + 2 * r;
  float top = -__builtin_inff();
  for (int s = lane; s < j.slots; s += 64) top = fmaxf(top, stat[s * step]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  float l = 0.0f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.0f;
  const bool inside = d < 32 * G;
#pragma unroll 4
  for (int s = group; s < j.slots; s += 4) {
    const v2f ml = *(const v2f*)(stat + s * step);
    const float* p = part + s * step + r * 32 * G + (inside ? d : 0);
    const v4f x = *(const v4f*)p, y = *(const v4f*)(p + 4);
    const float f = ml[0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((ml[0] - top) * a.scale_log2);
    l = fmaf(ml[1], f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = fmaf(x[e], f, o[e]);
      o[4 + e] = fmaf(y[e], f, o[4 + e]);
    }
  }
#pragma unroll
  for (int off = 16; off <= 32; off <<= 1) {
    l += __shfl_xor(l, off, 64);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] += __shfl_xor(o[e], off, 64);
  }
  if (group != 0 || d >= a.D) return;
  const int last = a.causal ? min(token + j.nk - j.nq, j.nk - 1) : j.nk - 1;
  const float inv = 1.0f / l;
  v4u out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = last < 0 ? 0u : T::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
  *(v4u*)(a.out + (j.q0 + (int64_t)token) * a.o_token + head * a.o_head + d) = out;
}

}  // namespace hf
