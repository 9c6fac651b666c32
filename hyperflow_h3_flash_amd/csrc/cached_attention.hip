// Attention of few rows over keys and values in pages of 4-bit codes (kv_cache.hip).
//
// Rows, items and the running maximum and sum are those of attention.hip: a row is a (token, head of the group) pair, here 16
// or 32 of them a workgroup (R blocks of 16), and scores are computed transposed. The four waves of a workgroup take the
// item's blocks of 32 keys in turn, each with sums of its own and no barrier, and join them at the end through LDS.
//
// Operands (matrix instructions of 16 x 16 x 32). Codes go from memory to registers: lane l takes the channels of quarter
// l / 16 (a group of 32 channels, or a quarter of a narrower head) of keys l % 16 and 16 + l % 16. For the scores that is
// already the order of the first product's operand, 8 channels a step, when the queries' channels are taken in the same
// order; codes become values of the type two at a time with the group's scale (exact). A lane's scores are of row l % 16 and
// keys 16 b + 4 (l / 16) + i: the second product's operand when its keys are numbered so. Values are turned through LDS, by
// wave: written by key, read transposed four keys at a time, as in attention.hip.
//
// Bound: the keys' bytes with long caches, a wave's own chain of about 0.7 us a step (codes, product, maximum, exponentials,
// LDS, product) with short ones. One token of 64 / 8 heads against 131072 keys: 29 us and 4 for the join, 4.9 TB/s (a copy:
// 5.0); 16 tokens of 32 / 8 heads against 77411 keys 16.6 and 3.0; 100 tokens of 32 / 8 heads against 16000 keys 57 us, 0.46
// PFLOP/s (codes become values for every 32 rows anew). Loads of the next block have no condition, and its page number is known
// a step earlier: with loads under a condition each wait was one for all of them (54 us for the 16 tokens). Blocks two or
// three steps ahead (25.5 -> 26.7, 27.7) and 64 keys a step (28.0 -> 30.0 for 64 caches of 2000) were slower: more registers,
// fewer waves.
#pragma once

#include "attention.hip"
#include "kv_cache.hip"

namespace hf {

constexpr int kCaRows = 16, kCaWaves = 4, kCaKeys = 32;  // of a block of rows, of a workgroup, of a step

// As AttentionItem; table0: where the sequence's pages begin among all; first: the page of each wave's first block (one load
// less one behind the other at a workgroup's start).
struct CachedItem {
  int32_t q0, nq, nk, row0, key_lo, key_hi, head, slot, table0, first[kCaWaves], pad[3];
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

// Floats of a workspace tile: O [16 R][32 G], then m and l per row.
__host__ __device__ constexpr int ca_slot_floats(int groups, int blocks) { return kCaRows * blocks * (32 * groups + 2); }
__host__ __device__ constexpr int ca_pitch(int groups) { return groups > 2 ? 256 : 128; }

// Chunk c (16 bytes) of row r lies at c ^ f(r): 16 rows' same chunk, as it is written, and two chunks of rows 4 q .. 4 q + 3
// for the two quarters q that the transposing read takes at a time touch every bank once (with at_swizzle, whose halves read
// other chunks, each such read takes two turns).
template <int PITCH>
__device__ __forceinline__ int ca_swizzle(int r) {
  const int q = ((r >> 1) & 2) | ((r >> 3) & 1);
  return PITCH == 256 ? ((r & 3) << 2) | q : (((r >> 1) & 1) << 2) | q;
}

__device__ __forceinline__ v4f ca_mfma(v4u a, v4u b, v4f c, Bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f ca_mfma(v4u a, v4u b, v4f c, Fp16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <class T, int G, int R>
__global__ __launch_bounds__(64 * kCaWaves, R > 1 ? 2 : G > 2 ? 3 : 4) void cached_rows_kernel(CachedArgs a) {
  constexpr int PITCH = ca_pitch(G);
  constexpr int W = G > 2 ? 4 : G;      // dwords of codes a lane takes of a key, steps of the first product
  constexpr int DB = 2 * G;             // blocks of 16 channels
  constexpr int kTile = kCaKeys * PITCH;
  constexpr int kSums = kCaWaves * DB * 1024;  // bytes of the waves' sums of a block of rows
  __shared__ __attribute__((aligned(1024))) unsigned char ca_mem[kCaWaves * kTile > kSums ? kCaWaves * kTile : kSums];
  __shared__ v2f ca_stat[kCaWaves][kCaRows * R];
  const CachedItem it = a.items[blockIdx.x];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int sub = lane & 15, quarter = lane >> 4;
  const int first_page = a.items[blockIdx.x].first[wave];  // (as it.first[wave] the whole item would go through memory)
  // The group of the lane's channels, and the dword of its codes where they begin.
  const int g = G > 2 ? min(quarter, G - 1) : G == 2 ? quarter >> 1 : 0;
  const int dword = G > 2 ? 0 : G == 2 ? 2 * (quarter & 1) : quarter;

  bool live[R];
  int token[R], head[R], last[R];
  v4u qf[R][W];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = (int64_t)it.row0 + kCaRows * r + sub;
    live[r] = row < (int64_t)it.nq * a.group;
    token[r] = live[r] ? (int)((uint32_t)row / (uint32_t)a.group) : 0;
    head[r] = it.head * a.group + (live[r] ? (int)(row - (int64_t)token[r] * a.group) : 0);
    last[r] = live[r] ? (a.causal ? min(token[r] + it.nk - it.nq, it.nk - 1) : it.nk - 1) : -1;
    // Queries in the order of the codes.
    const uint16_t* q = a.q + (it.q0 + (int64_t)token[r]) * a.q_token + head[r] * a.q_head;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int c = 8 * (W * quarter + w);
      qf[r][w] = live[r] && c < a.D ? *(const v4u*)(q + c) : (v4u){0, 0, 0, 0};
    }
  }
  const int first_last = __builtin_amdgcn_readfirstlane(last[0]);  // the first row sees the fewest keys

  typedef uint32_t Codes[W];
  struct Block {
    Codes k[2], v[2];
    uint32_t ks[2], vs[2];  // scale bytes of the key
  };
  const int page_shift = 31 - __builtin_clz(a.page);
  const int64_t slab_bytes = kv_slab(G, a.page);
  const int blocks = (it.key_hi - it.key_lo + kCaKeys - 1) / kCaKeys;
  // Past the item's last block its last one again: loads without a condition, so that waiting for one block's loads is not
  // waiting for the next one's.
  auto key_of = [&](int i) __attribute__((always_inline)) { return it.key_lo + kCaKeys * min(i, blocks - 1); };
  auto page_of = [&](int i) __attribute__((always_inline)) { return a.tables[it.table0 + (key_of(i) >> page_shift)]; };
  auto load = [&](int key0, int page, Block& b) __attribute__((always_inline)) {
    const unsigned char* slab = a.cache + (int64_t)page * a.page_bytes + it.head * slab_bytes;
    const int at = (key0 & (a.page - 1)) + sub;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* k = slab + (g * a.page + at + 16 * h) * 16 + 4 * dword;
      const unsigned char* v = k + G * a.page * 16;
      const unsigned char* s = slab + 2 * G * a.page * 16 + (at + 16 * h) * 2 * kv_scale_bytes(G);
      if constexpr (W == 4) {
        const v4u x = *(const v4u*)k, y = *(const v4u*)v;
        const uint2 z = *(const uint2*)s;
#pragma unroll
        for (int w = 0; w < 4; ++w) b.k[h][w] = x[w], b.v[h][w] = y[w];
        b.ks[h] = z.x, b.vs[h] = z.y;
      } else if constexpr (W == 2) {
        const uint2 x = *(const uint2*)k, y = *(const uint2*)v;
        const uint32_t z = *(const uint32_t*)s;
        b.k[h][0] = x.x, b.k[h][1] = x.y, b.v[h][0] = y.x, b.v[h][1] = y.y;
        b.ks[h] = z & 0xffffu, b.vs[h] = z >> 16;
      } else {
        const uint16_t z = *(const uint16_t*)s;
        b.k[h][0] = *(const uint32_t*)k, b.v[h][0] = *(const uint32_t*)v;
        b.ks[h] = z & 255u, b.vs[h] = z >> 8;
      }
    }
  };
  auto scale_of = [&](uint32_t scales) __attribute__((always_inline)) {
    return __uint_as_float(((scales >> (8 * g)) & 255u) << 23);
  };

  unsigned char HF_LDS* tile = (unsigned char HF_LDS*)ca_mem + wave * kTile;
  const uint32_t vwrite = (uint32_t)(sub * PITCH + (((W * quarter) ^ ca_swizzle<PITCH>(sub)) * 16));
  uint32_t vread;
  {
    const int r = 4 * quarter + (sub >> 2), ch = (lane & 3) >> 1;
    vread = (uint32_t)(r * PITCH + ((ch ^ ca_swizzle<PITCH>(r)) * 16) + (lane & 1) * 8);
  }
  auto vfrag = [&](int d) __attribute__((always_inline)) {  // channels 16 d + sub of keys 4 quarter + i, 16 + 4 quarter + i
    typedef short v8s __attribute__((ext_vector_type(8)));
    const unsigned char HF_LDS* at = tile + (vread ^ (uint32_t)(32 * d));
    const v4s f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)at);
    const v4s f1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(at + 16 * PITCH));
    return __builtin_bit_cast(v4u, (v8s)__builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  const float c = a.scale_log2;
  v4f o[R][DB];
  float m[R], l[R];

  // SAFE: groups of values that are NaN are taken out and their first keys kept (keys come in rising order).
  int nan_from[G];
  auto step = [&](auto safe_t, int key0, Block& b) __attribute__((always_inline)) {
    // What lies past the sequence in its last page counts nothing, whatever it is.
    if (key0 + kCaKeys > it.nk) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (key0 + 16 * h + sub >= it.nk) b.ks[h] = b.vs[h] = 0;
    }
    if constexpr (decltype(safe_t)::value) {
#pragma unroll
      for (int x = 0; x < G; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bool bad = ((b.vs[h] >> (8 * x)) & 255u) == 255u;
          const uint32_t keys = (uint32_t)__ballot(bad) & 0xffffu;
          if (keys) nan_from[x] = min(nan_from[x], key0 + 16 * h + __builtin_ctz(keys));
          if (bad) b.vs[h] &= ~(255u << (8 * x));
        }
    }
    v4f s[R][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float scale = scale_of(b.ks[h]);
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][h] = (v4f){0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const v4u k = kv_values<T>(b.k[h][w], scale);
#pragma unroll
        for (int r = 0; r < R; ++r) s[r][h] = ca_mfma(k, qf[r][w], s[r][h], T());
      }
    }
    // A lane's values of its keys to LDS.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float scale = scale_of(b.vs[h]);
      if (G != 3 || quarter < 3) {
#pragma unroll
        for (int w = 0; w < W; ++w)
          *(v4u HF_LDS*)(tile + (vwrite ^ (uint32_t)(16 * w)) + 16 * h * PITCH) = kv_values<T>(b.v[h][w], scale);
      }
    }
    v4u pf[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (key0 + kCaKeys - 1 > first_last) {  // value i of half h is key 16 h + 4 quarter + i of the block
        const int left = last[r] - key0 - 4 * quarter;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * h + i > left) s[r][h][i] = -__builtin_inff();
      }
      float top = s[r][0][0];
#pragma unroll
      for (int v = 1; v < 8; ++v) top = fmaxf(top, s[r][v >> 2][v & 3]);
      top = quad_max(top);
      // The maximum is taken anew where a weight would pass 2^8 (attention.hip on at_lift); each row goes by its own scores,
      // so that its bits do not depend on the rows that share its wave.
      const bool move = (top - m[r]) * c > 8.0f + at_lift<T>();
      if (__any(move)) {
        const float next = move ? top - a.lift : m[r];
        const float alpha = move ? __builtin_amdgcn_exp2f((m[r] - next) * c) : 1.0f;
        m[r] = next;
        l[r] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int v = 0; v < 4; ++v) o[r][d][v] *= alpha;
      }
      const float mc = m[r] == -__builtin_inff() ? 0.0f : m[r] * c;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        // Rounded to the type for the second product (attention.hip); the sum is of the unrounded ones.
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[r][p >> 1][2 * (p & 1)], c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[r][p >> 1][2 * (p & 1) + 1], c, -mc));
        l[r] += p0 + p1;
        pf[r][p] = T::pack(p0, p1);
      }
    }
    wave_lds_sync();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const v4u v = vfrag(d);
#pragma unroll
      for (int r = 0; r < R; ++r) o[r][d] = ca_mfma(v, pf[r], o[r][d], T());
    }
    wave_lds_sync();
  };
  auto run = [&](auto safe_t) __attribute__((always_inline)) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int d = 0; d < DB; ++d) o[r][d] = (v4f){0, 0, 0, 0};
      m[r] = -__builtin_inff(), l[r] = 0.0f;
    }
#pragma unroll
    for (int x = 0; x < G; ++x) nan_from[x] = 0x7fffffff;
    if (wave >= blocks) return;
    Block b[2];
    load(key_of(wave), first_page, b[0]);
    int page = page_of(wave + kCaWaves);
#pragma unroll 1
    for (int i = wave;;) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        load(key_of(i + kCaWaves), page, b[1 - x]);
        page = page_of(i + 2 * kCaWaves);
        step(safe_t, key_of(i), b[x]);
        i += kCaWaves;
        if (i >= blocks) return;
      }
    }
  };
  run(std::false_type{});
  // A value that is NaN poisons rows that do not see it (0 * NaN); then the wave's keys are taken again the safe way. Keys
  // that are NaN need none of it: scores that a row does not see are replaced.
  {
    bool again = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float all = 0.0f;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 4; ++v) all += o[r][d][v];
      again |= live[r] && all != all;
    }
    if (__any(again)) {
      run(std::true_type{});
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int d = 0; d < DB; ++d)
          if (nan_from[d >> 1] <= last[r]) o[r][d] = (v4f){1, 1, 1, 1} * __builtin_nanf("");
    }
  }

  // The waves' sums joined: each row's maximum over the waves, every wave's sums to that, then a block of 16 channels a wave
  // summed over the waves.
  float top[R], total[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    l[r] = quad_sum(l[r]);
    if (l[r] != l[r] && m[r] == -__builtin_inff()) m[r] = 0.0f;  // only scores that are NaN: seen, so not to be left out
    if (quarter == 0) ca_stat[wave][kCaRows * r + sub] = (v2f){m[r], l[r]};
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    top[r] = -__builtin_inff(), total[r] = 0.0f;
#pragma unroll
    for (int w = 0; w < kCaWaves; ++w) top[r] = fmaxf(top[r], ca_stat[w][kCaRows * r + sub][0]);
#pragma unroll
    for (int w = 0; w < kCaWaves; ++w) {
      const v2f ml = ca_stat[w][kCaRows * r + sub];
      total[r] += ml[0] == -__builtin_inff() ? 0.0f : ml[1] * __builtin_amdgcn_exp2f((ml[0] - top[r]) * c);
    }
    const float f = m[r] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m[r] - top[r]) * c);
    if (r > 0) __syncthreads();
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      v4f x = o[r][d];
#pragma unroll
      for (int v = 0; v < 4; ++v) x[v] = m[r] == -__builtin_inff() ? 0.0f : x[v] * f;
      *(v4f*)(ca_mem + ((wave * DB + d) * 64 + lane) * 16) = x;
    }
    __syncthreads();
    const float inv = 1.0f / total[r];
#pragma unroll
    for (int d0 = 0; d0 < DB; d0 += kCaWaves) {
      const int d = d0 + wave;
      if (d >= DB) break;
      v4f x = *(const v4f*)(ca_mem + (d * 64 + lane) * 16);
#pragma unroll
      for (int w = 1; w < kCaWaves; ++w) x += *(const v4f*)(ca_mem + ((w * DB + d) * 64 + lane) * 16);
      const int channel = 16 * d + 4 * quarter;
      if (!live[r]) continue;
      if (it.slot >= 0) {
        float* part = a.ws + (int64_t)it.slot * ca_slot_floats(G, R) + (kCaRows * r + sub) * 32 * G;
        *(v4f*)(part + channel) = x;
      } else if (channel < a.D) {
        uint16_t* out = a.out + (it.q0 + (int64_t)token[r]) * a.o_token + head[r] * a.o_head + channel;
        *(uint2*)out = last[r] < 0 ? make_uint2(0, 0) : make_uint2(T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv));
      }
    }
    if (it.slot >= 0 && wave == 0 && quarter == 0 && live[r])
      *(v2f*)(a.ws + (int64_t)it.slot * ca_slot_floats(G, R) + kCaRows * R * 32 * G + 2 * (kCaRows * r + sub)) =
          (v2f){top[r], total[r]};
  }
}

// The shares of a tile joined, as attention_join_kernel does. blockIdx.y takes kJoinRows rows of the tile.
template <class T, int G, int R>
__global__ __launch_bounds__(64 * kJoinRows) void cached_join_kernel(CachedArgs a) {
  const CachedJoin j = a.joins[blockIdx.x];
  const int lane = threadIdx.x & 63, group = lane >> 4;
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 6), d = 8 * (lane & 15);
  if (r >= j.rows) return;
  const int64_t row = (int64_t)j.row0 + r;
  const int token = (int)((uint32_t)row / (uint32_t)a.group);
  const int head = j.head * a.group + (int)(row - (int64_t)token * a.group);
  const int64_t step = ca_slot_floats(G, R);
  const float* part = a.ws + (int64_t)j.slot0 * step;
  const float* stat = part + kCaRows * R * 32 * G + 2 * r;
  // One pass: each group of lanes sums its shares to a maximum of its own, then the four are joined.
  float top = -__builtin_inff(), l = 0.0f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.0f;
  const bool inside = d < 32 * G;
  constexpr int kAtOnce = 4;
  for (int s0 = group; s0 < j.slots; s0 += 4 * kAtOnce) {
    v2f ml[kAtOnce];
    v4f x[kAtOnce], y[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t s = min(s0 + 4 * i, j.slots - 1);
      const float* p = part + s * step + r * 32 * G + (inside ? d : 0);
      ml[i] = *(const v2f*)(stat + s * step);
      x[i] = *(const v4f*)p;
      y[i] = *(const v4f*)(p + 4);
    }
    float next = top;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (s0 + 4 * i >= j.slots) ml[i] = (v2f){-__builtin_inff(), 0.0f};
      next = fmaxf(next, ml[i][0]);
    }
    // A share whose keys the row does not see has m = -inf and adds nothing.
    const float f0 = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - next) * a.scale_log2);
    top = next;
    l *= f0;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= f0;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (ml[i][0] == -__builtin_inff()) continue;
      const float f = __builtin_amdgcn_exp2f((ml[i][0] - top) * a.scale_log2);
      l = fmaf(ml[i][1], f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(x[i][e], f, o[e]);
        o[4 + e] = fmaf(y[i][e], f, o[4 + e]);
      }
    }
  }
  {
    const float all = quad_max(top);
    const float f = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - all) * a.scale_log2);
    l = quad_sum(top == -__builtin_inff() ? 0.0f : l * f);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = quad_sum(top == -__builtin_inff() ? 0.0f : o[e] * f);
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
