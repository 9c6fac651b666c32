// Attention over packed sequences: out_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys that query i sees.
//
// One pass over the keys with a running maximum and sum (Milakov and Gimelshein's online softmax): scores and weights
// live in registers only.
//
// Rows. The query heads that share a key head read the same keys, so a row is a (token, head of the group) pair and a
// wave takes 32 rows of one key head: single tokens of grouped heads fill a tile together, and the keys are read once a
// group. Work items come from the plan: a tile of rows of one sequence and key head, and its range of keys (the whole,
// or a share whose unnormalised sums go to a workspace and are joined by attention_join_kernel).
//
// Operands. Scores are computed transposed, S^T = K Q^T, so that one lane holds scores of one row only (row l % 32):
// maximum and sum need one exchange with lane l ^ 32. The accumulator layout of S^T is already the operand layout of
// the weights in O^T = V^T P^T when the keys of a step are numbered 8g + 4h + i (half h, value 4g + i), so the weights
// never leave their lane; V^T comes from LDS through gfx950's transposing 64-bit read in that same order.
//
// LDS. Tiles of 64 keys, K and V, double-buffered, loaded past the registers (16 bytes a lane) while the tile before is
// computed. Rows are 256 (D > 64) or 128 bytes; chunk c of row r lies at c ^ f(r) so that both the 16-row fragment reads
// of K and the 4-row transposing reads of V touch every bank once.
//
// Bound: the card's power with long sequences, the keys' bytes with single tokens. 37710 tokens x 7 heads of 128: 4.44 ms
// among other calls, 1148 TFLOP/s (a large library product of the same type: 1555); in a profiled run of 4.68 ms the matrix
// unit is busy 65 % at 1.64 GHz. On zeros the same launch takes 3.18 ms against 4.35 on random values, both in turn: so
// energy counts, not issue slots. Leaving out the search for the maximum saved 1 %; adding the weights up two at a time with
// dot products nothing; running the products of neighbouring tiles under the weights' arithmetic in one wave, with two tiles
// of scores in registers, raised the matrix unit's share of the cycles and lowered the clock as much (4.63 ms against 4.55):
// the two waves of a SIMD overlap well enough by themselves, once the products' operands are read four products ahead
// (at_order).
// Heads of at most 64 need 167 (bfloat16) and 168 (float16) vector registers, a third of them, and 32 KB of LDS, so three
// workgroups share a compute unit; two, by more LDS, are slower (37710 tokens x 7 heads of 64 2524 us against 2451, prompts
// 111 against 105, cross attention with 511 and 77 keys 70 against 60). A test holds the built kernels to 168: launch bounds
// of three make the compiler spill 2 and 4 registers, 0.3 % slower. Wider heads take two workgroups.
// 16 single tokens of 32 / 8 heads against 77411 keys: 56 us and 4 for the join, 5.6 TB/s (a copy: 5.2).
#pragma once

#include <type_traits>

#include "block_types.h"

namespace hf {

constexpr int kAtKeys = 64;
constexpr int kAtWaves = 4, kAtRows = 32 * kAtWaves;  // of a workgroup
// The largest weight is 2^at_lift when its maximum is taken, not 1: the factor is in the weights' sum too and leaves with
// the quotient. fp16 loses bits under 2^-14 and everything under 2^-25, so with a largest of 1, small weights beside a
// dominant one would be lost to the product and kept in the sum (40000 keys of weight 2^-25.06 beside one of 1: 1.1e-3 of
// the result). Six powers up they keep all bits down to 2^-20 and some down to 2^-31. bfloat16 has float32's exponents.
template <class T>
constexpr int at_lift() { return T::kNarrow ? 6 : 0; }
// What a lane's weights of one tile may sum to before their maximum is taken anew: 512 times the largest when that was
// taken. fp16 holds them (at most 2^15), and bfloat16's sums have as much room for large values as that many keys of equal
// weight take.
template <class T>
constexpr float at_most() { return (float)(512 << at_lift<T>()); }

// A work item: rows row0 .. of sequence (q0, nq, k0, nk) and key head `head`, over keys [key_lo, key_hi). slot < 0: the
// result goes to out; else the unnormalised sums go to workspace tile `slot`.
struct AttentionItem {
  int32_t q0, nq, k0, nk, row0, key_lo, key_hi, head, slot, pad[3];
};
// Workspace tiles slot0 .. slot0 + slots - 1 are the shares of one tile.
struct AttentionJoin {
  int32_t q0, nq, k0, nk, row0, head, slot0, slots;
};

struct AttentionArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  float* ws;
  const AttentionItem* items;
  const AttentionJoin* joins;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
  int group, D, causal;
  float scale_log2;
  float lift;  // at_lift in units of the scores
};

template <int PITCH>
__device__ __forceinline__ int at_swizzle(int r) {
  return PITCH == 256 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Floats of a workspace tile: O [kAtRows][32 DB], then m and l per row.
__host__ __device__ constexpr int at_slot_floats(int db) { return kAtRows * (32 * db + 2); }

// Every load has landed, the queries' among them: told to the compiler here, it need not wait for them inside a loop, where
// it would wait for the next tile too.
__device__ __forceinline__ void at_landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }
// The workgroup's barrier, after this wave's reads of LDS have returned and its loads to LDS have landed.
__device__ __forceinline__ void at_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}
// The order of N products with READS reads of LDS each: operands are on their way four products ahead. Left to itself, the
// compiler reads two and waits for them.
template <int N, int READS>
__device__ __forceinline__ void at_order() {
  constexpr int kAhead = 4;
  __builtin_amdgcn_sched_group_barrier(0x100, kAhead * READS, 0);  // LDS reads
#pragma unroll
  for (int i = 0; i < N - kAhead; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a product
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
  __builtin_amdgcn_sched_barrier(0);
}

// D up to 32 * DB channels.
template <class T, int DB>
__global__ __launch_bounds__(64 * kAtWaves, 2) void attention_kernel(AttentionArgs a) {
  constexpr int PITCH = DB > 2 ? 256 : 128, KS = 2 * DB;
  constexpr int kTile = kAtKeys * PITCH;           // bytes of one K or V tile
  constexpr int kLoads = kTile / 1024 / kAtWaves;  // 1 KiB loads of a wave a tile
  constexpr int kRowsPerLoad = 1024 / PITCH, kChunks = PITCH / 16;
  extern __shared__ __attribute__((aligned(1024))) unsigned char at_lds[];
  unsigned char HF_LDS* lds = (unsigned char HF_LDS*)at_lds;

  const AttentionItem it = a.items[blockIdx.x];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int sub = lane & 31, half = lane >> 5;

  // The lane's row.
  const int64_t row = (int64_t)it.row0 + wave * 32 + sub;
  const bool live = row < (int64_t)it.nq * a.group;
  const int token = live ? (int)((uint32_t)row / (uint32_t)a.group) : 0;
  const int head = it.head * a.group + (live ? (int)(row - (int64_t)token * a.group) : 0);
  // Last key the row sees; -1 for none.
  const int last = live ? (a.causal ? min(token + it.nk - it.nq, it.nk - 1) : it.nk - 1) : -1;
  // The least of the wave's live rows, its first one's (later rows see no less): tiles up to it need no mask.
  const int wave_first = __builtin_amdgcn_readfirstlane(live ? last : 0x7fffffff);

  v4u qf[KS];
  {
    const uint16_t* q = a.q + (it.q0 + (int64_t)token) * a.q_token + head * a.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[s] = live && 16 * s + 8 * half < a.D ? *(const v4u*)(q + 16 * s) : (v4u){0, 0, 0, 0};
  }

  // A wave's loads of a tile: load i fills rows kRowsPerLoad (4 i + wave) ..; lane l row l / kChunks, chunk l % kChunks of
  // LDS from chunk (l % kChunks) ^ f(row) of the key; f does not depend on i. Rows past the sequence and chunks past D read
  // as zero: their offset lies past the descriptor, which starts at the tile, so that offsets stay small however long the
  // sequence is.
  const uint16_t* kbase = a.k + ((int64_t)it.k0 + it.key_lo) * a.k_token + it.head * a.k_head;
  const uint16_t* vbase = a.v + ((int64_t)it.k0 + it.key_lo) * a.v_token + it.head * a.v_head;
  const int kstride = (int)a.k_token, vstride = (int)a.v_token;
  uint32_t kpart, vpart;
  {
    const int r = wave * kRowsPerLoad + lane / kChunks, c = (lane % kChunks) ^ at_swizzle<PITCH>(r);
    kpart = c * 8 < a.D ? (uint32_t)(lane / kChunks * kstride * 2 + c * 16) : 0x80000000u;
    vpart = c * 8 < a.D ? (uint32_t)(lane / kChunks * vstride * 2 + c * 16) : 0x80000000u;
  }
  auto load_tile = [&](const uint16_t* base, int stride, uint32_t part, int t,
                       unsigned char HF_LDS* dst) __attribute__((always_inline)) {
    const int rows = min(kAtKeys, it.nk - it.key_lo - t * kAtKeys);
    const __amdgpu_buffer_rsrc_t rsrc =
        make_rsrc(base + (int64_t)t * kAtKeys * stride, (uint32_t)((rows - 1) * stride * 2 + a.D * 2));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int blk = kAtWaves * i + wave;
      const uint32_t off = part + (uint32_t)(blk * kRowsPerLoad * stride * 2);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (void HF_LDS*)(dst + blk * 1024), 16, off, 0, 0, 0);
    }
  };

  // Fragment addresses within a tile. K: lane (key sub, half) reads chunk 2s + half of step s; V: 4 channels of key
  // 4 half + (lane % 16) / 4 (+ 8 for the second part p), channels 32 d + 16 ((lane / 16) % 2) + 4 (lane % 4). Steps,
  // parts and channel blocks change bits of the chunk that the swizzle changes too, so they are exclusive ors of one
  // address each.
  const uint32_t kaddr = (uint32_t)(sub * PITCH + ((half ^ at_swizzle<PITCH>(sub)) * 16));
  uint32_t vaddr;
  {
    const int r = 4 * half + ((lane & 15) >> 2), ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    vaddr = (uint32_t)(r * PITCH + ((ch ^ at_swizzle<PITCH>(r)) * 16) + (lane & 1) * 8);
  }
  auto kfrag = [&](const unsigned char HF_LDS* kt, int ks, int b) __attribute__((always_inline)) {
    return *(const v4u HF_LDS*)(kt + (kaddr ^ (uint32_t)(32 * ks)) + b * 32 * PITCH);
  };
  auto vfrag = [&](const unsigned char HF_LDS* vt, int ks, int d) __attribute__((always_inline)) {
    typedef short v8s __attribute__((ext_vector_type(8)));
    const unsigned char HF_LDS* at = vt + ks * 16 * PITCH;
    const v4s f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(at + (vaddr ^ (uint32_t)(64 * d))));
    const v4s f1 =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(at + 8 * PITCH + (vaddr ^ (uint32_t)(64 * d + 32))));
    return __builtin_bit_cast(v4u, (v8s)__builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7));
  };

  v16f o[DB];
  float m, l;
  const float c = a.scale_log2;

  // Scores of 64 keys against the wave's 32 rows: value 4g + i of block b is key 32b + 8g + 4h + i.
  auto scores = [&](const unsigned char HF_LDS* kt, v16f (&s)[2]) __attribute__((always_inline)) {
    s[0] = s[1] = (v16f){0};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int b = 0; b < 2; ++b)
        s[b] = T::mfma(kfrag(kt, ks, b), qf[ks], s[b]);
  };

  // Keys that a row does not see out of its scores; tiles that every row of the wave sees in full need none of it.
  auto mask = [&](int key0, v16f (&s)[2]) __attribute__((always_inline)) {
    if (key0 + kAtKeys - 1 > wave_first) {
      const int left = last - key0 - 4 * half;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          if (32 * b + 8 * (v >> 2) + (v & 3) > left) s[b][v] = -__builtin_inff();
          if (v & 1) __builtin_amdgcn_sched_barrier(0);  // two comparisons at a time: scalar registers are scarce
        }
    }
  };

  // Scores to weights, in the operand order of the second product: p = 2^(c (s - m)). m need not be the running maximum,
  // only near enough that the weights keep their precision and their sums stay in range: it is taken in the first tile
  // that a row sees, and anew when a tile's weights sum to more than at_most (or to NaN). Looking for the maximum in every
  // tile would be a seventh of the vector unit's work. Each row goes by its own scores alone, so that its bits do not
  // depend on the rows that share its wave. The sums over the keys are rescaled when m moves (`rescale`).
  auto exponentials = [&](const v16f (&s)[2], v4u (&pf)[4], int p, float mc, float (&part)[2])
                          __attribute__((always_inline)) {  // two of them, p of 16
    // Rounded to the inputs' type for the second product, whose matrix instructions take 16-bit operands (weights in two
    // parts would double its work); their sum is of the unrounded ones.
    const int b = p >> 3, v = 2 * (p & 7);
    const float p0 = __builtin_amdgcn_exp2f(fmaf(s[b][v], c, -mc));
    const float p1 = __builtin_amdgcn_exp2f(fmaf(s[b][v + 1], c, -mc));
    part[0] += p0;
    part[1] += p1;
    pf[p >> 2][p & 3] = T::pack(p0, p1);
  };
  auto centre = [&]() __attribute__((always_inline)) { return m == -__builtin_inff() ? 0.0f : m * c; };
  // After all 16: their sum, or, where m has to move, new weights first.
  auto settle = [&](const v16f (&s)[2], v4u (&pf)[4], float (&part)[2]) __attribute__((always_inline)) {
    float sum = part[0] + part[1];
    if (__any(!(sum <= at_most<T>()) || m == -__builtin_inff())) {
      float top = m;
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(fmaxf(top, s[0][v]), s[1][v]);
      top = half_max(top);
      const bool move = half_max(sum <= at_most<T>() ? 0.0f : 1.0f) > 0.0f || m == -__builtin_inff();
      if constexpr (at_lift<T>() > 0) top -= a.lift;
      m = move ? top : m;
      const float mc = centre();
      part[0] = part[1] = 0.0f;
#pragma unroll
      for (int p = 0; p < 16; ++p) exponentials(s, pf, p, mc, part);
      sum = part[0] + part[1];
    }
    return sum;
  };
  auto rescale = [&](float used) __attribute__((always_inline)) {
    if (__any(used != m)) {
      const float alpha = used != m ? __builtin_amdgcn_exp2f((used - m) * c) : 1.0f;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
    }
  };

  // Weights times the 64 keys' values, added to the sums.
  auto values = [&](const unsigned char HF_LDS* vt, const v4u (&pf)[4]) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
      for (int d = 0; d < DB; ++d)
        o[d] = T::mfma(vfrag(vt, ks, d), pf[ks], o[d]);
  };
  // The same with values that are not finite taken out of the product and added where they are seen.
  auto safe_values = [&](int key0, const unsigned char HF_LDS* vt, const v4u (&pf)[4]) __attribute__((always_inline)) {
    const int left = last - key0 - 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      v16f high = (v16f){0}, low = (v16f){0};  // how many +inf (or NaN) and -inf (or NaN) values a row sees
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const v4u f = vfrag(vt, ks, d);
        v4u fine, up, down, sees;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = 2 * e + x;
            const uint32_t bits = (f[e] >> (16 * x)) & 0xffffu;
            const bool finite = (bits & T::kExponent) != T::kExponent;
            const bool nan = !finite && (bits & 0x7fffu) != T::kExponent;
            w[0] |= (finite ? bits : 0u) << (16 * x);
            w[1] |= (!finite && (nan || !(bits & 0x8000u)) ? T::kOne : 0u) << (16 * x);
            w[2] |= (!finite && (nan || (bits & 0x8000u)) ? T::kOne : 0u) << (16 * x);
            // The key of operand element j in step ks: 16 ks + 8 (j / 4) + 4 h + j % 4.
            w[3] |= (16 * ks + 8 * (j >> 2) + (j & 3) <= left ? T::kOne : 0u) << (16 * x);
          }
          fine[e] = w[0], up[e] = w[1], down[e] = w[2], sees[e] = w[3];
        }
        o[d] = T::mfma(fine, pf[ks], o[d]);
        high = T::mfma(up, sees, high);
        low = T::mfma(down, sees, low);
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        if (high[v] > 0.0f) o[d][v] += __builtin_inff();
        if (low[v] > 0.0f) o[d][v] -= __builtin_inff();
      }
    }
  };

  const int tiles = (it.key_hi - it.key_lo + kAtKeys - 1) / kAtKeys;
  auto load_k = [&](int t) __attribute__((always_inline)) {
    if (t < tiles) load_tile(kbase, kstride, kpart, t, lds + (t & 1) * 2 * kTile);
  };
  auto load_v = [&](int t) __attribute__((always_inline)) {
    if (t < tiles) load_tile(vbase, vstride, vpart, t, lds + (t & 1) * 2 * kTile + kTile);
  };
  auto tile_at = [&](int t) __attribute__((always_inline)) -> const unsigned char HF_LDS* {
    return lds + (t & 1) * 2 * kTile;
  };

  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = (v16f){0};
    m = last >= it.key_lo ? -__builtin_inff() : 0.0f;  // rows that see none of the keys need no maximum
    l = 0.0f;
  };
  auto run = [&](auto safe_t) __attribute__((always_inline)) {
    clear();
    if (tiles <= 0) return;
    load_k(0);
    load_v(0);
    at_landed();
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      // This wave's loads of the tile have landed, and after the barrier everyone's; all have left the other buffer.
      at_barrier();
      load_k(t + 1);
      load_v(t + 1);
      const int key0 = it.key_lo + t * kAtKeys;
      v16f s[2];
      v4u pf[4];
      float part[2] = {0.0f, 0.0f};
      scores(tile_at(t), s);
      at_order<4 * DB, 1>();
      mask(key0, s);
      const float used = m, mc = centre();
#pragma unroll
      for (int p = 0; p < 16; ++p) exponentials(s, pf, p, mc, part);
      const float sum = settle(s, pf, part);
      rescale(used);
      l += sum;
      if constexpr (decltype(safe_t)::value) {
        safe_values(key0, tile_at(t) + kTile, pf);
      } else {
        __builtin_amdgcn_sched_barrier(0);
        values(tile_at(t) + kTile, pf);
        at_order<4 * DB, 2>();
      }
    }
  };
  run(std::false_type{});
  // A key whose values are not finite poisons rows that do not see it (0 * inf); that shows as a NaN in the sums, and
  // then the item runs again the safe way.
  {
    float all = 0.0f;  // NaN if one of the sums is, or infinities of both signs are
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) all += o[d][v];
    bool again = __any(live && all != all);
    // The workgroup decides together, through the buffer that the last tile, which may still be read, does not use.
    int HF_LDS* votes = (int HF_LDS*)(lds + (tiles & 1) * 2 * kTile);
    if (lane == 0) votes[wave] = again;
    at_barrier();
#pragma unroll
    for (int w = 0; w < kAtWaves; ++w) again |= votes[w] != 0;
    if (again) at_barrier();
    if (again) run(std::true_type{});
  }
  l = half_sum(l);
  if (last < it.key_lo) m = -__builtin_inff();

  if (it.slot >= 0) {
    // Shares go out as they are: row-major, and the row's maximum and sum behind them.
    float* part = a.ws + (int64_t)it.slot * at_slot_floats(DB);
    const int r = wave * 32 + sub;
    if (!live) return;  // the end of a tile's rows: nobody joins them
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(v4f*)(part + r * 32 * DB + 32 * d + 8 * g + 4 * half) =
            (v4f){o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) *(v2f*)(part + kAtRows * 32 * DB + 2 * r) = (v2f){m, l};
    return;
  }
  // A row that sees no key is zero; 1 / l otherwise (a row of weights that are all NaN stays NaN).
  const float inv = last < 0 ? 0.0f : 1.0f / l;
  uint16_t* out = a.out + (it.q0 + (int64_t)token) * a.o_token + head * a.o_head;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
      // Values 4g .. are channels 32 d + 8 g + 4 h ..; halves swap so that half h stores the 8 channels of g + h.
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

// The shares of a tile joined: out = sum_s 2^((m_s - M) c) O_s / sum_s 2^((m_s - M) c) l_s. A wave a row: lane group
// lane / 16 takes every fourth share, eight channels a lane. blockIdx.y takes kJoinRows rows of the tile.
constexpr int kJoinRows = 4;
template <class T, int DB>
__global__ __launch_bounds__(64 * kJoinRows) void attention_join_kernel(AttentionArgs a) {
  const AttentionJoin j = a.joins[blockIdx.x];
  const int lane = threadIdx.x & 63, group = lane >> 4;
  const int r = blockIdx.y * kJoinRows + (threadIdx.x >> 6), d = 8 * (lane & 15);
  const int64_t row = (int64_t)j.row0 + r;
  if (row >= (int64_t)j.nq * a.group) return;
  const int token = (int)((uint32_t)row / (uint32_t)a.group);
  const int head = j.head * a.group + (int)(row - (int64_t)token * a.group);
  const int64_t step = at_slot_floats(DB);
  const float* part = a.ws + (int64_t)j.slot0 * step;
  const float* stat = part + kAtRows * 32 * DB + 2 * r;
  float top = -__builtin_inff();
  for (int s = lane; s < j.slots; s += 64) top = fmaxf(top, stat[s * step]);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
  float l = 0.0f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.0f;
  const bool inside = d < 32 * DB;
#pragma unroll 4  // 147 shares: 28.5 us for the call against 29.8 two at a time and 30.6 eight
  for (int s = group; s < j.slots; s += 4) {
    const v2f ml = *(const v2f*)(stat + s * step);
    const float* p = part + s * step + r * 32 * DB + (inside ? d : 0);
    const v4f x = *(const v4f*)p, y = *(const v4f*)(p + 4);
    // A share whose keys the row does not see has m = -inf and adds nothing.
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

// The same for many tiles in few shares each: 16 lanes a row, eight shares' loads on their way at once. Its time is about 5 us
// and an eighth for each share of the tile that has most, whose reads go one behind the other, the other's about 6 us and a
// twenty-fifth for each tile, whose rows take a wave each: this one is taken where a tile has a quarter as many shares as there
// are tiles, or fewer (at_few_shares). us, this one and the other, by tiles joined and most shares of one: 266, 32 13.2 and
// 16.9; 266, 34 13.0 and 16.3; 259, 73 18.2 and 17.9; 232, 6 8.7 and 13.2; 256, 2 8.0 and 14.4; 182, 55 13.4 and 12.1; 96, 5
// 6.4 and 9.1; 56, 9 6.7 and 7.1; 48, 10 7.2 and 7.5; 12, 41 9.3 and 6.8; 8, 64 11.8 and 7.4; 5, 98 16.9 and 8.1.
constexpr int kJoinFewRows = 16, kJoinAtOnce = 8;  // rows of a workgroup
constexpr bool at_few_shares(int64_t most, int64_t joins) { return 4 * most <= joins; }
template <class T, int DB>
__global__ __launch_bounds__(256) void attention_join_few_kernel(AttentionArgs a) {
  const AttentionJoin j = a.joins[blockIdx.x];
  const int r = blockIdx.y * kJoinFewRows + (threadIdx.x >> 4), d = 8 * (threadIdx.x & 15);
  const int64_t row = (int64_t)j.row0 + r;
  if (row >= (int64_t)j.nq * a.group || d >= a.D) return;
  const int64_t step = at_slot_floats(DB);
  const float* part = a.ws + (int64_t)j.slot0 * step;
  const float* stat = part + kAtRows * 32 * DB + 2 * r;
  float top = -__builtin_inff(), l = 0.0f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.0f;
#pragma unroll 1
  for (int s0 = 0; s0 < j.slots; s0 += kJoinAtOnce) {
    v2f ml[kJoinAtOnce];
    v4f x[kJoinAtOnce], y[kJoinAtOnce];
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i) {
      ml[i] = (v2f){-__builtin_inff(), 0.0f};
      x[i] = y[i] = (v4f){0, 0, 0, 0};
      if (s0 + i < j.slots) {
        const float* p = part + (s0 + i) * step + r * 32 * DB + d;
        ml[i] = *(const v2f*)(stat + (s0 + i) * step);
        x[i] = *(const v4f*)p;
        y[i] = *(const v4f*)(p + 4);
      }
    }
    float next = top;
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i) next = fmaxf(next, ml[i][0]);
    if (s0 > 0) {
      const float f = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((top - next) * a.scale_log2);
      l *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] *= f;
    }
    top = next;
#pragma unroll
    for (int i = 0; i < kJoinAtOnce; ++i) {
      // A share whose keys the row does not see has m = -inf and adds nothing.
      const float f = ml[i][0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((ml[i][0] - top) * a.scale_log2);
      l = fmaf(ml[i][1], f, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(x[i][e], f, o[e]);
        o[4 + e] = fmaf(y[i][e], f, o[4 + e]);
      }
    }
  }
  const int token = (int)((uint32_t)row / (uint32_t)a.group);
  const int head = j.head * a.group + (int)(row - (int64_t)token * a.group);
  const int last = a.causal ? min(token + j.nk - j.nq, j.nk - 1) : j.nk - 1;
  const float inv = 1.0f / l;
  v4u out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = last < 0 ? 0u : T::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
  *(v4u*)(a.out + (j.q0 + (int64_t)token) * a.o_token + head * a.o_head + d) = out;
}

}  // namespace hf
