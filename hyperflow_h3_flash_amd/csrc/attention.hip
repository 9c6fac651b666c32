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
#pragma once

#include <type_traits>

#include "block_types.h"

namespace hf {

constexpr int kAtKeys = 64;

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
  int group, D, causal, items_count;
  float scale_log2;
};

template <int PITCH>
__device__ __forceinline__ int at_swizzle(int r) {
  return PITCH == 256 ? ((r & 3) << 2) | ((r >> 2) & 3) : (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
}

// Floats of a workspace tile of `rows` rows: O [rows][32 DB], then m and l per row.
__host__ __device__ constexpr int at_slot_floats(int rows, int db) { return rows * (32 * db + 2); }

// Lane l exchanges with lane l ^ 32: max of both.
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// NW waves of 32 rows; D up to 32 * DB channels.
template <class T, int DB, int NW>
__global__ __launch_bounds__(64 * NW, 2) void attention_kernel(AttentionArgs a) {
  constexpr int PITCH = DB > 2 ? 256 : 128, KS = 2 * DB;
  constexpr int kTile = kAtKeys * PITCH;       // bytes of one K or V tile
  constexpr int kLoads = kTile / 1024 / NW;    // 1 KiB loads of a wave a tile
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
  int wave_first = live ? last : 0x7fffffff;  // the least of the wave's rows: tiles up to it need no mask
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) wave_first = min(wave_first, __shfl_xor(wave_first, off, 64));
  wave_first = __builtin_amdgcn_readfirstlane(wave_first);

  v4u qf[KS];
  {
    const uint16_t* q = a.q + (it.q0 + (int64_t)token) * a.q_token + head * a.q_head + 8 * half;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qf[s] = live && 16 * s + 8 * half < a.D ? *(const v4u*)(q + 16 * s) : (v4u){0, 0, 0, 0};
  }

  // A wave's loads of a tile: load i fills rows (kLoads wave + i) kRowsPerLoad ..; lane l row l / kChunks, chunk
  // l % kChunks of LDS from chunk (l % kChunks) ^ f(row) of the key. Rows past the sequence and chunks past D read as
  // zero: their offset lies past the descriptor, which starts at the tile, so that offsets stay small however long the
  // sequence is.
  const uint16_t* kbase = a.k + (int64_t)it.k0 * a.k_token + it.head * a.k_head;
  const uint16_t* vbase = a.v + (int64_t)it.k0 * a.v_token + it.head * a.v_head;
  uint32_t kpart[kLoads], vpart[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = (kLoads * wave + i) * kRowsPerLoad + lane / kChunks;
    const int c = (lane % kChunks) ^ at_swizzle<PITCH>(r);
    kpart[i] = c * 8 < a.D ? (uint32_t)(lane / kChunks * (int)a.k_token * 2 + c * 16) : 0x80000000u;
    vpart[i] = c * 8 < a.D ? (uint32_t)(lane / kChunks * (int)a.v_token * 2 + c * 16) : 0x80000000u;
  }
  auto load_tile = [&](const uint16_t* base, int64_t stride, const uint32_t* part, int key0, unsigned char HF_LDS* dst) {
    const int rows = min(kAtKeys, it.nk - key0);
    const __amdgpu_buffer_rsrc_t rsrc =
        make_rsrc(base + (int64_t)key0 * stride, (uint32_t)((rows - 1) * (int)stride * 2 + a.D * 2));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int blk = kLoads * wave + i;
      const uint32_t off = part[i] + (uint32_t)(blk * kRowsPerLoad * (int)stride * 2);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (void HF_LDS*)(dst + blk * 1024), 16, off, 0, 0, 0);
    }
  };

  // Fragment addresses within a tile. K: lane (key sub, half) chunk 2s + half. V: lane reads 4 channels of key
  // 4 half + (lane % 16) / 4 (+ 8 for the second part), channels 16 ((lane / 16) % 2) + 4 (lane % 4).
  int kaddr[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) kaddr[s] = sub * PITCH + (((2 * s + half) ^ at_swizzle<PITCH>(sub)) * 16);
  int vaddr[DB][2];
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int r = 8 * p + 4 * half + ((lane & 15) >> 2);
      const int c = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
      vaddr[d][p] = r * PITCH + ((c ^ at_swizzle<PITCH>(r)) * 16) + (lane & 1) * 8;
    }

  v16f o[DB];
  float m, l;
  const float c = a.scale_log2;

  // SAFE: values that are not finite are taken out of the products and added where they are seen.
  auto run = [&](auto safe_t) {
    constexpr bool SAFE = decltype(safe_t)::value;
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = (v16f){0};
    m = -__builtin_inff();
    l = 0.0f;
    int buf = 0;
    if (it.key_lo < it.key_hi) {
      load_tile(kbase, a.k_token, kpart, it.key_lo, lds);
      load_tile(vbase, a.v_token, vpart, it.key_lo, lds + kTile);
    }
    for (int key0 = it.key_lo; key0 < it.key_hi; key0 += kAtKeys) {
      // This wave's loads of the tile have landed, and after the barrier everyone's; all have left the other buffer.
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      unsigned char HF_LDS* kt = lds + buf * 2 * kTile;
      unsigned char HF_LDS* vt = kt + kTile;
      buf ^= 1;
      if (key0 + kAtKeys < it.key_hi) {
        load_tile(kbase, a.k_token, kpart, key0 + kAtKeys, lds + buf * 2 * kTile);
        load_tile(vbase, a.v_token, vpart, key0 + kAtKeys, lds + buf * 2 * kTile + kTile);
      }
      v16f s[2];
      s[0] = s[1] = (v16f){0};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int b = 0; b < 2; ++b)
          s[b] = T::mfma(*(const v4u HF_LDS*)(kt + kaddr[ks] + b * 32 * PITCH), qf[ks], s[b]);
      if (key0 + kAtKeys - 1 > wave_first) {
        const int left = last - key0 - 4 * half;  // value 4g + i of block b is key 32b + 8g + 4h + i
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (32 * b + 8 * (v >> 2) + (v & 3) > left) s[b][v] = -__builtin_inff();
      }
      float top = m;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int v = 0; v < 16; ++v) top = fmaxf(top, s[b][v]);
      top = half_max(top);
      // The maximum that the weights are taken against follows the running one only when it falls 2^8 behind: the
      // weights then stay below 2^8, which costs no precision, and the sums are rescaled a few times a row at most.
      // Each row goes by its own scores alone, so that its bits do not depend on the rows that share its wave.
      const bool behind = (top - m) * c > 8.0f;  // also from -inf; NaN (still nothing seen) compares false
      if (__any(behind)) {
        const float alpha = behind ? __builtin_amdgcn_exp2f((m - top) * c) : 1.0f;
        m = behind ? top : m;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
      }
      const float mc = m == -__builtin_inff() ? 0.0f : m * c;
      v4u pf[4];
      float sum = 0.0f;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
          const float p0 = __builtin_amdgcn_exp2f(fmaf(s[b][v], c, -mc));
          const float p1 = __builtin_amdgcn_exp2f(fmaf(s[b][v + 1], c, -mc));
          sum += p0 + p1;
          pf[2 * b + (v >> 3)][(v & 7) >> 1] = T::pack(p0, p1);
        }
      l += sum;
      if constexpr (!SAFE) {
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int d = 0; d < DB; ++d) {
            const v4s f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(vt + vaddr[d][0] + ks * 16 * PITCH));
            const v4s f1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(vt + vaddr[d][1] + ks * 16 * PITCH));
            typedef short v8s __attribute__((ext_vector_type(8)));
            const v8s f = __builtin_shufflevector(f0, f1, 0, 1, 2, 3, 4, 5, 6, 7);
            o[d] = T::mfma(__builtin_bit_cast(v4u, f), pf[ks], o[d]);
          }
      } else {
        const int left = last - key0 - 4 * half;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          v16f high = (v16f){0}, low = (v16f){0};  // how many +inf (or NaN) and -inf (or NaN) values a row sees
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const v4s f0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(vt + vaddr[d][0] + ks * 16 * PITCH));
            const v4s f1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((v4s HF_LDS*)(vt + vaddr[d][1] + ks * 16 * PITCH));
            v4u fine, up, down, sees;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int j = 2 * e + x;
                const uint32_t bits = (uint16_t)(j < 4 ? f0[j & 3] : f1[j & 3]);
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
      }
    }
  };
  run(std::false_type{});
  // A key whose values are not finite poisons rows that do not see it (0 * inf); that shows as a NaN in the sums, and
  // then the item runs again the safe way. The vote goes through the buffers' first bytes.
  {
    bool nan = false;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int v = 0; v < 16; ++v) nan |= o[d][v] != o[d][v];
    bool again = __any(live && nan);
    if constexpr (NW > 1) {
      int HF_LDS* votes = (int HF_LDS*)lds;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      if (lane == 0) votes[wave] = again;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
      for (int w = 0; w < NW; ++w) again |= votes[w] != 0;
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (again) run(std::true_type{});
  }
  l = half_sum(l);

  if (it.slot >= 0) {
    // Shares go out as they are: row-major, and the row's maximum and sum behind them.
    float* part = a.ws + (int64_t)it.slot * at_slot_floats(32 * NW, DB);
    const int r = wave * 32 + sub;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(v4f*)(part + r * 32 * DB + 32 * d + 8 * g + 4 * half) =
            (v4f){o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
    if (half == 0) *(v2f*)(part + 32 * NW * 32 * DB + 2 * r) = (v2f){m, l};
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

// The shares of a tile joined: out = sum_s 2^((m_s - M) c) O_s / sum_s 2^((m_s - M) c) l_s. Eight channels a thread;
// blockIdx.y takes kJoinRows rows of the tile.
constexpr int kJoinThreads = 256;
template <class T, int DB>
__global__ __launch_bounds__(kJoinThreads) void attention_join_kernel(AttentionArgs a, int tile_rows) {
  constexpr int kLanes = 4 * DB, kRows = kJoinThreads / 16;
  const AttentionJoin j = a.joins[blockIdx.x];
  const int r = blockIdx.y * kRows + threadIdx.x / 16, d = threadIdx.x % 16 * 8;
  const int64_t row = (int64_t)j.row0 + r;
  if (threadIdx.x % 16 >= kLanes || d >= a.D || r >= tile_rows || row >= (int64_t)j.nq * a.group) return;
  const int token = (int)((uint32_t)row / (uint32_t)a.group);
  const int head = j.head * a.group + (int)(row - (int64_t)token * a.group);
  const int64_t step = at_slot_floats(tile_rows, DB);
  const float* part = a.ws + (int64_t)j.slot0 * step;
  const float* stat = part + tile_rows * 32 * DB + 2 * r;
  float top = -__builtin_inff();
  for (int s = 0; s < j.slots; ++s) top = fmaxf(top, stat[s * step]);
  float l = 0.0f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.0f;
  for (int s = 0; s < j.slots; ++s) {
    const v2f ml = *(const v2f*)(stat + s * step);
    // A share whose keys the row does not see has m = -inf and adds nothing.
    const float f = ml[0] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((ml[0] - top) * a.scale_log2);
    const float* p = part + s * step + r * 32 * DB + d;
    const v4f x = *(const v4f*)p, y = *(const v4f*)(p + 4);
    l = fmaf(ml[1], f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] = fmaf(x[e], f, o[e]);
      o[4 + e] = fmaf(y[e], f, o[4 + e]);
    }
  }
  const int last = a.causal ? min(token + j.nk - j.nq, j.nk - 1) : j.nk - 1;
  const float inv = 1.0f / l;
  v4u out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = last < 0 ? 0u : T::pack(o[2 * e] * inv, o[2 * e + 1] * inv);
  *(v4u*)(a.out + (j.q0 + (int64_t)token) * a.o_token + head * a.o_head + d) = out;
}

}  // namespace hf
