// Host launchers and planners behind the C ABI declared in include/hf_block.h, one translation unit with its kernels.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "../../include/hf_block.h"
#include "adapters.hip"
#include "attention.hip"
#include "qk_norm_rope.hip"

namespace {

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline int launch_status() { return hipGetLastError() == hipSuccess ? HF_OK : HF_ERR_LAUNCH; }
inline int64_t up_to(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// What the planners take: their host memory goes with both.
constexpr int32_t kMostUnits = 1 << 16, kMostAdapters = 1 << 24;

// Compute units of the current device, asked once per device (256 without one).
int compute_units() {
  static std::once_flag once[64];
  static int cus[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  std::call_once(once[dev], [dev] {
    int n = 0;
    cus[dev] = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0 ? n : 256;
  });
  return cus[dev];
}

// ------------------------------------------------------------------------------------------------ norms and rotation

template <class T, int LPR>
void launch_rope(const hf::RopeArgs& a, bool interleaved, bool norm, dim3 grid, size_t lds, hipStream_t stream) {
#define HF_ROPE(I, N)                                                                                            \
  hipLaunchKernelGGL((hf::qk_norm_rope_kernel<T, LPR, I, N>), grid, dim3(hf::kRopeThreads), lds, stream, a)
  if (interleaved) {
    if (norm) HF_ROPE(true, true); else HF_ROPE(true, false);
  } else {
    if (norm) HF_ROPE(false, true); else HF_ROPE(false, false);
  }
#undef HF_ROPE
}

template <class T>
void launch_rope_lanes(const hf::RopeArgs& a, int lanes, bool interleaved, bool norm, dim3 grid, size_t lds,
                       hipStream_t stream) {
  if (lanes <= 4) launch_rope<T, 4>(a, interleaved, norm, grid, lds, stream);
  else if (lanes <= 8) launch_rope<T, 8>(a, interleaved, norm, grid, lds, stream);
  else launch_rope<T, 16>(a, interleaved, norm, grid, lds, stream);
}

// -------------------------------------------------------------------------------------------------- attention's plan

constexpr int32_t kAttentionMagic = 0x48464154;
struct AttentionHeader {
  int32_t magic, heads, kv_heads, D, causal, items, joins, few;  // few: attention_join_few_kernel joins
  int64_t bytes, slots, q_rows, kv_rows;
  int32_t pad[16];
};
static_assert(sizeof(AttentionHeader) == 128, "items start on a 128-byte line");

bool attention_header(const void* plan, int64_t bytes, AttentionHeader* h) {
  if (!plan || bytes < (int64_t)sizeof(*h)) return false;
  memcpy(h, plan, sizeof(*h));
  return h->magic == kAttentionMagic && h->bytes == bytes;
}

inline int attention_db(int D) { return D <= 64 ? 2 : D <= 96 ? 3 : 4; }

struct AttentionWork {
  AttentionHeader head;
  std::vector<hf::AttentionItem> items;
  std::vector<hf::AttentionJoin> joins;
};

// Where the parts of each tile end, in key tiles.
typedef std::vector<std::vector<int64_t>> AttentionCuts;

// When the last place ends if each takes the longest part left whenever it is free, with `start` a part's start costs.
int64_t attention_end(const AttentionCuts& cuts, int64_t places, int64_t start) {
  const auto less = [](int64_t x, int64_t y) { return x > y; };
  std::vector<int64_t> costs, at((size_t)places, 0);
  for (const auto& ends : cuts)
    for (size_t i = 0; i < ends.size(); ++i) costs.push_back(ends[i] - (i > 0 ? ends[i - 1] : 0) + start);
  std::sort(costs.begin(), costs.end(), less);
  for (int64_t c : costs) {
    std::pop_heap(at.begin(), at.end(), less);
    at.back() += c;
    std::push_heap(at.begin(), at.end(), less);
  }
  return *std::max_element(at.begin(), at.end());
}

// Lays out the work; false when a size does not fit the kernels' indexes. q_starts: where each sequence's queries begin (NULL:
// one sequence behind the other). fill: tiles may also be cut to give each place what it lacks of an equal share, where that
// ends well before parts of one length (266 tiles of 590 on 512 places, 7 heads of 128: 603 us against 879 uncut, and cut in
// two they would fill one round and a twentieth of the next).
bool attention_layout(const int64_t* q_lens, const int64_t* kv_lens, int64_t count, int heads, int kv_heads, int D,
                      int causal, int cus, AttentionWork* w, const int64_t* q_starts = nullptr, bool fill = false) {
  const int64_t group = heads / kv_heads, limit = 0x7fffffff;
  int64_t q_rows = 0, kv_rows = 0;
  for (int64_t b = 0; b < count; ++b) {
    if (q_lens[b] < 0 || kv_lens[b] < 0 || q_lens[b] > limit || kv_lens[b] > limit) return false;
    q_rows += q_lens[b];
    kv_rows += kv_lens[b];
    if (q_rows > limit || kv_rows > limit || q_lens[b] * group > limit - 4096) return false;
  }
  struct Piece {
    hf::AttentionItem item;
    int64_t cost;
  };
  std::vector<Piece> tiles;
  int64_t total = 0;
  int64_t q0 = 0, k0 = 0;
  for (int64_t b = 0; b < count; ++b) {
    const int64_t nq = q_lens[b], nk = kv_lens[b];
    if (q_starts) q0 = q_starts[b];
    for (int h = 0; h < kv_heads; ++h)
      for (int64_t r = 0; r < nq * group; r += hf::kAtRows) {
        const int64_t last = std::min(r + hf::kAtRows, nq * group) - 1;
        const int64_t hi = causal ? std::min(std::max(last / group + nk - nq + 1, (int64_t)0), nk) : nk;
        Piece p;
        memset(&p, 0, sizeof(p));
        p.item.q0 = (int32_t)q0, p.item.nq = (int32_t)nq, p.item.k0 = (int32_t)k0, p.item.nk = (int32_t)nk;
        p.item.row0 = (int32_t)r, p.item.key_hi = (int32_t)hi, p.item.head = h, p.item.slot = -1;
        p.cost = (hi + hf::kAtKeys - 1) / hf::kAtKeys;
        total += p.cost;
        tiles.push_back(p);
        if ((int64_t)tiles.size() > limit / 64) return false;
      }
    q0 += nq;
    k0 += nk;
  }
  std::stable_sort(tiles.begin(), tiles.end(), [](const Piece& x, const Piece& y) { return x.cost > y.cost; });
  // The device takes `places` workgroups at a time, the longest tiles first (half as many again of heads of at most 64, but
  // shares laid out for all of those are shorter than they are worth: 37710 tokens x 7 heads of 64 2888 us against 2692, 16
  // single tokens against 77411 keys, 32 / 8 heads of 64, 33.2 against 31.1). Tiles that would end well after an equal share
  // of all work (few rows over many keys, or the last round of equal tiles) are cut along the keys into parts that fill
  // what the whole ones leave; a part costs about two tiles of keys more (its start, its sums' way through memory).
  const int64_t places = 2 * (int64_t)cus, share = (total + places - 1) / places;
  std::vector<int64_t> load((size_t)places, 0);  // a heap, the least loaded place first
  const auto less = [](int64_t x, int64_t y) { return x > y; };
  size_t whole = 0;
  int64_t left = total;
  for (; whole < tiles.size(); ++whole) {
    const int64_t end = load.front() + tiles[whole].cost;
    if (end > share + share / 16 + 4) break;
    std::pop_heap(load.begin(), load.end(), less);
    load.back() = end;
    std::push_heap(load.begin(), load.end(), less);
    left -= tiles[whole].cost;
  }
  // No more parts than places where they are about equal, so that none waits for another. A wave's n tiles in parts of p take it p steps and then n / p
  // reads in the join, a step about eleven reads long: p no less than sqrt(n / 11), and two, or three where a tile's many
  // rows make the join's reads many. Against six whatever n (us; heads / key heads of 128): one token, 131072 keys, 8 / 1
  // 37.6 -> 28.5, 4096 keys, 32 / 8 13.4 -> 11.3, 700 keys 12.7 -> 8.9; 300 tokens, 2000 keys, 8 / 8, three 17.6, two 19.5,
  // six 18.8.
  int64_t longest_cost = 0, most_rows = 0;
  for (size_t t = whole; t < tiles.size(); ++t) {
    const hf::AttentionItem& it = tiles[t].item;
    longest_cost = std::max(longest_cost, tiles[t].cost);
    most_rows = std::max(most_rows, std::min((int64_t)it.nq * group - it.row0, (int64_t)hf::kAtRows));
  }
  int64_t least = std::max((left + places - 1) / places, (int64_t)(most_rows <= 32 ? 2 : 3));
  least = std::max(least, (int64_t)ceil(sqrt((double)longest_cost / 11.0)));
  int64_t part = least;
  for (;; part += part / 32 + 1) {
    int64_t parts = 0;
    for (size_t t = whole; t < tiles.size(); ++t) parts += std::max((tiles[t].cost + part - 1) / part, (int64_t)1);
    if (parts <= places || part >= longest_cost) break;
    // With many short tiles beside long ones the number says nothing: parts longer than twice an equal share would be what
    // all others wait for, while short tiles fill places one behind the other.
    if (part > 2 * least) {
      part = least;
      break;
    }
  }
  AttentionCuts cuts(tiles.size());
  for (size_t t = 0; t < tiles.size(); ++t) {
    const int64_t cost = tiles[t].cost, n = t < whole ? 1 : std::max((cost + part - 1) / part, (int64_t)1);
    for (int64_t i = 1; i <= n; ++i) cuts[t].push_back(cost * i / n);
  }
  if (fill && whole < tiles.size()) {
    constexpr int64_t start = 3;
    const int64_t shortest = std::max(start, (int64_t)ceil(sqrt((double)longest_cost / 11.0)));
    const int64_t end = (total + start * (int64_t)tiles.size()) / places + start;
    AttentionCuts even(tiles.size());
    for (size_t t = 0; t < tiles.size(); ++t) {
      const int64_t cost = tiles[t].cost;
      if (t < whole) even[t].push_back(cost);
      for (int64_t at = 0; t >= whole && at < cost;) {
        int64_t n = std::max(end - load.front() - start, shortest);
        if (cost - at - n < shortest) n = cost - at;
        std::pop_heap(load.begin(), load.end(), less);
        load.back() += n + start;
        std::push_heap(load.begin(), load.end(), less);
        even[t].push_back(at += n);
      }
      if (even[t].empty()) even[t].push_back(cost);
    }
    // Tiles of rows that are not cut at the same keys share less of the L2s (2000 rows x 4000 keys, 16 heads: predicted 6 %
    // sooner, 81 us against 72), so only where it is worth an eighth.
    if (8 * attention_end(even, places, start) < 7 * attention_end(cuts, places, start)) cuts.swap(even);
  }
  int64_t slots = 0;
  for (size_t t = 0; t < tiles.size(); ++t) {
    const Piece& p = tiles[t];
    const std::vector<int64_t>& ends = cuts[t];
    const int64_t parts = (int64_t)ends.size();
    if (parts <= 1) {
      w->items.push_back(p.item);
      continue;
    }
    hf::AttentionJoin j = {p.item.q0, p.item.nq, p.item.k0, p.item.nk, p.item.row0, p.item.head, (int32_t)slots,
                           (int32_t)parts};
    w->joins.push_back(j);
    for (int64_t i = 0; i < parts; ++i) {
      hf::AttentionItem it = p.item;
      it.key_lo = (int32_t)((i > 0 ? ends[i - 1] : 0) * hf::kAtKeys);
      it.key_hi = (int32_t)std::min(ends[i] * hf::kAtKeys, (int64_t)p.item.key_hi);
      it.slot = (int32_t)slots++;
      w->items.push_back(it);
    }
  }
  if (fill)  // the longest first, as places take them
    std::stable_sort(w->items.begin(), w->items.end(), [](const hf::AttentionItem& x, const hf::AttentionItem& y) {
      return x.key_hi - x.key_lo > y.key_hi - y.key_lo;
    });
  memset(&w->head, 0, sizeof(w->head));
  w->head.magic = kAttentionMagic;
  w->head.heads = heads, w->head.kv_heads = kv_heads, w->head.D = D, w->head.causal = causal != 0;
  w->head.items = (int32_t)w->items.size(), w->head.joins = (int32_t)w->joins.size();
  if (fill) {  // (plans of packed sequences keep their order of sums)
    int32_t most = 0;
    for (const hf::AttentionJoin& j : w->joins) most = std::max(most, j.slots);
    w->head.few = hf::at_few_shares(most, w->head.joins);
  }
  w->head.slots = slots, w->head.q_rows = q_rows, w->head.kv_rows = kv_rows;
  w->head.bytes = (int64_t)sizeof(w->head) + (int64_t)(w->items.size() * sizeof(hf::AttentionItem)) +
                  (int64_t)(w->joins.size() * sizeof(hf::AttentionJoin));
  return true;
}

// The plan as its bytes.
void attention_write(const AttentionWork& w, unsigned char* to) {
  memcpy(to, &w.head, sizeof(w.head));
  to += sizeof(w.head);
  if (!w.items.empty()) memcpy(to, w.items.data(), w.items.size() * sizeof(w.items[0]));
  to += w.items.size() * sizeof(hf::AttentionItem);
  if (!w.joins.empty()) memcpy(to, w.joins.data(), w.joins.size() * sizeof(w.joins[0]));
}

int64_t attention_slot_bytes(const AttentionHeader& h) {
  return (int64_t)hf::at_slot_floats(attention_db(h.D)) * 4;
}

constexpr int attention_lds(int db) { return 4 * hf::kAtKeys * (db > 2 ? 256 : 128); }

template <class T, int DB>
int launch_attention(const hf::AttentionArgs& a, const AttentionHeader& h, hipStream_t stream) {
  constexpr int lds = attention_lds(DB);
  static_assert(lds <= 64 * 1024, "dynamic LDS that needs no attribute");
  hipLaunchKernelGGL((hf::attention_kernel<T, DB>), dim3(h.items), dim3(64 * hf::kAtWaves), lds, stream, a);
  if (int st = launch_status()) return st;
  if (h.joins > 0 && h.few) {
    hipLaunchKernelGGL((hf::attention_join_few_kernel<T, DB>), dim3(h.joins, hf::kAtRows / hf::kJoinFewRows), dim3(256), 0,
                       stream, a);
    return launch_status();
  }
  if (h.joins > 0) {
    hipLaunchKernelGGL((hf::attention_join_kernel<T, DB>), dim3(h.joins, hf::kAtRows / hf::kJoinRows),
                       dim3(64 * hf::kJoinRows), 0, stream,
                       a);
    return launch_status();
  }
  return HF_OK;
}

template <class T>
int launch_attention_of(const hf::AttentionArgs& a, const AttentionHeader& h, hipStream_t stream) {
  switch (attention_db(h.D)) {
    case 2: return launch_attention<T, 2>(a, h, stream);
    case 3: return launch_attention<T, 3>(a, h, stream);
    default: return launch_attention<T, 4>(a, h, stream);
  }
}

// -------------------------------------------------------------------------------------------------- adapters' plan

constexpr int32_t kAdapterMagic = 0x48464144;
struct AdapterHeader {
  int32_t magic, adapters, tiles, live_tiles;  // the first live_tiles tiles have an adapter
  int64_t bytes, rows, live_rows;
  int32_t tile_rows;
  int32_t pad[21];
};
static_assert(sizeof(AdapterHeader) == 128, "tiles start on a 128-byte line");

bool adapter_header(const void* plan, int64_t bytes, AdapterHeader* h) {
  if (!plan || bytes < (int64_t)sizeof(*h)) return false;
  memcpy(h, plan, sizeof(*h));
  return h->magic == kAdapterMagic && h->bytes == bytes;
}

// How the first product of a call is cut: rank blocks of 32 that a workgroup takes, rank parts, K shares, and whether a
// launch of its own joins them.
struct AdapterCut {
  int rank_blocks, parts, splits;
  bool join;
};
inline int adapter_waves(int rb, int nb) { return rb == 4 ? 3 : nb == 1 && rb == 1 ? 8 : nb == 1 ? 6 : 4; }
AdapterCut adapter_cut(const AdapterHeader& h, int64_t K, int r32, int32_t dtype, int cus) {
  AdapterCut c;
  c.rank_blocks = r32 <= 32 ? 1 : r32 <= 64 ? 2 : 4;
  c.parts = (r32 / 32 + c.rank_blocks - 1) / c.rank_blocks;
  // One K share while the waves have few steps of 64 k each; beyond that, as many as fill the device (4042 rows x 5376 ->
  // 7168, rank 64, 14 steps: both products 59 us whole, 55 us in two shares with their join; 64 single rows, 10 steps:
  // the join's launch would cost more than it gains).
  const int64_t steps = K / hf::kAdChunk / adapter_waves(c.rank_blocks, h.tile_rows / 32);
  const int64_t wgs = (int64_t)h.live_tiles * c.parts;
  c.splits = 1;
  if (wgs > 0 && steps >= 12 && 2 * wgs <= cus)
    c.splits = (int)std::min(std::min((int64_t)cus / wgs, steps / 6), (int64_t)16);
  c.join = c.splits > 1 || (dtype == HF_FP16 && c.parts > 1);
  return c;
}

// The workspace: rows' factors, u in operand order, and the shares where they are joined.
struct AdapterSpace {
  int64_t frags, planes, bytes;
};
AdapterSpace adapter_space(const AdapterHeader& h, int r32, const AdapterCut& c) {
  const int64_t rows = (int64_t)h.live_tiles * h.tile_rows;
  AdapterSpace s;
  s.frags = up_to(rows * 4, 256);
  s.planes = s.frags + rows * r32 * 4;
  s.bytes = s.planes + (c.join ? c.splits * rows * r32 * 4 : 0);
  return s;
}

// Dynamic LDS past 64 KiB has to be asked for, once per device and kernel.
void allow_lds(const void* kernel, std::once_flag* once, int bytes) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) dev = 0;
  std::once_flag spare;
  std::call_once(dev < 64 ? once[dev] : spare,
                 [&] { (void)hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes); });
}

template <class T, int RB, int NB, int NW>
void launch_adapter_down(const hf::AdapterArgs& a, int parts, hipStream_t stream) {
  static std::once_flag once[64];
  constexpr int lds = hf::ad_down_lds(RB, NB, NW);
  static_assert(lds >= 4096 * RB * NB * NW && lds >= NB * 32 * (RB * 32 + 4) * 4, "the sums fit the rings");
  allow_lds(reinterpret_cast<const void*>(&hf::adapter_down_kernel<T, RB, NB, NW>), once, lds);
  const dim3 grid(a.live_tiles, a.splits, parts);
  hipLaunchKernelGGL((hf::adapter_down_kernel<T, RB, NB, NW>), grid, dim3(64 * NW), lds, stream, a);
}

template <class T, bool VEC>
void launch_adapter_up(const hf::AdapterArgs& a, dim3 grid, hipStream_t stream) {
  static std::once_flag once[64];
  allow_lds(reinterpret_cast<const void*>(&hf::adapter_up_kernel<T, VEC>), once, 512 / 16 * 2048 + 4 * hf::kAdUpStage);
  hipLaunchKernelGGL((hf::adapter_up_kernel<T, VEC>), grid, dim3(hf::kAdUpThreads),
                     a.r32 / 16 * 2048 + 4 * hf::kAdUpStage, stream, a);
}

template <class T>
int launch_adapters(hf::AdapterArgs& a, const AdapterHeader& h, const AdapterCut& c, bool vec, hipStream_t stream) {
  const int cus = compute_units();
  if (h.live_tiles > 0) {
    switch (c.rank_blocks * 4 + a.tile_rows / 32) {
      case 1 * 4 + 1: launch_adapter_down<T, 1, 1, 8>(a, c.parts, stream); break;
      case 1 * 4 + 2: launch_adapter_down<T, 1, 2, 4>(a, c.parts, stream); break;
      case 2 * 4 + 1: launch_adapter_down<T, 2, 1, 6>(a, c.parts, stream); break;
      case 2 * 4 + 2: launch_adapter_down<T, 2, 2, 4>(a, c.parts, stream); break;
      case 4 * 4 + 1: launch_adapter_down<T, 4, 1, 3>(a, c.parts, stream); break;
      default: launch_adapter_down<T, 4, 2, 3>(a, c.parts, stream); break;
    }
    if (int st = launch_status()) return st;
    if (c.join) {
      static std::once_flag once[64];
      allow_lds(reinterpret_cast<const void*>(&hf::adapter_join_kernel<T>), once, 64 * 516 * 4);
      hipLaunchKernelGGL(hf::adapter_join_kernel<T>, dim3(h.live_tiles), dim3(256),
                         (size_t)a.tile_rows * (a.r32 + 4) * 4, stream, a);
      if (int st = launch_status()) return st;
    }
  }
  const int64_t row_blocks = (int64_t)(a.in_place ? h.live_tiles : h.tiles) * (a.tile_rows / 32);
  if (row_blocks == 0) return HF_OK;
  // Column blocks of a workgroup: one a wave with few rows; with many rows up to 4 a wave, for one reading of u (up to 8:
  // 475 -> 508 us at 32768 rows x 15360 columns).
  const int64_t blocks = (a.N + 63) / 64;
  const int64_t want = std::max((int64_t)1, (int64_t)8 * cus / row_blocks);  // workgroups a row block
  a.blocks_per_wg = (int)std::min(std::max(up_to((blocks + want - 1) / want, 4), (int64_t)4), (int64_t)16);
  // A y that the Infinity Cache (256 MiB) does not hold beside what was written with it is read past the caches.
  a.stream_y = h.rows * a.N * 2 > (int64_t)128 << 20;
  a.col_groups = (int)((blocks + a.blocks_per_wg - 1) / a.blocks_per_wg);
  if (row_blocks * a.col_groups > 0x7fffffff) return HF_ERR_SIZE;
  const dim3 grid((unsigned)(row_blocks * a.col_groups));
  if (vec) launch_adapter_up<T, true>(a, grid, stream);
  else launch_adapter_up<T, false>(a, grid, stream);
  return launch_status();
}

}  // namespace

extern "C" {

int hf_qk_norm_rope(const void* q, int64_t q_token, int64_t q_head, int32_t heads_q, const void* k, int64_t k_token,
                    int64_t k_head, int32_t heads_k, void* q_out, int64_t qo_token, int64_t qo_head, void* k_out,
                    int64_t ko_token, int64_t ko_head, const void* pos, int32_t pos_type, int64_t ld_pos, int32_t axes,
                    const double* turns, const int32_t* axis, int32_t pairs, int32_t interleaved, int32_t norm,
                    const void* qw, const void* kw, int32_t weight_f32, float eps, int64_t T, int32_t D, int32_t dtype,
                    hf_stream_t stream) {
  if (T < 0 || heads_q < 0 || heads_k < 0 || D <= 0 || pairs < 0 || axes < 0 || pos_type < 0 || pos_type > 2 ||
      (dtype != HF_BF16 && dtype != HF_FP16) || !(eps >= 0.0f))
    return HF_ERR_ARGUMENT;
  if (T > 0x7fffffff || D > 256 || axes > 16 || (int64_t)heads_q + heads_k > 65536) return HF_ERR_SIZE;
  if (D % 16 || pairs % 8) return HF_ERR_ALIGNMENT;
  if (2 * pairs > D) return HF_ERR_ARGUMENT;
  if (T == 0 || heads_q + heads_k == 0) return HF_OK;
  if (heads_q > 0 && (!q || !q_out)) return HF_ERR_ARGUMENT;
  if (heads_k > 0 && (!k || !k_out)) return HF_ERR_ARGUMENT;
  if (pairs > 0 && (!pos || !turns || !axis || axes < 1 || (T > 1 && ld_pos < axes))) return HF_ERR_ARGUMENT;
  const void* data[6] = {heads_q ? q : nullptr, heads_q ? q_out : nullptr, heads_k ? k : nullptr,
                         heads_k ? k_out : nullptr, norm ? qw : nullptr, norm ? kw : nullptr};
  for (const void* p : data)
    if (!aligned(p, 16)) return HF_ERR_ALIGNMENT;
  if (heads_q > 0 && (q_token % 8 || q_head % 8 || qo_token % 8 || qo_head % 8)) return HF_ERR_ALIGNMENT;
  if (heads_k > 0 && (k_token % 8 || k_head % 8 || ko_token % 8 || ko_head % 8)) return HF_ERR_ALIGNMENT;

  hf::RopeArgs a = {};
  a.side[0] = {(const uint16_t*)q, (uint16_t*)q_out, qw, q_token, q_head, qo_token, qo_head, heads_q};
  a.side[1] = {(const uint16_t*)k, (uint16_t*)k_out, kw, k_token, k_head, ko_token, ko_head, heads_k};
  a.pos = pos, a.ld_pos = ld_pos, a.turns = turns, a.axis = axis, a.T = T, a.pos_type = pos_type, a.pairs = pairs;
  a.D = D, a.weight_f32 = weight_f32, a.eps = eps;
  // A workgroup takes as many tokens of a side as give it three rounds of rows, while every compute unit gets two of them
  // (heads of 128, one round -> three: 37710 tokens x 7 heads each 60 -> 57 us, 16384 x 32 each 130 -> 105, 4099 x 32 and
  // 8 24 -> 20; four rounds and more: 37710 x 56 each 393 -> 411); a share of one token's heads, down to one round, when
  // there are few tokens.
  const int lanes = D <= 64 ? 4 : D <= 128 ? 8 : 16, round = hf::kRopeThreads / lanes;
  const int64_t cus = compute_units();
  int64_t blocks = 0;
  int most = 1;
  for (int i = 0; i < 2; ++i) {
    hf::RopeSide& s = a.side[i];
    s.tokens = 1, s.heads_per_wg = s.heads, s.parts = 1;
    if (s.heads == 0) continue;
    while (s.tokens < 16 && s.tokens * s.heads < 3 * round && T / (2 * s.tokens) >= 2 * cus) s.tokens *= 2;
    if (s.tokens == 1) {
      const int64_t want = std::min(std::max((int64_t)1, 4 * cus / T), (int64_t)(s.heads + round - 1) / round);
      s.heads_per_wg = (int)((s.heads + want - 1) / want);
      s.parts = (s.heads + s.heads_per_wg - 1) / s.heads_per_wg;
    }
    blocks += (T + s.tokens - 1) / s.tokens * s.parts;
    if (i == 0) a.q_blocks = (int)blocks;
    most = std::max(most, s.tokens);
  }
  if (blocks > 0x7fffffff) return HF_ERR_SIZE;
  const dim3 grid((unsigned)blocks);
  const size_t lds = (size_t)most * pairs * sizeof(float) * 2;
  if (dtype == HF_BF16) launch_rope_lanes<hf::Bf16>(a, lanes, interleaved, norm, grid, lds, (hipStream_t)stream);
  else launch_rope_lanes<hf::Fp16>(a, lanes, interleaved, norm, grid, lds, (hipStream_t)stream);
  return launch_status();
}

int64_t hf_attention_plan(const int64_t* q_lens, const int64_t* kv_lens, int64_t count, int32_t heads, int32_t kv_heads,
                          int32_t D, int32_t causal, int32_t cus, void* plan, int64_t bytes) {
  if (count < 0 || (count > 0 && (!q_lens || !kv_lens)) || heads < 1 || kv_heads < 1 || heads % kv_heads || D < 1 ||
      cus < 0 || cus > kMostUnits)
    return HF_ERR_ARGUMENT;
  if (D % 16) return HF_ERR_ALIGNMENT;
  if (D > 128) return HF_ERR_SIZE;
  for (int64_t b = 0; b < count; ++b)
    if (q_lens[b] < 0 || kv_lens[b] < 0) return HF_ERR_ARGUMENT;
  try {
    AttentionWork w;
    if (!attention_layout(q_lens, kv_lens, count, heads, kv_heads, D, causal, cus ? cus : compute_units(), &w))
      return HF_ERR_SIZE;
    if (plan) {
      if (bytes < w.head.bytes) return HF_ERR_SIZE;
      attention_write(w, (unsigned char*)plan);
    }
    return w.head.bytes;
  } catch (...) {  // no memory for that many
    return HF_ERR_SIZE;
  }
}

int64_t hf_attention_ws_bytes(const void* plan, int64_t bytes) {
  AttentionHeader h;
  if (!attention_header(plan, bytes, &h)) return HF_ERR_ARGUMENT;
  return h.slots * attention_slot_bytes(h);
}

int hf_attention(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                 const void* v, int64_t v_token, int64_t v_head, void* out, int64_t o_token, int64_t o_head,
                 float scale, const void* plan, const void* plan_dev, int64_t plan_bytes, void* ws, int64_t ws_bytes,
                 int32_t dtype, hf_stream_t stream) {
  AttentionHeader h;
  if (!attention_header(plan, plan_bytes, &h) || (dtype != HF_BF16 && dtype != HF_FP16)) return HF_ERR_ARGUMENT;
  if (!(scale > 0.0f) || !isfinite(scale)) return HF_ERR_ARGUMENT;
  if (h.items == 0) return HF_OK;
  if (!q || !out || !plan_dev || (h.kv_rows > 0 && (!k || !v))) return HF_ERR_ARGUMENT;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(plan_dev, 16) ||
      !aligned(ws, 16))
    return HF_ERR_ALIGNMENT;
  const int64_t strides[8] = {q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head};
  for (int64_t s : strides) {
    if (s < 0) return HF_ERR_ARGUMENT;
    if (s % 8) return HF_ERR_ALIGNMENT;
  }
  // A key row past the sequence is told by its offset, so rows may not overlap.
  if (h.kv_rows > 1 && (k_token < h.D || v_token < h.D)) return HF_ERR_ARGUMENT;
  if (k_token >= (1 << 23) || v_token >= (1 << 23)) return HF_ERR_SIZE;
  if (h.slots > 0 && (!ws || ws_bytes < h.slots * attention_slot_bytes(h))) return HF_ERR_ARGUMENT;

  hf::AttentionArgs a = {};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v, a.out = (uint16_t*)out;
  a.ws = (float*)ws;
  const unsigned char* dev = (const unsigned char*)plan_dev + sizeof(h);
  a.items = (const hf::AttentionItem*)dev;
  a.joins = (const hf::AttentionJoin*)(dev + (int64_t)h.items * (int64_t)sizeof(hf::AttentionItem));
  a.q_token = q_token, a.q_head = q_head, a.k_token = k_token, a.k_head = k_head;
  a.v_token = v_token, a.v_head = v_head, a.o_token = o_token, a.o_head = o_head;
  a.group = h.heads / h.kv_heads, a.D = h.D, a.causal = h.causal;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  // Finite however small the scale: there every weight is one, whatever is taken off.
  a.lift = (float)std::min((dtype == HF_FP16 ? hf::at_lift<hf::Fp16>() : 0) / (double)a.scale_log2, 0x1p127);
  return dtype == HF_BF16 ? launch_attention_of<hf::Bf16>(a, h, (hipStream_t)stream)
                          : launch_attention_of<hf::Fp16>(a, h, (hipStream_t)stream);
}

int64_t hf_adapter_plan(const int32_t* ids, const int64_t* lens, int64_t count, int32_t adapters, int32_t cus,
                        void* plan, int64_t bytes) {
  if (count < 0 || (count > 0 && !ids) || adapters < 0 || cus < 0 || cus > kMostUnits) return HF_ERR_ARGUMENT;
  if (adapters > kMostAdapters) return HF_ERR_SIZE;
  int64_t rows = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (ids[i] < -1 || ids[i] >= adapters || (lens && lens[i] < 0)) return HF_ERR_ARGUMENT;
    const int64_t n = lens ? lens[i] : 1;
    if (n > 0x7fffffff - rows) return HF_ERR_SIZE;
    rows += n;
  }
  try {
    // Rows sorted by adapter (those without one last), in their order within each: a counting sort over requests.
    const size_t keys = (size_t)adapters + 1;
    std::vector<int64_t> at(keys + 1, 0);
    for (int64_t i = 0; i < count; ++i) at[(ids[i] < 0 ? adapters : ids[i]) + 1] += lens ? lens[i] : 1;
    for (size_t i = 0; i < keys; ++i) at[i + 1] += at[i];
    // Tiles of 64 rows read the first product's weights half as often (the second takes 32 rows a workgroup either way),
    // tiles of 32 are twice as many: 64 once those fill the device
    // (rows, rank, tiles of 32 -> 64: 8192, 64: 75 -> 77 us; 16384, 32: 114 -> 108; 32768, 64: 330 -> 306; 32768, 128:
    // 475 -> 428; 300, 64: 20 -> 23).
    int64_t wide = 0;
    for (size_t key = 0; key + 1 < keys; ++key) wide += (at[key + 1] - at[key] + 63) / 64;
    const int tile_rows = wide >= (cus ? cus : compute_units()) ? 64 : 32;
    std::vector<hf::AdapterTile> tiles;
    int32_t live_tiles = 0;
    for (size_t key = 0; key < keys; ++key) {
      for (int64_t r = at[key]; r < at[key + 1]; r += tile_rows)
        tiles.push_back({key == (size_t)adapters ? -1 : (int32_t)key, (int32_t)r,
                         (int32_t)std::min((int64_t)tile_rows, at[key + 1] - r), 0});
      if (key + 1 < keys) live_tiles = (int32_t)tiles.size();
    }
    AdapterHeader h;
    memset(&h, 0, sizeof(h));
    h.magic = kAdapterMagic, h.adapters = adapters, h.tiles = (int32_t)tiles.size(), h.live_tiles = live_tiles;
    h.rows = rows, h.live_rows = at[keys - 1], h.tile_rows = tile_rows;
    h.bytes = (int64_t)sizeof(h) + (int64_t)(tiles.size() * sizeof(hf::AdapterTile)) + 4 * rows;
    if (plan) {
      if (bytes < h.bytes) return HF_ERR_SIZE;
      unsigned char* to = (unsigned char*)plan;
      memcpy(to, &h, sizeof(h));
      to += sizeof(h);
      if (!tiles.empty()) memcpy(to, tiles.data(), tiles.size() * sizeof(tiles[0]));
      int32_t* list = (int32_t*)(to + tiles.size() * sizeof(hf::AdapterTile));
      int32_t row = 0;
      for (int64_t i = 0; i < count; ++i) {
        int64_t& next = at[ids[i] < 0 ? adapters : ids[i]];
        for (int64_t n = lens ? lens[i] : 1; n > 0; --n) list[next++] = row++;
      }
    }
    return h.bytes;
  } catch (...) {  // no memory for that many
    return HF_ERR_SIZE;
  }
}

int64_t hf_adapter_ws_bytes(const void* plan, int64_t bytes, int64_t K, int32_t r, int32_t dtype) {
  AdapterHeader h;
  if (!adapter_header(plan, bytes, &h) || K <= 0 || r <= 0 || r > 512 || (dtype != HF_BF16 && dtype != HF_FP16))
    return HF_ERR_ARGUMENT;
  const int r32 = (int)up_to(r, 32);
  return adapter_space(h, r32, adapter_cut(h, K, r32, dtype, compute_units())).bytes;
}

int hf_adapter_add(const void* x, int64_t ldx, const void* y, int64_t ldy, const void* down, const void* up, int32_t r,
                   const float* scale, void* out, int64_t ldo, int64_t N, int64_t K, const void* plan,
                   const void* plan_dev, int64_t plan_bytes, void* ws, int64_t ws_bytes, int32_t dtype,
                   hf_stream_t stream) {
  AdapterHeader h;
  if (!adapter_header(plan, plan_bytes, &h) || (dtype != HF_BF16 && dtype != HF_FP16)) return HF_ERR_ARGUMENT;
  if (N < 0 || K <= 0 || r <= 0 || (h.rows > 1 && (ldx < K || ldy < N || ldo < N))) return HF_ERR_ARGUMENT;
  if (r > 512 || N > 0x7fffffff || K > 0x7fffffff) return HF_ERR_SIZE;
  if (K % 8 || r % 8 || ldx % 8) return HF_ERR_ALIGNMENT;
  if (h.rows == 0 || N == 0) return HF_OK;
  if (!y || !out || !plan_dev || (h.live_rows > 0 && (!x || !down || !up))) return HF_ERR_ARGUMENT;
  if (!aligned(x, 16) || !aligned(down, 16) || !aligned(up, 16) || !aligned(y, 2) || !aligned(out, 2) ||
      !aligned(plan_dev, 16) || !aligned(ws, 16) || !aligned(scale, 4))
    return HF_ERR_ALIGNMENT;
  const bool in_place = y == out;
  if (in_place && ldy != ldo && h.rows > 1) return HF_ERR_ARGUMENT;

  hf::AdapterArgs a = {};
  a.x = (const uint16_t*)x, a.y = (const uint16_t*)y, a.down = (const uint16_t*)down, a.up = (const uint16_t*)up;
  a.scale = scale, a.out = (uint16_t*)out;
  const unsigned char* dev = (const unsigned char*)plan_dev + sizeof(h);
  a.tiles = (const hf::AdapterTile*)dev;
  a.rows = (const int32_t*)(dev + (int64_t)h.tiles * (int64_t)sizeof(hf::AdapterTile));
  a.ldx = ldx, a.ldy = ldy, a.ldo = ldo, a.K = K, a.N = N, a.live_tiles = h.live_tiles, a.tile_rows = h.tile_rows;
  a.r = r, a.r32 = (int)up_to(r, 32), a.in_place = in_place;
  const AdapterCut cut = adapter_cut(h, K, a.r32, dtype, compute_units());
  a.splits = cut.splits;
  const AdapterSpace space = adapter_space(h, a.r32, cut);
  if (h.live_rows > 0 && (!ws || ws_bytes < space.bytes)) return HF_ERR_ARGUMENT;
  a.factors = (float*)ws;
  a.frags = (hf::v4u*)((unsigned char*)ws + space.frags);
  a.planes = (float*)((unsigned char*)ws + space.planes);
  const bool vec = aligned(y, 16) && aligned(out, 16) && ldy % 8 == 0 && ldo % 8 == 0 && N % 8 == 0;
  return dtype == HF_BF16 ? launch_adapters<hf::Bf16>(a, h, cut, vec, (hipStream_t)stream)
                          : launch_adapters<hf::Fp16>(a, h, cut, vec, (hipStream_t)stream);
}

int hf_qk_norm_rope_call(const hf_qk_norm_rope_args* a) {
  if (!a) return HF_ERR_ARGUMENT;
  return hf_qk_norm_rope(a->q, a->q_token, a->q_head, a->heads_q, a->k, a->k_token, a->k_head, a->heads_k, a->q_out,
                         a->qo_token, a->qo_head, a->k_out, a->ko_token, a->ko_head, a->pos, a->pos_type, a->ld_pos,
                         a->axes, a->turns, a->axis, a->pairs, a->interleaved, a->norm, a->qw, a->kw, a->weight_f32,
                         a->eps, a->T, a->D, a->dtype, a->stream);
}

int hf_attention_call(const hf_attention_args* a) {
  if (!a) return HF_ERR_ARGUMENT;
  return hf_attention(a->q, a->q_token, a->q_head, a->k, a->k_token, a->k_head, a->v, a->v_token, a->v_head, a->out,
                      a->o_token, a->o_head, a->scale, a->plan, a->plan_dev, a->plan_bytes, a->ws, a->ws_bytes,
                      a->dtype, a->stream);
}

int hf_adapter_add_call(const hf_adapter_add_args* a) {
  if (!a) return HF_ERR_ARGUMENT;
  return hf_adapter_add(a->x, a->ldx, a->y, a->ldy, a->down, a->up, a->r, a->scale, a->out, a->ldo, a->N, a->K,
                        a->plan, a->plan_dev, a->plan_bytes, a->ws, a->ws_bytes, a->dtype, a->stream);
}

}  // extern "C"

#include "cache_abi.hip"
