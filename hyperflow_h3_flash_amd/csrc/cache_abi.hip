// Host launchers and the planner behind include/hf_cache.h; the end of block_abi.hip's translation unit.
#pragma once

#include "../../include/hf_cache.h"
#include "cached_attention.hip"
#include "kv_cache.hip"
#include "residual_norm.hip"

namespace {

constexpr int32_t kCacheMagic = 0x48464b56;
struct CacheHeader {
  int32_t magic, heads, kv_heads, D, causal, page, items, joins;
  int64_t bytes, slots, q_rows, kv_rows, new_rows, wide_rows;  // wide_rows: of the pass that expands most
  int32_t reads, writes, wides, join_rows;  // join_rows: of the fullest tile that is joined
  // Where each part starts: items, joins, tables, segments read, written and expanded, the passes' plans (and their bytes).
  int64_t at_items, at_joins, at_tables, at_reads, at_writes, at_wides, at_attention, attention_bytes;
  int64_t pool_pages;
  int32_t row_blocks, passes;
  int64_t at_passes;
  int32_t pad[18];
};
static_assert(sizeof(CacheHeader) == 256, "parts start on 128-byte lines behind it");

// Sequences that are expanded and attended to at a time: their segments, rows of keys, and plan.
struct CachePass {
  int32_t first, count;
  int64_t rows, at_attention, attention_bytes;
};

bool cache_header(const void* plan, int64_t bytes, CacheHeader* h) {
  if (!plan || bytes < (int64_t)sizeof(*h)) return false;
  memcpy(h, plan, sizeof(*h));
  return h->magic == kCacheMagic && h->bytes == bytes;
}

inline int cache_groups(int D) { return (D + 31) / 32; }

int cache_sizes(int32_t kv_heads, int32_t D, int32_t page) {
  if (kv_heads < 1 || D < 1) return HF_ERR_ARGUMENT;
  if (page != 32 && page != 64 && page != 128 && page != 256) return HF_ERR_ARGUMENT;
  if (D % 16) return HF_ERR_ALIGNMENT;
  return D > 128 || kv_heads > 65535 ? HF_ERR_SIZE : HF_OK;
}

int64_t cache_page_bytes(const CacheHeader& h) { return h.kv_heads * hf::kv_slab(cache_groups(h.D), h.page); }

// Which sequences have their keys and values expanded to a workspace for attention_kernel, which multiplies about twice as
// fast as the kernel on the pages (that makes codes values anew for every 32 rows): those of many rows a key head, if their
// products together are worth the expansion and its launches. us, on the pages and expanded, 32 / 8 heads of 128: 600 rows x
// 16000 keys 74 and 71, 800 105 and 87, 1200 141 and 110; 8 x 800 x 4000 158 and 166, 8 x 1200 218 and 189; but 2000 x 1000
// 17 and 30, 2000 x 4000 50 and 53. 16 heads of 64: 200 x 16000 44 and 46, 400 77 and 64; 800 x 1000 11 and 24.
constexpr int64_t cache_wide_rows(int D) { return D > 64 ? 640 : 320; }
constexpr double kWidePairs = 64 << 20;  // of rows and keys, over the key heads
// Values of the keys of the other sequences up to which they are expanded too where some are: the kernel on the pages and its
// join would be two launches more, one behind the other (4096, 8191 keys expanded beside 733 and 2500, 8 heads of 128: 124 us
// with those on the pages, 108 with all expanded).
constexpr int64_t kWideRest = 6 << 20;

// Bytes of expanded keys and values up to which sequences share a pass. What is more is expanded pass by pass into the same
// workspace, so that it does not grow with the batch (a sequence is not divided). ms, in one pass and in passes of this size,
// and the workspaces, 8 key heads of 128: 24 x 200 tokens over 100000, 32 heads 13.8 and 11.0, 9.2 and 3.8 GiB; 100 x 160 over
// 30000 13.7 and 12.5, 11.4 and 3.9; 8 x 1000 over 300000, 8 heads 14.7 and 13.2, 9.2 and 3.5. Passes of a quarter of this end
// their attention more often than they gain: 3 x 1000 over 300000 4.7 in one, 5.4 in three.
constexpr int64_t kMostExpanded = (int64_t)1 << 32;

struct CacheWork {
  CacheHeader head;
  std::vector<hf::CachedItem> items;
  std::vector<hf::CachedJoin> joins;
  std::vector<int32_t> tables;
  std::vector<hf::CacheSegment> reads, writes, wides;
  std::vector<CachePass> passes;
  std::vector<AttentionWork> attentions;  // of each pass
};

// Segments of tokens lo .. hi - 1 of a sequence.
void cache_segments(std::vector<hf::CacheSegment>* to, const int32_t* table, int page, int64_t lo, int64_t hi, int64_t row0) {
  for (int64_t t = lo; t < hi;) {
    const int64_t end = std::min((t / page + 1) * page, hi);
    to->push_back({table[t / page], (int32_t)(t % page), (int32_t)(end - t), (int32_t)(row0 + t - lo)});
    t = end;
  }
}

// Lays out the work; HF_OK or an error.
int cache_layout(const int64_t* q_lens, const int64_t* kv_lens, const int64_t* new_lens, int64_t count,
                 const int32_t* pages, int64_t pool_pages, int page, int heads, int kv_heads, int D, int causal, int cus,
                 CacheWork* w) {
  const int64_t limit = 0x7fffffff, group = heads / kv_heads;
  int64_t q_rows = 0, kv_rows = 0, new_rows = 0, table = 0;
  for (int64_t b = 0; b < count; ++b) {
    if (q_lens[b] < 0 || kv_lens[b] < 0 || new_lens[b] < 0 || new_lens[b] > kv_lens[b]) return HF_ERR_ARGUMENT;
    if (q_lens[b] > limit || kv_lens[b] > limit) return HF_ERR_SIZE;
    q_rows += q_lens[b], kv_rows += kv_lens[b], new_rows += new_lens[b];
    if (q_rows > limit || kv_rows > limit - 4096 || q_lens[b] * group > limit - 4096) return HF_ERR_SIZE;
    const int64_t n = (kv_lens[b] + page - 1) / page;
    if (n > 0 && !pages) return HF_ERR_ARGUMENT;
    for (int64_t i = 0; i < n; ++i)
      if (pages[table + i] < 0 || pages[table + i] >= pool_pages) return HF_ERR_ARGUMENT;
    table += n;
  }
  w->tables.assign(pages, pages + table);
  double pairs = 0;
  int64_t rest = 0;
  for (int64_t b = 0; b < count; ++b)
    if (q_lens[b] * group >= cache_wide_rows(D)) pairs += (double)(q_lens[b] * group) * kv_lens[b] * kv_heads;
    else rest += kv_lens[b];
  const bool all = rest <= kWideRest / ((int64_t)kv_heads * D);
  const int64_t direct_rows = pairs < kWidePairs ? limit : all ? 0 : cache_wide_rows(D) - 1;  // of a sequence on its pages

  struct Tile {
    hf::CachedItem item;
    int64_t cost, rows;
  };
  // Rows of a tile: 16 hold the tokens and heads of most batches; two blocks where a sequence has more, so that its keys are
  // read and made values of once (16 x 5 tokens of 32 / 8 heads 26.1 us; beside such a one, fifteen single tokens 24.9 where
  // sixteen take 21.2).
  int64_t most = 0;
  for (int64_t b = 0; b < count; ++b)
    if (q_lens[b] * group <= direct_rows) most = std::max(most, q_lens[b] * group);
  const int row_blocks = most > hf::kCaRows ? 2 : 1, tile_rows = hf::kCaRows * row_blocks;
  std::vector<Tile> tiles;
  struct Wide {
    std::vector<int64_t> q, kv, q0;
  };
  std::vector<Wide> wides;  // of each pass
  const int64_t pass_rows = kMostExpanded / (4 * (int64_t)kv_heads * D);
  int64_t total = 0, q0 = 0, k0 = 0, n0 = 0;
  table = 0;
  for (int64_t b = 0; b < count; ++b) {
    const int64_t nq = q_lens[b], nk = kv_lens[b];
    const int32_t* mine = w->tables.data() + table;
    cache_segments(&w->reads, mine, page, 0, nk, k0);
    cache_segments(&w->writes, mine, page, nk - new_lens[b], nk, n0);
    if (nq * group > direct_rows) {
      if (wides.empty() || (w->passes.back().rows > 0 && w->passes.back().rows + nk > pass_rows)) {
        wides.emplace_back();
        w->passes.push_back({(int32_t)w->wides.size(), 0, 0, 0, 0});
      }
      CachePass& pass = w->passes.back();
      cache_segments(&w->wides, mine, page, 0, nk, pass.rows);
      pass.count = (int32_t)w->wides.size() - pass.first;
      pass.rows += nk;
      wides.back().q.push_back(nq), wides.back().kv.push_back(nk), wides.back().q0.push_back(q0);
    } else {
      for (int h = 0; h < kv_heads; ++h)
        for (int64_t r = 0; r < nq * group; r += tile_rows) {
          const int64_t last = std::min(r + tile_rows, nq * group) - 1;
          const int64_t hi = causal ? std::min(std::max(last / group + nk - nq + 1, (int64_t)0), nk) : nk;
          Tile t;
          memset(&t, 0, sizeof(t));
          t.item.q0 = (int32_t)q0, t.item.nq = (int32_t)nq, t.item.nk = (int32_t)nk, t.item.row0 = (int32_t)r;
          t.item.key_hi = (int32_t)hi, t.item.head = h, t.item.slot = -1, t.item.table0 = (int32_t)table;
          t.cost = (hi + hf::kCaKeys - 1) / hf::kCaKeys;
          t.rows = last + 1 - r;
          total += t.cost;
          tiles.push_back(t);
          if ((int64_t)tiles.size() > limit / 64) return HF_ERR_SIZE;
        }
    }
    q0 += nq, k0 += nk, n0 += new_lens[b];
    table += (nk + page - 1) / page;
  }
  std::stable_sort(tiles.begin(), tiles.end(), [](const Tile& x, const Tile& y) { return x.cost > y.cost; });
  // A tile of n blocks is cut into parts of about `part` blocks: no shorter than sqrt(n), where a wave's steps and the join's
  // reads take about as long (30000 keys, 32 / 8 heads: parts of 15 17.2 us, 30 15.0, 64 20.8). Up to kWhole blocks it is not
  // cut, for the join's launch costs as much (700 keys 8.6 us against 12.6). Of the lengths that make one to three parts a
  // compute unit, that with the soonest end: if each unit takes the longest part left (a start costs about kStart blocks),
  // and a join its tile's shares (four cost about a block). 131072 keys, 64 / 8 heads: one part a unit 32.9 us, one and a
  // quarter 38.8, two 34.7; 16 caches of 1 to 16384 keys, 32 / 8 heads: one 23.5, one and three quarters 21.9, two 25.2.
  constexpr int64_t kWhole = 32, kStart = 8;
  const int64_t longest = tiles.empty() ? 0 : tiles[0].cost;
  const auto less = [](int64_t x, int64_t y) { return x > y; };
  const auto parts_of = [&](int64_t cost, int64_t part) { return cost <= kWhole ? 1 : (cost + part - 1) / part; };
  int64_t part = std::max(longest, (int64_t)1), best = -1;
  // With many tiles a unit their order evens them out, and only long ones are cut.
  for (int quarters = tiles.size() > (size_t)8 * cus ? 12 : 4; quarters <= 12 && longest > kWhole; ++quarters) {
    const int64_t n = std::max({(4 * total + quarters * (int64_t)cus - 1) / (quarters * (int64_t)cus),
                                (int64_t)ceil(sqrt((double)longest)), (int64_t)2 * hf::kCaWaves});
    std::vector<int64_t> costs, units((size_t)cus, 0);
    for (const Tile& t : tiles) {
      const int64_t parts = parts_of(t.cost, n);
      costs.insert(costs.end(), (size_t)parts, (t.cost + parts - 1) / parts + kStart);
    }
    std::sort(costs.begin(), costs.end(), less);
    for (int64_t c : costs) {
      std::pop_heap(units.begin(), units.end(), less);
      units.back() += c;
      std::push_heap(units.begin(), units.end(), less);
    }
    const int64_t end = *std::max_element(units.begin(), units.end()) + parts_of(longest, n) / 4;
    if (best < 0 || end < best) best = end, part = n;
  }
  int64_t slots = 0;
  int32_t join_rows = 0;
  for (const Tile& t : tiles) {
    const int64_t parts = parts_of(t.cost, part);
    if (parts == 1) {
      w->items.push_back(t.item);
      continue;
    }
    if (slots + parts > limit) return HF_ERR_SIZE;
    w->joins.push_back({t.item.q0, t.item.nq, t.item.nk, t.item.row0, t.item.head, (int32_t)slots, (int32_t)parts,
                        (int32_t)t.rows});
    join_rows = std::max(join_rows, (int32_t)t.rows);
    for (int64_t i = 0; i < parts; ++i) {
      hf::CachedItem it = t.item;
      it.key_lo = (int32_t)(t.cost * i / parts * hf::kCaKeys);
      it.key_hi = (int32_t)std::min(t.cost * (i + 1) / parts * hf::kCaKeys, (int64_t)t.item.key_hi);
      it.slot = (int32_t)slots++;
      w->items.push_back(it);
    }
  }
  std::stable_sort(w->items.begin(), w->items.end(), [](const hf::CachedItem& x, const hf::CachedItem& y) {
    return x.key_hi - x.key_lo > y.key_hi - y.key_lo;
  });
  for (hf::CachedItem& it : w->items)
    for (int i = 0; i < hf::kCaWaves; ++i)
      if (it.key_lo + i * hf::kCaKeys < it.key_hi) it.first[i] = w->tables[it.table0 + (it.key_lo + i * hf::kCaKeys) / page];
  // A launch has fewer than 2^32 threads.
  constexpr size_t kMostGroups = (1 << 24) - 1;
  if (w->items.size() > kMostGroups || w->reads.size() > kMostGroups) return HF_ERR_SIZE;
  CacheHeader& h = w->head;
  memset(&h, 0, sizeof(h));
  h.magic = kCacheMagic;
  w->attentions.resize(wides.size());
  for (size_t i = 0; i < wides.size(); ++i) {
    if (!attention_layout(wides[i].q.data(), wides[i].kv.data(), (int64_t)wides[i].q.size(), heads, kv_heads, D, causal, cus,
                          &w->attentions[i], wides[i].q0.data(), true))
      return HF_ERR_SIZE;
    w->passes[i].attention_bytes = w->attentions[i].head.bytes;
    w->passes[i].at_attention = h.attention_bytes;
    h.attention_bytes = (i + 1 < wides.size() ? up_to(h.attention_bytes + w->passes[i].attention_bytes, 128)
                                              : h.attention_bytes + w->passes[i].attention_bytes);
    h.wide_rows = std::max(h.wide_rows, w->passes[i].rows);
  }
  h.heads = heads, h.kv_heads = kv_heads, h.D = D, h.causal = causal != 0, h.page = page;
  h.items = (int32_t)w->items.size(), h.joins = (int32_t)w->joins.size(), h.slots = slots, h.join_rows = join_rows;
  h.row_blocks = row_blocks;
  h.q_rows = q_rows, h.kv_rows = kv_rows, h.new_rows = new_rows, h.pool_pages = pool_pages;
  h.reads = (int32_t)w->reads.size(), h.writes = (int32_t)w->writes.size(), h.wides = (int32_t)w->wides.size();
  int64_t at = sizeof(h);
  const auto place = [&](int64_t* where, int64_t bytes) {
    *where = at;
    at = up_to(at + bytes, 128);
  };
  place(&h.at_items, h.items * (int64_t)sizeof(hf::CachedItem));
  place(&h.at_joins, h.joins * (int64_t)sizeof(hf::CachedJoin));
  place(&h.at_tables, (int64_t)w->tables.size() * 4);
  place(&h.at_reads, h.reads * (int64_t)sizeof(hf::CacheSegment));
  place(&h.at_writes, h.writes * (int64_t)sizeof(hf::CacheSegment));
  place(&h.at_wides, h.wides * (int64_t)sizeof(hf::CacheSegment));
  place(&h.at_attention, h.attention_bytes);
  h.passes = (int32_t)w->passes.size();
  place(&h.at_passes, h.passes * (int64_t)sizeof(CachePass));
  for (CachePass& pass : w->passes) pass.at_attention += h.at_attention;
  h.bytes = at;
  return HF_OK;
}

CachePass cache_pass(const CacheHeader& h, const void* plan, int i) {
  CachePass pass;
  memcpy(&pass, (const unsigned char*)plan + h.at_passes + i * (int64_t)sizeof(pass), sizeof(pass));
  return pass;
}

// The workspace of an attention call: shares of the rows computed on the pages, expanded keys and values of a pass, and the
// workspace of the attention over those.
struct CacheSpace {
  int64_t k, v, attention, bytes;
};
CacheSpace cache_space(const CacheHeader& h, int64_t attention_ws) {
  CacheSpace s;
  s.k = up_to(h.slots * hf::ca_slot_floats(cache_groups(h.D), h.row_blocks) * 4, 256);
  s.v = s.k + up_to(h.wide_rows * h.kv_heads * h.D * 2, 256);
  s.attention = s.v + up_to(h.wide_rows * h.kv_heads * h.D * 2, 256);
  s.bytes = s.attention + attention_ws;
  return s;
}

int64_t cache_attention_ws(const CacheHeader& h, const void* plan) {
  int64_t most = 0;
  for (int i = 0; i < h.passes; ++i) {
    const CachePass pass = cache_pass(h, plan, i);
    most = std::max(most, hf_attention_ws_bytes((const unsigned char*)plan + pass.at_attention, pass.attention_bytes));
  }
  return most;
}

#define HF_CACHE_GROUPS(G, CALL)  \
  switch (G) {                    \
    case 1: CALL(1); break;       \
    case 2: CALL(2); break;       \
    case 3: CALL(3); break;       \
    default: CALL(4); break;      \
  }

template <class CT>
void launch_cache_write(const hf::CacheWriteArgs& a, dim3 grid, hipStream_t stream) {
#define HF_CALL(G) hipLaunchKernelGGL((hf::cache_write_kernel<CT, G>), grid, dim3(hf::kCacheThreads), 0, stream, a)
  HF_CACHE_GROUPS(cache_groups(a.D), HF_CALL)
#undef HF_CALL
}

template <class CT>
void launch_cache_read(const hf::CacheReadArgs& a, dim3 grid, hipStream_t stream) {
#define HF_CALL(G) hipLaunchKernelGGL((hf::cache_read_kernel<CT, G>), grid, dim3(hf::kCacheThreads), 0, stream, a)
  HF_CACHE_GROUPS(cache_groups(a.D), HF_CALL)
#undef HF_CALL
}

int cache_read(const CacheHeader& h, const void* cache, void* k, void* v, const unsigned char* segments, int32_t count,
               int32_t dtype, hipStream_t stream) {
  hf::CacheReadArgs a = {};
  a.cache = (const unsigned char*)cache, a.out[0] = (uint16_t*)k, a.out[1] = (uint16_t*)v;
  a.segments = (const hf::CacheSegment*)segments;
  a.page_bytes = cache_page_bytes(h), a.D = h.D, a.page = h.page, a.heads = h.kv_heads;
  const dim3 grid(count, h.kv_heads);
  if (dtype == HF_BF16) launch_cache_read<hf::CacheTypeBf16>(a, grid, stream);
  else launch_cache_read<hf::CacheTypeFp16>(a, grid, stream);
  return launch_status();
}

template <class T, int G, int R>
int launch_cached_rows(const hf::CachedArgs& a, const CacheHeader& h, hipStream_t stream) {
  hipLaunchKernelGGL((hf::cached_rows_kernel<T, G, R>), dim3(h.items), dim3(64 * hf::kCaWaves), 0, stream, a);
  if (int st = launch_status()) return st;
  if (h.joins == 0) return HF_OK;
  hipLaunchKernelGGL((hf::cached_join_kernel<T, G, R>), dim3(h.joins, (h.join_rows + hf::kJoinRows - 1) / hf::kJoinRows),
                     dim3(64 * hf::kJoinRows), 0, stream, a);
  return launch_status();
}

template <class T, int R>
int launch_cached(const hf::CachedArgs& a, const CacheHeader& h, hipStream_t stream) {
  switch (cache_groups(h.D)) {
    case 1: return launch_cached_rows<T, 1, R>(a, h, stream);
    case 2: return launch_cached_rows<T, 2, R>(a, h, stream);
    case 3: return launch_cached_rows<T, 3, R>(a, h, stream);
    default: return launch_cached_rows<T, 4, R>(a, h, stream);
  }
}

template <class T>
int launch_cached_blocks(const hf::CachedArgs& a, const CacheHeader& h, hipStream_t stream) {
  return h.row_blocks > 1 ? launch_cached<T, 2>(a, h, stream) : launch_cached<T, 1>(a, h, stream);
}

template <class T, bool WIDE, bool VF32, bool Y, int W, int NV>
void launch_norm_rows(const hf::NormArgs& a, hipStream_t stream) {
  constexpr int kWaves = hf::norm_waves(W), kRows = kWaves / W;
  constexpr int64_t kMost = ((int64_t)1 << 31) / (64 * kWaves) * kRows;  // rows of a launch, of fewer than 2^32 threads
  for (int64_t t0 = 0; t0 < a.T; t0 += kMost) {
    hf::NormArgs part = a;
    part.t0 = t0, part.T = std::min(a.T, t0 + kMost);
    const dim3 grid((unsigned)((part.T - t0 + kRows - 1) / kRows));
    hipLaunchKernelGGL((hf::residual_norm_kernel<T, WIDE, VF32, Y, W, NV>), grid, dim3(64 * kWaves), 0, stream, part);
  }
}

template <class T, bool WIDE, bool VF32, bool Y>
void launch_norm_width(const hf::NormArgs& a, hipStream_t stream) {
  // Waves of a row by its width, two or three chunks of 8 channels a lane.
  const int chunks = a.C / 8;
  if (chunks <= 64) launch_norm_rows<T, WIDE, VF32, Y, 1, 1>(a, stream);
  else if (chunks <= 128) launch_norm_rows<T, WIDE, VF32, Y, 1, 2>(a, stream);
  else if (chunks <= 256) launch_norm_rows<T, WIDE, VF32, Y, 2, 2>(a, stream);
  else if (chunks <= 512) launch_norm_rows<T, WIDE, VF32, Y, 4, 2>(a, stream);
  else if (chunks <= 768) launch_norm_rows<T, WIDE, VF32, Y, 4, 3>(a, stream);
  else if (chunks <= 1024) launch_norm_rows<T, WIDE, VF32, Y, 8, 2>(a, stream);
  else if (chunks <= 1536) launch_norm_rows<T, WIDE, VF32, Y, 8, 3>(a, stream);
  else launch_norm_rows<T, WIDE, VF32, Y, 16, 2>(a, stream);
}

template <class T, bool VF32>
void launch_norm(const hf::NormArgs& a, bool wide, hipStream_t stream) {
  if (wide) a.y ? launch_norm_width<T, true, VF32, true>(a, stream) : launch_norm_width<T, true, VF32, false>(a, stream);
  else a.y ? launch_norm_width<T, false, VF32, true>(a, stream) : launch_norm_width<T, false, VF32, false>(a, stream);
}

}  // namespace

extern "C" {

int64_t hf_cache_page_bytes(int32_t kv_heads, int32_t D, int32_t page_size) {
  const int st = cache_sizes(kv_heads, D, page_size);
  return st ? st : kv_heads * hf::kv_slab(cache_groups(D), page_size);
}

int64_t hf_cache_plan(const int64_t* q_lens, const int64_t* kv_lens, const int64_t* new_lens, int64_t count,
                      const int32_t* pages, int64_t pool_pages, int32_t page_size, int32_t heads, int32_t kv_heads,
                      int32_t D, int32_t causal, int32_t cus, void* plan, int64_t bytes) {
  if (count < 0 || (count > 0 && (!q_lens || !kv_lens || !new_lens)) || heads < 1 || kv_heads < 1 || heads % kv_heads ||
      cus < 0 || cus > kMostUnits || pool_pages < 0)
    return HF_ERR_ARGUMENT;
  if (int st = cache_sizes(kv_heads, D, page_size)) return st;
  if (pool_pages > 0x7fffffff / page_size) return HF_ERR_SIZE;
  try {
    CacheWork w;
    const int st = cache_layout(q_lens, kv_lens, new_lens, count, pages, pool_pages, page_size, heads, kv_heads, D, causal,
                                cus ? cus : compute_units(), &w);
    if (st) return st;
    const CacheHeader& h = w.head;
    if (plan) {
      if (bytes < h.bytes) return HF_ERR_SIZE;
      unsigned char* to = (unsigned char*)plan;
      memset(to, 0, h.bytes);
      const auto put = [&](int64_t at, const auto& list) {
        if (!list.empty()) memcpy(to + at, list.data(), list.size() * sizeof(list[0]));
      };
      memcpy(to, &h, sizeof(h));
      put(h.at_items, w.items);
      put(h.at_joins, w.joins);
      put(h.at_tables, w.tables);
      put(h.at_reads, w.reads);
      put(h.at_writes, w.writes);
      put(h.at_wides, w.wides);
      put(h.at_passes, w.passes);
      for (size_t i = 0; i < w.passes.size(); ++i) attention_write(w.attentions[i], to + w.passes[i].at_attention);
    }
    return h.bytes;
  } catch (...) {  // no memory for that many
    return HF_ERR_SIZE;
  }
}

int64_t hf_cache_ws_bytes(const void* plan, int64_t bytes) {
  CacheHeader h;
  if (!cache_header(plan, bytes, &h)) return HF_ERR_ARGUMENT;
  return cache_space(h, cache_attention_ws(h, plan)).bytes;
}

int hf_cache_append(const hf_cache_append_args* p) {
  CacheHeader h;
  if (!p || !cache_header(p->plan, p->plan_bytes, &h) || (p->dtype != HF_BF16 && p->dtype != HF_FP16)) return HF_ERR_ARGUMENT;
  if (h.new_rows == 0) return HF_OK;
  if (!p->k || !p->v || !p->cache || !p->plan_dev) return HF_ERR_ARGUMENT;
  if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->cache, 16) || !aligned(p->plan_dev, 16))
    return HF_ERR_ALIGNMENT;
  for (int64_t s : {p->k_token, p->k_head, p->v_token, p->v_head}) {
    if (s < 0) return HF_ERR_ARGUMENT;
    if (s % 8) return HF_ERR_ALIGNMENT;
  }
  hf::CacheWriteArgs a = {};
  a.x[0] = (const uint16_t*)p->k, a.x[1] = (const uint16_t*)p->v;
  a.token[0] = p->k_token, a.token[1] = p->v_token, a.head[0] = p->k_head, a.head[1] = p->v_head;
  a.cache = (unsigned char*)p->cache, a.page_bytes = cache_page_bytes(h);
  a.segments = (const hf::CacheSegment*)((const unsigned char*)p->plan_dev + h.at_writes);
  a.D = h.D, a.page = h.page;
  const dim3 grid(h.writes, h.kv_heads);
  if (p->dtype == HF_BF16) launch_cache_write<hf::CacheTypeBf16>(a, grid, (hipStream_t)p->stream);
  else launch_cache_write<hf::CacheTypeFp16>(a, grid, (hipStream_t)p->stream);
  return launch_status();
}

int hf_cache_read(const hf_cache_read_args* p) {
  CacheHeader h;
  if (!p || !cache_header(p->plan, p->plan_bytes, &h) || (p->dtype != HF_BF16 && p->dtype != HF_FP16)) return HF_ERR_ARGUMENT;
  if (h.kv_rows == 0) return HF_OK;
  if (!p->k || !p->v || !p->cache || !p->plan_dev) return HF_ERR_ARGUMENT;
  if (!aligned(p->k, 16) || !aligned(p->v, 16) || !aligned(p->cache, 16) || !aligned(p->plan_dev, 16))
    return HF_ERR_ALIGNMENT;
  return cache_read(h, p->cache, p->k, p->v, (const unsigned char*)p->plan_dev + h.at_reads, h.reads, p->dtype,
                    (hipStream_t)p->stream);
}

int hf_cached_attention(const hf_cached_attention_args* p) {
  CacheHeader h;
  if (!p || !cache_header(p->plan, p->plan_bytes, &h) || (p->dtype != HF_BF16 && p->dtype != HF_FP16)) return HF_ERR_ARGUMENT;
  if (!(p->scale > 0.0f) || !isfinite(p->scale)) return HF_ERR_ARGUMENT;
  if (h.q_rows == 0) return HF_OK;
  if (!p->q || !p->out || !p->plan_dev || (h.kv_rows > 0 && !p->cache)) return HF_ERR_ARGUMENT;
  if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->cache, 16) || !aligned(p->plan_dev, 16) ||
      !aligned(p->ws, 16))
    return HF_ERR_ALIGNMENT;
  for (int64_t s : {p->q_token, p->q_head, p->o_token, p->o_head}) {
    if (s < 0) return HF_ERR_ARGUMENT;
    if (s % 8) return HF_ERR_ALIGNMENT;
  }
  const int64_t attention_ws = cache_attention_ws(h, p->plan);
  const CacheSpace space = cache_space(h, attention_ws);
  if (space.bytes > 0 && (!p->ws || p->ws_bytes < space.bytes)) return HF_ERR_ARGUMENT;
  unsigned char* ws = (unsigned char*)p->ws;
  const unsigned char* dev = (const unsigned char*)p->plan_dev;
  if (h.items > 0) {
    hf::CachedArgs a = {};
    a.q = (const uint16_t*)p->q, a.out = (uint16_t*)p->out, a.cache = (const unsigned char*)p->cache, a.ws = (float*)ws;
    a.items = (const hf::CachedItem*)(dev + h.at_items), a.joins = (const hf::CachedJoin*)(dev + h.at_joins);
    a.tables = (const int32_t*)(dev + h.at_tables);
    a.q_token = p->q_token, a.q_head = p->q_head, a.o_token = p->o_token, a.o_head = p->o_head;
    a.page_bytes = cache_page_bytes(h), a.group = h.heads / h.kv_heads, a.D = h.D, a.causal = h.causal, a.page = h.page;
    a.scale_log2 = (float)((double)p->scale * 1.4426950408889634);
    a.lift = (float)std::min((p->dtype == HF_FP16 ? hf::at_lift<hf::Fp16>() : 0) / (double)a.scale_log2, 0x1p127);
    const int st = p->dtype == HF_BF16 ? launch_cached_blocks<hf::Bf16>(a, h, (hipStream_t)p->stream)
                                       : launch_cached_blocks<hf::Fp16>(a, h, (hipStream_t)p->stream);
    if (st) return st;
  }
  const int64_t token = (int64_t)h.kv_heads * h.D;
  for (int i = 0; i < h.passes; ++i) {
    const CachePass pass = cache_pass(h, p->plan, i);
    if (pass.count > 0)
      if (int st = cache_read(h, p->cache, ws + space.k, ws + space.v,
                              dev + h.at_wides + pass.first * (int64_t)sizeof(hf::CacheSegment), pass.count, p->dtype,
                              (hipStream_t)p->stream))
        return st;
    if (int st = hf_attention(p->q, p->q_token, p->q_head, ws + space.k, token, h.D, ws + space.v, token, h.D, p->out,
                              p->o_token, p->o_head, p->scale, (const unsigned char*)p->plan + pass.at_attention,
                              dev + pass.at_attention, pass.attention_bytes, attention_ws ? ws + space.attention : nullptr,
                              attention_ws, p->dtype, p->stream))
      return st;
  }
  return HF_OK;
}

int hf_copy_pages(const hf_copy_pages_args* p) {
  if (!p || p->layers < 0 || p->pages < 0 || p->page_bytes < 0 || p->count < 0 || p->layer_bytes < 0) return HF_ERR_ARGUMENT;
  if (p->count > 0 && (!p->src || !p->dst)) return HF_ERR_ARGUMENT;
  if (p->layers > 65535) return HF_ERR_SIZE;
  if (p->page_bytes % 16 || p->layer_bytes % 16 || !aligned(p->pool, 16)) return HF_ERR_ALIGNMENT;
  for (int64_t i = 0; i < p->count; ++i)
    if (p->src[i] < 0 || p->src[i] >= p->pages || p->dst[i] < 0 || p->dst[i] >= p->pages) return HF_ERR_ARGUMENT;
  try {
    std::vector<int32_t> to(p->dst, p->dst + p->count), from(p->src, p->src + p->count);
    std::sort(to.begin(), to.end());
    std::sort(from.begin(), from.end());
    if (std::adjacent_find(to.begin(), to.end()) != to.end()) return HF_ERR_ARGUMENT;
    for (size_t i = 0, j = 0; i < to.size() && j < from.size();) {
      if (to[i] == from[j]) return HF_ERR_ARGUMENT;
      to[i] < from[j] ? ++i : ++j;
    }
  } catch (...) {
    return HF_ERR_SIZE;
  }
  const int64_t chunks = (p->page_bytes + hf::kCopyBytes - 1) / hf::kCopyBytes;
  if (p->layers == 0 || chunks == 0 || p->count == 0) return HF_OK;
  if (!p->pool) return HF_ERR_ARGUMENT;
  if (p->layers > 1 && p->layer_bytes < p->pages * p->page_bytes) return HF_ERR_ARGUMENT;
  if (chunks > 0x7fffffff) return HF_ERR_SIZE;
  for (int64_t i = 0; i < p->count; i += hf::kCopyPairs) {
    const int n = (int)std::min(p->count - i, (int64_t)hf::kCopyPairs);
    hf::CopyArgs a = {};
    a.pool = (unsigned char*)p->pool, a.layer_bytes = p->layer_bytes, a.page_bytes = p->page_bytes;
    memcpy(a.src, p->src + i, n * sizeof(int32_t));
    memcpy(a.dst, p->dst + i, n * sizeof(int32_t));
    hipLaunchKernelGGL(hf::copy_pages_kernel, dim3((unsigned)chunks, n, (unsigned)p->layers), dim3(hf::kCacheThreads), 0,
                       (hipStream_t)p->stream, a);
    if (int st = launch_status()) return st;
  }
  return HF_OK;
}

int hf_residual_norm(const hf_residual_norm_args* p) {
  if (!p || p->T < 0 || p->C < 0 || p->post < 0 || p->post > 2 || p->norm < 0 || p->norm > 2 || p->groups < 0 ||
      (p->dtype != HF_BF16 && p->dtype != HF_FP16) || !(p->eps >= 0.0f) || !isfinite(p->residual))
    return HF_ERR_ARGUMENT;
  if (p->T > 0x7fffffff || p->C > 16384) return HF_ERR_SIZE;
  if (p->C % 8) return HF_ERR_ALIGNMENT;
  if (p->T == 0 || p->C == 0) return HF_OK;
  if (!p->x || (p->y && !p->r) || (!p->y && !p->n)) return HF_ERR_ARGUMENT;
  if ((p->gate || p->scale || p->shift) && (p->groups < 1 || (!p->group && p->per_row && p->groups < p->T)))
    return HF_ERR_ARGUMENT;
  const void* data[9] = {p->x, p->y, p->y ? p->r : nullptr, p->n, p->gate, p->scale, p->shift, p->post_weight, p->weight};
  for (const void* d : data)
    if (!aligned(d, 16)) return HF_ERR_ALIGNMENT;
  const int64_t strides[7] = {p->ldx, p->y ? p->ldy : 0, p->y ? p->ldr : 0, p->n ? p->ldn : 0, p->gate ? p->ld_gate : 0,
                              p->scale ? p->ld_scale : 0, p->shift ? p->ld_shift : 0};
  for (int64_t s : strides) {
    if (s < 0) return HF_ERR_ARGUMENT;
    if (s % 8) return HF_ERR_ALIGNMENT;
  }
  if (p->T > 1 && ((p->y && p->ldr < p->C) || (p->n && p->ldn < p->C))) return HF_ERR_ARGUMENT;
  hf::NormArgs a = {};
  a.x = p->x, a.y = (const uint16_t*)p->y, a.r = p->r, a.n = (uint16_t*)p->n;
  a.gate = p->gate, a.scale = p->scale, a.shift = p->shift, a.post_weight = p->post_weight, a.weight = p->weight;
  a.group = p->group, a.ldx = p->ldx, a.ldy = p->ldy, a.ldr = p->ldr, a.ldn = p->ldn;
  a.ld_gate = p->ld_gate, a.ld_scale = p->ld_scale, a.ld_shift = p->ld_shift;
  a.T = p->T, a.C = p->C, a.post = p->post, a.norm = p->norm, a.per_row = p->per_row;
  a.residual = p->residual, a.eps = p->eps;
  // Results that the Infinity Cache (256 MiB) does not hold go past it (r and n of 37710 rows, us: of 5376 channels 284 ->
  // 278, of 2048 110 -> 107, of 1024, which it holds, 58.5 -> 61.7).
  a.stream = ((p->y ? (p->wide ? 4 : 2) : 0) + (p->n ? 2 : 0)) * p->T * p->C > (int64_t)256 << 20;
  hipStream_t stream = (hipStream_t)p->stream;
  const bool wide = p->wide != 0;
  if (p->dtype == HF_BF16)
    p->vectors_f32 ? launch_norm<hf::Bf16, true>(a, wide, stream) : launch_norm<hf::Bf16, false>(a, wide, stream);
  else
    p->vectors_f32 ? launch_norm<hf::Fp16, true>(a, wide, stream) : launch_norm<hf::Fp16, false>(a, wide, stream);
  return launch_status();
}

}  // extern "C"
