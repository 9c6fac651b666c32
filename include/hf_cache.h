/*
 * hf_cache — C ABI of the MI355X (gfx950) operators of a transformer block around the attention of hf_block.h, in the same
 * library: keys and values held in 4 bits in pages, attention over them, copies of pages, and the norms before and after a
 * block with its gate and residual.
 *
 * As in hf_block.h every launch works on `stream` of the current HIP device, never synchronizes, never allocates, and
 * returns HF_OK or a negative HF_ERR_* code. Each takes its parameters in a struct (host memory, read before the call
 * returns; NULL is HF_ERR_ARGUMENT). Strides are in elements, `dtype` is HF_BF16 or HF_FP16. Forward only.
 *
 * THE PAGES. A cache is [layers][pages][kv_heads][slab]: a page holds page_size tokens (32, 64, 128 or 256) of one layer,
 * and a slab a page's tokens of one head. With G = ceil(D / 32) groups of 32 channels (the last one filled with zeros) and
 * S = G, but 4 for G = 3, a slab is
 *   keys' codes [G][page_size][16 bytes], values' codes the same, scales [page_size][S bytes of keys, S bytes of values].
 * A group's 16 bytes are its 32 codes, the even channel in the low half of a byte. A code is a sign bit above three bits for
 * 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale byte E is the power of two 2^(E - 127), and 255 a group of which every value is NaN.
 * WRITING: scale = the least 2^e that is at least a seventh of the group's largest magnitude (so that the largest is rounded
 * by half a step of the codes at most), e from -125 to 125 for bfloat16 and -23 to 13 for float16, which keeps every code's
 * value finite and exact in the type; 2^-3 for a group of zeros. code = the nearest to x / scale, ties to the even one, values
 * past 6 to 6 (magnitudes above 7 2^125 or, in float16, 7 2^13 = 57344 among them: off by up to a step). A group with a value
 * that is not finite is written as NaN.
 */
#ifndef HF_CACHE_H
#define HF_CACHE_H

#include "hf_block.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one page of one layer (kv_heads slabs), or a negative HF_ERR_* for sizes that no cache has. */
int64_t hf_cache_page_bytes(int32_t kv_heads, int32_t D, int32_t page_size);

/*
 * The work of a batch over a cache (host): sequence b has q_lens[b] queries and kv_lens[b] tokens in the cache, of which the
 * last new_lens[b] are written by hf_cache_append. Its pages are ceil(kv_lens[b] / page_size) entries of `pages`, one
 * sequence behind the other, each in [0, pool_pages). Query heads share key heads and `causal` masks as in
 * hf_attention_plan. Used like that function: with plan == NULL it returns the plan's bytes, otherwise fills `plan`; the
 * caller copies it to the device. A plan serves all layers. hf_cache_ws_bytes gives hf_cached_attention's workspace: shares of
 * what is cut, and where many rows attend to many keys those keys and values in `dtype`, of one sequence or of several up to
 * 2^32 bytes at a time.
 * Requires: D a multiple of 16 up to 128; sums of lengths below 2^31; pool_pages * page_size below 2^31.
 */
int64_t hf_cache_plan(const int64_t* q_lens, const int64_t* kv_lens, const int64_t* new_lens, int64_t count,
                      const int32_t* pages, int64_t pool_pages, int32_t page_size, int32_t heads, int32_t kv_heads,
                      int32_t D, int32_t causal, int32_t cus, void* plan, int64_t bytes);
int64_t hf_cache_ws_bytes(const void* plan, int64_t bytes);

/*
 * Writes k, v [sum new_lens, kv_heads, D] (16-byte aligned, strides multiples of 8) to the pages of one layer. `cache`: the
 * layer's first page, 16-byte aligned. Other tokens of these pages are left as they are.
 */
typedef struct {
  const void* k; int64_t k_token; int64_t k_head; const void* v; int64_t v_token; int64_t v_head; void* cache;
  const void* plan; const void* plan_dev; int64_t plan_bytes; int32_t dtype; hf_stream_t stream;
} hf_cache_append_args;
int hf_cache_append(const hf_cache_append_args* args);

/* The sequences' keys and values as hf_attention takes them: k, v [sum kv_lens, kv_heads, D], contiguous, 16-byte aligned. */
typedef struct {
  const void* cache; void* k; void* v; const void* plan; const void* plan_dev; int64_t plan_bytes; int32_t dtype;
  hf_stream_t stream;
} hf_cache_read_args;
int hf_cache_read(const hf_cache_read_args* args);

/*
 * Attention of q [sum q_lens, heads, D] over the pages of one layer, as hf_attention's over what hf_cache_read gives (a
 * query with no key gets zeros; keys that a query does not see never reach it). out may be q itself, with q's strides, and
 * otherwise overlaps neither q nor the cache. q, out 16-byte aligned, strides multiples of 8.
 */
typedef struct {
  const void* q; int64_t q_token; int64_t q_head; const void* cache; void* out; int64_t o_token; int64_t o_head;
  float scale; const void* plan; const void* plan_dev; int64_t plan_bytes; void* ws; int64_t ws_bytes; int32_t dtype;
  hf_stream_t stream;
} hf_cached_attention_args;
int hf_cached_attention(const hf_cached_attention_args* args);

/*
 * Page src[i] of every layer copied to page dst[i], i < count (src, dst: host memory). No dst twice or among src:
 * HF_ERR_ARGUMENT. pool: [layers] of `pages` pages of page_bytes (a multiple of 16), layers layer_bytes apart (a multiple
 * of 16), 16-byte aligned.
 */
typedef struct {
  void* pool; int64_t layers; int64_t layer_bytes; int64_t pages; int64_t page_bytes; const int32_t* src;
  const int32_t* dst; int64_t count; hf_stream_t stream;
} hf_copy_pages_args;
int hf_copy_pages(const hf_copy_pages_args* args);

/*
 * The norms after and before a block with its gate and residual:
 *   r = residual * x + gate[g] * P(y) (y NULL: r = x, not written),   n = N(r) * (1 + scale[g]) + shift[g]
 * over rows of C channels, row t's group g = group[t] (int32 [T]; NULL: the row itself with per_row, else group 0). P and N
 * are nothing (HF_NORM_NONE), h / sqrt(mean(h^2) + eps) (HF_NORM_RMS) or (h - mean) / sqrt(var + eps) (HF_NORM_LAYER), times
 * a weight [C] each (NULL: ones). gate, scale, shift: [groups, C], NULL for ones, zeros, zeros. n NULL: not computed. All in
 * fp32, r and n rounded once each (n is taken of the unrounded r).
 * x, r: of `dtype`, or fp32 with wide != 0; y, n: of dtype; gate, scale, shift, weights: of dtype, or fp32 with vectors_f32.
 * r may be x and n may be y (or x, when not wide), with the same strides; other overlaps are not allowed.
 * Requires: C a multiple of 8 up to 16384; all 16-byte aligned, strides multiples of 8; T < 2^31.
 */
#define HF_NORM_NONE 0
#define HF_NORM_RMS 1
#define HF_NORM_LAYER 2
typedef struct {
  const void* x; int64_t ldx; const void* y; int64_t ldy; void* r; int64_t ldr; void* n; int64_t ldn; const void* gate;
  int64_t ld_gate; const void* scale; int64_t ld_scale; const void* shift; int64_t ld_shift; const void* post_weight;
  const void* weight; const int32_t* group; int64_t groups; int64_t T; int32_t C; int32_t post; int32_t norm;
  int32_t per_row; int32_t wide; int32_t vectors_f32; int32_t dtype; float residual; float eps; hf_stream_t stream;
} hf_residual_norm_args;
int hf_residual_norm(const hf_residual_norm_args* args);

#ifdef __cplusplus
}
#endif

#endif /* HF_CACHE_H */
