/*
 * hf_block — C ABI of the MI355X (gfx950) operators that an attention block runs around its INT8 convrot linears
 * (hf_convrot.h): the per-head norms of queries and keys with the rotation of positions on several axes, attention
 * over packed sequences, and low-rank adapters of many requests beside a shared projection.
 *
 * As in hf_convrot.h every entry point takes device pointers, strides in elements and sizes, launches on `stream` of
 * the current HIP device, never synchronizes, never allocates, and returns HF_OK or a negative HF_ERR_* code (the
 * codes of hf_convrot.h). The two planners are host functions: they read and write host memory only.
 *
 * `dtype` is HF_BF16 or HF_FP16, the type of every tensor passed as `void*` unless its comment says otherwise. Forward
 * only: the layers of this framework are frozen.
 */
#ifndef HF_BLOCK_H
#define HF_BLOCK_H

#include <stdint.h>

#include "hf_convrot.h"

#ifdef __cplusplus
extern "C" {
#endif

#define HF_BF16 0
#define HF_FP16 1

/*
 * Norm of each head and rotation of its channels by the token's position, q and k in one pass:
 *   n = norm ? x * (1 / sqrt(mean_d(x^2) + eps)) * w[d] : x                       (w NULL: ones)
 *   (a, b) -> (a cos - b sin, a sin + b cos), angle = 2 pi * pos[t, axis[p]] * turns[p], for the pairs p < pairs:
 *     interleaved != 0: channels (2p, 2p + 1);  interleaved == 0: channels (p, p + pairs)
 *   channels at and after 2 * pairs keep n. All in fp32 (the angle's whole turns are taken off in fp64), rounded once.
 * x: [T, heads, D] with strides (token, head), channels contiguous; out the same (may be x itself, with x's strides, and
 * otherwise overlaps neither side's x).
 * heads_k == 0 leaves k out (its pointers are not read). pos: [T, axes] of int32 (HF_POS_I32), int64 (HF_POS_I64) or
 * fp32 (HF_POS_F32), rows `ld_pos` apart; turns: fp64 [pairs], revolutions per position step (theta^(-2i/dim) / 2 pi);
 * axis: int32 [pairs], each in [0, axes). qw, kw: [D] of x's type, or fp32 with weight_f32 != 0, or NULL.
 * Requires: D a multiple of 16 up to 256; 2 * pairs a multiple of 16 up to D; x, out, weights 16-byte aligned with
 * strides that are multiples of 8; at most 16 axes; T < 2^31, heads_q + heads_k <= 65536.
 */
#define HF_POS_I32 0
#define HF_POS_I64 1
#define HF_POS_F32 2
int hf_qk_norm_rope(const void* q, int64_t q_token, int64_t q_head, int32_t heads_q, const void* k, int64_t k_token,
                    int64_t k_head, int32_t heads_k, void* q_out, int64_t qo_token, int64_t qo_head, void* k_out,
                    int64_t ko_token, int64_t ko_head, const void* pos, int32_t pos_type, int64_t ld_pos, int32_t axes,
                    const double* turns, const int32_t* axis, int32_t pairs, int32_t interleaved, int32_t norm,
                    const void* qw, const void* kw, int32_t weight_f32, float eps, int64_t T, int32_t D, int32_t dtype,
                    hf_stream_t stream);

/*
 * Attention over packed sequences. Sequence b has q_lens[b] queries and kv_lens[b] keys, one sequence behind the other
 * in q, out [sum q_lens, heads, D] and k, v [sum kv_lens, kv_heads, D]; query head h reads key head h / (heads /
 * kv_heads). out may be q itself, with q's strides, and otherwise overlaps none of them.
 * out_i = sum_j w_ij v_j, w_i = softmax_j(scale * q_i . k_j) over the sequence's keys; causal: over the keys
 * j <= i + kv_lens[b] - q_lens[b] (the last query sees every key). A query with no key gets zeros; keys that a query
 * does not see never reach it, whatever k and v hold there.
 *
 * hf_attention_plan (host) lays out the work of a batch once for all layers and steps of these lengths: with
 * plan == NULL it returns the plan's bytes (`cus`: the device's compute units, 0 for the current one's, up to 65536),
 * otherwise it fills `plan` (host memory of that many bytes; `bytes` is checked) and returns the bytes, or a negative
 * HF_ERR_*. hf_attention_ws_bytes gives the workspace that a filled plan needs (0: none), or HF_ERR_ARGUMENT for bytes
 * that hold no plan. The caller copies the plan to the device and passes both copies to hf_attention: `plan` (host) for
 * the launch, `plan_dev` for the kernels.
 * Requires: D a multiple of 16 up to 128; heads a multiple of kv_heads; scale > 0 and finite; q, k, v, out 16-byte
 * aligned, token and head strides multiples of 8, of k and v below 2^23; `ws` of at least hf_attention_ws_bytes,
 * 16-byte aligned. Sums of lengths below 2^31.
 */
int64_t hf_attention_plan(const int64_t* q_lens, const int64_t* kv_lens, int64_t count, int32_t heads, int32_t kv_heads,
                          int32_t D, int32_t causal, int32_t cus, void* plan, int64_t bytes);
int64_t hf_attention_ws_bytes(const void* plan, int64_t bytes);
int hf_attention(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                 const void* v, int64_t v_token, int64_t v_head, void* out, int64_t o_token, int64_t o_head,
                 float scale, const void* plan, const void* plan_dev, int64_t plan_bytes, void* ws, int64_t ws_bytes,
                 int32_t dtype, hf_stream_t stream);

/*
 * Low-rank adapters of many requests beside a shared projection: for row m with adapter a = ids[m],
 *   out[m] = y[m] + scale[a] * (x[m] @ down[a]^T) @ up[a]^T,   out[m] = y[m] for a = -1,
 * summed in fp32 with the rank-wide intermediate kept to 16 bits of mantissa or more, rounded once.
 * x: [M, K]; y, out: [M, N] (out may be y itself, with y's stride, and otherwise does not overlap it);
 * down: [adapters, r, K]; up: [adapters, N, r]; scale: fp32 [adapters] or NULL (ones).
 *
 * hf_adapter_plan (host) groups the rows by adapter once for all projections of a batch: `ids` holds one adapter or -1
 * for each of `count` requests, `lens` its rows (NULL: one each). Used like hf_attention_plan.
 * Requires: K, r, ldx multiples of 8, r <= 512; x, down, up 16-byte aligned; y, out 2-byte aligned (16-byte aligned with
 * strides and N multiples of 8 for whole-vector access); ws 16-byte aligned; M, N, K < 2^31; adapters <= 2^24.
 */
int64_t hf_adapter_plan(const int32_t* ids, const int64_t* lens, int64_t count, int32_t adapters, int32_t cus,
                        void* plan, int64_t bytes);
int64_t hf_adapter_ws_bytes(const void* plan, int64_t bytes, int64_t K, int32_t r, int32_t dtype);
int hf_adapter_add(const void* x, int64_t ldx, const void* y, int64_t ldy, const void* down, const void* up, int32_t r,
                   const float* scale, void* out, int64_t ldo, int64_t N, int64_t K, const void* plan,
                   const void* plan_dev, int64_t plan_bytes, void* ws, int64_t ws_bytes, int32_t dtype,
                   hf_stream_t stream);

/*
 * The three launches again with their parameters in a struct, in the order of the lists above: for callers to whom a
 * long list of arguments costs host time (a foreign-function call from Python converts one value instead of 31: 1.0 us
 * against 3.0). `args` is host memory, read before the call returns; NULL is HF_ERR_ARGUMENT.
 */
typedef struct {
  const void* q; int64_t q_token; int64_t q_head; int32_t heads_q; const void* k; int64_t k_token; int64_t k_head;
  int32_t heads_k; void* q_out; int64_t qo_token; int64_t qo_head; void* k_out; int64_t ko_token; int64_t ko_head;
  const void* pos; int32_t pos_type; int64_t ld_pos; int32_t axes; const double* turns; const int32_t* axis;
  int32_t pairs; int32_t interleaved; int32_t norm; const void* qw; const void* kw; int32_t weight_f32; float eps;
  int64_t T; int32_t D; int32_t dtype; hf_stream_t stream;
} hf_qk_norm_rope_args;
typedef struct {
  const void* q; int64_t q_token; int64_t q_head; const void* k; int64_t k_token; int64_t k_head; const void* v;
  int64_t v_token; int64_t v_head; void* out; int64_t o_token; int64_t o_head; float scale; const void* plan;
  const void* plan_dev; int64_t plan_bytes; void* ws; int64_t ws_bytes; int32_t dtype; hf_stream_t stream;
} hf_attention_args;
typedef struct {
  const void* x; int64_t ldx; const void* y; int64_t ldy; const void* down; const void* up; int32_t r;
  const float* scale; void* out; int64_t ldo; int64_t N; int64_t K; const void* plan; const void* plan_dev;
  int64_t plan_bytes; void* ws; int64_t ws_bytes; int32_t dtype; hf_stream_t stream;
} hf_adapter_add_args;
int hf_qk_norm_rope_call(const hf_qk_norm_rope_args* args);
int hf_attention_call(const hf_attention_args* args);
int hf_adapter_add_call(const hf_adapter_add_args* args);

#ifdef __cplusplus
}
#endif

#endif /* HF_BLOCK_H */
