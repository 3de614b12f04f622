/*
 * sgq_decoder.h — the fp32 operators that sit between the quantized linears of a LLaMA-style
 * decoder block (RMSNorm, rotary embedding + KV-cache store, single-query attention over the
 * cache, SiLU gate), and the INT8 form of that cache, exported from the same library as sgq.h.
 *
 * They exist so that a whole greedy-decode step (sixteen blocks, ~200 launches) can be recorded
 * into one CUDA graph and replayed without host work: every quantity that changes from step to
 * step (the position in the cache) is read from DEVICE memory, so the recorded launches stay valid.
 * Arithmetic is fp32 throughout and follows the reference's operators:
 *
 *   sgqd_add_rmsnorm     sovereigngrad::rms_norm            src/ops.cpp:1532-1564
 *   sgqd_rope_kv_store   sovereigngrad::rotary_embedding    src/ops.cpp:1714-1745
 *                        nn::RotaryEmbedding tables         include/sovereigngrad/nn.hpp:583-607
 *   sgqd_attn_decode     nn::CausalSelfAttention            include/sovereigngrad/nn.hpp:503-560
 *                        (last row of the causal softmax(q k^T / sqrt(d)) v; the reference has no
 *                        KV cache and recomputes every row, models.hpp:262-300) + rotary_embedding
 *   sgqd_attn_prefill    causal attention with online softmax  src/cuda_kernels.cu:1323-1394
 *   sgqd_silu_mul        nn::SwiGLU gate                    include/sovereigngrad/nn.hpp:151-156
 *                        simd::vec_silu                     include/sovereigngrad/simd.hpp:103-108
 *   sgqd_embedding       sovereigngrad::embedding           src/ops.cpp:2624-2659
 *   sgqd_rope_kv_store_int8, sgqd_kv_load_int8, sgqd_attn_decode_int8, sgqd_attn_decode_prefix_int8
 *                        rotary_embedding and CausalSelfAttention as above over keys and values
 *                        that are held as quantization::quantize_int8 holds a row
 *                        (src/quantization.cpp:22-78)
 *   sgqd_argmax_rows     greedy choice in NanoLLaMA::generate  include/sovereigngrad/models.hpp:291-298
 *
 * Conventions are those of sgq.h: device pointers owned by the caller, `stream` is a cudaStream_t
 * passed as void*, calls enqueue and return an sgq_status, nothing is allocated.
 */
#ifndef SGQ_DECODER_H
#define SGQ_DECODER_H

#include "sgq.h"

#ifdef __cplusplus
extern "C" {
#endif

/* h[rows, dim] += delta (skipped when delta is NULL), then out = h * rsqrt(mean(h^2) + eps) * gamma.
 * h is updated in place: it is the residual stream.  out may not alias h.
 * prepared_out (optional, NULL to skip): also writes out in the prepared-activation format of
 * sgq.h (sgq_prepared_x_bytes(rows, dim) bytes, 256-byte aligned) for sgq_linear_int4_prepared. */
SGQ_API int sgqd_add_rmsnorm(float* h, const float* delta, const float* gamma, float eps, int64_t rows, int64_t dim,
                             float* out, void* prepared_out, size_t prepared_bytes, void* stream);

/* qkv[batch * t_new, 3 * n_heads * head_dim] holds, per token, the query, key and value rows of
 * n_heads heads (token m = b * t_new + i is the i-th new token of sequence b, at position
 * *pos0 + i).  Rotates q in place, and stores the rotated k and the v of every new token into
 * k_cache / v_cache[batch, n_heads, max_seq, head_dim].  cos / sin are [max_seq, head_dim / 2]
 * tables (pair (d, d + head_dim/2), angle pos * base^(-2d/head_dim)).  pos0 is a DEVICE int32:
 * the number of tokens already in the cache.  Tokens whose position would be >= max_seq are
 * skipped (nothing is written out of bounds).  head_dim must be a multiple of 8. */
SGQ_API int sgqd_rope_kv_store(float* qkv, int64_t batch, int64_t t_new, int64_t n_heads, int64_t head_dim,
                               const float* cos_table, const float* sin_table, const int32_t* pos0,
                               float* k_cache, float* v_cache, int64_t max_seq, void* stream);

/* One decode step of attention for one NEW token per sequence, fused with that token's rotary
 * embedding and cache append.  qkv[batch, qkv_stride] holds the un-rotated query, key and value of
 * the token at position *pos0 (same layout as above, t_new = 1; qkv is not modified).  The kernel
 * rotates q and k, appends k and v to the caches at position *pos0, and writes
 *   out[b, h*head_dim + d] = sum_{t <= pos0} softmax_t(q . k_t / sqrt(head_dim)) v_t[d].
 * Do not call sgqd_rope_kv_store for the same token.  If *pos0 is outside [0, max_seq) nothing is
 * stored and the query attends to the cache contents only.  head_dim must be 64 or 128.
 * prepared_out (optional, prepared_bytes >= sgq_prepared_x_bytes(batch, n_heads * head_dim)): the rows
 * out[b, 0 .. n_heads*head_dim) additionally in the decode kernel's prepared form, bit-identical to
 * sgq_prepare_x on `out`, so that the linear behind the attention (sgq_linear_int4_prepared) needs no
 * conversion launch. */
SGQ_API int sgqd_attn_decode(float* qkv, int64_t qkv_stride, int64_t batch, int64_t n_heads, int64_t head_dim,
                             const float* cos_table, const float* sin_table, float* k_cache, float* v_cache,
                             int64_t max_seq, const int32_t* pos0, float* out, int64_t out_stride, void* prepared_out,
                             size_t prepared_bytes, void* stream);

/* Causal attention of t_new NEW tokens per sequence (the prompt pass), after sgqd_rope_kv_store has rotated
 * q in place and appended the rotated keys and the values: token i of sequence b (row b * t_new + i of qkv,
 * position *pos0 + i) attends to cache positions 0 .. *pos0 + i,
 *   out[b * t_new + i, h*head_dim + d] = sum_{t <= pos0 + i} softmax_t(q . k_t / sqrt(head_dim)) v_t[d],
 * computed with an online softmax over tiles of 32 keys like the reference's attention
 * (src/cuda_kernels.cu:1323-1394).  head_dim must be 64 or 128; batch * n_heads <= 65535. */
SGQ_API int sgqd_attn_prefill(const float* qkv, int64_t qkv_stride, int64_t batch, int64_t t_new, int64_t n_heads, int64_t head_dim,
                              const float* k_cache, const float* v_cache, int64_t max_seq, const int32_t* pos0, float* out,
                              int64_t out_stride, void* stream);

/* The same attention on the tensor cores, for prompt passes whose linears run on the bf16 tensor-core path anyway
 * (SGQ_PATH_TC_BF16): q, k, v and the softmax weights are rounded to bf16, the products accumulate in fp32, the
 * softmax is fp32.  Within 2e-2 of the largest output of sgqd_attn_prefill (measured ~3e-3).  head_dim must be 128.
 * (No counterpart in the reference, whose attention is fp32.) */
SGQ_API int sgqd_attn_prefill_bf16(const float* qkv, int64_t qkv_stride, int64_t batch, int64_t t_new, int64_t n_heads, int64_t head_dim,
                              const float* k_cache, const float* v_cache, int64_t max_seq, const int32_t* pos0, float* out,
                              int64_t out_stride, void* stream);

/* gate_up[rows, 2 * hidden] = [gate | up] per row; out[rows, hidden] = gate / (1 + exp(-gate)) * up.
 * prepared_out: as for sgqd_add_rmsnorm, the prepared form of out[rows, hidden]. */
SGQ_API int sgqd_silu_mul(const float* gate_up, int64_t rows, int64_t hidden, float* out, void* prepared_out,
                          size_t prepared_bytes, void* stream);

/* Column-sharded forms of the two operators whose output is a column slice per GPU (the heads of this rank, the
 * SwiGLU columns of this rank): the result goes straight into the full-width buffer of EVERY rank,
 * out_ranks[r][row * stride + col_offset + c] (plain peer stores; out_ranks is a HOST array of `world` device
 * pointers, as for sgq_linear_int4_allgather), so no copy kernel stands between the operator and sgq_peer_barrier.
 * Otherwise as sgqd_attn_decode (without the prepared form) and sgqd_silu_mul. */
SGQ_API int sgqd_attn_decode_allgather(float* qkv, int64_t qkv_stride, int64_t batch, int64_t n_heads, int64_t head_dim,
                                       const float* cos_table, const float* sin_table, float* k_cache, float* v_cache,
                                       int64_t max_seq, const int32_t* pos0, float* const* out_ranks, int world,
                                       int64_t out_stride, int64_t col_offset, void* stream);
SGQ_API int sgqd_silu_mul_allgather(const float* gate_up, int64_t rows, int64_t hidden, float* const* out_ranks, int world,
                                    int64_t ld, int64_t col_offset, void* stream);

/* out[i, :] = table[ids[i], :] for rows indices (ids: DEVICE int64).  An id outside [0, vocab) gives a row
 * of zeros, as in the reference (src/ops.cpp:2643-2649); the table is never read out of bounds. */
SGQ_API int sgqd_embedding(const float* table, int64_t vocab, int64_t dim, const int64_t* ids, int64_t rows, float* out,
                           void* stream);

/* out[r] = first index of the strict maximum of x[r, 0..n) (row stride ld), a DEVICE int64 per row: the
 * reference's greedy choice keeps the first of equal candidates (models.hpp:291-298).  NaN never wins;
 * a row of NaNs (or n == 0) gives 0. */
SGQ_API int sgqd_argmax_rows(const float* x, int64_t rows, int64_t n, int64_t ld, int64_t* out, void* stream);

/* ---- the INT8 key/value cache ------------------------------------------------------------------------------------
 *
 * Keys and values of a decoder block as INT8 codes with one fp32 scale per (sequence, kv head, position): head_dim + 4
 * bytes per row in the place of 4 * head_dim.  A row r is held as sgq_quantize_int8 holds a row (SGQ_PER_ROW), bit for bit:
 *   a = max(1e-8, max |r|),  scale = a / 127,  code = clamp(round_half_away(r * (127 / a)), -127, 127),
 * all in fp32 (a NaN gets code +127; an infinity makes the scale infinite), and stands for code * scale.  Keys are rotated
 * before they are quantized, every product and sum of the rotation rounded to fp32, so the codes depend on the inputs alone.
 * The struct holds DEVICE pointers owned by the caller; it is read during the call only.  codes: [batch, n_kv_heads,
 * max_seq, head_dim], 16-byte aligned; scales: [batch, n_kv_heads, max_seq].  The four arrays, rows, outputs and workspace of a
 * call share no memory (SGQ_ERR_BAD_ARGUMENT where they do), but for what is said below.  Query head h reads kv head
 * h / (n_heads / n_kv_heads).  `pos` is a DEVICE int32 per sequence (pos_stride 1) or one for all (pos_stride 0): the tokens
 * of the sequence that are in the cache.  Rows of qkv are [n_heads | n_kv_heads | n_kv_heads] heads of head_dim values,
 * qkv_stride floats apart; cos / sin tables as above, [table_rows, head_dim / 2], 16-byte aligned. */
typedef struct sgqd_cache_int8 {
    int8_t* k_codes;
    float* k_scales;
    int8_t* v_codes;
    float* v_scales;
    int64_t batch, n_kv_heads, max_seq, head_dim;
} sgqd_cache_int8;

/* t_new new tokens per sequence (row b * t_new + i of qkv: token i of sequence b, at position pos[b] + i): writes the rotated
 * queries to q_out (rows q_stride floats apart; q_out == qkv with the same stride rotates in place, any other overlap is
 * not allowed), and the rotated keys and the values, quantized, into the cache.  n_new (optional, DEVICE int32 per sequence):
 * only the first n_new[b] tokens of sequence b exist (padded prompts).  rope_offset (optional, ONE DEVICE int32): added to
 * the position for the rotation, for sequences behind a shared prefix.  table_rows >= max_seq.  A token that does not exist,
 * whose position lies outside [0, max_seq) or whose rotation lies outside the tables changes nothing: no query and no row
 * is written.
 * head_dim: a multiple of 8, at most 256. */
SGQ_API int sgqd_rope_kv_store_int8(const float* qkv, int64_t qkv_stride, int64_t t_new, int64_t n_heads, const float* cos_table,
                                    const float* sin_table, int64_t table_rows, const int32_t* pos, int64_t pos_stride, const int32_t* n_new,
                                    const int32_t* rope_offset, float* q_out, int64_t q_stride, const sgqd_cache_int8* cache,
                                    void* stream);

/* Reads positions [0, rows) back as fp32: k_out / v_out[b, h, out_row0 + t, :] = code * scale for b < batch, outputs
 * [batch, n_kv_heads, out_max_seq, head_dim] (what the prompt attention takes as its caches).  A cache of one sequence
 * (a shared prefix) is read into every one of `batch` sequences.  Other rows of the outputs are left as they were.
 * head_dim: a multiple of 8, at most 256. */
SGQ_API int sgqd_kv_load_int8(const sgqd_cache_int8* cache, int64_t rows, int64_t batch, float* k_out, float* v_out,
                              int64_t out_max_seq, int64_t out_row0, void* stream);

/* One decode step of attention for one NEW token per sequence (row b of qkv, position pos[b]): appends its rotated key and
 * its value to the cache, quantized as above, and writes
 *   out[b, h*head_dim + d] = sum_{t <= pos[b]} softmax_t(q_h . k_t / sqrt(head_dim)) v_t[d],
 * k_t and v_t being the values the cache then holds, the new token's included.  qkv is read only.  A sequence whose pos lies
 * outside [0, max_seq) takes no part: nothing is stored and its output row is zero.  Rows at positions behind pos may be read, as far as
 * max_seq, but do not enter: they may hold anything, and another stream may write them meanwhile.
 *   Range: a NaN or an infinity in a query gives NaN in its head's output, and so does a row with a scale that is not finite, a
 * rotated query value beyond 2^122 or a largest score beyond the fp32 range on either side.  Keys may have any size; values too behind
 * 2^18 positions, and up to FLT_MAX * 2^18 / n behind n; positions whose weight times value scale is below 2^-80 may count as nothing.
 *   Errors: scores are exact integer products of the codes with the query as 24-bit fixed point relative to the largest |value| of its row,
 * off by at most 2^-21 * max |q| * sum |k_t| / sqrt(head_dim).  That is an fp32 evaluation's error where the query's values are of one
 * order; where one is far larger than the others and its keys are small, it is larger than that by as much.  Softmax weights (times
 * value scale) are 23-bit fixed point relative to the largest of the 32 to 128 positions that are read together (for 33 query rows and
 * more per kv head behind a prefix the sum of two 16-bit floats, 22 bits of a weight and 2^-37 of the largest).  Exponentials are off
 * by 2 ulp; sums are fp32.  table_rows >= max_seq.  head_dim must be 64 or
 * 128, max_seq at most 2^30.  out may not overlap qkv.  prepared_out: as for sgqd_attn_decode.  workspace: as many bytes as the query says (0: none is read; caches that
 * may grow long need some), 256-byte aligned; it holds nothing from one call to the next, and calls that may run at the
 * same time need one each.  The query's answer follows from the sizes alone. */
SGQ_API size_t sgqd_attn_decode_int8_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                                     int64_t max_seq);
SGQ_API int sgqd_attn_decode_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table,
                                  const float* sin_table, int64_t table_rows, const int32_t* pos, int64_t pos_stride,
                                  const sgqd_cache_int8* cache, float* out, int64_t out_stride, void* prepared_out, size_t prepared_bytes, void* workspace, size_t workspace_bytes,
                                  void* stream);

/* The same for sequences that begin with the same *prefix_len tokens (ONE DEVICE int32, taken as at least 0 and at most
 * prefix->max_seq), whose rows lie once in `prefix`, a cache of one sequence with the same heads: every query attends to
 * the prefix rows and to its own rows 0 .. pos[b], which stand at positions *prefix_len + t of its sequence (the rotation of
 * the new token included; table_rows >= prefix->max_seq + max_seq).  The prefix is read once for the whole
 * batch and shares no memory with `cache` (refused).  workspace: as for sgqd_attn_decode_int8 (0 bytes only for sizes that are refused). */
SGQ_API size_t sgqd_attn_decode_prefix_int8_workspace_bytes(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                                            int64_t max_seq, int64_t prefix_max);
SGQ_API int sgqd_attn_decode_prefix_int8(const float* qkv, int64_t qkv_stride, int64_t n_heads, const float* cos_table,
                                         const float* sin_table, int64_t table_rows, const int32_t* pos,
                                         int64_t pos_stride, const sgqd_cache_int8* cache, const sgqd_cache_int8* prefix, const int32_t* prefix_len,
                                         float* out, int64_t out_stride, void* prepared_out, size_t prepared_bytes, void* workspace,
                                         size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SGQ_DECODER_H */
