/* b200serve - serving with drafted tokens over a paged 4-bit KV cache.
 *
 * The reference keeps one sequence's cache in fp32 or fp16 (KVCache, inference/kv_cache.h:11-138), rotates
 * whole heads by unscaled positions (rope_forward_cached, cuda/cuda_ops.h:92) and has neither pages nor
 * drafted tokens; nothing here replaces a function of its op API.  One step of a server that checks drafts:
 *
 *   b200_paged_plan            lengths and new rows of the requests -> pages, positions, slots, row offsets
 *   b200_rope_forward_scaled   rotary positions of the step's queries and keys
 *   b200_kv4_store             the step's keys and values into the 4-bit pages
 *   b200_attention_paged_kv4   every row against its sequence's pages
 *   b200_verify_drafts         drafts kept or refused, the next token drawn
 *
 * Conventions are those of b200ops.h: device pointers, the library's current stream, status codes.  None of
 * these calls allocates, synchronises or keeps anything between calls, so all of them can be captured into
 * CUDA graphs; where a call needs room, the caller gives it a workspace, any contents, 16-byte aligned, not shared by
 * calls that may overlap.
 * Lengths and offsets are read on the device when the call runs.
 *
 * The 4-bit pages.  `pages` holds num_pages pages of b200_kv4_page_bytes() bytes, 16-byte aligned, each of `page`
 * tokens: K codes [KV, page, hd/2], K scales [KV, page, hd/32], V codes, V scales, each part starting on a multiple of
 * 128 bytes from the page's start.  A token's row of hd elements (64 or 128) is cut in blocks of 32; element
 * 32 b + 4 g + i (b < hd/32, g < 8, i < 4) is nibble i, lowest first, of the row's 16-bit word g * (hd/32) + b.
 * kind 0 (Q4_0): a scale is one fp16 d, the value d * (code - 8); kind 1 (Q4_1): an fp16 pair d, m, the value
 * d * code + m.  kind 0 holds the codes and scales of b200_quantize, bit for bit; kind 1 as well, but that its step is
 * (max - min) * fp32(1/15), not a division: its last bit may differ and with it the code of a value on the border of two.  d and m beyond
 * the range of fp16 are kept as +-65504.  So every stored value is finite and no d is negative, which the attention counts on.  Slot s is token s % page of page s / page;
 * num_pages * page must fit in 31 bits, KV * page be at most 2^23. */
#ifndef B200SERVE_H
#define B200SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The pages and rows of the next step of `batch` (0 .. 2048) requests.
 *
 * ctx_lens [batch]: tokens in the cache; new_lens [batch]: rows to add (0: idle, negative: the request is finished and
 * gives its pages back); held [batch]: pages that page_table [batch, max_pages] already names for it, more than its
 * context needs after drafts were refused.  Free pages stand in a ring: free_ring [ring_size], the oldest at
 * ring_at[0] % ring_size, the end (exclusive) at ring_at[1] % ring_size, both counting up for ever (0 <= ring_at[0] <=
 * ring_at[1] <= ring_at[0] + ring_size, or the ring counts as empty and takes nothing); ring_size >= num_pages, so that no page
 * is ever lost.
 *
 * In order of b a request takes max(0, ceil((ctx + new) / page) - held) pages from the ring, until the first one that the
 * free pages or max_rows rows do not suffice for: it and every later request with new rows are refused, as is one that
 * would outgrow max_pages.  A refused request keeps what it had and gets no rows this step.  Pages given back this step are free
 * from the next one on.
 *
 * seq_lens [batch]: tokens after the step (0: finished); held_out [batch]; row_offsets [batch + 1]: rows of request b are
 * row_offsets[b] .. row_offsets[b+1] - 1; positions and slots [max_rows]: of every row, -1 behind the last one; ring_at_out [2];
 * counts [4]: rows, pages taken, pages given back, requests refused.  page_table and free_ring are updated in place;
 * seq_lens may be ctx_lens, held_out held, ring_at_out ring_at, otherwise the arrays must not overlap.  A page id of the ring or
 * table outside [0, num_pages) gives slot -1. */
int b200_paged_plan(const int32_t* ctx_lens, const int32_t* new_lens, const int32_t* held, int batch, int32_t* page_table,
                    int max_pages, int page, int num_pages, int32_t* free_ring, int ring_size, const int64_t* ring_at,
                    int64_t* ring_at_out, int32_t* seq_lens, int32_t* held_out, int32_t* row_offsets, int32_t* positions,
                    int32_t* slots, int max_rows, int32_t* counts);

/* inv_freq [rot_dim / 2] fp64 (device): base theta, frequency theta^(-2i / rot_dim), scaled for contexts longer than
 * orig_ctx by `factor` (>= 1): scaling 0 none; 1 linear (all divided by it); 2 theta * factor^(rot_dim / (rot_dim - 2))
 * as the base; 3 YaRN: divided where the original context holds fewer than `low` turns, kept where it holds more than `high`,
 * a ramp over the dimensions between (usual: 1, 32); 4 the same by wavelength, a ramp over the turns (usual: 1, 4).
 * *attn_factor_host (optional, host): what cos and sin are to be multiplied by, 1 + 0.1 ln(factor) for scaling 3, else 1. */
int b200_rope_frequencies(double* inv_freq, int rot_dim, double theta, int scaling, double factor, int orig_ctx, double low,
                          double high, double* attn_factor_host);
/* The first rot_dim (even, <= head_dim <= 1024) elements of every head turned by pos * inv_freq, the rest copied.  rope_type as
 * in b200_rope_forward_cached: 0 pairs (2i, 2i+1), 1 pairs (i, i + rot_dim/2).  q [ntok, n_heads, head_dim] with q_stride
 * floats from token to token, k [ntok, n_kv, head_dim] likewise, outputs with strides of their own; an output may be its
 * input (then with the same stride) or other columns of the same rows, else they must not overlap.  q (and q_out) or k (and k_out) may be NULL.  A row with a negative
 * position is left as it was.  The angle is taken in 64 bits and reduced before cos and sin. */
int b200_rope_forward_scaled(const float* q, const float* k, float* q_out, float* k_out, const int32_t* pos,
                             const double* inv_freq, int64_t ntok, int n_heads, int n_kv, int head_dim, int rot_dim,
                             int rope_type, int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride,
                             float attn_factor);

/* Bytes of one page (see above). */
int b200_kv4_page_bytes(int page, int KV, int hd, int kind, size_t* bytes);
/* Rows k, v [n, KV, hd] (strides in floats from row to row) into their slots; a row whose slot lies outside the cache is
 * left out.  Slots must differ; of two rows in one slot the result is some mixture. */
int b200_kv4_store(const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int32_t* slots, int64_t n,
                   void* pages, int num_pages, int page, int KV, int hd, int kind);
/* The values at the slots as fp32 rows (k or v may be NULL); a row whose slot lies outside the cache is left as it was. */
int b200_kv4_fetch(const void* pages, int num_pages, int page, const int32_t* slots, int64_t n, float* k, float* v,
                   int64_t k_stride, int64_t v_stride, int KV, int hd, int kind);

/* Attention of ragged rows over the 4-bit pages.  q, out: rows [H, hd] with q_stride / out_stride floats from row to row;
 * rows of sequence b are row_offsets[b] .. row_offsets[b+1] - 1 (NULL: row b alone), its last row the token seq_lens[b] - 1,
 * the row before it the token before, and so on (seq_lens counts the rows' own tokens, which have been stored).  A row sees the
 * tokens up to its own, with window > 0 the last `window` of them.  H a multiple of KV, hd 64 or 128.  max_rows: the most
 * rows of one sequence (it sizes the tiles; a sequence with more is still right).  page_table [batch, max_pages]; a length
 * beyond max_pages * page is cut to it; a page id outside [0, num_pages) reads as zeros.  A row before the sequence's first
 * token (more rows than tokens) is all zeros; rows of no sequence are left as they were.  fp32 accuracy: queries and
 * probabilities travel as two fp16 parts that hold 2^-24 of the largest among them (of a query's elements; of 32 tokens' weights), codes are
 * exact, sums are fp32.  q, out and pages 16-byte aligned, strides multiples of 4.  workspace: b200_attention_paged_kv4_workspace() bytes for the same H, KV, hd, max_rows (the batch
 * and the lengths do not matter). */
int b200_attention_paged_kv4_workspace(int H, int KV, int hd, int max_rows, size_t* bytes);
int b200_attention_paged_kv4(const float* q, int64_t q_stride, const int32_t* row_offsets, const void* pages, int num_pages,
                             const int32_t* page_table, const int32_t* seq_lens, float* out, int64_t out_stride, int batch,
                             int max_rows, int max_pages, int page, int H, int KV, int hd, int kind, float scale, int window,
                             void* workspace, size_t workspace_bytes);

/* Drafted tokens against the target's probabilities.  Row row_offsets[b] + j holds the target's logits after the j-th token
 * of sequence b that was fed this step, ids[row_offsets[b] + j]: the drafts are the ids of its second and later rows, checked
 * by the row before.  p = softmax(logits / temperature) (temperature <= 0: greedy, at most 1e30); q: the row of draft_probs [rows, V] that the
 * draft was drawn from (NULL: the drafter had no choice, q(x) = 1).  Draft x is kept iff u * q(x) < p(x), u = uniforms of the
 * checking row, in [0, 1); the first refusal draws from max(p - q, 0) (q = 1 at x alone if draft_probs is NULL), and if there is none
 * the next token is drawn from the p of the row behind the last draft: the first index whose cumulated mass exceeds u * (all of it), u = the
 * uniform of the sequence's last row, or from p itself where max(p - q, 0) has no mass.  Greedy: a draft is kept iff it is the arg-max
 * (the lowest index of equal ones), the next token is the arg-max.  NaN logits count as -inf; several +inf share the mass; a row
 * without any logit above -inf keeps no draft and draws -1, as does an id outside the vocabulary keep nothing.
 * accepted [batch]; tokens [batch, max_drafts + 1]: the drafts kept, the token drawn, then -1.  At most max_drafts (0 .. 255) drafts of
 * a sequence are looked at; a sequence without rows gets 0 and -1.  Masses are summed in 64 bits.  `rows`: how many rows
 * the arrays have; workspace: b200_verify_drafts_workspace(rows, V) bytes. */
int b200_verify_drafts_workspace(int rows, int V, size_t* bytes);
int b200_verify_drafts(const float* logits, int64_t logits_stride, const float* draft_probs, int64_t draft_stride,
                       const int32_t* ids, const int32_t* row_offsets, int batch, int rows, int V, float temperature,
                       const float* uniforms, int max_drafts, int32_t* accepted, int32_t* tokens, void* workspace,
                       size_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* B200SERVE_H */
