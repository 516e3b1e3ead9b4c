/*
 * mars5_paged.h  --  argument structures of the paged serving entry points of libmars5_hip.so.  Included by mars5_hip.h, which
 * declares the functions and states the conventions (device pointers, element strides, caller-owned buffers, status codes).
 */
#ifndef MARS5_PAGED_H
#define MARS5_PAGED_H
#include <stdint.h>

/* ------------------------------------------------------------------------------------
 * Paged serving: a KV cache in blocks that many requests share, several new tokens per request and step (prompt chunks, drafted
 * tokens), n_heads / n_kv_heads query heads per kv head.  One step = m5_paged_plan, then per layer m5_paged_rope_cache and
 * m5_paged_attention, then m5_draft_verify; its keep_len is the next step's (rejected drafts are rolled back there).  Blocks come
 * back from a request's end only: those behind a window stay with it until it ends.  All lengths live in device memory: a step is
 * capturable and needs no host read-back.  Caches: block, head and slot strides in elements, features contiguous; block_size a
 * power of two <= 1024; a block id outside [0, n_blocks) is never dereferenced.  Padding (rows from q_start[n_seq] on) is neither
 * computed nor written.
 * ------------------------------------------------------------------------------------ */

/* Block tables, slot map, positions and row offsets of one step, from the requests' lengths, in one launch.
 * Request b holds seq_len[b] positions in ceil(seq_len / block_size) blocks (block_table row b); it keeps the first keep_len[b] of
 * them (rejected drafts and finished requests, keep 0, are given back) and adds new_len[b].  Afterwards seq_len = keep + new.
 * keep_len may be seq_len itself (all is kept).
 *   q_start[n_seq + 1]  exclusive prefix sums of new_len: the step's rows, packed by request
 *   positions[r]        position of row r in its request;  slot_map[r] = block * block_size + offset;  rows past the last: -1
 *                       (both NULL: the rows are not described, n_rows is not looked at, e.g. a roll-back)
 *   free_blocks[n_blocks], state[M5_PST_FREE]   a stack of free block ids.  Blocks given back are pushed from the last request's last
 *                       page to the first's, blocks taken are popped by request and page: rolling a step back restores it.
 *                       What block_table holds behind a request's pages is not defined.
 *   state[M5_PST_STATUS] 0; > 0: that many blocks short; < 0: -1 - b = request b is not valid (a negative length, keep > held, more
 *                       positions than its table row holds), b = n_seq: more rows than n_rows, n_seq + 1: more blocks given back
 *                       than n_blocks.  Not 0 = nothing is taken or changed and the step has no rows: q_start 0, maps -1.
 * state: M5_PST_WORDS int32, zero-filled once, [M5_PST_FREE] set; words from 3 on are the library's.  n_seq <= 4096. */
#define M5_PST_FREE 0
#define M5_PST_STATUS 1
#define M5_PST_ROWS 2
#define M5_PST_WORDS 8
typedef struct {
    int32_t* seq_len; const int32_t* keep_len; const int32_t* new_len;
    int32_t n_seq, table_width, n_blocks, block_size, n_rows;
    int32_t* block_table; int64_t table_rs;
    int32_t* free_blocks; int32_t* state;
    int32_t* q_start; int32_t* slot_map; int32_t* positions;
} M5PagedPlanArgs;

/* Norms of the q and k heads, the position rotation and the cache write in one pass over the packed projections
 * (the paged form of m5_rope_cache).  Row r of qkv = [n_heads | n_kv_heads | n_kv_heads] x head_dim; q and k heads are
 * y = x rsqrt(mean(x^2) + eps) w when q_norm / k_norm (fp32 [head_dim]) are given, then the first 2 n_pairs features are
 * rotated by rope[positions[r]] (fp32 [n_pos][n_pairs][cos, sin]): features (2i, 2i + 1) when interleaved, (i, n_pairs + i)
 * otherwise.  fp32 throughout, rounded once.  q -> q_out, k and v -> slot slot_map[r] of the caches.  A row with a slot or position
 * out of range (padding: -1) is skipped and its q_out row left as it was; slots must be distinct (two rows of one slot: a mixture of
 * their values).  q_out may be the q part of qkv itself.  head_dim 64 or 128; 2 n_pairs <= head_dim, n_pairs % 8 == 0; pointers and strides multiples of 16 bytes. */
typedef struct {
    const void* qkv; int64_t qkv_rs;
    int32_t n_rows, n_heads, n_kv_heads, head_dim;
    const float* q_norm; const float* k_norm; float eps;
    const float* rope; int32_t n_pos, n_pairs, interleaved;
    const int32_t* positions; const int32_t* slot_map;
    void* q_out; int64_t q_rs, q_hs;
    void* k_cache; int64_t k_bs, k_hs, k_ss;
    void* v_cache; int64_t v_bs, v_hs, v_ss;
    int32_t n_blocks, block_size;
} M5PagedRopeArgs;

/* Attention of every request's new tokens over its paged cache: query row r of request b (rows q_start[b] .. q_start[b + 1])
 * stands at position p = seq_len[b] - (q_start[b + 1] - r) and sees the keys max(0, p - window + 1) .. p (window 0: from 0 on); query head
 * h reads kv head h / (n_heads / n_kv_heads).  Online softmax in fp32, scores never stored.  16-bit calls round a key's weight to their
 * type for the product with its value (once; sums in fp32, in bf16 tiles of 128 rows of the rounded weights); fp32 calls round none.
 * A row that sees no key, or only keys whose score is -inf, gets zeros; a NaN among the scores that a row sees makes the row NaN;
 * keys on a block id out of range are not seen.
 * Keys past a request's length and pages behind it are never used, whatever they hold; row offsets that do not ascend compute
 * nothing or rows of theirs twice, inside the buffers.  max_new: upper bound of the new tokens of one request (speed only: it
 * selects the tiling).
 * workspace (may be NULL): scratch for keys split over workgroups when there are few rows; zero-filled once by the caller, left
 * ready for the next call of any types and shapes that is given the same bytes; calls that may run at the same time need one
 * each; no other operator's; 16-byte aligned.  More bytes allow more splits; m5_paged_attention_workspace tells how many bytes
 * the largest split of these shapes uses.
 * head_dim 64 or 128; n_seq <= 4096; at most 2^30 positions per table row; strides of blocks below 64 GB, of slots below 64 MB; pointers
 * and strides multiples of 16 bytes. */
typedef struct {
    const void* q; int64_t q_rs, q_hs;
    const void* k_cache; int64_t k_bs, k_hs, k_ss;
    const void* v_cache; int64_t v_bs, v_hs, v_ss;
    const int32_t* block_table; int64_t table_rs; int32_t table_width, n_blocks, block_size;
    int32_t n_seq, n_rows, max_new, n_heads, n_kv_heads, head_dim, window;
    const int32_t* seq_len; const int32_t* q_start;
    float scale;
    void* out; int64_t o_rs, o_hs;
    void* workspace; int64_t workspace_bytes;
} M5PagedAttnArgs;

/* Drafted tokens against the target's probabilities (speculative sampling), one launch.  Request b owns the rows r0 = row_start[b]
 * .. r1 = row_start[b + 1]: row r's token tokens[r] was fed to the target, target[r] are the probabilities of what follows it, and
 * tokens[r + 1], r + 1 < r1, is a draft drawn from draft[r] (draft NULL: certain, probability 1).  Draft r + 1 is accepted iff
 * uniforms[r] * draft[r][d] < target[r][d], d = tokens[r + 1] (fp32; an id outside [0, vocab) is not accepted), up to the first that is
 * not.  Then one more token is drawn: after a rejection in row r from max(target[r] - draft[r], 0) (draft NULL: target[r] without d;
 * if nothing is left, target[r]), after the last row from target[r1 - 1]: the lowest v with the largest weight[v] / noise[b][v]
 * (noise: Exp(1) draws as in m5_ar_sample; NaN and weights <= 0 count as 0).
 *   out_tokens[b] = accepted drafts, the drawn token, then -1;  n_out[b] = their number (0 for a request without rows)
 *   keep_len[b] = seq_len[b] - (r1 - r0) + n_out[b] (both NULL: not wanted): positions that m5_paged_plan keeps in the next step
 * row_start is the plan's q_start only where a request's rows are one sampled token and the drafts behind it: a prompt's rows would be taken
 * for drafts.  Of a prompt's chunk only the last row is verified (none while more of the prompt is to come): rows and offsets of
 * their own; keep_len then keeps the chunk whole.
 * dtype: that of target and draft.  A request of more than out_width rows counts its first out_width rows.
 * plan_state (may be NULL): the state of the m5_paged_plan that opened the step.  If that refused the step (status not 0), every
 * request counts as one without rows and keep_len is left as it was: seq_len still holds what the step before rejected, so a keep_len
 * given to the plan must outlive it, and the step can be tried again once there are blocks.
 * workspace (may be NULL): M5_DRAFT_WS_BYTES per request, kept as m5_paged_attention's; lets a row be split over workgroups. */
#define M5_DRAFT_WS_BYTES 32
typedef struct {
    const void* target; int64_t t_rs;
    const void* draft; int64_t d_rs;
    int32_t n_rows, vocab, n_seq, out_width;
    const int64_t* tokens; const int32_t* row_start;
    const float* uniforms; const float* noise; int64_t noise_rs;
    int64_t* out_tokens; int64_t out_rs; int32_t* n_out;
    const int32_t* seq_len; int32_t* keep_len;
    void* workspace; int64_t workspace_bytes;
    const int32_t* plan_state;
} M5DraftVerifyArgs;

#endif /* MARS5_PAGED_H */
