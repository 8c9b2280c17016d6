/*
 * teeny_cache8 -- C ABI of the 8-bit key/value cache (libteeny_b200.so): appending tokens, causal attention over the cache with
 * the attention weight that every cached token received, and evicting tokens by those weights.
 *
 * A cache has slots, one for each sequence.  Keys k [slots, kv_heads, max_cached, dim] and values v [.., vdim] are E4M3 numbers,
 * one byte each, with a scale for each block of `block` tokens and kv head: k_scale, v_scale [slots, kv_heads, ceil(max_cached /
 * block)] f32.  A code c of a block with scale s stands for s * c.  Scales are powers of two, the smallest with |x| <= 448 s for
 * the block's numbers and not below 2^-126, so that a block whose scale grows can be held at the new one by shifting exponents:
 * only numbers that leave E4M3's normal range are rounded again.  weights [slots, kv_heads, max_cached] f32 or null: the attention
 * weight that each cached token received, summed over the query heads of its kv head.
 *
 * Step tables are those of teeny_hybrid.h: seqs, device int32 [n_seqs][4] = {slot, position, first row, tokens}; max_len: the longest
 * entry, or anything above it, and at least 1 (a call whose entries are all empty is refused).  host_seqs: the same table in host memory, or
 * null.  With it an entry that does not fit (slot, position + tokens, rows) and a slot that comes twice in a call that writes to it are refused.  The kernels go by the device's table, which a replayed graph may
 * have moved on since the call was made, and leave out entries that do not fit; one longer than max_len does not.  A position is the
 * index of a token's row in the cache; after an eviction that is no longer its position in the text, which only the caller's
 * rotations need.
 *
 * f32: element type of k, v, q, out and gate (0 bf16, 1 f32).  Row strides are in elements, heads lie side by side within a row.
 * dim and vdim are multiples of 16 up to 128, block is 16, 32, 64 or 128, the caches' bases are 16-byte aligned.
 * All pointers are device pointers owned by the caller unless stated; nothing here allocates device memory, and scratch holds
 * no results from one call to the next.  Status codes are those of teeny_b200.h.
 */
#ifndef TEENY_CACHE8_H_
#define TEENY_CACHE8_H_

#include "teeny_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  int slots, kv_heads, max_cached, dim, vdim, block;
} teeny_cache8_shape;

enum { TEENY_CACHE8_COUNTER_BYTES = 4096 };

/* Tokens k [rows, ldk], v [rows, ldv] of every entry into the cache, at its position and behind.  A block that holds older tokens of
 * the entry (those before its position) keeps at least its scale, and they are rounded to the new one; what a block held at or behind
 * the entry's position does not count.  NaN and infinities become NaN and do not count for the scale.  weights (or null) are set to zero for the new tokens. */
int teeny_cache8_append(int f32, const teeny_cache8_shape* shape, void* k, void* v, float* k_scale, float* v_scale, float* weights,
                        const void* k_new, long long ldk, const void* v_new, long long ldv, int rows, const int* seqs,
                        const int* host_seqs, int n_seqs, int max_len, teeny_stream_t stream);

/* Causal grouped-query attention of every entry's tokens over the cache, which holds their own keys and values already: score =
 * (q . k) * score_scale, with softcap > 0 softcap * tanh(score / softcap) (from 1e-30 to 1e30); sink [heads] or null: exp(sink) joins the softmax
 * denominator; gate [rows, ldg] (heads vdim apart) or null: the output is multiplied by sigmoid(gate).  lse [rows, heads] or
 * null: logarithm of the denominator, the sink's part included.  weights (or null): for every live token of the entries' slots
 * weights <- weight_decay * weights + the probabilities that the entry's tokens and query heads gave it; with weight_decay 0 what
 * was there is not read.  The gate does not count there.  Rows of out that belong to no entry stay as they are; no two entries have
 * a row in common (refused where host_seqs shows it).  Sums are made in
 * a fixed order: the same call gives the same bits.
 * Sums and statistics are f32.  Before the product with the values a probability is rounded to f16 (f32 calls: to 22 bits), and to bf16 in the entries of bf16
 * calls with max(32, 192 / (heads / kv_heads)) tokens and more whose rows lie on 16 bytes, which the tcgen05 kernel takes.  In f16 a probability
 * stands multiplied by its value block's scale, relative to the largest scale that the row sees: below 2^-28 that loses bits, below 2^-38 it is lost (f32 calls:
 * 2^-39, 2^-49).
 * scratch, on 32 bytes: its first TEENY_CACHE8_COUNTER_BYTES are zero before the first call, and every call leaves them zero (after a device error they have to be
 * made zero again).  Calls of any sizes may share it, evictions among them, as long as they follow one another.  out must not overlap q. */
size_t teeny_cache8_attention_scratch_bytes(const teeny_cache8_shape* shape, int f32, int heads, int rows, int n_seqs, int max_len,
                                            int with_weights);
int teeny_cache8_attention(int f32, const teeny_cache8_shape* shape, const void* k, const void* v, const float* k_scale,
                           const float* v_scale, float* weights, float weight_decay, const void* q, long long ldq, void* out,
                           long long ldo, int rows, int heads, float score_scale, float softcap, const float* sink, const void* gate,
                           long long ldg, float* lse, void* scratch, size_t scratch_bytes, const int* seqs, const int* host_seqs,
                           int n_seqs, int max_len, teeny_stream_t stream);

/* Thins out every entry's slot, whose live tokens are the first `position` of the cache (first row and tokens of an entry are not used): each kv
 * head keeps its last `recent` tokens and those of the others with the largest weights (equal ones: the lowest index; NaN counts as the
 * least), `keep` in all, and they move to the front in their order, with scales made anew from what is kept.  A slot with at most
 * `keep` tokens keeps them all.  The slot's next token belongs at min(position, keep).  kept [n_seqs, kv_heads, keep]: the kept
 * tokens' indices before, -1 behind the last.  Rows of the cache behind the kept tokens, and their weights, stay as they are.  scratch: on 16 bytes. */
size_t teeny_cache8_evict_scratch_bytes(const teeny_cache8_shape* shape, int n_seqs, int keep);
int teeny_cache8_evict(const teeny_cache8_shape* shape, void* k, void* v, float* k_scale, float* v_scale, float* weights, int keep,
                       int recent, int* kept, void* scratch, size_t scratch_bytes, const int* seqs, const int* host_seqs, int n_seqs,
                       teeny_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* TEENY_CACHE8_H_ */
