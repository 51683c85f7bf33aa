/* sx8_draft.h -- drafted tokens: the trees that they form and which of them the target model keeps (libsx8_hip.so).
 *
 * A pass over drafted tokens brings each slot n rows: row 0 is the slot's last token, whose K/V is not in the cache yet, the
 * others are drafted ones; row i follows row parents[i] < i of its slot.  The pass is sx8_draft_tree, for every layer
 * sx8_kv4_append_rope and sx8_kv4_attend_tree, then sx8_draft_verify on the logits and sx8_kv4_keep (sx8_paged.h); with their forms
 * sx8_draft_verify_within and *_marked nothing that was not written can become part of a sequence.
 * The reference has no counterpart (its runtime decodes one token a step, scripts/infer_sx8.py:109-173).
 * Conventions as in sx8_paged.h: rows are packed by slot (slot s has the rows cu[s] .. cu[s + 1] - 1; cu (n_slots + 1)
 * int32, kept within the call's rows), nothing is allocated and nothing synchronised, every call can be captured in
 * a graph.  n_slots <= 4096.
 */
#ifndef SX8_DRAFT_H
#define SX8_DRAFT_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Masks and depths of the slots' trees from parents (rows) int32: bit j of a row's mask (rows, words) uint64 is set where row j
 * is the row itself or an ancestor, depth (rows) int32 counts its ancestors.  A parent outside 0 .. i - 1 is none.  Rows of a
 * slot from 64 words on (words 1..4) are no part of a tree: mask 0 and depth -2^30, a place before every table.  Rows of no slot
 * are left as they are. */
int32_t sx8_draft_tree(const int32_t* parents, const int32_t* cu, int64_t n_slots, int64_t rows, int32_t words,
                       uint64_t* mask, int32_t* depth, void* stream);

/* Which drafted tokens the target keeps, and the token that follows them.  logits (rows, V) are the target's for the
 * token behind each row (row stride in elements; dtype 0 fp16, 1 bf16, 2 float32), tokens (rows) int64, u (rows) float32 random
 * numbers in [0, 1), temperature (n_slots) float32, or NULL: t for every slot.
 *   Where the temperature is above zero, p = softmax(logits / temperature) of the current row, row 0 at first.  Its children are
 *   tried in the order of their rows; child i with token x is kept if u[i] < p(x), and is the current row then.  Otherwise what
 *   is known of x is taken out of p and p is scaled to a sum of 1 for the next child:
 *     without draft probabilities (NULL): p(x) = 0 (drafts that were chosen, not drawn: no token is lost or favoured);
 *     with probs (rows, V), row r the distribution that the children of row r were drawn from: child i is kept if
 *     u[i] probs(x) < p(x), otherwise p = max(p - probs, 0).  Rows as logits have them, of probs_dtype.
 *   When no child is left, the next token is drawn from p: the lowest k with p(0) + .. + p(k) > u[row 0] (the sum of p).
 *   Where p has no sum left (u of 1 or more, or roundings) p is the target's own again.
 *   Elsewhere (temperature not above zero) a child is kept if its token is the first of the largest logits, which is the
 *   next token as well; u may be NULL if t and temperature say that for all slots (t <= 0, temperature NULL).
 * A NaN logit counts as -infinity; +infinities share a row between them; a row of -infinities keeps no child and gives no
 * token (-1).  A token outside 0 .. V - 1 is never kept.  Exponentials and sums are held in 64 bits, so that tokens do
 * not depend on the order of a sum.
 * sx8_draft_verify_within: with depth (rows) int32 as sx8_draft_tree gives it (NULL: as sx8_draft_verify).  A row whose depth is below
 * zero is no part of its tree: neither sx8_kv4_append_rope nor sx8_kv4_attend_tree knew it, so it is never kept; a slot whose
 * row 0 is such a row keeps nothing (counts 0, next -1).
 * path (rows) int32: slot s has the row numbers in the slot of what it keeps, row 0 first, in path[cu[s]] .. , then -1;
 * counts (n_slots) int32: how many (0: no rows); next (n_slots) int64: the token that follows (-1: none).
 * rows up to 2^22, V up to 2^27; workspace (256-byte aligned, sx8_draft_verify_workspace_bytes, no clearing needed). */
int64_t sx8_draft_verify_workspace_bytes(int64_t n_slots, int64_t rows, int64_t V);
int32_t sx8_draft_verify(const void* logits, int64_t logits_stride, int32_t dtype, const int64_t* tokens,
                         const int32_t* parents, const int32_t* cu, int64_t n_slots, int64_t rows, int64_t V,
                         const float* u, const float* temperature, float t, const void* probs, int64_t probs_stride,
                         int32_t probs_dtype, int32_t* path, int32_t* counts, int64_t* next, void* workspace,
                         int64_t workspace_bytes, void* stream);
int32_t sx8_draft_verify_within(const void* logits, int64_t logits_stride, int32_t dtype, const int64_t* tokens,
                                const int32_t* parents, const int32_t* depth, const int32_t* cu, int64_t n_slots, int64_t rows,
                                int64_t V, const float* u, const float* temperature, float t, const void* probs,
                                int64_t probs_stride, int32_t probs_dtype, int32_t* path, int32_t* counts, int64_t* next,
                                void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SX8_DRAFT_H */
