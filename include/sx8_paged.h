/* sx8_paged.h -- several sequences at once: attention of packed prompts, and a paged KV cache held
 * in 4 bits with its writer, reader, attention and page operations (libsx8_hip.so).
 *
 * These are the batched forms of the cache and attention ops of sx8_decoder.h.  The reference has no
 * counterpart (its runtime serves one sequence with the Hugging Face cache, scripts/infer_sx8.py:109-173).
 * Conventions as in sx8_hip.h: device pointers, int32_t status, stream as void*; nothing is allocated and
 * nothing synchronised, lengths and tables are read on the device, so every call can be captured in a
 * graph.  dtype: 0 = fp16, 1 = bf16 (both as 16-bit words).  Strides are in elements; a head's hd values
 * are contiguous; pointers of rows are 16-byte aligned and their strides
 * multiples of 8; output rows may not overlap each other or what the call reads, but for out on the rows of q alone.
 *
 * The cache.  A pool has n_pages pages for each layer, a page page_tokens (32, 64, 128 or 256) tokens of
 * all nk KV heads: sx8_kv4_page_bytes bytes, [head][block of 32 tokens][block bytes].  A block is
 *   K levels (16 hd bytes), V levels (16 hd), K scales, K minima, V scales, V minima (hd bytes each, fp16)
 * where each group of 64 values of a row has a scale s and a minimum m, and a 4-bit level stands for m + s level.
 *   levels: eight to a 32-bit word, value e at bit 4 (e / 2) + 16 (e % 2).
 *   K word j (hd / 32 of them, four or fewer side by side) of lane 16 h + c: token 16 tile + c, dimensions
 *     32 j + 8 h + e; order [tile][j / 4][lane][j % 4].
 *   V word of tile t and lane 16 h + c: dimension 16 t + c, tokens 16 (e / 4) + 4 h + e % 4; order
 *     [t / 4][lane][t % 4].
 *   K scales, V scales, V minima: [group][h][e] with the tokens of a V word; K minima: [token][group].
 * A group x is encoded as s = fp16(min(fl32(fl32(max x - min x) * fl32(1/15)), 65504)), m = fp16 of min x
 * kept within +-65504, level = (x - m) / s rounded to the nearest (ties to even) and kept within 0..15, exactly;
 * a group with a NaN or an infinity gets s = m = NaN.  4.5 bits a value.
 *
 * Slots.  table (n_slots, max_pages) int32 holds a slot's pages in order (-1: none), lens (n_slots) int32 its
 * tokens, refs (n_pages) int32 how many slots hold a page.  A call brings `rows` new rows: slot s the
 * rows cu[s] .. cu[s + 1] - 1 (cu (n_slots + 1) int32, or NULL: one row a slot, rows = n_slots), which are the
 * LAST tokens of the slot: lens counts them already (sx8_kv4_reserve).  A slot may bring none.  Rows behind
 * cu[n_slots] are left as they are.  Page numbers outside 0 .. n_pages - 1 are read as no tokens and never written;
 * lens is kept within the table.  n_slots <= 4096, max_pages * page_tokens <= 2^22.
 */
#ifndef SX8_PAGED_H
#define SX8_PAGED_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Attention of packed sequences.  q (Tq, nh, hd), k and v (Tk, nk, hd), out (Tq, nh, hd) with token and head
 * strides; sequence b has the query rows cu_q[b] .. cu_q[b + 1] - 1 and the keys cu_k[b] .. cu_k[b + 1] - 1
 * (cu_* (n_seq + 1) int32).  out = softmax(scale * q . k) v over its keys; causal != 0: row i of nq attends keys
 * 0 .. nk_b - nq + i (its own is the last).  A row with no key gives zeros; rows of no sequence are left as
 * they are.  hd 64, 128 or 256, nh a multiple of nk, scale > 0; n_seq <= 4096; one head's keys and values are
 * addressed in 64 bits.  Softmax sums and products are held in float32, probabilities rounded to dtype.
 * workspace (256-byte aligned, sx8_attn_varlen_workspace_bytes, no clearing needed) lets calls of few rows cut their
 * keys into parts that are added up by a second launch; without one (NULL) they run as one part. */
int64_t sx8_attn_varlen_workspace_bytes(int64_t n_seq, int64_t Tq, int64_t Tk, int32_t nh, int32_t hd);
int32_t sx8_attn_varlen(const void* q, const void* k, const void* v, void* out, const int32_t* cu_q,
                        const int32_t* cu_k, int64_t n_seq, int64_t Tq, int64_t Tk, int32_t nh, int32_t nk, int32_t hd,
                        int64_t q_ts, int64_t q_hs, int64_t k_ts, int64_t k_hs, int64_t v_ts, int64_t v_hs,
                        int64_t o_ts, int64_t o_hs, float scale, int32_t causal, int32_t dtype, void* workspace,
                        int64_t workspace_bytes, void* stream);

/* Bytes of a page (nk heads of hd 64, 128 or 256), or -1 for bad arguments. */
int64_t sx8_kv4_page_bytes(int32_t nk, int32_t hd, int32_t page_tokens);

/* Encode k and v (rows, nk, hd) into the slots' pages of one layer (pages: n_pages pages).  The pages of the new
 * tokens must be the slot's own (not shared); other tokens of their blocks keep their bits. */
int32_t sx8_kv4_append(uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu, int64_t n_slots,
                       int64_t max_pages, int64_t n_pages, const void* k, const void* v, int64_t rows, int64_t k_ts,
                       int64_t k_hs, int64_t v_ts, int64_t v_hs, int32_t nk, int32_t hd, int32_t page_tokens,
                       int32_t dtype, void* stream);

/* The values of the slots' last tokens (as sx8_kv4_append takes them), rounded to dtype.  Tokens without a page
 * and rows without a token (a slot with more rows than tokens) give zeros. */
int32_t sx8_kv4_read(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu, int64_t n_slots,
                     int64_t max_pages, int64_t n_pages, void* k, void* v, int64_t rows, int64_t k_ts, int64_t k_hs,
                     int64_t v_ts, int64_t v_hs, int32_t nk, int32_t hd, int32_t page_tokens, int32_t dtype,
                     void* stream);

/* Attention of the slots' new rows q (rows, nh, hd) over their pages: row i of a slot's n sits at position
 * lens - n + i and attends positions 0 .. that one; out (rows, nh, hd).  No position: zeros.  scale > 0,
 * nh a multiple of nk.  Levels and scales enter exactly, weights times scales as two fp16 numbers: to 22 bits, or within
 * 2^-35 of the largest weight (for scales of 2, 64 or 2048 on: 2^5, 2^10 or 2^15 times that); sums are held in float32.
 * Two launches;
 * workspace: sx8_kv4_attend_workspace_bytes(hd) bytes, 256-byte aligned, no clearing needed. */
int32_t sx8_kv4_attend(const uint8_t* pages, const int32_t* table, const int32_t* lens, const int32_t* cu,
                       int64_t n_slots, int64_t max_pages, int64_t n_pages, const void* q, void* out, int64_t rows,
                       int64_t q_ts, int64_t q_hs, int64_t o_ts, int64_t o_hs, int32_t nh, int32_t nk, int32_t hd,
                       int32_t page_tokens, float scale, int32_t dtype, void* workspace, int64_t workspace_bytes,
                       void* stream);
int64_t sx8_kv4_attend_workspace_bytes(int32_t hd);

/* Page operations.  Each takes free pages lowest number first, in the order of its slots or entries, and does all
 * of it or nothing: where it cannot, status (2 int32: code, slot or entry) is set if it was zero, and nothing
 * else changes.  Codes: 1 bad slot or count, 2 no free pages, 3 the slot's table row is full, 4 the target slot
 * is in use, named twice or a source.  workspace: sx8_kv4_pages_workspace_bytes bytes, 16-byte aligned.
 *
 * reserve: slot s grows by add[s] >= 0 tokens (lens[s] += add[s]), its new pages with one reference.
 * fork: for n entries, the empty slot dst[i] becomes a copy of slot src[i]: full pages are shared, a last page that is
 *   partly filled is copied (every layer: pages of layer l at pages + l * n_pages * page_bytes).
 * free: the slots' pages lose a reference, their rows become -1 and their lengths 0.  A slot named twice is freed
 *   once.  One launch, no workspace.
 * compact: the used pages above the number of used pages move to the free ones below it, highest
 *   free places last (i-th such page to the i-th such place); tables and refs follow. */
int64_t sx8_kv4_pages_workspace_bytes(int64_t n_slots, int64_t n_pages);
int32_t sx8_kv4_reserve(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* add, int64_t n_slots,
                        int64_t max_pages, int64_t n_pages, int32_t page_tokens, int32_t* status, void* workspace,
                        int64_t workspace_bytes, void* stream);
int32_t sx8_kv4_fork(uint8_t* pages, int64_t n_layers, int64_t page_bytes, int32_t* table, int32_t* lens, int32_t* refs,
                     const int32_t* src, const int32_t* dst, int64_t n, int64_t n_slots, int64_t max_pages,
                     int64_t n_pages, int32_t page_tokens, int32_t* status, void* workspace, int64_t workspace_bytes,
                     void* stream);
int32_t sx8_kv4_free(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* slots, int64_t n, int64_t n_slots,
                     int64_t max_pages, int64_t n_pages, int32_t* status, void* stream);
int32_t sx8_kv4_compact(uint8_t* pages, int64_t n_layers, int64_t page_bytes, int32_t* table, int32_t* refs,
                        int64_t n_slots, int64_t max_pages, int64_t n_pages, void* workspace, int64_t workspace_bytes,
                        void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SX8_PAGED_H */
