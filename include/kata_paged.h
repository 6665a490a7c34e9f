/* kata_paged.h - C ABI of the paged KV cache: a cache in pages instead of one contiguous arena per sequence (kata_attn.h), the kernel
 * that appends to it (per-head RMSNorm, rotary positions with up to three axes, gate split, quantise-on-append), the attention of the
 * newest tokens over it, and the eviction that keeps a sequence within a budget of slots by the attention its keys have received.
 *
 * The reference (wolfjpy/kata) serves one sequence from one contiguous cache and text positions only (src/engine.cpp:54-60, 119-127,
 * 161-178); nothing here has a counterpart there. Formulas, rounding points and row layouts are those of the contiguous path, so that rows can be
 * copied between the two (kata_paged_import).
 *
 * Layout. A context holds n_layers pools of n_pages pages of page_size slots; a slot is the K and V row of one token. Per layer:
 *   K, V         [n_pages][page_size][kv_heads][head_dim]  fp16, or int8 codes
 *   K, V scales  [n_pages][page_size][kv_heads]            fp16 (int8 only: scale = fp16(max |x| / 127), 1 for a row of zeros; value = code * scale)
 *   weight, age  [n_pages][kv_heads][page_size]            fp32, int32 (contexts with KATA_PAGED_WEIGHTS only)
 * A sequence's slot s lies in page table[s / page_size] at offset s % page_size; the table is the same for every layer. Slots are places in the cache,
 * not positions: after an eviction a slot holds whatever key was moved there, a different one per KV head (attention does not mind the order of its
 * keys; the rotary position was applied when the key was appended).
 *
 * Conventions are those of kata_attn.h: d_* is device memory of the caller, calls enqueue on the caller's stream and return at once, every function
 * returns KATA_OK or an error code, nothing is allocated after kata_paged_create. One context per GPU and one stream at a time: the context's scratch
 * (and two CUDA graphs captured from it) must not be in use twice at once. Device pointers must lie on 16-byte boundaries. */
#ifndef KATA_PAGED_H
#define KATA_PAGED_H

#include <stddef.h>
#include <stdint.h>
#include "kata_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KATA_PAGED_MAX_BATCH 256     /* sequences per call */
#define KATA_PAGED_MAX_SLOTS 524288  /* slots per sequence */
#define KATA_PAGED_MAX_KV_HEADS 16
#define KATA_PAGED_MAX_GROUP 16      /* query heads per KV head */

enum { KATA_PAGED_GATED = 1,         /* flags: the query rows of kata_paged_prep are [query | gate] per head, as KATA_QFULL_DIM rows are */
       KATA_PAGED_WEIGHTS = 2 };     /* flags: keep per slot and KV head the attention weight received and the token's age (kata_paged_evict); takes 32 or 64 bytes more per
                                      * slot of the pool and KV head for the scores of one launch (64 when a call can have more than 8 query rows per KV head) */
enum { KATA_PAGED_K = 0, KATA_PAGED_V = 1, KATA_PAGED_K_SCALE = 2, KATA_PAGED_V_SCALE = 3, KATA_PAGED_WEIGHT = 4, KATA_PAGED_AGE = 5, KATA_PAGED_PLANES = 6 };

/* ---- the page table (host only, no GPU): which pages belong to which sequence. A kata_paged context keeps one of its own. Free pages are handed
 * out lowest number first. Pages may be shared between sequences by kata_pages_fork; a page is free again when its last owner drops it. */
typedef struct kata_pages kata_pages;
int kata_pages_create(int32_t n_pages, int32_t page_size, int32_t n_seqs, int32_t max_slots, kata_pages** out);
int kata_pages_destroy(kata_pages* p);
int kata_pages_reserve(kata_pages* p, int32_t seq, int32_t n_slots);                 /* at least ceil(n_slots / page_size) pages; KATA_ERR_NOMEM (nothing changed) when they run out */
int kata_pages_trim(kata_pages* p, int32_t seq, int32_t n_slots);                    /* at most that many pages: drops the others */
/* dst (without pages) becomes a copy of the first n_slots slots of src: whole pages are shared, a last partial page is a page of its own, to be
 * copied by the caller: *copy_from, *copy_to (pages) and *copy_slots, -1, -1, 0 when there is none. */
int kata_pages_fork(kata_pages* p, int32_t src, int32_t dst, int32_t n_slots, int32_t* copy_from, int32_t* copy_to, int32_t* copy_slots);
int32_t kata_pages_count(const kata_pages* p, int32_t seq);                          /* pages of a sequence, -1 for a bad argument */
int32_t kata_pages_get(const kata_pages* p, int32_t seq, int32_t* out, int32_t cap); /* writes up to cap of them; returns their number */
int32_t kata_pages_free_count(const kata_pages* p);
int32_t kata_pages_owners(const kata_pages* p, int32_t page);                        /* sequences that hold a page */

/* ---- the context */
typedef struct kata_paged_ctx kata_paged_ctx;

typedef struct kata_paged_config {
    int32_t device, n_layers, n_seqs, n_pages;
    int32_t page_size;      /* a power of two, 16 .. 1024 */
    int32_t max_slots;      /* most slots of one sequence, <= KATA_PAGED_MAX_SLOTS */
    int32_t heads, kv_heads, head_dim;   /* head_dim 128 or 256; heads a multiple of kv_heads */
    int32_t kv_mode;        /* KATA_KV_FP16 or KATA_KV_INT8 (rounding: ties to even) */
    int32_t rot_dim;        /* leading dims of a head that are rotated, pairs (i, i + rot_dim / 2); a multiple of 16, 0 .. head_dim */
    int32_t section[3];     /* frequencies that take their position from axis 0, 1, 2 (time, height, width); sum = rot_dim / 2 */
    int32_t interleaved;    /* 0: the axes' frequencies lie one after the other. 1: frequency i belongs to axis i % 3 while i < 3 * section[i % 3], else to axis 0 */
    int32_t flags;          /* KATA_PAGED_* */
    double rope_theta;      /* frequency i: rope_theta ^ (-2 i / rot_dim) */
    void* planes[KATA_PAGED_PLANES];   /* device memory of the caller for a plane ([n_layers] times the layout above, 128-byte aligned, left as it is); NULL: allocated here, zero-filled */
} kata_paged_config;

int kata_paged_create(const kata_paged_config* cfg, kata_paged_ctx** out);
int kata_paged_destroy(kata_paged_ctx* ctx);
const char* kata_paged_last_error(const kata_paged_ctx* ctx);
uint64_t kata_paged_launch_count(const kata_paged_ctx* ctx);
int kata_paged_check(kata_paged_ctx* ctx, void* stream);   /* synchronises the stream; KATA_ERR_DEVICE_WAIT after a bounded device wait that ran out */
void* kata_paged_plane_ptr(kata_paged_ctx* ctx, int32_t layer, int32_t plane);   /* device address of a layer's plane, NULL when the context has none */

/* The page table. The host's side changes at once, the device's copy in stream order (kata_paged_reserve and _fork enqueue it), so the calls that use the
 * new pages belong on the same stream or behind it. Not inside a stream capture (KATA_ERR_MODE). A trim or release enqueues nothing: freed
 * pages are reused in stream order. */
int kata_paged_reserve(kata_paged_ctx* ctx, int32_t seq, int32_t n_slots, void* stream);
int kata_paged_trim(kata_paged_ctx* ctx, int32_t seq, int32_t n_slots);
/* As kata_pages_fork, the partial page copied for all layers. Shared pages are read-only: kata_paged_prep and _import refuse to write them.
 * A context with KATA_PAGED_WEIGHTS cannot share pages (weights belong to one sequence): KATA_ERR_MODE. */
int kata_paged_fork(kata_paged_ctx* ctx, int32_t src, int32_t dst, int32_t n_slots, void* stream);
const kata_pages* kata_paged_table(const kata_paged_ctx* ctx);

/* Norm, rotary position and append of T tokens per sequence into slots slot0[b] .. slot0[b] + T - 1 (reserved before, each sequence once per call).
 *   x = v * rsqrt(mean(v^2) + 1e-6) * w; angle_i = p_axis(i) * theta^(-2i/rot_dim); (x_i, x_j) <- (x_i cos - x_j sin, x_i sin + x_j cos), j = i + rot_dim / 2.
 * The angle is taken modulo a full turn in 64-bit fixed point before its sine and cosine are formed: positions far out lose nothing
 * (kata_attn_prep forms it in fp32, as the reference does: at position 130,000 that is 0.007 off).
 *   d_q [n][T][heads][head_dim, or 2 head_dim when gated], d_k, d_v [n][T][kv_heads][head_dim]: act_dtype; d_qnorm, d_knorm fp32 [head_dim]
 *   d_axis_pos [n][T][3] int32 (device), or NULL: all three axes are at age0[b] + t (text)
 *   age0 [n]: tokens the sequence has seen before this call, the age of its first token here; NULL: slot0, which is right until kata_paged_evict has cut the sequence: from then on
 *   a slot's number is not its token's age (nor its text position), and the caller says it
 *   d_q16 [n][T][heads][head_dim] fp16: the query times 1/sqrt(head_dim); d_gate [n][T][heads][head_dim] fp32, NULL when not gated (or not wanted)
 * d_q NULL appends K and V alone. With KATA_PAGED_WEIGHTS the appended slots get weight 0 and their age. */
int kata_paged_prep(kata_paged_ctx* ctx, int32_t layer, int32_t n, const int32_t* seq_ids, const int32_t* slot0, int32_t T, const int32_t* d_axis_pos, const int32_t* age0,
                    const void* d_q, const void* d_k, const void* d_v, int32_t act_dtype, const float* d_qnorm, const float* d_knorm, void* d_q16, float* d_gate, void* stream);

/* Attention of the T newest tokens of each sequence (1..KATA_MAX_VERIFY) over its n_slots[b] slots: token t sees slots [0, n_slots[b] - T + 1 + t).
 *   d_out [n][T][heads][head_dim] out_dtype = softmax(q k^T) v (* sigmoid(gate) when d_gate is given); a token that sees no slot gets zeros.
 * The probabilities go into the matrix product in two fp16 terms (about 22 bits); for int8 caches with bf16 or fp16 outputs in one (2^-11 relative). They are carried relative to the
 * row's largest probability so far and, int8, times the V scale relative to the largest of its tile of 32 or 64 slots, whatever the size of either; parts below 2^-40 of these are lost.
 * accumulate != 0 (KATA_PAGED_WEIGHTS; each sequence once per call): weight[head][slot] += the slot's probability, summed over the tokens and over the
 * query heads of the KV head. No atomics: the sums come out the same in every run. */
int kata_paged_decode(kata_paged_ctx* ctx, int32_t layer, int32_t n, const int32_t* seq_ids, const int32_t* n_slots, int32_t T,
                      const void* d_q16, const float* d_gate, void* d_out, int32_t out_dtype, int32_t accumulate, void* stream);

/* Cuts each sequence of the call (each once) from n_slots[b] to min(n_slots[b], keep) slots, in layers [layer, layer + n_layers), per layer and KV head: kept are the
 * `keep` slots with the largest weight, where slots of age < sink or >= seen[b] - recent (the newest `recent` of the seen[b] tokens) count as
 * infinitely heavy, equal weights go to the lowest slots, and NaN is lighter than everything. Kept slots below `keep` stay where they are; the kept slots behind it move, in order, into
 * the free slots below it (K, V, scales, weight, age). d_src [n_layers][n][kv_heads][keep] int32 (required): the slot each slot's content came from, -1 behind a sequence's end.
 * Slots >= keep are left as they were; kata_paged_trim gives their pages back. */
int kata_paged_evict(kata_paged_ctx* ctx, int32_t layer, int32_t n_layers, int32_t n, const int32_t* seq_ids, const int32_t* n_slots, const int32_t* seen, int32_t keep, int32_t sink, int32_t recent,
                     int32_t* d_src, void* stream);

/* Copies n_rows cache rows of a contiguous context (sequence src_seq, layer src_layer, positions src_pos ..) into slots slot0 .. of a sequence: a prompt
 * that kata_attn_prefill has worked on goes on in pages. Same kv_mode, 24 heads, 4 KV heads, head_dim 256, same device; KATA_ERR_MODE for a source
 * that kata_attn_set_kv_heads has restricted (it never wrote the other heads' rows). Weights start at 0, ages at age0. */
int kata_paged_import(kata_paged_ctx* ctx, int32_t layer, int32_t seq, int32_t slot0, int32_t n_rows, int32_t age0, kata_attn_ctx* src, int32_t src_layer, int32_t src_seq, int32_t src_pos, void* stream);

/* How a decode launch would be shared out (host only, no GPU): tile_keys (16, 32 or 64) keys per tile, the tiles of all (sequence, KV head) segments in one list, CTA c works on tiles
 * [first_tile[c], first_tile[c + 1]). Returns the number of CTAs, -1 for arguments out of range; *max_contrib: CTAs of the most-cut segment. */
int kata_paged_decode_plan(int32_t n, const int32_t* n_keys, int32_t kv_heads, int32_t tile_keys, int32_t sm_count, int32_t* first_tile, int32_t first_tile_cap, int32_t* max_contrib);

#ifdef __cplusplus
}
#endif
#endif /* KATA_PAGED_H */
