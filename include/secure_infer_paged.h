/*
 * secure_infer_paged.h -- operators on the paged KV cache that reloads fill.
 *
 * No reference counterpart: the reference leaves a layer's attention, the
 * writing of new keys and values into pages and the bookkeeping of pages to
 * its serving engine.  A layer's cache is K and V of [pages][128 tokens]
 * [KV heads][128], as secure_infer_h2d_reload_layer scatters it.
 *
 * Streams are cudaStream_t passed as void*; every other pointer is a device
 * pointer of the device that is current, unless said otherwise.  Nothing here
 * waits for the device (but secure_infer_attend_status) or allocates.  Functions return 0, or -1 when an argument is refused (nothing is
 * launched) or a launch fails.  Contents of device arrays cannot be refused:
 * page ids outside the cache read as zeros and are never written, lengths are
 * clamped to the block table, ranges of tokens to the token count.
 */
#ifndef SECURE_INFER_PAGED_H
#define SECURE_INFER_PAGED_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SECURE_INFER_PAGE_TOKENS 128u
#define SECURE_INFER_HEAD_DIM 128u
#define SECURE_INFER_BF16 0u
#define SECURE_INFER_FP16 1u

/* One layer's paged cache.  Strides are in elements: page, token, head; the
 * 128 values of a head are adjacent.  Base addresses and strides are multiples
 * of 16 bytes. */
typedef struct {
    void* k;
    void* v;
    int64_t k_stride[3];
    int64_t v_stride[3];
    uint32_t pages;
    uint32_t heads;
    uint32_t dtype;
    uint32_t reserved;
} secure_infer_pages;

/* The new tokens of a step, ragged over sequences: sequence s owns tokens
 * [cu_q[s], cu_q[s+1]) of `tokens` and holds kv_lens[s] tokens in all, these
 * new ones last.  Position p of s lives in page block_table[s][p / 128], slot
 * p % 128.  A sequence may have no new token.  max_q: no sequence has more
 * (0: unknown).  Tokens past cu_q[seqs] belong to nobody. */
typedef struct {
    const int32_t* block_table;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    int64_t table_stride;
    uint32_t table_width;
    uint32_t seqs;
    uint32_t tokens;
    uint32_t max_q;
} secure_infer_chunk;

/* Attention of the chunk over the pages.  q: [tokens][q_heads][128] with its
 * strides in elements, q_heads a multiple of the KV
 * heads (query head h reads KV head h / (q_heads / heads)).  out:
 * [tokens][q_heads][128], dense.  lse: null, or [tokens][q_heads] natural
 * logarithms of the softmax sums, for joining with attention over other keys.
 * causal: the token at position p sees keys 0..p (else all of its sequence),
 * and with window > 0 only the last `window` of them.  A row that sees no key
 * gives zeros and -inf.  Keys that a row does not see take no part in it,
 * whatever they hold; an infinite value that it sees makes it infinite, or NaN
 * where the key's weight rounds to zero.  Rows of tokens that belong to nobody are
 * not written.  workspace: secure_infer_paged_attend_workspace() bytes
 * (41 MB on a device of 148 SMs; it is asked with that device current),
 * 256-byte aligned, zero before its first use, used by one stream at a time
 * (host threads that share the stream may share it too);
 * calls leave it ready for the next. */
#define SECURE_INFER_ATTEND_STATE_BYTES 4096u   /* of a workspace, from its start: all that has to be zero */
/* Waits inside the kernels have a limit of some seconds.  One that runs out ends
 * its call with NaN in the rows that it concerns and makes the first word of the
 * workspace non-zero, and from then on calls with this workspace give NaN in
 * every row that sees a key. */
uint64_t secure_infer_paged_attend_workspace(void);
/* The stream capture that `stream` takes part in, 0 outside of one.  A captured
 * call uses its workspace wherever the graph is replayed, so it needs one that
 * no other stream's calls use meanwhile. */
uint64_t secure_infer_capture_id(void* stream);
/* 1 where a call of this size is not refused, 0 where it has more than 2^31 - 1
 * units of work (a page for a tile of rows and a KV head), by the longest context
 * that the table's width can hold. */
int secure_infer_attend_fits(const secure_infer_pages* pages, const secure_infer_chunk* chunk, uint32_t q_heads);
/* The same for a call with a window and sinks, whose tiles count a page more.
 * (A shared prefix refuses nothing: where its work would pass that the call goes
 * without it.) */
int secure_infer_attend_fits_window(const secure_infer_pages* pages, const secure_infer_chunk* chunk, uint32_t q_heads,
                                    uint32_t window, uint32_t sinks);
/* Waits for the stream, which is the one exception here.  *status: 0, or 1 if a
 * wait ran out in a call with this workspace; then its state is zero again and
 * the next call computes.  -1 while the stream is captured. */
int secure_infer_attend_status(void* workspace, uint32_t* status, void* stream);
int secure_infer_paged_attend(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                              int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* out, float* lse,
                              float scale, uint32_t causal, uint32_t window, void* workspace, void* stream);

/* The same with more of it.  sinks, with a window: the first `sinks` tokens of a
 * sequence stay visible behind it, so the token at position p sees the keys j <= p
 * with j > p - window or j < sinks; what lies between is not read, and its pages
 * may be given back (secure_infer_trim).
 *
 * plan, from secure_infer_shared_prefix of this chunk: groups of sequences attend
 * the pages that they have in common once for all of their rows, which gives what
 * the call without it gives, up to the order of sums and the rounding of weights:
 * these are rounded to the cache's type beside the largest of their part of the
 * keys, and many rows of common keys go through the kernel for many rows (in bf16
 * errors of 0.0023 relative where single tokens alone have 0.0017).  Not with a
 * window.  It is done where it saves time, which is judged on the host by the sizes
 * alone: max_common says that no group has more tokens in common (0: as many as the
 * table holds, which in tables much wider than the prefixes may take the slower
 * way).  parts: secure_infer_attend_parts() bytes, 16-byte aligned, for
 * this call alone; null where that is 0, else 1040 bytes for every token of the call
 * and query head.  options may be null. */
typedef struct {
    const int32_t* plan;
    float* parts;
    uint32_t groups;
    uint32_t max_common;
    uint32_t sinks;
    uint32_t reserved;
} secure_infer_attend_options;
int secure_infer_attend(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                        int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* out, float* lse,
                        float scale, uint32_t causal, uint32_t window, const secure_infer_attend_options* options,
                        void* workspace, void* stream);
uint64_t secure_infer_attend_parts(const secure_infer_pages* pages, const secure_infer_chunk* chunk, uint32_t q_heads,
                                   const secure_infer_attend_options* options);

/* What the sequences of a chunk have in common.  Group g is the sequences
 * [cu_seqs[g], cu_seqs[g+1]), 1 <= groups <= seqs; cu_seqs may be null for one
 * group of all.  Common are the pages from the first on that every sequence of the
 * group with new tokens names in the same places, as far as all their tokens lie
 * before the new ones of each.  plan: secure_infer_shared_prefix_ints() int32,
 * 16-byte aligned: the common tokens of each sequence [seqs], then the kernels'
 * own.  It goes with the chunk's contents when this runs: offsets, lengths and
 * tables that change need another.  Only kv_lens may grow meanwhile, under the same
 * cu_q: rows that the plan does not know would read what nobody has written. */
uint64_t secure_infer_shared_prefix_ints(uint32_t seqs, uint32_t groups);
int secure_infer_shared_prefix(const secure_infer_chunk* chunk, const int32_t* cu_seqs, uint32_t groups, int32_t* plan,
                               void* stream);

/* Attention over all keys from attention over n sets of them that have none in
 * common, 1 <= n <= SECURE_INFER_JOIN_PARTS: lse = log sum e^lse_i and out = sum
 * e^(lse_i - lse) out_i.  A part with lse_i = -inf counts for nothing, whatever
 * its out_i holds; where all are, out is 0 and lse -inf.  One of NaN, as attention
 * that failed gives it, makes out and lse NaN beside any others.  A part's out:
 * [tokens][heads][128] of `dtype` with its strides (token, head) in elements,
 * multiples of 16 bytes; its lse: [tokens][heads] with strides.  out, lse: dense;
 * out may be one part's own where that is dense. */
#define SECURE_INFER_JOIN_PARTS 8u
typedef struct {
    const void* out;
    const float* lse;
    int64_t out_stride[2];
    int64_t lse_stride[2];
} secure_infer_attend_part;
int secure_infer_attend_join(const secure_infer_attend_part* parts, uint32_t n, uint32_t tokens, uint32_t heads,
                             uint32_t dtype, void* out, float* lse, void* stream);

/* Rotary positions and the chunk's way into its pages.  q (may be null), k and
 * v: [tokens][heads][128] with their strides (token, head).  Pair i of a head
 * (elements i and i + 64, or 2i and 2i + 1 where `interleaved`) turns by
 * positions[axis[i]][token] * phase[i] revolutions / 2^64.  phase: 64 uint64,
 * axis: 64 uint32, device; both null: no rotation.  positions: int32
 * [axes][tokens] with axis stride position_stride, or null for the position in
 * the sequence.  Turned q goes to q_out, dense; turned k and plain v to their
 * slots.  Tokens whose slot lies outside the cache are not written. */
int secure_infer_paged_append(const secure_infer_pages* pages, const secure_infer_chunk* chunk, const void* q,
                              int64_t q_token_stride, int64_t q_head_stride, uint32_t q_heads, void* q_out,
                              const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                              int64_t v_token_stride, int64_t v_head_stride, const uint64_t* phase,
                              const uint32_t* axis, const int32_t* positions, int64_t position_stride, uint32_t axes, uint32_t interleaved, void* stream);

/* Tables of a cache: block_table [seqs][width], tokens held per sequence, and
 * how many rows hold each page (0: free).  A sequence of n tokens holds
 * ceil(n / 128) pages, less those that secure_infer_trim took (-1). */
typedef struct {
    int32_t* block_table;
    int32_t* lens;
    int32_t* refs;
    uint32_t seqs;
    uint32_t width;
    uint32_t pages;
    uint32_t reserved;
} secure_infer_tables;

/* A tensor whose pages are copied: page p at base + p * page_stride bytes,
 * page_bytes of it, all multiples of 16. */
typedef struct {
    void* base;
    int64_t page_stride;
} secure_infer_page_tensor;

/* Scratch of the calls below for tables of this size and n requests. */
uint64_t secure_infer_paged_scratch(const secure_infer_tables* tables, uint32_t n);

/* Copies pages src[i] to dst[i] of every tensor.  Pairs outside [0, pages) are
 * skipped.  No page may be written twice, or written and read. */
int secure_infer_paged_copy(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes,
                            uint32_t pages, const int32_t* src, const int32_t* dst, uint32_t n, void* stream);

/* The calls below read `in` and write all of `out` (no array of which may
 * overlap one of `in`), so work in flight may go on reading the old tables.
 *
 * fork: request i gives the empty sequence children[i] the tokens of
 * parents[i].  It shares the full pages and gets a copy of a partial last one,
 * in the lowest free page; requests are served in order, and granted[i] = 0
 * where the child is not empty or given twice, an index is out of range, or no
 * page is left for it. */
int secure_infer_paged_fork(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes,
                            const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* parents,
                            const int32_t* children, uint32_t n, int32_t* granted, void* scratch, void* stream);

/* reserve: sequence seqs[i] grows to new_lens[i] tokens, on the lowest free
 * pages in order; granted[i] = 0 where it would shrink, does not fit the table,
 * is given twice, its partial last page is shared, or fewer pages are left than
 * it needs (later requests may still have them). */
int secure_infer_paged_reserve(const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* seqs,
                               const int32_t* new_lens, uint32_t n, int32_t* granted, void* scratch, void* stream);

/* free: the sequences give up their pages and become empty. */
int secure_infer_paged_free(const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* seqs,
                            uint32_t n, void* scratch, void* stream);

/* trim: the sequences give up the pages that no later token sees when it is
 * attended with this window and these sinks: those behind the first `sinks`
 * tokens that lie wholly before the window of the token at position lens.
 * 1 <= window < 2^31, sinks < 2^31 - 128.  Their entries become -1, lengths stay. */
int secure_infer_trim(const secure_infer_tables* in, const secure_infer_tables* out, const int32_t* seqs, uint32_t n,
                      uint32_t window, uint32_t sinks, void* scratch, void* stream);

/* compact: with `live` pages in use, the i-th used page at or above `live`
 * moves to the i-th free page below it.  moved[p]: where page p is now, -1 for
 * a free one; live: the count. */
int secure_infer_paged_compact(const secure_infer_page_tensor* tensors, uint32_t n_tensors, uint64_t page_bytes,
                               const secure_infer_tables* in, const secure_infer_tables* out, int32_t* moved,
                               int32_t* live, void* scratch, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SECURE_INFER_PAGED_H */
