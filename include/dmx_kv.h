/*
 * dmx_kv.h — the C ABI of the operators between a decoder's q/k/v and o
 * projections, in libdmx_radix.so: rotary positions, the append to a paged
 * key/value cache held in 4 bits, its read and the attention over it, over all
 * of a sequence or over pages that a score selects; and the pages' handing out. No
 * drinkme counterpart: drinkme leaves these to the model's own code.
 *
 * Conventions are dmx_radix.h's: int status (0, or 1 with a message in
 * `err`), caller-owned buffers, host checks before any launch, no
 * synchronisation, buffers and stream of the current device. What only the device can see (lengths, positions, page
 * numbers) is checked by the kernels: none of it leads a read or a write out
 * of the buffers described here.
 *
 * The cache. Each token and head of keys and of values is held as blocks of
 * 32 channels: one exponent byte e, the block's scale 2^(e - 127), and 32
 * four-bit codes: a sign, then 0 0.5 1 1.5 2 3 4 6. e is the smallest (2 at
 * least, 252 at most) for which the block's largest magnitude is below
 * 7 * 2^(e - 127), the values that round to the grid's top or lower; a value
 * goes to the nearest of the grid, ties to the even code, and to the top
 * where it is larger. A block that holds a NaN or an infinity has e = 255 and
 * reads as NaN. Every value read is exactly a bf16 number. 253 and 254 are
 * never written; what a block with one reads as is left open.
 *
 *   k_codes   u32 [pages, heads, page, dim / 8]: nibble n of word w is
 *             channel 8 w + n
 *   k_scales  u8  [pages, heads, page, dim / 32]
 *   v_codes   u32 [pages, heads, page / 8, dim / 8, 8]: the words of eight
 *             tokens side by side, as a lane of the attention reads them
 *   v_scales  u8  [pages, heads, page / 8, dim / 32, 8]
 */
#ifndef DMX_KV_H
#define DMX_KV_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* pairs of channels that a rotation turns: (i, i + rotary_dim / 2), or (2 i, 2 i + 1) */
#define DMX_ROTARY_HALF 0
#define DMX_ROTARY_INTERLEAVED 1

typedef struct dmx_kv_cache {
    uint32_t* k_codes;  /* 16-byte aligned, as v_codes; the scales 8-byte aligned */
    uint32_t* v_codes;
    uint8_t* k_scales;
    uint8_t* v_scales;
    uint32_t pages;
    uint32_t heads;
    uint32_t page; /* tokens a page: a power of two, 8..1024 */
    uint32_t dim;  /* 64, 96, 128, 192 or 256 */
} dmx_kv_cache;

/* The sequences of a call. Sequence b has n_b new tokens: total / batch each
 * (cu NULL), or cu[b + 1] - cu[b], cu[0] = 0 and cu[batch] = total. Its new
 * token m sits at position lengths[b] - n_b + m; position p is in page
 * table[b, p / page]. */
typedef struct dmx_kv_seqs {
    const int32_t* table;   /* [batch, table_cols] page numbers */
    const int32_t* lengths; /* [batch] tokens of each sequence, the new ones included */
    const int32_t* cu;      /* [batch + 1], or NULL */
    uint32_t batch;
    uint32_t table_cols;
    uint32_t total;      /* new tokens of all sequences */
    uint32_t max_tokens; /* no sequence has more new tokens (cu given, attention alone) */
} dmx_kv_seqs;

/* x [tokens, heads, dim] of dtype DMX_BF16 or DMX_F32, channels adjacent;
 * strides in elements */
typedef struct dmx_rows {
    void* at;
    int64_t token_stride;
    int64_t head_stride;
    uint32_t heads;
} dmx_rows;

/* A rotary table: cos, sin of position p's angle i at at[p, i, 0 and 1]. */
typedef struct dmx_rotary_table {
    const float* at; /* [positions, dim / 2, 2], 16-byte aligned */
    uint32_t positions;
    uint32_t dim;    /* channels turned, the first ones: even, at most the head's */
    int layout;      /* DMX_ROTARY_HALF or DMX_ROTARY_INTERLEAVED */
} dmx_rotary_table;

/* out[i] = in[i] rotated, for n = 1 or 2 tensors of `tokens` tokens: a pair
 * (a, b) of angle t becomes a cos t - b sin t, b cos t + a sin t, each product
 * and sum rounded in fp32, then once to dtype; the channels past table->dim
 * are copied. positions: device int32 (wide 0) or int64 (wide 1) [tokens]; a
 * token whose position is outside the table becomes NaN in its turned
 * channels. out may be in itself (the same addresses and strides). */
int dmx_rotary(const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
               const void* positions, int wide, const dmx_rotary_table* table, void* stream, char* err, size_t errn);

/* The new tokens' keys k (rotated by their positions where table is given)
 * and values v [total, heads, dim] into the cache; and q, if given, rotated
 * to q_out as dmx_rotary does. A token whose position is negative or past the
 * table's columns, whose page is not one of the cache's, or which is of no
 * sequence (before cu[0], from cu[batch] on) is not stored; of the latter q_out
 * is left open. */
int dmx_kv_append(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, const dmx_rows* k, const dmx_rows* v,
                  const dmx_rows* q, const dmx_rows* q_out, int dtype, const dmx_rotary_table* table, void* stream,
                  char* err, size_t errn);

/* The new tokens' keys and values as the cache holds them, to bf16 k and v
 * [total, heads, dim], dense. Tokens that dmx_kv_append does not store read
 * NaN. */
int dmx_kv_read(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint16_t* k, uint16_t* v, void* stream, char* err,
                size_t errn);

/* How the attention of a call is split (a function of these alone): bytes of
 * device workspace that dmx_kv_attention needs, 16-byte aligned; 0 for none.
 * max_length: no sequence is longer (0: the table's columns). */
uint64_t dmx_kv_attention_workspace(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint32_t q_heads, int dtype,
                                    uint32_t max_length, uint32_t window);

/* The new tokens' queries q [total, q_heads, dim] (rotated already) against
 * the cached tokens of their sequences: out [total, q_heads, dim] of q's
 * dtype, dense, and lse fp32 [total, q_heads] (or NULL), the natural logarithm
 * of each row's sum of exponentials. q_heads is a multiple of the cache's
 * heads; query head g reads cache head g / (q_heads / heads). A query at
 * position p sees positions below its sequence's length, with causal no later
 * than p, with window > 0 later than p - window. A query that sees nothing
 * gives zeros and -inf. What a query does not see never reaches its result,
 * whatever bytes are there; a position that it sees but whose page is not one
 * of the cache's gives NaN. So does every token that the call does not
 * compute: a sequence's past max_tokens, and those of no sequence (before
 * cu[0], from cu[batch] on).
 *
 * Sums are divided at the end: a result is finite where the values that it sees
 * stay below 2^107 / (the tokens that it sees) in magnitude, and may overflow
 * past that, though the cache holds up to 1.5 * 2^127. */
int dmx_kv_attention(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, const dmx_rows* q, int dtype, float scale,
                     int causal, uint32_t window, uint32_t max_length, void* out, float* lse, void* workspace,
                     uint64_t workspace_bytes, void* stream, char* err, size_t errn);

/* ---- positions of several axes ---- */

/* Which axis of the positions turns each angle: two bits an angle, 16 angles a
 * word, the first lowest. */
typedef struct dmx_rotary_axes {
    uint32_t count;    /* axes, 1..4 */
    uint32_t of[16];   /* of angles 0 .. table->dim / 2 - 1, 256 at most */
} dmx_rotary_axes;

/* As dmx_rotary, with positions [count, tokens]: angle i of token t is turned by
 * the table's row positions[axis of i, t]. */
int dmx_rotary_by_axes(const dmx_rows* in, const dmx_rows* out, uint32_t n, uint32_t tokens, uint32_t dim, int dtype,
                       const void* positions, int wide, const dmx_rotary_axes* axes, const dmx_rotary_table* table,
                       void* stream, char* err, size_t errn);

/* ---- pages ---- */

/* The pages that no sequence has, as a stack: free[0 .. count - 1]. */
typedef struct dmx_kv_pool {
    int32_t* free;   /* [pages] */
    int32_t* count;  /* [1] */
    int32_t* lacking; /* [1]: pages that the last dmx_kv_reserve had not */
    uint32_t pages;  /* of the cache, fewer than 2^30 */
} dmx_kv_pool;

/* Room for each sequence's new tokens, and where they lie. table [batch,
 * table_cols] and lengths [batch] are updated in place; added [batch] (or NULL:
 * total / batch each) are the new tokens, negative ones 0; where their sum passes
 * `total` the sequences that pass it get what is left. In order of the sequences, and of a
 * sequence's columns, each column between the last one that holds a token and
 * the new end gets the page on top of the stack; -1 from where it is empty. Then cu
 * [batch + 1] holds the offsets of the new tokens, and positions and slots
 * [total] where each lies: its position (-1 behind the last), and page * page_size
 * + position % page_size, -1 where it has no page of the cache. lengths count
 * the tokens without one, too; before the new ones they count as 2^30 - 1 at most. */
int dmx_kv_reserve(const dmx_kv_pool* pool, int32_t* table, int32_t* lengths, const int32_t* added, uint32_t batch,
                   uint32_t table_cols, uint32_t page, uint32_t total, int32_t* cu, int32_t* positions, int64_t* slots,
                   void* stream, char* err, size_t errn);

/* Sequences cut to their first keep [batch] tokens (none where negative, all
 * where there are not that many): lengths become that, columns past it -1, and
 * their pages go back so that dmx_kv_reserve gives them out in the order they
 * had. Numbers that are no page's are dropped, and so is what a full stack does
 * not hold. */
int dmx_kv_trim(const dmx_kv_pool* pool, int32_t* table, int32_t* lengths, const int32_t* keep, uint32_t batch,
                uint32_t table_cols, uint32_t page, void* stream, char* err, size_t errn);

/* ---- attention over selected pages ---- */

/* Of each page and head: of every channel the largest and the smallest key of
 * its tokens (NaNs apart; 0 where there is no other), in whole numbers of
 * 2^(scale - 127), the largest rounded up and the smallest down. scale - 127 is the
 * least exponent, -126 or more, that leaves no number over 127. */
typedef struct dmx_kv_summaries {
    int8_t* bounds;   /* [pages, heads, 2, dim], 16-byte aligned: largest, smallest */
    uint8_t* scales;  /* [pages, heads] */
} dmx_kv_summaries;

/* The summaries of the pages that the new tokens lie in, from all of their
 * sequence's tokens there; of a page that several of them have, from the most that one has there. */
int dmx_kv_summarize(const dmx_kv_cache* cache, const dmx_kv_summaries* summaries, const dmx_kv_seqs* seqs, void* stream,
                     char* err, size_t errn);

/* The columns of the block table that score highest for each new token and
 * cache head: blocks [total, heads, count], ascending, -1 behind the last. Of the
 * columns that hold a position which the token sees (causal: up to its own) the
 * first `first` and the last `last` are among them (first + last at most
 * count); the others by their score, ties to the lower column, columns without a
 * page of the cache last. A score is 2^(scale - 127) times the largest sum, of
 * the query heads that share the cache head, over channels of x * (x > 0 ?
 * largest : smallest): x the query in whole numbers (to the nearest, even) of the least power
 * of two, 2^-126 or more, that leaves none of these heads' over 127; values that are not finite
 * are 0. Sums are below 2^24 and compared as fp32. Tokens of no sequence list nothing. A block
 * table has at most DMX_KV_MAX_COLUMNS columns here. workspace: as dmx_kv_select_workspace says, 16-byte
 * aligned device bytes, 0 for none. */
#define DMX_KV_MAX_COLUMNS 16384
uint64_t dmx_kv_select_workspace(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint32_t q_heads);
int dmx_kv_select(const dmx_kv_cache* cache, const dmx_kv_summaries* summaries, const dmx_kv_seqs* seqs,
                  const dmx_rows* q, int dtype, uint32_t count, uint32_t first, uint32_t last, int causal,
                  int32_t* blocks, void* workspace, uint64_t workspace_bytes, void* stream, char* err, size_t errn);

/* As dmx_kv_attention without a window, over the listed columns alone: a query
 * of token t and cache head h sees of the positions that it would see there those in
 * columns blocks[t, h, 0 .. count - 1]. Their order does not matter, a column
 * listed twice counts once, and one that is negative or past the token's position is
 * nothing; one that the table has no page for gives NaN. A sequence has fewer than 2^31 rows (new tokens, at most
 * max_tokens, times the query heads that share a cache head). */
uint64_t dmx_kv_attention_blocks_workspace(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, uint32_t q_heads,
                                           int dtype, uint32_t count, uint32_t max_length);
int dmx_kv_attention_blocks(const dmx_kv_cache* cache, const dmx_kv_seqs* seqs, const dmx_rows* q, int dtype, float scale,
                            int causal, const int32_t* blocks, uint32_t count, uint32_t max_length, void* out, float* lse,
                            void* workspace, uint64_t workspace_bytes, void* stream, char* err, size_t errn);

#ifdef __cplusplus
}
#endif

#endif /* DMX_KV_H */
