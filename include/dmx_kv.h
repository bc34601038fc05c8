/*
 * dmx_kv.h — the C ABI of the operators between a decoder's q/k/v and o
 * projections, in libdmx_radix.so: rotary positions, the append to a paged
 * key/value cache held in 4 bits, its read and the attention over it. No
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

#ifdef __cplusplus
}
#endif

#endif /* DMX_KV_H */
