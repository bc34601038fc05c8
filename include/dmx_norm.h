/*
 * dmx_norm.h — the C ABI of the norms around a decoder's blocks, in
 * libdmx_radix.so: a norm of rows (of heads, before the rotary positions), and
 * a block's output into the residual stream with the norm after the block, its
 * gate and factor, and the norm and modulation before the next one, in one pass. No
 * drinkme counterpart: drinkme leaves these to the model's own code.
 *
 * Conventions are dmx_radix.h's: int status (0, or 1 with a message in
 * `err`), caller-owned buffers, host checks before any launch, no
 * synchronisation, buffers and stream of the current device.
 *
 * N(v; w, b), of a row v of `dim` numbers:
 *   DMX_NORM_RMS    v / sqrt(mean(v^2) + eps) * (w + offset) + b
 *   DMX_NORM_LAYER  (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * (w + offset) + b
 * without w the factor is 1, without b there is no term. Everything is computed in
 * fp32 and rounded once, to each output's type.
 */
#ifndef DMX_NORM_H
#define DMX_NORM_H

#include <stddef.h>
#include <stdint.h>

#include "dmx_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DMX_NORM_RMS 0
#define DMX_NORM_LAYER 1
#define DMX_NORM_MAX_DIM 32768

/* Rows of `dim` numbers, dense, of DMX_BF16 or DMX_F32 (at NULL: none). */
typedef struct dmx_vectors {
    const void* at;
    int dtype;
    uint32_t rows; /* 1: for every row of the call; else `rows` of them, see cu */
} dmx_vectors;

typedef struct dmx_norm_form {
    int kind; /* DMX_NORM_RMS or DMX_NORM_LAYER */
    float eps;
    float offset;
    float factor;        /* dmx_block_norm: of what the block adds */
    dmx_vectors weight;  /* of N in front of the next block (dmx_norm: of N); weight, bias and post have one row */
    dmx_vectors bias;
    dmx_vectors post;    /* w of N after the block (at NULL: no such norm) */
    dmx_vectors gate;
    dmx_vectors scale;   /* both or neither */
    dmx_vectors shift;
    const int32_t* cu;   /* device [batch + 1]: gate, scale and shift of `batch` rows have one for the rows cu[b] ..
                            cu[b + 1] - 1 (those before and behind: as the nearest). NULL: row r of a call of R takes
                            row r / (R / rows), and R is a multiple of rows */
    uint32_t batch;
} dmx_norm_form;

/* out [tokens, x->heads, dim], dense, of x's dtype: N of each token's and head's row.
 * post, gate, scale, shift and cu are not used. */
int dmx_norm(const dmx_rows* x, void* out, uint32_t tokens, uint32_t dim, int dtype, const dmx_norm_form* form,
             void* stream, char* err, size_t errn);

/* Of each of `rows` rows:
 *   r'  = residual + factor * gate * (post ? N(y; post) : y)
 *   out = N(r'; weight, bias) * (1 + scale) + shift
 * r' goes into the second norm as it is, before its rounding. y and out are of
 * dtype, residual and residual_out of residual_dtype: dtype, or DMX_F32. Strides are of rows, in elements;
 * residual_out and out are dense. residual_out may be residual, and out may be y, where those are dense. */
int dmx_block_norm(const void* y, int64_t y_stride, const void* residual, int64_t residual_stride, void* residual_out,
                   void* out, uint32_t rows, uint32_t dim, int dtype, int residual_dtype, const dmx_norm_form* form,
                   void* stream, char* err, size_t errn);

#ifdef __cplusplus
}
#endif

#endif /* DMX_NORM_H */
