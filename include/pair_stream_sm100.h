/*
 * pair_stream_sm100.h -- C ABI of the pair-stream operators in libtrimul_sm100.so: what makes, updates and
 * reads the pair representation (b, i, j, d) around the triangle update of trimul_sm100.h.
 *
 *   pair_sm100_add_norm        z = residual + dropout(update); optionally y = rms_norm(z), in the activations' type
 *                              or in e4m3 with fp32 scales
 *   pair_sm100_add_norm_grad   its gradients
 *   pair_sm100_embed           out = base + scale * table[index]
 *   pair_sm100_embed_grad      the table's gradient
 *
 * The conventions of trimul_sm100.h hold: 0 or a negative TRIMUL_ERR_* code with a message in
 * trimul_sm100_last_error(), caller-owned device memory, no allocation, no hidden stream, nothing throws.
 * Nothing is kept between calls: two calls need two workspaces only if they overlap on the GPU.
 * Tensors are described by a base pointer and the element strides of their b, i and j axes (0 for a
 * broadcast axis); channels are contiguous.  Outputs are contiguous unless a stride is named.  The device that
 * owns the buffers and the stream is the current one.
 */
#ifndef PAIR_STREAM_SM100_H_
#define PAIR_STREAM_SM100_H_

#include <stdint.h>

#include "trimul_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PAIR_BF16 0
#define PAIR_FP16 1
#define PAIR_FP32 2

#define PAIR_MAX_WIDTH 8192 /* channels */
#define PAIR_MAX_BATCH 65536 /* batch coordinates of the dropout's counter */

/* Axis the dropout's mask is shared over. */
#define PAIR_SHARED_NONE 0
#define PAIR_SHARED_ROWS 1    /* one mask for all i */
#define PAIR_SHARED_COLUMNS 2 /* one mask for all j */

/* Dropout without a stored mask.  Element (b, i, j, c) of the WHOLE grid is kept when
 *     h(b, i, j, c) < keep,   h = half word c % 8 of Philox4x32-10(counter, key)
 *     counter = ((b << 16) | (c / 8), j, i, offset),  key = (seed low, seed high)
 * with i = 0 when the mask is shared over rows and j = 0 when it is shared over columns; kept elements are
 * multiplied by 65536 / keep.  A rank that holds a block of the grid passes the block's first (b, i, j) as
 * `origin`, so that every way of splitting the grid draws the same mask.  Half word 2k (2k + 1) is the low
 * (high) half of output word k. */
typedef struct pair_dropout {
  uint64_t seed;
  uint32_t offset;
  uint32_t keep; /* values of 65536 that are kept; 65536 = no dropout, 0 = everything is dropped */
  const uint64_t* device_seed; /* nullable: {seed, offset} in device memory, read when the kernel runs */
  int32_t shared; /* PAIR_SHARED_* */
  int32_t origin_b;
  int32_t origin_i;
  int32_t origin_j;
} pair_dropout_t;

typedef struct pair_tensor {
  void* data;
  int64_t stride_b; /* elements */
  int64_t stride_i;
  int64_t stride_j;
} pair_tensor_t;

typedef struct pair_norm_desc {
  int32_t b;
  int32_t i;
  int32_t j;
  int32_t d;
  int32_t dtype;        /* PAIR_*: update, residual, stream, y, dy, dz, and the gradients of the activations */
  int32_t weight_dtype; /* PAIR_*: weight and its gradient */
  int32_t group;        /* y in e4m3 with one scale per `group` channels (32, 64, 128 or d); 0: y in dtype */
  float eps;
  pair_dropout_t dropout;
} pair_norm_desc_t;

/* z = round(residual + dropout(update)), y = z / sqrt(mean(z^2) + eps) * weight of the stored z.
 * residual.data may be NULL (z = dropout(update)); stream (contiguous) may be NULL when z is not wanted, and may be
 * the residual's or the update's own memory where that is contiguous; weight and y are both NULL for the addition alone.
 * scales: (b, i, j, d / group) fp32 for an e4m3 output: max|y| of the group / 448, at least 2^-126, 1 where that is 0;
 * y is then the quotient y / scale rounded once, ties to even. */
int pair_sm100_add_norm(const pair_norm_desc_t* desc, const pair_tensor_t* update, const pair_tensor_t* residual,
                        const void* weight, void* stream, void* y, float* scales, trimul_stream_t cuda_stream);

/* Bytes of workspace that pair_sm100_add_norm_grad needs on the current device. */
int pair_sm100_add_norm_grad_workspace(const pair_norm_desc_t* desc, uint64_t* bytes);

/* Gradients of the norm form.  stream: z as pair_sm100_add_norm stored it; dy and dz: gradients of y and of z
 * (either may have data = NULL: zero).  d_stream (nullable) receives the residual's gradient, d_update (nullable) the
 * update's; without dropout they are the same values and one of them is enough.  d_weight may be NULL. */
int pair_sm100_add_norm_grad(const pair_norm_desc_t* desc, const pair_tensor_t* stream, const pair_tensor_t* dy,
                             const pair_tensor_t* dz, const void* weight, void* d_stream, void* d_update,
                             void* d_weight, void* workspace, trimul_stream_t cuda_stream);

typedef struct pair_embed_desc {
  int64_t tokens;
  int32_t d;
  int32_t rows;        /* of the table */
  int32_t index_bits;  /* 32 or 64 */
  int32_t dtype;       /* PAIR_*: out, base, d_out */
  int32_t table_dtype; /* PAIR_*: table and its gradient */
  float scale;
} pair_embed_desc_t;

/* out[t] = base[t] + scale * table[index[t]]; an index outside [0, rows) adds nothing.  All tensors contiguous; base
 * may be NULL and may be out itself. */
int pair_sm100_embed(const pair_embed_desc_t* desc, const void* index, const void* table, const void* base, void* out,
                     trimul_stream_t cuda_stream);

int pair_sm100_embed_grad_workspace(const pair_embed_desc_t* desc, uint64_t* bytes);

/* d_table[v] = scale * sum of d_out[t] over the tokens with index v, in a fixed order (the same bits every
 * time); rows that no token names become 0. */
int pair_sm100_embed_grad(const pair_embed_desc_t* desc, const void* index, const void* d_out, void* d_table,
                          void* workspace, trimul_stream_t cuda_stream);

#ifdef __cplusplus
}
#endif
#endif /* PAIR_STREAM_SM100_H_ */
