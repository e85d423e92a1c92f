/* SPDX-License-Identifier: Apache-2.0
 *
 * point_features: operators on the points' features for B200 (sm_100a):
 * rotary positions, cross attention between two levels of a hierarchy, and
 * attention along the rows of a radius or 3NN query, with their gradients.
 * Shared library: gsa_b200/_native/point_features.so
 *
 * They have no counterpart in GSA.  All tensors are DEVICE memory of the
 * current CUDA device; the argument structs and `turns` are host memory, read
 * during the call.  `stream` is a cudaStream_t; every call is stream-ordered,
 * allocates nothing and does not synchronise, so it can be captured.
 *
 * Return codes: 0 success; a cudaError_t value; -2 an invalid argument (a
 * size, type or stride out of range, a null or misaligned buffer, a workspace
 * that is too small).
 *
 * Rows are packed scene after scene: scene i owns rows seg[i] .. seg[i + 1],
 * seg[0] = 0 and seg[scenes] = the number of rows.  A row holds `heads` heads
 * of `dim` elements; rows and heads have strides, elements follow one another.
 */
#ifndef GSA_B200_POINT_FEATURES_H
#define GSA_B200_POINT_FEATURES_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define POINT_FEATURES_F32 0
#define POINT_FEATURES_F16 1
#define POINT_FEATURES_BF16 2

/* A tensor of rows: strides in elements.  Attention reads and writes 16 bytes
 * at a time: its tensors start on 16 bytes and their strides are multiples of
 * 16 bytes. */
typedef struct {
  const void* data;
  int64_t row, head;
} feature_rows;

typedef struct {
  int64_t type, rows, heads, dim;
  feature_rows x, y;        /* y may be x, else they do not overlap */
  const void* positions;    /* rows x axes, strides in elements */
  int64_t pos_type;         /* 0 float32, 1 int32, 2 int64 */
  int64_t pos_row, pos_axis;
  int64_t axes, pairs;      /* pairs per axis, at most 128 */
  const double* turns;      /* HOST [pairs]: whole turns per unit */
  double amplitude;
  int64_t interleaved;      /* pairs (2p, 2p+1), else (p, p + axes*pairs) */
  int64_t transposed;       /* turn back: the gradient */
  void* stream;
} rotary_args;

/* Pair p = axis * pairs + i of every head's first 2 * axes * pairs elements
 * turns by positions[row][axis] * turns[i] whole turns and is multiplied by
 * the amplitude; the other elements are copied. */
int rotary_positions(const rotary_args* a);

typedef struct {
  int64_t type, scenes, n_q, n_k;
  int64_t max_q, max_k;     /* longest scene */
  int64_t heads, kv_heads;  /* heads a multiple of kv_heads: head h reads
                               head h / (heads / kv_heads) of the keys; cross
                               attention: at most 64 heads per kv_head, 65535
                               kv_heads and 65535 scenes */
  int64_t dim;              /* a multiple of 8, at most 128 */
  double scale;             /* 2^-24 to 2^24 */
  feature_rows q, k, v;     /* cross: no strides of 0 or from 2^40 bytes on;
                               neighbor: row strides of what is gathered (k,
                               v; backward q and dout too) below 2^32 bytes */
  feature_rows out;         /* written forward, read backward */
  feature_rows dout;
  float* lse;               /* [n_q][heads], natural log; may be null forward */
  void *dq, *dk, *dv;       /* contiguous, of the inputs' type */
  const int32_t *q_seg, *k_seg;
  const uint8_t* mask;      /* cross: [n_k], 0 shuts a key out; may be null */
  const int32_t* ids;       /* neighbor: [n_q][width] scene-local key rows */
  int64_t width;            /* 1 .. 32 */
  int64_t padded;           /* entries that repeat the first do not count */
  void* workspace;          /* 16-byte aligned, private to the call until its
                               work is done; null when none is needed */
  int64_t workspace_bytes;
  int32_t* error;           /* cross: set to 1 if a bounded wait ran out */
  void* stream;
} attention_args;

/* out = softmax(scale q k^T) v over the open keys of each query's scene, for
 * float16 and bfloat16; lse = log sum exp of the scores.  A row without open
 * keys gives 0 and lse = -inf; one of open keys whose scores are all -inf gives
 * NaN and lse = NaN.  Shut keys may hold anything.
 * The workspace calls read the sizes only and return bytes, or -2. */
int cross_attention(const attention_args* a);
int64_t cross_attention_workspace(const attention_args* a);

/* The gradients of cross_attention's out, from its out and lse: dq [n_q]
 * [heads][dim], dk and dv [n_k][kv_heads][dim], all of them written.  Weights
 * are taken again from lse, whose 32 bits leave them off by some 2^-22 |lse| of
 * themselves (float16: beyond an |lse| of 2^22 they may overflow).  For
 * float16, rows whose |lse| / scale or |<dout, out>| is 2^31 or more make dk and
 * dv of their scene NaN. */
int cross_attention_grad(const attention_args* a);
int64_t cross_attention_grad_workspace(const attention_args* a);

/* The same over the keys that a query's row names, for float32 too (a row
 * without entries is one without open keys).  An entry outside the scene's keys
 * is absent; with `padded`, so is one behind the first that repeats it.  Other
 * repeats count each time. */
int neighbor_attention(const attention_args* a);
int neighbor_attention_grad(const attention_args* a);
int64_t neighbor_attention_grad_workspace(const attention_args* a);

/* Kernel launches issued by this library so far in the process. */
int launch_counter(unsigned long long* total);

#ifdef __cplusplus
}
#endif
#endif
