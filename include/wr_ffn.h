/*
 * wr_ffn.h -- C-ABI of the dense gated FFN and the int8 products of
 * libwarp_route_hip.so: the FFN (or shared expert) that stands beside a
 * routed MoE layer, its backward pass, and its int8 form.  Conventions are
 * those of warp_route.h: plain device pointers and sizes, wr_status codes,
 * every argument checked before the first HIP call, work enqueued on `stream`,
 * nothing allocated, nothing synchronised.  No counterpart in the reference.
 *
 * With g = x Wg^T, u = x Wu^T, s = 1 / (1 + exp(-g)):
 *   a  = g s u                              [T, I]
 *   y  = a Wd^T                             [T, h]
 * and for a gradient dy of y, with da = dy Wd:
 *   du = da g s,  dg = da u s (1 + g (1 - s))
 *   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T a
 * Sums are fp32.  a, dg and du are rounded to the call's dtype, in which the
 * matrix cores read them; g and u are kept in fp32, so that the gradients
 * see one rounding before their last product, as y does.
 *
 * Matrices are row-major and contiguous; pointers are 16-byte aligned.
 * A call may be recorded into a HIP graph.
 */
#ifndef WR_FFN_H
#define WR_FFN_H

#include "warp_route.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest hidden_dim, intermediate_dim, and rows or columns of a weight. */
#define WR_FFN_MAX_DIM (1 << 20)
/* Most rows (tokens) of a call, and most columns that wr_quantize_int8 takes. */
#define WR_FFN_MAX_ROWS (1 << 28)
#define WR_INT8_MAX_COLS (1 << 30)
/* Largest K of an int8 product: 128 * 128 * K stays inside an int32. */
#define WR_INT8_MAX_K 131071

typedef struct wr_ffn_args {
  const void *x;        /* [T, h]                                               */
  const void *w_gate;   /* [I, h]                                               */
  const void *w_up;     /* [I, h]                                               */
  const void *w_down;   /* [h, I]                                               */
  void *out;            /* forward: y [T, h]                                    */
  float *saved_gate;    /* g, u (fp32) and a (dtype), [T, wr_ffn_saved_row(I)]  */
  float *saved_up;      /*   each.  Forward: written when all three are given,  */
  void *saved_act;      /*   all NULL: not kept.  Backward: as forward wrote.   */
  const void *dout;     /* backward: dy [T, h]                                  */
  void *dx;             /* backward: gradients, each optional (NULL: not       */
  void *dw_gate;        /*   computed)                                          */
  void *dw_up;
  void *dw_down;
  int32_t dtype;        /* WR_F32, WR_F16 or WR_BF16, of every matrix           */
  int32_t batch_size;   /* T >= 0                                               */
  int32_t hidden_dim;   /* h                                                    */
  int32_t intermediate_dim; /* I                                                */
  void *workspace;      /* device scratch, >= wr_ffn_workspace_bytes(...)       */
  size_t workspace_bytes;
} wr_ffn_args;

/* Elements of one row of a saved buffer: I rounded up to a multiple of 64; 0
 * for an invalid I. */
WR_API int64_t wr_ffn_saved_row(int intermediate_dim);

/* Workspace of a forward (backward = 0) or backward (1) call, or 0 for
 * invalid arguments. */
WR_API size_t wr_ffn_workspace_bytes(int backward, int dtype, int hidden_dim,
                                     int intermediate_dim, int batch_size);

WR_API int wr_ffn_forward(const wr_ffn_args *args, void *stream);
WR_API int wr_ffn_backward(const wr_ffn_args *args, void *stream);

/* int8 codes and scales of rows: with m = max |row|,
 *   scale = m / 127 (fp32),  code = 127 x / m rounded to nearest, ties to even
 * (the exact quotient's rounding).  A row of zeros gets scale 1; a row with a
 * non-finite value gets codes 0 and scale NaN, so that whatever is computed
 * from it is NaN.  codes [rows, cols], scales [rows]. */
WR_API int wr_quantize_int8(const void *x, int dtype, int rows, int cols, int8_t *codes,
                            float *scales, void *stream);

typedef struct wr_int8_args {
  const int8_t *x;        /* [M, K] codes                                        */
  const float *x_scale;   /* [M]                                                 */
  const int8_t *w;        /* [N, K] codes                                        */
  const float *w_scale;   /* [N]                                                 */
  void *out;              /* [M, N]                                              */
  int32_t out_dtype;      /* WR_F32, WR_F16 or WR_BF16                           */
  int32_t rows;           /* M >= 0                                              */
  int32_t out_features;   /* N                                                   */
  int32_t in_features;    /* K <= WR_INT8_MAX_K                                  */
  void *workspace;        /* >= wr_int8_workspace_bytes(...)                     */
  size_t workspace_bytes;
} wr_int8_args;

/* out[m][n] = (sum_k x[m][k] w[n][k]) x_scale[m] w_scale[n], the sum exact. */
WR_API size_t wr_int8_workspace_bytes(int rows, int out_features, int in_features);
WR_API int wr_int8_matmul(const wr_int8_args *args, void *stream);

/* The gated FFN on int8 weights: x is quantised per token (wr_quantize_int8),
 * g and u are int8 products, a is computed in fp32 and quantised per token,
 * y is an int8 product of out's dtype (= x's). */
typedef struct wr_ffn_int8_args {
  const void *x;          /* [T, h]                                              */
  const int8_t *w_gate;   /* [I, h] codes                                        */
  const float *s_gate;    /* [I]                                                 */
  const int8_t *w_up;     /* [I, h]                                              */
  const float *s_up;      /* [I]                                                 */
  const int8_t *w_down;   /* [h, I]                                              */
  const float *s_down;    /* [h]                                                 */
  void *out;              /* [T, h]                                              */
  int32_t dtype;          /* of x and out                                        */
  int32_t batch_size;     /* T >= 0                                              */
  int32_t hidden_dim;     /* h <= WR_INT8_MAX_K                                  */
  int32_t intermediate_dim; /* I <= WR_INT8_MAX_K                                */
  void *workspace;
  size_t workspace_bytes;
} wr_ffn_int8_args;

WR_API size_t wr_ffn_int8_workspace_bytes(int hidden_dim, int intermediate_dim, int batch_size);
WR_API int wr_ffn_int8(const wr_ffn_int8_args *args, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* WR_FFN_H */
