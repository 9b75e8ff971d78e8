/*
 * vectra_dense.h -- C ABI of the MI355X (gfx950) dense operators of a Transformer
 * block: the linear layers around its attention, forward and backward, and the 8-bit
 * form in which a training step may keep their input.
 *
 *   linear   y = act(x W^T + b) + r        x [rows, width_in], W [width_out, width_in],
 *                                          b [width_out], r and y [rows, width_out]
 *   gated    y = act(x G^T + b_g) * (x U^T + b_u)
 *                                          W [2 width_out, width_in]: the rows of G, then
 *                                          those of U; b [2 width_out] likewise
 *
 * Products are accumulated in fp32; bias, activation, product and residual are applied
 * to the fp32 sums, and the result is rounded once to the output's type.
 *
 * Gradients of y's sum weighted by g [rows, width_out]:
 *   linear   dz = g * act'(z), z = x W^T + b
 *   gated    dz = [g * u * act'(a), g * act(a)], [a, u] = x W^T + b
 *   dx = dz W      dW = dz^T x      db = column sums of dz      (dr = g)
 * dz is kept in the operands' type (one rounding) for the products; db sums it in fp32
 * before that rounding where the product that forms it can, else after.
 * z is computed again from x (or from x's 8-bit form): nothing but the inputs is needed.
 *
 * 8-bit rows: every 32 consecutive elements of a row share a power of two 2^e, the
 * smallest for which no finite element exceeds 448 2^e in magnitude (e >= -117; for
 * fp16 rows e >= -15), and an element x is kept as x / 2^e rounded to OCP e4m3 (ties
 * to even).  codes [rows, width] holds e4m3 bytes, scales [rows, ceil(width / 32)]
 * holds e + 127 as bytes.  A non-finite element becomes e4m3's NaN.  An element
 * whose rounding would pass its type's largest value takes the next code below.
 *
 * Contract (as vectra_rbf.h):
 *  - Plain pointers, sizes and strides; matrices are row-major with unit element
 *    stride and a row stride in ELEMENTS (codes and scales: in bytes, contiguous rows
 *    need not be adjacent) of at least a row; that of a single row is not read.
 *  - Every buffer is owned by the caller.  Calls that need scratch memory take a
 *    workspace whose size the _workspace_bytes function tells; it needs no set-up,
 *    holds nothing between calls, and must not be shared by calls that can overlap.
 *  - Work is enqueued on `stream` of the current device, without synchronising; calls
 *    are reentrant and may be captured into a HIP graph.  Results do not depend on the
 *    order in which workgroups run.
 *  - Errors are status codes (vectra_dense_status_string); on an argument error nothing
 *    was enqueued.
 */
#ifndef VECTRA_DENSE_H_
#define VECTRA_DENSE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* hipStream_t without pulling in the HIP headers. */
typedef struct ihipStream_t* vectra_dense_stream_t;

typedef enum vectra_dense_dtype {
  VECTRA_DENSE_F32 = 0,
  VECTRA_DENSE_F16 = 1,
  VECTRA_DENSE_BF16 = 2
} vectra_dense_dtype;

typedef enum vectra_dense_activation {
  VECTRA_DENSE_NONE = 0,      /* z                                  */
  VECTRA_DENSE_RELU = 1,      /* max(z, 0); slope 0 at 0            */
  VECTRA_DENSE_GELU = 2,      /* z Phi(z), Phi the normal distribution function */
  VECTRA_DENSE_GELU_TANH = 3, /* z / 2 (1 + tanh(sqrt(2/pi) (z + 0.044715 z^3))) */
  VECTRA_DENSE_SILU = 4       /* z / (1 + exp(-z))                  */
} vectra_dense_activation;

enum {
  VECTRA_DENSE_OK = 0,
  VECTRA_DENSE_ERR_NULL_ARGUMENT = 1,
  VECTRA_DENSE_ERR_BAD_DTYPE = 2,
  VECTRA_DENSE_ERR_BAD_SHAPE = 3,      /* negative sizes, strides smaller than a row  */
  VECTRA_DENSE_ERR_BAD_STRUCT = 4,     /* struct_size does not match this build       */
  VECTRA_DENSE_ERR_TOO_LARGE = 5,      /* a size exceeds the kernels' index range     */
  VECTRA_DENSE_ERR_LAUNCH = 6,         /* the HIP launch itself failed                */
  VECTRA_DENSE_ERR_BAD_ACTIVATION = 7,
  VECTRA_DENSE_ERR_WORKSPACE = 8       /* workspace missing, too small or not 256-byte aligned */
};

typedef struct vectra_dense_args {
  int64_t struct_size; /* sizeof(vectra_dense_args) as compiled by the caller */

  const void* x;
  const void* weight;
  const void* bias;     /* NULL: none */
  const void* residual; /* NULL: none; linear only */
  void* out;

  int32_t dtype;      /* of x, weight, residual and out */
  int32_t bias_dtype; /* dtype, or F32 */
  int32_t activation; /* VECTRA_DENSE_* */
  int32_t gated;      /* 0: linear, 1: gated */

  int64_t rows, width_in, width_out;
  int64_t x_stride, weight_stride, residual_stride, out_stride;
} vectra_dense_args;

typedef struct vectra_dense_grad_args {
  int64_t struct_size; /* sizeof(vectra_dense_grad_args) */

  const void* x;      /* the input, or NULL where codes and scales give it in 8 bits; neither is
                         read, and all may be NULL, for dx and db of an ungated layer without activation */
  const void* codes;
  const void* scales;
  const void* weight;
  const void* bias; /* NULL: none (db may still be asked for) */
  const void* grad; /* gradient of y */
  void* dx;         /* NULL: not wanted */
  void* dweight;    /* NULL: not wanted */
  void* dbias;      /* NULL: not wanted */

  int32_t dtype;      /* of x, weight, grad, dx, dweight */
  int32_t bias_dtype; /* of bias and dbias: dtype, or F32 */
  int32_t activation;
  int32_t gated;

  int64_t rows, width_in, width_out;
  int64_t x_stride, codes_stride, scales_stride, weight_stride, grad_stride;
  int64_t dx_stride, dweight_stride;
} vectra_dense_grad_args;

/* y.  rows == 0 or width_out == 0 is a successful no-op; width_in == 0 leaves
 * act(b) + r.  `out` may be the residual itself (the same pointer and stride);
 * any other overlap of out with an input is not allowed. */
int vectra_dense_forward(const vectra_dense_args* args, void* workspace, int64_t workspace_bytes,
                         vectra_dense_stream_t stream);
/* Bytes of workspace vectra_dense_forward needs for these arguments (0: none);
 * negative: -status. */
int64_t vectra_dense_forward_workspace_bytes(const vectra_dense_args* args);

/* dx, dW and db, those that are wanted.  rows == 0 sets dW and db to zero.  No
 * output may overlap an input or another output. */
int vectra_dense_backward(const vectra_dense_grad_args* args, void* workspace, int64_t workspace_bytes,
                          vectra_dense_stream_t stream);
int64_t vectra_dense_backward_workspace_bytes(const vectra_dense_grad_args* args);

/* The 8-bit form of x [rows, width] (dtype F32, F16 or BF16). */
int vectra_rows_quantize(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride,
                         void* codes, int64_t codes_stride, void* scales, int64_t scales_stride,
                         vectra_dense_stream_t stream);
/* What codes and scales stand for, in `dtype`, the type of the rows that were
 * quantised (another type rounds, and may overflow). */
int vectra_rows_dequantize(const void* codes, int64_t codes_stride, const void* scales, int64_t scales_stride,
                           int32_t dtype, int64_t rows, int64_t width, void* out, int64_t out_stride,
                           vectra_dense_stream_t stream);

const char* vectra_dense_status_string(int status);
/* (major << 16) | minor. */
int vectra_dense_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* VECTRA_DENSE_H_ */
