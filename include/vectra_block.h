/*
 * vectra_block.h -- C ABI of the MI355X (gfx950) operators between the dense products
 * of a Transformer block, and of those products in 8 bits.
 *
 *   dropout   y = k * x                  k = 65536 / (65536 - t) where an element is kept, else 0
 *   norm      h = s r + gate * k * post(x)        the residual stream with a branch's output
 *             n = norm(h)                         what the next branch reads
 *   linear    y = act(x^ W^T + b) + r    x^: x in 8 bits, W kept in 8 bits
 *   gated     y = act(x^ G^T + b_g) * (x^ U^T + b_u)
 *
 * Norms over a row of `width` elements, w and b per column (absent: 1 and 0):
 *   RMS       x / sqrt(mean(x^2) + eps) * w + b
 *   LAYER     (x - mean) / sqrt(var + eps) * w + b, var the mean of (x - mean)^2
 * Everything is computed in fp32 and rounded once, h and n apart (n from the unrounded h).
 *
 * Which elements are kept: Philox 4x32 with ten rounds (Salmon, Moraes, Dror, Shaw:
 * Parallel random numbers: as easy as 1, 2, 3; SC 2011).  Key: the 64-bit seed rng[0].
 * Counter, four 32-bit words: group, group >> 32, stream, rng[1] (its low 32 bits), where
 * group = row * ceil(width / 8) + column / 8.  Of its four words, element column % 8 = 2 j
 * takes the low half of word j, 2 j + 1 the high one, and is kept where those 16 bits are
 * at least t (0 <= t <= 65535: elements are dropped with probability t / 65536).  rng is
 * read on the device when the kernel runs: a captured graph draws anew when the program
 * changes it between replays.
 *
 * Gradients of the norm, for gradients gh of h and gn of n:
 *   gt = gh + norm'(h)^T gn     dr = s gt     dgate = sum of gt * k * post(x)
 *   du = gate * k * gt          dx = post'(x)^T du (du itself without a post norm)
 *   dw = sum of gn * normalised h, db = sum of gn, likewise post's from du.
 *
 * 8-bit blocks: elements that share a power of two 2^e, the smallest for which no finite
 * one exceeds 448 2^e in magnitude (e >= -117), are kept as x / 2^e rounded to OCP e4m3
 * (ties to even); non-finite ones become NaN, and one that would round past fp32's
 * largest value (e = 120) takes the code below.  Rows: 128 consecutive elements of a row.
 * Tiles: 128 rows of 128.  codes [rows, depth], depth = width rounded up to 128 (the
 * padding is zero); scales [ceil(rows / 1 or 128), 4 ceil(width / 512)] hold e + 127 as
 * bytes (those past ceil(width / 128) are 0 and not used); rows are adjacent.
 * Products take any byte b from 0 to 254 as 2^(b - 127), and 255 as NaN.  A code that
 * stands for more than fp32's largest value, as no call here makes one, counts as infinite
 * there, or, on the 8-bit matrix cores, as the value that it has.
 *
 * Sums of the products: F32 results, and results of at most 32 rows, are exact products
 * added in fp32.  Larger products with 16-bit results run on the 8-bit matrix cores: of
 * each 16 products of a row and a column those bits are dropped that lie below 2^-13 of
 * the largest one's power of two, and the sums are added in fp32.
 * (1.6e-5 of a result of normal operands; 1e-2 of one beside which products of 500 times
 * its size cancel.  F32 results of the same codes, rounded by the caller, are without it.)
 *
 * Contract (as vectra_dense.h):
 *  - Plain pointers, sizes and strides; matrices are row-major with unit element stride
 *    and a row stride in ELEMENTS of at least a row; that of a single row is not read.
 *    Rows are at most 2^21 wide (of a norm VECTRA_BLOCK_NORM_WIDTH), and rows * (width + 512)
 *    is below 2^35.
 *    Codes begin at a multiple of 16 bytes, scales of 4.
 *  - Every buffer is owned by the caller.  Calls that need scratch memory take a workspace
 *    whose size the _workspace_bytes function tells; it needs no set-up, holds nothing
 *    between calls, and must not be shared by calls that can overlap.
 *  - Work is enqueued on `stream` of the current device, without synchronising; calls are
 *    reentrant and may be captured into a HIP graph.  Results do not depend on the order
 *    in which workgroups run.
 *  - Errors are status codes (vectra_block_status_string); on an argument error nothing
 *    was enqueued.
 */
#ifndef VECTRA_BLOCK_H_
#define VECTRA_BLOCK_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* hipStream_t without pulling in the HIP headers. */
typedef struct ihipStream_t* vectra_block_stream_t;

typedef enum vectra_block_dtype {
  VECTRA_BLOCK_F32 = 0,
  VECTRA_BLOCK_F16 = 1,
  VECTRA_BLOCK_BF16 = 2
} vectra_block_dtype;

typedef enum vectra_block_norm {
  VECTRA_BLOCK_NO_NORM = 0, /* post only */
  VECTRA_BLOCK_RMS = 1,
  VECTRA_BLOCK_LAYER = 2
} vectra_block_norm;

enum {
  VECTRA_BLOCK_OK = 0,
  VECTRA_BLOCK_ERR_NULL_ARGUMENT = 1,
  VECTRA_BLOCK_ERR_BAD_DTYPE = 2,
  VECTRA_BLOCK_ERR_BAD_SHAPE = 3,  /* negative sizes, strides smaller than a row, unaligned codes */
  VECTRA_BLOCK_ERR_BAD_STRUCT = 4, /* struct_size does not match this build      */
  VECTRA_BLOCK_ERR_TOO_LARGE = 5,  /* a size exceeds the kernels' range          */
  VECTRA_BLOCK_ERR_LAUNCH = 6,     /* the HIP launch itself failed               */
  VECTRA_BLOCK_ERR_BAD_OPTION = 7, /* unknown norm or activation, threshold, eps */
  VECTRA_BLOCK_ERR_WORKSPACE = 8   /* workspace missing, too small or not 256-byte aligned */
};

/* Widest row of a norm. */
#define VECTRA_BLOCK_NORM_WIDTH 16384

/* y = k * x.  `rng`: two int64 on the device; not read (and may be NULL) for threshold 0. */
int vectra_dropout(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, void* y,
                   int64_t y_stride, int32_t threshold, const int64_t* rng, uint32_t stream_id,
                   vectra_block_stream_t stream);

typedef struct vectra_norm_args {
  int64_t struct_size; /* sizeof(vectra_norm_args) as compiled by the caller */

  const void* x;           /* [rows, width] */
  const void* residual;    /* [rows, width] */
  const void* weight;      /* [width]; this and the next four may be NULL */
  const void* bias;        /* [width] */
  const void* gate;        /* [ceil(rows / gate_rows), width]: a row for each gate_rows consecutive ones */
  const void* post_weight; /* [width] */
  const void* post_bias;   /* [width] */
  const int64_t* rng;      /* as above */
  void* h;                 /* [rows, width] */
  void* n;                 /* [rows, width], or NULL where codes and scales take it in 8-bit rows */
  void* codes;
  void* scales;

  int32_t dtype;        /* of x and n */
  int32_t stream_dtype; /* of residual and h: dtype, or F32 */
  /* Of the vectors, each dtype or F32; those of NULL pointers are not read. */
  int32_t weight_dtype, bias_dtype, gate_dtype, post_weight_dtype, post_bias_dtype;
  int32_t norm; /* RMS or LAYER */
  int32_t post; /* NO_NORM, RMS or LAYER */
  int32_t threshold;
  uint32_t stream_id;
  float eps, residual_scale;

  int64_t rows, width, gate_rows;
  int64_t x_stride, residual_stride, gate_stride, h_stride, n_stride;
} vectra_norm_args;

typedef struct vectra_norm_grad_args {
  int64_t struct_size; /* sizeof(vectra_norm_grad_args) */

  const void* grad_h; /* NULL: zero */
  const void* grad_n; /* NULL: zero */
  /* With a gate, a post norm or a stream of 16 bits: x and residual.  Else h, in fp32. */
  const void* x;
  const void* residual;
  const void* h;
  const void* weight;
  const void* gate;
  const void* post_weight;
  const void* post_bias;
  const int64_t* rng;
  /* The gradients that are wanted; NULL: not wanted. */
  void* dx;
  void* dresidual;
  void* dweight;
  void* dbias;
  void* dgate;
  void* dpost_weight;
  void* dpost_bias;

  int32_t dtype, stream_dtype; /* dtype: x, grad_n, dx; stream_dtype: residual, h, grad_h, dresidual */
  int32_t weight_dtype, bias_dtype, gate_dtype, post_weight_dtype, post_bias_dtype; /* of the vectors and their gradients */
  int32_t norm, post, threshold;
  uint32_t stream_id;
  float eps, residual_scale;

  int64_t rows, width, gate_rows;
  int64_t grad_h_stride, grad_n_stride, x_stride, residual_stride, h_stride, gate_stride;
  int64_t dx_stride, dresidual_stride, dgate_stride;
} vectra_norm_grad_args;

/* h and n.  rows == 0 or width == 0 is a successful no-op.  No output may overlap an input. */
int vectra_norm_forward(const vectra_norm_args* args, vectra_block_stream_t stream);

/* rows == 0 sets the gradients of `width` elements to zero (the gate's has no rows then). */
int vectra_norm_backward(const vectra_norm_grad_args* args, void* workspace, int64_t workspace_bytes,
                         vectra_block_stream_t stream);
int64_t vectra_norm_backward_workspace_bytes(const vectra_norm_grad_args* args);

/* 8-bit rows (tiles == 0) or tiles (tiles == 1) of x [rows, width]. */
int vectra_blocks_quantize(const void* x, int32_t dtype, int64_t rows, int64_t width, int64_t x_stride, int32_t tiles,
                           void* codes, void* scales, vectra_block_stream_t stream);

typedef struct vectra_linear8_args {
  int64_t struct_size; /* sizeof(vectra_linear8_args) */

  const void* x;             /* [rows, width], or NULL where codes and scales give it in 8-bit rows */
  const void* codes;         /* [rows, depth] */
  const void* scales;        /* [rows, 4 ceil(width / 512)] */
  const void* weight;        /* codes of 8-bit tiles, [width_out (gated: 2 width_out), depth] */
  const void* weight_scales; /* [ceil(that / 128), 4 ceil(width / 512)] */
  const void* bias;          /* NULL: none */
  const void* residual;      /* NULL: none; linear only */
  void* out;                 /* [rows, width_out] */

  int32_t dtype;      /* of x, residual and out */
  int32_t bias_dtype; /* dtype, or F32 */
  int32_t activation; /* as vectra_dense_activation of vectra_dense.h */
  int32_t gated;

  int64_t rows, width, width_out;
  int64_t x_stride, residual_stride, out_stride;
} vectra_linear8_args;

/* y.  rows == 0 or width_out == 0 is a successful no-op; width == 0 leaves act(b) + r.
 * `out` may be the residual itself (the same pointer and stride); any other overlap of
 * out with an input is not allowed. */
int vectra_linear8_forward(const vectra_linear8_args* args, void* workspace, int64_t workspace_bytes,
                           vectra_block_stream_t stream);
int64_t vectra_linear8_workspace_bytes(const vectra_linear8_args* args);

const char* vectra_block_status_string(int status);
/* (major << 16) | minor. */
int vectra_block_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* VECTRA_BLOCK_H_ */
