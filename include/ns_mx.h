/* ns_mx.h: C-ABI of the MI355X layer operators around attention and logits: the root-mean-square norm, the gated
 * activation, and products of microscaled (MX) rows with 4-bit weights.
 *
 * Replaces, in the reference's forward pass:
 *   nanoserve/model/llama.py:31-37    (RMSNorm) with the residual's addition around it (:75-85): ns_mx_rms_norm
 *   nanoserve/model/llama.py:53-56    (the MLP's silu(gate) * up): ns_mx_silu_mul
 *   its linear projections (llama.py:53-56, attention.py:97-135, compute_logits llama.py:136-143), with weights of 4
 *   bits: ns_mx_quantize once at load, ns_mx_linear.  The reference has 16-bit weights only.
 *
 * MX rows.  A row of `cols` values is padded with zeros to `k`, the next multiple of 128, and cut into blocks of 32.  A
 * block's values are codes times one power of two, 2^(s - 127) of its scale byte s; s = 255 makes every value of the
 * block NaN.  Codes: NS_MX_FP4 e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6; sign in bit 3), two to a byte, the even value in the
 * low half; NS_MX_FP8 e4m3 (up to 448).  Quantisation: s - 127 = floor(log2 of the block's largest magnitude) - 2 (FP4)
 * or - 8 (FP8), at least -127; codes are value / 2^(s - 127) to nearest even, saturating.  A block that holds a NaN or an
 * infinity gets s = 255 and zero codes.  A row's codes are contiguous and 16-byte aligned (k / 2 or k bytes), its scales
 * are k / 32 contiguous bytes, 4-byte aligned.
 *
 * All pointers are device pointers; nothing is read on the host, no call synchronizes or allocates, and every call can
 * be captured into a graph.  Calls keep nothing between them.
 */
#ifndef NS_MX_H
#define NS_MX_H

#include <stddef.h>
#include <stdint.h>
#include <hip/hip_runtime_api.h>

#ifdef __cplusplus
extern "C" {
#endif

#define NS_MX_ABI_VERSION 1

#define NS_MX_F32 0
#define NS_MX_BF16 1
#define NS_MX_F16 2
#define NS_MX_FP4 4    /* MX rows of e2m1 codes */
#define NS_MX_FP8 8    /* MX rows of e4m3 codes */

/* values a row is padded to a multiple of */
#define NS_MX_ROW_ALIGN 128

/* MX rows */
typedef struct ns_mx_rows {
  void*    codes;
  uint8_t* scales;
  int64_t  stride_codes;    /* bytes from row to row, a multiple of 16 */
  int64_t  stride_scales;   /* bytes from row to row, a multiple of 4 */
  int32_t  format;          /* NS_MX_FP4 or NS_MX_FP8 */
} ns_mx_rows;

/* h = x, or x + residual rounded to their type; y = h * weight / sqrt(mean(h^2) + eps), formed in float32 (the squares'
 * sum in float64) and rounded once, to the type or to MX codes.  Output row i is of input row rows[i] (i without rows);
 * an index outside the input gives a row of NaN.  With heads > 1 each of a row's heads is a norm of its own.
 * out and sum may be x or residual themselves where rows is NULL; otherwise they lie apart from what is read. */
typedef struct ns_mx_norm_args {
  const void*    x;                /* (n_x, heads, cols) */
  const void*    residual;         /* like x, or NULL */
  const void*    weight;           /* (cols), of x's type or float32 */
  const int64_t* rows;             /* (n), or NULL with n == n_x */
  void*          sum;              /* (n, heads, cols) of x's type: receives h; NULL: not wanted */
  void*          out;              /* (n, heads, cols) of x's type; NULL with out_mx */
  ns_mx_rows     out_mx;           /* (n) rows of cols values, heads == 1; format 0 with out */
  int64_t        n_x, n;
  int64_t        stride_x, stride_x_head;                 /* elements */
  int64_t        stride_residual, stride_residual_head;
  int64_t        stride_sum, stride_sum_head;
  int64_t        stride_out, stride_out_head;
  int32_t        heads, cols;
  int32_t        dtype, weight_dtype;   /* NS_MX_F32, _BF16, _F16 */
  float          eps;
} ns_mx_norm_args;

/* ns_mx_silu_mul: silu(gate) * up = gate / (1 + exp(-gate)) * up in float32, rounded once.  ns_mx_quantize: x = gate alone
 * (up NULL, out NULL), row i of input row rows[i] as for the norm.  ns_mx_silu_mul's out may be gate or up themselves. */
typedef struct ns_mx_gate_args {
  const void*    gate;             /* (n_x, cols) */
  const void*    up;               /* like gate */
  const int64_t* rows;             /* ns_mx_quantize alone: (n), or NULL with n == n_x */
  void*          out;              /* (n, cols) of gate's type; NULL with out_mx */
  ns_mx_rows     out_mx;
  int64_t        n_x, n;
  int64_t        stride_gate, stride_up, stride_out;      /* elements */
  int32_t        cols, dtype;
} ns_mx_gate_args;

/* out[i][j] = sum over c of x[i][c] w[j][c], products whole, their sums float32, rounded once to out's type.  Strides of x
 * and weight are below 2^23 bytes. */
typedef struct ns_mx_linear_args {
  ns_mx_rows     x;                /* (m) rows, either format */
  ns_mx_rows     weight;           /* (n) rows, NS_MX_FP4 */
  void*          out;              /* (m, n) */
  int64_t        stride_out;       /* elements */
  int64_t        m, n;
  int32_t        k;                /* padded width of both, a multiple of NS_MX_ROW_ALIGN */
  int32_t        dtype;            /* out's: NS_MX_F32, _BF16, _F16 */
} ns_mx_linear_args;

/* Version of this ABI (NS_MX_ABI_VERSION). */
int ns_mx_abi_version(void);

/* Message of the last failed call on this thread. */
const char* ns_mx_last_error(void);

/* Every function below returns 0, or nonzero on invalid arguments. */
int ns_mx_rms_norm(const ns_mx_norm_args* args, hipStream_t stream);
int ns_mx_silu_mul(const ns_mx_gate_args* args, hipStream_t stream);
int ns_mx_quantize(const ns_mx_gate_args* args, hipStream_t stream);
int ns_mx_linear(const ns_mx_linear_args* args, hipStream_t stream);

/* The first cols values of n MX rows as floats of a type, out (n, cols) with stride_out elements from row to row. */
int ns_mx_dequantize(const ns_mx_rows* rows, int64_t n, int32_t cols, void* out, int64_t stride_out, int32_t dtype,
                     hipStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* NS_MX_H */
