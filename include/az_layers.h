/* az_layers.h -- C ABI of the network layers outside the search (libaz_mcts.so, gfx950): a dense
 * layer with bias, activation and residual, a layer norm, both with their backward passes, and the
 * draw of an action from truncated policy logits.
 *
 * The reference's networks are flax Dense / activation stacks (networks/networks.py:25-48); these
 * entry points are their layers, and the residual blocks' built from them, as single operators.
 *
 * Conventions of az_mcts.h: device pointers owned by the caller, row-major and contiguous; calls
 * enqueue on `stream` of the current device and do not synchronise, allocate or keep anything
 * between calls; return codes and az_last_error() as there.  Workspaces are scratch of one call:
 * calls that may overlap need workspaces of their own.
 */
#ifndef AZ_LAYERS_H_
#define AZ_LAYERS_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define AZ_TYPE_F32 0
#define AZ_TYPE_BF16 1
#define AZ_TYPE_F16 2

/* activations */
#define AZ_ACT_NONE 0
#define AZ_ACT_RELU 1
#define AZ_ACT_SWISH 2 /* z / (1 + exp(-z)) */
#define AZ_ACT_GELU 3  /* z * (1 + erf(z / sqrt 2)) / 2 */

#define AZ_DENSE_MAX_WIDTH 1048576     /* fan_in, fan_out */
#define AZ_NORM_MAX_WIDTH 1048576
#define AZ_SAMPLE_MAX_ACTIONS 1048576

/* y[rows, fan_out] = act(x[rows, fan_in] kernel[fan_in, fan_out] + bias[fan_out]) + residual
 *
 * x, kernel, bias (may be NULL), residual [rows, fan_out] (may be NULL) and y have the type `dtype`;
 * sums are held in float32 and rounded once, into y.  z (may be NULL; only with an activation)
 * receives the pre-activation for az_dense_backward: float32 for AZ_TYPE_F32, otherwise float16
 * whatever the 16-bit type.  y may be `residual` itself.
 * workspace: az_dense_workspace_bytes(dtype, rows, fan_in, fan_out, 0) bytes, 16-byte aligned (NULL if 0).
 * rows = 0 is allowed and does nothing. */
int az_dense_forward(int32_t dtype, int32_t act, int32_t rows, int32_t fan_in, int32_t fan_out,
                     const void* x, const void* kernel, const void* bias, const void* residual, void* y,
                     void* z, void* workspace, int64_t workspace_bytes, void* stream);

/* The gradients of az_dense_forward for dy[rows, fan_out]: with dz = dy act'(z) (for the 16-bit types, whose
 * matrix instructions take it, as the sum of two values of that type: to 2^-16 of itself, AZ_TYPE_F16 2^-22),
 *   dx = dz kernel^T,  dkernel = x^T dz,  dbias = column sums of dz in float32.
 * (the residual's gradient is dy).  Any of dx, dkernel, dbias may be NULL.  x is read for dkernel,
 * kernel for dx, z with an activation.  Sums have a fixed order: results do not depend on timing.
 * rows = 0 sets dkernel and dbias to zero.
 * workspace: az_dense_workspace_bytes(dtype, rows, fan_in, fan_out, 1) bytes, 16-byte aligned. */
int az_dense_backward(int32_t dtype, int32_t act, int32_t rows, int32_t fan_in, int32_t fan_out,
                      const void* x, const void* kernel, const void* z, const void* dy, void* dx,
                      void* dkernel, void* dbias, void* workspace, int64_t workspace_bytes, void* stream);

/* Bytes of the workspace of a forward (pass 0) or backward (pass 1) call; -1 for sizes the calls refuse. */
int64_t az_dense_workspace_bytes(int32_t dtype, int32_t rows, int32_t fan_in, int32_t fan_out, int32_t pass);

/* y = (x - mean) * rstd * scale + bias over the last axis of x[rows, width], with the biased variance
 * and rstd = 1 / sqrt(variance + eps).  scale and bias [width] may each be NULL (1 and 0); they have the type
 * `param_dtype`, which is `dtype` or AZ_TYPE_F32.  mean and rstd [rows] float32 (both or neither NULL) are
 * kept for az_layer_norm_backward.  Sums are float32: a row whose values or squared differences add up to more than
 * that holds (deviations around 1e19) has an infinite variance. */
int az_layer_norm_forward(int32_t dtype, int32_t param_dtype, int32_t rows, int32_t width, const void* x,
                          const void* scale, const void* bias, float eps, void* y, float* mean, float* rstd,
                          void* stream);

/* With xhat = (x - mean) * rstd and h = dy * scale:
 *   dx = rstd * (h - mean(h) - xhat * mean(h * xhat)),  dscale = column sums of dy * xhat,
 *   dbias = column sums of dy  (the last two of type `param_dtype`).  Any of the three may be NULL.
 * workspace: az_layer_norm_workspace_bytes(rows, width) bytes, 16-byte aligned; read only if dscale or dbias is
 * asked for.  Sums have a fixed order. */
int az_layer_norm_backward(int32_t dtype, int32_t param_dtype, int32_t rows, int32_t width, const void* x,
                           const void* scale, const float* mean, const float* rstd, const void* dy, void* dx,
                           void* dscale, void* dbias, void* workspace, int64_t workspace_bytes, void* stream);

int64_t az_layer_norm_workspace_bytes(int32_t rows, int32_t width);

/* Draws one action a row from truncated policy logits.
 *
 * Weights w = exp((l - max l) / temperature) over the row's legal actions.  Of their descending order (equal
 * logits by index) the first top_k are kept, of these the fewest that hold top_p of the mass of the top_k
 * (one at least), of these the ones with w >= max(min_p, 2^-40).  With the kept weights' sum W, the action is
 * the first in INDEX order whose cumulative kept weight exceeds uniform * W, log_prob = log(w / W).
 * An illegal action has invalid != 0; -inf and NaN logits count as illegal.  Where +inf logits are present they
 * share the mass.  A row without a legal action gives action 0 and log_prob -inf.
 *
 * Each parameter is a number or, if its pointer is not NULL, one value a row: temperature (0, negative, NaN or
 * below 1e-300: the likeliest action), top_k (<= 0: all), top_p (>= 1 or NaN: all), min_p (<= 0 or NaN: none; above 1 it is 1).
 * Weights are summed as 64-bit integers (unit: the largest weight / 2^41 or finer; each is rounded to a whole one): draws
 * do not depend on the order of the additions. */
typedef struct az_sample_desc {
  int32_t dtype, rows, actions, top_k;
  double temperature, top_p, min_p;
  const void* logits;              /* [rows, actions] of type dtype */
  const float* uniform;            /* [rows], in [0, 1) */
  const uint8_t* invalid;          /* [rows, actions], may be NULL */
  const float* temperature_rows;   /* [rows], may be NULL; likewise below */
  const int32_t* top_k_rows;
  const float* top_p_rows;
  const float* min_p_rows;
} az_sample_desc;

int az_sample_actions(const az_sample_desc* d, int32_t* action, float* log_prob /* may be NULL */, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* AZ_LAYERS_H_ */
