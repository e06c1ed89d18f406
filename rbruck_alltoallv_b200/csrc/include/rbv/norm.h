/* The norms behind and in front of a transformer block, fused with the block's gate, the residual scale and the residual
 * sum, forward and backward.  The reference library has no compute kernels.
 *
 *   zhat = z / sqrt(mean(z^2) + eps)            r2 = r + scale * gate * w1 * zhat
 *   xhat = r2 / sqrt(mean(r2^2) + eps)          u  = xhat * w2
 */
#ifndef RBV_NORM_H_
#define RBV_NORM_H_

#ifdef __cplusplus
extern "C" {
#endif

enum { RBV_NORM_BF16 = 0, RBV_NORM_FP16 = 1, RBV_NORM_FP32 = 2 };
enum { RBV_GATE_NONE = 0, RBV_GATE_CHANNEL = 1, RBV_GATE_TOKEN = 2, RBV_GATE_FULL = 3 };   /* 1, [H], [T], [T, H] */
#define RBV_NORM_MAX_HIDDEN 16384

/* One call of T >= 1 rows.  Rows of H elements, `*_ld` elements apart; written tensors are packed.  z, u, dz, du (and a full gate) have the
 * type z_type; r, r2, dr, dr2 the type r_type, which is z_type or fp32.  Each weight and the gate is fp32 where its flag is
 * set and of z_type otherwise.  z null: no block (r2 = r, not written); w2 null: no second norm (u not written). */
typedef struct {
  long long T;
  int H, z_type, r_type, gate_kind, w1_f32, w2_f32, gate_f32;
  float scale, eps;
  const void *z, *r, *w1, *gate, *w2;
  long long z_ld, r_ld, gate_ld;
  float *rstd1, *rstd2;             /* [T] each: written by the forward pass (may be null), read by the backward pass */
  void *r2, *u;                     /* forward only */
  /* backward only: gradients of r2 and u (null: zero), of z and r, of a gate per token or element, and of what is summed over
   * the tokens (each may be null); partial: fp32 [rbv_block_norm_parts(T, H, z_type)][2][H] workspace, null if no gradient
   * of a weight or of a gate per channel is asked for */
  const void *dr2, *du;
  long long dr2_ld, du_ld;
  void *dz, *dr, *dgate, *dw1, *dw2;
  float* partial;
} rbv_norm_t;

/* Both return 0 or a CUDA error code. */
int rbv_block_norm(const rbv_norm_t* call, void* cuda_stream);
int rbv_block_norm_backward(const rbv_norm_t* call, void* cuda_stream);
/* Rows of the workspace that the backward pass wants (for the current device). */
int rbv_block_norm_parts(long long T, int H, int z_type);

#ifdef __cplusplus
}
#endif
#endif
