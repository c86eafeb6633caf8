/* fermix_b200: the operators of the attention blocks whose orbitals the determinants take
 * (part of libfermix_b200.so, same conventions as fermix_b200.h: stream-ordered, no
 * allocation, FX_* status codes, caller-owned memory).
 *
 *   fermix_residual_norm     u = norm(f), r = x + scale gate u, z = norm(r)
 *   fermix_position_bias     out[b, h, i, j] = table[h, bucket(k_pos[b, j] - q_pos[b, i])]
 *   fermix_biased_attention  softmax(scale q k^T + bias) v with the same bias inside
 *
 * and the gradients of each (*_grad). dtype is FX_F32 or FX_BF16; statistics, sums and
 * softmax are float32. The channel and table gradients are summed in a fixed order, so
 * repeated calls give the same bits.
 */
#ifndef FERMIX_B200_BLOCK_H
#define FERMIX_B200_BLOCK_H

#include <stddef.h>
#include <stdint.h>

#include "fermix_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FX_BF16 4

/* ---- gated residual with its norms ---------------------------------------------------
 * Rows are (groups, rows) of `width` contiguous entries. kind 0: x / rms(x); kind 1: the
 * mean is taken off first. gate_mode: 0 none, 1 an entry per entry, 2 one per row,
 * 3 one vector per group (dgate_f32: modes 1 and 3 write float32 gradients of the gate, for a
 * caller that sums them further). post_* act on f, pre_* on r; scale, *_bias and gate may be NULL.
 * 1 <= width <= FX_NORM_MAX_WIDTH. */
#define FX_NORM_MAX_WIDTH 8192
#define FX_GATE_NONE 0
#define FX_GATE_FULL 1
#define FX_GATE_ROW 2
#define FX_GATE_GROUP 3

typedef struct {
  int32_t dtype, kind, gate_mode, dgate_f32;
  float eps;
  int32_t reserved;
  int64_t groups, rows, width;
  const void *x, *f, *gate, *scale, *post_weight, *post_bias, *pre_weight, *pre_bias;
  /* forward */
  void *r, *z;
  /* backward: grad_r / grad_z may be NULL (zero). dx, df and the weights' gradients are
   * required, the others where their input is given. */
  const void *grad_r, *grad_z;
  void *dx, *df, *dgate, *dscale, *dpost_weight, *dpost_bias, *dpre_weight, *dpre_bias;
} fx_norm_args;

int fermix_residual_norm(void* stream, const fx_norm_args* args);
int fermix_residual_norm_grad(void* stream, const fx_norm_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_residual_norm_grad_workspace_bytes(const fx_norm_args* args);

/* ---- position buckets ----------------------------------------------------------------
 * With d = k_pos - q_pos: two-sided, bucket = #(edges <= |d|), plus num_buckets / 2 where
 * d > 0; one-sided, bucket = #(edges <= max(-d, 0)). edges is a HOST array, ascending,
 * edges[0] >= 1, num_edges < num_buckets (two-sided: < num_buckets / 2), and
 * edges[num_edges - 1] <= FX_BUCKET_MAX_EDGE. Positions are within +-2^29. */
#define FX_BUCKET_MAX 256
#define FX_BUCKET_MAX_EDGE 2048

typedef struct {
  int32_t num_buckets, two_sided, num_edges, reserved;
  const int32_t* edges;
  /* (q_len) or, with a batch stride, (batch, q_len); NULL: k_pos[j] = j and
   * q_pos[i] = k_len - q_len + i */
  const int32_t *q_pos, *k_pos;
  int64_t q_pos_stride, k_pos_stride;
} fx_buckets;

typedef struct {
  int32_t dtype, reserved;
  int64_t batch, heads, q_len, k_len;
  fx_buckets buckets;
  const void* table; /* (heads, num_buckets) */
  void* out;         /* (batch, heads, q_len, k_len) */
  const void* grad;  /* backward: of out, contiguous */
  void* dtable;
} fx_bias_args;

int fermix_position_bias(void* stream, const fx_bias_args* args);
int fermix_position_bias_grad(void* stream, const fx_bias_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_position_bias_grad_workspace_bytes(const fx_bias_args* args);

/* ---- attention with the position bias ------------------------------------------------
 * q (batch, heads, q_len, dim), k and v (batch, kv_heads, k_len, dim), heads a multiple of
 * kv_heads, 1 <= dim <= FX_ATTN_MAX_DIM, by element strides (batch, head, token); the
 * entries of a token are contiguous. key_mask (batch, k_len) bytes or NULL: 0 leaves the
 * key out whatever it holds; causal leaves out keys with k_pos > q_pos. A row with no key
 * gives 0, and no gradient. table NULL: no bias. lse (batch, heads, q_len) float32, the
 * logarithm (base 2) of each row's sum of exponentials: written by the forward when not
 * NULL, read by the backward. lse_low, of the same shape: what lse's rounding left out of it,
 * written (where lse is) and read alike; NULL: taken as zero, which is near enough unless a
 * row's bias is huge beside its scores (log2 n of a row whose n keys all carry -1e9 is in
 * lse_low alone). */
#define FX_ATTN_MAX_DIM 128

typedef struct {
  int32_t dtype, causal;
  int64_t batch, heads, kv_heads, q_len, k_len, dim;
  float scale;
  int32_t reserved;
  fx_buckets buckets;
  const void *q, *k, *v, *table;
  int64_t q_stride[3], k_stride[3], v_stride[3];
  const uint8_t* key_mask;
  int64_t mask_stride;
  void* out;
  int64_t out_stride[3];
  float* lse;
  /* backward */
  const void* dout;
  int64_t dout_stride[3];
  void *dq, *dk, *dv, *dtable;
  int64_t dq_stride[3], dk_stride[3], dv_stride[3];
  float* lse_low;
} fx_attn_args;

int fermix_biased_attention(void* stream, const fx_attn_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_biased_attention_workspace_bytes(const fx_attn_args* args);
int fermix_biased_attention_grad(void* stream, const fx_attn_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_biased_attention_grad_workspace_bytes(const fx_attn_args* args);

#ifdef __cplusplus
}
#endif
#endif
