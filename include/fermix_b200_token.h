/* fermix_b200: the operators around the attention blocks whose orbitals the determinants take
 * (part of libfermix_b200.so, same conventions as fermix_b200.h: stream-ordered, no
 * allocation, FX_* status codes, caller-owned memory).
 *
 *   fermix_token_embedding   out[i] = scale table[token[i]]
 *   fermix_linear            y = residual + act(x W^T + b)
 *   fermix_token_logprobs    log p[i, token[i]] of softmax(scale logits), entropy, likeliest entries
 *
 * and the gradients of each (*_grad). dtype is FX_F32 or FX_BF16; sums, statistics and
 * log probabilities are float32. Every gradient is summed in a fixed order, so repeated calls
 * give the same bits. Tokens are whole numbers of token_bytes 1 (unsigned), 2, 4 or 8 (signed).
 */
#ifndef FERMIX_B200_TOKEN_H
#define FERMIX_B200_TOKEN_H

#include <stddef.h>
#include <stdint.h>

#include "fermix_b200_block.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- embedding -------------------------------------------------------------------------
 * weight (rows, width), out and grad (count, width), contiguous. A token equal to `padding`
 * (where has_padding) gives zeros and has no gradient; any other token outside [0, rows) gives
 * NaN and has no gradient. dweight gets every row, zeros where no token is. count and rows
 * < 2^31 - 1, 1 <= width <= FX_EMBED_MAX_WIDTH. */
#define FX_EMBED_MAX_WIDTH (1 << 23)

typedef struct {
  int32_t dtype, token_bytes;
  int64_t count, rows, width, padding;
  int32_t has_padding;
  float scale;
  const void *tokens, *weight;
  void* out;
  /* backward */
  const void* grad;
  void* dweight;
} fx_embed_args;

int fermix_token_embedding(void* stream, const fx_embed_args* args);
int fermix_token_embedding_grad(void* stream, const fx_embed_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_token_embedding_grad_workspace_bytes(const fx_embed_args* args);

/* ---- linear map with its epilogue ------------------------------------------------------
 * h = x W^T + b, y = residual + act(h). x (rows, inner), weight (outer, inner), residual and dy
 * (rows, outer) by the element stride of a row, entries contiguous; y, slope and the
 * gradients contiguous. bias and residual may be NULL. slope (rows, outer), act'(h): written
 * by the forward where not NULL, required by the backward unless act is FX_ACT_NONE; IEEE half
 * for FX_BF16 (a derivative lies within +-1.2 and needs more bits, not more range), float32
 * for FX_F32. The backward computes the gradients whose pointers are given: with
 * g = dy act'(h), dx = g W, dweight = g^T x, dbias = the sum of g over the rows. rows, inner and
 * outer < 2^30. The workspace depends on sizes, types, strides, the alignment of x, weight and dy, and on
 * which gradients are asked for (dx, dweight, dbias not NULL): the queries read all of these from the call's
 * own arguments. x, weight and dy that are NULL in a query count as off every alignment, which is enough for any. */
#define FX_ACT_NONE 0
#define FX_ACT_RELU 1
#define FX_ACT_SILU 2
#define FX_ACT_GELU 3      /* h (1 + erf(h / sqrt 2)) / 2 */
#define FX_ACT_GELU_TANH 4 /* h (1 + tanh(sqrt(2 / pi) (h + 0.044715 h^3))) / 2 */
#define FX_ACT_TANH 5

typedef struct {
  int32_t dtype, activation;
  int64_t rows, inner, outer;
  const void *x, *weight, *bias, *residual;
  int64_t x_stride, weight_stride, residual_stride;
  void *y, *slope;
  /* backward */
  const void* dy;
  int64_t dy_stride;
  void *dx, *dweight, *dbias;
} fx_linear_args;

int fermix_linear(void* stream, const fx_linear_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_linear_workspace_bytes(const fx_linear_args* args);
int fermix_linear_grad(void* stream, const fx_linear_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_linear_grad_workspace_bytes(const fx_linear_args* args);

/* ---- log probabilities of tokens ---------------------------------------------------------
 * logits and mask (rows, entries) by the element stride of a row (mask: bytes, 0 leaves the entry
 * out, stride 0: one for all rows; NULL: none). Per row: logp of its token, entropy (in nats),
 * and the `top` <= FX_TOP_MAX likeliest entries, ties to the lowest index, with -inf and index -1
 * behind the last entry of any probability. A row without such an entry has entropy 0 and
 * dlogits 0, whether the mask or logits of -inf leave none; a token
 * that is masked or whose logit is -inf has logp -inf. A live NaN or +inf makes the row's numbers
 * NaN and its indices -1. A token equal to `padding` (where has_padding) leaves its row out: logp
 * and entropy 0, top -inf and -1, dlogits 0, whatever the logits hold; any other token outside
 * [0, entries) has logp NaN and no gradient through it. 1e-30 <= scale <= 1e30. stats (2, rows): written where
 * not NULL, read by the backward with entropy: dlogits = scale (grad_logp (hit - p) -
 * grad_entropy p (log p + entropy)), 0 where masked; grad_logp and grad_entropy may be NULL. */
#define FX_TOP_MAX 32
#define FX_LOGPROBS_MAX (1 << 30) /* entries of a row */

typedef struct {
  int32_t dtype, token_bytes;
  int64_t rows, entries, padding;
  int32_t has_padding, top;
  float scale;
  int32_t reserved;
  const void *logits, *tokens;
  const uint8_t* mask;
  int64_t logits_stride, mask_stride;
  float *logp, *entropy, *top_logp;
  int64_t* top_index;
  float* stats;
  /* backward */
  const float *grad_logp, *grad_entropy;
  void* dlogits; /* (rows, entries), contiguous */
} fx_logprobs_args;

int fermix_token_logprobs(void* stream, const fx_logprobs_args* args, void* workspace, size_t workspace_bytes);
size_t fermix_token_logprobs_workspace_bytes(const fx_logprobs_args* args);
int fermix_token_logprobs_grad(void* stream, const fx_logprobs_args* args);

#ifdef __cplusplus
}
#endif
#endif
