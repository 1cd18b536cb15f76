/*
 * Operators of mixture-of-experts layers on packed weights (libtgm_mi355x.so): the choice of each
 * token's experts and the experts' feed-forward products.
 *
 * The reference has no model code; these are what a serving loop around its packed matmul
 * (alexandreteles/tinygrad-dx12 src/tinygrad_dx12/codegen/decomp/dx12.py:108-112) needs for layers
 * whose feed-forward block is one of many.
 *
 * Every function returns TGM_OK or a negative tgm_status (message in tgm_last_error()); none allocates
 * memory or issues a memset.
 */
#ifndef TGM_EXPERTS_H
#define TGM_EXPERTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum tgm_route_score { TGM_ROUTE_SOFTMAX = 0, TGM_ROUTE_SIGMOID = 1 };

/* The top_k experts of every token from its router logits [tokens, experts] (F32, F16 or BF16, row
 * stride ld), at most 1024 experts.
 *
 *   p    = softmax(logits) or sigmoid(logits)
 *   key  = p + bias (bias: float32 [experts] or NULL)
 *   groups > 1: expert e is in group e / (experts / groups); a group counts by the sum of its two
 *          largest keys (its only one in groups of one), and all but top_groups groups are left out
 *   ids[t, j]     the expert of the j-th largest key (of the j-th largest logit without a bias)
 *   weights[t, j] = scale p, divided by the chosen ones' sum with renormalize
 *
 * Equal keys rank by index, groups too.  The choice is that of keys in 64 bits.  A NaN key ranks behind
 * every other and counts as -infinity in its group's sum; a row with a NaN among its logits, or with
 * +infinity under a softmax, has NaN weights, and under a softmax its keys are NaN.  Renormalised weights
 * are those of the chosen logits however far below the row's largest, or 0, they lie; chosen logits of
 * -infinity alone have the weights 0.  ids int32 and weights float32 are [tokens, top_k]. */
int tgm_route(const void* logits, int64_t dtype, int64_t tokens, int64_t experts, int64_t ld, const float* bias,
              int64_t score, int64_t groups, int64_t top_groups, int64_t top_k, int64_t renormalize, double scale,
              int32_t* ids, float* weights, void* stream);

/* The packed weights of a layer's experts: gate_up [experts, 2 ffn, hidden] with gate (2 i) and up
 * (2 i + 1) rows in turn, down [experts, hidden, ffn], each a bit stream of codes (enum tgm_format) and
 * 16-byte aligned.  FP4 / FP6: scales E8M0 per 32 values of a row, or none, activations BF16.  INT4 /
 * UINT4: scales F16, BF16 or F32 per 32, 64 or 128, or none, activations F16.  hidden and ffn are
 * multiples of 128; scales are 4-byte aligned. */
typedef struct tgm_experts {
  const void* gate_up;
  const void* gate_up_scales; /* NULL: none */
  const void* down;
  const void* down_scales;
  int64_t experts;
  int64_t hidden;
  int64_t ffn;
  int64_t format;
  int64_t scale_dtype; /* TGM_NONE without scales */
  int64_t block_size;
} tgm_experts;

/* y[t] = sum_j weights[t, j] down_e . (silu(gate_e . x[t]) * (up_e . x[t])),  e = ids[t, j]
 *
 * x [tokens, hidden] (row stride ldx, a multiple of 8; 16-byte aligned), ids and weights [tokens, top_k]
 * contiguous, y [tokens, hidden] (row stride ldy) of x's type or F32; y may be x and shares no memory
 * with weights.  An id outside [0, experts) names no expert and adds nothing; the same expert may be
 * named twice.  Products and sums over K, experts and tokens are float32; silu(gate) * up is rounded to
 * x's type on its way into the down product.  Repeated calls agree to the bit.  A token's result depends
 * on the other tokens of the call in the rounding of sums alone, whose order goes by the call's sizes
 * and, for up to 16 tokens, by the experts that they name.  tokens times top_k must be less than 2^24, x
 * less than 2 GiB and the weight of an expert less than 4 GiB.
 * workspace: tgm_experts_workspace() bytes, 16-byte aligned. */
int64_t tgm_experts_workspace(const tgm_experts* experts, int64_t tokens, int64_t top_k);
int tgm_experts_apply(const tgm_experts* experts, const void* x, int64_t x_dtype, int64_t tokens, int64_t ldx,
                      const int32_t* ids, const float* weights, int64_t top_k, void* y, int64_t y_dtype, int64_t ldy,
                      void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TGM_EXPERTS_H */
