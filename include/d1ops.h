/* d1ops — operators of a policy update beside the fused MLP step (C ABI), gfx950.
 *
 *   d1_tokens_*   log probabilities of given tokens (actions) with the row's entropy, its most
 *                 probable alternatives, and the gradient of the logits
 *   d1_norm_*     layer norm, its backward pass and the reduction of the weight's and the bias's gradient
 *   d1_adamw_*    one AdamW step over many tensors, moments in 32 or 8 bits, clip by the global norm
 *   d1_policy_loss*   the clipped policy loss with value, entropy and reference-KL terms, and its gradients
 *   d1_scan_*     a gated linear recurrence over long sequences, forward and backward
 *   d1_muon_*     updates orthogonalised by Newton-Schulz products, and the momentum step made of them
 *
 * Conventions as in d1hip.h: device pointers unless said otherwise, asynchronous on `stream`
 * (0 = the null stream), 0 on success, a hipError_t code for launch failures or a negative D1_E_*
 * code for arguments rejected before any launch. The library allocates nothing and keeps no state:
 * scratch memory is the caller's (`work`, sized by the *_work_bytes function, contents free to
 * change between calls). Element types are D1_FP32, D1_BF16 and D1_FP16; rows are addressed by a
 * stride in elements, elements of a row are adjacent. No pointer needs more than its element's
 * alignment.
 */
#ifndef D1OPS_H
#define D1OPS_H
#include <stdint.h>

#include "d1hip.h"

#ifdef __cplusplus
extern "C" {
#endif

#define D1_FP32 0
#define D1_BF16 1
#define D1_FP16 2

#define D1_TOKENS_MAX_TOP 64
#define D1_TOKENS_MAX_VOCAB (1 << 24)
#define D1_NORM_MAX_WIDTH 16384
#define D1_SCAN_MAX_WIDTH (1 << 24)
#define D1_SCAN_MAX_STEPS (1 << 30)
#define D1_MUON_MAX_SIDE (1 << 17)
#define D1_MUON_MAX_STEPS 32
#define D1_ADAMW_BLOCK 256            /* elements of an 8-bit moment that share an exponent */

/* For row i of logits [rows, vocab] over its allowed entries (mask[i * mask_stride + j] != 0; all
 * when mask is null; mask_stride 0: one mask row for every row):
 *   logp[i]     x[t] - log sum_j exp x[j] for t = tokens[i]
 *   entropy[i]  -sum_j p[j] log p[j], an entry of probability 0 adding 0
 *   stats[2i], stats[2i+1]   the largest allowed entry (0 when there is none above -inf) and
 *               sum_j exp(x[j] - it), read again by d1_tokens_bwd
 *   top_ids, top_logp [rows, top]   the `top` most probable allowed entries in falling order, the
 *               lowest index first among equal ones, and their log probabilities (a NaN logit
 *               counts as the largest); -1 and -inf where a row has fewer
 * A negative token is padding: logp 0. A token of vocab or more gives NaN, a masked one -inf. A
 * row with nothing allowed, or with -inf alone, has logp -inf (padding: 0), entropy 0. A +inf or
 * NaN entry that is allowed makes logp, entropy and top_logp NaN; what stands in masked places is
 * not looked at. top is 0 (top_ids, top_logp unused) to min(vocab, 64). */
int64_t d1_tokens_work_bytes(int64_t rows, int vocab, int top);
int d1_tokens_fwd(const void *logits, int type, int64_t rows, int vocab, int64_t stride, const int64_t *tokens,
                  const uint8_t *mask, int64_t mask_stride, int top, float *logp, float *entropy, float *stats,
                  int64_t *top_ids, float *top_logp, void *work, int64_t work_bytes, void *stream);
/* dlogits [rows, vocab] (contiguous, the logits' type) from the gradients of logp and entropy
 * (either may be null: zero): dlogp (1[j = t] - p[j]) - dentropy p[j] (log p[j] + entropy). Masked
 * entries and rows without an allowed entry get 0, padding no dlogp part; a token of vocab or more
 * makes its row's allowed entries NaN when dlogp is given. dlogits must not overlap the logits: an
 * entry may be read again after its gradient was written (dlogits == logits is rejected). */
int d1_tokens_bwd(const void *logits, int type, int64_t rows, int vocab, int64_t stride, const int64_t *tokens,
                  const uint8_t *mask, int64_t mask_stride, const float *stats, const float *entropy,
                  const float *dlogp, const float *dentropy, void *dlogits, void *stream);

/* y = (x - mean) * rstd * w + b over each row of x [rows, width], rstd = 1/sqrt(var + eps) with the
 * biased variance. w and b [width] may be null (1 and 0); `wtype` is x's type or D1_FP32. y
 * [rows, width] is contiguous; mean and rstd [rows] fp32 are kept for the backward pass. */
int d1_norm_fwd(const void *x, int type, int64_t rows, int width, int64_t stride, const void *w, const void *b,
                int wtype, float eps, void *y, float *mean, float *rstd, void *stream);
/* dx [rows, width] (contiguous, x's type), dw and db [width] (wtype; either may be null, then it is
 * not made). The sums over rows are made in fp32 in a fixed order: the same inputs give the same
 * bits. `work` is only needed with dw or db. */
int64_t d1_norm_work_bytes(int64_t rows, int width, int type);
int d1_norm_bwd(const void *dy, int64_t dy_stride, const void *x, int type, int64_t rows, int width, int64_t stride,
                const void *w, int wtype, const float *mean, const float *rstd, void *dx, void *dw, void *db,
                void *work, int64_t work_bytes, void *stream);

/* One tensor of an AdamW step. With 8-bit moments m and v are bytes and m_exp, v_exp hold one byte
 * for each D1_ADAMW_BLOCK elements; with 32-bit moments they are fp32 and the exponents unused. */
typedef struct D1AdamWTensor {
    void *p;                  /* parameter, fp32 or bf16 */
    const void *g;            /* gradient, fp32 or bf16 */
    void *m, *v;
    uint8_t *m_exp, *v_exp;
    void *copy;               /* bf16 copy of the new parameter, or null */
    int64_t n;                /* elements */
    int64_t counter;          /* 8-bit: first counter of the tensor's rounding draws */
    double lr, weight_decay;
    int32_t lag;              /* steps that this tensor has missed (its step count is the shared one less this, 1 at least) */
    uint8_t ptype, gtype;     /* D1_FP32 or D1_BF16 */
    uint8_t pad[2];
} D1AdamWTensor;

typedef struct D1AdamW {
    double beta1, beta2, eps;
    double max_norm;          /* clip by the global norm of all gradients; 0: no clip and no check */
    uint64_t seed;            /* of the 8-bit moments' rounding */
    int32_t bits;             /* 32 or 8 */
    int32_t pad;
} D1AdamW;

/* ctl: int32 [8] on the device, zero before the first step: [0] steps made, [1] steps skipped,
 * [5] the last global norm (fp32 bits); the rest is the step's own. `t` and `h` are host arrays,
 * read before the call returns.
 *   g' = g * min(1, max_norm / (norm + 1e-6));  m = beta1 m + (1 - beta1) g';
 *   v = beta2 v + (1 - beta2) g'^2;
 *   p = p (1 - lr wd) - lr/(1 - beta1^t) * m / (sqrt(v)/sqrt(1 - beta2^t) + eps)
 * With max_norm > 0 a norm that is not finite changes nothing but ctl[1]. The step count and the
 * norm stay on the device, so a captured graph of this call makes a new step on each replay.
 * 8-bit moments: x = +-(code) 2^exp with 3 bits of mantissa, 4 bits of exponent and a sign for m, 5
 * bits of exponent for v; the parameter's step is made from the moments before they are rounded;
 * rounding goes up or down by chance, a hash of (seed, step, counter + element) against the part
 * that is dropped, so that its expectation is the value; a v that is not 0 never becomes 0. An element
 * whose m or v is not finite after the step (a gradient that is not, or whose square overflows, with
 * max_norm 0) leaves the others of its block as they are and gets finite moments: m 0 and its block's
 * largest v where they were infinite, codes of its block's largest where they were NaN; with 32-bit moments it keeps what is not finite. The parameter is what the formula gives either way (v
 * past 2^104 counts as infinite for the 8-bit step: the parameter only decays). */
int64_t d1_adamw_work_bytes(const D1AdamWTensor *t, int count, const D1AdamW *h);
int d1_adamw_step(const D1AdamWTensor *t, int count, const D1AdamW *h, int32_t *ctl, void *work, int64_t work_bytes,
                  void *stream);
/* The same, made or skipped together with another step that has decided but changed nothing yet: `other` is the ctl of a
 * d1_muon_step with part 1 before this call on the stream. Where that one is skipped so is this; where this one's norm is not finite
 * (max_norm > 0) that one's decision is taken back, and its part 2 changes nothing. */
int d1_adamw_step_with(const D1AdamWTensor *t, int count, const D1AdamW *h, int32_t *ctl, int32_t *other, void *work,
                       int64_t work_bytes, void *stream);
/* out[i] (fp32) = the value that an 8-bit moment's code stands for; is_signed 1 for m, 0 for v. */
int d1_adamw_read(const uint8_t *code, const uint8_t *exp, int64_t n, int is_signed, float *out, void *stream);

/* An input of the policy loss: element t of sequence r is at data[r * row + t * step], strides in elements, none
 * negative; data null: not given. */
typedef struct D1LossInput {
    const void *data;
    int64_t row, step;
    int32_t type;             /* D1_FP32, D1_BF16 or D1_FP16; not read for the mask, whose elements are bytes */
    int32_t pad;
} D1LossInput;

typedef struct D1PolicyLoss {
    D1LossInput logp, old_logp, advantages;
    D1LossInput ref_logp, entropy, values, returns, old_values, mask;      /* each may be null; values need returns */
    int64_t rows, length;     /* `rows` sequences of `length` tokens */
    double clip_low, clip_high;          /* 0 <= clip_low <= 1, clip_high >= 0 */
    double value_clip;        /* 0: none, else it needs old_values */
    double kl_coef, value_coef, entropy_coef;
    int32_t sequence;         /* 0: every token counts alike; 1: every sequence with a token does, its tokens sharing its weight */
    int32_t fp32_grads;       /* 0: gradients in the type of their input, 1: all in fp32 */
} D1PolicyLoss;

/* With d = logp - old_logp, r = e^d, x = ref_logp - logp and w a token's weight (0 where mask is 0, whatever the other
 * inputs hold there; 1/tokens, or 1/(tokens of its sequence * sequences with a token)):
 *   terms[0] loss = policy + value_coef * value - entropy_coef * entropy + kl_coef * kl
 *   terms[1] policy = -sum w min(r A, min(max(r, 1 - clip_low), 1 + clip_high) A)
 *   terms[2] value = sum w max((v - R)^2, (v' - R)^2) / 2, v' = v held within value_clip of old_values
 *   terms[3] entropy = sum w entropy;  terms[4] kl = sum w (e^x - x - 1)
 *   terms[5] clipped = sum of the weights of tokens whose clip is active;  terms[6] drift = sum w (e^d - d - 1)
 *   terms[7] the tokens, or the sequences with one
 * A term whose input is not given is 0, all are where no token is left. dlogp, dentropy and dvalues (each may be null,
 * then it is not made; contiguous [rows, length], the type of their input, or fp32 with fp32_grads) are the gradients of
 * the loss. They must not overlap the inputs. The same inputs give the same bits. */
int64_t d1_policy_loss_work_bytes(const D1PolicyLoss *h);
int d1_policy_loss(const D1PolicyLoss *h, float *terms, void *dlogp, void *dentropy, void *dvalues, void *work,
                   int64_t work_bytes, void *stream);
/* out[0..n) = data[0..n) * *by (D1_FP32, D1_BF16 or D1_FP16); out may be data. */
int d1_scale(const void *data, void *out, int type, int64_t n, const float *by, void *stream);
/* The same of fp32 data, rounded to `type` once, after the product; out must not overlap data unless type is D1_FP32. */
int d1_scale_to(const float *data, void *out, int type, int64_t n, const float *by, void *stream);

/* h[t] = (1 - z[t]) m[t] h[t-1] + z[t] x[t] with z = sigmoid(gate), for `rows` sequences of `steps` steps of `width`
 * channels; m[t] is 0 where reset[t * reset_t + row * reset_n] is not (what was before is dropped, whatever it holds),
 * else 1. Element (t, row, c) of x is x[t * x_t + row * x_n + c], likewise the others; strides in elements. All of a
 * call's sequences are of one type; states are fp32 [rows, width], contiguous, and everything is computed in fp32. */
typedef struct D1Scan {
    const void *x, *gate;
    const uint8_t *reset;     /* or null: none */
    const float *state;       /* before the first step, or null: zeros */
    float *marks;             /* fp32 [d1_scan_marks(h), rows, width]: written by d1_scan_fwd where it is not null, read by
                                 d1_scan_bwd, which needs it where d1_scan_marks is not 0 */
    int64_t x_t, x_n, gate_t, gate_n, reset_t, reset_n;
    int64_t steps, rows;
    int32_t width, type;
} D1Scan;

int64_t d1_scan_marks(const D1Scan *h);             /* by steps, rows and width */
int64_t d1_scan_work_bytes(const D1Scan *h);       /* of either call */
/* out (x's type) and, where it is not null, last [rows, width] = the state after the last step. With no steps nothing
 * is written. Outputs must not overlap inputs. */
int d1_scan_fwd(const D1Scan *h, void *out, int64_t out_t, int64_t out_n, float *last, void *work, int64_t work_bytes, void *stream);
/* The gradients of x, gate and (where dstate is not null) the state from those of the outputs; dlast may be null (zero). */
int d1_scan_bwd(const D1Scan *h, const void *dh, int64_t dh_t, int64_t dh_n, const float *dlast, void *dx, int64_t dx_t,
                int64_t dx_n, void *dgate, int64_t dgate_t, int64_t dgate_n, float *dstate, void *work, int64_t work_bytes,
                void *stream);

/* One matrix [rows, cols], contiguous. With `momentum` (fp32) it is a parameter's step, else out = O(g). */
typedef struct D1MuonTensor {
    const void *g;            /* gradient, or the matrix that is orthogonalised */
    float *momentum;
    void *out;                /* the parameter (D1_FP32 or D1_BF16), or the result (any type) */
    void *copy;               /* of a step: bf16 copy of the new parameter, or null */
    int64_t rows, cols;
    double lr, scale, weight_decay;
    int32_t type, gtype;      /* of out and of g; of a step D1_FP32 or D1_BF16 */
} D1MuonTensor;

typedef struct D1Muon {
    double a, b, c;           /* of the quintic a s + b s^3 + c s^5 */
    double eps, momentum;
    int32_t steps, nesterov;
    int32_t terms;            /* operands of the products: 1: fp16, 3: two fp16 halves (22 bits), 0: 3 for fp32 results
                                 and matrices with a side under 16, 1 for others */
    int32_t part;             /* 0: the whole step; 1: its norms and whether it is made, in ctl; 2: the rest of it */
} D1Muon;

/* 0 where the coefficients can be used: `steps` times the quintic, from singular values in [0, 1], stays under 3.8 and its
 * factor a + b s^2 + c s^4 under 15, the range of what the products hold; else D1_E_ARG. */
int d1_muon_check(const D1Muon *h);
/* O(U): X = U / (|U|_F + eps), then `steps` times X = a X + (b A + c A A) X with A = X X^T (on the smaller side).
 * Of a step: m = momentum m + g;  U = nesterov ? g + momentum m : m;  p = p (1 - lr weight_decay) - lr scale O(U).
 * ctl as in d1_adamw_step, [0] steps made, [1] steps skipped, or null: with it a step with a U whose norm is not finite
 * changes nothing but ctl[1]. Parts 1 and 2 need ctl, and part 2 the `work` that part 1 left, with the same arguments otherwise and
 * nothing that they name changed between. `t` and `h` are host arrays, read before the call returns. Matrices with no elements are left
 * out. Results must not overlap each other or gradients. The same inputs give the same bits. */
int64_t d1_muon_work_bytes(const D1MuonTensor *t, int count, const D1Muon *h);
int d1_muon_step(const D1MuonTensor *t, int count, const D1Muon *h, int32_t *ctl, void *work, int64_t work_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif
