/*
 * minispeed_ops.h — C ABI of the language-model operators around the boundary
 * step on MI355X (gfx950): the token embedding and its gradient, log
 * probabilities of given tokens and their gradient, and activations held in
 * 8 bits between forward and backward.
 *
 * Conventions (as minispeed_boundary.h)
 *   - Every pointer is caller-owned device memory [dev]; scalars are read
 *     during the call.  Element types are MS_OPS_F32 / F16 / BF16.
 *   - Every entry point is asynchronous on `stream` (a hipStream_t passed as
 *     void*; NULL is the legacy default stream) and allocates nothing.
 *     Scratch memory is the caller's `workspace`, at least as large as the
 *     matching *_workspace() says, 16-byte aligned, its contents free.
 *   - Return value: 0, a negative MS_OPS_E* code for an argument error found
 *     on the host (nothing was launched), or a positive hipError_t from the
 *     launch.  ms_ops_error_string() names both kinds.
 *   - The same call gives the same bits: no floating-point atomics, every sum
 *     in a fixed order.  (That of a row of logits follows from the row's
 *     address modulo 16, and of its gradient's where lse is beyond +-256; nothing
 *     else depends on addresses.)
 *   - Row-strided operands are given as (inner, outer_stride, inner_stride):
 *     row r starts at (r / inner) * outer_stride + (r % inner) * inner_stride
 *     elements; elements of a row are consecutive.  Token lists are the same
 *     with one element per row.  A plain list has inner = its length.
 *     Lists, rows and vocabularies hold fewer than 2^31 entries; offsets are
 *     64-bit.  A launch has fewer than 2^32 threads: a call that would take
 *     more (some 2^35 values) is refused with MS_OPS_EINVAL.
 */
#ifndef MINISPEED_OPS_H
#define MINISPEED_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MS_OPS_ABI_VERSION 1

enum { MS_OPS_F32 = 0, MS_OPS_F16 = 1, MS_OPS_BF16 = 2 };

enum {
  MS_OPS_OK = 0,
  MS_OPS_EINVAL = -1,     /* bad size, stride, type or NULL where required */
  MS_OPS_EWORKSPACE = -2  /* workspace smaller than needed or misaligned   */
};

/* values that share one scale of the 8-bit form */
#define MS_OPS_BLOCK 32
/* most alternatives per row of ms_logprobs */
#define MS_OPS_MAX_TOP 64

enum {
  MS_ACT_GELU = 0,        /* x Phi(x)                                     */
  MS_ACT_GELU_TANH = 1,   /* x / (1 + exp(-2 sqrt(2/pi) (x + .044715 x^3))) */
  MS_ACT_SILU = 2,        /* x / (1 + exp(-x))                            */
  MS_ACT_SWIGLU = 3       /* silu(x) * up                                 */
};

/* A list of n token numbers, 4 or 8 bytes each (`wide`). */
typedef struct ms_tokens {
  const void* data;
  int64_t n;
  int64_t inner;
  int64_t outer_stride;
  int64_t inner_stride;
  int32_t wide;
  int32_t reserved;
} ms_tokens_t;

/* `n` rows of `width` consecutive elements. */
typedef struct ms_rows {
  const void* data;
  int64_t n;
  int64_t width;
  int64_t inner;
  int64_t outer_stride;
  int64_t inner_stride;
  int32_t dtype;
  int32_t reserved;
} ms_rows_t;

int ms_ops_abi_version(void);
const char* ms_ops_error_string(int code);

/*
 * Embedding lookup: out[t, :] = scale * table[id_t, :], computed in fp32 and
 * rounded once to the table's type.  `table->n` rows at one stride (inner >= n);
 * out is dense
 * [ids->n, width].  An id outside [0, table->n) gives a row of NaN.
 */
int ms_embedding(const ms_tokens_t* ids, const ms_rows_t* table, float scale,
                 void* out, void* stream);

/*
 * Its gradient: dtable[v, :] = scale * sum over the tokens t with id_t = v, in
 * increasing t, of grad[t, :]; dtable is dense [vocab, width] of the
 * gradient's type and written whole (rows without tokens are zeros).  Sums
 * are fp32 in an order that follows from the ids, the sizes and the type, and
 * is the same for every column; they are multiplied by scale and rounded once.  Ids outside [0, vocab) and `padding_idx` (-1: none) add
 * nothing.  dtable is 16-byte aligned; at most 2^30 tokens.
 */
int64_t ms_embedding_grad_workspace(int64_t n, int64_t vocab, int64_t width);
int ms_embedding_grad(const ms_tokens_t* ids, const ms_rows_t* grad, int64_t vocab,
                      float scale, int64_t padding_idx, void* dtable,
                      void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Log probabilities.  Per row x of logits, with p = softmax(x):
 *   lse      = log sum exp x
 *   logprob  = x[target] - lse           (0 where target == ignore_index)
 *   entropy  = -sum p log p              (NULL: not computed)
 *   top      the `top` largest p in falling order, equal ones by rising
 *            index: top_logprob fp32, top_id int64, both [n, top]
 * All outputs fp32 and dense.  A row of -inf has lse = -inf, logprob and
 * top_logprob -inf, entropy 0.  A row that holds NaN or +inf has NaN in lse,
 * logprob, entropy and top_logprob (top_id then orders NaN above +inf).  A
 * target outside [0, vocab) that is not ignore_index gives NaN.
 */
int64_t ms_logprobs_workspace(int64_t n, int64_t vocab, int32_t dtype, int32_t top);
int ms_logprobs(const ms_rows_t* logits, const ms_tokens_t* targets, int64_t ignore_index,
                int32_t top, float* logprob, float* entropy, float* lse,
                float* top_logprob, int64_t* top_id, void* workspace,
                int64_t workspace_bytes, void* stream);

/*
 * Gradient of the logits, dense [n, vocab] of the logits' type:
 *   dlogits[j] = g (1[j = target] - p_j) - h p_j (log p_j + entropy)
 * with g = grad_logprob of the row (0 where target == ignore_index, and where
 * NULL) and h = grad_entropy (NULL: 0; then `entropy` is not read).  lse and entropy are
 * those that ms_logprobs gave.  Rows of -inf get zeros, a NaN logit NaN
 * whatever lse is; a target outside
 * [0, vocab) that is not ignore_index makes g NaN.  A row whose lse is beyond
 * +-256 costs another pass over its logits: its maximum and sum are found again,
 * as an fp32 lse no longer tells them from each other.
 */
int ms_logprobs_grad(const ms_rows_t* logits, const ms_tokens_t* targets, int64_t ignore_index,
                     const float* lse, const float* entropy, const float* grad_logprob,
                     const float* grad_entropy, void* dlogits, void* stream);

/*
 * The 8-bit form of n values: blocks of MS_OPS_BLOCK consecutive values (the
 * last may be short) share the scale 2^(e - 127), e in [1, 254] the smallest
 * for which every |value| rounds to at most 127 steps; code = value / scale
 * rounded to nearest even.  The error is at most half a step, below 1/127 of
 * the block's largest magnitude (values below 2^-126 aside).  A block that
 * holds an inf or NaN has e = 255 and stands for NaN throughout.
 * codes: n int8; exponents: ceil(n / MS_OPS_BLOCK) uint8.
 */
int ms_pack8(const void* x, int32_t dtype, int64_t n, int8_t* codes, uint8_t* exponents,
             void* stream);
int ms_unpack8(const int8_t* codes, const uint8_t* exponents, int64_t n, int32_t dtype,
               void* out, void* stream);

/*
 * An activation function that leaves the 8-bit form of its input.
 *   a = f(h), or f(h) * up for MS_ACT_SWIGLU; dense [h->n, h->width].
 * codes / exponents hold h, up_codes / up_exponents hold up, as ms_pack8 of
 * the dense [n * width] values.  `up` and its two outputs are NULL unless
 * kind is MS_ACT_SWIGLU.
 */
int ms_act8(const ms_rows_t* h, const ms_rows_t* up, int32_t kind, void* a,
            int8_t* codes, uint8_t* exponents, int8_t* up_codes, uint8_t* up_exponents,
            void* stream);

/*
 * Its backward pass from the 8-bit form, n dense values:
 *   dh = grad * f'(h^) (* up^),  dup = grad * f(h^),  a = f(h^) (* up^)
 * with h^, up^ the values that the codes stand for.  `a`, the activation
 * again for the weight gradient of the product behind it, may be NULL.
 */
int ms_act8_grad(const int8_t* codes, const uint8_t* exponents, const int8_t* up_codes,
                 const uint8_t* up_exponents, const void* grad, int32_t dtype, int32_t kind,
                 int64_t n, void* dh, void* dup, void* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
