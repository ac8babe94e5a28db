/*
 * b200policy — C ABI of the learned-policy operators that run beside the
 * batched physics step: the memory, the normalisation and the gradient
 * clipping of a policy that reads the worlds' observation slab and writes
 * their actions, on the device that steps them.
 *
 * Conventions (those of b200phys.h):
 *   - all device buffers are caller-owned; launches allocate nothing and are
 *     graph-capturable; argument structs are read before a launch returns;
 *   - launch functions return a cudaError_t value (0 == success) and
 *     cudaErrorInvalidValue (1) for rejected arguments;
 *   - every *_bytes() export is checked by the host against its own layout;
 *   - strides are in elements; the innermost dimension is contiguous;
 *   - pointers are aligned to their elements, those marked so to more; what is
 *     not marked "or NULL" has to be there unless it holds no element.
 */
#ifndef B200POLICY_H
#define B200POLICY_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Element types. */
#define B200_FP32 0
#define B200_FP16 1
#define B200_BF16 2

/* Widest head of decay attention. */
#define B200_HEAD_MAX 128

/* Decay attention.  Per world b and head h, with lambda = exp(log_decay[h]):
 *   S_t = lambda * (first[b, t] ? 0 : S_{t-1}) + k_t v_t^T      t < lengths[b]
 *   o_t = scale * q_t S_t
 * S is [dk, dv] and starts at `state` (NULL: zero).  Tokens at or past
 * lengths[b] leave S alone, and their output rows (and gradients) are zero;
 * their q, k, v are never used.  Query head h reads key / value head
 * h / (heads / kv_heads). */
typedef struct B200AttentionArgs {
  const void *q;           /* [batch, time, heads, dk] */
  const void *k;           /* [batch, time, kv_heads, dk] */
  const void *v;           /* [batch, time, kv_heads, dv] */
  const float *log_decay;  /* [heads] */
  const float *state;      /* [batch, heads, dk, dv] or NULL */
  const uint8_t *first;    /* [batch, time] or NULL: no token starts an episode */
  const int32_t *lengths;  /* [batch] or NULL: every row holds `time` tokens */
  void *out;               /* [batch, time, heads, dv], dense (forward) */
  float *state_out;        /* [batch, heads, dk, dv], dense (forward); may alias state */
  const void *dout;        /* [batch, time, heads, dv] (backward) */
  const float *dstate_out; /* [batch, heads, dk, dv] or NULL: zero (backward) */
  void *dq;                /* like q, dense (backward) */
  void *dk_out;            /* like k, dense (backward) */
  void *dv_out;            /* like v, dense (backward) */
  float *dstate;           /* [batch, heads, dk, dv] or NULL: not wanted (backward) */
  void *workspace;         /* b200policy_attention_workspace() bytes, 16-byte aligned */
  int32_t *status;         /* not zero once a bounded wait of a launch has run out: that launch's outputs are void,
                            * others are not, but a captured one's replays are until it is set to zero.  NULL: only
                            * kernels without such waits run (long rows of wide bf16 heads take longer) */
  int64_t q_batch, q_time, q_head;
  int64_t k_batch, k_time, k_head;
  int64_t v_batch, v_time, v_head;
  int64_t g_batch, g_time, g_head; /* dout */
  int64_t first_batch, first_time;
  int32_t batch, time, heads, kv_heads, dk, dv;
  int32_t dtype; /* of q, k, v, out, dout, dq, dk_out, dv_out */
  float scale;
} B200AttentionArgs;

/* Layer norm over rows of `width` elements:
 *   y = (x - mean) * rstd * weight + bias,  rstd = 1 / sqrt(var + eps). */
typedef struct B200NormArgs {
  const void *x;      /* [rows, width], row stride x_row */
  const void *weight; /* [width] or NULL: one */
  const void *bias;   /* [width] or NULL: zero */
  void *y;            /* [rows, width], dense (forward) */
  float *stats;       /* [rows, 2]: mean, rstd, 8-byte aligned (forward writes, backward reads; forward: NULL if not
                       * wanted) */
  const void *dy;     /* [rows, width], row stride dy_row (backward) */
  void *dx;           /* [rows, width], dense, or NULL (backward) */
  void *dweight;      /* [width], weight's type, or NULL (backward) */
  void *dbias;        /* [width], weight's type, or NULL (backward) */
  void *workspace;    /* b200policy_norm_workspace() bytes, 16-byte aligned (backward) */
  int64_t rows, x_row, dy_row;
  int32_t width;
  int32_t dtype;        /* of x, y, dy, dx */
  int32_t weight_dtype; /* of weight, bias, dweight, dbias: dtype or fp32 */
  float eps;
} B200NormArgs;

/* One tensor of the global norm: dst receives src scaled (dst may be src). */
typedef struct B200ClipTensor {
  const void *src;
  void *dst;
  int64_t count;
  int64_t dtype;
} B200ClipTensor;

const char *b200policy_source_id(void);
int b200policy_arch(void);
size_t b200policy_attention_bytes(void); /* sizeof(B200AttentionArgs) */
size_t b200policy_norm_bytes(void);      /* sizeof(B200NormArgs) */
size_t b200policy_clip_bytes(void);      /* sizeof(B200ClipTensor) */

/* Device workspace of a forward (backward == 0) or backward launch, in bytes. */
size_t b200policy_attention_workspace(const B200AttentionArgs *a, int backward);
int b200policy_attention_forward(const B200AttentionArgs *a, void *stream);
int b200policy_attention_backward(const B200AttentionArgs *a, void *stream);

/* Device workspace of a backward launch, in bytes. */
size_t b200policy_norm_workspace(const B200NormArgs *a);
int b200policy_norm_forward(const B200NormArgs *a, void *stream);
int b200policy_norm_backward(const B200NormArgs *a, void *stream);

/* norm[0] = sqrt(sum over all tensors of |src|^2); every dst = src *
 * min(1, max_norm / (norm[0] + eps)).  `tensors` is a host array; memory that
 * is written through one entry may not be read or written through another, and
 * within an entry only dst == src may overlap (rejected otherwise). */
size_t b200policy_clip_workspace(const B200ClipTensor *tensors, int count);
int b200policy_clip(const B200ClipTensor *tensors, int count, float max_norm, float eps, float *norm,
                    void *workspace, void *stream);

#ifdef __cplusplus
}
#endif
#endif
