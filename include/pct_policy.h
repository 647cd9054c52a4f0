/*
 * pct_policy.h -- C ABI of the policy operators that stand between an observation and a step (libpct_hip.so).
 *
 *   pct_choice_pick      one choice per row from masked logits (+ noise), its log-probability, the row's entropy
 *   pct_choice_log_probs log-probabilities of given choices, entropy, the best alternatives
 *   pct_choice_backward  the gradient of pct_choice_log_probs with respect to the logits
 *   pct_attend           attention of queries to the allowed keys of a batch
 *   pct_attend_backward  its gradients
 *
 * The conventions are those of pct_env.h: int status (PCT_OK == 0, text from pct_last_error()), `stream` is a hipStream_t,
 * work is only enqueued on it, every pointer is device memory on the current device that the caller owns; nothing is
 * allocated, kept or synchronised.  Strides count elements.  Sizes that are zero enqueue nothing.  Workspaces and statistics start
 * on 16 bytes.
 */
#ifndef PCT_POLICY_H
#define PCT_POLICY_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element types */
#define PCT_F32 0
#define PCT_BF16 1
#define PCT_F16 2
/* mask types: an entry allows its choice (key) where it is not zero */
#define PCT_MASK_NONE 0
#define PCT_MASK_U8 1  /* bool, uint8, int8 */
#define PCT_MASK_F16 2 /* 16-bit floats of either kind */
#define PCT_MASK_F32 3
#define PCT_MASK_I32 4

#define PCT_CHOICE_MAX_GIVEN 64
#define PCT_CHOICE_MAX_TOP 64

typedef struct pct_choice {
  int32_t struct_size;
  int32_t dtype;        /* of the logits */
  int32_t rows, choices;
  const void* logits;   /* [rows, choices], unit stride along the choices */
  int64_t logits_row;
  const void* mask;     /* [rows, choices] or NULL */
  int64_t mask_row, mask_col;
  int32_t mask_type;
  int32_t given_count;  /* 0 .. PCT_CHOICE_MAX_GIVEN */
  const int64_t* given; /* [rows, given_count], contiguous; -1: no choice */
  int32_t top;          /* 0 .. PCT_CHOICE_MAX_TOP */
  int32_t pad;
  const float* noise;   /* pick: [rows, choices] float32, unit stride, or NULL */
  int64_t noise_row;
  int64_t* actions;     /* pick: [rows] */
  float* log_probs;     /* pick: [rows]; otherwise [rows, given_count] */
  float* entropy;       /* [rows] */
  float* top_log_probs; /* [rows, top] */
  int64_t* top_actions; /* [rows, top] */
  float* stats;         /* [rows, 4] for pct_choice_backward, or NULL */
  void* workspace;      /* pct_choice_workspace() bytes */
  int64_t workspace_bytes;
} pct_choice;

typedef struct pct_choice_grad {
  int32_t struct_size;
  int32_t dtype;
  int32_t rows, choices;
  const void* logits;
  int64_t logits_row;
  const void* mask;
  int64_t mask_row, mask_col;
  int32_t mask_type;
  int32_t given_count;
  const int64_t* given;
  int32_t top;
  int32_t pad;
  const int64_t* top_actions;   /* as pct_choice_log_probs wrote them */
  const float* stats;           /* as pct_choice_log_probs wrote them */
  const float* d_log_probs;     /* [rows, given_count] contiguous, or NULL (zero) */
  const float* d_entropy;       /* [rows] or NULL */
  const float* d_top_log_probs; /* [rows, top] or NULL */
  void* d_logits;               /* [rows, choices] contiguous, dtype */
} pct_choice_grad;

/* bytes of workspace that the two forward calls need for these sizes (0: none) */
int64_t pct_choice_workspace(int32_t rows, int32_t choices, int32_t top);
int pct_choice_pick(const pct_choice* c, void* stream);
int pct_choice_log_probs(const pct_choice* c, void* stream);
int pct_choice_backward(const pct_choice_grad* c, void* stream);

typedef struct pct_attention {
  int32_t struct_size;
  int32_t dtype;
  int32_t batch, q_len, k_len, heads, kv_heads, dim; /* heads a multiple of kv_heads; dim a multiple of 8, 8 .. 128 */
  const void *q, *k, *v;                             /* [batch, length, heads, dim], unit stride along dim; rows start on 16 bytes */
  int64_t q_stride[3], k_stride[3], v_stride[3];     /* batch, length, head */
  const void* key_mask;                              /* [batch, k_len] or NULL; the backward only looks whether it is NULL */
  int64_t mask_row, mask_col;
  int32_t mask_type;
  int32_t lengths_type;    /* 4: int32, 8: int64 */
  const void* key_lengths; /* [batch] or NULL: key j is allowed where j < length */
  float scale;             /* positive */
  int32_t pad;
  void* out;               /* [batch, q_len, heads, dim] contiguous */
  float* stats;            /* [batch, kv_heads, q_len * heads / kv_heads, 2]: written by pct_attend (may be NULL there), read by the backward */
  int32_t* key_list;       /* [batch, k_len + 1] workspace: written by pct_attend with a key_mask, read by the backward; else NULL */
  void* workspace;         /* pct_attend_workspace() bytes */
  int64_t workspace_bytes;
  /* backward only */
  const void* d_out;       /* [batch, q_len, heads, dim], as q; `out` and `stats` are inputs then */
  int64_t d_out_stride[3];
  void *d_q, *d_k, *d_v;   /* contiguous, dtype */
} pct_attention;

/* bytes of workspace that pct_attend (backward == 0) or pct_attend_backward needs for the sizes in *a (0: none) */
int64_t pct_attend_workspace(const pct_attention* a, int32_t backward);
int pct_attend(const pct_attention* a, void* stream);
int pct_attend_backward(const pct_attention* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif
