// C ABI of the operators of a training step that surround the exchange: the product with its epilogue, the loss over
// a vocabulary and the AdamW step over many tensors.  Same conventions as cx_common.h: plain structs, `dev` picks the
// back end, the return value is 0 or negative with the reason in cx_last_error().
#pragma once
#include "cx_common.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- AdamW over many tensors ------------------------------------------------------------------------------------ */
#define CX_ADAMW_BLOCK 256    /* elements that share a scale of the 8-bit states; tensors start on multiples of it */
#define CX_ADAMW_CLASSES 64   /* tensors with the same settings and the same step count */

typedef struct CxAdamWClass {
  float decay;          /* 1 - lr * weight decay */
  float b1, ob1;        /* beta1, 1 - beta1 */
  float b2, ob2;
  float rate;           /* lr / (1 - beta1^t) */
  float norm;           /* 1 / sqrt(1 - beta2^t) */
  float eps;
} CxAdamWClass;

typedef struct CxAdamW {
  const int32_t* blk_seg;      /* [blocks] tensor of every block of the flat states */
  const int64_t* seg_blk;      /* [segs] first block of a tensor */
  const int64_t* seg_len;      /* [segs] its elements */
  void* const* seg_param;      /* [segs] the tensors */
  const void* const* seg_grad; /* [segs] and their gradients, of the same type; NULL: the tensor is left as it is */
  const int32_t* seg_class;    /* [segs] row of settings; those of this call are first_class + index into cls */
  float* master;               /* flat 32-bit weights behind 16-bit tensors; NULL for tensors of 32 bits */
  void* m;                     /* flat first moments: float, or e4m3 with 8 bits */
  void* v;                     /* flat second moments: float, or with 8 bits e4m3 of their square roots */
  float* m_scale;              /* [blocks], 8 bits only */
  float* v_scale;
  int64_t blocks;
  int32_t segs;
  int32_t dtype;               /* CX_F32, CX_BF16, CX_F16 */
  int32_t bits;                /* 32 or 8 */
  uint32_t noise;              /* of this step: cx_adamw_noise(seed + step) */
  int32_t first_class;         /* tensors of other rows are left as they are: more rows are more calls */
  int32_t pad;
  CxAdamWClass cls[CX_ADAMW_CLASSES];
} CxAdamW;

uint32_t cx_adamw_noise(uint32_t number);
int cx_adamw_step(int dev, const CxAdamW* a, void* stream);

/* ---- y = act(x w^T + bias) + residual --------------------------------------------------------------------------- */
#define CX_ACT_NONE 0
#define CX_ACT_RELU 1
#define CX_ACT_GELU 2        /* u Phi(u) */
#define CX_ACT_GELU_TANH 3   /* its tanh form */
#define CX_ACT_SILU 4

/* Matrices are row-major with rows `ld*` elements apart (ldpre: 16-byte aligned rows are the fast case); y, dx, dw are
 * written without gaps.  All of one type. */
typedef struct CxLinear {
  int64_t rows, inner, outer;
  int64_t ldx, ldw, ldr, ldg, ldpre;
  const void* x;         /* [rows][inner] */
  const void* w;         /* [outer][inner] */
  const void* bias;      /* [outer] or NULL */
  const void* residual;  /* [rows][outer] or NULL */
  void* y;               /* forward: [rows][outer] */
  void* pre;             /* x w^T + bias: written by the forward call when not NULL, read by the backward call where the
                            activation needs it; [rows][outer], rows ldpre apart */
  const void* grad;      /* backward: of y */
  void* dx;              /* each may be NULL */
  void* dw;
  void* dbias;
  void* workspace;       /* cx_linear_workspace_bytes */
  int64_t ws_bytes;
  int32_t dtype, act;
} CxLinear;

int64_t cx_linear_workspace_bytes(int dev, const CxLinear* l, int backward);
int cx_linear_forward(int dev, const CxLinear* l, void* stream);
int cx_linear_backward(int dev, const CxLinear* l, void* stream);

/* ---- softmax cross entropy of h w^T over a vocabulary, without the logits ---------------------------------------- */
#define CX_REDUCE_NONE 0
#define CX_REDUCE_SUM 1
#define CX_REDUCE_MEAN 2     /* over the rows that are not ignored */

typedef struct CxVocabLoss {
  int64_t rows, vocab, dim;
  int64_t ldh, ldw;
  const void* h;           /* [rows][dim] */
  const void* w;           /* [vocab][dim] */
  const int64_t* targets;  /* [rows]; ignore_index: the row counts for nothing; any other value outside [0, vocab) makes
                              the row's loss and gradients NaN */
  int64_t ignore_index;
  float* loss;             /* [rows] for CX_REDUCE_NONE, else [1] */
  float* lse;              /* [rows] log sum exp of the logits: written by the forward call, read by the backward call */
  float* count;            /* [1] rows that are not ignored: likewise (CX_REDUCE_MEAN) */
  const float* grad;       /* backward: of the loss */
  int64_t grad_stride;     /* CX_REDUCE_NONE: from row to row (0 for a broadcast one) */
  void* dh;                /* [rows][dim], may be NULL */
  void* dw;                /* [vocab][dim], may be NULL */
  void* workspace;         /* cx_vocab_loss_workspace_bytes */
  int64_t ws_bytes;
  int32_t dtype, reduction;
} CxVocabLoss;

int64_t cx_vocab_loss_workspace_bytes(int dev, const CxVocabLoss* l, int backward);
int cx_vocab_loss_forward(int dev, const CxVocabLoss* l, void* stream);
int cx_vocab_loss_backward(int dev, const CxVocabLoss* l, void* stream);

int64_t cx_ops_sizeof(int what); /* 0 CxAdamW, 1 CxLinear, 2 CxVocabLoss */

#ifdef __cplusplus
}
#endif
