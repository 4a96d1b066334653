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
  const int32_t* seg_class;    /* [segs] index into cls */
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
  CxAdamWClass cls[CX_ADAMW_CLASSES];
} CxAdamW;

uint32_t cx_adamw_noise(uint32_t number);
int cx_adamw_step(int dev, const CxAdamW* a, void* stream);

int64_t cx_ops_sizeof(int what); /* 0 CxAdamW */

#ifdef __cplusplus
}
#endif
