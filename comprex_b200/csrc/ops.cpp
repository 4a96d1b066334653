// Entry points of the operators of cx_ops.h: checks of the descriptors, then the back end that `dev` names.
#include "cx_adamw.h"
#include "cx_ops.h"

int cx_set_error(const char* where, int cuda_err);
int cx_adamw_step_cuda(const CxAdamW*, void*);
int cx_adamw_step_host(const CxAdamW*);

namespace {
bool type_ok(int dtype) { return dtype == CX_F32 || dtype == CX_BF16 || dtype == CX_F16; }
}  // namespace

extern "C" {

uint32_t cx_adamw_noise(uint32_t number) { return cxadam::mix(number); }

int cx_adamw_step(int dev, const CxAdamW* a, void* stream) {
  if (!a || !type_ok(a->dtype)) return cx_set_error("cx_adamw_step: bad element type", 0);
  if (a->bits != 8 && a->bits != 32) return cx_set_error("cx_adamw_step: states have 8 or 32 bits", 0);
  if (a->blocks < 0 || a->segs < 0) return cx_set_error("cx_adamw_step: negative size", 0);
  if (a->blocks == 0) return 0;
  if (!a->blk_seg || !a->seg_blk || !a->seg_len || !a->seg_param || !a->seg_grad || !a->seg_class || !a->m || !a->v ||
      (a->bits == 8 && (!a->m_scale || !a->v_scale)) || (a->dtype != CX_F32 && !a->master))
    return cx_set_error("cx_adamw_step: a table or state is missing", 0);
  return dev == CX_DEV_CUDA ? cx_adamw_step_cuda(a, stream) : cx_adamw_step_host(a);
}

int64_t cx_ops_sizeof(int what) {
  switch (what) {
    case 0: return (int64_t)sizeof(CxAdamW);
    default: return -1;
  }
}

}  // extern "C"
