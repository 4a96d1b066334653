// Entry points of the operators of cx_ops.h: checks of the descriptors, then the back end that `dev` names.
#include <exception>

#include "cx_adamw.h"
#include "cx_ops.h"

int cx_set_error(const char* where, int cuda_err);
void cx_note_stream(const void* stream, bool early);
int cx_adamw_step_cuda(const CxAdamW*, void*);
int cx_adamw_step_host(const CxAdamW*);
int64_t cx_linear_workspace_bytes_cuda(const CxLinear*, int);
int cx_linear_forward_cuda(const CxLinear*, void*);
int cx_linear_backward_cuda(const CxLinear*, void*);
int cx_linear_forward_host(const CxLinear*);
int cx_linear_backward_host(const CxLinear*);
int64_t cx_vocab_loss_workspace_bytes_cuda(const CxVocabLoss*, int);
int cx_vocab_loss_forward_cuda(const CxVocabLoss*, void*);
int cx_vocab_loss_backward_cuda(const CxVocabLoss*, void*);
int cx_vocab_loss_forward_host(const CxVocabLoss*);
int cx_vocab_loss_backward_host(const CxVocabLoss*);

namespace {

bool type_ok(int dtype) { return dtype == CX_F32 || dtype == CX_BF16 || dtype == CX_F16; }
// No exception leaves a C entry: the host back end allocates.
template <typename F, typename D>
int on_host(F f, const D* d) {
  try {
    return f(d);
  } catch (const std::exception& e) {
    return cx_set_error(e.what(), 0);
  }
}

// The products' kernels let the kernel behind them in at their start: a receive kernel that comes next waits first.
void* noted(void* stream) {
  cx_note_stream(stream, true);
  return stream;
}

constexpr int64_t kMost = 0x7FFFFF00;      // rows, columns and entries of the vocabulary: 32-bit coordinates
bool size_ok(int64_t n) { return n >= 1 && n <= kMost; }

const char* wrong(const CxLinear* l) {
  if (!l || !type_ok(l->dtype)) return "cx_linear: bad element type";
  if (!size_ok(l->rows) || !size_ok(l->inner) || !size_ok(l->outer)) return "cx_linear: a size is zero, negative or too large";
  if (l->act < CX_ACT_NONE || l->act > CX_ACT_SILU) return "cx_linear: unknown activation";
  return nullptr;
}
const char* wrong(const CxVocabLoss* l) {
  if (!l || !type_ok(l->dtype)) return "cx_vocab_loss: bad element type";
  if (!size_ok(l->rows) || !size_ok(l->vocab) || !size_ok(l->dim)) return "cx_vocab_loss: a size is zero, negative or too large";
  if (l->reduction < CX_REDUCE_NONE || l->reduction > CX_REDUCE_MEAN) return "cx_vocab_loss: unknown reduction";
  if (l->ldh < l->dim || l->ldw < l->dim) return "cx_vocab_loss: rows overlap";
  if (!l->h || !l->w || !l->targets || !l->lse || !l->count) return "cx_vocab_loss: an operand is missing";
  return nullptr;
}

}  // namespace

extern "C" {

uint32_t cx_adamw_noise(uint32_t number) { return cxadam::mix(number); }

int cx_adamw_step(int dev, const CxAdamW* a, void* stream) {
  if (!a || !type_ok(a->dtype)) return cx_set_error("cx_adamw_step: bad element type", 0);
  if (a->bits != 8 && a->bits != 32) return cx_set_error("cx_adamw_step: states have 8 or 32 bits", 0);
  if (a->blocks < 0 || a->segs < 0 || a->first_class < 0) return cx_set_error("cx_adamw_step: negative size", 0);
  if (a->blocks == 0) return 0;
  if (!a->blk_seg || !a->seg_blk || !a->seg_len || !a->seg_param || !a->seg_grad || !a->seg_class || !a->m || !a->v ||
      (a->bits == 8 && (!a->m_scale || !a->v_scale)) || (a->dtype != CX_F32 && !a->master))
    return cx_set_error("cx_adamw_step: a table or state is missing", 0);
  return dev == CX_DEV_CUDA ? cx_adamw_step_cuda(a, stream) : on_host(cx_adamw_step_host, a);
}

int64_t cx_linear_workspace_bytes(int dev, const CxLinear* l, int backward) {
  return dev == CX_DEV_CUDA && !wrong(l) ? cx_linear_workspace_bytes_cuda(l, backward) : 0;
}

int cx_linear_forward(int dev, const CxLinear* l, void* stream) {
  if (const char* why = wrong(l)) return cx_set_error(why, 0);
  if (!l->x || !l->w || !l->y) return cx_set_error("cx_linear_forward: an operand is missing", 0);
  if (l->ldx < l->inner || l->ldw < l->inner || (l->residual && l->ldr < l->outer) || (l->pre && l->ldpre < l->outer))
    return cx_set_error("cx_linear_forward: rows overlap", 0);
  return dev == CX_DEV_CUDA ? cx_linear_forward_cuda(l, noted(stream)) : on_host(cx_linear_forward_host, l);
}

int cx_linear_backward(int dev, const CxLinear* l, void* stream) {
  if (const char* why = wrong(l)) return cx_set_error(why, 0);
  if (!l->grad || (l->dx && !l->w) || (l->dw && !l->x) || (l->act != CX_ACT_NONE && !l->pre))
    return cx_set_error("cx_linear_backward: an operand is missing", 0);
  if (l->ldg < l->outer || (l->act != CX_ACT_NONE && l->ldpre < l->outer) || (l->dw && l->ldx < l->inner) || (l->dx && l->ldw < l->inner))
    return cx_set_error("cx_linear_backward: rows overlap", 0);
  return dev == CX_DEV_CUDA ? cx_linear_backward_cuda(l, noted(stream)) : on_host(cx_linear_backward_host, l);
}

int64_t cx_vocab_loss_workspace_bytes(int dev, const CxVocabLoss* l, int backward) {
  return dev == CX_DEV_CUDA && !wrong(l) ? cx_vocab_loss_workspace_bytes_cuda(l, backward) : 0;
}

int cx_vocab_loss_forward(int dev, const CxVocabLoss* l, void* stream) {
  if (const char* why = wrong(l)) return cx_set_error(why, 0);
  if (!l->loss) return cx_set_error("cx_vocab_loss_forward: an operand is missing", 0);
  return dev == CX_DEV_CUDA ? cx_vocab_loss_forward_cuda(l, noted(stream)) : on_host(cx_vocab_loss_forward_host, l);
}

int cx_vocab_loss_backward(int dev, const CxVocabLoss* l, void* stream) {
  if (const char* why = wrong(l)) return cx_set_error(why, 0);
  if (!l->grad) return cx_set_error("cx_vocab_loss_backward: an operand is missing", 0);
  if (!l->dh && !l->dw) return 0;
  return dev == CX_DEV_CUDA ? cx_vocab_loss_backward_cuda(l, noted(stream)) : on_host(cx_vocab_loss_backward_host, l);
}

int64_t cx_ops_sizeof(int what) {
  switch (what) {
    case 0: return (int64_t)sizeof(CxAdamW);
    case 1: return (int64_t)sizeof(CxLinear);
    case 2: return (int64_t)sizeof(CxVocabLoss);
    default: return -1;
  }
}

}  // extern "C"
