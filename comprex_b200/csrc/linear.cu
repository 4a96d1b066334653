// y = act(x w^T + bias) + residual and its gradients.
//
//   u = x w^T + b    y = act(u) + r        du = dy act'(u)    dx = du w    dw = du^T x    db = sum of du over the rows
//
// Forward is one product with everything else in its epilogue.  Backward is one pass that makes du (where there is an
// activation) and its column sums, and the two products, which read du, w and x where they lie: none is transposed in
// memory.
#include "cx_product.cuh"

namespace {

constexpr int kThreads = 256, kRowsPer = 64;

struct Du {
  const void* grad;
  const void* pre;
  void* du;             // NULL: not stored
  float* part;          // [chunks][outer], NULL: no sums
  int64_t rows, outer, ldg, ldd;
  int32_t act;
};

// du and the sums of its columns over kRowsPer rows; a thread has a column
template <typename T>
__global__ void __launch_bounds__(kThreads) du_kernel(const Du d) {
  using E = cx::Elem<T>;
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= d.outer) return;
  const int64_t r0 = (int64_t)blockIdx.y * kRowsPer, r1 = min(d.rows, r0 + kRowsPer);
  float sum = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    float g = E::to_f(reinterpret_cast<const T*>(d.grad)[r * d.ldg + c]);
    if (d.act != CX_ACT_NONE) g *= cxprod::slope(E::to_f(reinterpret_cast<const T*>(d.pre)[r * d.outer + c]), d.act);
    sum += g;
    if (d.du) reinterpret_cast<T*>(d.du)[r * d.ldd + c] = E::from_f(g);
  }
  if (d.part) d.part[blockIdx.y * d.outer + c] = sum;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) column_sum_kernel(const float* part, int64_t chunks, int64_t outer, T* out) {
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= outer) return;
  float sum = 0.f;
  for (int64_t i = 0; i < chunks; ++i) sum += part[i * outer + c];
  out[c] = cx::Elem<T>::from_f(sum);
}

template <typename T>
int du_pass(const Du& d, void* dbias, cudaStream_t s) {
  const int64_t chunks = (d.rows + kRowsPer - 1) / kRowsPer, cols = (d.outer + kThreads - 1) / kThreads;
  du_kernel<T><<<dim3((unsigned)cols, (unsigned)chunks), kThreads, 0, s>>>(d);
  cx_note_launch();
  if (dbias) {
    column_sum_kernel<T><<<(unsigned)cols, kThreads, 0, s>>>(d.part, chunks, d.outer, reinterpret_cast<T*>(dbias));
    cx_note_launch();
  }
  return cx_check_launch("cx_linear_backward");
}

// Both calls also run without a workspace: they launch nothing then and count the bytes that they need.
int forward(const CxLinear& l, cxprod::Arena& ws, cudaStream_t s) {
  CxProduct p = {};
  p.m = l.rows; p.n = l.outer; p.k = l.inner;
  p.a = l.x; p.lda = l.ldx; p.b = l.w; p.ldb = l.ldw;
  p.layout = kNT; p.dtype = l.dtype; p.act = l.act;
  p.out = l.y; p.ldo = l.outer; p.bias = l.bias; p.residual = l.residual; p.ldr = l.ldr; p.pre = l.pre;
  int rc = cx_product_operand(&p.a, &p.lda, l.dtype, l.rows, l.inner, ws, s);
  if (!rc) rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.outer, l.inner, ws, s);
  return rc ? rc : cx_product(p, ws, s);
}

int backward(const CxLinear& l, cxprod::Arena& ws, cudaStream_t s) {
  const int64_t size = l.dtype == CX_F32 ? 4 : 2;
  Du d = {};
  d.grad = l.grad; d.pre = l.pre;
  d.rows = l.rows; d.outer = l.outer; d.ldg = l.ldg; d.act = l.act;
  const void* du = l.grad;
  int64_t ldd = l.ldg;
  if (l.act != CX_ACT_NONE && (l.dx || l.dw)) {
    d.ldd = ldd = (l.outer + 7) / 8 * 8;
    du = d.du = ws.take(l.rows * ldd * size);
  }
  if (l.dbias) d.part = reinterpret_cast<float*>(ws.take((l.rows + kRowsPer - 1) / kRowsPer * l.outer * 4));
  int rc = 0;
  if (ws.base && !ws.ok()) return cx_set_error("cx_linear_backward: workspace too small", 0);
  if (ws.base && (d.du || d.part))
    rc = l.dtype == CX_F32 ? du_pass<float>(d, l.dbias, s)
         : l.dtype == CX_BF16 ? du_pass<__nv_bfloat16>(d, l.dbias, s) : du_pass<__half>(d, l.dbias, s);
  if (!rc && (l.dx || l.dw)) rc = cx_product_operand(&du, &ldd, l.dtype, l.rows, l.outer, ws, s);
  if (l.dx && !rc) {
    CxProduct p = {};
    p.m = l.rows; p.n = l.inner; p.k = l.outer;
    p.a = du; p.lda = ldd; p.b = l.w; p.ldb = l.ldw;
    p.layout = kNN; p.dtype = l.dtype; p.out = l.dx; p.ldo = l.inner;
    rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.outer, l.inner, ws, s);
    if (!rc) rc = cx_product(p, ws, s);
  }
  if (l.dw && !rc) {
    CxProduct p = {};
    p.m = l.outer; p.n = l.inner; p.k = l.rows;
    p.a = du; p.lda = ldd; p.b = l.x; p.ldb = l.ldx;
    p.layout = kTN; p.dtype = l.dtype; p.out = l.dw; p.ldo = l.inner;
    rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.rows, l.inner, ws, s);
    if (!rc) rc = cx_product(p, ws, s);
  }
  return rc;
}

}  // namespace

int64_t cx_linear_workspace_bytes_cuda(const CxLinear* l, int back) {
  cxprod::Arena ws = {nullptr, 0, 0};
  (back ? backward : forward)(*l, ws, nullptr);
  return ws.used + 256;          // never none: without a base nothing runs
}
int cx_linear_forward_cuda(const CxLinear* l, void* stream) {
  cxprod::Arena ws = {reinterpret_cast<char*>(l->workspace), 0, l->ws_bytes};
  return ws.base ? forward(*l, ws, static_cast<cudaStream_t>(stream)) : cx_set_error("cx_linear_forward: no workspace", 0);
}
int cx_linear_backward_cuda(const CxLinear* l, void* stream) {
  cxprod::Arena ws = {reinterpret_cast<char*>(l->workspace), 0, l->ws_bytes};
  return ws.base ? backward(*l, ws, static_cast<cudaStream_t>(stream)) : cx_set_error("cx_linear_backward: no workspace", 0);
}
