// y = act(x w^T + bias) + residual and its gradients.
//
//   u = x w^T + b    y = act(u) + r        du = dy act'(u)    dx = du w    dw = du^T x    db = sum of du over the rows
//
// Forward is one product with everything else in its epilogue.  Backward is one pass that makes du (where there is an
// activation) and its column sums, and the two products, which read du, w and x where they lie: none is transposed in
// memory.
#include "cx_product.cuh"

namespace {

constexpr int kThreads = 256, kRowsPer = 64;      // a block of du_kernel: 64 rows of 256 columns

struct Du {
  const void* grad;
  const void* pre;
  void* du;             // NULL: not stored
  float* part;          // [chunks][outer], NULL: no sums
  int64_t rows, outer, ldg, ldd;
  int32_t act;
  int32_t wide_in, wide_out;       // 16-byte accesses are aligned
};

// du, and the sums of its columns over 64 rows.  Bound by memory: a thread has 8 neighbouring columns of 8 rows, all of
// them under way at once; the 8 threads of a column join their sums in shared memory, in a fixed order.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) du_kernel(const __grid_constant__ Du d) {
  __shared__ float sums[8][256 + 8];
  cx::pdl_trigger();
  cx::pdl_wait();
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 256 + lane * 8, r0 = (int64_t)blockIdx.y * kRowsPer + group;
  const int left = (int)max((int64_t)0, min((int64_t)8, d.outer - c));
  constexpr bool act = ACT != CX_ACT_NONE;
  float sum[8] = {};
  const T* grad = reinterpret_cast<const T*>(d.grad) + c;
  const T* pre = reinterpret_cast<const T*>(d.pre) + c;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float g[4][8], u[4][8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + 8 * (4 * h + j);
      const int have = r < d.rows ? left : 0;
      cxprod::load8(grad + r * d.ldg, have == 8 && d.wide_in, have, g[j]);
      if (act) cxprod::load8(pre + r * d.outer, have == 8 && d.wide_in, have, u[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + 8 * (4 * h + j);
      if (r >= d.rows || left == 0) continue;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (act) g[j][i] *= cxprod::slope<ACT>(u[j][i]);
        sum[i] += i < left ? g[j][i] : 0.f;
      }
      if (d.du) cxprod::store8(reinterpret_cast<T*>(d.du) + r * d.ldd + c, left == 8 && d.wide_out, left, g[j]);
    }
  }
  if (!d.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[group][lane * 8 + i] = sum[i];
  __syncthreads();
  const int64_t mine = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (mine >= d.outer) return;
  float all = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) all += sums[j][threadIdx.x];
  d.part[blockIdx.y * d.outer + mine] = all;
}

struct ColumnSums {
  const float* part;
  int64_t chunks, outer;
  void* out;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) column_sum_kernel(const __grid_constant__ ColumnSums d) {
  __shared__ float sums[8][33];
  cx::pdl_trigger();
  cx::pdl_wait();
  const int lane = threadIdx.x % 32, group = threadIdx.x / 32;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float sum = 0.f;
  if (c < d.outer) {
#pragma unroll 4
    for (int64_t i = group; i < d.chunks; i += 8) sum += d.part[i * d.outer + c];
  }
  sums[group][lane] = sum;
  __syncthreads();
  if (group || c >= d.outer) return;
#pragma unroll
  for (int j = 1; j < 8; ++j) sum += sums[j][lane];
  reinterpret_cast<T*>(d.out)[c] = cx::Elem<T>::from_f(sum);
}

template <typename T>
int du_pass(Du& d, void* dbias, cudaStream_t s) {
  const int64_t chunks = (d.rows + kRowsPer - 1) / kRowsPer;
  const uintptr_t in = reinterpret_cast<uintptr_t>(d.grad) | (d.act != CX_ACT_NONE ? reinterpret_cast<uintptr_t>(d.pre) : 0);
  d.wide_in = (in & 15) == 0 && d.ldg % 8 == 0 && (d.act == CX_ACT_NONE || d.outer % 8 == 0);
  d.wide_out = (reinterpret_cast<uintptr_t>(d.du) & 15) == 0 && d.ldd % 8 == 0;
  for (int64_t first = 0; first < chunks; first += 65535) {        // a grid's second dimension ends there
    Du part = d;
    part.grad = reinterpret_cast<const T*>(d.grad) + first * kRowsPer * d.ldg;
    if (d.pre) part.pre = reinterpret_cast<const T*>(d.pre) + first * kRowsPer * d.outer;
    if (d.du) part.du = reinterpret_cast<T*>(d.du) + first * kRowsPer * d.ldd;
    if (d.part) part.part = d.part + first * d.outer;
    part.rows = d.rows - first * kRowsPer;
    const dim3 grid((unsigned)((d.outer + 255) / 256), (unsigned)(chunks - first < 65535 ? chunks - first : 65535));
    switch (d.act) {
      case CX_ACT_RELU: cx_launch_pdl2(du_kernel<T, CX_ACT_RELU>, grid, kThreads, s, part); break;
      case CX_ACT_GELU: cx_launch_pdl2(du_kernel<T, CX_ACT_GELU>, grid, kThreads, s, part); break;
      case CX_ACT_GELU_TANH: cx_launch_pdl2(du_kernel<T, CX_ACT_GELU_TANH>, grid, kThreads, s, part); break;
      case CX_ACT_SILU: cx_launch_pdl2(du_kernel<T, CX_ACT_SILU>, grid, kThreads, s, part); break;
      default: cx_launch_pdl2(du_kernel<T, CX_ACT_NONE>, grid, kThreads, s, part);
    }
    cx_note_launch();
  }
  if (dbias) {
    const ColumnSums c = {d.part, chunks, d.outer, dbias};
    cx_launch_pdl2(column_sum_kernel<T>, dim3((unsigned)((d.outer + 31) / 32)), kThreads, s, c);
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
  return rc ? rc : cx_product(&p, 1, ws, s);
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
  CxProduct both[2] = {};
  int count = 0;
  if (l.dx && !rc) {
    CxProduct& p = both[count++];
    p.m = l.rows; p.n = l.inner; p.k = l.outer;
    p.a = du; p.lda = ldd; p.b = l.w; p.ldb = l.ldw;
    p.layout = kNN; p.dtype = l.dtype; p.out = l.dx; p.ldo = l.inner;
    rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.outer, l.inner, ws, s);
  }
  if (l.dw && !rc) {
    CxProduct& p = both[count++];
    p.m = l.outer; p.n = l.inner; p.k = l.rows;
    p.a = du; p.lda = ldd; p.b = l.x; p.ldb = l.ldx;
    p.layout = kTN; p.dtype = l.dtype; p.out = l.dw; p.ldo = l.inner;
    rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.rows, l.inner, ws, s);
  }
  return rc || !count ? rc : cx_product(both, count, ws, s);
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
