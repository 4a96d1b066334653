// y = act(x w^T + bias) + residual and its gradients.
//
//   u = x w^T + b    y = act(u) + r        du = dy act'(u)    dx = du w    dw = du^T x    db = sum of du over the rows
//
// Forward is one product with everything else in its epilogue.  Backward is one pass that makes du (where there is an
// activation) and its column sums, and the two products, which read du, w and x where they lie: none is transposed in
// memory.
//
// Bound by the tensor cores for many rows and by reading w for few.  8192 rows in bf16: 1024 -> 4096 with bias and tanh GELU
// 69 us with u kept and 59 without (48 without any epilogue), its gradients 48 us for du and db and 93 for the two products
// (1.48 PFLOP/s); 4096 -> 1024 with bias and residual 56 us, its gradients 85.
#include "cx_product.cuh"

namespace {

constexpr int kThreads = 256, kRowsPer = 64;      // a block of du_kernel: 64 rows of 256 columns

struct Du {
  const void* grad;
  const void* pre;
  void* du;             // NULL: not stored
  float* part;          // [chunks][outer], NULL: no sums
  int64_t rows, outer, ldg, ldpre, ldd;
  int32_t act;
  int32_t wide_grad, wide_pre, wide_out;       // 16-byte accesses are aligned
};

// 8 neighbouring elements as they lie in memory
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool wide, int have) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = make_uint4(0, 0, 0, 0);
    if (wide) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < have) reinterpret_cast<T*>(w)[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = cx::Elem<T>::to_f(reinterpret_cast<const T*>(w)[i]);
  }
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
  const bool wide = left == 8 && d.wide_grad && (!act || d.wide_pre);
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    // as they lie in memory until they are used: 16 loads of 16 bytes (of 16-bit types) under way in 64 registers
    Raw8<T> g[4], u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + 8 * (4 * h + j);
      const int have = r < d.rows ? left : 0;
      g[j].load(grad + r * d.ldg, wide && have, have);
      if (act) u[j].load(pre + r * d.ldpre, wide && have, have);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t r = r0 + 8 * (4 * h + j);
      if (r >= d.rows || left == 0) continue;
      float x[8], y[8];
      g[j].get(x);
      if (act) u[j].get(y);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (act) x[i] *= cxprod::slope<T, ACT>(y[i]);
        sum[i] += x[i];                                   // (zero from `left` on)
      }
      if (d.du) cxprod::store8(reinterpret_cast<T*>(d.du) + r * d.ldd + c, left == 8 && d.wide_out, left, x);
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
  d.wide_grad = (reinterpret_cast<uintptr_t>(d.grad) & 15) == 0 && d.ldg % 8 == 0;
  d.wide_pre = (reinterpret_cast<uintptr_t>(d.pre) & 15) == 0 && d.ldpre % 8 == 0;
  d.wide_out = (reinterpret_cast<uintptr_t>(d.du) & 15) == 0 && d.ldd % 8 == 0;
  for (int64_t first = 0; first < chunks; first += 65535) {        // a grid's second dimension ends there
    Du part = d;
    part.grad = reinterpret_cast<const T*>(d.grad) + first * kRowsPer * d.ldg;
    if (d.pre) part.pre = reinterpret_cast<const T*>(d.pre) + first * kRowsPer * d.ldpre;
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

// ---- few rows: tokens that are being decoded ------------------------------------------------------------------------
// Bound by reading w, and at these sizes by latency: every weight is used once per row, so the tensor cores have nothing to
// do.  A warp has four rows of w and a share of k, 256 elements at a time, all loads of a turn under way at once; `share`
// warps of a block join their sums in a fixed order, and one thread per result does the rest.
constexpr int kFewColumns = 4, kWarps = kThreads / 32;

struct Few {
  const void* x;
  const void* w;
  const void* bias;
  const void* residual;
  void* y;
  void* pre;
  int64_t inner, outer, ldx, ldw, ldr, ldpre;
  int rows, act, share;
};

// Sums of V values (4 to 16) over the warp, each in the lanes whose highest bits are its number.  A step halves what a lane
// holds, so that V values take about V shuffles instead of 5 V.
template <int V>
__device__ __forceinline__ void warp_sums(float (&v)[V], int lane) {
  int have = V;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (have > 1) {
      have /= 2;
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        if (i < have) {
          const float give = lane & o ? v[i] : v[i + have], keep = lane & o ? v[i + have] : v[i];
          v[i] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
        }
    } else {
      v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
    }
  }
}

template <typename T, int R, bool WIDE>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(const __grid_constant__ Few d) {
  constexpr int V = R * kFewColumns;
  __shared__ float sums[kWarps][V];
  cx::pdl_trigger();
  cx::pdl_wait();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, groups = kWarps / d.share;
  const int64_t c0 = ((int64_t)blockIdx.x * groups + warp / d.share) * kFewColumns;
  const T* x = reinterpret_cast<const T*>(d.x);
  const T* w = reinterpret_cast<const T*>(d.w) + c0 * d.ldw;
  const int columns = (int)max((int64_t)0, min((int64_t)kFewColumns, d.outer - c0));
  float acc[V] = {};
  for (int64_t k = (warp % d.share) * 256 + lane * 8; k < d.inner; k += d.share * 256) {
    const int left = (int)min((int64_t)8, d.inner - k);
    float b[kFewColumns][8];
#pragma unroll
    for (int c = 0; c < kFewColumns; ++c) cxprod::load8(w + c * d.ldw + k, WIDE && left == 8 && c < columns, c < columns ? left : 0, b[c]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float a[8];
      cxprod::load8(x + r * d.ldx + k, WIDE && left == 8 && r < d.rows, r < d.rows ? left : 0, a);
#pragma unroll
      for (int c = 0; c < kFewColumns; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[r * kFewColumns + c] = __fmaf_rn(a[i], b[c][i], acc[r * kFewColumns + c]);
    }
  }
  warp_sums<V>(acc, lane);
  // a lane holds the value that its number says, highest bit first
  constexpr int kBits = V == 16 ? 4 : V == 8 ? 3 : 2;
  int at = 0, size = V;
#pragma unroll
  for (int i = 0; i < kBits; ++i) {
    size /= 2;
    at += lane & (16 >> i) ? size : 0;
  }
  sums[warp][at] = acc[0];
  __syncthreads();
  for (int i = threadIdx.x; i < groups * V; i += kThreads) {
    const int g = i / V, r = i % V / kFewColumns;
    const int64_t c = ((int64_t)blockIdx.x * groups + g) * kFewColumns + i % kFewColumns;
    if (r >= d.rows || c >= d.outer) continue;
    float v[1] = {0.f};
    for (int j = 0; j < d.share; ++j) v[0] += sums[g * d.share + j][i % V];
    using E = cx::Elem<T>;
    if (d.bias) v[0] += E::to_f(reinterpret_cast<const T*>(d.bias)[c]);
    if (d.pre) reinterpret_cast<T*>(d.pre)[r * d.ldpre + c] = E::from_f(v[0]);
    cxprod::activate<T>(v, d.act);
    if (d.residual) v[0] += E::to_f(reinterpret_cast<const T*>(d.residual)[r * d.ldr + c]);
    reinterpret_cast<T*>(d.y)[r * d.outer + c] = E::from_f(v[0]);
  }
}

template <typename T, int R>
void few_rows_of(const Few& d, bool wide, dim3 grid, cudaStream_t s) {
  if (wide) cx_launch_pdl2(few_rows_kernel<T, R, true>, grid, kThreads, s, d);
  else cx_launch_pdl2(few_rows_kernel<T, R, false>, grid, kThreads, s, d);
}

template <typename T>
int few_rows(const CxLinear& l, cudaStream_t s) {
  Few d = {l.x, l.w, l.bias, l.residual, l.y, l.pre, l.inner, l.outer, l.ldx, l.ldw, l.ldr, l.ldpre, (int)l.rows, l.act, 1};
  while (d.share < kWarps && d.share * 512 < l.inner) d.share *= 2;
  constexpr int64_t per = 16 / sizeof(T);
  const bool wide = ((reinterpret_cast<uintptr_t>(l.x) | reinterpret_cast<uintptr_t>(l.w)) & 15) == 0 && l.ldx % per == 0 && l.ldw % per == 0;
  const int64_t columns = kFewColumns * kWarps / d.share;
  const dim3 grid((unsigned)((l.outer + columns - 1) / columns));
  if (l.rows == 1) few_rows_of<T, 1>(d, wide, grid, s);
  else if (l.rows <= 2) few_rows_of<T, 2>(d, wide, grid, s);
  else few_rows_of<T, 4>(d, wide, grid, s);
  cx_note_launch();
  return cx_check_launch("cx_linear_forward");
}

// Both calls also run without a workspace: they launch nothing then and count the bytes that they need.
int forward(const CxLinear& l, cxprod::Arena& ws, cudaStream_t s) {
  // On the CUDA cores up to two rows, and up to four where w is small or of 32 bits, which the tensor cores do not multiply.  Weights
  // from memory, one row, then four; here / as tiles, us: bf16 1024 x 1024 3.5 / 5.4, 4.3 / 5.5; 2048 x 4096 5.5 / 10.0, 10.7 / 10.1;
  // 4096 x 4096 9.6 / 12.6, 15.7 / 12.8 (two rows 13.6 / 12.7); float32 1024 x 1024 3.6 / 102, 4.9 / 105; 4096 x 4096 11.7 / 425, 17.2 / 428.
  if (l.rows <= 2 || (l.rows <= 4 && (l.dtype == CX_F32 || l.outer * l.inner <= (8 << 20)))) {
    if (!ws.base) return 0;
    return l.dtype == CX_F32 ? few_rows<float>(l, s) : l.dtype == CX_BF16 ? few_rows<__nv_bfloat16>(l, s) : few_rows<__half>(l, s);
  }
  CxProduct p = {};
  p.m = l.rows; p.n = l.outer; p.k = l.inner;
  p.a = l.x; p.lda = l.ldx; p.b = l.w; p.ldb = l.ldw;
  p.layout = kNT; p.dtype = l.dtype; p.act = l.act;
  p.out = l.y; p.ldo = l.outer; p.bias = l.bias; p.residual = l.residual; p.ldr = l.ldr; p.pre = l.pre; p.ldpre = l.ldpre;
  int rc = cx_product_operand(&p.a, &p.lda, l.dtype, l.rows, l.inner, ws, s);
  if (!rc) rc = cx_product_operand(&p.b, &p.ldb, l.dtype, l.outer, l.inner, ws, s);
  if (!rc && p.residual) rc = cx_product_operand(&p.residual, &p.ldr, l.dtype, l.rows, l.outer, ws, s);
  return rc ? rc : cx_product(&p, 1, ws, s);
}

int backward(const CxLinear& l, cxprod::Arena& ws, cudaStream_t s) {
  const int64_t size = l.dtype == CX_F32 ? 4 : 2;
  Du d = {};
  d.grad = l.grad; d.pre = l.pre;
  d.rows = l.rows; d.outer = l.outer; d.ldg = l.ldg; d.ldpre = l.ldpre; d.act = l.act;
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
