// The product of cx_product.cuh for operands of 32 bits, on the CUDA cores (the tensor cores round them to 11 bits): any
// layout and stride.  Not what this package trains large models in; 20 TFLOP/s.
#include "cx_product.cuh"

namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

__device__ __forceinline__ void finish(const CxProduct& p, int64_t row, int64_t col, float v) {
  if (p.mode == kSums) {
    float* at = p.addend + row * p.ldadd + col;
    *at = p.has_addend ? *at + v : v;
    return;
  }
  if (p.mode == kProb) {
    const float q = exp2f(v * cxprod::kLog2e - p.lse[row]) - (p.targets[row] == p.col0 + col ? 1.f : 0.f);
    const float f = p.row_factor[row];
    reinterpret_cast<float*>(p.out)[row * p.ldo + col] = f == 0.f ? 0.f : q * f;
    return;
  }
  if (p.has_addend) v += p.addend[row * p.ldadd + col];
  if (p.scale) v *= *p.scale;
  if (p.bias) v += reinterpret_cast<const float*>(p.bias)[col];
  if (p.pre) reinterpret_cast<float*>(p.pre)[row * p.ldpre + col] = v;
  float one[1] = {v};
  cxprod::activate<float>(one, p.act);
  v = one[0];
  if (p.residual) v += reinterpret_cast<const float*>(p.residual)[row * p.ldr + col];
  reinterpret_cast<float*>(p.out)[row * p.ldo + col] = v;
}

__global__ void __launch_bounds__(kThreads) product_kernel(const __grid_constant__ CxProduct p) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  __shared__ float2 stat[kTile][16];
  // neighbouring blocks have the same columns; one dimension, since a grid's second one ends at 65535
  const uint32_t tiles_m = (uint32_t)((p.m + kTile - 1) / kTile), tile_n = blockIdx.x / tiles_m;
  const int64_t row0 = (int64_t)(blockIdx.x - tile_n * tiles_m) * kTile, col0 = (int64_t)tile_n * kTile;
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  const float* a = reinterpret_cast<const float*>(p.a);
  const float* b = reinterpret_cast<const float*>(p.b);
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.k; k0 += kDepth) {
#pragma unroll
    for (int j = 0; j < kTile * kDepth / kThreads; ++j) {
      const int i = threadIdx.x + j * kThreads;
      // neighbouring threads along the operand's consecutive elements
      const int ka = p.layout == kTN ? i / kTile : i % kDepth, ma = p.layout == kTN ? i % kTile : i / kDepth;
      const int kb = p.layout == kNT ? i % kDepth : i / kTile, nb = p.layout == kNT ? i / kDepth : i % kTile;
      const int64_t r = row0 + ma, c = col0 + nb;
      const bool in_a = r < p.m && k0 + ka < p.k, in_b = c < p.n && k0 + kb < p.k;
      sa[ka][ma] = !in_a ? 0.f : p.layout == kTN ? a[(k0 + ka) * p.lda + r] : a[r * p.lda + k0 + ka];
      sb[kb][nb] = !in_b ? 0.f : p.layout == kNT ? b[c * p.ldb + k0 + kb] : b[(k0 + kb) * p.ldb + c];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
      float x[4], y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = sa[k][tr * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = sb[k][tc * 4 + i];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __fmaf_rn(x[i], y[j], acc[i][j]);
    }
    __syncthreads();
  }
  if (p.mode != kStats) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t r = row0 + tr * 4 + i, c = col0 + tc * 4 + j;
        if (r < p.m && c < p.n) finish(p, r, c, acc[i][j]);
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t r = row0 + tr * 4 + i;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t c = col0 + tc * 4 + j;
      if (c >= p.n || r >= p.m) continue;
      if (p.targets[r] == p.col0 + c) p.target_logit[r] = acc[i][j];
      top = acc[i][j] > top || acc[i][j] != acc[i][j] ? acc[i][j] : top;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col0 + tc * 4 + j < p.n && top != -INFINITY) sum += exp2f((acc[i][j] - top) * cxprod::kLog2e);
    stat[tr * 4 + i][tc] = make_float2(top, sum);
  }
  __syncthreads();
  if (threadIdx.x < kTile && row0 + threadIdx.x < p.m) {
    float top = -INFINITY, sum = 0.f;
    for (int j = 0; j < 16; ++j) {
      const float t = stat[threadIdx.x][j].x;
      top = t > top || t != t ? t : top;
    }
    for (int j = 0; j < 16; ++j) {
      const float2 s = stat[threadIdx.x][j];
      if (s.x != -INFINITY) sum += s.y * exp2f((s.x - top) * cxprod::kLog2e);
    }
    p.part[(int64_t)tile_n * p.m + row0 + threadIdx.x] = make_float2(top, sum);
  }
}

struct Align {
  const uint16_t* from;
  uint16_t* to;
  int64_t ld, rows, cols, to_ld;
};

// rows of `cols` elements, `ld` apart, to rows of `to_ld` (a multiple of 8); what is beyond a row's end is zero
__global__ void __launch_bounds__(kThreads) align_kernel(const __grid_constant__ Align d) {
  cx::pdl_trigger();
  cx::pdl_wait();
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x, per = d.to_ld / 8;
  if (i >= d.rows * per) return;
  const int64_t row = i / per, col = i % per * 8;
  uint16_t v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = col + k < d.cols ? d.from[row * d.ld + col + k] : 0;
  uint4 t;
  memcpy(&t, v, 16);
  *reinterpret_cast<uint4*>(d.to + row * d.to_ld + col) = t;
}

}  // namespace

int cx_product_operand(const void** base, int64_t* ld, int dtype, int64_t rows, int64_t cols, cxprod::Arena& ws, cudaStream_t s) {
  if (dtype == CX_F32 || ((reinterpret_cast<uintptr_t>(*base) & 15) == 0 && *ld % 8 == 0)) return 0;
  const int64_t to_ld = (cols + 7) / 8 * 8;
  void* to = ws.take(rows * to_ld * 2);
  const void* from = *base;
  const int64_t from_ld = *ld;
  *base = to;
  *ld = to_ld;
  if (!ws.base) return 0;
  if (!ws.ok()) return cx_set_error("cx_product: workspace too small", 0);
  const Align d = {reinterpret_cast<const uint16_t*>(from), reinterpret_cast<uint16_t*>(to), from_ld, rows, cols, to_ld};
  cx_launch_pdl2(align_kernel, dim3((unsigned)((rows * (to_ld / 8) + kThreads - 1) / kThreads)), kThreads, s, d);
  cx_note_launch();
  return cx_check_launch("cx_product");
}

int cx_product_stat_columns(const CxProduct& p) { return p.dtype != CX_F32 ? cx_tensor_product_stat_columns(p) : kTile; }

int cx_product(CxProduct* p, int count, cxprod::Arena& ws, cudaStream_t s) {
  if (p[0].dtype != CX_F32) return cx_tensor_product(p, count, ws, s);
  if (!ws.base) return 0;
  if (!ws.ok()) return cx_set_error("cx_product: workspace too small", 0);
  for (int i = 0; i < count; ++i) {
    const int64_t tiles = ((p[i].m + kTile - 1) / kTile) * ((p[i].n + kTile - 1) / kTile);
    if (tiles > 0x7FFFFFFF) return cx_set_error("cx_product: too many tiles", 0);
    product_kernel<<<(unsigned)tiles, kThreads, 0, s>>>(p[i]);
    cx_note_launch();
  }
  return cx_check_launch("cx_product");
}
