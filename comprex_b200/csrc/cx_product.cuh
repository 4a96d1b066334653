// A product of two matrices with what is done to each of its elements: the core of the linear operator and of the
// vocabulary loss.  C[m][n] = sum_k A(m, k) B(n, k), sums in 32 bits.
#pragma once
#include "cx_device.cuh"
#include "cx_ops.h"

enum CxLayout {       // how the operands lie in memory (rows of consecutive elements)
  kNT = 0,            // A[m][k], B[n][k]
  kNN = 1,            // A[m][k], B[k][n]
  kTN = 2             // A[k][m], B[k][n]
};
enum CxProductMode {
  kOut = 0,           // out = act((C + addend) * scale + bias) + residual
  kSums = 1,          // addend = C (+ addend): 32-bit sums that a later product goes on with
  kStats = 2,         // per row and tile of columns: largest logit and sum of exponentials; the target's logit
  kProb = 3           // out = (exp(C - lse) - [column is the target]) * row factor
};

struct CxProduct {
  int64_t m, n, k;
  const void* a;
  const void* b;
  int64_t lda, ldb;
  int32_t layout, mode, dtype, act;
  void* out;               // kOut, kProb
  int64_t ldo;
  const void* bias;        // kOut: [n]
  const void* residual;    // kOut
  int64_t ldr;
  void* pre;               // kOut: (C + addend) * scale + bias, rounded
  int64_t ldpre;
  float* addend;           // [m][ldadd], 32-byte aligned rows
  int64_t ldadd;
  int32_t has_addend;      // it holds sums already
  const float* scale;      // device cell, NULL: 1
  float2* part;            // kStats: [tile][m]
  float* target_logit;     // kStats: [m]
  const int64_t* targets;  // kStats, kProb: [m]
  int64_t col0;            // kStats, kProb: column 0 is this entry of the vocabulary
  const float* lse;        // kProb: [m], in units of log 2
  const float* row_factor; // kProb: [m]
  void* workspace;
  int64_t ws_bytes;
};

namespace cxprod {

struct Arena {                 // workspace handed out front to back; without a base it only counts
  char* base;
  int64_t used, size;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += (bytes + 255) / 256 * 256;
    return p;
  }
  bool ok() const { return used <= size; }
};

}  // namespace cxprod

// One product, or two that do not depend on one another and share the GPU.  Takes their own workspace from `ws`;
// without a base nothing is launched and the arena counts.
int cx_product(CxProduct* p, int count, cxprod::Arena& ws, cudaStream_t s);
// An operand as the tensor cores can read it: itself, or a copy in `ws` whose rows are 16-byte aligned (16-bit types).
int cx_product_operand(const void** base, int64_t* ld, int dtype, int64_t rows, int64_t cols, cxprod::Arena& ws, cudaStream_t s);
// columns of a kStats tile
int cx_product_stat_columns(const CxProduct& p);

// tensor_product.cu: 16-bit types, operands as cx_product_operand leaves them
int cx_tensor_product_stat_columns(const CxProduct& p);
// about how long that takes, in us
double cx_tensor_product_time(const CxProduct* p, int count);
int cx_tensor_product(CxProduct* p, int count, cxprod::Arena& ws, cudaStream_t s);

// A launch that may become resident while the kernel in front is ending; every kernel launched so calls cx::pdl_wait
// before it touches memory.
template <typename K, typename P>
void cx_launch_pdl2(K kernel, dim3 grid, int threads, cudaStream_t s, const P& params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cx_pdl_enabled() ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, params);           // (an error is the next cx_check_launch's)
}

namespace cxprod {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Activations in terms of u = x w^T + b.  gelu_tanh(u) = u sigmoid(2 z), z = sqrt(2 / pi) (u + 0.044715 u^3): the same
// function as u / 2 (1 + tanh z), with one exponential and without the sum's cancellation.
//
// For results of 16 bits power of two and reciprocal are the hardware's: each is about 2 units of 2^-23 off, the argument's
// rounding 1.44 |2 z| more of 2^-24 (z = -40: 5e-6 of the result, which is rounded to 2^-9 or 2^-12 of itself), and a gate below
// 2^-126 is 0.  Results of 32 bits take expf of an argument that is rounded once, and a true quotient.
constexpr float kGelu = 1.5957691216057308f;       // 2 sqrt(2 / pi)
__device__ __forceinline__ float sigmoid_full(float z) {
  const float t = expf(-fabsf(z));
  return (z >= 0.f ? 1.f : t) / (1.f + t);
}
template <bool FULL>
__device__ __forceinline__ float sigmoid(float z) {
  return FULL ? sigmoid_full(z) : inverse(1.f + pow2(-kLog2e * z));
}
template <bool FULL>
__device__ __forceinline__ float gelu_gate(float u) {
  return FULL ? sigmoid_full(u * __fmaf_rn(u * u, 0.044715f * kGelu, kGelu)) : inverse(1.f + pow2(u * __fmaf_rn(u * u, -0.044715f * kGelu * kLog2e, -kGelu * kLog2e)));
}
// T: of the results
template <typename T, int N>
__device__ __forceinline__ void activate(float (&v)[N], int act) {
  constexpr bool full = sizeof(T) == 4;
  if (act == CX_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] > 0.f || v[i] != v[i] ? v[i] : 0.f;
  } else if (act == CX_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.5f * v[i] * (1.f + erff(v[i] * 0.70710678118654752f));
  } else if (act == CX_ACT_GELU_TANH) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= gelu_gate<full>(v[i]);
  } else if (act == CX_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= sigmoid<full>(v[i]);
  }
}
template <typename T, int ACT>
__device__ __forceinline__ float slope(float u) {
  constexpr bool full = sizeof(T) == 4;
  if (ACT == CX_ACT_RELU) return u > 0.f ? 1.f : 0.f;
  if (ACT == CX_ACT_GELU) {
    const float bell = full ? expf(-0.5f * u * u) : pow2(-0.5f * kLog2e * u * u);
    return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * 0.39894228040143268f * bell;
  }
  if (ACT == CX_ACT_GELU_TANH) {
    const float q = gelu_gate<full>(u);
    return q + u * q * (1.f - q) * kGelu * __fmaf_rn(u * u, 0.134145f, 1.f);
  }
  if (ACT == CX_ACT_SILU) {
    const float q = sigmoid<full>(u);
    return q * __fmaf_rn(u, 1.f - q, 1.f);
  }
  return 1.f;
}

// 8 neighbouring elements of a row, as 16 bytes where `wide`, else the first `left` one by one
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool wide, int left, float (&v)[8]) {
  if (wide) {
    float lo[4], hi[4];
    if (sizeof(T) == 2) {
      const uint4 t = *reinterpret_cast<const uint4*>(p);
      cx::Raw4<T>::to_f(reinterpret_cast<const typename cx::Raw4<T>::type*>(&t)[0], lo);
      cx::Raw4<T>::to_f(reinterpret_cast<const typename cx::Raw4<T>::type*>(&t)[1], hi);
    } else {
      cx::load4(p, lo);
      cx::load4(p + 4, hi);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = lo[i];
      v[4 + i] = hi[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? cx::Elem<T>::to_f(p[i]) : 0.f;
  }
}
__device__ __forceinline__ void pack4(const float* v, uint2* out, __nv_bfloat16) {
  const float t[4] = {v[0], v[1], v[2], v[3]};
  cx::store4(reinterpret_cast<__nv_bfloat16*>(out), t);
}
__device__ __forceinline__ void pack4(const float* v, uint2* out, __half) {
  const float t[4] = {v[0], v[1], v[2], v[3]};
  cx::store4(reinterpret_cast<__half*>(out), t);
}
__device__ __forceinline__ void pack4(const float*, uint2*, float) {}
template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, int left, const float* v) {
  if (wide && sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else if (wide) {
    uint2 t[2];
    pack4(v, t, T());
    pack4(v + 4, t + 1, T());
    *reinterpret_cast<uint4*>(p) = make_uint4(t[0].x, t[0].y, t[1].x, t[1].y);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = cx::Elem<T>::from_f(v[i]);
  }
}

}  // namespace cxprod
