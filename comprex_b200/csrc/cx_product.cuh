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
  void* pre;               // kOut: (C + addend) * scale + bias, rounded, rows ldo apart
  float* addend;           // [m][n] without gaps
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

// Takes the product's own workspace from `ws`; without a base nothing is launched and the arena counts.
int cx_product(CxProduct& p, cxprod::Arena& ws, cudaStream_t s);
// An operand as the tensor cores can read it: itself, or a copy in `ws` whose rows are 16-byte aligned (16-bit types).
int cx_product_operand(const void** base, int64_t* ld, int dtype, int64_t rows, int64_t cols, cxprod::Arena& ws, cudaStream_t s);
// columns of a kStats tile
int cx_product_stat_columns(const CxProduct& p);

// tensor_product.cu: 16-bit types, operands that a tile copy can read (16-byte aligned rows)
bool cx_tensor_product_takes(const CxProduct& p);
int cx_tensor_product_stat_columns(const CxProduct& p);
int64_t cx_tensor_product_workspace_bytes(const CxProduct& p);
int cx_tensor_product(const CxProduct& p, cudaStream_t s);

namespace cxprod {

constexpr float kLog2e = 1.4426950408889634f;

// Activations in terms of u = x w^T + b.  gelu_tanh(u) = u / (1 + exp(-2 z)), z = sqrt(2 / pi) (u + 0.044715 u^3): the
// same function as u / 2 (1 + tanh z), with one exponential.
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
__device__ __forceinline__ float activate(float u, int act) {
  switch (act) {
    case CX_ACT_RELU: return u > 0.f || u != u ? u : 0.f;
    case CX_ACT_GELU: return 0.5f * u * (1.f + erff(u * 0.70710678118654752f));
    case CX_ACT_GELU_TANH: return u * sigmoid(1.5957691216057308f * (u + 0.044715f * u * u * u));
    case CX_ACT_SILU: return u * sigmoid(u);
    default: return u;
  }
}
__device__ __forceinline__ float slope(float u, int act) {
  switch (act) {
    case CX_ACT_RELU: return u > 0.f ? 1.f : 0.f;
    case CX_ACT_GELU: return 0.5f * (1.f + erff(u * 0.70710678118654752f)) + u * 0.39894228040143268f * __expf(-0.5f * u * u);
    case CX_ACT_GELU_TANH: {
      const float q = sigmoid(1.5957691216057308f * (u + 0.044715f * u * u * u));
      return q + u * q * (1.f - q) * 1.5957691216057308f * (1.f + 0.134145f * u * u);
    }
    case CX_ACT_SILU: {
      const float q = sigmoid(u);
      return q * (1.f + u * (1.f - q));
    }
    default: return 1.f;
  }
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
template <typename T>
__device__ __forceinline__ void store8(T* p, bool wide, int left, const float (&v)[8]) {
  if (wide) {
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
