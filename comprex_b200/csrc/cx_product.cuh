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

// columns of a kStats tile
int cx_product_stat_columns(const CxProduct& p);
int64_t cx_product_workspace_bytes(const CxProduct& p);
int cx_product(const CxProduct& p, cudaStream_t s);

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

}  // namespace cxprod
