// AdamW step over all tensors of a model in one launch, states in 32 bits or in 8 (the mathematics: cx_adamw.h).
//
// Bound by memory: an element moves its gradient, its 32-bit weight both ways, its 16-bit copy and two states both
// ways, 16 bytes for a bf16 tensor with 8-bit states and 28 with 32-bit ones.  One warp takes one block of 256
// elements at a time: the block is what shares a scale, so its largest values are two warp-wide integer maxima and
// nothing crosses warps, and a lane's two groups of four consecutive elements make every access of the warp whole
// lines.  Tensors are found through a table of blocks, so a model of many small tensors is one launch as well.
#include <cuda_fp8.h>

#include "cx_adamw.h"
#include "cx_device.cuh"

namespace {

constexpr int kThreads = 256;

struct State4 {
  float p[4], m[4], v[4];
};

__device__ __forceinline__ void step1(const CxAdamWClass& c, float g, float& p, float& m, float& v, float& root) {
  m = m * c.b1 + g * c.ob1;
  v = v * c.b2 + (g * c.ob2) * g;
  root = sqrtf(v);
  p = p * c.decay - (m * c.rate) / (root * c.norm + c.eps);
}

// |x| < 256 with 16 random bits under the mantissa's end: they are added below the sign, and what is below is cut off
__device__ __forceinline__ float cut(float x, uint32_t bits16) { return __uint_as_float((__float_as_uint(x) + (bits16 << 4)) & 0xFFF00000u); }
__device__ __forceinline__ uint32_t pack4(const float (&x)[4]) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
__device__ __forceinline__ void unpack4(uint32_t w, float scale, float (&x)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
    const float2 f = __half22float2(__half2(r));
    x[2 * h] = f.x * scale;
    x[2 * h + 1] = f.y * scale;
  }
}

template <typename T, bool EIGHT>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ CxAdamW a) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t b = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); b < a.blocks; b += warps) {
    const int seg = a.blk_seg[b];
    const T* grad = reinterpret_cast<const T*>(a.seg_grad[seg]);
    if (grad == nullptr) continue;
    const CxAdamWClass& c = a.cls[a.seg_class[seg]];
    const int64_t at = (b - a.seg_blk[seg]) * CX_ADAMW_BLOCK;          // in the tensor
    const int64_t flat = b * CX_ADAMW_BLOCK;
    const int left = (int)min((int64_t)CX_ADAMW_BLOCK, a.seg_len[seg] - at);
    T* param = reinterpret_cast<T*>(a.seg_param[seg]) + at;
    grad += at;
    constexpr uintptr_t kWide = 4 * sizeof(T) - 1;
    const bool wide = left == CX_ADAMW_BLOCK && (((uintptr_t)param | (uintptr_t)grad) & kWide) == 0;
    float scale_m = 0.f, scale_v = 0.f;
    if (EIGHT) {
      scale_m = a.m_scale[b];
      scale_v = a.v_scale[b];
    }
    State4 s[2];
    float g[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = h * 128 + lane * 4;
      if (wide) {
        cx::load4(grad + e, g[h]);
        if (sizeof(T) == 4) cx::load4(reinterpret_cast<const float*>(param) + e, s[h].p);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          g[h][k] = e + k < left ? cx::Elem<T>::to_f(grad[e + k]) : 0.f;
          if (sizeof(T) == 4) s[h].p[k] = e + k < left ? cx::Elem<T>::to_f(param[e + k]) : 0.f;
        }
      }
      if (sizeof(T) != 4) cx::load4(a.master + flat + e, s[h].p);
      if (EIGHT) {
        unpack4(reinterpret_cast<const uint32_t*>(a.m)[(flat + e) / 4], scale_m, s[h].m);
        unpack4(reinterpret_cast<const uint32_t*>(a.v)[(flat + e) / 4], scale_v, s[h].v);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[h].v[k] *= s[h].v[k];
      } else {
        cx::load4(reinterpret_cast<const float*>(a.m) + flat + e, s[h].m);
        cx::load4(reinterpret_cast<const float*>(a.v) + flat + e, s[h].v);
      }
    }
    float root[2][4];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        step1(c, g[h][k], s[h].p[k], s[h].m[k], s[h].v[k], root[h][k]);
        if (EIGHT) {
          top_m = max(top_m, __float_as_uint(s[h].m[k]) & 0x7FFFFFFFu);
          top_v = max(top_v, __float_as_uint(s[h].v[k]) & 0x7FFFFFFFu);
        }
      }
    float inv_m = 0.f, inv_v = 0.f;
    bool fine = true;                     // no element of the block is infinite or no number
    if (EIGHT) {
      top_m = __reduce_max_sync(0xFFFFFFFFu, top_m);
      top_v = __reduce_max_sync(0xFFFFFFFFu, top_v);
      const uint32_t e_m = top_m >> 23, e_v = cxadam::root_exponent(top_v >> 23);
      fine = max(top_m, top_v) < 0x7F800000u;
      inv_m = __uint_as_float(cxadam::inverse_bits(e_m));
      inv_v = __uint_as_float(cxadam::inverse_bits(e_v));
      if (lane == 0) {
        a.m_scale[b] = __uint_as_float(cxadam::scale_bits(e_m));
        a.v_scale[b] = __uint_as_float(cxadam::scale_bits(e_v));
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = h * 128 + lane * 4;
      if (wide) {
        if (sizeof(T) == 4) cx::store4(reinterpret_cast<float*>(param) + e, s[h].p);
        else cx::store4(param + e, s[h].p);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (e + k < left) param[e + k] = cx::Elem<T>::from_f(s[h].p[k]);
      }
      if (sizeof(T) != 4) cx::store4(a.master + flat + e, s[h].p);
      if (EIGHT) {
        float qm[4], qv[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t bits = cxadam::random_bits((uint32_t)(flat + e + k), a.noise);
          qm[k] = cut(s[h].m[k] * inv_m, bits & 0xFFFFu);
          const float q = fmaxf(cut(root[h][k] * inv_v, bits >> 16), 0x1p-9f);
          qv[k] = s[h].v[k] == 0.f ? 0.f : q;
        }
        if (!fine) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (!(fabsf(s[h].m[k]) < INFINITY)) qm[k] = NAN;
            if (!(s[h].v[k] < INFINITY)) qv[k] = NAN;
          }
        }
        reinterpret_cast<uint32_t*>(a.m)[(flat + e) / 4] = pack4(qm);
        reinterpret_cast<uint32_t*>(a.v)[(flat + e) / 4] = pack4(qv);
      } else {
        cx::store4(reinterpret_cast<float*>(a.m) + flat + e, s[h].m);
        cx::store4(reinterpret_cast<float*>(a.v) + flat + e, s[h].v);
      }
    }
  }
}

template <typename T, bool EIGHT>
int launch(const CxAdamW& a, cudaStream_t s) {
  static const int per_sm = [] {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, adamw_kernel<T, EIGHT>, kThreads, 0) != cudaSuccess || n < 1) n = 4;
    return n;
  }();
  const int64_t ctas = (a.blocks + kThreads / 32 - 1) / (kThreads / 32);
  const int grid = (int)(ctas < (int64_t)per_sm * cx_sm_count() ? ctas : (int64_t)per_sm * cx_sm_count());
  adamw_kernel<T, EIGHT><<<grid, kThreads, 0, s>>>(a);
  cx_note_launch();
  return cx_check_launch("cx_adamw_step");
}

}  // namespace

int cx_adamw_step_cuda(const CxAdamW* a, void* stream) {
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->bits == 8) {
    if (a->dtype == CX_F32) return launch<float, true>(*a, s);
    if (a->dtype == CX_BF16) return launch<__nv_bfloat16, true>(*a, s);
    return launch<__half, true>(*a, s);
  }
  if (a->dtype == CX_F32) return launch<float, false>(*a, s);
  if (a->dtype == CX_BF16) return launch<__nv_bfloat16, false>(*a, s);
  return launch<__half, false>(*a, s);
}
