// AdamW step over all tensors of a model in one launch, states in 32 bits or in 8 (the mathematics: cx_adamw.h).
//
// An element moves its gradient, its 32-bit weight both ways, its 16-bit copy and two states both ways: 16 bytes for a bf16
// tensor with 8-bit states, 28 with 32-bit ones.  With 32 bits that bounds it (268 M elements bf16 / fp32 1146 / 1127 us, 6.6
// / 6.7 TB/s); with 8 it is instructions as well, 73 an element, 18 of them the random bits (830 / 803 us, 5.2 / 5.3 TB/s).  One warp takes one block of 256 elements at a time: the block is what shares a scale,
// so its largest values are two warp-wide integer maxima and nothing crosses warps, and a lane's two groups of four
// consecutive elements make every access of the warp whole lines.  Tensors are found through a table of blocks, so a model of
// many small tensors is one launch as well.
#include <cuda_fp8.h>

#include "cx_adamw.h"
#include "cx_device.cuh"

namespace {

constexpr int kThreads = 256;

// The hardware's reciprocal, 2^-23 off, one instruction instead of ten: the step that it makes is lr-sized.  The root is the
// exact one: what is kept of it is rounded at random, and must be the same whoever computes it (with an approximate root one
// code in 500 000 differed, and the weights a step later).
__device__ __forceinline__ float approx_inverse(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two products, sums or multiply-adds in one instruction, each rounded as one alone is
struct Two {
  unsigned long long w;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(w)); }
};
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.w) : "l"(a.w), "l"(b.w));
  return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return d;
}
// a b + c d as three roundings.  (The sum is one of single numbers: as two in one instruction it would be joined with a
// product into a multiply-add, and the moments would not be the host's.)
__device__ __forceinline__ void sum_of_products(Two a, Two b, Two c, Two d, float& x, float& y) {
  float p, q, r, s;
  (a * b).get(p, q);
  (c * d).get(r, s);
  x = __fadd_rn(p, r);
  y = __fadd_rn(q, s);
}
// The larger magnitude of three; NaN where one is
__device__ __forceinline__ float top3(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// |x| < 256 with 16 random bits under the mantissa's end: they are added below the sign, and what is below is cut off
__device__ __forceinline__ float cut(float x, uint32_t bits16) { return __uint_as_float((__float_as_uint(x) + (bits16 << 4)) & 0xFFF00000u); }
__device__ __forceinline__ uint32_t pack4(const float (&x)[4]) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
__device__ __forceinline__ void unpack4(uint32_t w, float (&x)[4]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
    const float2 f = __half22float2(__half2(r));
    x[2 * h] = f.x;
    x[2 * h + 1] = f.y;
  }
}

// four elements as they lie in memory, and what a lane holds of a block: elements 4 lane to 4 lane + 3 of both halves
template <typename T, bool EIGHT>
struct Loaded {
  typename cx::Raw4<T>::type g[2];
  float4 p[2];
  float4 m[EIGHT ? 1 : 2], v[EIGHT ? 1 : 2];
  uint32_t m8[2], v8[2];
};

template <typename T, bool EIGHT>
__global__ void __launch_bounds__(kThreads, EIGHT ? 4 : 2) adamw_kernel(const __grid_constant__ CxAdamW a, const int64_t run) {
  using Raw = cx::Raw4<T>;
  const int lane = threadIdx.x & 31;
  // A CTA takes `run` neighbouring blocks, mostly of one tensor, its warps in turn, then those of its next turn: all CTAs
  // together stay in a window of each array, and the tensors' tables are seldom read.  (355 M elements in 292 tensors, bf16,
  // 8 bits, runs of 8 / 32 / 128 / 512 blocks and one range a CTA: 1387 / 1233 / 1147 / 1096 / 1223 us; 268 M in one tensor
  // with 32 bits, 8 / 16 / 32 / 128: 1174 / 1137 / 1147 / 1185.)
  constexpr int64_t warps = kThreads / 32;
  // a tensor's row of the tables is read when a block of another tensor comes; which tensor that is, a block ahead
  int seg = 0, known = -1;
  const T* grad0 = nullptr;
  T* param0 = nullptr;
  int64_t first = 0, len = 0;
  int cls = 0;
  // With 8 bits the next block's lines are asked into L2 while this one is worked on, a lane has one of them: there are
  // more instructions then than 32 warps an SM hide the loads behind (268 M elements, bf16 / fp32: with it 8 / 1 % faster).
  // With 32 bits 16 warps without it are fastest (1150 / 1125 us; 24 warps 1259 / 1208, 32 warps with it 1450 / 1417).
  constexpr int kT = (int)sizeof(T) * 2, kState = EIGHT ? 2 : 8;           // lines of a block: of a tensor, of a state
  constexpr int kLines = kT + 8 + 2 * kState;                              // gradient, weights, two states
  const int part = lane < kT ? 0 : lane < kT + 8 ? 1 : lane < kT + 8 + kState ? 2 : 3;
  const int64_t per = part == 0 ? kT * 128 : part == 1 ? 1024 : kState * 128;
  const char* line = nullptr;
  for (int64_t turn = blockIdx.x; turn * run < a.blocks; turn += gridDim.x) {
    const int64_t last = min(a.blocks, (turn + 1) * run);
    int64_t b = turn * run + (threadIdx.x >> 5);
    if (b >= last) continue;
    seg = a.blk_seg[b];
    for (; b < last; b += warps) {
      if (seg != known) {
        known = seg;
        grad0 = reinterpret_cast<const T*>(a.seg_grad[seg]);
        param0 = reinterpret_cast<T*>(a.seg_param[seg]);
        first = a.seg_blk[seg];
        len = a.seg_len[seg];
        cls = a.seg_class[seg] - a.first_class;
        if ((uint32_t)cls >= CX_ADAMW_CLASSES) grad0 = nullptr;      // its settings are another launch's
        const char* base = part == 0 ? reinterpret_cast<const char*>(grad0) - first * per
                           : part == 1 ? (sizeof(T) == 4 ? reinterpret_cast<const char*>(param0) - first * per : reinterpret_cast<const char*>(a.master))
                           : reinterpret_cast<const char*>(part == 2 ? a.m : a.v);
        line = base + 128 * (part == 0 ? lane : part == 1 ? lane - kT : part == 2 ? lane - kT - 8 : lane - kT - 8 - kState);
      }
      if (b + warps < last) seg = a.blk_seg[b + warps];
      if (grad0 == nullptr) continue;
      if (EIGHT && lane < kLines && b + warps < last && seg == known && (b + warps - first + 1) * CX_ADAMW_BLOCK <= len)       // whole, and of this tensor
        asm volatile("prefetch.global.L2 [%0];" ::"l"(line + (b + warps) * per));
      const int64_t at = (b - first) * CX_ADAMW_BLOCK, flat = b * CX_ADAMW_BLOCK;
      const int left = (int)min((int64_t)CX_ADAMW_BLOCK, len - at);
      const T* grad = grad0 + at;
      T* param = param0 + at;
      constexpr uintptr_t kWide = 4 * sizeof(T) - 1;
      const bool wide = left == CX_ADAMW_BLOCK && (((uintptr_t)param | (uintptr_t)grad) & kWide) == 0;
      Loaded<T, EIGHT> in;
      const CxAdamWClass& c = a.cls[cls];
      // of what is kept, this much stays: with 8 bits times the scale, or its square (powers of two: the products with beta
      // are what they are without them)
      float keep_m = c.b1, keep_v = c.b2;
      if (EIGHT) {
        const float scale = a.v_scale[b];
        keep_m *= a.m_scale[b];
        keep_v *= scale * scale;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = h * 128 + lane * 4;
        if (wide) {
          in.g[h] = Raw::load(grad + e);
          if (sizeof(T) == 4) in.p[h] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(param) + e);
        } else {
          T g[4];
          float p[4] = {};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            g[k] = e + k < left ? grad[e + k] : cx::Elem<T>::from_f(0.f);
            if (sizeof(T) == 4 && e + k < left) p[k] = cx::Elem<T>::to_f(param[e + k]);
          }
          memcpy(&in.g[h], g, sizeof(g));
          in.p[h] = make_float4(p[0], p[1], p[2], p[3]);
        }
        if (sizeof(T) != 4) in.p[h] = *reinterpret_cast<const float4*>(a.master + flat + e);
        if (EIGHT) {
          in.m8[h] = reinterpret_cast<const uint32_t*>(a.m)[(flat + e) / 4];
          in.v8[h] = reinterpret_cast<const uint32_t*>(a.v)[(flat + e) / 4];
        } else {
          in.m[h] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.m) + flat + e);
          in.v[h] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.v) + flat + e);
        }
      }
      // the step; what is done with an element is stored at once, but for the states of 8 bits, which wait for their scale
      float m[2][4], root[2][4], most_m = 0.f, most_v = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = h * 128 + lane * 4;
        float g[4], p[4] = {in.p[h].x, in.p[h].y, in.p[h].z, in.p[h].w}, v[4];
        Raw::to_f(in.g[h], g);
        if (EIGHT) {
          unpack4(in.m8[h], m[h]);
          unpack4(in.v8[h], v);
#pragma unroll
          for (int k = 0; k < 4; k += 2) {                     // 4 bits squared: exact
            const Two r(v[k], v[k + 1]);
            (r * r).get(v[k], v[k + 1]);
          }
        } else {
          const float4 x = in.m[h], y = in.v[h];
          m[h][0] = x.x, m[h][1] = x.y, m[h][2] = x.z, m[h][3] = x.w;
          v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
        }
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const Two g2(g[k], g[k + 1]);
          sum_of_products(Two(m[h][k], m[h][k + 1]), Two(keep_m, keep_m), g2, Two(c.ob1, c.ob1), m[h][k], m[h][k + 1]);
          sum_of_products(Two(v[k], v[k + 1]), Two(keep_v, keep_v), g2 * Two(c.ob2, c.ob2), g2, v[k], v[k + 1]);
          const Two m2(m[h][k], m[h][k + 1]);
          root[h][k] = sqrtf(v[k]);
          root[h][k + 1] = sqrtf(v[k + 1]);
          float low0, low1;
          fma2(Two(root[h][k], root[h][k + 1]), Two(c.norm, c.norm), Two(c.eps, c.eps)).get(low0, low1);
          fma2(Two(p[k], p[k + 1]), Two(c.decay, c.decay), m2 * Two(-c.rate, -c.rate) * Two(approx_inverse(low0), approx_inverse(low1))).get(p[k], p[k + 1]);
        }
        if (EIGHT) {
          most_m = top3(most_m, m[h][0], top3(m[h][1], m[h][2], m[h][3]));
          most_v = top3(most_v, v[0], top3(v[1], v[2], v[3]));
        }
        if (wide) {
          if (sizeof(T) == 4) cx::store4(reinterpret_cast<float*>(param) + e, p);
          else cx::store4(param + e, p);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (e + k < left) param[e + k] = cx::Elem<T>::from_f(p[k]);
        }
        if (sizeof(T) != 4) cx::store4(a.master + flat + e, p);
        if (!EIGHT) {
          cx::store4(reinterpret_cast<float*>(a.m) + flat + e, m[h]);
          cx::store4(reinterpret_cast<float*>(a.v) + flat + e, v);
        }
      }
      if (!EIGHT) continue;
      const uint32_t top_m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most_m) & 0x7FFFFFFFu);
      const uint32_t top_v = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(most_v) & 0x7FFFFFFFu);
      const uint32_t e_m = top_m >> 23, e_v = cxadam::root_exponent(top_v >> 23);
      const bool fine = max(top_m, top_v) < 0x7F800000u;       // no element of the block is infinite or no number
      const float inv_m = __uint_as_float(cxadam::inverse_bits(e_m)), inv_v = __uint_as_float(cxadam::inverse_bits(e_v));
      if (lane == 0) {
        a.m_scale[b] = __uint_as_float(cxadam::scale_bits(e_m));
        a.v_scale[b] = __uint_as_float(cxadam::scale_bits(e_v));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = h * 128 + lane * 4;
        float qm[4], qv[4];
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          (Two(m[h][k], m[h][k + 1]) * Two(inv_m, inv_m)).get(qm[k], qm[k + 1]);
          (Two(root[h][k], root[h][k + 1]) * Two(inv_v, inv_v)).get(qv[k], qv[k + 1]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t bits = cxadam::random_bits((uint32_t)(flat + e + k), a.noise);
          qm[k] = cut(qm[k], bits & 0xFFFFu);
          const float q = fmaxf(cut(qv[k], bits >> 16), 0x1p-9f);
          qv[k] = root[h][k] == 0.f ? 0.f : q;                 // (only the root of zero is zero)
        }
        if (!fine) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (!(fabsf(m[h][k]) < INFINITY)) qm[k] = NAN;
            if (!(root[h][k] < INFINITY)) qv[k] = NAN;
          }
        }
        reinterpret_cast<uint32_t*>(a.m)[(flat + e) / 4] = pack4(qm);
        reinterpret_cast<uint32_t*>(a.v)[(flat + e) / 4] = pack4(qv);
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
  constexpr int64_t most = EIGHT ? 512 : 32;
  int64_t run = (a.blocks + grid - 1) / grid;
  run = run < most ? (run + 7) / 8 * 8 : most;
  adamw_kernel<T, EIGHT><<<grid, kThreads, 0, s>>>(a, run);
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
