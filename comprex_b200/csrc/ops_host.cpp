// Host back end of the operators of cx_ops.h: the same formulas as the kernels, element by element.
#include <math.h>

#include <algorithm>
#include <vector>

#include "cx_adamw.h"
#include "cx_host_elem.h"
#include "cx_ops.h"

int cx_set_error(const char* where, int cuda_err);

namespace {

inline uint32_t bits_of(float x) {
  uint32_t u;
  memcpy(&u, &x, 4);
  return u;
}
inline float float_of(uint32_t u) {
  float x;
  memcpy(&x, &u, 4);
  return x;
}

// e4m3: 4 bits of exponent (bias 7), 3 of mantissa, no infinities, 0x7F is NaN
inline float e4m3_to_f(uint8_t c) {
  const int e = (c >> 3) & 15, man = c & 7;
  float x = e ? ldexpf((float)(8 + man), e - 10) : ldexpf((float)man, -9);
  if ((c & 0x7F) == 0x7F) x = NAN;
  return c & 0x80 ? -x : x;
}
// of a number below 448 with at most 3 bits of mantissa, or NaN
inline uint8_t f_to_e4m3(float x) {
  const uint8_t sign = (uint8_t)(bits_of(x) >> 31 << 7);
  if (x != x) return sign | 0x7F;
  x = fabsf(x);
  if (x < 0x1p-6f) return sign | (uint8_t)nearbyintf(x * 512.f);
  return sign | (uint8_t)((bits_of(x) >> 20) - (120u << 3));
}
inline float cut(float x, uint32_t bits16) {
  const uint32_t raw = bits_of(x) & 0x7FFFFFFFu;
  return raw < 0x7F800000u ? float_of(((raw + (bits16 << 4)) & ~0xFFFFFu) | (bits_of(x) & 0x80000000u)) : NAN;
}

}  // namespace

int cx_adamw_step_host(const CxAdamW* a) {
  std::vector<float> m(CX_ADAMW_BLOCK), v(CX_ADAMW_BLOCK), root(CX_ADAMW_BLOCK);
  for (int64_t b = 0; b < a->blocks; ++b) {
    const int32_t seg = a->blk_seg[b];
    const void* grad = a->seg_grad[seg];
    if (!grad) continue;
    const CxAdamWClass& c = a->cls[a->seg_class[seg]];
    const int64_t at = (b - a->seg_blk[seg]) * CX_ADAMW_BLOCK, flat = b * CX_ADAMW_BLOCK;
    const int left = (int)std::min<int64_t>(CX_ADAMW_BLOCK, a->seg_len[seg] - at);
    uint32_t top_m = 0, top_v = 0;
    uint8_t *m8 = reinterpret_cast<uint8_t*>(a->m) + flat, *v8 = reinterpret_cast<uint8_t*>(a->v) + flat;
    float *m32 = reinterpret_cast<float*>(a->m) + flat, *v32 = reinterpret_cast<float*>(a->v) + flat;
    for (int e = 0; e < left; ++e) {
      if (a->bits == 8) {
        m[e] = e4m3_to_f(m8[e]) * a->m_scale[b];
        v[e] = e4m3_to_f(v8[e]) * a->v_scale[b];
        v[e] *= v[e];
      } else {
        m[e] = m32[e];
        v[e] = v32[e];
      }
      const float g = load_elem(a->dtype, grad, at + e);
      float p = a->master ? a->master[flat + e] : load_elem(a->dtype, a->seg_param[seg], at + e);
      m[e] = m[e] * c.b1 + g * c.ob1;
      v[e] = v[e] * c.b2 + (g * c.ob2) * g;
      root[e] = sqrtf(v[e]);
      p = p * c.decay - (m[e] * c.rate) / (root[e] * c.norm + c.eps);
      if (a->master) a->master[flat + e] = p;
      store_elem(a->dtype, a->seg_param[seg], at + e, p);
      top_m = std::max(top_m, bits_of(m[e]) & 0x7FFFFFFFu);
      top_v = std::max(top_v, bits_of(v[e]) & 0x7FFFFFFFu);
    }
    if (a->bits == 8) {
      const uint32_t e_m = top_m >> 23, e_v = cxadam::root_exponent(top_v >> 23);
      const float inv_m = float_of(cxadam::inverse_bits(e_m)), inv_v = float_of(cxadam::inverse_bits(e_v));
      a->m_scale[b] = float_of(cxadam::scale_bits(e_m));
      a->v_scale[b] = float_of(cxadam::scale_bits(e_v));
      for (int e = 0; e < left; ++e) {
        const uint32_t bits = cxadam::random_bits((uint32_t)(flat + e), a->noise);
        m8[e] = f_to_e4m3(cut(m[e] * inv_m, bits & 0xFFFFu));
        const float q = cut(root[e] * inv_v, bits >> 16);
        v8[e] = f_to_e4m3(v[e] == 0.f ? 0.f : q < 0x1p-9f ? 0x1p-9f : q);
      }
    } else {
      for (int e = 0; e < left; ++e) {
        m32[e] = m[e];
        v32[e] = v[e];
      }
    }
  }
  return 0;
}
