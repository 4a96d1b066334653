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
    const uint32_t row = (uint32_t)(a->seg_class[seg] - a->first_class);
    if (!grad || row >= CX_ADAMW_CLASSES) continue;      // (of another call)
    const CxAdamWClass& c = a->cls[row];
    const int64_t at = (b - a->seg_blk[seg]) * CX_ADAMW_BLOCK, flat = b * CX_ADAMW_BLOCK;
    const int left = (int)std::min<int64_t>(CX_ADAMW_BLOCK, a->seg_len[seg] - at);
    uint32_t top_m = 0, top_v = 0;
    uint8_t *m8 = reinterpret_cast<uint8_t*>(a->m) + flat, *v8 = reinterpret_cast<uint8_t*>(a->v) + flat;
    float *m32 = reinterpret_cast<float*>(a->m) + flat, *v32 = reinterpret_cast<float*>(a->v) + flat;
    for (int e = 0; e < left; ++e) {
      // with 8 bits what is kept is a power of two times what is stored: it goes with beta, as in the kernel
      float keep_m = c.b1, keep_v = c.b2;
      if (a->bits == 8) {
        m[e] = e4m3_to_f(m8[e]);
        v[e] = e4m3_to_f(v8[e]);
        v[e] *= v[e];
        keep_m *= a->m_scale[b];
        keep_v *= a->v_scale[b] * a->v_scale[b];
      } else {
        m[e] = m32[e];
        v[e] = v32[e];
      }
      const float g = load_elem(a->dtype, grad, at + e);
      float p = a->master ? a->master[flat + e] : load_elem(a->dtype, a->seg_param[seg], at + e);
      m[e] = m[e] * keep_m + g * c.ob1;
      v[e] = v[e] * keep_v + (g * c.ob2) * g;
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

// ---- linear -----------------------------------------------------------------------------------------------------
namespace {

float sigmoid_host(float z) {
  const float t = expf(-fabsf(z));
  return (z >= 0.f ? 1.f : t) / (1.f + t);
}
float act_host(float u, int act, float* slope) {
  const float k = 1.5957691216057308f;      // 2 sqrt(2 / pi)
  switch (act) {
    case CX_ACT_RELU:
      *slope = u > 0.f ? 1.f : 0.f;
      return u > 0.f || u != u ? u : 0.f;
    case CX_ACT_GELU: {
      const float cdf = 0.5f * (1.f + erff(u * 0.70710678118654752f));
      *slope = cdf + u * 0.39894228040143268f * expf(-0.5f * u * u);
      return u * cdf;
    }
    case CX_ACT_GELU_TANH: {
      const float q = sigmoid_host(u * (0.044715f * k * (u * u) + k));
      *slope = q + u * q * (1.f - q) * k * (0.134145f * (u * u) + 1.f);
      return u * q;
    }
    case CX_ACT_SILU: {
      const float q = sigmoid_host(u);
      *slope = q * (1.f + u * (1.f - q));
      return u * q;
    }
    default:
      *slope = 1.f;
      return u;
  }
}

std::vector<float> widen(int dtype, const void* p, int64_t rows, int64_t cols, int64_t ld) {
  std::vector<float> out((size_t)(rows * cols));
  for (int64_t r = 0; r < rows; ++r)
    for (int64_t c = 0; c < cols; ++c) out[(size_t)(r * cols + c)] = load_elem(dtype, p, r * ld + c);
  return out;
}
// out[c] += sum over i of a[i] b[i][c]  (also where a[i] is zero: b may be no number)
void add_product(const float* a, const float* b, float* out, int64_t inner, int64_t cols) {
  for (int64_t i = 0; i < inner; ++i)
    for (int64_t c = 0; c < cols; ++c) out[c] += a[i] * b[i * cols + c];
}
float dot(const float* a, const float* b, int64_t n) {
  float sum = 0.f;
  for (int64_t i = 0; i < n; ++i) sum += a[i] * b[i];
  return sum;
}

}  // namespace

int cx_linear_forward_host(const CxLinear* l) {
  const std::vector<float> x = widen(l->dtype, l->x, l->rows, l->inner, l->ldx), w = widen(l->dtype, l->w, l->outer, l->inner, l->ldw);
  for (int64_t r = 0; r < l->rows; ++r)
    for (int64_t c = 0; c < l->outer; ++c) {
      float u = dot(&x[(size_t)(r * l->inner)], &w[(size_t)(c * l->inner)], l->inner), slope;
      if (l->bias) u += load_elem(l->dtype, l->bias, c);
      if (l->pre) store_elem(l->dtype, l->pre, r * l->ldpre + c, u);
      u = act_host(u, l->act, &slope);
      if (l->residual) u += load_elem(l->dtype, l->residual, r * l->ldr + c);
      store_elem(l->dtype, l->y, r * l->outer + c, u);
    }
  return 0;
}

int cx_linear_backward_host(const CxLinear* l) {
  std::vector<float> du = widen(l->dtype, l->grad, l->rows, l->outer, l->ldg), sum((size_t)l->outer);
  for (int64_t r = 0; r < l->rows; ++r)
    for (int64_t c = 0; c < l->outer; ++c) {
      float& d = du[(size_t)(r * l->outer + c)];
      float slope = 1.f;
      if (l->act != CX_ACT_NONE) act_host(load_elem(l->dtype, l->pre, r * l->ldpre + c), l->act, &slope);
      d *= slope;
      sum[(size_t)c] += d;
    }
  if (l->dbias)
    for (int64_t c = 0; c < l->outer; ++c) store_elem(l->dtype, l->dbias, c, sum[(size_t)c]);
  std::vector<float> row((size_t)l->inner);
  if (l->dx) {
    const std::vector<float> w = widen(l->dtype, l->w, l->outer, l->inner, l->ldw);
    for (int64_t r = 0; r < l->rows; ++r) {
      std::fill(row.begin(), row.end(), 0.f);
      add_product(&du[(size_t)(r * l->outer)], w.data(), row.data(), l->outer, l->inner);
      for (int64_t i = 0; i < l->inner; ++i) store_elem(l->dtype, l->dx, r * l->inner + i, row[(size_t)i]);
    }
  }
  if (l->dw) {
    const std::vector<float> x = widen(l->dtype, l->x, l->rows, l->inner, l->ldx);
    for (int64_t c = 0; c < l->outer; ++c) {
      std::fill(row.begin(), row.end(), 0.f);
      for (int64_t r = 0; r < l->rows; ++r) add_product(&du[(size_t)(r * l->outer + c)], &x[(size_t)(r * l->inner)], row.data(), 1, l->inner);
      for (int64_t i = 0; i < l->inner; ++i) store_elem(l->dtype, l->dw, c * l->inner + i, row[(size_t)i]);
    }
  }
  return 0;
}

// ---- loss over a vocabulary ---------------------------------------------------------------------------------------
int cx_vocab_loss_forward_host(const CxVocabLoss* l) {
  const std::vector<float> h = widen(l->dtype, l->h, l->rows, l->dim, l->ldh), w = widen(l->dtype, l->w, l->vocab, l->dim, l->ldw);
  std::vector<float> s((size_t)l->vocab);
  float sum = 0.f, count = 0.f;
  for (int64_t r = 0; r < l->rows; ++r) {
    const int64_t t = l->targets[r];
    float top = -INFINITY, z = 0.f;
    for (int64_t v = 0; v < l->vocab; ++v) {
      s[(size_t)v] = dot(&h[(size_t)(r * l->dim)], &w[(size_t)(v * l->dim)], l->dim);
      if (s[(size_t)v] > top || s[(size_t)v] != s[(size_t)v]) top = s[(size_t)v];
    }
    for (int64_t v = 0; v < l->vocab; ++v) z += expf(s[(size_t)v] - top);
    const bool ignored = t == l->ignore_index, inside = t >= 0 && t < l->vocab;
    l->lse[r] = !ignored && !inside ? NAN : top + logf(z);
    const float loss = ignored ? 0.f : inside ? l->lse[r] - s[(size_t)t] : NAN;
    if (l->reduction == CX_REDUCE_NONE) l->loss[r] = loss;
    sum += loss;
    count += ignored ? 0.f : 1.f;
  }
  *l->count = count;
  if (l->reduction != CX_REDUCE_NONE) *l->loss = l->reduction == CX_REDUCE_MEAN ? sum / count : sum;
  return 0;
}

int cx_vocab_loss_backward_host(const CxVocabLoss* l) {
  const std::vector<float> h = widen(l->dtype, l->h, l->rows, l->dim, l->ldh), w = widen(l->dtype, l->w, l->vocab, l->dim, l->ldw);
  std::vector<float> p((size_t)l->vocab), dh((size_t)l->dim), dw((size_t)(l->vocab * l->dim));
  for (int64_t r = 0; r < l->rows; ++r) {
    const int64_t t = l->targets[r];
    float g = l->grad[l->reduction == CX_REDUCE_NONE ? r * l->grad_stride : 0];
    if (l->reduction == CX_REDUCE_MEAN) g /= *l->count;
    if (t == l->ignore_index) g = 0.f;
    const float* hr = &h[(size_t)(r * l->dim)];
    std::fill(dh.begin(), dh.end(), 0.f);
    if (g != 0.f) {
      for (int64_t v = 0; v < l->vocab; ++v)
        p[(size_t)v] = (expf(dot(hr, &w[(size_t)(v * l->dim)], l->dim) - l->lse[r]) - (v == t ? 1.f : 0.f)) * g;
      add_product(p.data(), w.data(), dh.data(), l->vocab, l->dim);
      if (l->dw)
        for (int64_t v = 0; v < l->vocab; ++v) add_product(&p[(size_t)v], hr, &dw[(size_t)(v * l->dim)], 1, l->dim);
    }
    if (l->dh)
      for (int64_t i = 0; i < l->dim; ++i) store_elem(l->dtype, l->dh, r * l->dim + i, dh[(size_t)i]);
  }
  if (l->dw)
    for (int64_t i = 0; i < l->vocab * l->dim; ++i) store_elem(l->dtype, l->dw, i, dw[(size_t)i]);
  return 0;
}
