// Element types on the host: conversions that agree bit for bit with the device's (round to nearest even).
#pragma once
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include "cx_common.h"

namespace {

inline float bf16_to_f(uint16_t h) {
  uint32_t u = (uint32_t)h << 16;
  float f;
  memcpy(&f, &u, 4);
  return f;
}
inline uint16_t f_to_bf16(float f) {
  uint32_t u;
  memcpy(&u, &f, 4);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);  // NaN
  const uint32_t lsb = (u >> 16) & 1u;
  u += 0x7fffu + lsb;
  return (uint16_t)(u >> 16);
}
inline float f16_to_f(uint16_t h) {
  const uint32_t sign = (uint32_t)(h & 0x8000u) << 16;
  uint32_t exp = (h >> 10) & 0x1fu, man = h & 0x3ffu, u;
  if (exp == 0) {
    if (man == 0) u = sign;
    else {
      exp = 127 - 15 + 1;
      while (!(man & 0x400u)) { man <<= 1; --exp; }
      u = sign | (exp << 23) | ((man & 0x3ffu) << 13);
    }
  } else if (exp == 31) u = sign | 0x7f800000u | (man << 13);
  else u = sign | ((exp + 127 - 15) << 23) | (man << 13);
  float f;
  memcpy(&f, &u, 4);
  return f;
}
inline uint16_t f_to_f16(float f) {
  uint32_t x;
  memcpy(&x, &f, 4);
  const uint32_t sign = (x >> 16) & 0x8000u;
  x &= 0x7fffffffu;
  if (x >= 0x7f800000u) return (uint16_t)(sign | 0x7c00u | (x > 0x7f800000u ? 0x200u : 0));
  if (x >= 0x477ff000u) return (uint16_t)(sign | 0x7c00u);  // rounds to inf
  if (x < 0x33000001u) return (uint16_t)sign;                // rounds to zero
  int exp = (int)(x >> 23) - 127 + 15;
  uint32_t man = x & 0x7fffffu;
  if (exp <= 0) {  // subnormal half
    man |= 0x800000u;
    const int shift = 14 - exp;
    uint32_t half = man >> shift;
    const uint32_t rem = man & ((1u << shift) - 1), mid = 1u << (shift - 1);
    if (rem > mid || (rem == mid && (half & 1))) ++half;
    return (uint16_t)(sign | half);
  }
  uint32_t half = ((uint32_t)exp << 10) | (man >> 13);
  const uint32_t rem = man & 0x1fffu;
  if (rem > 0x1000u || (rem == 0x1000u && (half & 1))) ++half;
  return (uint16_t)(sign | half);
}

inline float load_elem(int dtype, const void* p, int64_t i) {
  switch (dtype) {
    case CX_F32: return reinterpret_cast<const float*>(p)[i];
    case CX_BF16: return bf16_to_f(reinterpret_cast<const uint16_t*>(p)[i]);
    default: return f16_to_f(reinterpret_cast<const uint16_t*>(p)[i]);
  }
}
inline void store_elem(int dtype, void* p, int64_t i, float v) {
  switch (dtype) {
    case CX_F32: reinterpret_cast<float*>(p)[i] = v; break;
    case CX_BF16: reinterpret_cast<uint16_t*>(p)[i] = f_to_bf16(v); break;
    default: reinterpret_cast<uint16_t*>(p)[i] = f_to_f16(v); break;
  }
}
inline size_t elem_size(int dtype) { return dtype == CX_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == CX_F32 || dtype == CX_BF16 || dtype == CX_F16; }

}  // namespace
