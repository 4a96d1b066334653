// One element of an AdamW step, and how its 8-bit states are rounded: shared by the CUDA kernel and the host back end.
//
//   m = b1 m + (1 - b1) g     v = b2 v + (1 - b2) g^2     p = (1 - lr wd) p - lr / c1 * m / (sqrt(v / c2) + eps)
//
// (Decoupled weight decay; c1, c2 are the bias corrections.)  All of it in 32 bits; the moments without multiply-add
// contraction, so that both back ends have the same ones, bit for bit.
//
// States of 8 bits: a block of 256 elements keeps m and r = sqrt(v) as e4m3 numbers times a power of two per block,
// chosen so that the block's largest magnitude lies in [128, 256) (r: [128, 256)).  The root halves the range that the
// second moment needs: e4m3 holds 2^-9 .. 448, so r reaches 2^17 below the block's largest, v 2^34.  A moving average
// with b2 = 0.999 changes by less than a tenth of a percent per step, a step of e4m3 is 6 to 12 %: rounded to
// nearest, v would stay where it is for good, so both are rounded at random, up with a probability equal to the part
// that is cut off (16 random bits below the mantissa's end; below 2^-6, in the subnormals, what is left is rounded to
// nearest).  An r above zero stays above zero: an element never loses its denominator to the rounding.
#pragma once
#include <stdint.h>

#include "cx_ops.h"

#ifdef __CUDACC__
#define CX_HD __host__ __device__ __forceinline__
#else
#include <math.h>
#include <string.h>
#define CX_HD inline
#endif

namespace cxadam {

// Integer hash with the multipliers of Chris Wellons' search for low-bias 32-bit functions ("lowbias32", 2018).
CX_HD uint32_t mix(uint32_t v) {
  v = (v ^ (v >> 16)) * 0x7FEB352Du;
  v = (v ^ (v >> 15)) * 0x846CA68Bu;
  return v ^ (v >> 16);
}
// 32 random bits of a flat position: the lower half rounds m, the upper half r
CX_HD uint32_t random_bits(uint32_t place, uint32_t noise) { return mix(mix(place) + noise); }

// Biased exponent that a block's scale is made from: the one of the largest |m|, or of the root of the largest v.
// The scale is 2^(max(e, 8) - 134): largest / scale lies in [128, 256) and neither scale nor 1 / scale leaves the
// normal numbers (e <= 255).
CX_HD uint32_t root_exponent(uint32_t e) { return (uint32_t)(((int)e - 127) >> 1) + 127u; }
CX_HD uint32_t scale_bits(uint32_t e) { return ((e < 8 ? 8 : e) - 134 + 127) << 23; }
CX_HD uint32_t inverse_bits(uint32_t e) { return (134 - (e < 8 ? 8 : e) + 127) << 23; }

}  // namespace cxadam
