// Symmetric 8-bit codes of 16-bit values: code = rint(127 x / top), ties to even, correctly rounded; top = max|x| of the row.
//
// The largest magnitude is found on the bit patterns (16-bit floats order like their magnitude bits; infinities and NaN come
// out as patterns from the infinity's upwards).
//
// The code is found without a division per value.  r = fl(127 / top) and v = fl(x r) are within 2^-23 of the exact quotient q
// (relative).  127 x is a whole number of at most 18 bits times a power of two and top one of at most 11 bits, so a q that is
// no tie (no odd multiple of 1/2) differs from every tie by at least 1 / (254 * 2047) > 2^-19 of itself.  v cut to 20
// significant bits (Veltkamp's splitting, round to nearest) is therefore the tie itself where q is one - ties have 8 bits - and
// stays strictly on q's side of it where q is not: half a unit of 20 bits is at most 2^-20 of q.  Rounding it to an integer
// gives q's own code.
#pragma once
#include "dense.cuh"

namespace dense {

__device__ __forceinline__ uint32_t magnitude_max(uint32_t top2, uint4 v) {   // two running maxima, low and high half
  top2 = __vmaxu2(top2, v.x & 0x7fff7fffu);
  top2 = __vmaxu2(top2, v.y & 0x7fff7fffu);
  top2 = __vmaxu2(top2, v.z & 0x7fff7fffu);
  return __vmaxu2(top2, v.w & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t magnitude_join(uint32_t top2) { return max(top2 & 0xffffu, top2 >> 16); }

struct RowScale {
  float scale;     // what a code step stands for: top / 127, or NaN for a row with an infinity or a NaN
  float r;         // 127 / top; 0 where all codes are 0
  float up;        // rows of tiny values are scaled by a power of two first, so that r stays finite
};
__device__ __forceinline__ RowScale row_scale(uint32_t top_bits, bool bf16) {
  const bool odd = top_bits >= (bf16 ? 0x7f80u : 0x7c00u);
  const float top = unpack16(top_bits, bf16);
  RowScale s;
  s.scale = odd ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 127.f);
  s.up = top < 0x1p-100f ? 0x1p64f : 1.f;
  s.r = (odd || top == 0.f) ? 0.f : __fdiv_rn(127.f, top * s.up);
  return s;
}
// The code in the lowest byte (two's complement); x * up, r of the row.  A row without codes has r = 0 and may hold anything.
__device__ __forceinline__ uint32_t code_bits(float x, float r) {
  const float v = __fmul_rn(x, r);
  const float c = __fmul_rn(v, 17.f);
  const float cut = __fsub_rn(c, __fsub_rn(c, v));
  return __float_as_uint(__fadd_rn(cut, 12582912.f));   // 1.5 * 2^23: the sum's unit is 1
}
__device__ __forceinline__ uint2 codes8(uint4 v, const RowScale& s, bool bf16) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float lo, hi;
    if (bf16) {
      lo = __uint_as_float(w[j] << 16), hi = __uint_as_float(w[j] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      lo = f.x, hi = f.y;
    }
    if (s.up != 1.f) lo *= s.up, hi *= s.up;
    c[2 * j] = code_bits(lo, s.r), c[2 * j + 1] = code_bits(hi, s.r);
  }
  uint2 o;
  o.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
  o.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  return s.r == 0.f ? make_uint2(0u, 0u) : o;
}

}  // namespace dense
