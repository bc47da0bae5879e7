// Signed 8-bit rows with one fp32 scale each: the quantiser shared by the row
// kernels and by the transform's epilogue. Nothing here is part of the public C ABI.
//
// A row v is held as s = fp32(max|v| / 127) and q_i = v_i / s rounded to the
// nearest integer, ties to even. The rounding is decided on the exact quotient,
// not on its fp32 neighbour: n = rint(v * (1/s)) is off by at most one, and the
// residual v - n*s is exact in one fused multiply-add (|v - n*s| <= s, a multiple
// of the smaller of both units in the last place), so comparing it with s/2
// settles the integer. A row of zeros, or one whose scale underflows, has s = 0
// and q = 0; a row that holds a NaN or an infinity has s = NaN and q = 0, so that
// whatever is computed from it is NaN.
#pragma once

#include <stdint.h>

namespace gnnb200 {

// max(a, |b|), NaN if either is
__device__ __forceinline__ float max_abs_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}

struct RowQuant {
  float s;     // the scale that is stored
  float sw;    // the scale, times 2^80 where it is tiny, so that it is a normal number
  float inv;   // 1 / sw
  float half;  // sw / 2
  bool tiny;
  uint32_t mask;  // 0 where q = 0 throughout
};

__device__ __forceinline__ RowQuant row_quant(float amax) {
  RowQuant r;
  const bool bad = !(amax < __int_as_float(0x7f800000));  // infinity or NaN
  r.s = bad ? __int_as_float(0x7fffffff) : __fdiv_rn(amax, 127.0f);
  const bool none = bad || r.s == 0.0f;
  r.mask = none ? 0u : 0xffffffffu;
  r.tiny = !none && r.s < 0x1p-60f;
  r.sw = none ? 1.0f : (r.tiny ? r.s * 0x1p80f : r.s);
  r.inv = __frcp_rn(r.sw);
  r.half = 0.5f * r.sw;
  return r;
}

constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23: adding it leaves the rounded integer in the low bits

// Four values of a row as four bytes.
__device__ __forceinline__ uint32_t quant4(const RowQuant& r, float a, float b, float c, float d) {
  float v[4] = {a, b, c, d};
  if (r.tiny) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= 0x1p80f;
  }
  float t[4], e[4];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t[i] = __fmaf_rn(v[i], r.inv, kRoundMagic);
    e[i] = __fmaf_rn(-__fsub_rn(t[i], kRoundMagic), r.sw, v[i]);  // exact residual
    near |= fabsf(e[i]) >= r.half;
  }
  if (near || r.tiny) {  // at or beyond a border: ties go to the even neighbour
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float f = fabsf(e[i]);
      if (f > r.half || (f == r.half && (__float_as_int(t[i]) & 1))) t[i] = __fadd_rn(t[i], copysignf(1.0f, e[i]));
      // a subnormal scale can be so coarse that the row's largest value lies past 127 steps
      t[i] = fminf(fmaxf(t[i], kRoundMagic - 127.0f), kRoundMagic + 127.0f);
    }
  }
  const uint32_t lo = __byte_perm(__float_as_uint(t[0]), __float_as_uint(t[1]), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(t[2]), __float_as_uint(t[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410) & r.mask;
}

__device__ __forceinline__ int8_t quant1(const RowQuant& r, float a) {
  return static_cast<int8_t>(quant4(r, a, 0.0f, 0.0f, 0.0f) & 0xffu);
}

}  // namespace gnnb200
