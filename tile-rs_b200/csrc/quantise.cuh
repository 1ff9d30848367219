// Rows of f32 as whole numbers of steps of their largest magnitude: step = max|x| * (1/127), q = x / step rounded to nearest even (the quotient in f32).  A row with an
// infinity, or with a NaN if the largest is taken with fmax_nan, has a step of NaN, and so has q * step all along.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace tsm100 {
namespace quant {

struct Step {
  float step, inv;
};
__device__ __forceinline__ Step step_of(float top) {
  Step s;
  s.step = top * static_cast<float>(1.0 / 127.0);
  // among the smallest numbers, where a step is a few times 2^-149, the nearest one may be too short for the largest x (190 over 1) or be 0: the next one then
  if (s.step < 0x1p-120f && 255.f * s.step <= 2.f * top && top > 0.f) s.step = __uint_as_float(__float_as_uint(s.step) + 1u);
  if (top == INFINITY) s.step = __uint_as_float(0x7fffffffu);
  // 0 for a row of zeros; NaN where the reciprocal is no use (far from 1, not finite): every number then takes the division
  s.inv = top == 0.f ? 0.f : s.step >= 0x1p-120f && s.step <= 0x1p120f ? 1.f / s.step : __uint_as_float(0x7fffffffu);
  return s;
}
// Four numbers as bytes.  A product with the reciprocal is within 4e-5 of the quotient, so both round alike unless that ends near a half; only then is it divided
// (a tenth of the warps; dividing always, the norm of 8192 x 4096 took 45 us, this way 36).  Adding 1.5 * 2^23 rounds to nearest
// even and leaves the number in the low byte.
__device__ __forceinline__ uint32_t quantise4(const float* x, const Step& s) {
  constexpr float kMagic = 12582912.f;
  float u[4];
  bool divide = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = x[i] * s.inv;
    u[i] = t + kMagic;
    divide |= !(fabsf(t - (u[i] - kMagic)) <= 0.4999f);
  }
  if (divide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = x[i] / s.step + kMagic;
  }
  const uint32_t lo = __byte_perm(__float_as_uint(u[0]), __float_as_uint(u[1]), 0x0040), hi = __byte_perm(__float_as_uint(u[2]), __float_as_uint(u[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// Byte i of x, a whole number, as f32: behind 0x4b0000 it is 2^23 + 128 + q.
__device__ __forceinline__ float number(uint32_t x, int i) {
  return __uint_as_float(__byte_perm(x ^ 0x80808080u, 0x4b000000u, 0x7540 + i)) - 8388736.f;
}

// Two of the four whole numbers of x, bytes 0 and 1 (or 2 and 3: `upper`), as 16-bit numbers, exactly.  f16: a byte behind 0x64 is 1024 + byte.  bf16: 128 and the lower
// seven bits, less 128, or 256 where the sign is set.
template <bool kIsBf16>
__device__ __forceinline__ uint32_t pair_of(uint32_t x, bool upper) {
  uint32_t r;
  if (kIsBf16) {
    const uint32_t h = __byte_perm(x, 0u, upper ? 0x4342 : 0x4140);
    uint32_t a, b;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(a) : "r"(h), "r"(0x007f007fu), "r"(0x43004300u));
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(b) : "r"(h), "r"(0x00800080u), "r"(0x43004300u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    const uint32_t h = __byte_perm(x ^ 0x80808080u, 0x64646464u, upper ? 0x4342 : 0x4140);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));
  }
  return r;
}

}  // namespace quant
}  // namespace tsm100
