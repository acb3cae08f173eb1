// How a row of a 4-bit cache comes to its scale, factors and codes.
#pragma once
#include "attn_dev.cuh"

namespace vq2 {

// Maximum that a NaN passes through.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float reciprocal(float x) {   // off by 2^-22 at most, above 2^126 too
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// A 4-bit group's factor (e4m3, as a byte and as a number): its largest magnitude over the row's, rounded up so that
// no value passes 7 steps. 2^-9 at least unless the group is 0. `inverse`: of the row. A share of 2^-20 less keeps quotients that
// are such numbers from the next one; no other quotient of 16-bit values is within 2^-14 of one.
__device__ __forceinline__ uint32_t factor_of(float group, float inverse, float& u) {
  const float r = group * (inverse * (1.f - 1.f / 1048576.f));
  const uint32_t b = r >= 0.015625f * (1.f - 1.f / 1048576.f) ? ((__float_as_uint(r) + 0xfffffu) >> 20) - 960u
                                                              : max((uint32_t)ceilf(r * 512.f), (uint32_t)(group > 0.f));
  u = e4m3_value(b);
  return b;
}

// A group's factor, what turns its values into codes -7..7 (0: they are 0) and the row's scale, of the largest magnitudes of the
// group and the row. The code is the nearest integer to 7 x / (row * factor), a tie away from zero: a share of 2^-20 more
// lifts every tie, and no quotient of 16-bit values (a tie is 2^-16 away if it is not met) over it, the reciprocals' 2^-22 included;
// so one multiplication rounds as an exact division would. A row that is not finite has scale NaN (beside finite
// factors), one below 1e-30 is zeros.
__device__ __forceinline__ float quantiser4(float group, float row, uint32_t& byte, float& scale) {
  const bool bad = !(row < INFINITY);
  byte = bad ? 0x38u : 0u;
  scale = bad ? __uint_as_float(0x7fc00000u) : 0.f;
  if (bad || row < 1e-30f) return 0.f;
  float u;
  byte = factor_of(group, reciprocal(row), u);
  scale = row * (1.f / 7.f);
  scale = fmaf(fmaf(-7.f, scale, row), 1.f / 7.f, scale);   // a Newton step from the exact remainder: row / 7 rounded once
  return u == 0.f ? 0.f : reciprocal(row * u) * (7.f + 7.f / 1048576.f);
}

// The codes of 8 values, plus 8, value 0's in the low bits.
__device__ __forceinline__ uint32_t codes8(const float* f, float per) {
  uint32_t u[8];   // adding 1.5 * 2^23 + 8 rounds to an integer and leaves it in the low bits
#pragma unroll
  for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(fmaf(f[j], per, 12582920.f));
  const uint32_t even = __byte_perm(__byte_perm(u[0], u[2], 0x0040), __byte_perm(u[4], u[6], 0x0040), 0x5410);
  const uint32_t odd = __byte_perm(__byte_perm(u[1], u[3], 0x0040), __byte_perm(u[5], u[7], 0x0040), 0x5410);
  return (even & 0x0f0f0f0fu) | (odd & 0x0f0f0f0fu) << 4;
}

// Keys and values that need no turning into a 4-bit cache, and out of one (kv_cache4.cu).
int launch_store4(const PagedKV& kv, const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs,
                  bool half, int64_t tokens, int64_t D, cudaStream_t st);
int launch_load4(const PagedKV& kv, void* k, void* v, bool half, int64_t tokens, int64_t D, cudaStream_t st);

}  // namespace vq2
