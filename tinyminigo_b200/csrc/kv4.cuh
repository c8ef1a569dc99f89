// The 4-bit KV cache: its layout and the arithmetic of one group.
//
// A cache row (stream m, kv head h, position p) holds head_dim codes of 4
// bits, element 2i in the low half of byte i, at codes + ((m * nkv + h) * cap
// + p) * d / 2, and one 32-bit word per group of g = min(d, 32) elements at
// params + ((m * nkv + h) * cap + p) * d / g: the bf16 minimum in the high
// half, the bf16 step in the low half.  Head-major, so that the positions of
// one head are one contiguous stretch for the attention that reads them.
//
// A group x_0 .. x_{g-1}: m = the largest bf16 <= min x, s = the smallest
// bf16 with 15 s >= max x - m, code = rint((x - m) / s) (0 where s = 0), and
// the code stands for fma(code, s, m).  Rounding m down and s up keeps every
// code in 0..15 without a clamp and every |x - value| <= s / 2 (+ the f32
// rounding of the value).  bf16 and not fp16 for the two: it holds every
// magnitude that f32 does, and since the codes are chosen against the rounded
// pair its 8 bits only widen the step by up to 2^-7.  A group with a value
// that is not finite, or whose range or rounded bounds leave f32 / bf16,
// stands for NaN as a whole (m and s NaN).
#pragma once

#include "common.cuh"
#include "kernels.cuh"

namespace tmg {

__host__ __device__ __forceinline__ int kv4_group(int d) { return d < 32 ? d : 32; }
__host__ __device__ __forceinline__ int kv4_groups(int d) { return d / kv4_group(d); }

__device__ __forceinline__ float kv4_min(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float kv4_step(uint32_t w) { return __uint_as_float(w << 16); }

// The parameter word of a group with extremes lo and hi; ok = every value
// of the group is finite.
__device__ __forceinline__ uint32_t kv4_params(float lo, float hi, bool ok) {
  const uint32_t lb = __float_as_uint(lo);
  uint32_t m = lb & 0xffff0000u;
  if ((lb >> 31) && m != lb) m += 0x10000u;  // towards -inf
  // the smallest bf16 s with 15 s >= hi - m: 15 s (12 bits) is an f32, so the
  // range may be rounded up first.  A product that is not below range / 15
  // gives s or the bf16 above it.
  const float range = __fsub_ru(hi, __uint_as_float(m));
  uint32_t s = (__float_as_uint(__fmul_ru(range, 0x1.111112p-4f)) + 0xffffu) & 0xffff0000u;
  if (s > 0u && 15.0f * __uint_as_float(s - 0x10000u) >= range) s -= 0x10000u;
  ok = ok && (m & 0x7f800000u) != 0x7f800000u && (s & 0x7f800000u) != 0x7f800000u &&
       range <= 3.402823466e38f;
  return ok ? (m | (s >> 16)) : 0x7fc07fc0u;
}

// The code of x in a group with parameter word `word`.
__device__ __forceinline__ uint32_t kv4_code(float x, uint32_t word) {
  const float s = kv4_step(word);
  return s > 0.0f ? uint32_t(rint((double(x) - double(kv4_min(word))) / double(s))) : 0u;
}

// The 8 codes of x in a group with parameter word `word`, lowest first.  The
// f32 quotient (x - m) / s is off by less than 4e-6 (15 times 2^-22: the
// difference, the reciprocal and the product), so it decides except next to a
// tie, or where 1 / s leaves f32; there the 64-bit quotient does.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], uint32_t word) {
  const float m = kv4_min(word), s = kv4_step(word);
  if (!(s > 0.0f)) return 0u;  // a constant group, or one that stands for NaN
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  // a sum with 1.5 * 2^23 has the rounded t in its low bits, above them
  // 0x4b400000, which the codes' places take off again
  constexpr float kMagic = 12582912.0f;
  uint32_t codes = 0u - 0x4b400000u * 0x11111111u;
  uint32_t sum = 0u;
  float off = 0.0f;
#pragma unroll
  for (int j = 7; j >= 0; --j) {
    const float t = (x[j] - m) * inv, r = t + kMagic;
    off = fmaxf(off, fabsf(t - (r - kMagic)));
    sum = sum * 16u + __float_as_uint(r);
  }
  codes += sum;
  if (off > 0.5f - 1e-5f || s < 0x1p-126f) {
    codes = 0u;
#pragma unroll 1
    for (int j = 7; j >= 0; --j) codes = codes * 16u + kv4_code(x[j], word);
  }
  return codes;
}

}  // namespace tmg
