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
  // the smallest bf16 s with 15 s >= hi - m: each step rounds up, and 15 s
  // (12 bits) is an f32, so rounding up twice picks no larger one
  const float range = __fsub_ru(hi, __uint_as_float(m));
  const uint32_t sb = __float_as_uint(__fdiv_ru(range, 15.0f));
  const uint32_t s = (sb + 0xffffu) & 0xffff0000u;
  ok = ok && (m & 0x7f800000u) != 0x7f800000u && (s & 0x7f800000u) != 0x7f800000u &&
       range <= 3.402823466e38f;
  return ok ? (m | (s >> 16)) : 0x7fc07fc0u;
}

// The code of x in a group with parameters (m, s), inv = 1 / s.  The f32
// quotient is off by less than 4e-6 (three roundings of a value below 16),
// so it decides except next to a tie; there the 64-bit quotient does.
__device__ __forceinline__ uint32_t kv4_code(float x, float m, float s, float inv) {
  const float t = (x - m) * inv;
  const float r = rintf(t);
  if (fabsf(fabsf(t - r) - 0.5f) > 1e-5f) return uint32_t(r);
  if (!(s > 0.0f)) return 0u;
  return uint32_t(rint((double(x) - double(m)) / double(s)));
}

}  // namespace tmg
