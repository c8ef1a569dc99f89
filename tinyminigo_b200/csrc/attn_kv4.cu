// Decode attention over the 4-bit KV cache (kv4.cuh): per query head of each
// stream, o = sum_t p_t v_t with p = softmax(q . k_t / sqrt(d)) over the
// stream's cached positions (the attention of src/model.rs:434-459, whose
// cache is f32).
#include <math.h>

#include "kv4.cuh"

namespace tmg {

namespace {

constexpr int kWarps = 4;

// One CTA per (query head, stream).  A warp takes 32 positions at a time:
// a lane scores one of them, then the lanes share the values' columns and
// walk the 32 positions; online softmax per warp, the warps meet at the end.
template <int D>
__global__ void __launch_bounds__(kWarps * 32) attn_kv4_simple_kernel(const AttnKv4Args a) {
  constexpr int G = D < 32 ? D : 32, NG = D / G, C = D < 32 ? 1 : D / 32;
  __shared__ float qs[D];
  __shared__ float os[kWarps][D], ms[kWarps], ls[kWarps];
  const int h = blockIdx.x, m = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kvh = h / (a.nq / a.kv.nkv);
  int len = a.lens[m];
  if (len < 0 || len > a.max_len) {
    if (threadIdx.x == 0 && a.err) atomicCAS(a.err, 0, kErrLength);
    len = len < 0 ? 0 : int(a.max_len);
  }
  for (int i = threadIdx.x; i < D; i += blockDim.x) qs[i] = a.q[int64_t(m) * a.q_ld + h * D + i];
  __syncthreads();
  const int64_t row0 = (int64_t(m) * a.kv.nkv + kvh) * a.kv.cap;
  float mx = -INFINITY, l = 0.f, o[C] = {};
  for (int t0 = warp * 32; t0 < len; t0 += kWarps * 32) {
    const int t = t0 + lane;
    float s = -INFINITY;
    if (t < len) {
      const uint32_t* c = reinterpret_cast<const uint32_t*>(a.kv.kc + (row0 + t) * (D / 2));
      float acc = 0.f;
      for (int g = 0; g < NG; ++g) {
        const uint32_t w = a.kv.kp[(row0 + t) * NG + g];
        const float mn = kv4_min(w), st = kv4_step(w);
        for (int j = 0; j < G / 8; ++j) {
          const uint32_t cw = c[g * (G / 8) + j];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            acc = fmaf(qs[g * G + j * 8 + i], fmaf(float((cw >> (4 * i)) & 15u), st, mn), acc);
        }
      }
      s = acc * a.scale;
    }
    const float nm = fmaxf(mx, warp_max(s));
    const float ref = nm == -INFINITY ? 0.f : nm;
    const float al = expf(mx - ref), p = t < len ? expf(s - ref) : 0.f;
    mx = nm;
    l = l * al + p;
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] *= al;
    const int n = min(32, len - t0);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const int64_t r = row0 + t0 + j;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int e = i * 32 + lane;
        if (e < D) {
          const uint32_t w = a.kv.vp[r * NG + e / G];
          const uint32_t b = a.kv.vc[r * (D / 2) + e / 2];
          o[i] = fmaf(pj, fmaf(float((b >> (4 * (e & 1))) & 15u), kv4_step(w), kv4_min(w)), o[i]);
        }
      }
    }
  }
  l = warp_sum(l);
  if (lane == 0) ms[warp] = mx, ls[warp] = l;
#pragma unroll
  for (int i = 0; i < C; ++i)
    if (i * 32 + lane < D) os[warp][i * 32 + lane] = o[i];
  __syncthreads();
  float M = -INFINITY;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ms[w]);
  const float ref = M == -INFINITY ? 0.f : M;
  for (int e = threadIdx.x; e < D; e += blockDim.x) {
    float tot = 0.f, acc = 0.f;
    for (int w = 0; w < kWarps; ++w) {
      const float f = expf(ms[w] - ref);
      tot += ls[w] * f;
      acc = fmaf(os[w][e], f, acc);
    }
    a.out[int64_t(m) * a.out_ld + h * D + e] = len > 0 ? acc / tot : 0.f;
  }
}

}  // namespace

size_t attn_kv4_ws(const Kv4&, int, int) { return 0; }

cudaError_t launch_attn_kv4(const AttnKv4Args& a, cudaStream_t s) {
  const dim3 grid(a.nq, a.kv.M);
  switch (a.kv.d) {
    case 16: attn_kv4_simple_kernel<16><<<grid, kWarps * 32, 0, s>>>(a); break;
    case 32: attn_kv4_simple_kernel<32><<<grid, kWarps * 32, 0, s>>>(a); break;
    case 64: attn_kv4_simple_kernel<64><<<grid, kWarps * 32, 0, s>>>(a); break;
    case 128: attn_kv4_simple_kernel<128><<<grid, kWarps * 32, 0, s>>>(a); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace tmg
