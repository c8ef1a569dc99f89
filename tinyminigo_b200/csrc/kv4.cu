// Rows of keys and values quantised to 4 bits as they are written into the
// cache, and read back to f32 (kv4.cuh has the layout and the arithmetic).
// No counterpart in the reference, whose cache holds f32 rows
// (src/model.rs:250-332).
//
// Both kernels move data: 8 f32 a thread, 4 threads a group of 32 (two of 16
// for head dim 16), a warp for 256 / d consecutive rows of one head, so a
// warp reads 1 KB of f32 in segments of d floats and its codes (128 bytes)
// and parameters (32 or 64) are whole sectors of the cache.
#include "kv4.cuh"

namespace tmg {

namespace {

constexpr int kThreads = 256;

struct Rows {
  Kv4 kv;
  const float *k_in, *v_in;
  float *k_out, *v_out;
  int64_t ld, T;
  const int32_t *pos, *count;
  int32_t* err;
};

// A warp's work: rows t0 .. of one head of one stream, keys or values.
struct Work {
  bool value;
  int h, m;
  int64_t t0;
};
template <int D>
__device__ __forceinline__ bool warp_work(const Rows& a, int64_t w, Work* o) {
  const int64_t nt = (a.T + 256 / D - 1) / (256 / D);
  const int n = 2 * a.kv.nkv;
  const int c = int(w % n);
  w /= n;
  o->value = c >= a.kv.nkv;
  o->h = o->value ? c - a.kv.nkv : c;
  o->t0 = w % nt * (256 / D);
  w /= nt;
  o->m = int(w);
  return w < a.kv.M;
}

// The row of this thread and whether it takes part; its cache row.
template <int D>
__device__ __forceinline__ bool thread_row(const Rows& a, const Work& w, int lane, int64_t* t,
                                           int64_t* crow) {
  *t = w.t0 + lane / (D / 8);
  int64_t n = a.T;
  if (a.count) n = min(n, int64_t(max(a.count[w.m], 0)));
  if (*t >= n) return false;
  const int64_t p = int64_t(a.pos[w.m]) + *t;
  if (p < 0 || p >= a.kv.cap) {
    if (a.err) atomicCAS(a.err, 0, kErrPosition);
    return false;
  }
  *crow = (int64_t(w.m) * a.kv.nkv + w.h) * a.kv.cap + p;
  return true;
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const Rows a) {
  constexpr int G = D < 32 ? D : 32, LG = G / 8;  // lanes a group
  Work w;
  const int lane = threadIdx.x & 31;
  if (!warp_work<D>(a, int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32, &w)) return;
  int64_t t, crow;
  const bool on = thread_row<D>(a, w, lane, &t, &crow);
  const int e = lane % (D / 8) * 8;  // first element of the head's row
  float x[8] = {};
  if (on) {
    const float* p = (w.value ? a.v_in : a.k_in) + (int64_t(w.m) * a.T + t) * a.ld + w.h * D + e;
    const float4 u = __ldg(reinterpret_cast<const float4*>(p));
    const float4 v = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  }
  float lo = x[0], hi = x[0];
  bool ok = true;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    ok = ok && fabsf(x[i]) <= 3.402823466e38f;
  }
#pragma unroll
  for (int o = 1; o < LG; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    ok = __shfl_xor_sync(0xffffffffu, int(ok), o) && ok;
  }
  const uint32_t word = kv4_params(lo, hi, ok);
  const float m = kv4_min(word), s = kv4_step(word), inv = 1.0f / s;
  uint32_t codes = 0;
  if (s == s)
#pragma unroll
    for (int i = 0; i < 8; ++i) codes |= kv4_code(x[i], m, s, inv) << (4 * i);
  if (!on) return;
  uint8_t* cb = w.value ? a.kv.vc : a.kv.kc;
  uint32_t* pb = w.value ? a.kv.vp : a.kv.kp;
  *reinterpret_cast<uint32_t*>(cb + crow * (D / 2) + e / 2) = codes;
  if (lane % LG == 0) pb[crow * (D / G) + e / G] = word;
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const Rows a) {
  constexpr int G = D < 32 ? D : 32;
  Work w;
  const int lane = threadIdx.x & 31;
  if (!warp_work<D>(a, int64_t(blockIdx.x) * (kThreads / 32) + threadIdx.x / 32, &w)) return;
  float* ob = w.value ? a.v_out : a.k_out;
  int64_t t, crow;
  if (ob == nullptr || !thread_row<D>(a, w, lane, &t, &crow)) return;
  const int e = lane % (D / 8) * 8;
  const uint8_t* cb = w.value ? a.kv.vc : a.kv.kc;
  const uint32_t* pb = w.value ? a.kv.vp : a.kv.kp;
  const uint32_t c = __ldg(reinterpret_cast<const uint32_t*>(cb + crow * (D / 2) + e / 2));
  const uint32_t word = __ldg(pb + crow * (D / G) + e / G);
  const float m = kv4_min(word), s = kv4_step(word);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(float((c >> (4 * i)) & 15u), s, m);
  float4* p = reinterpret_cast<float4*>(ob + (int64_t(w.m) * a.T + t) * a.ld + w.h * D + e);
  p[0] = make_float4(x[0], x[1], x[2], x[3]);
  p[1] = make_float4(x[4], x[5], x[6], x[7]);
}

template <int D>
cudaError_t launch_rows(const Rows& a, bool append, cudaStream_t s) {
  const int64_t warps = 2ll * a.kv.M * a.kv.nkv * ((a.T + 256 / D - 1) / (256 / D));
  const int64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  if (append)
    kv4_append_kernel<D><<<unsigned(blocks), kThreads, 0, s>>>(a);
  else
    kv4_read_kernel<D><<<unsigned(blocks), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_rows_d(const Rows& a, bool append, cudaStream_t s) {
  if (a.T <= 0) return cudaSuccess;
  switch (a.kv.d) {
    case 16: return launch_rows<16>(a, append, s);
    case 32: return launch_rows<32>(a, append, s);
    case 64: return launch_rows<64>(a, append, s);
    case 128: return launch_rows<128>(a, append, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4& kv, const float* k, const float* v, int64_t row_ld,
                              int64_t T, const int32_t* pos, const int32_t* count, int32_t* err,
                              cudaStream_t s) {
  return launch_rows_d({kv, k, v, nullptr, nullptr, row_ld, T, pos, count, err}, true, s);
}

cudaError_t launch_kv4_read(const Kv4& kv, const int32_t* pos, const int32_t* count, int64_t T,
                            float* k, float* v, int64_t row_ld, int32_t* err, cudaStream_t s) {
  return launch_rows_d({kv, nullptr, nullptr, k, v, row_ld, T, pos, count, err}, false, s);
}

}  // namespace tmg
