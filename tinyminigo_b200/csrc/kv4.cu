// Rows of keys and values quantised to 4 bits as they are written into the
// cache, and read back to f32 (kv4.cuh has the layout and the arithmetic).
// No counterpart in the reference, whose cache holds f32 rows
// (src/model.rs:250-332).
//
// Both kernels move data.  A warp's unit is 256 / d consecutive rows of one
// head: 1 KB of f32 in segments of d floats, and codes (128 bytes) and
// parameters (32 or 64) that are whole sectors of the cache.  The f32 side
// goes 16 bytes a lane, a warp's 512 in one piece; 4 units a warp, their loads
// in flight together, once there are enough rows to fill the GPU so.
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

// A warp's work: U units from row t0 of one head of one stream, keys or values.
struct Work {
  bool value;
  int h, m;
  int64_t t0;
};
template <int D, int U>
__device__ __forceinline__ bool warp_work(const Rows& a, Work* o) {
  constexpr int R = 256 / D * U;  // rows
  const unsigned nt = unsigned((a.T + R - 1) / R), n = 2u * a.kv.nkv;
  unsigned w = blockIdx.x * (kThreads / 32) + threadIdx.x / 32;
  const unsigned c = w % n;
  w /= n;
  o->value = int(c) >= a.kv.nkv;
  o->h = o->value ? int(c) - a.kv.nkv : int(c);
  o->t0 = int64_t(w % nt) * R;
  o->m = int(w / nt);
  return o->m < a.kv.M;
}

// Rows of stream m that are no padding, and the first one's position.
__device__ __forceinline__ int64_t row_count(const Rows& a, int m) {
  return a.count ? min(a.T, int64_t(max(a.count[m], 0))) : a.T;
}
// The cache row of position p, or -1 (reported) outside the cache.
__device__ __forceinline__ int64_t cache_row(const Rows& a, const Work& w, int64_t p) {
  if (p < 0 || p >= a.kv.cap) {
    if (a.err) atomicCAS(a.err, 0, kErrPosition);
    return -1;
  }
  return (int64_t(w.m) * a.kv.nkv + w.h) * a.kv.cap + p;
}

// 8 elements a lane: a group's arithmetic (a division among it) is repeated
// by 4 lanes and not by 8.
template <int D, int U>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const Rows a) {
  constexpr int G = D < 32 ? D : 32, LG = G / 8;  // lanes a group
  Work w;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  if (!warp_work<D, U>(a, &w)) return;
  const int64_t n = row_count(a, w.m), p0 = a.pos[w.m];
  const float* in = (w.value ? a.v_in : a.k_in) + int64_t(w.m) * a.T * a.ld + w.h * D;
  const int t0 = lane * 8 / D, e = lane * 8 % D;  // the lane's row of a unit, and column
  float4 v[U][2];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t t = w.t0 + i * (256 / D) + t0;
    v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (t < n) {
      const float4* p = reinterpret_cast<const float4*>(in + t * a.ld + e);
      v[i][0] = __ldg(p);
      v[i][1] = __ldg(p + 1);
    }
  }
  uint8_t* cb = w.value ? a.kv.vc : a.kv.kc;
  uint32_t* pb = w.value ? a.kv.vp : a.kv.kp;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const float x[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w,
                        v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
    float lo = x[0], hi = x[0];
    bool ok = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo = fminf(lo, x[j]);
      hi = fmaxf(hi, x[j]);
      ok = ok && fabsf(x[j]) <= 3.402823466e38f;
    }
    // the group's extremes over its lanes; +inf above stands for a value that
    // is not finite
    hi = ok ? hi : INFINITY;
#pragma unroll
    for (int o = 1; o < LG; o <<= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const uint32_t word = kv4_params(lo, hi, hi < INFINITY);
    const uint32_t codes = kv4_codes(x, word);
    const int64_t t = w.t0 + i * (256 / D) + t0;
    const int64_t row = t < n ? cache_row(a, w, p0 + t) : -1;
    if (row < 0) continue;
    *reinterpret_cast<uint32_t*>(cb + row * (D / 2) + e / 2) = codes;
    if (lane % LG == 0) pb[row * (D / G) + e / G] = word;
  }
}

// The f32 side in pieces of 128 elements, 4 a lane: element 4 lane of piece i
// is in row (128 i + 4 lane) / d of the warp's, column (128 i + 4 lane) % d.
template <int D, int U>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const Rows a) {
  constexpr int G = D < 32 ? D : 32;
  Work w;
  const int lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  if (!warp_work<D, U>(a, &w)) return;
  float* out = w.value ? a.v_out : a.k_out;
  if (out == nullptr) return;
  const int64_t n = row_count(a, w.m), p0 = a.pos[w.m];
  const uint8_t* cb = w.value ? a.kv.vc : a.kv.kc;
  const uint32_t* pb = w.value ? a.kv.vp : a.kv.kp;
  // codes 8 a lane, as whole sectors
  uint32_t c[U], word[U];
  bool on[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int e = i * 256 + lane * 8;
    const int64_t t = w.t0 + e / D;
    const int64_t row = t < n ? cache_row(a, w, p0 + t) : -1;
    on[i] = row >= 0;
    c[i] = word[i] = 0;
    if (on[i]) {
      c[i] = __ldg(reinterpret_cast<const uint32_t*>(cb + row * (D / 2) + e % D / 2));
      word[i] = __ldg(pb + row * (D / G) + e % D / G);
    }
  }
  out += int64_t(w.m) * a.T * a.ld + w.h * D;
#pragma unroll
  for (int i = 0; i < 2 * U; ++i) {
    // 4 of the 8 codes that lane 16 (i % 2) + lane / 2 has loaded
    const int src = 16 * (i % 2) + lane / 2;
    const uint32_t cc = __shfl_sync(0xffffffffu, c[i / 2], src) >> (16 * (lane & 1));
    const uint32_t ww = __shfl_sync(0xffffffffu, word[i / 2], src);
    if (!__shfl_sync(0xffffffffu, int(on[i / 2]), src)) continue;
    const float m = kv4_min(ww), s = kv4_step(ww);
    const int e = i * 128 + lane * 4;
    __stcs(reinterpret_cast<float4*>(out + (w.t0 + e / D) * a.ld + e % D),
           make_float4(fmaf(float(cc & 15u), s, m), fmaf(float((cc >> 4) & 15u), s, m),
                       fmaf(float((cc >> 8) & 15u), s, m), fmaf(float((cc >> 12) & 15u), s, m)));
  }
}

// One decode step's rows (q | k | v of every stream, before RoPE): rotates q in
// place, rotates and quantises k, quantises v, at the stream's position, and
// gives the attention its length.  A warp a head; the arithmetic of RoPE as
// everywhere (src/tensor.rs:1026-1037), each product and sum rounded.
template <int D>
__global__ void __launch_bounds__(32) kv4_step_kernel(const Kv4 kv, float* qkv, int64_t ld, int nq,
                                                      StreamState st, const float* rope_cos,
                                                      const float* rope_sin, int cap,
                                                      int32_t* lens) {
  constexpr int G = D < 32 ? D : 32, NG = D / G, E = NG;  // elements a lane: one of each group
  const int m = blockIdx.y, head = blockIdx.x, lane = threadIdx.x;
  pdl_trigger();
  pdl_wait();
  const int pos = st.pos[m];
  const bool append = st.done[m] == 0 && pos < cap;
  if (head == 0 && lane == 0) lens[m] = append ? pos + 1 : min(pos, cap);
  if (!append && head >= nq) return;
  float* row = qkv + m * ld + head * D;
  const bool on = lane < G;
  float x[E];
#pragma unroll
  for (int i = 0; i < E; ++i) x[i] = on ? row[i * G + lane] : 0.f;
  const bool value = head >= nq + kv.nkv;
  if (!value) {
    // element e pairs with e + d / 2: another group of the lane, or another lane
    const int at = min(pos, cap - 1);  // a finished stream may stand behind the last
    const float* c = rope_cos + int64_t(at) * (D / 2);
    const float* s = rope_sin + int64_t(at) * (D / 2);
    float y[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = i * G + (lane % G), j = e % (D / 2);
      const float other = E > 1 ? x[(i + E / 2) % E] : __shfl_xor_sync(0xffffffffu, x[i], D / 2);
      const float cs = c[j], sn = s[j];
      y[i] = e < D / 2 ? __fsub_rn(__fmul_rn(x[i], cs), __fmul_rn(other, sn))
                       : __fadd_rn(__fmul_rn(other, sn), __fmul_rn(x[i], cs));
    }
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = y[i];
  }
  if (head < nq) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (on) row[i * G + lane] = x[i];
    return;
  }
  const int h = value ? head - nq - kv.nkv : head - nq;
  const int64_t crow = (int64_t(m) * kv.nkv + h) * kv.cap + pos;
  uint8_t* cb = (value ? kv.vc : kv.kc) + crow * (D / 2);
  uint32_t* pb = (value ? kv.vp : kv.kp) + crow * NG;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const bool ok = fabsf(x[i]) <= 3.402823466e38f;
    const float lo = -warp_max(on ? -x[i] : -INFINITY), hi = warp_max(on ? x[i] : -INFINITY);
    const uint32_t word = kv4_params(lo, hi, __all_sync(0xffffffffu, ok || !on));
    const uint32_t code = on ? kv4_code(x[i], word) : 0u;
    const uint32_t next = __shfl_down_sync(0xffffffffu, code, 1);
    if (on && lane % 2 == 0) cb[(i * G + lane) / 2] = uint8_t(code | (next << 4));
    if (lane == 0) pb[i] = word;
  }
}

template <typename K>
cudaError_t launch_units(K kern, int U, const Rows& a, cudaStream_t s) {
  const int64_t rows = 256 / a.kv.d * U;  // a warp's
  const int64_t warps = 2ll * a.kv.M * a.kv.nkv * ((a.T + rows - 1) / rows);
  const int64_t blocks = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (blocks > INT32_MAX / (kThreads / 32)) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <int D>
cudaError_t launch_rows(const Rows& a, bool append, cudaStream_t s) {
  // several units a warp from about two waves of 148 x 64 warps on; 2 to write
  // (4 took 30 us where 2 take 28), 4 to read
  const bool many = 2ll * a.kv.M * a.kv.nkv * ((a.T + 256 / D - 1) / (256 / D)) >= 18944;
  if (append)
    return many ? launch_units(kv4_append_kernel<D, 2>, 2, a, s)
                : launch_units(kv4_append_kernel<D, 1>, 1, a, s);
  return many ? launch_units(kv4_read_kernel<D, 4>, 4, a, s)
              : launch_units(kv4_read_kernel<D, 1>, 1, a, s);
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

template <int D>
cudaError_t launch_step(const Kv4& kv, float* qkv, int64_t ld, int nq, const StreamState& st,
                        const float* rope_cos, const float* rope_sin, int cap, int32_t* lens,
                        cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(nq + 2 * kv.nkv, kv.M);
  cfg.blockDim = dim3(32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_step_kernel<D>, kv, qkv, ld, nq, st, rope_cos, rope_sin,
                            cap, lens);
}

template <int D>
cudaError_t carveouts() {
  TMG_CUDA_TRY(set_carveout(kv4_step_kernel<D>));
  TMG_CUDA_TRY(set_carveout(kv4_append_kernel<D, 1>));
  TMG_CUDA_TRY(set_carveout(kv4_append_kernel<D, 2>));
  TMG_CUDA_TRY(set_carveout(kv4_read_kernel<D, 1>));
  return set_carveout(kv4_read_kernel<D, 4>);
}

}  // namespace

cudaError_t kv4_prepare() {
  TMG_CUDA_TRY(carveouts<16>());
  TMG_CUDA_TRY(carveouts<32>());
  TMG_CUDA_TRY(carveouts<64>());
  return carveouts<128>();
}

cudaError_t launch_kv4_step(const Kv4& kv, float* qkv, int64_t ld, int nq, const StreamState& st,
                            const float* rope_cos, const float* rope_sin, int cap, int32_t* lens,
                            cudaStream_t s) {
  switch (kv.d) {
    case 16: return launch_step<16>(kv, qkv, ld, nq, st, rope_cos, rope_sin, cap, lens, s);
    case 32: return launch_step<32>(kv, qkv, ld, nq, st, rope_cos, rope_sin, cap, lens, s);
    case 64: return launch_step<64>(kv, qkv, ld, nq, st, rope_cos, rope_sin, cap, lens, s);
    case 128: return launch_step<128>(kv, qkv, ld, nq, st, rope_cos, rope_sin, cap, lens, s);
  }
  return cudaErrorInvalidValue;
}

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
