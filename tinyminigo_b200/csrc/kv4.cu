// Rows of keys and values quantised to 4 bits as they are written into the
// cache, and read back to f32 (kv4.cuh has the layout and the arithmetic).
// No counterpart in the reference, whose cache holds f32 rows
// (src/model.rs:250-332).
//
// Both kernels move data.  A warp's unit is 256 / d consecutive rows of one
// head: 1 KB of f32 in segments of d floats, and codes (128 bytes) and
// parameters (32 or 64) that are whole sectors of the cache.  The f32 side
// goes 16 bytes a lane, a warp's 512 in one piece; several units a warp, their
// loads in flight together, once there are enough rows to fill the GPU so.
//
// Reading 65536 rows (8 heads of 128: 84 MB of cache, 537 MB of f32) takes 98
// us, 6.3 TB/s, 96% of a plain copy's rate.  Writing 4000 rows (32.8 MB in, 5.1
// MB out) takes 11.8 us a call in a graph, where the bytes are 5.8: 2000 blocks, of
// which 592 are resident (4 an SM, at 61 registers a thread), so 3.4 waves at half
// the warps that an SM holds, each with its own latency of loads, the group's
// extremes by 2 rounds of shuffles, 183 instructions a unit of 256 values, and
// stores.  A few rows (a step of 16 streams) take a launch's time, 2.4 us in a graph
// and about 4 from the host.
#include <algorithm>

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

// Blocks: x the head (keys, then values; all heads of a row at once, since
// they are neighbours in memory), y a stretch of rows, z the stream.  A warp's
// rows w.t0 .. w.t0 + 256 / d * U - 1 of that head.
struct Work {
  bool value;
  int h;
  int64_t n;     // rows of the stream that are no padding
  int64_t p0;    // position of row 0
  int64_t row0;  // cache row of position 0
};
__device__ __forceinline__ Work block_work(const Rows& a) {
  Work w;
  const int m = blockIdx.z;
  w.value = int(blockIdx.x) >= a.kv.nkv;
  w.h = int(blockIdx.x) - (w.value ? a.kv.nkv : 0);
  w.n = a.count ? min(a.T, int64_t(max(a.count[m], 0))) : a.T;
  w.p0 = a.pos[m];
  w.row0 = (int64_t(m) * a.kv.nkv + w.h) * a.kv.cap;
  return w;
}
// Whether position p lies in the cache (reported if not).
__device__ __forceinline__ bool in_cache(const Rows& a, int64_t p) {
  if (p >= 0 && p < a.kv.cap) return true;
  if (a.err) atomicCAS(a.err, 0, kErrPosition);
  return false;
}

// The smaller / larger of two, NaN if either is.
__device__ __forceinline__ float min_nan(float a, float b) {
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// 8 elements a lane: a group's arithmetic is repeated by 4 lanes and not by 8.
template <int D, int U>
__global__ void __launch_bounds__(kThreads) kv4_append_kernel(const Rows a) {
  constexpr int G = D < 32 ? D : 32, LG = G / 8;  // lanes a group
  constexpr int R = 256 / D;                      // rows a unit
  pdl_trigger();
  pdl_wait();
  const Work w = block_work(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = lane * 8 % D;  // the lane's column; its row of a unit: lane * 8 / D
  const float* in = (w.value ? a.v_in : a.k_in) + int64_t(blockIdx.z) * a.T * a.ld + w.h * D + e;
  uint8_t* cb = (w.value ? a.kv.vc : a.kv.kc) + e / 2;
  uint32_t* pb = (w.value ? a.kv.vp : a.kv.kp) + e / G;
  constexpr int kBlock = kThreads / 32 * U * R;  // rows a block and round
#pragma unroll 1
  for (int64_t tb = int64_t(blockIdx.y) * kBlock; tb < w.n; tb += int64_t(gridDim.y) * kBlock) {
    const int64_t t0 = tb + warp * (U * R) + lane * 8 / D;
    const float* src = in + t0 * a.ld;
    float4 v[U][2];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (t0 + i * R < w.n) {
        v[i][0] = __ldg(reinterpret_cast<const float4*>(src));
        v[i][1] = __ldg(reinterpret_cast<const float4*>(src) + 1);
      }
      src += R * a.ld;
    }
    const int64_t row = w.row0 + w.p0 + t0;
    uint8_t* cd = cb + row * (D / 2);
    uint32_t* pd = pb + row * (D / G);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const float x[8] = {v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w,
                          v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w};
      float lo = x[0], hi = x[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) {
        lo = min_nan(lo, x[j]);
        hi = max_nan(hi, x[j]);
      }
#pragma unroll
      for (int o = 1; o < LG; o <<= 1) {
        lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      const uint32_t word =
          kv4_params(lo, hi, lo >= -3.402823466e38f && hi <= 3.402823466e38f);
      const uint32_t codes = kv4_codes(x, word);
      const int64_t t = t0 + i * R;
      if (t < w.n && in_cache(a, w.p0 + t)) {
        *reinterpret_cast<uint32_t*>(cd + i * R * (D / 2)) = codes;
        if (lane % LG == 0) pd[i * R * (D / G)] = word;
      }
    }
  }
}

// The f32 side in pieces of 128 elements, 4 a lane: element 4 lane of piece i
// is in row (128 i + 4 lane) / d of the warp's, column (128 i + 4 lane) % d.
template <int D, int U>
__global__ void __launch_bounds__(kThreads) kv4_read_kernel(const Rows a) {
  constexpr int G = D < 32 ? D : 32, R = 256 / D;
  pdl_trigger();
  pdl_wait();
  const Work w = block_work(a);
  float* out = w.value ? a.v_out : a.k_out;
  if (out == nullptr) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e = lane * 8 % D;
  const uint8_t* cb = (w.value ? a.kv.vc : a.kv.kc) + e / 2;
  const uint32_t* pb = (w.value ? a.kv.vp : a.kv.kp) + e / G;
  out += int64_t(blockIdx.z) * a.T * a.ld + w.h * D;
  constexpr int kBlock = kThreads / 32 * U * R;
#pragma unroll 1
  for (int64_t tb = int64_t(blockIdx.y) * kBlock; tb < w.n; tb += int64_t(gridDim.y) * kBlock) {
    const int64_t tw = tb + warp * (U * R), t0 = tw + lane * 8 / D;
    const int64_t row = w.row0 + w.p0 + t0;
    const uint8_t* cs = cb + row * (D / 2);
    const uint32_t* ps = pb + row * (D / G);
    // codes 8 a lane, as whole sectors
    uint32_t c[U], word[U];
    bool on[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int64_t t = t0 + i * R;
      on[i] = t < w.n && in_cache(a, w.p0 + t);
      c[i] = word[i] = 0;
      if (on[i]) {
        c[i] = __ldg(reinterpret_cast<const uint32_t*>(cs + i * R * (D / 2)));
        word[i] = __ldg(ps + i * R * (D / G));
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * U; ++i) {
      // 4 of the 8 codes that lane 16 (i % 2) + lane / 2 has loaded
      const int from = 16 * (i % 2) + lane / 2;
      const uint32_t cc = __shfl_sync(0xffffffffu, c[i / 2], from) >> (16 * (lane & 1));
      const uint32_t ww = __shfl_sync(0xffffffffu, word[i / 2], from);
      const bool store = __shfl_sync(0xffffffffu, int(on[i / 2]), from);
      const float m = kv4_min(ww), s = kv4_step(ww);
      const int q = i * 128 + lane * 4;
      if (store)
        __stcs(reinterpret_cast<float4*>(out + (tw + q / D) * a.ld + q % D),
               make_float4(fmaf(float(cc & 15u), s, m), fmaf(float((cc >> 4) & 15u), s, m),
                           fmaf(float((cc >> 8) & 15u), s, m), fmaf(float((cc >> 12) & 15u), s, m)));
    }
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
  const int64_t rows = int64_t(kThreads / 32) * U * 256 / a.kv.d;  // a block's
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * a.kv.nkv, unsigned(std::min<int64_t>((a.T + rows - 1) / rows, 65535)), a.kv.M);
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
