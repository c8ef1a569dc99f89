// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives, per row of logits.  The reference has the softmax of
// its sampler only (src/tensor.rs:1142-1213).
//
// With y_i = x_i - max x, Z = sum e^{y_i}: log p_i = y_i - ln Z and H = ln Z -
// sum e^{y_i} y_i / Z, so one pass that keeps (max, Z, sum e^y y) online gives
// both.  y is taken before the change to base 2 (not x log2 e - max log2 e in
// one fma), so that rows at the type's lowest value stay finite.
#include <math.h>

#include "common.cuh"
#include "kernels.cuh"

namespace tmg {

namespace {

constexpr int kThreads = 512;
constexpr int kCand = 2048;  // candidates of a row held in shared memory
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

using u64 = unsigned long long;

// Larger key = earlier alternative: value first, ties to the lower index;
// NaN counts as -inf.  Every element's key is above 0 and its own.
__device__ __forceinline__ u64 order_key(float v, uint32_t idx) {
  if (!(v == v)) v = -INFINITY;
  uint32_t b = __float_as_uint(v + 0.0f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (u64(b) << 32) | uint32_t(~idx);
}
__device__ __forceinline__ float key_value(u64 k) {
  uint32_t b = uint32_t(k >> 32);
  b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
  return __uint_as_float(b);
}

// 2^x by the SFU's ex2 instruction (relative error about 2^-22; 2^-inf = 0)
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The online state: the largest x, l = sum e^y, w = sum e^y y (y = (x_i - x)
// log2 e).
struct Soft {
  float x = -INFINITY, l = 0.f, w = 0.f;
};
constexpr float kFloor = -1000.f;  // 2^kFloor = 0: what a y of -inf weighs in w

// Move s to the reference point x >= s.x: w moves by the change per unit of l.
__device__ __forceinline__ void move(Soft& s, float x) {
  const float d = fmaxf((s.x - x) * kLog2e, kFloor), f = ex2_approx(d);
  s.w = fmaf(s.l, d, s.w) * f;
  s.l *= f;
  s.x = x;
}
__device__ __forceinline__ void merge(Soft& a, Soft b) {
  const float x = fmaxf(a.x, b.x);
  if (x > -INFINITY) {  // else both sums are 0, or NaN
    move(a, x);
    move(b, x);
  }
  a.l += b.l;
  a.w += b.w;
}

// 4 floats of the row at chunk c of the 16-byte grid its first element
// lies `shift` floats into; elements outside the row read as -inf and
// have no key.
struct Row {
  const float* base;  // 16-byte aligned: the row's start - shift
  int shift;
  int64_t V;
  __device__ __forceinline__ float4 load(int64_t c) const {
    const int64_t i = 4 * c - shift;
    if (i >= 0 && i + 4 <= V) return __ldg(reinterpret_cast<const float4*>(base) + c);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j >= 0 && i + j < V ? __ldg(base + 4 * c + j) : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ u64 key(float x, int64_t c, int j) const {
    const int64_t i = 4 * c - shift + j;
    return i >= 0 && i < V ? order_key(x, uint32_t(i)) : 0ull;
  }
};

__device__ __forceinline__ void accumulate(Soft& s, const float4& v) {
  const float mx = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
  if (mx > s.x) move(s, mx);
  const float x[4] = {v.x, v.y, v.z, v.w}, ref = s.x == -INFINITY ? 0.f : s.x;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float y = (x[j] - ref) * kLog2e, e = ex2_approx(y);
    s.l += e;
    s.w = fmaf(e, fmaxf(y, kFloor), s.w);
  }
}

__global__ void __launch_bounds__(kThreads) logprobs_kernel(const LogprobsArgs a) {
  __shared__ Soft soft_s[kThreads / 32];
  __shared__ u64 cand[kCand];
  __shared__ int owner[kMaxTopK];
  __shared__ int n_owner, n_cand;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x;
  const float* row = a.logits + r * a.ld;
  Row R;
  R.shift = int((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
  R.base = row - R.shift;
  R.V = a.V;
  const int64_t nc = (a.V + R.shift + 3) / 4;

  Soft s;
  float best = -INFINITY;
  int64_t bc = tid;
  for (int64_t c = tid; c < nc; c += kThreads) {
    const float4 v = R.load(c);
    const float mx = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
    if (mx > best) best = mx, bc = c;
    accumulate(s, v);
  }
  auto shfl = [&](const Soft& t, int o) {
    Soft u;
    u.x = __shfl_xor_sync(0xffffffffu, t.x, o);
    u.l = __shfl_xor_sync(0xffffffffu, t.l, o);
    u.w = __shfl_xor_sync(0xffffffffu, t.w, o);
    return u;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(s, shfl(s, o));
  if (lane == 0) soft_s[warp] = s;
  if (tid == 0) n_owner = n_cand = 0;
  __syncthreads();
  s = soft_s[0];
  for (int w = 1; w < kThreads / 32; ++w) merge(s, soft_s[w]);
  const float lz = logf(s.l);  // ln Z
  if (tid == 0) {
    if (a.logprob) {
      const uint32_t t = a.targets[r];
      float lp = NAN;
      if (t < uint64_t(a.V)) lp = (row[t] - s.x) - lz;
      else if (a.err) atomicCAS(a.err, 0, kErrToken);
      a.logprob[r] = lp;
    }
    if (a.entropy) a.entropy[r] = lz - s.w / s.l * kLn2;
  }
  if (a.n_top == 0) return;

  // Alternatives.  Each thread's best key is an element; the n_top-th largest
  // of them bounds the row's n_top-th largest element from below, and only the
  // n_top threads at or above it can hold an element that is: their elements
  // are looked at again.
  u64 mine = 0ull;
  if (bc < nc) {
    const float4 v = R.load(bc);
    const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const u64 k = R.key(x[j], bc, j);
      mine = k > mine ? k : mine;
    }
  }
  u64 tau = 0ull;
  for (int b = 63; b >= 0; --b) {
    const u64 t = tau | (1ull << b);
    const int n = __syncthreads_count(mine >= t);
    if (n >= a.n_top) tau = t;
    if (n == a.n_top) break;
  }
  const int64_t per = (nc + kThreads - 1) / kThreads;
  if (mine >= tau && mine != 0ull) owner[min(atomicAdd(&n_owner, 1), kMaxTopK - 1)] = tid;
  __syncthreads();
  const bool all = n_owner < a.n_top;  // fewer threads with elements than wanted
  const int64_t todo = all ? nc : per * n_owner;
  auto chunk = [&](int64_t i) { return all ? i : i / n_owner * kThreads + owner[i % n_owner]; };
  auto collect = [&](u64 t, bool keep) {
    int n = 0;
    for (int64_t i = tid; i < todo; i += kThreads) {
      const int64_t c = chunk(i);
      if (c >= nc) continue;
      const float4 v = R.load(c);
      const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 k = R.key(x[j], c, j);
        if (k != 0ull && k >= t) {
          ++n;
          if (keep) {
            const int at = atomicAdd(&n_cand, 1);
            if (at < kCand) cand[at] = k;
          }
        }
      }
    }
    return n;
  };
  collect(tau, true);
  __syncthreads();
  if (n_cand > kCand) {
    // more at or above the bound than fit (few threads hold the large ones):
    // raise it, bit by bit, to a value that n_top or a few more reach
    __shared__ int n_s;
    u64 up = 0ull;
    for (int b = 63; b >= 0; --b) {
      const u64 t = up | (1ull << b);
      if (tid == 0) n_s = 0;
      __syncthreads();
      const int n = collect(t > tau ? t : tau, false);
      if (n) atomicAdd(&n_s, n);
      __syncthreads();
      const int total = n_s;
      __syncthreads();
      if (total >= a.n_top) up = t;
      if (total >= a.n_top && total <= kCand) break;
    }
    if (tid == 0) n_cand = 0;
    __syncthreads();
    collect(up > tau ? up : tau, true);
    __syncthreads();
  }
  const int n = min(n_cand, kCand);
  for (int i = tid; i < n; i += kThreads) {
    const u64 k = cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > k;
    if (rank < a.n_top) {
      a.top_ids[r * a.n_top + rank] = ~uint32_t(k);
      a.top_logprobs[r * a.n_top + rank] = (key_value(k) - s.x) - lz;
    }
  }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, cudaStream_t s) {
  if (a.rows == 0) return cudaSuccess;
  logprobs_kernel<<<unsigned(a.rows), kThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace tmg
