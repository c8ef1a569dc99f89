// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives, per row of logits.  The reference has the softmax of
// its sampler only (src/tensor.rs:1142-1213).
//
// With y_i = x_i - max x, Z = sum e^{y_i}: log p_i = y_i - ln Z and H = ln Z -
// sum e^{y_i} y_i / Z, so one pass that keeps (max, Z, sum e^y y) online gives
// both.  y is taken before the change to base 2 (not x log2 e - max log2 e in
// one fma), so that rows at the type's lowest value stay finite.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "kernels.cuh"

namespace tmg {

namespace cg = cooperative_groups;

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

// The largest of the row's elements in v, as keys; elements outside have none.
__device__ __forceinline__ u64 best_key(const Row& R, const float4& v, int64_t c) {
  const float x[4] = {v.x, v.y, v.z, v.w};
  u64 b = 0ull;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const u64 k = R.key(x[j], c, j);
    b = k > b ? k : b;
  }
  return b;
}

// A thread's pass over its chunks: the online state, and the first chunk that
// holds its largest element.
struct Pass {
  Soft s;
  float best = -INFINITY;
  int64_t at;
  template <int U>
  __device__ __forceinline__ void take(const float4 (&v)[U], int64_t c) {
    float m[U], mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      m[u] = fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w));
      mx = fmaxf(mx, m[u]);
    }
    if (mx > best) {
      best = mx;
#pragma unroll
      for (int u = U - 1; u >= 0; --u)
        if (m[u] == mx) at = c + int64_t(u) * kThreads;
      move(s, mx);
    }
    const float ref = s.x == -INFINITY ? 0.f : s.x;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = (x[j] - ref) * kLog2e, e = ex2_approx(y);
        s.l += e;
        s.w = fmaf(e, fmaxf(y, kFloor), s.w);
      }
    }
  }
};

// The CTA's result, for the cluster's first CTA to join.
struct Part {
  Soft s;
  int n;  // alternatives in the list, largest first
  u64 top[kMaxTopK];
};

__global__ void __launch_bounds__(kThreads, 3) logprobs_kernel(const LogprobsArgs a) {
  __shared__ Soft soft_s[kThreads / 32];
  __shared__ u64 cand[kCand];
  __shared__ int owner[kMaxTopK];
  __shared__ int n_owner, n_cand, n_s;
  __shared__ Part part;
  cg::cluster_group cluster = cg::this_cluster();
  const int slices = int(cluster.num_blocks()), slice = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / slices;
  const float* row = a.logits + r * a.ld;
  Row R;
  R.shift = int((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
  R.base = row - R.shift;
  R.V = a.V;
  // this slice's chunks [c0, c1): thread t has c0 + t, c0 + t + kThreads, ..
  const int64_t nc = (a.V + R.shift + 3) / 4;
  const int64_t per_slice = (nc + slices - 1) / slices;
  const int64_t c0 = min(nc, slice * per_slice), c1 = min(nc, c0 + per_slice);
  if (tid == 0) n_owner = n_cand = 0;
  pdl_trigger();
  pdl_wait();

  Pass ps;
  ps.at = c0 + tid;
  {
    constexpr int U = 4;  // 16-byte loads in flight a thread
    int64_t c = c0 + tid;
    // whole chunks only: not the row's first if it is not aligned, nor its last
    const int64_t whole = min(c1, (a.V + R.shift) / 4);
    const float4* p = reinterpret_cast<const float4*>(R.base);
    if (c < c1 && c == 0 && R.shift != 0) {
      const float4 v[1] = {R.load(c)};
      ps.take(v, c);
      c += kThreads;
    }
    for (; c + (U - 1) * kThreads < whole; c += U * kThreads) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = __ldg(p + c + u * kThreads);
      ps.take(v, c);
    }
    for (; c < c1; c += kThreads) {
      const float4 v[1] = {R.load(c)};
      ps.take(v, c);
    }
  }
  auto across = [&](Soft s, int from) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (o > from) continue;
      Soft u;
      u.x = __shfl_xor_sync(0xffffffffu, s.x, o);
      u.l = __shfl_xor_sync(0xffffffffu, s.l, o);
      u.w = __shfl_xor_sync(0xffffffffu, s.w, o);
      merge(s, u);
    }
    return s;
  };
  Soft s = across(ps.s, 16);
  if (lane == 0) soft_s[warp] = s;
  __syncthreads();
  s = across(soft_s[lane % (kThreads / 32)], kThreads / 64);

  // Alternatives.  Each thread's largest key is an element; the n_top-th
  // largest of them bounds the slice's n_top-th largest element from below, and
  // only the n_top threads at or above it can hold an element that is: their
  // elements are looked at again.
  int n = 0;
  if (a.n_top) {
    const u64 mine = ps.at < c1 ? best_key(R, R.load(ps.at), ps.at) : 0ull;
    u64 tau = 0ull;
    for (int b = 63; b >= 0; --b) {
      const u64 t = tau | (1ull << b);
      const int m = __syncthreads_count(mine >= t);
      if (m >= a.n_top) tau = t;
      if (m == a.n_top) break;
    }
    const int64_t per = (c1 - c0 + kThreads - 1) / kThreads;
    if (mine >= tau && mine != 0ull) owner[min(atomicAdd(&n_owner, 1), kMaxTopK - 1)] = tid;
    __syncthreads();
    const bool all = n_owner < a.n_top;  // fewer threads with elements than wanted
    const int64_t todo = all ? c1 - c0 : per * n_owner;
    auto collect = [&](u64 t, bool keep) {
      int m = 0;
      for (int64_t i = tid; i < todo; i += kThreads) {
        const int64_t c = c0 + (all ? i : i / n_owner * kThreads + owner[i % n_owner]);
        if (c >= c1) continue;
        const float4 v = R.load(c);
        const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const u64 k = R.key(x[j], c, j);
          if (k != 0ull && k >= t) {
            ++m;
            if (keep) {
              const int at = atomicAdd(&n_cand, 1);
              if (at < kCand) cand[at] = k;
            }
          }
        }
      }
      return m;
    };
    collect(tau, true);
    __syncthreads();
    if (n_cand > kCand) {
      // more at or above the bound than fit (few threads hold the large ones):
      // raise it, bit by bit, to a value that n_top or a few more reach
      u64 up = 0ull;
      for (int b = 63; b >= 0; --b) {
        const u64 t = up | (1ull << b);
        if (tid == 0) n_s = 0;
        __syncthreads();
        const int m = collect(t > tau ? t : tau, false);
        if (m) atomicAdd(&n_s, m);
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
    const int m = min(n_cand, kCand);
    n = min(m, a.n_top);
    for (int i = tid; i < m; i += kThreads) {
      const u64 k = cand[i];
      int rank = 0;
      for (int j = 0; j < m; ++j) rank += cand[j] > k;
      if (rank < a.n_top) part.top[rank] = k;
    }
  }
  if (tid == 0) part.s = s, part.n = n;

  // The slices meet in the first one's CTA: the states merge, and an
  // alternative's rank is the sum of its ranks in the sorted lists.
  if (slices > 1) {
    cluster.sync();
    if (slice == 0)
      for (int q = 1; q < slices; ++q) merge(s, cluster.map_shared_rank(&part, q)->s);
  } else {
    __syncthreads();
  }
  if (slice == 0) {
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
    for (int i = tid; i < slices * a.n_top; i += kThreads) {
      const int q = i / a.n_top, j = i - q * a.n_top;
      const Part* own = slices > 1 ? cluster.map_shared_rank(&part, q) : &part;
      if (j >= own->n) continue;
      const u64 k = own->top[j];
      int rank = j;
      for (int o = 0; o < slices; ++o) {
        if (o == q) continue;
        const Part* other = cluster.map_shared_rank(&part, o);
        int lo = 0, hi = other->n;  // the number of its keys above k
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (other->top[mid] > k) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      if (rank < a.n_top) {
        a.top_ids[r * a.n_top + rank] = ~uint32_t(k);
        a.top_logprobs[r * a.n_top + rank] = (key_value(k) - s.x) - lz;
      }
    }
  }
  if (slices > 1) cluster.sync();  // no CTA leaves while its part is read
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, cudaStream_t s, int num_sms) {
  if (a.rows == 0) return cudaSuccess;
  // Few rows: a cluster of CTAs a row, up to two CTAs an SM in all and no
  // slice below 4 loads a thread.
  int slices = 1;
  while (slices < 8 && a.rows * slices * 2 <= 2 * num_sms &&
         a.V >= int64_t(slices) * 2 * kThreads * 16)
    slices *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows * slices));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = slices;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel, a);
}

}  // namespace tmg
