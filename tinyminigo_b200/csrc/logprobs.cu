// Log probabilities of given tokens, the entropy of their distributions and
// the top alternatives, per row of logits.  The reference has the softmax of
// its sampler only (src/tensor.rs:1142-1213).
//
// With y_i = x_i - max x, Z = sum e^{y_i}: log p_i = y_i - ln Z and H = ln Z -
// sum e^{y_i} y_i / Z, so one pass that keeps (max, Z, sum e^y y) online gives
// both.  y is taken before the change to base 2 (not x log2 e - max log2 e in
// one fma), so that rows at the type's lowest value stay finite.
//
// The alternatives: every thread remembers the largest of its elements and
// whether a second could count too (its second largest value).  A bound that n
// of the threads' maxima reach is not above the n-th largest element, so the
// elements at or above it hold the answer: the maxima themselves, and those of
// the few threads whose second value reaches it, which alone are read again.
//
// It is bound by the one read of the logits: 2047 rows of 128256 (1.05 GB) take
// 167 us, 6.3 TB/s, 96% of a plain copy's rate, with 8 alternatives and 182
// with 64; in a long run at the power cap's clocks 184.  By 16-byte loads, four
// of them in flight a thread; through a ring of bulk copies in shared memory it
// took 232 us.  One row of 128256 takes 6.6 us (a cluster of 8 CTAs; of 4 7.2,
// one CTA 24.9).
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "kernels.cuh"

namespace tmg {

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
constexpr int kCand = 2048;  // candidates of a slice held in shared memory
constexpr int kSlack = 2;    // threads more than wanted that a bound may let through
constexpr int kMaxSlices = 8;
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
// 4 floats of the row at chunk c of the 16-byte grid its first element
// lies `shift` floats into; elements outside the row read as -inf and
// have no key.
struct Row {
  const float* base;  // 16-byte aligned: the row's start - shift
  int shift;
  int V;
  __device__ __forceinline__ float4 load(int c) const {
    const int i = 4 * c - shift;
    if (i >= 0 && i <= V - 4) return __ldg(reinterpret_cast<const float4*>(base) + c);
    float v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = i + j >= 0 && i < V - j ? __ldg(base + 4 * int64_t(c) + j) : -INFINITY;
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  __device__ __forceinline__ u64 key(float x, int c, int j) const {
    const int i = 4 * c - shift + j;
    return i >= 0 && i < V ? order_key(x, uint32_t(i)) : 0ull;
  }
};

// A thread's pass over its chunks: the online state, the index of the first of
// its largest elements, and the second largest value.
struct Pass {
  Soft s;
  uint32_t idx;
  float second = -INFINITY;
  template <int U>
  __device__ __forceinline__ void take(const float4 (&v)[U], int c, int shift) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      mx = fmaxf(mx, fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w)));
    if (mx > second) {  // a few times a row
      float best = s.x;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float x[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          second = fmaxf(second, fminf(best, x[j]));
          if (x[j] > best) {
            best = x[j];
            idx = uint32_t(4 * (c + u * kThreads) + j - shift);
          }
        }
      }
      if (best > s.x) move(s, best);
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

// The states of a warp's lanes (of lanes that agree in the bits above `from`)
// as one: the largest x first, then sums relative to it.
__device__ __forceinline__ Soft across(Soft s, int from) {
  float x = s.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o <= from) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  if (x > -INFINITY) move(s, x);  // else the sums are 0, or NaN
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o <= from) {
      s.l += __shfl_xor_sync(0xffffffffu, s.l, o);
      s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
    }
  return s;
}

// The slices' results, in the shared memory of the cluster's first CTA.
struct Parts {
  float x[kMaxSlices], l[kMaxSlices], w[kMaxSlices];
  int n[kMaxSlices];  // alternatives in the list, largest first
  u64 top[kMaxSlices][kMaxTopK];
};

__global__ void __launch_bounds__(kThreads, 3) logprobs_kernel(const LogprobsArgs a) {
  constexpr int kW = kThreads / 32;
  __shared__ float soft_s[3][kW];
  __shared__ unsigned or_s[kW], and_s[kW];
  __shared__ u64 cand[kCand];
  __shared__ int owner[kMaxTopK + kSlack];
  __shared__ u64 owner_key[kMaxTopK + kSlack];
  __shared__ int n_owner, n_cand, n_s;
  __shared__ Parts parts;
  cg::cluster_group cluster = cg::this_cluster();
  const int slices = int(cluster.num_blocks()), slice = int(cluster.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r = blockIdx.x / unsigned(slices);
  const float* row = a.logits + r * a.ld;
  const int V = int(a.V);
  Row R;
  R.shift = int((reinterpret_cast<uintptr_t>(row) >> 2) & 3);
  R.base = row - R.shift;
  R.V = V;
  // this slice's chunks [c0, c1): thread t has c0 + t, c0 + t + kThreads, ..
  const int nc = V / 4 + (V % 4 + R.shift + 3) / 4;
  const int per_slice = (nc + slices - 1) / slices;
  const int c0 = min(nc, slice * per_slice), c1 = min(nc, c0 + per_slice);
  if (tid == 0) n_owner = n_cand = 0;
  pdl_trigger();
  pdl_wait();
  // no CTA writes into the first one's memory before that has started
  if (slices > 1) cluster.barrier_arrive();

  float at_target = 0.f;  // thread 0: the target's logit, fetched early
  uint32_t target = 0;
  if (tid == 0 && slice == 0 && a.logprob) {
    target = a.targets[r];
    if (target < uint32_t(V)) at_target = row[target];
  }

  Pass ps;
  ps.idx = uint32_t(max(4 * (c0 + tid) - R.shift, 0));
  {
    constexpr int U = 4;  // 16-byte loads in flight a thread
    int c = c0 + tid;
    // whole chunks only: not the row's first if it is not aligned, nor its last
    const int whole = min(c1, V / 4 + (V % 4 + R.shift) / 4);
    const float4* p = reinterpret_cast<const float4*>(R.base);
    if (c < c1 && c == 0 && R.shift != 0) {
      const float4 v[1] = {R.load(c)};
      ps.take(v, c, R.shift);
      c += kThreads;
    }
    for (; c < whole - (U - 1) * kThreads; c += U * kThreads) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = __ldg(p + c + u * kThreads);
      ps.take(v, c, R.shift);
    }
    // the rest: its loads in flight together too where no other CTA's fill the
    // wait (elsewhere the loads that it has not cost 6 of 167 us)
    if (slices > 1 && c < c1) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = c + u * kThreads;
        v[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at < whole) v[u] = __ldg(p + at);
        else if (at < c1) v[u] = R.load(at);
      }
      ps.take(v, c, R.shift);
      c = c1;
    }
#pragma unroll 1
    for (; c < c1; c += kThreads) {
      const float4 v[1] = {R.load(c)};
      ps.take(v, c, R.shift);
    }
  }
  // for the alternatives, each thread's largest key; and the bits in which
  // their upper halves differ
  u64 mine = 0ull;
  if (a.n_top) {
    if (c0 + tid < c1) mine = order_key(ps.s.x, ps.idx);
    const unsigned hi = unsigned(mine >> 32);
    const unsigned any = __reduce_or_sync(0xffffffffu, hi);
    const unsigned every = __reduce_and_sync(0xffffffffu, mine ? hi : ~0u);
    if (lane == 0) or_s[warp] = any, and_s[warp] = every;
  }
  Soft s = across(ps.s, 16);
  if (lane == 0) soft_s[0][warp] = s.x, soft_s[1][warp] = s.l, soft_s[2][warp] = s.w;
  __syncthreads();
  s.x = soft_s[0][lane % kW], s.l = soft_s[1][lane % kW], s.w = soft_s[2][lane % kW];
  s = across(s, kW / 2);

  // Alternatives.  A thread's largest key is an element; the n_top-th largest of
  // them (or a bound that a few more reach) bounds the slice's n_top-th largest
  // element from below.  The threads at or above it (owners) bring theirs; an
  // owner has others there only if its second largest value reaches the bound
  // too, and only such owners' elements are looked at again: by then they may
  // have left L2 (reading every owner's cost 75 of 250 us for 64 alternatives of
  // 2047 x 128256).
  int n = 0;
  if (a.n_top) {
    const unsigned any = __reduce_or_sync(0xffffffffu, or_s[lane % kW]);
    const unsigned every = __reduce_and_sync(0xffffffffu, and_s[lane % kW]);
    // the bits above the first in which two keys differ are everybody's
    int b = 63 - __clz(any ^ every);
    if (any == every) b = 31;
    u64 tau = b == 63 ? 0ull : u64(every) << 32 >> (b + 1) << (b + 1);
    // (a thread without elements, or fewer than n_top threads: tau stays below)
    if (__syncthreads_count(mine >= tau && mine != 0ull) >= a.n_top) {
#pragma unroll 1
      for (; b >= 0; --b) {
        const u64 t = tau | (1ull << b);
        const int m = __syncthreads_count(mine >= t);
        if (m >= a.n_top) tau = t;
        if (m >= a.n_top && m <= a.n_top + kSlack) break;
      }
    } else {
      tau = 0ull;
    }
    if (mine >= tau && mine != 0ull && order_key(ps.second, 0u) >= tau) {
      const int w = atomicAdd(&n_owner, 1);  // at most n_top + kSlack
      if (w < kMaxTopK + kSlack) owner[w] = tid, owner_key[w] = mine;
    }
    __syncthreads();
    const int owners = min(n_owner, kMaxTopK + kSlack);
    const int per = (c1 - c0 + kThreads - 1) / kThreads;
    auto collect = [&](u64 t, bool keep) {
      int m = 0;
      if (mine >= t && mine != 0ull) {
        ++m;
        if (keep) {
          const int at = atomicAdd(&n_cand, 1);
          if (at < kCand) cand[at] = mine;
        }
      }
#pragma unroll 1
      for (int w = warp; w < owners; w += kW) {
        const int first = c0 + owner[w];
        const u64 had = owner_key[w];
#pragma unroll 1
        for (int i = lane; i < per; i += 32) {
          const int c = first + i * kThreads;
          if (c >= c1) continue;
          const float4 v = R.load(c);
          const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const u64 k = R.key(x[j], c, j);
            if (k != 0ull && k >= t && k != had) {
              ++m;
              if (keep) {
                const int at = atomicAdd(&n_cand, 1);
                if (at < kCand) cand[at] = k;
              }
            }
          }
        }
      }
      return m;
    };
    // more at or above the bound than fit (few threads hold the large ones):
    // raise it, bit by bit, to a value that n_top or a few more reach
#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
      collect(tau, true);
      __syncthreads();
      if (n_cand <= kCand) break;
      u64 up = 0ull;
#pragma unroll 1
      for (int q = 63; q >= 0; --q) {
        const u64 t = up | (1ull << q);
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
      tau = up > tau ? up : tau;
      if (tid == 0) n_cand = 0;
      __syncthreads();
    }
    const int m = min(n_cand, kCand);
    n = min(m, a.n_top);
    if (slices > 1) cluster.barrier_wait();
    u64* top = slices > 1 ? cluster.map_shared_rank(&parts.top[slice][0], 0) : parts.top[0];
#pragma unroll 1
    for (int i = tid; i < m; i += kThreads) {
      const u64 k = cand[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < m; ++j) rank += cand[j] > k;
      if (rank < a.n_top) top[rank] = k;
    }
  } else if (slices > 1) {
    cluster.barrier_wait();
  }

  // The slices meet in the first one's CTA: the states merge, and an
  // alternative's rank is the sum of its ranks in the sorted lists.
  if (slices > 1) {
    if (tid == 0) {
      Parts* p = cluster.map_shared_rank(&parts, 0);
      p->x[slice] = s.x;
      p->l[slice] = s.l;
      p->w[slice] = s.w;
      p->n[slice] = n;
    }
    cluster.sync();
    if (slice != 0) return;
    const int q = lane % kMaxSlices;
    s.x = q < slices ? parts.x[q] : -INFINITY;
    s.l = q < slices ? parts.l[q] : 0.f;
    s.w = q < slices ? parts.w[q] : 0.f;
    s = across(s, kMaxSlices / 2);
  } else {
    if (tid == 0) parts.n[0] = n;
    __syncthreads();
  }
  const float lz = logf(s.l);  // ln Z
  if (tid == 0) {
    if (a.logprob) {
      float lp = NAN;
      if (target < uint32_t(V)) lp = (at_target - s.x) - lz;
      else if (a.err) atomicCAS(a.err, 0, kErrToken);
      a.logprob[r] = lp;
    }
    if (a.entropy) a.entropy[r] = lz - s.w / s.l * kLn2;
  }
  auto put = [&](u64 k, int rank) {
    a.top_ids[r * a.n_top + rank] = ~uint32_t(k);
    a.top_logprobs[r * a.n_top + rank] = (key_value(k) - s.x) - lz;
  };
  if (slices == 1) {
    if (tid < n) put(parts.top[0][tid], tid);
    return;
  }
  // 8 lanes an alternative, a list each: the number of its keys above, bit by bit
#pragma unroll 1
  for (int i = tid; i - lane < slices * a.n_top * kMaxSlices; i += kThreads) {
    const int o = i % kMaxSlices, q = i / kMaxSlices / a.n_top, j = i / kMaxSlices % a.n_top;
    const bool on = q < slices && j < parts.n[q];
    const u64 k = on ? parts.top[q][j] : 0ull;
    const int len = on && o < slices && o != q ? parts.n[o] : 0;
    int above = 0;
#pragma unroll 1
    for (int step = 1 << (31 - __clz(a.n_top)); step > 0; step >>= 1) {
      const u64 v = parts.top[o][min(above + step, kMaxTopK) - 1];
      if (above + step <= len && v > k) above += step;
    }
#pragma unroll
    for (int s = 1; s < kMaxSlices; s <<= 1) above += __shfl_xor_sync(0xffffffffu, above, s);
    if (on && o == 0 && above + j < a.n_top) put(k, above + j);
  }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobsArgs& a, cudaStream_t s, int num_sms) {
  if (a.rows == 0) return cudaSuccess;
  // Few rows: a cluster of CTAs a row, up to the three CTAs that an SM holds
  // and no slice below 4 loads a thread (16 rows of 32003: 7.5 us so, 8.5 with 2).
  int slices = 1;
  while (slices < kMaxSlices && a.rows * slices * 2 <= 3 * num_sms &&
         a.V >= int64_t(slices) * 2 * kThreads * 16)
    slices *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows * slices));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = slices;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel, a);
}

}  // namespace tmg
