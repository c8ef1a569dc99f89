// Decode attention over the 4-bit KV cache (kv4.cuh): per query head of each
// stream, o = sum_t p_t v_t with p = softmax(q . k_t / sqrt(d)) over the
// stream's cached positions (the attention of src/model.rs:434-459, whose
// cache is f32).
//
// With k_t = m + s c over each group of 32 elements (codes c, minimum m, step
// s), q . k_t = sum over groups of s (q . c) + m (sum of q): the products
// with codes are exact 4-bit integers times q, which the warp matrix
// instruction takes as f16, and s and m are applied to 32-bit sums.  q is
// carried as two f16 parts (22 bits, and 2^-35 of the head's largest element at
// least; scaled per head by a power of two so that neither part leaves f16's
// range), the parts as neighbouring columns of one instruction.  Likewise o =
// sum_t (p_t s_t) (c_t - 8) + sum_t p_t (m_t + 8 s_t): p s in two f16 parts; the
// codes centred, since the sums of c and of m alone are hundreds of times larger
// than their sum over a long row.  p is scaled for the sizes of s and m (windows,
// below); values that no such scale serves are summed another way (wide_tile).
//
// What bounds it: at 5 bits an element the memory brings 37 elements a clock
// and SM, so 3.4 lane-instructions an element are all there are; a tile of 64
// positions x 64 (keys and values) takes about 750, 2.9 an element, and the
// schedulers issue in 61 of 100 clocks (both with the fixed parts).  16 streams
// of 32768 positions (32 / 8 heads of 64, 336 MB) take 73 us, 4.6 TB/s, and 77 to
// 81 in a long run at the power cap's clocks; with the arithmetic left out 61 us
// where the whole took 78, and the bytes alone are 51.  One stream of 131072
// positions takes 26 us for 12.8 of bytes: the list's scan and the first tiles
// 3.5 us, the joins 5.  The matrix instructions are mma.sync (m16n8k16): a key
// tile meets 4 heads' two parts in 8 columns, so tcgen05's 128-row tiles with
// operands in shared memory would spend more on writing widened codes than they
// save; the tensor pipe is busy a fifth of the time.  With 5 to 8 query heads a
// kv head (two column tiles) a warp needs up to 254 registers, so an SM has 8
// warps; 9 to 16 make two head groups, each of which loads and widens its kv
// head's tiles for itself.
//
// Tiles come by bulk copies into a ring of each warp's own, so no warp waits for
// another before its head group ends.  (By 16-byte cp.async those 61 us are 76.)
// All tiles of all streams are one list that the CTAs, and in them the warps,
// take equal runs of; a head group that several warps share is joined in shared
// memory, one that several CTAs share by a second kernel.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <math.h>

#include <algorithm>

#include "kv4.cuh"

namespace tmg {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// A warp's tile is TK positions of one head: 64, and 32 for head dim 128, so
// that a tile is 5 KB in both (2560 and 1536 bytes for the small head dims).
// NC: column tiles of 4 query heads.
template <int D, int NC>
struct Cfg {
  static constexpr int G = D < 32 ? D : 32, NG = D / G, TK = D == 128 ? 32 : 64;
  static constexpr int HB = 4 * NC;
  static constexpr int CODE = TK * D / 2, PAR = TK * NG * 4, STAGE = 2 * (CODE + PAR);
  // One CTA an SM: of two, the one that started first runs ahead of the other
  // (65 and 82 us of the same work), of one's warps none does.
  static constexpr int W = NC == 1 ? 16 : 8;        // warps (128 and 255 registers a thread)
  static constexpr int NST = NC == 1 ? 2 : 4;       // stages of a warp's ring
  static constexpr int SLOT = HB * (D + 2);         // floats of a partial result (a multiple of 4)
  static constexpr bool MAP = D == 128;             // tiles by tensor map (swizzled)
  static constexpr int WPL = TK * NG / 32;          // a lane's share of a tile's parameter words
  static constexpr int SMEM = W * (NST * STAGE + SLOT * 4) + 1024;
};

// 2^x by the SFU's ex2 instruction (relative error about 2^-22; 2^-inf = 0)
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / x by the SFU's rcp instruction (relative error about 2^-23)
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8x8 transpose of 16-bit elements over the warp (row = lane / 4)
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
// x's two f16 parts, the upper 11 bits (cut) and the rest, in one word
__device__ __forceinline__ uint32_t two_parts(float x) {
  const float h = __uint_as_float(__float_as_uint(x) & 0xffffe000u);
  return pack_f16(h, x - h);
}
// (x & m) | o in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(m), "r"(o));
  return y;
}
// Two codes in bits 0-3 (or 4-7) of the halves of x to f16 c - 8: 0x6400 | c
// is 1024 + c, 0x6400 | 16 c is 1024 + 16 c; both steps are exact.  (Kim et al., "Who
// Says Elephants Can't Run: Bringing Large Scale MoE Models into Cloud Scale
// Production", 2022, widen integers by such an exponent.)
__device__ __forceinline__ uint32_t centred_lo(uint32_t x) {
  uint32_t y;
  asm("add.rn.f16x2 %0, %1, %2;"
      : "=r"(y)
      : "r"(and_or(x, 0x000f000fu, 0x64006400u)), "r"(0xe408e408u));
  return y;  // - 1032
}
__device__ __forceinline__ uint32_t centred_hi(uint32_t x) {
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;"
      : "=r"(y)
      : "r"(and_or(x, 0x00f000f0u, 0x64006400u)), "r"(0x2c002c00u), "r"(0xd480d480u));
  return y;  // / 16 - 72
}
// Four 8x8 matrices of 16-bit elements, rows of 16 bytes: lane i gives the
// address of row i % 8 of matrix i / 8, and receives of each matrix word t of
// row g (lane = 4 g + t), or, transposed, element g of rows 2 t and 2 t + 1.
__device__ __forceinline__ void ldsm(uint32_t a, uint32_t (&w)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm_t(uint32_t a, uint32_t (&w)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "r"(a));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[N]) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(a));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
  else
    w[0] = lds32(a);
}
__device__ __forceinline__ void tma_tile(void* dst, const CUtensorMap* map, uint64_t* bar, int line,
                                         int seg) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(0), "r"(line), "r"(seg)
      : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
// Byte offset in a tile of 16-byte chunk `c` of row `r`.  Rows of 64 bytes lie
// in 128-byte lines as the tensor map's swizzle writes them (chunk ^ line % 8
// of the line's 8 chunks), so that the words of one chunk of 8 rows lie in 32
// banks.  Shorter rows lie as in memory: 8 rows of 32 bytes meet each bank
// twice at most, which costs less than the swizzle's addresses (82.3 and 88.3 us for 16 x 32768).
template <int D>
__device__ __forceinline__ uint32_t chunk_off(int r, int c) {
  if constexpr (D == 128) {
    constexpr int R = 2;  // rows a line
    return (r / R) * 128 + ((((r % R) * (D / 32) + c) ^ (r / R % 8)) << 4);
  }
  return r * (D / 2) + c * 16;
}
// a b + c of two f32 pairs in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 twice(float x) { return make_float2(x, x); }

// A tile's window: a power of two 2^K, as its bf16 pattern (K + 127) << 7, such
// that every step s and minimum m of the tile's values has
//   max(s, |m| / 8) >= 2^(K - kDepth),  s <= 2^K,  |m| <= 2^(K + kMinima)
// (a group of zeros aside, see the kernel), K within +-kFar.  Weights are scaled so
// that p 2^K is at most 2^16, thus p s fits f16, and 2^11 at least for the largest
// weight when it comes, where p max(s, |m| / 8) is then 2^-1: what the two f16 parts
// of p s leave out of a position (2^-25, times codes of up to 8) is as small beside
// that as a rounding of f32.  Sums of p |m| over up to 2^31 positions stay below
// 2^(16 + 36 + 31), and moved to another window (by 2^40) below 2^123.
constexpr int kDepth = 12, kMinima = 36, kFar = 20;
constexpr int kNoWindow = 0x7fff;  // no value passes it
__device__ __forceinline__ int window_of(int K) { return (K + 127) << 7; }
// The window that steps up to s_max, minima up to m_max and a least max(s, |m| / 8)
// of `low` fit (all as bf16 patterns; without any, s_max = m_max = 0 and low =
// 0x7f80): `now` if it does, else one with some room for larger steps, `cap` at most.
__device__ __forceinline__ int fit_window(int now, int cap, int s_max, int m_max, int low) {
  if (s_max <= now && m_max <= now + (kMinima << 7) && low >= now - (kDepth << 7)) return now;
  const int least = max(max((s_max + 0x7f) & ~0x7f, ((m_max + 0x7f) & ~0x7f) - (kMinima << 7)),
                        window_of(-kFar));
  const int most = min((low & ~0x7f) + (kDepth << 7), cap);
  return least <= most ? min(least + (3 << 7), most) : kNoWindow;
}

// The tiles of all streams, in order of (stream, head group, tile).
struct Plan {
  AttnKv4Args a;
  int gh, gsh;    // query heads a head group; log2 of a kv head's head groups
  int VH;         // head groups a stream
  bool split;     // CTAs take equal runs of tiles (else one head group each)
  float* part;    // [grid, 2] partial results: weighted means, reference points, sums of weights
};
// Tiles of TK that hold n positions (n up to 2^31 - 1).
template <int TK>
__device__ __forceinline__ int tiles_of(int n) {
  return int((uint32_t(n) + (TK - 1)) / TK);
}
__device__ __forceinline__ int clamped_len(const AttnKv4Args& a, int m) {
  return min(max(a.lens[m], 0), int(a.max_len));
}
// `total` tiles dealt out to n CTAs (n <= total): the first r take q + 1, the
// others q.
struct Deal {
  int q, r;
  __device__ __forceinline__ Deal(int total, int n) : q(total / n) { r = total - q * n; }
  __device__ __forceinline__ int first(int b) const { return b * q + min(b, r); }
  // the CTA that takes tile T
  __device__ __forceinline__ int owner(int T) const {
    const int wide = r * (q + 1);
    return T < wide ? T / (q + 1) : r + (T - wide) / q;
  }
};

// A head group and the tile that a warp has reached in it.
struct Cursor {
  int m, vh, tile, nt;
};

// Wide mode: values that no window holds (steps or minima of one tile far apart,
// near the ends of f32, or much larger than those before).  There p is at most 1, cm
// is 0 and o counts in units of 2^unit[head][group], a bound of p |v| so far, to
// which each product goes as a 64-bit number; so it is as exact as 32-bit sums, and
// neither |v| nor what p leaves of it can leave f32.  A tile takes some 10 times as
// long so (all of 16 x 32768: 804 us).  It ends with a tile whose window holds what
// the sums hold, too.  A function of its own, called
// for such tiles only: in the loop its registers would cost every tile (8 heads of
// 128 a kv head: 130 us and not 115).
template <int D, int NC>
struct Wide {
  using C = Cfg<D, NC>;
  static constexpr int NG = C::NG, KB = C::TK / 16, OD = D == 16 ? 2 : 4;
  float x[NC][2 * KB], cq[NC], ref[NC], l[NC], cm[NC][NG], o[NC][NG][OD];
  float shift[NC];  // log2 of what the sums so far are multiplied by
};
template <int D, int NC>
__device__ __noinline__ void wide_tile(Wide<D, NC>& w, int (*unit)[Cfg<D, NC>::NG], uint32_t base,
                                       int valid, bool first) {
  using C = Cfg<D, NC>;
  constexpr int NG = C::NG, KB = C::TK / 16, OD = D == 16 ? 2 : 4;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  __syncwarp();
#pragma unroll 1
  for (int k = 0; k < NC; ++k) {
    const float al = ex2_approx(w.shift[k]);
    w.l[k] *= al;
#pragma unroll
    for (int i = 0; i < 2 * KB; ++i) {
      w.x[k][i] = ex2_approx(fmaf(w.x[k][i], w.cq[k], -w.ref[k]));  // p from here on
      w.l[k] += w.x[k][i];
    }
#pragma unroll 1
    for (int j = 0; j < NG; ++j) {
      float o[OD];
#pragma unroll
      for (int i = 0; i < OD; ++i) o[i] = w.o[k][j][i];
      int e = unit[4 * k + t][j];
      if (first) {  // o and cm as the other tiles left them
        float c = w.cm[k][j], big = 0.f;
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) c += __shfl_xor_sync(0xffffffffu, c, s);
#pragma unroll
        for (int i = 0; i < OD; ++i) big = fmaxf(big, fabsf(o[i] += c));
#pragma unroll
        for (int s = 4; s < 32; s <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
        e = big > 0.f ? ilogbf(big) + 1 : -4000;
#pragma unroll
        for (int i = 0; i < OD; ++i) o[i] = scalbnf(o[i], -e);
      }
      // times 2^shift
      const float whole = floorf(w.shift[k]);
      const float part = w.shift[k] <= -4000.f ? 0.f : ex2_approx(w.shift[k] - whole);
      e = max(e + int(fmaxf(whole, -4000.f)), -4000);
      // the exponent above the largest p |v| of the tile
      int up = e;
#pragma unroll 1
      for (int i = 0; i < 2 * KB; ++i) {
        const uint32_t par = 8 * i + g < valid
            ? lds32(base + 2 * C::CODE + C::PAR + ((8 * i + g) * NG + j) * 4) : 0u;
        const double m = kv4_min(par), s = kv4_step(par);
        const double y = double(w.x[k][i]) * fmax(fabs(m), fabs(fma(15.0, s, m)));
        if (y > 0.0) up = max(up, (__double2hiint(y) >> 20) - 1022);
      }
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) up = max(up, __shfl_xor_sync(0xffffffffu, up, s));
#pragma unroll
      for (int i = 0; i < OD; ++i) o[i] = scalbnf(o[i] * part, e - up);
      const double to_unit = __hiloint2double((1023 - max(up, -1000)) << 20, 0);
#pragma unroll 1
      for (int i = 0; i < 2 * KB; ++i)
#pragma unroll 1
        for (int r = 8 * i; r < min(8 * i + 8, valid); ++r) {
          const double p =
              double(__shfl_sync(0xffffffffu, w.x[k][i], 4 * (r & 7) + t)) * to_unit;
          const uint32_t par = lds32(base + 2 * C::CODE + C::PAR + (r * NG + j) * 4);
          uint32_t codes;
          if constexpr (D == 16) codes = lds8(base + C::CODE + r * 8 + g);
          else codes = lds16(base + C::CODE + chunk_off<D>(r, j) + 2 * g);
#pragma unroll
          for (int n = 0; n < OD; ++n)
            o[n] += float(p * double(fmaf(float(codes >> (4 * n) & 15u), kv4_step(par),
                                          kv4_min(par))));
        }
#pragma unroll
      for (int i = 0; i < OD; ++i) w.o[k][j][i] = o[i];
      __syncwarp();
      if (g == 0) unit[4 * k + t][j] = up;
    }
  }
  __syncwarp();
}

template <int D, int NC>
__global__ void __launch_bounds__(Cfg<D, NC>::W * 32, 1)
    attn_kv4_kernel(const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap, const Plan pl) {
  using C = Cfg<D, NC>;
  constexpr int G = C::G, NG = C::NG, TK = C::TK, KB = TK / 16, HB = C::HB, kWarps = C::W;
  constexpr int OD = D == 16 ? 2 : 4;  // output dims a lane and group
  extern __shared__ uint8_t smem[];
  // 1024: the period of the swizzle (a stage is a multiple of it)
  uint8_t* ring = smem + (-smem_u32(smem) & 1023u);
  __shared__ __align__(8) uint64_t full[kWarps][C::NST];
  __shared__ int pre[kKv4MaxStreams + 1];  // tiles before each stream
  __shared__ int scan_s[kWarps];
  __shared__ float far_s[kWarps][2][HB];
  // a head group's window as two bounds (set_window), and as it is; the groups of zeros
  // and others that it has had
  __shared__ __align__(16) uint32_t bounds_s[kWarps][4];
  __shared__ int window_s[kWarps][2];
  __shared__ int unit_s[kWarps][HB][NG];  // exponents of o (wide mode)
  __shared__ int slot_seg[2 * kWarps];  // head group of each warp's partials, -1: none
  const AttnKv4Args& a = pl.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int M = a.kv.M, VH = pl.VH;

  if (tid < kWarps * C::NST) mbar_init(&full[0][0] + tid, 1);
  if (tid < 2 * kWarps) slot_seg[tid] = -1;
  if constexpr (C::MAP)
    if (tid == 0) {
      prefetch_map(&kmap);
      prefetch_map(&vmap);
    }
  mbar_fence_init();
  pdl_wait();
  // The join may start.  It reads lens before it waits for this kernel, so the
  // trigger stays behind the wait: what wrote lens has then ended.
  pdl_trigger();

  auto checked_tiles = [&](int m) {
    const int len = a.lens[m];
    if ((len < 0 || len > a.max_len) && a.err) atomicCAS(a.err, 0, kErrLength);
    return tiles_of<TK>(clamped_len(a, m));
  };
  // this CTA's tiles [c0, c1)
  int c0, c1;
  if (pl.split) {
    // tiles (of one head group) before each stream: by the first warp, or 4
    // streams a thread, scanned over the CTA
    if (M <= 32) {
      if (warp == 0) {
        const int n = lane < M ? checked_tiles(lane) : 0;
        int inc = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        if (lane <= M) pre[lane] = inc - n;
        if (M == 32 && lane == 31) pre[32] = inc;
      }
    } else {
      int n[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        n[i] = 4 * tid + i < M ? checked_tiles(4 * tid + i) : 0;
        sum += n[i];
      }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (lane == 31) scan_s[warp] = inc;
      __syncthreads();
      int at = inc - sum;
      for (int w = 0; w < warp; ++w) at += scan_s[w];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (4 * tid + i <= M) pre[4 * tid + i] = at;
        at += n[i];
      }
      if (M == kKv4MaxStreams && tid == kWarps * 32 - 1) pre[M] = at;
    }
    __syncthreads();
    const int total = pre[M] * VH, ctas = min(int(gridDim.x), total);
    if (int(blockIdx.x) >= ctas) return;
    const Deal deal(total, ctas);
    c0 = deal.first(blockIdx.x);
    c1 = deal.first(blockIdx.x + 1);
  } else {  // one head group: its tiles count from 0
    const int m = blockIdx.x / VH, vh = blockIdx.x - m * VH;
    c0 = 0;
    c1 = checked_tiles(m);
    if (c1 == 0) {  // an empty stream
      const int per = a.nq / a.kv.nkv, h0 = (vh & ((1 << pl.gsh) - 1)) * pl.gh;
      float* o = a.out + int64_t(m) * a.out_ld + int64_t((vh >> pl.gsh) * per + h0) * D;
      for (int i = tid; i < min(pl.gh, per - h0) * D; i += blockDim.x) o[i] = 0.f;
      return;
    }
    __syncthreads();  // the mbarriers and slots above
  }
  const int w0 = c0 + (c1 - c0) * warp / kWarps, w1 = c0 + (c1 - c0) * (warp + 1) / kWarps;

  uint8_t* my_ring = ring + warp * C::NST * C::STAGE;
  float* first_slot = reinterpret_cast<float*>(ring + kWarps * C::NST * C::STAGE) + warp * C::SLOT;
  float* last_slot = reinterpret_cast<float*>(my_ring);  // once the ring is done with
  bool alive = true;

  auto locate = [&](int tile) {
    Cursor c;
    if (!pl.split) {
      c.m = blockIdx.x / VH;
      c.vh = blockIdx.x - c.m * VH;
      c.tile = tile;
      c.nt = c1;
      return c;
    }
    int lo = 0, hi = M - 1;  // the last stream with pre[m] VH <= tile
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] * VH <= tile) lo = mid;
      else hi = mid - 1;
    }
    c.m = lo;
    c.nt = pre[lo + 1] - pre[lo];
    const int r = tile - pre[lo] * VH;
    c.vh = r / c.nt;
    c.tile = r - c.vh * c.nt;
    return c;
  };
  auto advance = [&](Cursor& c) {
    if (++c.tile < c.nt) return;
    c.tile = 0;
    if (!pl.split || ++c.vh < VH) return;
    c.vh = 0;
    do ++c.m;
    while (c.m < M && pre[c.m + 1] == pre[c.m]);
    if (c.m < M) c.nt = pre[c.m + 1] - pre[c.m];
  };
  // the query heads of head group vh: the first and their number
  const int per = a.nq / a.kv.nkv, gmask = (1 << pl.gsh) - 1;
  auto first_head = [&](int vh) { return (vh >> pl.gsh) * per + (vh & gmask) * pl.gh; };
  auto n_heads = [&](int vh) { return min(pl.gh, per - (vh & gmask) * pl.gh); };
  // load tile `c` into stage st (one lane)
  auto load = [&](const Cursor& c, int64_t par, int seg, int st) {
    const int row = c.tile * TK;
    const int n = min(TK, int(a.kv.cap) - row);  // a multiple of 4
    uint8_t* s = my_ring + st * C::STAGE;
    uint64_t* bar = &full[warp][st];
    const uint32_t pb = n * NG * 4;
    if constexpr (C::MAP) {
      mbar_expect_tx(bar, 2 * (C::CODE + pb));
      tma_tile(s, &kmap, bar, row / (256 / D), seg);
      tma_tile(s + C::CODE, &vmap, bar, row / (256 / D), seg);
    } else {
      const uint32_t cb = n * (D / 2);
      mbar_expect_tx(bar, 2 * (cb + pb));
      bulk_g2s(s, a.kv.kc + par * (G / 2), cb, bar);
      bulk_g2s(s + C::CODE, a.kv.vc + par * (G / 2), cb, bar);
    }
    bulk_g2s(s + 2 * C::CODE, a.kv.kp + par, pb, bar);
    bulk_g2s(s + 2 * C::CODE + C::PAR, a.kv.vp + par, pb, bar);
  };
  // cache head and index of the first parameter word of tile `c`
  auto head_of = [&](const Cursor& c) { return c.m * a.kv.nkv + (c.vh >> pl.gsh); };
  auto par_of = [&](const Cursor& c) {
    return (int64_t(head_of(c)) * a.kv.cap + c.tile * TK) * NG;
  };

  // state of the head group: query head t (+ 4 c) of the lane; its output
  // dims 4 g .. (2 g .. for head dim 16) of each group
  float ref[NC], l[NC], cm[NC][NG], o[NC][NG][OD], cq[NC], qs[NC][NG];
  uint32_t qb[NC][NG][4];
  // as an operand the lane holds head g / 2 (part g % 2), of each group the
  // elements that lane t's code words hold
  constexpr int E = D == 16 ? 4 : 8;
  auto load_q = [&](const Cursor& c, float4 (&v)[NC][NG][E / 4]) {
    const int heads = n_heads(c.vh);
    const float* q = a.q + int64_t(c.m) * a.q_ld + int64_t(first_head(c.vh)) * D;
#pragma unroll
    for (int k = 0; k < NC; ++k)
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
          const int h = 4 * k + g / 2;
          v[k][j][i] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (h < heads)
            v[k][j][i] = *reinterpret_cast<const float4*>(q + h * D + j * G + t * E + 4 * i);
        }
  };
  // Scores beyond 2^20 (in powers of two), where one rounding of a reference
  // point would be a factor, or queries whose cq would leave f32: from there on
  // to the head group's end x holds e - M, e the rounded exponent and M the
  // largest so far, cq is 1 (which a product with log2 e never is) and ref
  // counts from M.  cq (without its 2^24) and M of head h: far_s[warp][..][h].
  auto go_far = [&](float room) {
    __syncwarp();
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      far_s[warp][0][4 * k + t] = cq[k];
      far_s[warp][1][4 * k + t] = ref[k] + room;
      if (ref[k] > -INFINITY) ref[k] = -room;
      cq[k] = 1.f;
    }
    __syncwarp();
  };
  // The head group's window; that which the next tile is tested against (none: always
  // off); its groups of zeros (bits 0-3) and others (4-7).
  auto set_window = [&](int now, int test, unsigned zn) {
    __syncwarp();
    if (lane == 0) {
      bounds_s[warp][0] = test * 0x10001u + (kMinima << 23);
      bounds_s[warp][1] = 0x80000000u | (test - (kDepth << 7));
      bounds_s[warp][2] =
          __float_as_uint(test == kNoWindow ? -INFINITY : 15.98f + 127 - (test >> 7));
      window_s[warp][0] = now, window_s[warp][1] = zn;
    }
    __syncwarp();
  };
  auto start = [&](const float4 (&q)[NC][NG][E / 4]) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float x[NG][E];
      float big = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int i = 0; i < E; i += 4) {
          const float4 v = q[k][j][i / 4];
          x[j][i] = v.x, x[j][i + 1] = v.y, x[j][i + 2] = v.z, x[j][i + 3] = v.w;
          big = fmaxf(big, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      // a power of two that takes the largest |q| to 2^14 .. 2^15
      const int e = min(268 - int(__float_as_uint(big) >> 23), 253);
      const float up = __uint_as_float(uint32_t(e) << 23);
      const int src = 8 * t;  // a lane that holds head t (+ 4 k) as an operand
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float sum = 0.f;
        uint32_t w[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
          x[j][i] *= up;
          sum += x[j][i];
          // odd codes enter as 16 c
          w[i] = two_parts(x[j][i] * (i & 1 ? 0.0625f : 1.f));
          w[i] = g & 1 ? w[i] >> 16 : w[i] & 0xffffu;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        // codes enter as f16 numbers c * 2^-24
        qs[k][j] = __shfl_sync(0xffffffffu, sum, src) * 0x1p-24f;
        constexpr int S = E / 2;  // the two codes of an operand word
#pragma unroll
        for (int i = 0; i < S; ++i) qb[k][j][i] = w[i] | (w[i + S] << 16);
        if constexpr (E == 4) qb[k][j][2] = qb[k][j][3] = 0u;
      }
      const float un = __uint_as_float(uint32_t(254 - e) << 23);
      cq[k] = __shfl_sync(0xffffffffu, un, src) * (a.scale * kLog2e);
      ref[k] = -INFINITY;
      l[k] = 0.f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        cm[k][j] = 0.f;
#pragma unroll
        for (int i = 0; i < OD; ++i) o[k][j][i] = 0.f;
      }
    }
    set_window(window_of(0), window_of(0), 0);  // a first guess, for values of ordinary size
    bool over = false;
#pragma unroll
    for (int k = 0; k < NC; ++k) over |= cq[k] >= 0x1p100f;
    if (__any_sync(0xffffffffu, over)) {
      go_far(0.f);
    } else {
#pragma unroll
      for (int k = 0; k < NC; ++k) cq[k] *= 0x1p24f;
    }
  };
  // the sums over the lanes that share a head (each had its own positions): o
  // becomes the weighted mean of the values, which f32 holds whatever they are
  auto finish = [&]() {
    __syncwarp();
    const bool wide = window_s[warp][0] == kNoWindow;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
#pragma unroll
      for (int s = 4; s < 32; s <<= 1) {
        l[k] += __shfl_xor_sync(0xffffffffu, l[k], s);
#pragma unroll
        for (int j = 0; j < NG; ++j) cm[k][j] += __shfl_xor_sync(0xffffffffu, cm[k][j], s);
      }
      const float f = rcp_approx(l[k]);
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int i = 0; i < OD; ++i) {
          o[k][j][i] = (o[k][j][i] + cm[k][j]) * f;
        }
    }
    if (wide) {
#pragma unroll
      for (int k = 0; k < NC; ++k)
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          const int e = max(unit_s[warp][4 * k + t][j], -252), h = e >> 1;
#pragma unroll
          for (int i = 0; i < OD; ++i)
            o[k][j][i] = o[k][j][i] * __int_as_float((h + 127) << 23) *
                         __int_as_float((e - h + 127) << 23);
        }
    }
    if (cq[0] == 1.f) {  // sums relative to M, so that M alone is the reference point
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const float f = ex2_approx(0.5f * ref[k]);
        l[k] = l[k] * f * f;
        ref[k] = far_s[warp][1][4 * k + t];
      }
    }
  };
  auto write_out = [&](const Cursor& c) {
    const int heads = n_heads(c.vh);
    float* out = a.out + int64_t(c.m) * a.out_ld + int64_t(first_head(c.vh)) * D;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int h = 4 * k + t;
      if (h >= heads) continue;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float* p = out + h * D + j * G + g * OD;
        if constexpr (OD == 4)
          *reinterpret_cast<float4*>(p) = make_float4(o[k][j][0], o[k][j][1], o[k][j][2], o[k][j][3]);
        else
          *reinterpret_cast<float2*>(p) = make_float2(o[k][j][0], o[k][j][1]);
      }
    }
  };
  auto write_slot = [&](float* s) {
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int h = 4 * k + t;
#pragma unroll
      for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int i = 0; i < OD; ++i) s[h * D + j * G + g * OD + i] = o[k][j][i];
      if (g == 0) s[HB * D + h] = ref[k], s[HB * D + HB + h] = l[k];
    }
  };

  if (w0 < w1) {
    Cursor cur = locate(w0), nxt = cur;
    int64_t nxt_par = par_of(nxt);
    int nxt_head = head_of(nxt);
    auto fetch = [&](int st) {
      if (lane == 0) load(nxt, nxt_par, nxt_head, st);
      advance(nxt);
      nxt_par += TK * NG;
      if (nxt.tile == 0) {
        nxt_par = par_of(nxt);
        nxt_head = head_of(nxt);
      }
    };
    float4 q[NC][NG][E / 4];
    load_q(cur, q);
    int len = clamped_len(a, cur.m);
    for (int i = 0; i < C::NST && w0 + i < w1; ++i) fetch(i);
    const int seg_first = cur.m * VH + cur.vh;
    start(q);
    bool whole = cur.tile == 0;  // the head group began in this warp
    int st = 0;
    uint32_t phase = 0;
    for (int T = w0; T < w1; ++T) {
      if (!mbar_wait_warp(&full[warp][st], phase)) {
        if (lane == 0 && a.err) atomicCAS(a.err, 0, 2);
        alive = false;
        break;
      }
      const uint32_t base = smem_u32(my_ring + st * C::STAGE);
      const int valid = len - cur.tile * TK;  // positions of the tile in the row

      // scores of positions 16 b + 8 i + g, x[][2 b + i]
      float x[NC][2 * KB];
#pragma unroll
      for (int b = 0; b < KB; ++b) {
#pragma unroll
        for (int k = 0; k < NC; ++k) x[k][2 * b] = x[k][2 * b + 1] = 0.f;
      }
#pragma unroll
      for (int b2 = 0; b2 < KB; b2 += 2) {
        uint32_t par[4][NG];  // parameters of the rows 16 b2 + 8 i + g
#pragma unroll
        for (int i = 0; i < 4; ++i)
          lds_words<NG>(base + 2 * C::CODE + (16 * b2 + 8 * i + g) * NG * 4, par[i]);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          uint32_t w[4];  // code words of those rows
          if constexpr (D == 16) {  // two bytes: one to each half
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = __byte_perm(lds32(base + (16 * b2 + 8 * i + g) * 8 + (t >> 1) * 4), 0u,
                                 t & 1 ? 0x4342u : 0x4140u);
          } else {
            ldsm(base + chunk_off<D>(16 * b2 + lane, j), w);
          }
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const int b = b2 + i / 2;
            const uint32_t u = w[i], v = w[i + 1];
            const float s0 = kv4_step(par[i][j]), m0 = kv4_min(par[i][j]);
            const float s1 = kv4_step(par[i + 1][j]), m1 = kv4_min(par[i + 1][j]);
#pragma unroll
            for (int k = 0; k < NC; ++k) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              // codes as f16 numbers below 1: c * 2^-24, 16 c * 2^-24
              mma_f16(c, u & 0x000f000fu, v & 0x000f000fu, u & 0x00f000f0u, v & 0x00f000f0u,
                      qb[k][j][0], qb[k][j][1]);
              if constexpr (D > 16)
                mma_f16(c, (u >> 8) & 0x000f000fu, (v >> 8) & 0x000f000fu,
                        (u >> 8) & 0x00f000f0u, (v >> 8) & 0x00f000f0u, qb[k][j][2], qb[k][j][3]);
              const float2 v2 =
                  fma2(make_float2(s0, s1), make_float2(c[0] + c[1], c[2] + c[3]),
                       fma2(make_float2(m0, m1), twice(qs[k][j]),
                            make_float2(x[k][2 * b], x[k][2 * b + 1])));
              x[k][2 * b] = v2.x;
              x[k][2 * b + 1] = v2.y;
            }
          }
        }
      }
      uint32_t pv[2 * KB][NG];  // the values' parameters of the same positions
#pragma unroll
      for (int i = 0; i < 2 * KB; ++i)
        lds_words<NG>(base + 2 * C::CODE + C::PAR + (8 * i + g) * NG * 4, pv[i]);
      // a share of them: word i is of position (lane WPL + i) / NG, group i % NG
      uint32_t pw[C::WPL];
      lds_words<C::WPL>(base + 2 * C::CODE + C::PAR + lane * C::WPL * 4, pw);
      uint32_t bounds[4];
      lds_words<4>(smem_u32(bounds_s[warp]), bounds);
      if (valid < TK) {
#pragma unroll
        for (int i = 0; i < 2 * KB; ++i)
          if (8 * i + g >= valid) {  // whatever the rows behind the last hold
#pragma unroll
            for (int k = 0; k < NC; ++k) x[k][i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < NG; ++j) pv[i][j] = 0u;
          }
#pragma unroll
        for (int i = 0; i < C::WPL; ++i)
          if ((lane * C::WPL + i) / NG >= valid) pw[i] = bounds[0] & 0xffffu;  // m = 0, s = 2^K
      }

      // p = 2^(x cq - ref), where ref is a bound of the row's exponents so far plus K
      // less 12: p times a step stays in f16's range, with 2^4 to spare before ref has
      // to grow.  The tile's parameters are held against the window (fit_window) as
      // pairs of 16 bits, signed and unsigned: the unsigned maximum has the steps' and
      // the largest negative minimum, the signed one the largest positive minimum.  A
      // NaN step is above all.
      uint32_t most = __vmaxu2(pw[0], pw[1]), most_s = __vmaxs2(pw[0], pw[1]);
      uint32_t least = __vmins2(pw[0], pw[1]);
      if constexpr (C::WPL == 4) {
        most = __vimax3_u16x2(most, pw[2], pw[3]);
        most_s = __vimax3_s16x2(most_s, pw[2], pw[3]);
        least = __vimin3_s16x2(least, pw[2], pw[3]);
      }
      const bool off = __vimax3_s16x2(most & 0x7fffffffu, most_s, bounds[0]) != bounds[0] ||
                       __vmins2(least, bounds[1]) != bounds[1];
      float p[NC][2 * KB];
      float top[NC];
      bool grow = off || cq[0] == 1.f;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        top[k] = x[k][0];
#pragma unroll
        for (int i = 1; i < 2 * KB; ++i) top[k] = fmaxf(top[k], x[k][i]);
        grow |= !(fmaf(top[k], cq[k], -ref[k]) <= __uint_as_float(bounds[2]));
      }
      bool wide = false;
      if (__any_sync(0xffffffffu, grow)) {
        int was_w = window_s[warp][0], now = was_w;
        if (__any_sync(0xffffffffu, off)) {
          // the tile's window (NaN groups do not count), and which of its groups have
          // zeros (z) or others (n)
          int s_max = 0, m_max = 0, low = 0x7f80;
          unsigned zn = 0;
#pragma unroll
          for (int i = 0; i < C::WPL; ++i) {
            const int s = pw[i] & 0x7fff, m = pw[i] >> 16 & 0x7fff;
            if (s >= 0x7f80 || (lane * C::WPL + i) / NG >= valid) continue;
            const int b = max(s, m - (3 << 7));
            zn |= (b > 0 ? 16u : 1u) << (i % NG);
            if (b > 0) s_max = max(s_max, s), m_max = max(m_max, m), low = min(low, b);
          }
          zn = __reduce_or_sync(0xffffffffu, zn);
          unsigned had = window_s[warp][1];
          int cap = window_of(kFar);
          if (was_w != kNoWindow) {
            // What the tiles before hold is 2^(K - kDepth) at least, by their window, so
            // it may fall but not rise (but before the first).
            if (had) cap = was_w;
          } else {
            // What the sums hold by now: 2^(e - 1) at least, max(s, |m| / 8) being a
            // quarter of b or more.
            had = 0;
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
              for (int j = 0; j < NG; ++j) {
                const int e = unit_s[warp][4 * k + t][j];
                if (e == -4000 && (zn >> j & 0x11u) == 1u) continue;  // zeros, and still
                had |= 16u << j;
                low = min(low, max(e - 3 + 127, 0) << 7);
                m_max = max(m_max, max(e + 127, 0) << 7);
              }
            had = __reduce_or_sync(0xffffffffu, had);
          }
          s_max = __reduce_max_sync(0xffffffffu, s_max);
          m_max = __reduce_max_sync(0xffffffffu, m_max);
          low = __reduce_min_sync(0xffffffffu, low);
          // A group with zeros and others has no window: the zeros may have all the
          // weight that ref counts from.
          zn |= had;
          now = zn & zn >> 4 & 15u ? kNoWindow : fit_window(was_w, cap, s_max, m_max, low);
          wide = now == kNoWindow;
          if (was_w == kNoWindow && !wide) {  // o as other tiles have it
#pragma unroll
            for (int k = 0; k < NC; ++k)
#pragma unroll
              for (int j = 0; j < NG; ++j) {
                const float f =
                    __int_as_float((max(unit_s[warp][4 * k + t][j], -126) + 127) << 23);
#pragma unroll
                for (int i = 0; i < OD; ++i) o[k][j][i] *= f;
              }
          }
          // (tiles that pass the test later have no group of zeros)
          if (wide || (zn & 15u)) set_window(now, kNoWindow, zn);
          else set_window(now, now, 0xf0u);
        } else if (lane == 0) {
          window_s[warp][1] = 0xf0;
        }
        // (of wide mode: p of at most 1)
        auto room_of = [](int w) { return w == kNoWindow ? 0.f : float(12 + 127 - (w >> 7)); };
        const float room = room_of(now), was_room = room_of(was_w);
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int s = 4; s < 32; s <<= 1)
            top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], s));
        if (cq[0] != 1.f) {
          bool over = false;
#pragma unroll
          for (int k = 0; k < NC; ++k) over |= fabsf(top[k] * cq[k]) >= 0x1p20f;
          if (__any_sync(0xffffffffu, over)) {
#pragma unroll
            for (int k = 0; k < NC; ++k) cq[k] *= 0x1p-24f;
            go_far(was_room);
          }
        }
        float shift[NC];  // log2 of what the sums so far are multiplied by
#pragma unroll
        for (int k = 0; k < NC; ++k) shift[k] = 0.f;
        if (cq[0] == 1.f) {
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            const float c = far_s[warp][0][4 * k + t], was = far_s[warp][1][4 * k + t];
            // (the order in which no product leaves f32 that e does not)
            const float c0 = c < 1.f ? c : 0x1p24f, c1 = c < 1.f ? 0x1p24f : c;
            auto e = [&](float x) { return __fmul_rn(__fmul_rn(x, c0), c1); };  // (no fma: M is one)
            top[k] = e(top[k]);
            const float M = fmaxf(was, top[k]);
            if (M > -INFINITY) {
              shift[k] = was - M;
#pragma unroll
              for (int i = 0; i < 2 * KB; ++i) x[k][i] = e(x[k][i]) - M;
              top[k] -= M;
            }
            __syncwarp();
            far_s[warp][1][4 * k + t] = M;
            __syncwarp();
          }
        }
        // ref moves with the window and grows, in whole numbers, so that the sums
        // move by powers of two
#pragma unroll
        for (int k = 0; k < NC; ++k) {
          const float r = fmaxf(ref[k] + (was_room - room), ceilf(top[k] * cq[k]) - room);
          shift[k] += ref[k] - r;
          ref[k] = r;
        }
        if (wide) {
          Wide<D, NC> w;
#pragma unroll
          for (int k = 0; k < NC; ++k) {
#pragma unroll
            for (int i = 0; i < 2 * KB; ++i) w.x[k][i] = x[k][i];
            w.cq[k] = cq[k], w.ref[k] = ref[k], w.l[k] = l[k], w.shift[k] = shift[k];
#pragma unroll
            for (int j = 0; j < NG; ++j) {
              w.cm[k][j] = cm[k][j];
              cm[k][j] = 0.f;
#pragma unroll
              for (int i = 0; i < OD; ++i) w.o[k][j][i] = o[k][j][i];
            }
          }
          wide_tile<D, NC>(w, unit_s[warp], base, valid, was_w != kNoWindow);
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            l[k] = w.l[k];
#pragma unroll
            for (int j = 0; j < NG; ++j)
#pragma unroll
              for (int i = 0; i < OD; ++i) o[k][j][i] = w.o[k][j][i];
          }
        } else {
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            const float al = ex2_approx(shift[k]);
            l[k] *= al;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
              cm[k][j] *= al;
#pragma unroll
              for (int i = 0; i < OD; ++i) o[k][j][i] *= al;
            }
          }
        }
      }
      if (!wide) {
#pragma unroll
        for (int k = 0; k < NC; ++k)
#pragma unroll
          for (int i = 0; i < 2 * KB; ++i) {
            p[k][i] = ex2_approx(fmaf(x[k][i], cq[k], -ref[k]));
            l[k] += p[k][i];
          }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          uint32_t pb[NC][2 * KB];
#pragma unroll
          for (int i = 0; i < 2 * KB; ++i) {
            const float s = kv4_step(pv[i][j]), c8 = fmaf(8.f, s, kv4_min(pv[i][j]));
#pragma unroll
            for (int k = 0; k < NC; ++k) {
              cm[k][j] = fmaf(p[k][i], c8, cm[k][j]);
              pb[k][i] = transpose8(two_parts(p[k][i] * s));
            }
          }
          float c[NC][2][4] = {};
          uint32_t w[4];
#pragma unroll
          for (int b = 0; b < KB; ++b) {
            // the codes of 4 dims of positions 16 b + 2 t, + 1 (u) and + 8, + 9 (v)
            uint32_t u, v;
            if constexpr (D == 16) {  // byte g of the rows
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = lds32(base + C::CODE + (16 * b + 8 * (i >> 1) + 2 * t + (i & 1)) * 8 +
                             (g >> 2) * 4);
              const uint32_t sel = (g & 3) | (4 + (g & 3)) << 8;
              u = __byte_perm(w[0], w[1], sel);
              v = __byte_perm(w[2], w[3], sel);
            } else {
              if (b % 2 == 0) ldsm_t(base + C::CODE + chunk_off<D>(16 * b + lane, j), w);
              u = w[b % 2 * 2], v = w[b % 2 * 2 + 1];
            }
            const uint32_t a0 = centred_lo(u), a1 = centred_hi(u);
            const uint32_t a2 = centred_lo(v), a3 = centred_hi(v);
#pragma unroll
            for (int k = 0; k < NC; ++k)
              mma_f16(c[k][0], a0, a1, a2, a3, pb[k][2 * b], pb[k][2 * b + 1]);
            if constexpr (D > 16) {
              const uint32_t b0 = centred_lo(u >> 8), b1 = centred_hi(u >> 8);
              const uint32_t b2 = centred_lo(v >> 8), b3 = centred_hi(v >> 8);
#pragma unroll
              for (int k = 0; k < NC; ++k)
                mma_f16(c[k][1], b0, b1, b2, b3, pb[k][2 * b], pb[k][2 * b + 1]);
            }
          }
#pragma unroll
          for (int k = 0; k < NC; ++k)
#pragma unroll
            for (int i = 0; i < OD; ++i)
              o[k][j][i] += c[k][i / 2][i % 2 * 2] + c[k][i / 2][i % 2 * 2 + 1];
        }
      }

      // the stage is read: fetch the tile NST ahead into it
      __syncwarp();
      if (T + C::NST < w1) fetch(st);
      if (++st == C::NST) st = 0, phase ^= 1;

      const Cursor was = cur;
      advance(cur);
      if (cur.tile == 0 || T + 1 == w1) {  // the head group, or this warp's part of it, ends
        finish();
        const int seg = was.m * VH + was.vh;
        if (whole && cur.tile == 0) {
          write_out(was);
        } else {
          const bool first = seg == seg_first;
          if (T + 1 == w1) __syncwarp();
          write_slot(T + 1 == w1 ? last_slot : first_slot);
          if (lane == 0) slot_seg[2 * warp + (first ? 0 : 1)] = seg;
          if (lane == 0 && first && T + 1 == w1) slot_seg[2 * warp] = seg | 0x40000000;
        }
        if (T + 1 < w1) {
          load_q(cur, q);
          len = clamped_len(a, cur.m);
          start(q);
          whole = true;
        }
      }
    }
    if (!alive)  // let the copies in flight land before the CTA leaves
      for (int i = 0; i < C::NST; ++i) mbar_wait(&full[warp][i], i < st ? phase ^ 1 : phase);
  }
  __syncthreads();

  // Partial results of neighbouring warps with the same head group meet: runs
  // of slots in warp order, a warp for each of a run's heads.  A run that is
  // the whole head group is written out, another goes to the CTA's workspace
  // slot (0: it holds the CTA's first tile, else 1).
  constexpr unsigned kAll = 0xffffffffu, kInLast = 0x40000000u;
  const int sg = lane < 2 * kWarps ? slot_seg[lane] : -1;
  const int id = sg < 0 ? -1 : sg & ~int(kInLast);
  const unsigned used = __ballot_sync(kAll, sg >= 0);
  const unsigned below = used & ((1u << lane) - 1);
  const int before = __shfl_sync(kAll, id, below ? 31 - __clz(below) : lane);
  unsigned heads_of_runs = __ballot_sync(kAll, sg >= 0 && (!below || before != id));
  const unsigned in_last = __ballot_sync(kAll, (lane & 1) || (sg & int(kInLast)));
  auto slot = [&](int s) {
    return reinterpret_cast<const float*>(
        (in_last >> s & 1) ? ring + (s >> 1) * C::NST * C::STAGE
                           : ring + kWarps * C::NST * C::STAGE + (s >> 1) * C::SLOT * 4);
  };
  while (heads_of_runs) {
    const int i = __ffs(heads_of_runs) - 1;
    heads_of_runs &= heads_of_runs - 1;
    const unsigned upto = heads_of_runs ? (1u << (__ffs(heads_of_runs) - 1)) - 1 : kAll;
    const unsigned run = used & upto & ~((1u << i) - 1);
    const int seg = __shfl_sync(kAll, id, i), m = seg / VH, vh = seg - m * VH;
    int s0 = 0, nt = c1;
    if (pl.split) {
      nt = pre[m + 1] - pre[m];
      s0 = pre[m] * VH + vh * nt;
    }
    const bool complete = s0 >= c0 && s0 + nt <= c1;
    float* out = a.out + int64_t(m) * a.out_ld + int64_t(first_head(vh)) * D;
    float* part = pl.part + (int64_t(blockIdx.x) * 2 + (s0 <= c0 ? 0 : 1)) * C::SLOT;
    for (int h = warp; h < n_heads(vh); h += kWarps) {
      // lanes as slots: their reference points and sums
      const bool on = run >> lane & 1;
      const float rs = on ? slot(lane)[HB * D + h] : -INFINITY;
      const float r = warp_max(rs);
      const float fl = on ? ex2_approx(rs - r) * slot(lane)[HB * D + HB + h] : 0.f;
      const float ls = warp_sum(fl), f = fl * rcp_approx(ls);
      constexpr int Q = (D + 31) / 32;
      float acc[Q] = {};
      // each warp from the run's first to its last has one of its slots, or none
      const int wb = (31 - __clz(run)) >> 1;
#pragma unroll 4
      for (int w = i >> 1; w <= wb; ++w) {
        const unsigned which = run >> (2 * w) & 3;
        const int s = 2 * w + (which >> 1);
        const float fs = __shfl_sync(kAll, f, s);
        const float* p = slot(s) + h * D;
#pragma unroll
        for (int q = 0; q < Q; ++q)
          if (which && q * 32 + lane < D) acc[q] = fmaf(p[q * 32 + lane], fs, acc[q]);
      }
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (q * 32 + lane < D) {
          if (complete) out[h * D + q * 32 + lane] = acc[q];
          else part[h * D + q * 32 + lane] = acc[q];
        }
      if (!complete && lane == 0) part[HB * D + h] = r, part[HB * D + HB + h] = ls;
    }
  }
}

// The head groups that several CTAs shared, joined from the workspace, and
// zeros for empty streams.  A CTA a head group; or, for MANY of them, CTA b
// takes the one that begins in the main kernel's CTA b and goes on behind it.
// A thread takes 4 columns of one head of every SL-th partial result, so that
// their loads are in flight together.
constexpr int kJoinThreads = 512;
template <int D, int NC, bool MANY>
__global__ void __launch_bounds__(kJoinThreads) attn_kv4_join_kernel(const Plan pl, int grid) {
  using C = Cfg<D, NC>;
  constexpr int HB = C::HB, ITEMS = HB * D / 4;
  constexpr int SL = kJoinThreads / ITEMS;  // 2 or more
  constexpr int PF = 4;                      // loads of the partials that do not wait for the weights
  extern __shared__ float fac[];  // [partial][HB] reference points, then weights; then sums
  __shared__ int sums[2][kJoinThreads / 32], at_s[3];
  __shared__ float4 acc_s[kJoinThreads];
  const AttnKv4Args& a = pl.a;
  const int VH = pl.VH, M = a.kv.M, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kW = kJoinThreads / 32;
  pdl_trigger();
  // everything but the partial results may be read before the main kernel ends:
  // the stream m, its tiles and those before it, and all
  auto tiles = [&](int i) { return tiles_of<C::TK>(clamped_len(a, i)); };
  int m, nt, before = 0, total = 0, T = 0;
  if constexpr (MANY) {
    // two streams a thread, scanned over the CTA; the one that holds the first
    // tile behind main CTA b's
    static_assert(kKv4MaxStreams <= 2 * kJoinThreads);
    const int n0 = 2 * tid < M ? tiles(2 * tid) : 0, n1 = 2 * tid + 1 < M ? tiles(2 * tid + 1) : 0;
    int at = n0 + n1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) sums[0][warp] = at;
    __syncthreads();
    const int of_warp = lane < kW ? sums[0][lane % kW] : 0;
    total = __reduce_add_sync(0xffffffffu, of_warp) * VH;
    at += __reduce_add_sync(0xffffffffu, lane < warp ? of_warp : 0) - n0 - n1;
    pdl_wait();
    for (int i = blockIdx.x; i < M; i += gridDim.x)
      if (tiles(i) == 0)
        for (int j = tid; j < a.nq * D; j += kJoinThreads) a.out[int64_t(i) * a.out_ld + j] = 0.f;
    if (int(blockIdx.x) + 1 >= min(grid, total)) return;
    T = Deal(total, min(grid, total)).first(blockIdx.x + 1);
    if (T >= at * VH && T < (at + n0 + n1) * VH) {
      const bool second = T >= (at + n0) * VH;
      at_s[0] = 2 * tid + second, at_s[1] = second ? at + n0 : at, at_s[2] = second ? n1 : n0;
    }
    __syncthreads();
    m = at_s[0], before = at_s[1], nt = at_s[2];
  } else {
    m = blockIdx.x / VH;
#pragma unroll 1
    for (int i = tid; i < M; i += kJoinThreads) {
      const int n = tiles(i);
      total += n;
      if (i < m) before += n;
    }
    nt = tiles(m);
    before = __reduce_add_sync(0xffffffffu, before);
    total = __reduce_add_sync(0xffffffffu, total);
    if (lane == 0) sums[0][warp] = before, sums[1][warp] = total;
    __syncthreads();
    before = __reduce_add_sync(0xffffffffu, lane < kW ? sums[0][lane % kW] : 0);
    total = __reduce_add_sync(0xffffffffu, lane < kW ? sums[1][lane % kW] : 0) * VH;
  }
  const int vh = MANY ? (T - before * VH) / nt : int(blockIdx.x) - m * VH;
  const int per = a.nq / a.kv.nkv, g0 = (vh & ((1 << pl.gsh) - 1)) * pl.gh;
  const int heads = min(pl.gh, per - g0);
  float* out = a.out + int64_t(m) * a.out_ld + int64_t((vh >> pl.gsh) * per + g0) * D;
  int b0 = 0, nb = 1, first = 0;
  if (nt > 0) {
    const int s0 = before * VH + vh * nt;
    const Deal deal(total, min(grid, total));
    b0 = deal.owner(s0);
    nb = deal.owner(s0 + nt - 1) - b0 + 1;
    // only the first of the CTAs can have begun before this head group
    first = s0 <= deal.first(b0) ? 0 : 1;
    // (T may be a head group's first tile, or an earlier CTA's head group)
    if (MANY && (s0 == T || b0 != int(blockIdx.x))) return;
  }
  if constexpr (!MANY) {
    pdl_wait();
    if (nt == 0) {
#pragma unroll 1
      for (int i = tid; i < heads * D; i += kJoinThreads) out[i] = 0.f;
      return;
    }
    if (nb == 1) return;
  }
  auto slot = [&](int i) {
    return pl.part + (int64_t(b0 + i) * 2 + (i == 0 ? first : 0)) * C::SLOT;
  };
  const int it = tid % ITEMS, h = it / (D / 4);
  const bool on = h < heads;
  float4 v[PF];
#pragma unroll
  for (int u = 0; u < PF; ++u) {
    const int i = tid / ITEMS + u * SL;
    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (on && i < nb) v[u] = __ldcg(reinterpret_cast<const float4*>(slot(i)) + it);
  }
  if (warp < heads) {  // a warp a head
    float r = -INFINITY, ls = 0.f;
#pragma unroll 1
    for (int base = lane; base < nb; base += 32 * PF) {
      float x[PF], l[PF];
#pragma unroll
      for (int u = 0; u < PF; ++u) {
        const int i = base + 32 * u;
        x[u] = -INFINITY, l[u] = 0.f;
        if (i < nb) {
          x[u] = __ldcg(slot(i) + HB * D + warp);
          l[u] = __ldcg(slot(i) + HB * D + HB + warp);
        }
      }
#pragma unroll
      for (int u = 0; u < PF; ++u) {
        const int i = base + 32 * u;
        if (i >= nb) break;
        fac[i * HB + warp] = x[u];
        fac[(nb + i) * HB + warp] = l[u];
        // (the sum so far moves with the reference point)
        const float n = fmaxf(r, x[u]);
        ls = fmaf(ls, ex2_approx(r - n), l[u] * ex2_approx(x[u] - n));
        r = n;
      }
    }
    const float top = warp_max(r);
    const float f = rcp_approx(warp_sum(lane < nb ? ls * ex2_approx(r - top) : 0.f));
#pragma unroll 1
    for (int i = lane; i < nb; i += 32)
      fac[i * HB + warp] = ex2_approx(fac[i * HB + warp] - top) * fac[(nb + i) * HB + warp] * f;
  }
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& v, int i) {
    const float f = fac[i * HB + h];
    acc.x = fmaf(v.x, f, acc.x);
    acc.y = fmaf(v.y, f, acc.y);
    acc.z = fmaf(v.z, f, acc.z);
    acc.w = fmaf(v.w, f, acc.w);
  };
  if (on) {
#pragma unroll
    for (int u = 0; u < PF; ++u)
      if (tid / ITEMS + u * SL < nb) add(v[u], tid / ITEMS + u * SL);
#pragma unroll 8
    for (int i = tid / ITEMS + PF * SL; i < nb; i += SL)
      add(__ldcg(reinterpret_cast<const float4*>(slot(i)) + it), i);
  }
  acc_s[tid] = acc;
  __syncthreads();
  if (tid < ITEMS && on) {
#pragma unroll
    for (int s = 1; s < SL; ++s) {
      const float4 o = acc_s[s * ITEMS + tid];
      acc.x += o.x, acc.y += o.y, acc.z += o.z, acc.w += o.w;
    }
    reinterpret_cast<float4*>(out)[it] = acc;
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_tiled() {
  static const auto fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// A map over the codes (head dim 128) as 128-byte lines of two rows of each
// head [M * nkv, cap / 2, 128] with a box of `rows` rows: TMA moves a line a
// step.  A box reaching behind a head's last line reads zeros there.
bool code_map(CUtensorMap* map, const uint8_t* base, const Kv4& kv, int rows) {
  auto fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t lines = cuuint64_t(kv.cap) * kv.d / 256;  // cap % 4 == 0
  const cuuint64_t dims[3] = {128, lines, cuuint64_t(kv.M) * kv.nkv};
  const cuuint64_t strides[2] = {128, lines * 128};
  const cuuint32_t box[3] = {128, cuuint32_t(rows * kv.d / 256), 1}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(base), dims, strides, box,
            estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K, typename... A>
cudaError_t launch(K kern, int grid, int threads, int smem, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// Head groups of a kv head: one or two of at most 8 query heads (two column
// tiles).
int head_groups(int per) { return (per + 7) / 8; }

template <int D, int NC>
cudaError_t run(const AttnKv4Args& a, cudaStream_t s) {
  using C = Cfg<D, NC>;
  Plan pl;
  const int per = a.nq / a.kv.nkv;
  pl.a = a;
  const int groups_kv = head_groups(per);
  pl.gsh = groups_kv - 1;
  pl.gh = (per + groups_kv - 1) / groups_kv;
  pl.VH = a.kv.nkv * groups_kv;
  pl.part = static_cast<float*>(a.ws);
  CUtensorMap km = {}, vm = {};
  if (C::MAP && (!code_map(&km, a.kv.kc, a.kv, C::TK) || !code_map(&vm, a.kv.vc, a.kv, C::TK)))
    return cudaErrorInvalidValue;
  const int64_t groups = int64_t(a.kv.M) * pl.VH;
  // A CTA a head group, or every CTA an equal run of the tiles and a join: the
  // join and what prepares it cost about 4 us, so up to 32 tiles a head group
  // (2 a warp; 64 where the head groups fill the GPU by half) go without.
  // 2048 positions of 8 heads of 64: 10.2 and 10.6 us; 4096: 14.8 and 10.9; 128
  // groups of 2048 (heads of 128): 16.4 and 20.5 us.  So do a few more head
  // groups than SMs, where one column tile makes them short: 192 of up to 300
  // positions (heads of 64) 8.9 and 11.2 us, of up to 2000 15.5 and 17.7; 256 of
  // up to 300 11.8 and 10.7.
  const int64_t most = NC == 1 ? a.num_sms + a.num_sms / 3 : a.num_sms;
  const bool half_full = 2 * groups > a.num_sms && groups <= a.num_sms;
  pl.split = groups > most || a.max_len > (half_full ? 64 : 32) * C::TK;
  const int grid = pl.split ? a.num_sms : int(groups);
  TMG_CUDA_TRY(launch(attn_kv4_kernel<D, NC>, grid, C::W * 32, C::SMEM, s, km, vm, pl));
  if (!pl.split) return cudaSuccess;
  // Streams of up to 300 positions, 8 heads of 64, all in all: 800 head groups 20.3
  // us with a CTA each and 20.1 by main CTAs, 2048: 33.3 and 27.8, 8192: 91 and 57;
  // 192: 11.2 and 12.2
  const int fac = 2 * grid * C::HB * 4;
  if (groups > 4 * grid)
    return launch(attn_kv4_join_kernel<D, NC, true>, grid, kJoinThreads, fac, s, pl, grid);
  return launch(attn_kv4_join_kernel<D, NC, false>, int(groups), kJoinThreads, fac, s, pl, grid);
}

template <int D, int NC>
cudaError_t prepare() {
  TMG_CUDA_TRY(set_carveout(attn_kv4_kernel<D, NC>, Cfg<D, NC>::SMEM));
  TMG_CUDA_TRY((set_carveout(attn_kv4_join_kernel<D, NC, true>)));
  return set_carveout(attn_kv4_join_kernel<D, NC, false>);
}

int column_tiles(int per) {
  const int n = head_groups(per);
  return (per + n - 1) / n > 4 ? 2 : 1;
}

}  // namespace

cudaError_t attn_kv4_prepare() {
  TMG_CUDA_TRY((prepare<16, 1>()));
  TMG_CUDA_TRY((prepare<16, 2>()));
  TMG_CUDA_TRY((prepare<32, 1>()));
  TMG_CUDA_TRY((prepare<32, 2>()));
  TMG_CUDA_TRY((prepare<64, 1>()));
  TMG_CUDA_TRY((prepare<64, 2>()));
  TMG_CUDA_TRY((prepare<128, 1>()));
  return prepare<128, 2>();
}

size_t attn_kv4_ws(const Kv4& kv, int nq, int num_sms) {
  const int nc = column_tiles(nq / kv.nkv);
  return size_t(num_sms) * 2 * (4 * nc) * (kv.d + 2) * 4;  // two of Cfg's SLOT a CTA
}

cudaError_t launch_attn_kv4(const AttnKv4Args& a, cudaStream_t s) {
  const int nc = column_tiles(a.nq / a.kv.nkv);
  switch (a.kv.d * 10 + nc) {
    case 161: return run<16, 1>(a, s);
    case 162: return run<16, 2>(a, s);
    case 321: return run<32, 1>(a, s);
    case 322: return run<32, 2>(a, s);
    case 641: return run<64, 1>(a, s);
    case 642: return run<64, 2>(a, s);
    case 1281: return run<128, 1>(a, s);
    case 1282: return run<128, 2>(a, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace tmg
