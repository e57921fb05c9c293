// AdamW over many tensors with 8-bit moments, for sm_100a.
//
// The first moment m and the root r of the second are e4m3 codes, 256 consecutive elements sharing a power of two
// (biased exponent e, value = code 2^(e - 127)): the smallest with absmax <= 448 2^(e - 127), so that scaling is exact and only the
// code is a rounding (half a step is 2^-4 of the value). r is held instead of v = r^2 because its logarithmic
// range is half of v's: e4m3 spans 2^17.8, which in v would be gradients a factor of 480 apart. An r that is not zero never
// becomes code 0, for a step divides by it.
//
//   m' = b1 m + (1 - b1) g,  r' = sqrt(b2 r^2 + (1 - b2) g^2),  p' = p (1 - lr wd) - lr (m' / (1 - b1^t)) / (r' / sqrt(1 - b2^t) + eps)
//
// The new moments are formed in fp32, one rounding to an operation (no contraction), so that the codes rounded to nearest
// are those of the same operations anywhere else; the parameter's step uses them before they are rounded.
//
// Bound by memory: 10 bytes and 1/64 an element in bf16, 218 M elements in 334 us, 6.5 TB/s (336 to 356 a call, one behind the other), with the moments and
// parameters rounded to nearest (fp32: 16 bytes, 530 us); with random bits, as by default, 432 us, two Philox calls to eight elements, where bf16
// moments take 575.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "chained_launch.cuh"
#include "launchers.h"
#include "philox.cuh"

namespace ss {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int A8_THREADS = 256, A8_WARPS = A8_THREADS / 32, A8_BLOCK = 256, A8_TENSORS = 48;

struct Tensor8 {
  void* p;
  const void* g;
  uint8_t *m, *r, *m_exp, *r_exp;
  long long n;
  unsigned long long offset;   // global element offset of the range: what the random bits are drawn by
  int first;                   // the launch's first CTA of this tensor
};
struct Table8 {
  Tensor8 t[A8_TENSORS];
  int count, run;              // run: blocks that each warp of a CTA walks
};
struct Args8 {
  float beta1, beta2, c1, c2, eps, keep, minus_lr, inv_bias2, grad_scale, one;   // minus_lr: with the first bias correction
  unsigned long long seed;
};

// The eight elements of a lane, by pairs: two fp32 operations to an instruction. Each operation is rounded by itself.
struct Eight {
  float2 v[4];
};
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// A sum of two rounded products by itself: packed products and sums are joined to fused multiply-adds, which round once,
// whatever their spelling, so the sum is spelled a * one + b with a `one` that the compiler does not know.
__device__ __forceinline__ float2 add2(float2 a, float2 b, float one) { return __ffma2_rn(a, both(one), b); }

__device__ __forceinline__ void decode8(uint2 codes, float unit, Eight& out) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
    out.v[i] = __fmul2_rn(__half22float2(__half2(h)), both(unit));
  }
}
// Eight scaled values -> codes, to nearest or by eight random bits each.
__device__ __forceinline__ uint2 encode8(const Eight& f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(f.v[i], __NV_SATFINITE, __NV_E4M3);
  return make_uint2(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410));
}
__device__ __forceinline__ uint2 encode8(const Eight& f, uint32_t r0, uint32_t r1) {
  uint2 out;
  asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;"
      : "=r"(out.x) : "f"(f.v[1].y), "f"(f.v[1].x), "f"(f.v[0].y), "f"(f.v[0].x), "r"(r0));
  asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;"
      : "=r"(out.y) : "f"(f.v[3].y), "f"(f.v[3].x), "f"(f.v[2].y), "f"(f.v[2].x), "r"(r1));
  return out;
}
// Biased exponent of a block whose largest magnitude has these bits. 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(unsigned bits) {
  if (bits == 0) return 0;
  const int e = static_cast<int>(bits >> 23) - ((bits & 0x7fffffu) > 0x600000u ? 7 : 8);
  return e > 1 ? e : 1;
}
__device__ __forceinline__ float unit_of(int exponent) { return __uint_as_float(static_cast<uint32_t>(exponent) << 23); }
__device__ __forceinline__ unsigned warp_top(float lane_top) { return __reduce_max_sync(0xffffffffu, __float_as_uint(lane_top)); }
__device__ __forceinline__ float sqrt_near(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal_near(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float largest(const Eight& f) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) t = fmaxf(t, fmaxf(fabsf(f.v[i].x), fabsf(f.v[i].y)));
  return t;
}

// What a lane reads of a block.
template <class T> struct Piece8;
template <> struct Piece8<bf16> {
  uint4 u;
  __device__ __forceinline__ void load(const uint4* x) { u = x[0]; }
  __device__ __forceinline__ void set(int e, bf16 x) {
    reinterpret_cast<unsigned short*>(&u)[e] = __bfloat16_as_ushort(x);
  }
  __device__ __forceinline__ void get(Eight& f) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
};
template <> struct Piece8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const uint4* x) {
    a = *reinterpret_cast<const float4*>(x);
    b = *reinterpret_cast<const float4*>(x + 1);
  }
  __device__ __forceinline__ void set(int e, float x) { (e < 4 ? reinterpret_cast<float*>(&a) : reinterpret_cast<float*>(&b))[e & 3] = x; }
  __device__ __forceinline__ void get(Eight& f) const {
    f.v[0] = make_float2(a.x, a.y); f.v[1] = make_float2(a.z, a.w); f.v[2] = make_float2(b.x, b.y); f.v[3] = make_float2(b.z, b.w);
  }
};
template <class P, class G> struct Read8 {
  Piece8<P> p;
  Piece8<G> g;
  uint2 m, r;
  int m_exp, r_exp;
};

// fp32 -> bf16 bits: to nearest, or 16 random bits below the kept mantissa and a cut (inf and NaN are only cut).
template <bool SR>
__device__ __forceinline__ uint32_t bf16_bits(float f, uint32_t rnd16) {
  if (!SR) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  const uint32_t u = __float_as_uint(f);
  return ((u & 0x7f800000u) == 0x7f800000u ? u : u + rnd16) >> 16;
}

// One block of 256 elements, eight to a lane: `x` becomes what is written, the parameters as fp32 in `p`.
//
// The root is needed as its code and for the parameter's step. sqrt.approx (relative error 2^-23) gives both, unless
// its value lies within 2^-21 of a border between two codes, where it is taken again with a correct rounding: that is one
// element in 30,000. So it is for a block whose exponent is in doubt, and for one with roots so small that their squares
// lose bits. (With the correctly rounded root everywhere: +10 instructions an element.)
template <bool SR_PARAM, bool SR_STATE, class P, class G>
__device__ __forceinline__ void update8(Read8<P, G>& x, const Args8& a, unsigned long long element, Eight& p, uint4& random) {
  Eight g, m, v, r;
  x.p.get(p);
  x.g.get(g);
  decode8(x.m, unit_of(x.m_exp), m);
  decode8(x.r, unit_of(x.r_exp), r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 gg = __fmul2_rn(g.v[i], both(a.grad_scale));
    m.v[i] = add2(__fmul2_rn(both(a.beta1), m.v[i]), __fmul2_rn(both(a.c1), gg), a.one);
    v.v[i] = add2(__fmul2_rn(both(a.beta2), __fmul2_rn(r.v[i], r.v[i])), __fmul2_rn(__fmul2_rn(both(a.c2), gg), gg), a.one);
    r.v[i] = make_float2(sqrt_near(v.v[i].x), sqrt_near(v.v[i].y));
  }
  auto exact_roots = [&] {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = make_float2(__fsqrt_rn(v.v[i].x), __fsqrt_rn(v.v[i].y));
  };
  x.m_exp = block_exponent(warp_top(largest(m)));
  unsigned top = warp_top(largest(r));
  const unsigned off = (top & 0x7fffffu) - 0x5ffffcu;          // four steps to either side of the border
  if (top < 0x2b800000u || (!SR_STATE && off <= 8u)) {         // 2^-40
    exact_roots();
    top = warp_top(largest(r));
  }
  x.r_exp = block_exponent(top);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 d = __ffma2_rn(r.v[i], both(a.inv_bias2), both(a.eps));
    const float2 step = __fmul2_rn(m.v[i], both(a.minus_lr));
    p.v[i] = __ffma2_rn(step, make_float2(reciprocal_near(d.x), reciprocal_near(d.y)), __fmul2_rn(p.v[i], both(a.keep)));
  }
  uint4 rs = make_uint4(0, 0, 0, 0);
  if (SR_PARAM || SR_STATE) {
    const unsigned long long at = element >> 3;
    const uint2 key = make_uint2(static_cast<uint32_t>(a.seed), static_cast<uint32_t>(a.seed >> 32));
    const uint32_t c0 = static_cast<uint32_t>(at), c1 = static_cast<uint32_t>(at >> 32);
    if (SR_PARAM) random = philox4x32(make_uint4(c0, c1, 0u, 0x3838u), key);
    if (SR_STATE) rs = philox4x32(make_uint4(c0, c1, 1u, 0x3838u), key);
  }
  const float m_inv = unit_of(254 - x.m_exp), r_inv = unit_of(254 - x.r_exp);
  constexpr float FLOOR = 0.001953125f;                        // code 1
  auto scaled = [&](Eight& out) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 y = __fmul2_rn(r.v[i], both(r_inv));
      out.v[i] = make_float2(v.v[i].x > 0.f ? fmaxf(y.x, FLOOR) : y.x, v.v[i].y > 0.f ? fmaxf(y.y, FLOOR) : y.y);
    }
  };
  Eight y;
#pragma unroll
  for (int i = 0; i < 4; ++i) m.v[i] = __fmul2_rn(m.v[i], both(m_inv));
  scaled(y);
  if (SR_STATE) {
    x.m = encode8(m, rs.x, rs.y);
    x.r = encode8(y, rs.z, rs.w);
  } else {
    x.m = encode8(m);
    Eight low, high;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      low.v[i] = __fmul2_rn(y.v[i], both(1.f - 0x1p-21f));
      high.v[i] = __fmul2_rn(y.v[i], both(1.f + 0x1p-21f));
    }
    x.r = encode8(low);
    const uint2 other = encode8(high);
    if (x.r.x != other.x || x.r.y != other.y) {
      exact_roots();
      scaled(y);
      x.r = encode8(y);
    }
  }
}

__device__ __forceinline__ void copy16(const void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy8(const void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}

// A warp walks `run` blocks, a CTA's eight warps side by side. Blocks to come are on their way in shared memory, copied and stored by
// whole sectors: eight fp32 elements of a lane are 32 bytes, which two instructions of 16 would each ask for by halves. (With the next block in registers instead the
// compiler moves the loads down to their use for want of registers: 218 M elements 668 us.)
template <class P, class G> struct Ring8 {
  static constexpr int P16 = sizeof(P) / 2, G16 = sizeof(G) / 2;       // 16-byte pieces of a lane
  static constexpr int STAGE = 32 * (16 * P16 + 16 * G16 + 16), STAGES = 48 * 1024 / A8_WARPS / STAGE;
};
// STAGED: tensors off the boundaries of their pieces. Neighbouring elements go by neighbouring lanes, and through shared memory to the eight
// of a lane and back: 50 M bf16 elements, one element off, 186 us (on the boundaries 109; by each lane's elements 3.7 times that). A kernel of its own: with
// this in the other one a layer of 218 M elements took 376 us instead of 361.
template <class P, class G, bool SR_PARAM, bool SR_STATE, bool STAGED>
__global__ void __launch_bounds__(A8_THREADS, 3)
adamw8_kernel(const __grid_constant__ Table8 tab, Args8 a) {
  using Ring = Ring8<P, G>;
  __shared__ __align__(16) unsigned char ring[A8_WARPS][Ring::STAGES][Ring::STAGE];
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int lo = 0, hi = tab.count - 1;                // the last tensor that starts at or before this CTA
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first <= static_cast<int>(blockIdx.x)) lo = mid; else hi = mid - 1;
  }
  const Tensor8 t = tab.t[lo];
  P* const p = static_cast<P*>(t.p);
  const G* const g = static_cast<const G*>(t.g);
  const long long first = static_cast<long long>(blockIdx.x - t.first) * tab.run * A8_WARPS + warp;
  const long long blocks = (t.n + A8_BLOCK - 1) / A8_BLOCK, whole = STAGED ? 0 : t.n / A8_BLOCK;
  auto walked = [&](long long end) {             // blocks of this warp's run before `end`
    const long long n = first < end ? (end - first + A8_WARPS - 1) / A8_WARPS : 0;
    return n < tab.run ? static_cast<int>(n) : tab.run;
  };
  const int mine = walked(blocks), full = walked(whole);
  // the exponents of all blocks of the run, one to a lane
  const long long kept = first + static_cast<long long>(lane) * A8_WARPS;
  int m_exp = lane < mine ? t.m_exp[kept] : 0, r_exp = lane < mine ? t.r_exp[kept] : 0;
  auto fetch = [&](int i) {
    if (i < full) {
      const long long e0 = (first + static_cast<long long>(i) * A8_WARPS) * A8_BLOCK + lane * 8;
      uint4* q = reinterpret_cast<uint4*>(ring[warp][i % Ring::STAGES]);
      const long long block = e0 - lane * 8;
#pragma unroll
      for (int k = 0; k < Ring::P16; ++k) copy16(q + lane + 32 * k, reinterpret_cast<const uint4*>(p + block) + lane + 32 * k);
      q += 32 * Ring::P16;
#pragma unroll
      for (int k = 0; k < Ring::G16; ++k) copy16(q + lane + 32 * k, reinterpret_cast<const uint4*>(g + block) + lane + 32 * k);
      uint2* c = reinterpret_cast<uint2*>(q + 32 * Ring::G16) + lane;
      copy8(c, t.m + e0);
      copy8(c + 32, t.r + e0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Eight out;
  uint4 random;
  Read8<P, G> x = {};
  auto rounded = [&] {                           // the new parameters in bf16
    const uint32_t rw[4] = {random.x, random.y, random.z, random.w};
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (SR_PARAM) {
        w[k] = bf16_bits<true>(out.v[k].x, rw[k] & 0xffffu) | bf16_bits<true>(out.v[k].y, rw[k] >> 16) << 16;
      } else {
        const __nv_bfloat162 two = __float22bfloat162_rn(out.v[k]);
        w[k] = *reinterpret_cast<const uint32_t*>(&two);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  if constexpr (STAGED) {
    int i = 0;
    P* const sp = reinterpret_cast<P*>(ring[warp][0]);
    G* const sg = reinterpret_cast<G*>(sp + A8_BLOCK);
    uint8_t *const sm = reinterpret_cast<uint8_t*>(sg + A8_BLOCK), *const sr = sm + A8_BLOCK;
    for (; i < mine; ++i) {
      const long long block = (first + static_cast<long long>(i) * A8_WARPS) * A8_BLOCK;
      const int n = static_cast<int>(min(t.n - block, static_cast<long long>(A8_BLOCK)));
      P pe[8];
      G ge[8];
      uint8_t me[8], re[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = lane + 32 * k;
        pe[k] = e < n ? p[block + e] : P(0.f);
        ge[k] = e < n ? g[block + e] : G(0.f);
        me[k] = e < n ? t.m[block + e] : uint8_t(0);
        re[k] = e < n ? t.r[block + e] : uint8_t(0);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = lane + 32 * k;
        sp[e] = pe[k];
        sg[e] = ge[k];
        sm[e] = me[k];
        sr[e] = re[k];
      }
      __syncwarp();
      x.p.load(reinterpret_cast<const uint4*>(sp) + lane * Ring::P16);
      x.g.load(reinterpret_cast<const uint4*>(sg) + lane * Ring::G16);
      x.m = reinterpret_cast<const uint2*>(sm)[lane];
      x.r = reinterpret_cast<const uint2*>(sr)[lane];
      x.m_exp = __shfl_sync(0xffffffffu, m_exp, i);
      x.r_exp = __shfl_sync(0xffffffffu, r_exp, i);
      update8<SR_PARAM, SR_STATE>(x, a, t.offset + static_cast<unsigned long long>(block + lane * 8), out, random);
      if (sizeof(P) == 4) {
        float4* to4 = reinterpret_cast<float4*>(sp) + 2 * lane;
        to4[0] = make_float4(out.v[0].x, out.v[0].y, out.v[1].x, out.v[1].y);
        to4[1] = make_float4(out.v[2].x, out.v[2].y, out.v[3].x, out.v[3].y);
      } else {
        reinterpret_cast<uint4*>(sp)[lane] = rounded();
      }
      reinterpret_cast<uint2*>(sm)[lane] = x.m;
      reinterpret_cast<uint2*>(sr)[lane] = x.r;
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int e = lane + 32 * k;
        if (e >= n) continue;
        p[block + e] = sp[e];
        t.m[block + e] = sm[e];
        t.r[block + e] = sr[e];
      }
      __syncwarp();
      if (lane == i) {
        m_exp = x.m_exp;
        r_exp = x.r_exp;
      }
    }
  } else {
    for (int i = 0; i < Ring::STAGES - 1; ++i) fetch(i);
    int i = 0;
    for (; i < full; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(Ring::STAGES - 2) : "memory");
      const long long e0 = (first + static_cast<long long>(i) * A8_WARPS) * A8_BLOCK + lane * 8;
      __syncwarp();                                // copies of other lanes, where a lane's eight elements are two pieces
      const uint4* q = reinterpret_cast<const uint4*>(ring[warp][i % Ring::STAGES]);
      x.p.load(q + lane * Ring::P16);
      q += 32 * Ring::P16;
      x.g.load(q + lane * Ring::G16);
      const uint2* c = reinterpret_cast<const uint2*>(q + 32 * Ring::G16) + lane;
      x.m = c[0];
      x.r = c[32];
      x.m_exp = __shfl_sync(0xffffffffu, m_exp, i);
      x.r_exp = __shfl_sync(0xffffffffu, r_exp, i);
      fetch(i + Ring::STAGES - 1);                 // into the stage of the block before this one
      update8<SR_PARAM, SR_STATE>(x, a, t.offset + static_cast<unsigned long long>(e0), out, random);
      if (sizeof(P) == 4) {
        // two lanes write the halves of the even one's eight elements, then those of the odd one's: whole sectors
        const bool odd = lane & 1;
        float2 own[2], other[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float2 gives = odd ? out.v[k] : out.v[2 + k];
          own[k] = odd ? out.v[2 + k] : out.v[k];
          other[k] = make_float2(__shfl_xor_sync(0xffffffffu, gives.x, 1), __shfl_xor_sync(0xffffffffu, gives.y, 1));
        }
        const float4 mine = make_float4(own[0].x, own[0].y, own[1].x, own[1].y),
                     its = make_float4(other[0].x, other[0].y, other[1].x, other[1].y);
        float4* to4 = reinterpret_cast<float4*>(p + e0 - (odd ? 4 : 0));         // even: 0 and 8, odd: 4 and 12 from the pair's first
        to4[0] = odd ? its : mine;
        to4[2] = odd ? mine : its;
      } else {
        *reinterpret_cast<uint4*>(p + e0) = rounded();
      }
      *reinterpret_cast<uint2*>(t.m + e0) = x.m;
      *reinterpret_cast<uint2*>(t.r + e0) = x.r;
      if (lane == i) {
        m_exp = x.m_exp;
        r_exp = x.r_exp;
      }
    }
    for (; i < mine; ++i) {                        // a tensor's last block
      const long long e0 = (first + static_cast<long long>(i) * A8_WARPS) * A8_BLOCK + lane * 8;
      x.m = x.r = make_uint2(0, 0);
      x.m_exp = __shfl_sync(0xffffffffu, m_exp, i);
      x.r_exp = __shfl_sync(0xffffffffu, r_exp, i);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = e0 + e < t.n;
        x.p.set(e, in ? p[e0 + e] : P(0.f));
        x.g.set(e, in ? g[e0 + e] : G(0.f));
        const uint32_t m = in ? t.m[e0 + e] : 0, r = in ? t.r[e0 + e] : 0;
        (e < 4 ? x.m.x : x.m.y) |= m << (8 * (e & 3));
        (e < 4 ? x.r.x : x.r.y) |= r << (8 * (e & 3));
      }
      update8<SR_PARAM, SR_STATE>(x, a, t.offset + static_cast<unsigned long long>(e0), out, random);
      const uint32_t rw[4] = {random.x, random.y, random.z, random.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e0 + e >= t.n) continue;
        const float f = (e & 1) ? out.v[e >> 1].y : out.v[e >> 1].x;
        if (sizeof(P) == 4) reinterpret_cast<float*>(p)[e0 + e] = f;
        else reinterpret_cast<unsigned short*>(p)[e0 + e] =
            static_cast<unsigned short>(bf16_bits<SR_PARAM>(f, (e & 1) ? rw[e >> 1] >> 16 : rw[e >> 1] & 0xffffu));
        t.m[e0 + e] = static_cast<uint8_t>((e < 4 ? x.m.x : x.m.y) >> (8 * (e & 3)));
        t.r[e0 + e] = static_cast<uint8_t>((e < 4 ? x.r.x : x.r.y) >> (8 * (e & 3)));
      }
      if (lane == i) {
        m_exp = x.m_exp;
        r_exp = x.r_exp;
      }
    }
  }
  if (lane < mine) {
    t.m_exp[kept] = static_cast<uint8_t>(m_exp);
    t.r_exp[kept] = static_cast<uint8_t>(r_exp);
  }
}

template <class P, class G, bool STAGED>
int launch8(const Table8& tab, const Args8& a, int ctas, int sr_param, int sr_state, cudaStream_t s) {
  auto go = [&](auto kern) {
    launch_chained(kern, ctas, A8_THREADS, 0, s, tab, a);
    return (int)cudaGetLastError();
  };
  if (sizeof(P) == 2 && sr_param)
    return sr_state ? go(adamw8_kernel<P, G, true, true, STAGED>) : go(adamw8_kernel<P, G, true, false, STAGED>);
  return sr_state ? go(adamw8_kernel<P, G, false, true, STAGED>) : go(adamw8_kernel<P, G, false, false, STAGED>);
}

}  // namespace
}  // namespace ss

extern "C" {
using namespace ss;

// `tensors`: eight values per tensor, {p, g, m, r, m_exp, r_exp, elements, offset}, and `hyper`, {lr, beta1, beta2, eps, weight decay,
// gradient scale}, in host memory, read before the call returns. No element is in two tensors; all parameters are of
// one type, and all gradients. `launched` receives the number of kernels: one to 48 tensors, and to 48 off the boundaries of their pieces.
int ss_adamw8_many(const long long* tensors, int count, int p_f32, int g_f32, const double* hyper, int step, long long seed,
                   int sr_param, int sr_state, int* launched, void* stream) {
  *launched = 0;
  const double lr = hyper[0], beta1 = hyper[1], beta2 = hyper[2], eps = hyper[3], weight_decay = hyper[4], grad_scale = hyper[5];
  if (step < 1) return -2;
  long long total = 0;
  for (int i = 0; i < count; ++i) {
    const long long* t = tensors + 8 * i;
    if (t[6] < 0 || t[7] < 0 || t[7] % 8) return -2;
    total += (t[6] + A8_BLOCK - 1) / A8_BLOCK;
  }
  Args8 a;
  a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.eps = (float)eps;
  a.c1 = (float)(1.0 - beta1); a.c2 = (float)(1.0 - beta2); a.keep = (float)(1.0 - lr * weight_decay);
  a.minus_lr = (float)(-lr / (1.0 - pow(beta1, step)));
  a.inv_bias2 = (float)(1.0 / sqrt(1.0 - pow(beta2, step)));
  a.grad_scale = (float)grad_scale;
  a.one = 1.f;
  a.seed = static_cast<unsigned long long>(seed) ^ (0x9E3779B97F4A7C15ull * (unsigned long long)(step + 1));
  // One wave of the three CTAs that fit on an SM while no warp walks more than 16 blocks; then the run from 8
  // on that leaves the last wave fullest (20 M elements: runs of 16 are 1.4 waves, 43 us in bf16 and 67 in fp32, of 11 two waves, 39.5 and 57; from 218 M
  // on it makes no difference).
  const long long each = (total + 148 * 24 - 1) / (148 * 24);
  long long run = each < 1 ? 1 : each;
  if (each > 16) {
    long long least = LLONG_MAX;
    for (long long r = 8; r <= 16; ++r) {
      const long long walked = (each + r - 1) / r * r;
      if (walked <= least) { least = walked; run = r; }
    }
  }
  // are all pointers of a tensor on the boundaries of their 8-element pieces?
  auto whole = [&](const long long* t) { return t[0] % 16 == 0 && t[1] % 16 == 0 && t[2] % 8 == 0 && t[3] % 8 == 0; };
  auto launches = [&](auto staged) {
    for (int done = 0; done < count;) {
      Table8 tab;
      tab.count = 0;
      tab.run = (int)run;
      long long ctas = 0;
      for (; done < count && tab.count < A8_TENSORS; ++done) {
        const long long* t = tensors + 8 * done;
        if (t[6] == 0 || whole(t) == decltype(staged)::value) continue;
        const long long mine = ((t[6] + A8_BLOCK - 1) / A8_BLOCK + run * A8_WARPS - 1) / (run * A8_WARPS);
        if (ctas + mine > 0x3fffffff) {
          if (tab.count == 0) return -2;
          break;
        }
        tab.t[tab.count++] = {(void*)t[0], (const void*)t[1], (uint8_t*)t[2], (uint8_t*)t[3], (uint8_t*)t[4], (uint8_t*)t[5],
                              t[6], (unsigned long long)t[7], (int)ctas};
        ctas += mine;
      }
      if (tab.count == 0) break;
      constexpr bool STAGED = decltype(staged)::value;
      cudaStream_t s = (cudaStream_t)stream;
      const int n = (int)ctas;
      const int e = p_f32 ? (g_f32 ? launch8<float, float, STAGED>(tab, a, n, sr_param, sr_state, s)
                                   : launch8<float, bf16, STAGED>(tab, a, n, sr_param, sr_state, s))
                          : (g_f32 ? launch8<bf16, float, STAGED>(tab, a, n, sr_param, sr_state, s)
                                   : launch8<bf16, bf16, STAGED>(tab, a, n, sr_param, sr_state, s));
      if (e) return e;
      ++*launched;
    }
    return 0;
  };
  const int e = launches(std::false_type());
  return e ? e : launches(std::true_type());
}
}  // extern "C"
