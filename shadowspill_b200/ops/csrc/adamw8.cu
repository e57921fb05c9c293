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
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

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
  int first;                   // the launch's first run of this tensor
  int vectors;                 // are all pointers on the boundaries of their 8-element pieces?
};
struct Table8 {
  Tensor8 t[A8_TENSORS];
  int count, run;              // run: blocks that a warp walks
};
struct Args8 {
  float lr, beta1, beta2, c1, c2, eps, keep, inv_bias1, inv_bias2, grad_scale;
  unsigned long long seed;
};

// Philox4x32-10, as the other update kernels use it.
__device__ __forceinline__ uint4 philox(uint4 c, uint2 key) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint32_t h0 = __umulhi(0xD2511F53u, c.x), l0 = 0xD2511F53u * c.x;
    const uint32_t h1 = __umulhi(0xCD9E8D57u, c.z), l1 = 0xCD9E8D57u * c.z;
    c = make_uint4(h1 ^ c.y ^ key.x, l1, h0 ^ c.w ^ key.y, l0);
    key.x += 0x9E3779B9u;
    key.y += 0xBB67AE85u;
  }
  return c;
}

__device__ __forceinline__ void decode8(uint2 codes, float unit, float (&f)[8]) {
  const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    f[2 * i] = v.x * unit;
    f[2 * i + 1] = v.y * unit;
  }
}
// Eight scaled values -> codes, to nearest or by eight random bits each.
template <bool SR>
__device__ __forceinline__ uint2 encode8(const float (&f)[8], uint32_t r0, uint32_t r1) {
  uint2 out;
  if (SR) {
    asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;"
        : "=r"(out.x) : "f"(f[3]), "f"(f[2]), "f"(f[1]), "f"(f[0]), "r"(r0));
    asm("cvt.rs.satfinite.e4m3x4.f32 %0, {%1, %2, %3, %4}, %5;"
        : "=r"(out.y) : "f"(f[7]), "f"(f[6]), "f"(f[5]), "f"(f[4]), "r"(r1));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i], f[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    out = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
  }
  return out;
}
// Biased exponent of the block whose largest magnitude is `top` (this lane's; the warp's is meant). 448 = 1.75 * 2^8.
__device__ __forceinline__ int block_exponent(float top) {
  const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (bits == 0) return 0;
  const int e = static_cast<int>(bits >> 23) - ((bits & 0x7fffffu) > 0x600000u ? 7 : 8);
  return e > 1 ? e : 1;
}

template <class T> __device__ __forceinline__ float one(const T* x, long long i);
template <> __device__ __forceinline__ float one(const float* x, long long i) { return x[i]; }
template <> __device__ __forceinline__ float one(const bf16* x, long long i) { return __bfloat162float(x[i]); }
template <class T> __device__ __forceinline__ void load8(const T* x, float (&f)[8]);
template <> __device__ __forceinline__ void load8(const float* x, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(x)[0], b = reinterpret_cast<const float4*>(x)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <> __device__ __forceinline__ void load8(const bf16* x, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(x);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// fp32 -> bf16 bits: to nearest, or 16 random bits below the kept mantissa and a cut (inf and NaN are only cut).
template <bool SR>
__device__ __forceinline__ uint32_t bf16_bits(float f, uint32_t rnd16) {
  if (!SR) return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  const uint32_t u = __float_as_uint(f);
  return ((u & 0x7f800000u) == 0x7f800000u ? u : u + rnd16) >> 16;
}

template <class P, class G, bool SR_PARAM, bool SR_STATE>
__global__ void __launch_bounds__(A8_THREADS)
adamw8_kernel(const __grid_constant__ Table8 tab, Args8 a) {
  const int lane = threadIdx.x & 31, run = blockIdx.x * A8_WARPS + (threadIdx.x >> 5);
  int lo = 0, hi = tab.count - 1;                // the last tensor that starts at or before this run
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].first <= run) lo = mid; else hi = mid - 1;
  }
  const Tensor8& t = tab.t[lo];
  P* const p = static_cast<P*>(t.p);
  const G* const g = static_cast<const G*>(t.g);
  const long long blocks = (t.n + A8_BLOCK - 1) / A8_BLOCK, from = static_cast<long long>(run - t.first) * tab.run;
  const long long to = from + tab.run < blocks ? from + tab.run : blocks;
  for (long long b = from; b < to; ++b) {
    const long long e0 = b * A8_BLOCK + lane * 8;
    const bool whole = t.vectors && (b + 1) * A8_BLOCK <= t.n;
    float pf[8], gf[8], mf[8], rf[8];
    const float m_unit = __uint_as_float(static_cast<uint32_t>(t.m_exp[b]) << 23);
    const float r_unit = __uint_as_float(static_cast<uint32_t>(t.r_exp[b]) << 23);
    uint2 mc = make_uint2(0, 0), rc = make_uint2(0, 0);
    if (whole) {
      load8(p + e0, pf);
      load8(g + e0, gf);
      mc = *reinterpret_cast<const uint2*>(t.m + e0);
      rc = *reinterpret_cast<const uint2*>(t.r + e0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool in = e0 + e < t.n;
        pf[e] = in ? one(p, e0 + e) : 0.f;
        gf[e] = in ? one(g, e0 + e) : 0.f;
        const uint32_t m = in ? t.m[e0 + e] : 0, r = in ? t.r[e0 + e] : 0;
        (e < 4 ? mc.x : mc.y) |= m << (8 * (e & 3));
        (e < 4 ? rc.x : rc.y) |= r << (8 * (e & 3));
      }
    }
    decode8(mc, m_unit, mf);
    decode8(rc, r_unit, rf);
    float m_top = 0.f, r_top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float gg = __fmul_rn(gf[e], a.grad_scale);
      mf[e] = __fadd_rn(__fmul_rn(a.beta1, mf[e]), __fmul_rn(a.c1, gg));
      rf[e] = __fsqrt_rn(__fadd_rn(__fmul_rn(a.beta2, __fmul_rn(rf[e], rf[e])), __fmul_rn(__fmul_rn(a.c2, gg), gg)));
      m_top = fmaxf(m_top, fabsf(mf[e]));
      r_top = fmaxf(r_top, rf[e]);
      pf[e] = pf[e] * a.keep - a.lr * __fdividef(mf[e] * a.inv_bias1, rf[e] * a.inv_bias2 + a.eps);
    }
    const int m_exp = block_exponent(m_top), r_exp = block_exponent(r_top);
    const float m_inv = __uint_as_float(static_cast<uint32_t>(254 - m_exp) << 23);
    const float r_inv = __uint_as_float(static_cast<uint32_t>(254 - r_exp) << 23);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mf[e] *= m_inv;
      rf[e] = rf[e] > 0.f ? fmaxf(rf[e] * r_inv, 0.001953125f) : rf[e];
    }
    uint4 rp = make_uint4(0, 0, 0, 0), rs = rp;
    if (SR_PARAM || SR_STATE) {
      const unsigned long long at = (t.offset + static_cast<unsigned long long>(e0)) >> 3;
      const uint2 key = make_uint2(static_cast<uint32_t>(a.seed), static_cast<uint32_t>(a.seed >> 32));
      const uint32_t c0 = static_cast<uint32_t>(at), c1 = static_cast<uint32_t>(at >> 32);
      if (SR_PARAM) rp = philox(make_uint4(c0, c1, 0u, 0x3838u), key);
      if (SR_STATE) rs = philox(make_uint4(c0, c1, 1u, 0x3838u), key);
    }
    mc = encode8<SR_STATE>(mf, rs.x, rs.y);
    rc = encode8<SR_STATE>(rf, rs.z, rs.w);
    const uint32_t rw[4] = {rp.x, rp.y, rp.z, rp.w};
    if (whole) {
      if (sizeof(P) == 4) {
        float4* out = reinterpret_cast<float4*>(p + e0);
        out[0] = make_float4(pf[0], pf[1], pf[2], pf[3]);
        out[1] = make_float4(pf[4], pf[5], pf[6], pf[7]);
      } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = bf16_bits<SR_PARAM>(pf[2 * i], rw[i] & 0xffffu) | bf16_bits<SR_PARAM>(pf[2 * i + 1], rw[i] >> 16) << 16;
        *reinterpret_cast<uint4*>(p + e0) = make_uint4(w[0], w[1], w[2], w[3]);
      }
      *reinterpret_cast<uint2*>(t.m + e0) = mc;
      *reinterpret_cast<uint2*>(t.r + e0) = rc;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (e0 + e >= t.n) continue;
        if (sizeof(P) == 4) reinterpret_cast<float*>(p)[e0 + e] = pf[e];
        else reinterpret_cast<unsigned short*>(p)[e0 + e] =
            static_cast<unsigned short>(bf16_bits<SR_PARAM>(pf[e], (e & 1) ? rw[e >> 1] >> 16 : rw[e >> 1] & 0xffffu));
        t.m[e0 + e] = static_cast<uint8_t>((e < 4 ? mc.x : mc.y) >> (8 * (e & 3)));
        t.r[e0 + e] = static_cast<uint8_t>((e < 4 ? rc.x : rc.y) >> (8 * (e & 3)));
      }
    }
    if (lane == 0) {
      t.m_exp[b] = static_cast<uint8_t>(m_exp);
      t.r_exp[b] = static_cast<uint8_t>(r_exp);
    }
  }
}

template <class P, class G>
int launch8(const Table8& tab, const Args8& a, int runs, int sr_param, int sr_state, cudaStream_t s) {
  auto go = [&](auto kern) {
    kern<<<(runs + A8_WARPS - 1) / A8_WARPS, A8_THREADS, 0, s>>>(tab, a);
    return (int)cudaGetLastError();
  };
  if (sizeof(P) == 2 && sr_param)
    return sr_state ? go(adamw8_kernel<P, G, true, true>) : go(adamw8_kernel<P, G, true, false>);
  return sr_state ? go(adamw8_kernel<P, G, false, true>) : go(adamw8_kernel<P, G, false, false>);
}

}  // namespace
}  // namespace ss

extern "C" {
using namespace ss;

// `tensors`: eight values per tensor, {p, g, m, r, m_exp, r_exp, elements, offset}, in host memory, read before the call
// returns; no element is in two of them. All parameters are of one type, and all gradients.
int ss_adamw8_many(const long long* tensors, int count, int p_f32, int g_f32, double lr, double beta1, double beta2, double eps,
                   double weight_decay, int step, double grad_scale, unsigned long long seed, int sr_param, int sr_state,
                   void* stream) {
  if (step < 1) return -2;
  long long total = 0;
  for (int i = 0; i < count; ++i) {
    const long long* t = tensors + 8 * i;
    if (t[6] < 0 || t[7] < 0 || t[7] % 8) return -2;
    total += (t[6] + A8_BLOCK - 1) / A8_BLOCK;
  }
  Args8 a;
  a.lr = (float)lr; a.beta1 = (float)beta1; a.beta2 = (float)beta2; a.eps = (float)eps;
  a.c1 = (float)(1.0 - beta1); a.c2 = (float)(1.0 - beta2); a.keep = (float)(1.0 - lr * weight_decay);
  a.inv_bias1 = (float)(1.0 / (1.0 - pow(beta1, step)));
  a.inv_bias2 = (float)(1.0 / sqrt(1.0 - pow(beta2, step)));
  a.grad_scale = (float)grad_scale;
  a.seed = seed ^ (0x9E3779B97F4A7C15ull * (unsigned long long)(step + 1));
  long long run = total / (148 * 40);
  run = run < 1 ? 1 : run > 16 ? 16 : run;
  for (int done = 0; done < count;) {
    Table8 tab;
    tab.count = 0;
    tab.run = (int)run;
    long long runs = 0;
    for (; done < count && tab.count < A8_TENSORS; ++done) {
      const long long* t = tensors + 8 * done;
      if (t[6] == 0) continue;
      const long long mine = ((t[6] + A8_BLOCK - 1) / A8_BLOCK + run - 1) / run;
      if (runs + mine > 0x3fffffff) {
        if (tab.count == 0) return -2;
        break;
      }
      const int vectors = t[0] % 16 == 0 && t[1] % 16 == 0 && t[2] % 8 == 0 && t[3] % 8 == 0;
      tab.t[tab.count++] = {(void*)t[0], (const void*)t[1], (uint8_t*)t[2], (uint8_t*)t[3], (uint8_t*)t[4], (uint8_t*)t[5],
                            t[6], (unsigned long long)t[7], (int)runs, vectors};
      runs += mine;
    }
    if (tab.count == 0) break;
    cudaStream_t s = (cudaStream_t)stream;
    const int e = p_f32 ? (g_f32 ? launch8<float, float>(tab, a, (int)runs, sr_param, sr_state, s)
                                 : launch8<float, bf16>(tab, a, (int)runs, sr_param, sr_state, s))
                        : (g_f32 ? launch8<bf16, float>(tab, a, (int)runs, sr_param, sr_state, s)
                                 : launch8<bf16, bf16>(tab, a, (int)runs, sr_param, sr_state, s));
    if (e) return e;
  }
  return 0;
}
}  // extern "C"
