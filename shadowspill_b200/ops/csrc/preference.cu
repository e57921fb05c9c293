// Paired preference loss on a block of logits for sm_100a, forward and gradient.
//
// Sequences 2p and 2p + 1 of the block are the chosen and the rejected answer of pair p:
//   logp_r = x_r[t_r] - lse(x_r);  sum_q = sum over its rows of w_r (logp_r - ref_r) [/ sum of w_r]
//   z_p = beta (sum_2p - sum_2p+1);  L = sum_p f(z_p)
//   dL/dx_r = coef_r (softmax(x_r) - onehot(t_r)),  coef_r = -+ beta f'(z_p) w_r [/ sum of w_r]
// with f = -(1 - e) log sigma(z) - e log sigma(-z), max(0, 1 - z) or (z / beta - 1 / (2 beta))^2.
//
// A row's gradient needs every row of its pair first, so the block is read twice: once for the rows' statistics (a running
// maximum and sum), once for the gradient.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

namespace ss {
namespace {

typedef __nv_bfloat16 bf16;
constexpr int PF_THREADS = 512;

template <class L> struct Vec;                   // one 16-byte piece of a row
template <> struct Vec<bf16> {
  static constexpr int N = 8;
  __device__ static void load(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static uint4 store(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ static float get(bf16 v) { return __bfloat162float(v); }
  __device__ static bf16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  __device__ static void load(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 store(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  __device__ static float get(float v) { return v; }
  __device__ static float put(float v) { return v; }
};

// The c-th piece of a row that may start anywhere: the same elements to a thread, hence the same bits, as of aligned rows.
template <class L>
__device__ __forceinline__ void load_piece(const L* x, int c, bool aligned, float (&f)[Vec<L>::N]) {
  if (aligned) return Vec<L>::load(reinterpret_cast<const uint4*>(x)[c], f);
#pragma unroll
  for (int e = 0; e < Vec<L>::N; ++e) f[e] = Vec<L>::get(x[c * Vec<L>::N + e]);
}
template <class L>
__device__ __forceinline__ void store_piece(L* x, int c, bool aligned, const float (&f)[Vec<L>::N]) {
  if (aligned) {
    reinterpret_cast<uint4*>(x)[c] = Vec<L>::store(f);
    return;
  }
#pragma unroll
  for (int e = 0; e < Vec<L>::N; ++e) x[c * Vec<L>::N + e] = Vec<L>::put(f[e]);
}

struct Rows {
  const long long* targets;
  const float* weights;      // null: one each
  int R, V;
  // Does row r carry loss? `t` and `w` receive its target and weight.
  __device__ bool scored(int r, long long& t, float& w) const {
    t = targets[r];
    w = weights != nullptr ? weights[r] : 1.f;
    return t >= 0 && t < V && w != 0.f;
  }
};

// What the kernels hand on, in one allocation of the caller's: per row the coefficient, the largest logit, the sum's
// reciprocal and what logp lost when it was rounded to fp32; the pairs' losses; a counter.
struct Work {
  float *coef, *top, *inv, *low, *pair_loss;
  int* done;
};

// exp(d) for d <= 0. The argument of ex2 carries log2(e) in two parts: __expf's single constant shifts every probability
// the same way, by up to 1e-6 at d = -20, and sequences of thousands of rows add that up.
__device__ __forceinline__ float exp_below(float d) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(d, 1.925963e-8f, d * 1.44269502f)));
  return e;
}
// The mean relative error of ex2.approx (4 M arguments over [-1, 0], [-12, 0] and [-20, 0]: -4.92e-8, -5.02e-8 and -5.05e-8, with a
// deviation of 3.0e-8 around it): what a sum of exponentials is short of.
constexpr double EX2_SHORT = 5.0e-8;

template <class L>
__global__ void __launch_bounds__(PF_THREADS)
preference_rows_kernel(const L* __restrict__ logits, long long ld, bool aligned, Rows rows, Work work, float* __restrict__ logp) {
  __shared__ float red_m[16], red_s[16];
  const int row = blockIdx.x;
  if (row == 0 && threadIdx.x == 0) *work.done = 0;
  if (row >= rows.R) return;
  long long target;
  float weight;
  if (!rows.scored(row, target, weight)) {
    if (threadIdx.x == 0) work.coef[row] = work.low[row] = logp[row] = 0.f;
    return;
  }
  const L* x = logits + row * ld;
  constexpr int N = Vec<L>::N;
  float m = -FLT_MAX, s = 0.f;
  auto add = [&](const float (&f)[N]) {
    float lm = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) lm = fmaxf(lm, f[e]);
    if (lm > m) {
      s *= exp_below(m - lm);
      m = lm;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) s += exp_below(f[e] - m);
  };
  for (int c = threadIdx.x; c < rows.V / N; c += PF_THREADS) {
    float f[N];
    load_piece(x, c, aligned, f);
    add(f);
  }
  for (int c = rows.V / N * N + threadIdx.x; c < rows.V; c += PF_THREADS) {
    const float f = Vec<L>::get(x[c]);
    if (f > m) {
      s *= exp_below(m - f);
      m = f;
    }
    s += exp_below(f - m);
  }
  auto merge = [&](float om, float os) {
    const float top = fmaxf(m, om);
    s = s * exp_below(m - top) + os * exp_below(om - top);
    m = top;
  };
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
  if ((threadIdx.x & 31) == 0) {
    red_m[threadIdx.x >> 5] = m;
    red_s[threadIdx.x >> 5] = s;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    m = threadIdx.x < 16 ? red_m[threadIdx.x] : -FLT_MAX;
    s = threadIdx.x < 16 ? red_s[threadIdx.x] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) merge(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    if (threadIdx.x == 0) {
      const double sum = s + (s - 1.0) * EX2_SHORT;     // the largest logit's own 1 is exact
      const double exact = (static_cast<double>(Vec<L>::get(x[target])) - m) - log(sum);
      const float rounded = static_cast<float>(exact);
      logp[row] = rounded;
      work.low[row] = isfinite(rounded) ? static_cast<float>(exact - rounded) : 0.f;
      work.top[row] = m;
      work.inv[row] = 1.f / s;
      work.coef[row] = 0.f;
    }
  }
}

struct PairArgs {
  const int* cu_seqlens;
  const float* ref_logp;     // optional, per row
  float beta, smoothing, grad_scale;
  int kind, average;
};
__device__ __forceinline__ double block_sum64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
  for (int i = 0; i < (blockDim.x >> 5); ++i) v += red[i];
  return v;
}

// One block per pair. Sums of a sequence's log ratios are held in 64 bits: they cancel between the two sides.
__global__ void __launch_bounds__(256)
preference_pairs_kernel(Rows rows, PairArgs a, Work work, const float* __restrict__ logp, float* __restrict__ sums,
                        float* __restrict__ loss_sum) {
  __shared__ double red[8];
  __shared__ bool last;
  const int p = blockIdx.x;
  double sum[2], mass[2];
  int first[2], end[2];
  bool some = true;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    first[side] = min(max(a.cu_seqlens[2 * p + side], 0), rows.R);
    end[side] = min(max(a.cu_seqlens[2 * p + side + 1], 0), rows.R);
    double ratio = 0.0, weight = 0.0;
    bool any = false;
    for (int r = first[side] + threadIdx.x; r < end[side]; r += blockDim.x) {
      long long t;
      float w;
      if (!rows.scored(r, t, w)) continue;
      any = true;
      weight += w;
      const double whole = static_cast<double>(logp[r]) + work.low[r];
      ratio += w * (a.ref_logp != nullptr ? whole - a.ref_logp[r] : whole);
    }
    sum[side] = block_sum64(ratio, red);
    mass[side] = a.average ? block_sum64(weight, red) : 1.0;
    if (a.average) sum[side] = mass[side] != 0.0 ? sum[side] / mass[side] : 0.0;
    some = __syncthreads_or(any) && some;
    if (threadIdx.x == 0 && sums != nullptr) sums[2 * p + side] = static_cast<float>(sum[side]);
  }
  const double beta = a.beta, e = a.smoothing, z = beta * (sum[0] - sum[1]);
  double loss, slope;                            // slope: dL / d sum[0]
  if (a.kind == 0) {
    const double tail = log1p(exp(-fabs(z)));
    loss = (1.0 - e) * (fmax(-z, 0.0) + tail) + e * (fmax(z, 0.0) + tail);
    slope = beta * (e - 1.0 / (1.0 + exp(z)));
  } else if (a.kind == 1) {
    loss = z < 1.0 ? 1.0 - z : z >= 1.0 ? 0.0 : z;       // NaN stays one
    slope = z < 1.0 ? -beta : 0.0;
  } else {
    const double gap = sum[0] - sum[1] - 0.5 / beta;
    loss = gap * gap;
    slope = 2.0 * gap;
  }
  if (!some) loss = slope = 0.0;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const double each = mass[side] != 0.0 ? (side ? slope : -slope) * a.grad_scale / mass[side] : 0.0;
    for (int r = first[side] + threadIdx.x; r < end[side]; r += blockDim.x) {
      long long t;
      float w;
      if (rows.scored(r, t, w)) work.coef[r] = static_cast<float>(each * w);
    }
  }
  // the last block to get here adds the pairs' losses, in their order
  if (threadIdx.x == 0) {
    work.pair_loss[p] = static_cast<float>(loss);
    __threadfence();
    last = atomicAdd(work.done, 1) == static_cast<int>(gridDim.x) - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double total = 0.0;
  for (int i = threadIdx.x; i < static_cast<int>(gridDim.x); i += blockDim.x) total += __ldcg(work.pair_loss + i);
  total = block_sum64(total, red);
  if (threadIdx.x == 0) *loss_sum += static_cast<float>(total);
}

// Not __restrict__: the gradient may go over the logits.
template <class L>
__global__ void __launch_bounds__(PF_THREADS)
preference_grad_kernel(const L* logits, long long ld, bool aligned, const long long* __restrict__ targets, Work work, int V,
                       L* grad, long long ldg) {
  const int row = blockIdx.x;
  constexpr int N = Vec<L>::N;
  const L* x = logits + row * ld;
  L* g = grad + row * ldg;
  const float coef = work.coef[row];
  if (coef == 0.f) {
    const float zero[N] = {};
    for (int c = threadIdx.x; c < V / N; c += PF_THREADS) store_piece(g, c, aligned, zero);
    for (int c = V / N * N + threadIdx.x; c < V; c += PF_THREADS) g[c] = Vec<L>::put(0.f);
    return;
  }
  const float top = work.top[row], each = coef * work.inv[row];
  const int target = static_cast<int>(targets[row]);
  for (int c = threadIdx.x; c < V / N; c += PF_THREADS) {
    float f[N];
    load_piece(x, c, aligned, f);
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = each * exp_below(f[e] - top) - (c * N + e == target ? coef : 0.f);
    store_piece(g, c, aligned, f);
  }
  for (int c = V / N * N + threadIdx.x; c < V; c += PF_THREADS)
    g[c] = Vec<L>::put(each * exp_below(Vec<L>::get(x[c]) - top) - (c == target ? coef : 0.f));
}

template <class L>
int preference(const L* logits, long long ld, const Rows& rows, const PairArgs& a, int pairs, const Work& work, float* logp,
               float* sums, float* loss_sum, L* grad, long long ldg, cudaStream_t s) {
  constexpr int N = Vec<L>::N;
  auto aligned16 = [&](const L* x, long long pitch) { return reinterpret_cast<uintptr_t>(x) % 16 == 0 && pitch % N == 0; };
  const bool aligned = aligned16(logits, ld) && (grad == nullptr || aligned16(grad, ldg));
  preference_rows_kernel<<<rows.R > 0 ? rows.R : 1, PF_THREADS, 0, s>>>(logits, ld, aligned, rows, work, logp);
  if (pairs > 0) preference_pairs_kernel<<<pairs, 256, 0, s>>>(rows, a, work, logp, sums, loss_sum);
  if (grad != nullptr && rows.R > 0)
    preference_grad_kernel<<<rows.R, PF_THREADS, 0, s>>>(logits, ld, aligned, rows.targets, work, rows.V, grad, ldg);
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace ss

extern "C" {
using namespace ss;

// work: 4 R + pairs + 1 words. logp: R words. grad null: the loss alone.
int ss_preference(const void* logits, int fp32_logits, long long ld, const long long* targets, const float* weights,
                  const int* cu_seqlens, int R, int V, int pairs, const float* ref_logp, float beta, int kind, float smoothing,
                  int average, float grad_scale, float* logp, float* sums, float* loss_sum, void* grad, long long ldg, void* work,
                  void* stream) {
  if (R < 0 || V < 1 || pairs < 0 || kind < 0 || kind > 2 || ld < V || (grad != nullptr && ldg < V)) return -2;
  const Rows rows{targets, weights, R, V};
  const PairArgs a{cu_seqlens, ref_logp, beta, smoothing, grad_scale, kind, average};
  float* w = (float*)work;
  const long long n = R;
  const Work handed{w, w + n, w + 2 * n, w + 3 * n, w + 4 * n, (int*)(w + 4 * n + pairs)};
  if (fp32_logits)
    return preference((const float*)logits, ld, rows, a, pairs, handed, logp, sums, loss_sum, (float*)grad, ldg, (cudaStream_t)stream);
  return preference((const bf16*)logits, ld, rows, a, pairs, handed, logp, sums, loss_sum, (bf16*)grad, ldg, (cudaStream_t)stream);
}
}  // extern "C"
