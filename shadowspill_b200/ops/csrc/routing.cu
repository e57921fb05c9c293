// Selection of experts for sm_100a: softmax or sigmoid scores, a bias that only selects, groups, top-k, renormalised and
// scaled weights, a histogram; and the gradient of the weights.
//
//   s = sigmoid(x) or softmax(x), key = s + bias; a group's score is the sum of its two largest keys; the k largest keys of
//   the best groups are the picks, ties to the lowest index; w_j = scale s_j / (sum_i s_i + 1e-20), or scale s_j.
//
// Which experts are picked is defined by keys in 64 bits. The kernel forms them in 32 and looks at the gaps between the picks,
// to the best key left over, and between the groups kept and dropped: a token with a gap within the error of its keys is
// done again in 64 bits. Where nothing is added to the scores and there are no groups the logits themselves are compared,
// which needs neither.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

namespace ss {
namespace {

constexpr int RT_THREADS = 128, RT_WARPS = RT_THREADS / 32;
constexpr int RT_MAX_E = 512, RT_MAX_K = 32, RT_MAX_GROUPS = 32;
constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ float load_logit(const float* p) { return *p; }
__device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_logit(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_logit(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float warp_sum32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
// Signed integers in the order of the floats; -inf and NaN compare lowest and equal.
__device__ __forceinline__ int ordered(float v) {
  const int b = __float_as_int(v + 0.f);         // -0 and 0 are equal
  return v > -INFINITY ? b ^ ((b >> 31) & 0x7fffffff) : INT_MIN;
}
__device__ __forceinline__ float unordered(int o) {
  return o == INT_MIN ? -INFINITY : __int_as_float(o ^ ((o >> 31) & 0x7fffffff));
}
__device__ __forceinline__ float row_max(float v) { return unordered(__reduce_max_sync(FULL, ordered(v))); }

struct RouteArgs {
  int T, E, k, groups, keep, sigmoid, renormalize;
  long long ld;
  float scale;
  const float* bias;
};

// The two largest of (a, b) and (c, d), both in decreasing order.
template <class F>
__device__ __forceinline__ void merge_top2(F& a, F& b, F c, F d) {
  const F low = a < c ? a : c;
  a = a < c ? c : a;
  const F rest = b < d ? d : b;
  b = rest < low ? low : rest;
}

// Which groups stay, as bits, from the keys of all experts in `keys` (shared memory, NaN already -inf). Each group is
// looked at by 32 / (groups rounded up to a power of two) lanes. `gap` receives how far the worst group kept lies above
// the best one dropped.
template <class F>
__device__ unsigned kept_groups(const F* keys, const RouteArgs& a, int lane, F& gap) {
  const int per = a.groups > 1 ? 32 >> (32 - __clz(a.groups - 1)) : 32;     // lanes to a group
  const int group = lane / per, sub = lane % per, size = a.E / a.groups;
  F best = -INFINITY, second = -INFINITY;
  if (group < a.groups)
    for (int i = sub; i < size; i += per) {
      const F v = keys[group * size + i];
      if (v > best) { second = best; best = v; } else if (v > second) second = v;
    }
  for (int o = per >> 1; o > 0; o >>= 1) {
    const F c = __shfl_xor_sync(FULL, best, o), d = __shfl_xor_sync(FULL, second, o);
    merge_top2(best, second, c, d);
  }
  const F score = size > 1 ? best + second : best;
  int ahead = 0;                                 // groups that come before this one
  for (int g = 0; g < a.groups; ++g) {
    const F other = __shfl_sync(FULL, score, g * per);
    ahead += other > score || (other == score && g < group);
  }
  const bool real = group < a.groups, kept = real && ahead < a.keep;
  F worst = kept ? score : F(INFINITY), left = real && !kept ? score : F(-INFINITY);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const F w = __shfl_xor_sync(FULL, worst, o), l = __shfl_xor_sync(FULL, left, o);
    worst = w < worst ? w : worst;
    left = l > left ? l : left;
  }
  gap = worst - left;                            // NaN where both are -inf: no gap
  unsigned bits = 0;
  for (int g = 0; g < a.groups; ++g) bits |= __shfl_sync(FULL, static_cast<unsigned>(kept), g * per) << g;
  return bits;
}

// The picks with keys in 64 bits; lane j returns the j-th.
template <int PER, class L>
__device__ __noinline__ int picks_exact(const L* row, const RouteArgs& a, const unsigned char* group_of, double* keys, int lane) {
  float top = -INFINITY;
  for (int e = lane; e < a.E; e += 32) top = fmaxf(top, load_logit(row + e));
  top = row_max(top);
  double total = 0.0;
  if (!a.sigmoid) {
    for (int e = lane; e < a.E; e += 32) {
      const float x = load_logit(row + e);
      if (x > -INFINITY) total += exp(static_cast<double>(x) - top);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
  }
  for (int e = lane; e < a.E; e += 32) {
    const double x = load_logit(row + e);
    double v = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : (x > -INFINITY ? exp(x - top) / total : x * 0.0);
    if (!a.sigmoid && x == -INFINITY) v = 0.0;
    if (a.bias != nullptr) v += a.bias[e];
    keys[e] = v == v ? v : -INFINITY;
  }
  __syncwarp();
  if (a.groups > 1) {
    double gap;
    const unsigned bits = kept_groups(keys, a, lane, gap);
    __syncwarp();
    for (int e = lane; e < a.E; e += 32)
      if (!((bits >> group_of[e]) & 1)) keys[e] = -INFINITY;
    __syncwarp();
  }
  unsigned taken = 0;                            // this lane's experts that are picked, by place
  int mine = 0;
  for (int j = 0; j < a.k; ++j) {
    double best = -INFINITY;
    int at = INT_MAX;
    for (int i = 0; i < PER; ++i) {
      const int e = lane + 32 * i;
      if (e < a.E && !((taken >> i) & 1) && (at == INT_MAX || keys[e] > best)) { best = keys[e]; at = e; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const double ob = __shfl_xor_sync(FULL, best, o);
      const int oa = __shfl_xor_sync(FULL, at, o);
      if (oa != INT_MAX && (at == INT_MAX || ob > best || (ob == best && oa < at))) { best = ob; at = oa; }
    }
    if ((at & 31) == lane) taken |= 1u << (at >> 5);
    if (lane == j) mine = at;
  }
  __syncwarp();
  return mine;
}

// One warp to a token, expert lane + 32 i in the lane's register i.
template <int PER, bool LOGITS, class L>
__global__ void __launch_bounds__(RT_THREADS)
select_experts_kernel(const L* __restrict__ logits, RouteArgs a, int* __restrict__ ids, float* __restrict__ weights,
                      int* __restrict__ counts) {
  __shared__ int hist[RT_MAX_E];
  __shared__ unsigned char group_of[RT_MAX_E];
  extern __shared__ double warp_keys[];          // E per warp, where keys may have to be formed in 64 bits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < a.E; e += RT_THREADS) {
    hist[e] = 0;
    group_of[e] = static_cast<unsigned char>(e / (a.E / a.groups));
  }
  __syncthreads();
  for (int t = blockIdx.x * RT_WARPS + warp; t < a.T; t += gridDim.x * RT_WARPS) {
    const L* row = logits + static_cast<long long>(t) * a.ld;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = lane + 32 * i < a.E ? load_logit(row + lane + 32 * i) : -INFINITY;
    float top = 0.f, total = 1.f;
    bool bad = false;                            // a softmax with a NaN or +inf in it
    if (!a.sigmoid) {
#pragma unroll
      for (int i = 0; i < PER; ++i) bad = bad || !(v[i] < INFINITY);
      bad = __any_sync(FULL, bad);
    }
    if (!a.sigmoid && !(LOGITS && a.renormalize)) {
      top = v[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
      top = row_max(top);
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < PER; ++i) sum += v[i] > -INFINITY ? __expf(v[i] - top) : 0.f;
      total = warp_sum32(sum);
    }
    bool again = false;
    float slack = 0.f;
    if (!LOGITS) {
      // errors of a key: the score's (a relative 2^-21 of the largest: exp, its sum, the division) and the sum's rounding
      slack = a.sigmoid ? 1.5e-6f : 1.5e-6f * __fdividef(1.f, fmaxf(total, 1.f));
      const float inv = __fdividef(1.f, fmaxf(total, 1.f));
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        if (a.sigmoid) v[i] = e < a.E ? __fdividef(1.f, 1.f + __expf(-v[i])) : -INFINITY;
        else if (e < a.E) v[i] = v[i] == -INFINITY ? 0.f : __expf(v[i] - top) * inv;
        if (e < a.E && a.bias != nullptr) v[i] += a.bias[e];
      }
    }
    int key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = lane + 32 * i < a.E ? ordered(v[i]) : INT_MIN;
    if (!LOGITS && a.groups > 1) {
      float* keys = reinterpret_cast<float*>(warp_keys + warp * a.E);
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < a.E) keys[lane + 32 * i] = unordered(key[i]);
      __syncwarp();
      float gap;
      const unsigned bits = kept_groups(keys, a, lane, gap);
      float big = 0.f;                           // group scores are sums of two keys
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (key[i] != INT_MIN) big = fmaxf(big, fabsf(v[i]));
      big = row_max(big);
      again = a.keep < a.groups && !(gap > 4.f * slack + 5e-7f * big);
      __syncwarp();
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (lane + 32 * i < a.E && !((bits >> group_of[lane + 32 * i]) & 1)) key[i] = INT_MIN;
    }
    int best = INT_MIN, place = 0;
    auto rescan = [&] {
      best = key[0];
      place = 0;
#pragma unroll
      for (int i = 1; i < PER; ++i)
        if (key[i] > best) { best = key[i]; place = i; }
    };
    rescan();
    int mine = 0, found = 0;
    float last = INFINITY;
    for (; found < a.k && !again; ++found) {
      const int m = __reduce_max_sync(FULL, best);
      if (m == INT_MIN) break;
      const int e = __reduce_min_sync(FULL, best == m ? lane + 32 * place : INT_MAX);
      if (!LOGITS) {
        const float f = unordered(m);
        again = last - f <= 2.f * slack + 2.5e-7f * fabsf(f);
        last = f;
      }
      if (lane == found) mine = e;
      if ((e & 31) == lane) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (i == place) key[i] = INT_MIN;
        rescan();
      }
    }
    if (!LOGITS) {
      if (!again && found == a.k) {
        const int m = __reduce_max_sync(FULL, best);
        const float f = unordered(m);
        again = m != INT_MIN && last - f <= 2.f * slack + 2.5e-7f * fabsf(f);
      }
      again = again || found < a.k;
      if (again) mine = picks_exact<PER>(row, a, group_of, warp_keys + warp * a.E, lane);
    } else if (found < a.k) {                    // fewer than k comparable logits: the first experts not yet picked
      unsigned taken = 0;
      for (int j = 0; j < found; ++j) {
        const int e = __shfl_sync(FULL, mine, j);
        if ((e & 31) == lane) taken |= 1u << (e >> 5);
      }
      for (; found < a.k; ++found) {
        int left = INT_MAX;
        for (int i = PER - 1; i >= 0; --i)
          if (lane + 32 * i < a.E && !((taken >> i) & 1)) left = lane + 32 * i;
        const int e = __reduce_min_sync(FULL, left);
        if ((e & 31) == lane) taken |= 1u << (e >> 5);
        if (lane == found) mine = e;
      }
    }
    const bool pick = lane < a.k;
    const float x = pick ? load_logit(row + mine) : -INFINITY;
    float s;
    if (a.sigmoid) {
      s = pick ? __fdividef(1.f, 1.f + __expf(-x)) : 0.f;
    } else {
      if (LOGITS && a.renormalize) top = row_max(x);      // the scores' common factor leaves with the renormalisation
      s = !pick || x == -INFINITY ? 0.f : __expf(x - top);
      if (!(LOGITS && a.renormalize)) s = __fdividef(s, fmaxf(total, 1.f));
      if (bad) s = NAN;
    }
    const float w = a.renormalize ? a.scale * __fdividef(s, warp_sum32(s) + 1e-20f) : a.scale * s;
    if (pick) {
      ids[static_cast<long long>(t) * a.k + lane] = mine;
      weights[static_cast<long long>(t) * a.k + lane] = w;
      atomicAdd(&hist[mine], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += RT_THREADS) {
    if (gridDim.x == 1) counts[e] = hist[e];
    else if (hist[e]) atomicAdd(counts + e, hist[e]);
  }
}

// With c_j the picked scores, S their sum: dc_j = scale / S (dw_j - sum_i dw_i c_i / S) or scale dw_j, and
//   sigmoid  dx_e = dc_e s_e (1 - s_e);   softmax  dx_e = s_e (dc_e - sum_j dc_j s_j), whose sum is zero if renormalised.
template <class L>
__global__ void __launch_bounds__(RT_THREADS)
select_experts_bwd_kernel(const L* __restrict__ logits, RouteArgs a, const int* __restrict__ ids,
                          const float* __restrict__ dweights, L* __restrict__ dlogits) {
  const int lane = threadIdx.x & 31;
  for (int t = blockIdx.x * RT_WARPS + (threadIdx.x >> 5); t < a.T; t += gridDim.x * RT_WARPS) {
    const L* row = logits + static_cast<long long>(t) * a.ld;
    L* out = dlogits + static_cast<long long>(t) * a.E;
    const bool pick = lane < a.k;
    const int id = pick ? ids[static_cast<long long>(t) * a.k + lane] : 0;
    const bool in = pick && id >= 0 && id < a.E;
    const float dw = in ? dweights[static_cast<long long>(t) * a.k + lane] : 0.f;
    const float x = in ? load_logit(row + id) : -INFINITY;
    float top = 0.f, total = 1.f, s, inner = 0.f;
    const bool whole = !a.sigmoid && !a.renormalize;
    if (whole) {
      top = -INFINITY;
      for (int e = lane; e < a.E; e += 32) top = fmaxf(top, load_logit(row + e));
      top = row_max(top);
      float sum = 0.f;
      for (int e = lane; e < a.E; e += 32) {
        const float y = load_logit(row + e);
        sum += y == -INFINITY ? 0.f : __expf(y - top);
      }
      total = warp_sum32(sum);
    } else if (!a.sigmoid) {
      top = row_max(x);
    }
    if (a.sigmoid) s = in ? __fdividef(1.f, 1.f + __expf(-x)) : 0.f;
    else s = x == -INFINITY ? 0.f : __fdividef(__expf(x - top), fmaxf(total, 1.f));
    float d = a.scale * dw;
    if (a.renormalize) {
      const float inv = __fdividef(1.f, warp_sum32(s) + 1e-20f);
      d = d * inv - warp_sum32(d * s * inv) * inv;
    }
    if (whole) {
      inner = warp_sum32(d * s);
      for (int e = lane; e < a.E; e += 32) {
        const float y = load_logit(row + e);
        store_logit(out + e, y == -INFINITY ? 0.f : -__fdividef(__expf(y - top), fmaxf(total, 1.f)) * inner);
      }
    } else {
      for (int e = lane; e < a.E; e += 32) store_logit(out + e, 0.f);
    }
    __syncwarp();                                // the picks overwrite what another lane wrote above
    if (in) store_logit(out + id, a.sigmoid ? d * s * __fdividef(1.f, 1.f + __expf(x)) : s * (d - inner));
  }
}

bool fits(const RouteArgs& a) {
  return a.T >= 0 && a.E >= 1 && a.E <= RT_MAX_E && a.k >= 1 && a.k <= RT_MAX_K && a.k <= a.E && a.groups >= 1 &&
         a.groups <= RT_MAX_GROUPS && a.E % a.groups == 0 && a.keep >= 1 && a.keep <= a.groups &&
         a.k <= a.keep * (a.E / a.groups) && a.ld >= a.E;
}

}  // namespace
}  // namespace ss

extern "C" {
using namespace ss;

int ss_select_experts(const void* logits, int bf16_logits, long long ld, const float* bias, int T, int E, int k, int groups,
                      int keep_groups, int sigmoid, int renormalize, float scale, int* ids, float* weights, int* counts,
                      void* stream) {
  const RouteArgs a{T, E, k, groups, keep_groups, sigmoid, renormalize, ld, scale, bias};
  if (!fits(a)) return -2;
  cudaStream_t s = (cudaStream_t)stream;
  const int blocks = (T + RT_WARPS - 1) / RT_WARPS, grid = blocks < 1 ? 1 : blocks < 148 * 8 ? blocks : 148 * 8;
  if (grid > 1) {                                // a single block writes the counts whole
    const cudaError_t e = cudaMemsetAsync(counts, 0, sizeof(int) * E, s);
    if (e != cudaSuccess) return (int)e;
  }
  const bool plain = bias == nullptr && groups == 1;
  auto go = [&](auto kern, auto* x) {
    kern<<<grid, RT_THREADS, plain ? 0 : sizeof(double) * E * RT_WARPS, s>>>(x, a, ids, weights, counts);
    return (int)cudaGetLastError();
  };
  auto by_type = [&](auto* x) {
    using L = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    if (plain) {
      if (E <= 64) return go(select_experts_kernel<2, true, L>, x);
      if (E <= 128) return go(select_experts_kernel<4, true, L>, x);
      if (E <= 256) return go(select_experts_kernel<8, true, L>, x);
      return go(select_experts_kernel<16, true, L>, x);
    }
    if (E <= 64) return go(select_experts_kernel<2, false, L>, x);
    if (E <= 128) return go(select_experts_kernel<4, false, L>, x);
    if (E <= 256) return go(select_experts_kernel<8, false, L>, x);
    return go(select_experts_kernel<16, false, L>, x);
  };
  return bf16_logits ? by_type((const __nv_bfloat16*)logits) : by_type((const float*)logits);
}

// dlogits [T, E] contiguous, in the logits' type, every element written.
int ss_select_experts_bwd(const void* logits, int bf16_logits, long long ld, const int* ids, const float* dweights, int T, int E,
                          int k, int sigmoid, int renormalize, float scale, void* dlogits, void* stream) {
  const RouteArgs a{T, E, k, 1, 1, sigmoid, renormalize, ld, scale, nullptr};
  if (!fits(a)) return -2;
  if (T == 0) return 0;
  const int blocks = (T + RT_WARPS - 1) / RT_WARPS, grid = blocks < 148 * 16 ? blocks : 148 * 16;
  if (bf16_logits)
    select_experts_bwd_kernel<<<grid, RT_THREADS, 0, (cudaStream_t)stream>>>((const __nv_bfloat16*)logits, a, ids, dweights,
                                                                             (__nv_bfloat16*)dlogits);
  else
    select_experts_bwd_kernel<<<grid, RT_THREADS, 0, (cudaStream_t)stream>>>((const float*)logits, a, ids, dweights,
                                                                             (float*)dlogits);
  return (int)cudaGetLastError();
}
}  // extern "C"
