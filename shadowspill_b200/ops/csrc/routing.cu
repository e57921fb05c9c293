// Selection of experts for sm_100a: softmax or sigmoid scores, a bias that only selects, groups, top-k, renormalised and
// scaled weights, a histogram; and the gradient of the weights.
//
//   s = sigmoid(x) or softmax(x), key = s + bias; a group's score is the sum of its two largest keys; the k largest keys of
//   the best groups are the picks, ties to the lowest index; w_j = scale s_j / (sum_i s_i + 1e-20), or scale s_j.
//
// Which experts are picked is defined by keys in 64 bits. The kernel forms them in 32 and looks at the gaps between the picks,
// to the best key left over, and between the groups kept and dropped: where a gap is within the error of its keys, the groups or the
// candidates are compared again in 64 bits. Where nothing is added to the scores and there are no groups the logits themselves are compared,
// which needs neither.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "chained_launch.cuh"
#include "launchers.h"

namespace ss {
namespace {

constexpr int RT_THREADS = 128, RT_WARPS = RT_THREADS / 32;
constexpr int RT_MAX_E = 512, RT_MAX_GROUPS = 32;
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
__device__ __forceinline__ float warp_max32(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}

// exp and 1 / (1 + exp(-x)) for keys, whose errors are allowed for: the argument's product is rounded, 6e-8 |x| of the result, and denormal
// results are zero.
constexpr float LOG2E = 1.44269504f;
__device__ __forceinline__ float ex2(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}
__device__ __forceinline__ float exp_of(float x) { return ex2(x * LOG2E); }
__device__ __forceinline__ float sigmoid_of(float x) {
  float s;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.f + exp_of(-x)));
  return s;
}

// A quotient by a normal denominator: the approximate reciprocal, then a Newton step on the quotient by its remainder, after which it is off by
// little more than its own rounding. (The compiler's division keeps registers for ranges that do not come up here: 65,537 x 512 in groups 145 ->
// 158 us.)
__device__ __forceinline__ float quotient(float x, float by) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(by));
  const float q = x * y;
  return fmaf(fmaf(-by, q, x), y, q);
}
// 1 / (1 + exp(-x)) as weights and gradients have it: 2 steps of exp's and one each of the sum's and the quotient's, denormal results kept.
// `other` receives 1 / (1 + exp(x)).
__device__ __forceinline__ float sigmoid_score(float x, float& other) {
  const float e = expf(-fabsf(x)), high = quotient(1.f, 1.f + e), low = quotient(e, 1.f + e);
  other = x < 0.f ? high : low;
  return x < 0.f ? low : high;
}

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
  F score = size > 1 ? best + second : best;
  score = score == score ? score : F(-INFINITY);             // inf - inf
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
  gap = fabs(worst) < F(3e38) ? worst - left : F(NAN);       // near the end of fp32's range a sum says nothing, nor do two of -inf
  unsigned bits = 0;
  for (int g = 0; g < a.groups; ++g) bits |= __shfl_sync(FULL, static_cast<unsigned>(kept), g * per) << g;
  return bits;
}

// A row's softmax's sum in 64 bits, of the lanes' own values where LANES share a row: 1 for a row of -inf, NaN for one with a NaN or +inf, whose
// keys are then all NaN.
__device__ __forceinline__ double term64(float x, float top) { return x == -INFINITY ? 0.0 : exp(static_cast<double>(x) - top); }
template <int LANES>
__device__ __forceinline__ double sum64(double part) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) part += __shfl_xor_sync(FULL, part, o);
  return part == 0.0 ? 1.0 : part;
}
__device__ __forceinline__ double score64(float x, float top, double total, bool sigmoid) {
  return sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(x))) : term64(x, top) / total;
}
__device__ __forceinline__ double key64(float x, float top, double total, const float* bias, int e, bool sigmoid) {
  double v = score64(x, top, total, sigmoid);
  if (bias != nullptr) v += bias[e];
  return v == v ? v : -INFINITY;
}

// A row's largest logit and its softmax's sum in 64 bits, by a whole warp.
template <class L>
__device__ __forceinline__ double whole_sum64(const L* row, const RouteArgs& a, int lane, float& top) {
  top = -INFINITY;
  for (int e = lane; e < a.E; e += 32) top = fmaxf(top, load_logit(row + e));
  top = warp_max32(top);
  double part = 0.0;
  if (!a.sigmoid)
    for (int e = lane; e < a.E; e += 32) part += term64(load_logit(row + e), top);
  return sum64<32>(part);
}
// All keys of a row in 64 bits into shared memory, by a whole warp, and the groups that stay, as bits.
template <class L>
__device__ __noinline__ unsigned exact_keys(const L* row, const RouteArgs& a, double* keys, int lane) {
  float top;
  const double total = whole_sum64(row, a, lane, top);
  for (int e = lane; e < a.E; e += 32) keys[e] = key64(load_logit(row + e), top, total, a.bias, e, a.sigmoid);
  __syncwarp();
  unsigned bits = FULL;
  if (a.groups > 1) {
    double gap;
    bits = kept_groups(keys, a, lane, gap);
    __syncwarp();
  }
  return bits;
}

// Keys of the groups that do not stay become -inf.
__device__ __forceinline__ void drop_groups(const RouteArgs& a, unsigned bits, const unsigned char* group_of, double* keys, int lane) {
  for (int e = lane; e < a.E; e += 32)
    if (!((bits >> group_of[e]) & 1)) keys[e] = -INFINITY;
  __syncwarp();
}
// The largest key that is not picked yet, by a whole warp; `taken`: this lane's experts that are, by place.
__device__ __forceinline__ int next_pick(const RouteArgs& a, const double* keys, int lane, unsigned& taken) {
  double best = -INFINITY;
  int at = INT_MAX;
  for (int i = 0; lane + 32 * i < a.E; ++i) {
    const int e = lane + 32 * i;
    if (!((taken >> i) & 1) && (at == INT_MAX || keys[e] > best)) { best = keys[e]; at = e; }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ob = __shfl_xor_sync(FULL, best, o);
    const int oa = __shfl_xor_sync(FULL, at, o);
    if (oa != INT_MAX && (at == INT_MAX || ob > best || (ob == best && oa < at))) { best = ob; at = oa; }
  }
  if ((at & 31) == lane) taken |= 1u << (at >> 5);
  return at;
}
// The picks among those keys; lane j returns the j-th.
__device__ __noinline__ int picks_exact(const RouteArgs& a, unsigned bits, const unsigned char* group_of, double* keys, int lane) {
  drop_groups(a, bits, group_of, keys, lane);
  unsigned taken = 0;
  int mine = 0;
  for (int j = 0; j < a.k; ++j) {
    const int at = next_pick(a, keys, lane, taken);
    if (lane == j) mine = at;
  }
  __syncwarp();
  return mine;
}

// Among the `n` candidates of a token, one to a lane (`id`, or -1), the number that come before this lane's by keys in 64 bits.
// `top`: the row's largest logit; `most`: the largest n of the warp.
template <int LANES, class L>
__device__ __noinline__ int exact_places(const L* row, const RouteArgs& a, float top, int lane, int id, int n, int most) {
  const int rank = lane % LANES, base = lane - rank;
  double part = 0.0;
  if (!a.sigmoid)
    for (int e = rank; e < a.E; e += LANES) part += term64(load_logit(row + e), top);
  const double total = sum64<LANES>(part);
  const double mine = id >= 0 ? key64(load_logit(row + id), top, total, a.bias, id, a.sigmoid) : -INFINITY;
  int ahead = 0;
  for (int c = 0; c < most; ++c) {
    const double other = __shfl_sync(FULL, mine, base + min(c, LANES - 1));
    const int whose = __shfl_sync(FULL, id, base + min(c, LANES - 1));
    ahead += c < n && (other > mine || (other == mine && whose < id));
  }
  return ahead;
}

// PER consecutive values of a row from expert `first` on, -inf behind the last expert.
template <int PER, class L>
__device__ __forceinline__ void load_row(const L* row, int first, int E, bool vectors, float (&v)[PER]) {
  constexpr int BYTES = PER * sizeof(L) < 16 ? PER * sizeof(L) : 16, N = BYTES / sizeof(L);
  if (vectors && first + PER <= E) {
#pragma unroll
    for (int c = 0; c < PER / N; ++c) {
      alignas(16) L piece[N];
      if (BYTES == 16) *reinterpret_cast<uint4*>(piece) = *reinterpret_cast<const uint4*>(row + first + c * N);
      else if (BYTES == 8) *reinterpret_cast<uint2*>(piece) = *reinterpret_cast<const uint2*>(row + first + c * N);
      else *reinterpret_cast<uint32_t*>(piece) = *reinterpret_cast<const uint32_t*>(row + first + c * N);
#pragma unroll
      for (int i = 0; i < N; ++i) v[c * N + i] = load_logit(piece + i);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = first + i < E ? load_logit(row + first + i) : -INFINITY;
}

// LANES to a token, PER consecutive experts to a lane. Bound by instructions: 8,192 tokens of 64 experts take 8 us, of 256
// with a bias 19, and 65,537 of 512 in groups 124 us, 1,300 instructions a token with 60 % of the issue slots
// used; their memory would take 0.5, 1.4 and 11. At the registers that eight (seven) blocks an SM leave, the kernels that form keys spill
// 84 to 220 bytes a thread, most of it around the rare paths.
//
// The k-th largest of the lanes' own maxima bounds the k-th largest key from below: the keys from it on, a dozen where k
// is 8, are gathered by one place to a lane and sorted. Where they are more than the lanes (one token in twenty for k = 8 of 16
// lanes; many equal keys), or fewer than k can be compared, the picks are taken one by one instead. A doubt among those is settled
// over the whole row, one among the gathered, which hold whatever may come before the k-th, between them.
constexpr int rt_resident(int per) { return per == 16 ? 7 : 8; }     // blocks that an SM's registers hold
template <int LANES, int PER, bool LOGITS, class L>
__global__ void __launch_bounds__(RT_THREADS, rt_resident(PER))
select_experts_kernel(const L* logits, bool vectors, bool bias_vectors, RouteArgs a, int* ids, float* weights, int* counts) {
  // Several blocks count behind the kernel that clears the counts, which lets this one start beside it, after its own wait for
  // all work before: what it waits for itself is the cleared counts alone, at the end (chained_launch.cuh: the exception).
  const bool alone = gridDim.x == 1;
  if (alone) chain_wait();
  constexpr int TOKENS = 32 / LANES;             // of a warp
  __shared__ int hist[RT_MAX_E];
  __shared__ unsigned char group_of[RT_MAX_E];
  __shared__ float2 gathered[RT_WARPS][32];
  extern __shared__ double warp_keys[];          // E per warp, where keys may have to be formed in 64 bits
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = lane % LANES, base = lane - rank;
  const unsigned own = LANES == 32 ? FULL : ((1u << LANES) - 1) << base;         // the lanes of this token
  const int size = a.E / a.groups, group_lanes = size / PER;
  const bool lane_groups = size % PER == 0 && (group_lanes & (group_lanes - 1)) == 0;
  for (int e = threadIdx.x; e < a.E; e += RT_THREADS) {
    hist[e] = 0;
    if (!LOGITS) group_of[e] = static_cast<unsigned char>(e / size);
  }
  __syncthreads();
  double* const keys64 = warp_keys + warp * a.E;
  unsigned ups = 0;                              // the sorting steps in which this lane keeps the larger of two
  {
    int step = 0;
#pragma unroll
    for (int n = 2; n <= LANES; n *= 2)
#pragma unroll
      for (int o = n / 2; o > 0; o >>= 1, ++step) ups |= static_cast<unsigned>(((rank & n) == 0) == ((rank & o) == 0)) << step;
  }
  const int tokens = gridDim.x * RT_WARPS * TOKENS;
  for (int t0 = (blockIdx.x * RT_WARPS + warp) * TOKENS; t0 < a.T; t0 += tokens) {
    const int t = t0 + base / LANES;
    const bool real = t < a.T;
    const L* row = logits + static_cast<long long>(real ? t : t0) * a.ld;
    const int first = rank * PER;
    float v[PER];
    load_row<PER>(row, first, a.E, vectors, v);
    float top = 0.f, total = 1.f;
    bool bad = false;                            // a softmax with a NaN or +inf in it
    const bool whole = !a.sigmoid && !(LOGITS && a.renormalize);         // the softmax's sum is needed
    if (!a.sigmoid && !whole) {
#pragma unroll
      for (int i = 0; i < PER; ++i) bad = bad || !(v[i] < INFINITY);
      bad = (__ballot_sync(FULL, bad) & own) != 0;
    }
    if (whole) {
      top = v[0];
#pragma unroll
      for (int i = 1; i < PER; ++i) top = fmaxf(top, v[i]);
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
      total = 0.f;
      const float none = top == -INFINITY ? 0.f : top;       // a row of -inf: exponentials of zero
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float e = exp_of(v[i] - none);
        if (!LOGITS) v[i] = e;
        total += e;
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) total += __shfl_xor_sync(FULL, total, o);
      bad = !(total < INFINITY);                 // exponentials of NaN and of inf - inf
      total = fmaxf(total, 1.f);                 // the largest alone is 1
    }
    // v becomes the keys: -inf for what cannot be picked or compared
    float slack = 0.f;
    if (!LOGITS) {
      // errors of a key before its sum is rounded. sigmoid: exp's |x| 6e-8 + 2.4e-7 times s (1 - s), the reciprocal's 6e-8 s and the
      // sum 1 + exp's as much; softmax: exp's times exp(-|x|), its sum's and the reciprocal's, 4e-7 together, of the largest
      const float inv = bad ? NAN : __fdividef(1.f, total);            // no key of a bad row compares
      slack = a.sigmoid ? 3e-7f : 1e-6f * inv;
      float b[PER];
      if (a.bias != nullptr) load_row<PER>(a.bias, first, a.E, bias_vectors, b);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        v[i] = a.sigmoid ? sigmoid_of(v[i]) : v[i] * inv;
        if (a.bias != nullptr) v[i] += b[i];     // -inf behind the last expert
        else if (first + i >= a.E) v[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = fmaxf(v[i], -INFINITY);         // NaN
    if (!LOGITS && a.groups > 1) {
      unsigned stay = 0;
      float gap, big;                            // big: the largest of the keys that group scores are sums of
      if (lane_groups) {
        float best = -INFINITY, second = -INFINITY;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          second = fmaxf(second, fminf(best, v[i]));
          best = fmaxf(best, v[i]);
        }
        for (int o = group_lanes >> 1; o > 0; o >>= 1) {
          const float c = __shfl_xor_sync(FULL, best, o), d = __shfl_xor_sync(FULL, second, o);
          second = fmaxf(fmaxf(second, d), fminf(best, c));
          best = fmaxf(best, c);
        }
        const float score = size > 1 ? fmaxf(best + second, -INFINITY) : best;             // NaN of inf - inf: -inf
        const int group = rank / group_lanes;
        int ahead = 0;                           // groups that come before this lane's
        for (int g = 0; g < a.groups; ++g) {
          const float other = __shfl_sync(FULL, score, base + g * group_lanes);
          ahead += other > score || (other == score && g < group);
        }
        const bool in = group < a.groups, kept = in && ahead < a.keep;
        float worst = kept ? score : INFINITY, left = in && !kept ? score : -INFINITY;
        big = fmaxf(best > -INFINITY ? fabsf(best) : 0.f, second > -INFINITY ? fabsf(second) : 0.f);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
          worst = fminf(worst, __shfl_xor_sync(FULL, worst, o));
          left = fmaxf(left, __shfl_xor_sync(FULL, left, o));
          big = fmaxf(big, __shfl_xor_sync(FULL, big, o));
        }
        gap = fabsf(worst) < 3e38f ? worst - left : NAN;     // as in kept_groups
        stay = kept ? 1u << group : 0u;          // this lane's own group
      } else {
        float* keys = reinterpret_cast<float*>(keys64);
        gap = big = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) big = fmaxf(big, v[i] > -INFINITY ? fabsf(v[i]) : 0.f);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(FULL, big, o));
        for (int part = 0; part < TOKENS; ++part) {          // the warp's tokens one after the other
          if (base == part * LANES) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
              if (first + i < a.E) keys[first + i] = v[i];
          }
          __syncwarp();
          float g;
          const unsigned b = kept_groups(keys, a, lane, g);
          if (base == part * LANES) { stay = b; gap = g; }
          __syncwarp();
        }
      }
      const bool doubtful = a.keep < a.groups && !(gap > 4.f * slack + 5e-7f * big);
      unsigned redo = __ballot_sync(FULL, doubtful && rank == 0 && real);
      while (redo) {                             // the whole warp, token by token: the groups by keys in 64 bits
        const int at = __ffs(redo) - 1;
        redo &= redo - 1;
        const unsigned bits = exact_keys(logits + static_cast<long long>(t0 + at / LANES) * a.ld, a, keys64, lane);
        if (base == at) stay = bits;
        __syncwarp();
      }
      if (lane_groups) {
        if (!((stay >> (rank / group_lanes)) & 1)) {
#pragma unroll
          for (int i = 0; i < PER; ++i) v[i] = -INFINITY;
        }
      } else {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (first + i < a.E && !((stay >> group_of[first + i]) & 1)) v[i] = -INFINITY;
      }
    }
    // the k-th largest of the lanes' maxima
    float most = v[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) most = fmaxf(most, v[i]);
    int step = 0;
#pragma unroll
    for (int n = 2; n <= LANES; n *= 2)
#pragma unroll
      for (int o = n / 2; o > 0; o >>= 1, ++step) {
        const float other = __shfl_xor_sync(FULL, most, o);
        most = (ups >> step) & 1 ? fmaxf(most, other) : fminf(most, other);
      }
    const float least = __shfl_sync(FULL, most, base + min(a.k, LANES) - 1);
    const float from = LOGITS ? least : least - (2.f * slack + 2.5e-7f * fabsf(least));      // and what an error may put before it
    unsigned chosen = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) chosen |= static_cast<unsigned>(v[i] >= from) << i;
    int place = __popc(chosen), all;
    {
      const int n = place;
#pragma unroll
      for (int o = 1; o < LANES; o *= 2) {
        const int before = __shfl_up_sync(FULL, place, o, LANES);
        if (rank >= o) place += before;
      }
      all = __shfl_sync(FULL, place, base + LANES - 1);
      place -= n;
    }
    const bool sorted = least > -INFINITY && all >= a.k && all <= LANES;     // a key of inf leaves nothing to choose by
    int mine = 0;
    if (__any_sync(FULL, sorted)) {
      if (sorted) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if ((chosen >> i) & 1) gathered[warp][base + place++] = make_float2(v[i], __int_as_float(first + i));
      }
      __syncwarp();
      float key = -INFINITY;
      int id = INT_MAX;
      const bool holds = sorted && rank < all;
      if (holds) {
        const float2 c = gathered[warp][lane];
        key = c.x;
        id = __float_as_int(c.y);
      }
      __syncwarp();
      step = 0;
#pragma unroll
      for (int n = 2; n <= LANES; n *= 2)
#pragma unroll
        for (int o = n / 2; o > 0; o >>= 1, ++step) {
          const float other = __shfl_xor_sync(FULL, key, o);
          const int whose = __shfl_xor_sync(FULL, id, o);
          const bool ahead = other > key || (other == key && whose < id);
          if (ahead == static_cast<bool>((ups >> step) & 1)) { key = other; id = whose; }
        }
      if (!LOGITS) {
        const float next = __shfl_down_sync(FULL, key, 1, LANES);
        const bool close = holds && rank < a.k && rank + 1 < all && key - next <= 2.f * slack + 2.5e-7f * fabsf(key);
        const unsigned near = __ballot_sync(FULL, close);
        if (near != 0) {                         // some pick of the warp's is in doubt: the candidates again, by their keys in 64 bits
          const int n = sorted ? all : 0, most_of = LANES == 32 ? n : max(n, __shfl_xor_sync(FULL, n, 16));
          const int ahead = exact_places<LANES>(row, a, top, lane, holds ? id : -1, n, most_of);
          if (holds) gathered[warp][base + ahead].y = __int_as_float(id);
          __syncwarp();
          if (holds) id = __float_as_int(gathered[warp][lane].y);
        }
      }
      __syncwarp();                              // the next token's candidates come into the same place
      mine = id;
    }
    const bool one_by_one = !sorted;
    bool doubt = false;
    if (__any_sync(FULL, one_by_one)) {
      float last_key = INFINITY;                 // the pick before, of those that compare, then of the rest
      int last_id = -1, left = -1, found = -1;
      for (int j = 0; j < a.k + !LOGITS; ++j) {  // one more where the last pick's lead counts
        float best = -INFINITY;                  // the largest behind the last pick
        int at = INT_MAX;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const bool behind = v[i] < last_key || (v[i] == last_key && first + i > last_id);
          if (behind && v[i] > best) { best = v[i]; at = first + i; }
        }
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
          const float b = __shfl_xor_sync(FULL, best, o);
          const int w = __shfl_xor_sync(FULL, at, o);
          if (b > best || (b == best && w < at)) { best = b; at = w; }
        }
        if (!LOGITS) doubt = doubt || (best == -INFINITY ? j < a.k : last_key - best <= 2.f * slack + 2.5e-7f * fabsf(best));
        // nothing left that compares: the first experts that do not, in their order (looked for by all lanes: the warp's tokens
        // differ in this)
        int rest = INT_MAX;
        if (LOGITS) {
#pragma unroll
          for (int i = PER - 1; i >= 0; --i)
            if (first + i < a.E && v[i] == -INFINITY && first + i > left) rest = first + i;
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) rest = min(rest, __shfl_xor_sync(FULL, rest, o));
        }
        if (best == -INFINITY) {
          at = left = rest;
        } else {
          last_key = best;
          last_id = at;
        }
        if (rank == j) found = at;
      }
      if (one_by_one) mine = found;
    }
    if (!LOGITS) {
      unsigned redo = __ballot_sync(FULL, one_by_one && doubt && rank == 0 && real);
      while (redo) {                             // the whole warp, token by token
        const int at = __ffs(redo) - 1;
        redo &= redo - 1;
        const unsigned bits = exact_keys(logits + static_cast<long long>(t0 + at / LANES) * a.ld, a, keys64, lane);
        const int pick = picks_exact(a, bits, group_of, keys64, lane);
        const int moved = __shfl_sync(FULL, pick, rank);
        if (base == at) mine = moved;
      }
    }
    const bool pick = real && rank < a.k;
    const float x = pick ? load_logit(row + mine) : -INFINITY;
    float s;
    if (a.sigmoid) {
      float other;
      s = sigmoid_score(x, other);               // -inf where there is no pick
    } else {
      if (!whole) {                              // the scores' common factor leaves with the renormalisation
        top = x > -INFINITY ? x : -INFINITY;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
      }
      s = x == -INFINITY ? 0.f : expf(x - top);
      if (whole) s = quotient(s, total);
      if (bad) s = NAN;
    }
    float sum = s;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    const float w = a.renormalize ? a.scale * quotient(s, sum + 1e-20f) : a.scale * s;
    if (pick) {
      ids[static_cast<long long>(t) * a.k + rank] = mine;
      weights[static_cast<long long>(t) * a.k + rank] = w;
      atomicAdd(&hist[mine], 1);
    }
  }
  if (!alone) chain_wait();
  chain_release();
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += RT_THREADS) {
    if (alone) counts[e] = hist[e];
    else if (hist[e]) atomicAdd(counts + e, hist[e]);
  }
}

// More picks than a warp has lanes: all keys in 64 bits, picked one by one, a warp to a token. 8,192 tokens, 40 of 256 experts by sigmoid: 126 us.
template <class L>
__global__ void __launch_bounds__(RT_THREADS)
select_many_kernel(const L* logits, RouteArgs a, int* ids, float* weights, int* counts) {
  chain_wait();
  chain_release();
  __shared__ int hist[RT_MAX_E];
  __shared__ unsigned char group_of[RT_MAX_E];
  extern __shared__ double warp_keys[];          // E to a warp; then the warps' picks
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, size = a.E / a.groups;
  double* const keys = warp_keys + warp * a.E;
  int* const picks = reinterpret_cast<int*>(warp_keys + RT_WARPS * a.E) + warp * a.k;
  for (int e = threadIdx.x; e < a.E; e += RT_THREADS) {
    hist[e] = 0;
    group_of[e] = static_cast<unsigned char>(e / size);
  }
  __syncthreads();
  for (int t = blockIdx.x * RT_WARPS + warp; t < a.T; t += gridDim.x * RT_WARPS) {
    const L* row = logits + static_cast<long long>(t) * a.ld;
    float top;
    const double total = whole_sum64(row, a, lane, top);
    if (a.bias == nullptr && a.groups == 1) {    // the logits themselves, as above
      for (int e = lane; e < a.E; e += 32) keys[e] = fmaxf(load_logit(row + e), -INFINITY);
      __syncwarp();
    } else {
      drop_groups(a, exact_keys(row, a, keys, lane), group_of, keys, lane);
    }
    unsigned taken = 0;
    for (int j = 0; j < a.k; ++j) {
      const int at = next_pick(a, keys, lane, taken);
      if (lane == 0) picks[j] = at;
    }
    __syncwarp();
    double sum = 0.0;
    for (int j = lane; j < a.k; j += 32) sum += score64(load_logit(row + picks[j]), top, total, a.sigmoid);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    const double by = a.renormalize ? a.scale / (sum + 1e-20) : a.scale;
    for (int j = lane; j < a.k; j += 32) {
      const int e = picks[j];
      ids[static_cast<long long>(t) * a.k + j] = e;
      weights[static_cast<long long>(t) * a.k + j] = static_cast<float>(score64(load_logit(row + e), top, total, a.sigmoid) * by);
      atomicAdd(&hist[e], 1);
    }
    __syncwarp();                                // keys and picks of the next token come into the same place
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += RT_THREADS)
    if (hist[e]) atomicAdd(counts + e, hist[e]);
}

__global__ void clear_counts_kernel(int* counts, int E) {
  chain_wait();                                  // ahead of the release: what comes behind reads inputs without a wait of its own
  chain_release();
  for (int e = threadIdx.x; e < E; e += blockDim.x) counts[e] = 0;
}

// A row by its lanes: pieces of N elements, lane + 32 c the c-th of a lane, so that an instruction takes consecutive ones. WHOLE: the row starts on a
// piece's boundary and has whole pieces; by element otherwise.
template <int PER, bool WHOLE, class L> struct Spread {
  static constexpr int MOST = 16 / static_cast<int>(sizeof(L)), N = !WHOLE ? 1 : PER < MOST ? PER : MOST;
  using Piece = std::conditional_t<N * sizeof(L) == 16, uint4, std::conditional_t<N * sizeof(L) == 8, uint2, std::conditional_t<N * sizeof(L) == 4, uint32_t, uint16_t>>>;
  __device__ static int first(int lane, int c) { return (lane + 32 * c) * N; }
  __device__ static void load(const L* row, int lane, int E, float (&v)[PER]) {
#pragma unroll
    for (int c = 0; c < PER / N; ++c) {
      const int e = first(lane, c);
      alignas(16) L piece[N];
      if (e < E) *reinterpret_cast<Piece*>(piece) = *reinterpret_cast<const Piece*>(row + e);
#pragma unroll
      for (int i = 0; i < N; ++i) v[c * N + i] = e < E ? load_logit(piece + i) : -INFINITY;
    }
  }
  __device__ static void store(L* row, int lane, int E, const float (&v)[PER]) {
#pragma unroll
    for (int c = 0; c < PER / N; ++c) {
      const int e = first(lane, c);
      alignas(16) L piece[N];
#pragma unroll
      for (int i = 0; i < N; ++i) store_logit(piece + i, v[c * N + i]);
      if (e < E) *reinterpret_cast<Piece*>(row + e) = *reinterpret_cast<const Piece*>(piece);
    }
  }
};

// With c_j the picked scores, S = sum_j c_j + 1e-20, A = sum_j dw_j c_j / S: dc_j = scale (dw_j - A) / S, or scale dw_j as they are, and
//   sigmoid  dx_e = dc_e s_e (1 - s_e);   softmax  dx_e = s_e (dc_e - B) with B = sum_j dc_j s_j, which is scale A 1e-20 / S if renormalised.
// B counts there where the picks' scores are next to nothing: a bias can bring that about, and the row's largest logit shows it. With a pick
// within 20 of that, the picks hold e^-20 / 512 = 4e-12 of the row or more, 1e-20 is under the rounding of their sum, and scores are taken
// relative to the largest pick; experts that were not picked get zero.
// A warp to a token. 65,537 x 512 bf16: sigmoid 22 us (67 MB written), softmax renormalised 25.5 (67 MB read too, for the largest logit), not
// renormalised 33 (an exponential for each, kept in registers). 8,192 x 256 fp32, sigmoid: 4.3, of which a launch is half.
constexpr float PICKS_NEAR = 20.f;
__device__ __forceinline__ float max_or_nan(float x, float y) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}
__device__ __forceinline__ float below(float x, float top) { return x == -INFINITY ? 0.f : exp_of(x - top); }
enum { SIGMOID, SOFTMAX_RENORMALISED, SOFTMAX };
constexpr int bwd_resident(int mode, int per) { return mode != SOFTMAX || per <= 4 ? 16 : per == 8 ? 12 : 10; }
// MANY: more picks than lanes, every 32nd to a lane.
template <int MODE, int PER, bool WHOLE, bool MANY, class L>
__global__ void __launch_bounds__(RT_THREADS, MANY ? 4 : bwd_resident(MODE, PER))
select_experts_bwd_kernel(const L* logits, RouteArgs a, const int* ids, const float* dweights, L* dlogits) {
  using Row = Spread<PER, WHOLE, L>;
  constexpr int OWN = MANY ? RT_MAX_E / 32 : 1;
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31;
  for (int t = blockIdx.x * RT_WARPS + (threadIdx.x >> 5); t < a.T; t += gridDim.x * RT_WARPS) {
    const L* row = logits + static_cast<long long>(t) * a.ld;
    L* out = dlogits + static_cast<long long>(t) * a.E;
    int id[OWN];                                 // -1: none
    float d[OWN], x[OWN], s[OWN], other[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) id[i] = lane + 32 * i < a.k ? ids[static_cast<long long>(t) * a.k + lane + 32 * i] : -1;
    float v[PER], top = -INFINITY;
    if (MODE != SIGMOID) {
      Row::load(row, lane, a.E, v);
#pragma unroll
      for (int i = 0; i < PER; ++i) top = max_or_nan(top, v[i]);
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (id[i] >= a.E) id[i] = -1;
      d[i] = id[i] >= 0 ? a.scale * dweights[static_cast<long long>(t) * a.k + lane + 32 * i] : 0.f;
      x[i] = id[i] >= 0 ? load_logit(row + id[i]) : -INFINITY;
    }
    float total = 1.f, inner = 0.f;
    bool others = MODE == SOFTMAX;               // do experts that were not picked have gradients?
    if (MODE == SIGMOID) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) s[i] = sigmoid_score(x[i], other[i]);
    } else {
      float base = x[0];
#pragma unroll
      for (int i = 1; i < OWN; ++i) base = fmaxf(base, x[i]);
      base = warp_max32(base);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = max_or_nan(top, __shfl_xor_sync(FULL, top, o));
      const bool bad = !(top < INFINITY);        // a NaN or +inf in the row: scores, weights and gradients are NaN
      if (MODE == SOFTMAX_RENORMALISED) others = bad || !(base >= top - PICKS_NEAR);
      if (others) {
        total = 0.f;
        if (MODE == SOFTMAX) {
#pragma unroll
          for (int i = 0; i < PER; ++i) {
            v[i] = below(v[i], top);
            total += v[i];
          }
        } else {
          for (int e = lane; e < a.E; e += 32) total += below(load_logit(row + e), top);
        }
        total = fmaxf(warp_sum32(total), 1.f);
        base = top;
      }
#pragma unroll
      for (int i = 0; i < OWN; ++i) s[i] = bad ? NAN : x[i] == -INFINITY ? 0.f : quotient(expf(x[i] - base), total);
    }
    float mine[OWN], part = 0.f;                 // dc_j s_j
    if (a.renormalize) {
#pragma unroll
      for (int i = 0; i < OWN; ++i) part += s[i];
      const float sum = warp_sum32(part) + 1e-20f;
      part = 0.f;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        mine[i] = quotient(s[i], sum);
        part += d[i] * mine[i];
      }
      const float mean = warp_sum32(part);
#pragma unroll
      for (int i = 0; i < OWN; ++i) mine[i] *= d[i] - mean;
      if (others) inner = mean * quotient(1e-20f, sum);
    } else {
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        mine[i] = d[i] * s[i];
        part += mine[i];
      }
      if (MODE == SOFTMAX) inner = warp_sum32(part);
    }
    const float each = others ? -quotient(inner, total) : 0.f;
    if (MODE == SOFTMAX) {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] *= each;
      Row::store(out, lane, a.E, v);
    } else if (others) {                         // hardly ever: read again instead of kept in registers
      for (int e = lane; e < a.E; e += 32) store_logit(out + e, below(load_logit(row + e), top) * each);
    } else {
      const float zero[PER] = {};
      Row::store(out, lane, a.E, zero);
    }
    __syncwarp();                                // the picks overwrite what another lane wrote above
#pragma unroll
    for (int i = 0; i < OWN; ++i)
      if (id[i] >= 0) store_logit(out + id[i], MODE == SIGMOID ? mine[i] * other[i] : mine[i] - s[i] * inner);
  }
}

bool fits(const RouteArgs& a) {
  return a.T >= 0 && a.T <= 0x7fff0000 && a.E >= 1 && a.E <= RT_MAX_E && a.k >= 1 && a.k <= a.E && a.groups >= 1 &&
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
  if (k > 32) {
    const int blocks = (T + RT_WARPS - 1) / RT_WARPS, grid = blocks < 1 ? 1 : blocks < 148 * 8 ? blocks : 148 * 8;
    const size_t smem = RT_WARPS * (sizeof(double) * E + sizeof(int) * k);
    launch_chained(clear_counts_kernel, 1, 128, 0, s, counts, E);
    if (bf16_logits) launch_chained(select_many_kernel<__nv_bfloat16>, grid, RT_THREADS, smem, s, (const __nv_bfloat16*)logits, a, ids, weights, counts);
    else launch_chained(select_many_kernel<float>, grid, RT_THREADS, smem, s, (const float*)logits, a, ids, weights, counts);
    return (int)cudaGetLastError();
  }
  const bool plain = bias == nullptr && groups == 1;
  // Half a warp to a token where the candidates are hardly ever more than its lanes: a token too many in twenty at k = 8 of 16
  // costs little where logits are compared, but what is doubtful of it is settled over a whole row, which the launch waits for (8,192
  // tokens, k = 8: 64 experts by logits 10.1 us, with whole warps 12.6; 256 with a bias 24.5, with whole warps 19.9).
  const bool halves = (plain ? 2 : 3) * k * groups <= 16 * keep_groups && E <= 256;
  const int lanes = halves ? 16 : 32, per_block = RT_WARPS * (halves ? 2 : 1);
  const int per = (E + lanes - 1) / lanes, most = 148 * rt_resident(per <= 8 ? 8 : 16);
  const int blocks = (T + per_block - 1) / per_block, grid = blocks < 1 ? 1 : blocks < most ? blocks : most;
  if (grid > 1) launch_chained(clear_counts_kernel, 1, 128, 0, s, counts, E);          // a single block writes the counts whole
  auto go = [&](auto kern, auto* x) {
    const bool vectors = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * sizeof(*x) % 16 == 0;
    launch_chained(kern, grid, RT_THREADS, plain ? 0 : sizeof(double) * E * RT_WARPS, s, x, vectors, reinterpret_cast<uintptr_t>(bias) % 16 == 0,
                   a, ids, weights, counts);
    return (int)cudaGetLastError();
  };
  auto by_mode = [&](auto* x, auto logits_only) {
    using X = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
    constexpr bool P = decltype(logits_only)::value;
    if (halves) {
      if (per <= 2) return go(select_experts_kernel<16, 2, P, X>, x);
      if (per <= 4) return go(select_experts_kernel<16, 4, P, X>, x);
      if (per <= 8) return go(select_experts_kernel<16, 8, P, X>, x);
      return go(select_experts_kernel<16, 16, P, X>, x);
    }
    if (per <= 2) return go(select_experts_kernel<32, 2, P, X>, x);
    if (per <= 4) return go(select_experts_kernel<32, 4, P, X>, x);
    if (per <= 8) return go(select_experts_kernel<32, 8, P, X>, x);
    return go(select_experts_kernel<32, 16, P, X>, x);
  };
  auto by_type = [&](auto* x) { return plain ? by_mode(x, std::true_type()) : by_mode(x, std::false_type()); };
  return bf16_logits ? by_type((const __nv_bfloat16*)logits) : by_type((const float*)logits);
}

// dlogits [T, E] contiguous, in the logits' type, every element written.
int ss_select_experts_bwd(const void* logits, int bf16_logits, long long ld, const int* ids, const float* dweights, int T, int E,
                          int k, int sigmoid, int renormalize, float scale, void* dlogits, void* stream) {
  const RouteArgs a{T, E, k, 1, 1, sigmoid, renormalize, ld, scale, nullptr};
  if (!fits(a)) return -2;
  if (T == 0) return 0;
  const int per = (E + 31) / 32, blocks = (T + RT_WARPS - 1) / RT_WARPS;
  auto launch = [&](auto kern, int resident, auto* x, auto* out) {
    launch_chained(kern, blocks < 148 * resident ? blocks : 148 * resident, RT_THREADS, 0, (cudaStream_t)stream, x, a, ids, dweights, out);
    return (int)cudaGetLastError();
  };
  auto go = [&](auto mode, auto n, auto whole, auto* x, auto* out) {
    constexpr int M = decltype(mode)::value, N = decltype(n)::value;
    using X = std::remove_pointer_t<decltype(out)>;
    return launch(select_experts_bwd_kernel<M, N, decltype(whole)::value, false, X>, bwd_resident(M, N), x, out);
  };
  auto by_length = [&](auto mode, auto whole, auto* x, auto* out) {
    if (k > 32) return launch(select_experts_bwd_kernel<decltype(mode)::value, 16, false, true, std::remove_pointer_t<decltype(out)>>, 4, x, out);
    if (per <= 2) return go(mode, std::integral_constant<int, 2>(), whole, x, out);
    if (per <= 4) return go(mode, std::integral_constant<int, 4>(), whole, x, out);
    if (per <= 8) return go(mode, std::integral_constant<int, 8>(), whole, x, out);
    return go(mode, std::integral_constant<int, 16>(), whole, x, out);
  };
  auto by_mode = [&](auto whole, auto* x, auto* out) {
    if (sigmoid) return by_length(std::integral_constant<int, SIGMOID>(), whole, x, out);
    if (renormalize) return by_length(std::integral_constant<int, SOFTMAX_RENORMALISED>(), whole, x, out);
    return by_length(std::integral_constant<int, SOFTMAX>(), whole, x, out);
  };
  auto by_type = [&](auto* x, auto* out) {
    const bool whole = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld * sizeof(*x) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                       E * sizeof(*x) % 16 == 0;
    return whole ? by_mode(std::true_type(), x, out) : by_mode(std::false_type(), x, out);
  };
  return bf16_logits ? by_type((const __nv_bfloat16*)logits, (__nv_bfloat16*)dlogits) : by_type((const float*)logits, (float*)dlogits);
}
}  // extern "C"
