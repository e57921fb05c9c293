// Paired preference loss on a block of logits for sm_100a, forward and gradient.
//
// Sequences 2p and 2p + 1 of the block are the chosen and the rejected answer of pair p:
//   logp_r = x_r[t_r] - lse(x_r);  sum_q = sum over its rows of w_r (logp_r - ref_r) [/ sum of w_r]
//   z_p = beta (sum_2p - sum_2p+1);  L = sum_p f(z_p)
//   dL/dx_r = coef_r (softmax(x_r) - onehot(t_r)),  coef_r = -+ beta f'(z_p) w_r [/ sum of w_r]
// with f = -(1 - e) log sigma(z) - e log sigma(-z), max(0, 1 - z) or (z / beta - 1 / (2 beta))^2.
//
// A row's gradient needs every row of its pair first, so the block is read twice: once for the rows' statistics, where the last row of a
// pair to be done forms the pair's loss and slopes, once for the gradient. Both are bound by memory where the block is large: 4,096 rows of
// 128,256 bf16 words, 70 % of them scored, take 418 to 430 us of which 388 are two reads and a write at the copy rate; 24 rows of 4,096
// are three launches, 15 to 17 us.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "chained_launch.cuh"
#include "launchers.h"

namespace ss {
namespace {

typedef __nv_bfloat16 bf16;

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

// The c-th of a row's `pieces` where the row starts anywhere: the same elements to a thread, hence the same bits, as of aligned rows. The two
// aligned 16 bytes that hold it are read and moved together; the first and last piece go by element, so that nothing
// outside the row is read. (4,096 rows of 50,257 words, without the gradient: 149 us by elements throughout, 100 for 50,256.)
template <class L>
__device__ __forceinline__ void load_piece(const L* x, int c, int pieces, float (&f)[Vec<L>::N]) {
  const L* at = x + static_cast<long long>(c) * Vec<L>::N;
  if (c == 0 || c == pieces - 1) {
#pragma unroll
    for (int e = 0; e < Vec<L>::N; ++e) f[e] = Vec<L>::get(at[e]);
    return;
  }
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15);
  const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(at) - off);
  const uint4 u = q[0], v = q[1];
  uint32_t w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = off & 2 ? __funnelshift_r(w[i], w[i + 1], 16) : w[i];
  Vec<L>::load(make_uint4(w[0], w[1], w[2], w[3]), f);
}

template <class L>
__device__ __forceinline__ void store_elements(L* to, const float (&f)[Vec<L>::N]) {
#pragma unroll
  for (int e = 0; e < Vec<L>::N; ++e) to[e] = Vec<L>::put(f[e]);
}

struct Rows {
  const long long* targets;
  const float* weights;      // null: one each
  const float* ref_logp;     // optional
  const int* cu_seqlens;
  int R, V, pairs;
  // Does row r carry loss? `t` and `w` receive its target and weight.
  __device__ bool scored(int r, long long& t, float& w) const {
    t = targets[r];
    w = weights != nullptr ? weights[r] : 1.f;
    return t >= 0 && t < V && w != 0.f;
  }
  __device__ int bound(int i) const { return min(max(cu_seqlens[i], 0), R); }
  // How many bounds are no larger than row r: by a warp, a 32nd of what is left at each step. In [0, 2 pairs + 1] whatever they hold.
  __device__ int bounds_up_to(int r) const {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = 2 * pairs + 1;
    while (lo < hi) {
      const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step - 1;
      lo += step * __popc(__ballot_sync(0xffffffffu, at < hi && bound(at) <= r));
      hi = min(hi, lo + step - 1);
    }
    return lo;
  }
};
struct PairArgs {
  float beta, smoothing, grad_scale;
  int kind, average;
};
// What the kernels hand on, in one allocation of the caller's. Per row: its weighted log ratio, its weight (0 if nothing is
// scored), its sequence (-1: none), the reference of its exponentials and the reciprocal of their sum. Per sequence, zero at the
// start: the coefficient of its rows by their weight. The pairs' losses; and counters, zero at the start: rows done of each pair, pairs
// done.
struct Work {
  double *ratio, *slope;
  float *weight, *ref, *inv, *pair_loss;
  int *sequence, *rows_done, *pairs_done;
};

// Exponentials are taken of x - ref, where a row's reference is a multiple of 8 no less than its largest logit: most threads of a row
// arrive at the same one, so that few sums are scaled. log2(e) comes in two parts, the smaller product first: a single constant
// shifts every probability the same way, by 1e-7 at 8 below the top, as does a second part that is added after a rounding,
// and sequences of thousands of rows add that up.
constexpr float LOG2E = 1.44269502f, LOG2E_REST = 1.925963e-8f;
// What ex2.approx leaves a sum short of, relatively, where no argument is positive (4 M of them: -5.03e-8 over [-1, 0], -5.08e-8
// over [-20, 0], -4.97e-8 and -5.06e-8 for normal logits of deviation 2 and 1; positive ones are 3.3e-8 over).
constexpr double EX2_SHORT = 5.0e-8;
// Rows whose largest logit is beyond this size, or none, are done by exp(x - top).
constexpr float PLAIN_TOP = 65536.f;

__device__ __forceinline__ float ex2(float x) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
  return e;
}
__device__ __forceinline__ float2 exponents(float x, float y, float minus_ref) {
  const float2 d = __fadd2_rn(make_float2(x, y), make_float2(minus_ref, minus_ref));
  return __ffma2_rn(d, make_float2(LOG2E, LOG2E), __fmul2_rn(d, make_float2(LOG2E_REST, LOG2E_REST)));
}

// A thread's share of a row's sum, exp(-ref) of it.
struct Sum {
  float ref = -1e30f, s = 0.f, top = -INFINITY;
  __device__ __forceinline__ void reach(float largest) {
    top = fmaxf(top, largest);
    if (largest > ref) {
      const float next = 8.f * ceilf(0.125f * largest);
      s *= expf(ref - next);
      ref = next;
    }
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&f)[N]) {
    float largest = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) largest = fmaxf(largest, f[e]);
    reach(largest);
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 x = exponents(f[e], f[e + 1], -ref);
      sum = __fadd2_rn(sum, make_float2(ex2(x.x), ex2(x.y)));
    }
    s += sum.x + sum.y;
  }
};

__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// A row's team: a warp, several of them to a block, or a whole block.
constexpr int BLOCK_OF_WARPS = 128;
template <int TEAM> struct Team {
  static constexpr int BLOCK = TEAM == 32 ? BLOCK_OF_WARPS : TEAM, ROWS = BLOCK / TEAM;
  __device__ static int rank() { return threadIdx.x % TEAM; }
  __device__ static int row() { return blockIdx.x * ROWS + threadIdx.x / TEAM; }
  __device__ static void sync() {
    if (TEAM == 32) __syncwarp(); else __syncthreads();
  }
  __device__ static bool any(bool x) { return TEAM == 32 ? __any_sync(0xffffffffu, x) : __syncthreads_or(x); }
};
template <int TEAM>
__device__ __forceinline__ double team_sum64(double v, double* red) {
  v = warp_sum64(v);
  if (TEAM == 32) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < TEAM / 32; ++i) v += red[i];
  return v;
}

// The pairs' losses in their order into the sum: by the team that has finished the last of them.
template <int TEAM>
__device__ void add_losses(const Rows& rows, const Work& work, float* loss_sum, double* red) {
  __threadfence();
  double total = 0.0;
  for (int i = Team<TEAM>::rank(); i < rows.pairs; i += TEAM) total += __ldcg(work.pair_loss + i);
  total = team_sum64<TEAM>(total, red);
  if (Team<TEAM>::rank() == 0) *loss_sum += static_cast<float>(total);
}

// The loss of pair p from its rows' log ratios, and its sequences' slopes. By one team, when all rows are done. Sums are held
// in 64 bits: they cancel between the two sides.
template <int TEAM>
__device__ void finish_pair(int p, const Rows& rows, const PairArgs& a, const Work& work, float* sums, float* loss_sum,
                            double (*red)[TEAM / 32]) {
  const int rank = Team<TEAM>::rank();
  const int from = rows.bound(2 * p), between = rows.bound(2 * p + 1), end = rows.bound(2 * p + 2);
  double sum[2] = {0.0, 0.0}, mass[2] = {0.0, 0.0};
  bool any0 = false, any1 = false;
  constexpr int AT_ONCE = 8;                     // loads on their way, the last few of them too
  for (int r0 = from + rank; r0 < end; r0 += AT_ONCE * TEAM) {
    double ratio[AT_ONCE];
    float w[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int r = r0 + i * TEAM;
      ratio[i] = r < end ? __ldcg(work.ratio + r) : 0.0;
      w[i] = r < end ? __ldcg(work.weight + r) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int side = r0 + i * TEAM >= between;
      sum[0] += side ? 0.0 : ratio[i];
      sum[1] += side ? ratio[i] : 0.0;
      mass[0] += side ? 0.f : w[i];
      mass[1] += side ? w[i] : 0.f;
      any0 = any0 || (!side && w[i] != 0.f);
      any1 = any1 || (side && w[i] != 0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sum[i] = warp_sum64(sum[i]);
    mass[i] = warp_sum64(mass[i]);
    if ((rank & 31) == 0) {
      red[i][rank >> 5] = sum[i];
      red[2 + i][rank >> 5] = mass[i];
    }
  }
  const bool some = Team<TEAM>::any(any0) & Team<TEAM>::any(any1);
  double loss = 0.0;
  if (rank < 32) {                        // one warp: 64-bit arithmetic has few units
    const int w = rank;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] = warp_sum64(w < TEAM / 32 ? red[i][w] : 0.0);
      mass[i] = warp_sum64(w < TEAM / 32 ? red[2 + i][w] : 0.0);
      if (!a.average) mass[i] = 1.0;
      else sum[i] = mass[i] != 0.0 ? sum[i] / mass[i] : 0.0;
      if (w == 0 && sums != nullptr) sums[2 * p + i] = static_cast<float>(sum[i]);
    }
    const double beta = a.beta, e = a.smoothing, z = beta * (sum[0] - sum[1]);
    double slope;                                  // dL / d sum[0]
    if (a.kind == 0) {
      const double far = exp(-fabs(z)), tail = log1p(far);
      loss = (1.0 - e) * (fmax(-z, 0.0) + tail) + e * (fmax(z, 0.0) + tail);
      slope = beta * (e - (z >= 0.0 ? far : 1.0) / (1.0 + far));
    } else if (a.kind == 1) {
      loss = z < 1.0 ? 1.0 - z : z >= 1.0 ? 0.0 : z;       // NaN stays one
      slope = z < 1.0 ? -beta : 0.0;
    } else {
      const double gap = sum[0] - sum[1] - 0.5 / beta;
      loss = gap * gap;
      slope = 2.0 * gap;
    }
    if (!some) loss = slope = 0.0;
    if (w < 2) {
      const double size = w ? mass[1] : mass[0];
      work.slope[2 * p + w] = size != 0.0 ? (w ? slope : -slope) * a.grad_scale / size : 0.0;
    }
  }
  if (rows.pairs == 1) {
    if (rank == 0) *loss_sum += static_cast<float>(loss);
    return;
  }
  bool last = false;
  if (rank == 0) {
    work.pair_loss[p] = static_cast<float>(loss);
    __threadfence();
    last = atomicAdd(work.pairs_done, 1) == rows.pairs - 1;
  }
  if (Team<TEAM>::any(last)) add_losses<TEAM>(rows, work, loss_sum, red[0]);
}

// The pairs without rows, by one team.
template <int TEAM>
__device__ void finish_empty(const Rows& rows, const Work& work, float* sums, float* loss_sum, double* red) {
  const int rank = Team<TEAM>::rank();
  int empty = 0;
  for (int p = rank; p < rows.pairs; p += TEAM) {
    if (rows.bound(2 * p) < rows.bound(2 * p + 2)) continue;
    if (sums != nullptr) sums[2 * p] = sums[2 * p + 1] = 0.f;
    work.pair_loss[p] = 0.f;
    ++empty;
  }
  __threadfence();
  Team<TEAM>::sync();
  const int all = static_cast<int>(team_sum64<TEAM>(empty, red));
  bool last = false;
  if (rank == 0 && all > 0) last = atomicAdd(work.pairs_done, all) == rows.pairs - all;
  if (Team<TEAM>::any(last)) add_losses<TEAM>(rows, work, loss_sum, red);
}

__global__ void clear_counters_kernel(int* words, int n) {
  chain_wait();                                  // ahead of the release: what comes behind reads its inputs without a wait of its own
  chain_release();
  for (int i = threadIdx.x; i < n; i += blockDim.x) words[i] = 0;
}

// A team per row, and one more for the pairs without rows. 735 MB of rows of 128,256 words: 133 us, 5.5 TB/s, the units of ex2 busy in 74 % of
// the cycles and half the issue slots; without exponentials it would be 122. Loads through a ring in shared memory, a part
// of the exponentials by multiply-adds and blocks that stay while one warp finishes rows for the others were no faster.
template <class L, int TEAM>
__global__ void __launch_bounds__(Team<TEAM>::BLOCK, TEAM == 512 ? 3 : 1)      // 512: 2 otherwise
preference_rows_kernel(const L* logits, long long ld, bool aligned, Rows rows, PairArgs a, Work work, float* logp, float* sums,
                       float* loss_sum) {
  constexpr int WARPS = TEAM / 32;
  __shared__ double red_of[Team<TEAM>::ROWS][4][WARPS];
  __shared__ double parts[WARPS];                // of teams of several warps
  __shared__ float refs[WARPS], tops[WARPS];
  const int rank = Team<TEAM>::rank(), row = Team<TEAM>::row();
  double (*red)[WARPS] = red_of[threadIdx.x / TEAM];
  // This kernel starts beside the one that clears its counters, which has waited for all work before; the
  // counters alone have to be waited for (chained_launch.cuh: the exception). Every block has a row up to the R-th and so waits.
  if (row > rows.R) return;
  if (row == rows.R) {
    chain_wait();
    finish_empty<TEAM>(rows, work, sums, loss_sum, red[0]);
    return;
  }
  long long target;
  float weight;
  const bool scored = rows.scored(row, target, weight);
  if (scored) {
    const L* x = logits + row * ld;
    const float mine = rank == 0 ? Vec<L>::get(x[target]) : 0.f;
    constexpr int N = Vec<L>::N, AHEAD = 4;      // pieces of a thread on their way at once
    Sum part;
    const int pieces = rows.V / N;
    int c = rank;
    if (aligned) {
      const uint4* xv = reinterpret_cast<const uint4*>(x);
      for (; c + (AHEAD - 1) * TEAM < pieces; c += AHEAD * TEAM) {
        uint4 u[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) u[i] = xv[c + i * TEAM];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
          float f[N];
          Vec<L>::load(u[i], f);
          part.add(f);
        }
      }
    }
    for (; c < pieces; c += TEAM) {
      float f[N];
      load_piece(x, c, pieces, f);
      part.add(f);
    }
    for (c = pieces * N + rank; c < rows.V; c += TEAM) {
      const float f[2] = {Vec<L>::get(x[c]), -INFINITY};
      part.add(f);
    }
    float ref = part.ref, top = part.top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    double sum = part.s;
    if (part.ref != ref) sum *= exp(static_cast<double>(part.ref) - ref);
    sum = warp_sum64(sum);
    if (WARPS > 1) {
      if ((rank & 31) == 0) {
        refs[rank >> 5] = ref;
        tops[rank >> 5] = top;
        parts[rank >> 5] = sum;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < WARPS; ++i) {
        ref = fmaxf(ref, refs[i]);
        top = fmaxf(top, tops[i]);
      }
    }
    const bool plain = !(fabsf(top) <= PLAIN_TOP);
    if (plain) {
      sum = 0.0;
      for (c = rank; c < rows.V; c += TEAM) sum += expf(Vec<L>::get(x[c]) - top);
      sum = team_sum64<TEAM>(sum, red[0]);
      ref = top;
    } else if (WARPS > 1 && rank == 0) {
      sum = 0.0;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) sum += refs[i] == ref ? parts[i] : parts[i] * exp(static_cast<double>(refs[i]) - ref);
    }
    if (rank == 0) {
      const double lse = ref + log(plain ? sum : sum + sum * EX2_SHORT);
      const double value = mine - lse;
      logp[row] = static_cast<float>(value);
      work.ratio[row] = weight * (rows.ref_logp != nullptr ? value - rows.ref_logp[row] : value);
      work.ref[row] = ref;
      work.inv[row] = plain ? -1.f / static_cast<float>(sum) : 1.f / static_cast<float>(sum);  // the sign: which exponentials
    }
  } else if (rank == 0) {
    logp[row] = 0.f;
    work.ratio[row] = 0.0;
  }
  const int before = rows.bounds_up_to(row);
  chain_wait();
  const int sequence = before > 0 && before <= 2 * rows.pairs ? before - 1 : -1, pair = sequence >> 1;
  bool last = false;
  if (rank == 0) {
    work.weight[row] = scored ? weight : 0.f;
    work.sequence[row] = sequence;
    if (pair >= 0) {
      const int all = rows.bound(2 * pair + 2) - rows.bound(2 * pair);
      __threadfence();
      last = atomicAdd(work.rows_done + pair, 1) == all - 1;
    }
  }
  if (!Team<TEAM>::any(last)) return;
  __threadfence();
  finish_pair<TEAM>(pair, rows, a, work, sums, loss_sum, red);
}

// From the last row to the first: the rows read last are still in the L2. Nothing is summed here, so a thread may have any elements: the pieces
// on the row's 16-byte boundaries and the few elements before and behind them, stored by element where the
// gradient's boundaries lie elsewhere. Bound by memory: 1.05 GB written and 0.74 read in 272 us, 6.5 TB/s (4,096 rows of 128,256 words, 70 % scored).
// 4,096 rows of 50,257 words, whole calls, 70 % scored: 243 us, by element from the row's start 2.3 times that; of 50,256 words 194. (The choice at the
// store stays in the loop: without it a thread's four stores leave together, 6 % slower.)
template <class L, int TEAM>
__global__ void __launch_bounds__(Team<TEAM>::BLOCK)
preference_grad_kernel(const L* logits, long long ld, const long long* targets, Work work, int R, int V, L* grad, long long ldg) {
  chain_wait();
  const int row = R - 1 - Team<TEAM>::row(), rank = Team<TEAM>::rank();
  if (row < 0) return;
  constexpr int N = Vec<L>::N, AHEAD = 4;
  const L* x = logits + row * ld;
  L* g = grad + row * ldg;
  const int sequence = work.sequence[row];
  const float weight = work.weight[row], coef = sequence >= 0 && weight != 0.f ? static_cast<float>(work.slope[sequence] * weight) : 0.f;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15);
  const bool together = off == static_cast<int>(reinterpret_cast<uintptr_t>(g) & 15);
  const int head = min(static_cast<int>(((16 - off) & 15) / sizeof(L)), V), pieces = (V - head) / N;
  const int rest = V - pieces * N;
  auto single = [&](int i) { return i < head ? i : i + pieces * N; };          // the i-th element outside the pieces
  uint4* gv = reinterpret_cast<uint4*>(g + head);
  if (coef == 0.f) {
    const float zero[N] = {};
    for (int c = rank; c < pieces; c += TEAM) {
      if (together) gv[c] = make_uint4(0, 0, 0, 0);
      else store_elements(g + head + c * N, zero);
    }
    for (int i = rank; i < rest; i += TEAM) g[single(i)] = Vec<L>::put(0.f);
    return;
  }
  const float ref = work.ref[row], inv = work.inv[row], each = coef * fabsf(inv);
  const int target = static_cast<int>(targets[row]);
  if (inv < 0.f) {
    for (int c = rank; c < V; c += TEAM)
      g[c] = Vec<L>::put(each * expf(Vec<L>::get(x[c]) - ref) - (c == target ? coef : 0.f));
    return;
  }
  const int among = target - head, target_piece = among >= 0 ? among / N : -1;         // from the first piece on; -1: in none
  auto piece = [&](const uint4& u, int c) {
    float f[N];
    Vec<L>::load(u, f);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 y = exponents(f[e], f[e + 1], -ref);
      const float2 v = __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), make_float2(each, each));
      f[e] = v.x;
      f[e + 1] = v.y;
    }
    if (c == target_piece) {
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = __fadd_rn(f[e], e == among % N ? -coef : 0.f);
    }
    if (together) gv[c] = Vec<L>::store(f);
    else store_elements(g + head + c * N, f);
  };
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  int c = rank;
  for (; c + (AHEAD - 1) * TEAM < pieces; c += AHEAD * TEAM) {
    uint4 u[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) u[i] = xv[c + i * TEAM];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) piece(u[i], c + i * TEAM);
  }
  for (; c < pieces; c += TEAM) piece(xv[c], c);
  for (int i = rank; i < rest; i += TEAM) {
    const int at = single(i);
    const float2 y = exponents(Vec<L>::get(x[at]), 0.f, -ref);
    g[at] = Vec<L>::put(__fadd_rn(__fmul_rn(ex2(y.x), each), at == target ? -coef : 0.f));     // as in a piece
  }
}

template <class L>
int preference(const L* logits, long long ld, const Rows& rows, const PairArgs& a, const Work& work, float* logp, float* sums,
               float* loss_sum, L* grad, long long ldg, cudaStream_t s) {
  const bool aligned = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && ld % Vec<L>::N == 0;
  // The rows kernel starts beside the kernel that clears its counters. Behind short ones the host is waited for, and a memset is
  // less of its time than a third kernel: 24 rows of 4,096 words 15.0 us with it and 15.7 with a kernel, 333 rows of 32,003 36 and 33.5.
  if (static_cast<long long>(rows.R) * rows.V < 1 << 21) cudaMemsetAsync(work.slope, 0, sizeof(int) * (5ll * rows.pairs + 1), s);
  else launch_chained(clear_counters_kernel, 1, rows.pairs < 64 ? 128 : 1024, 0, s, reinterpret_cast<int*>(work.slope), 5 * rows.pairs + 1);
  const int pieces = rows.V / Vec<L>::N;
  auto statistics = [&](auto team) {
    using T = Team<decltype(team)::value>;
    launch_chained(preference_rows_kernel<L, decltype(team)::value>, rows.R / T::ROWS + 1, T::BLOCK, 0, s, logits, ld, aligned, rows, a, work,
                   logp, sums, loss_sum);
  };
  auto gradient = [&](auto team) {
    using T = Team<decltype(team)::value>;
    launch_chained(preference_grad_kernel<L, decltype(team)::value>, (rows.R + T::ROWS - 1) / T::ROWS, T::BLOCK, 0, s, logits, ld,
                   rows.targets, work, rows.R, rows.V, grad, ldg);
  };
  // A row's team grows while all rows have a place on the GPU in teams of the next size and no thread has less than four pieces then. Calls without
  // the gradient, us, by team of 32 / 128 / 256 / 512: 8,000 rows of 2,500 words 40 / 48 / 73 / 128; 2,000 of 4,096 19.6 / 21.5 / 28;
  // 600 of 8,192 21.5 / 17.4 / 17.4; 1,021 of 50,304 63 / 37 / 43 / 49; 4,096 of 128,256 - / 148 / 150 / 184; 250 of 128,256 - / 45 / 35 / 31 (1,024: 41).
  const int places[3][2] = {{128, 148 * 8}, {256, 148 * 5}, {512, 148 * 3}};
  int team = pieces <= 1024 ? 32 : 128;
  for (const auto& [next, rows_at_once] : places)
    if (next > team && rows.R <= rows_at_once && pieces >= 4 * next) team = next;
  if (team == 32) statistics(std::integral_constant<int, 32>());
  else if (team == 128) statistics(std::integral_constant<int, 128>());
  else if (team == 256) statistics(std::integral_constant<int, 256>());
  else statistics(std::integral_constant<int, 512>());
  if (grad == nullptr || rows.R == 0) return (int)cudaGetLastError();
  // The gradient has nothing to reduce: by length alone. 8,000 rows of 1,000 words 39 / 41 / 45 / 60 / 93; 8,192 of 5,000 72 / 69 / 78 / 100 / 135;
  // 2,000 of 20,000 69 / 60 / 60 / 64 / 80; 4,096 of 128,256 466 / 454 / 442 / 429 / 457.
  if (pieces <= 256) gradient(std::integral_constant<int, 32>());
  else if (pieces <= 1024) gradient(std::integral_constant<int, 128>());
  else if (pieces <= 4096) gradient(std::integral_constant<int, 256>());
  else gradient(std::integral_constant<int, 512>());
  return (int)cudaGetLastError();
}

}  // namespace
}  // namespace ss

extern "C" {
using namespace ss;

// work: 6 R + 6 pairs + 1 words on a boundary of 8 bytes. logp: R words. grad null: the loss alone.
int ss_preference(const void* logits, int fp32_logits, long long ld, const long long* targets, const float* weights,
                  const int* cu_seqlens, int R, int V, int pairs, const float* ref_logp, float beta, int kind, float smoothing,
                  int average, float grad_scale, float* logp, float* sums, float* loss_sum, void* grad, long long ldg, void* work,
                  void* stream) {
  if (R < 0 || R > 0x7fff0000 || V < 1 || pairs < 0 || pairs > 0xfffffff || kind < 0 || kind > 2 || ld < V || (grad != nullptr && ldg < V)) return -2;
  const Rows rows{targets, weights, ref_logp, cu_seqlens, R, V, pairs};
  const PairArgs a{beta, smoothing, grad_scale, kind, average};
  const long long n = R, p = pairs;
  double* d = (double*)work;                     // ratio, slope; then the counters, which are cleared with the slopes; then the rest
  int* c = (int*)(d + n + 2 * p);
  float* w = (float*)(c + p + 1);
  const Work handed{d, d + n, w, w + n, w + 2 * n, w + 4 * n, (int*)(w + 3 * n), c, c + p};
  cudaStream_t s = (cudaStream_t)stream;
  if (fp32_logits) return preference((const float*)logits, ld, rows, a, handed, logp, sums, loss_sum, (float*)grad, ldg, s);
  return preference((const bf16*)logits, ld, rows, a, handed, logp, sums, loss_sum, (bf16*)grad, ldg, s);
}
}  // extern "C"
