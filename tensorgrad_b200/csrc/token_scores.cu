// Scores of tokens under a language model's logits, class axis last (no reference counterpart;
// next to the cross entropy of ops/loss.py:23-97): per row x with m = max x, s = sum e^(x - m)
//   log p_t  = (x_t - m) - log s                     the given token
//   H        = log s - (1 / s) sum e^(x - m) (x - m) the entropy of the whole distribution
//   (log p_i, i) of the k largest x_i, equal ones by ascending i
// and their VJP. The largest entry's own 1 is kept out of the sum: r = s - 1 and log1p(r) hold the
// log probability and the entropy of a nearly certain token to their last digits, where 1 + r
// would have rounded r away. m and r are kept apart for the VJP (p = e^(x - m) / (1 + r)): one
// log-sum-exp would round p to that sum's spacing.
#include <cooperative_groups.h>

#include <limits>

#include "common.cuh"

namespace tg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 128;
constexpr int64_t kMaxClasses = 1 << 30;

// ---------------------------------------------------------------- order of the alternatives
// A value's place in the order as an unsigned key: larger value, larger key; both zeros alike;
// NaN below everything.
template <typename T>
struct OrderKey;
template <>
struct OrderKey<float> {
  using U = uint32_t;
  static __device__ __forceinline__ U of(float x) {
    if (x != x) return 0;
    const U u = __float_as_uint(x + 0.f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
  }
};
template <>
struct OrderKey<double> {
  using U = unsigned long long;
  static __device__ __forceinline__ U of(double x) {
    if (x != x) return 0;
    const U u = (U)__double_as_longlong(x + 0.0);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
  }
};

// One alternative: its key and its class.
template <typename U>
struct Alt {
  U key;
  int id;
};

// a before b: the larger key, then the lower class.
template <typename U>
__device__ __forceinline__ bool before(Alt<U> a, Alt<U> b) {
  return a.key > b.key || (a.key == b.key && a.id < b.id);
}

// ---------------------------------------------------------------- row statistics
// Running maximum m (the type's lowest value before the first), r = sum e^(x - m) - 1 without the
// rounding of that 1 (-1 before the first) and u = sum e^(x - m) (x - m).
template <typename T>
struct Stats {
  T m, r, u;
};

template <typename T>
constexpr T kLowest = std::numeric_limits<T>::lowest();

template <typename T>
__device__ __forceinline__ Stats<T> no_stats() {
  return {kLowest<T>, T(-1), T(0)};
}

// Exponentials are dev_exp's, a step off or two, except in a lane's own sums (push): there the
// argument is in base 2, off by (4 + 2.4 |x|) half steps. Its x is below that lane's own maximum,
// whose term is an exact 1, so of n values a lane's sum is off by about 4 + 3.4 log n half steps at
// most; whatever lies far below the row's maximum is moved there by one exact exponential a lane.
// 8192 x 50304 forward and backward: 801 us, with dev_exp there too 814; with base 2 everywhere 796,
// and a class 80 below the maximum off by 61 half steps.
__device__ __forceinline__ float lane_exp(float x) { return __expf(x); }
__device__ __forceinline__ double lane_exp(double x) { return exp(x); }
__device__ __forceinline__ float log_1p(float x) { return log1pf(x); }
__device__ __forceinline__ double log_1p(double x) { return log1p(x); }

// The statistics of two sets of values as one: the lower maximum's set is scaled by
// c = e^(its m - the other m), every x - m of it moves by the difference d. A set so low that c is
// 0 (classes closed by the type's lowest value, say) adds nothing: its sum is scaled before d
// multiplies it, as sum times d may overflow, and d itself is kept finite.
template <typename T>
__device__ __forceinline__ Stats<T> join(Stats<T> a, Stats<T> b) {
  if (b.m > a.m) {
    const Stats<T> t = a;
    a = b;
    b = t;
  }
  const T s = T(1) + b.r;
  if (s == T(0)) return a;  // nothing in it
  const T d = fmax(b.m - a.m, kLowest<T>), c = dev_exp(d), moved = s * c;
  return {a.m, a.r + moved, a.u + (c * b.u + moved * d)};
}

// What one lane has read: its maximum m, s = sum e^(x - m) and u = sum e^(x - m) (x - m).
template <typename T>
struct Seen {
  T m, s, u;
};

// N more values at a time: the maximum moves at most once, each value costs one exponential. A
// value of -inf adds nothing (0 times the lowest value); NaN and +inf make s NaN.
template <int N, typename T>
__device__ __forceinline__ void push(Seen<T>& a, const T (&x)[N]) {
  T top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmax(top, x[i]);
  if (top > a.m) {
    const T d = fmax(a.m - top, kLowest<T>), c = dev_exp(d);
    a.s *= c;
    a.u = c * a.u + a.s * d;  // finite as in join
    a.m = top;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const T z = x[i] - a.m, e = lane_exp(z);
    a.s += e;
    a.u += e * fmax(z, kLowest<T>);
  }
}

// Statistics over every group of LANES lanes.
template <int LANES, typename T>
__device__ __forceinline__ Stats<T> lanes_join(Stats<T> a) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1)
    a = join(a, Stats<T>{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.r, o),
                         __shfl_xor_sync(0xffffffffu, a.u, o)});
  return a;
}

template <typename T, int VE>
struct alignas(sizeof(T) * VE) Vec {
  T v[VE];
};

// ---------------------------------------------------------------- the alternatives
constexpr int kList = 1024;  // entries that are ranked against each other

template <typename T>
struct Shared {
  using U = typename OrderKey<T>::U;
  Stats<T> stats[kThreads / 32];
  T tops_of[kThreads / 32];  // the warps' maxima
  T rest[kThreads / 32];     // their shares of what the maximum's lane has read: the terms
  T rest_u[kThreads / 32];   // beside the maximum's own, and those times x - m
  int equal[kThreads / 32];
  int holder;               // the first lane that has the maximum
  Stats<T> mine;            // the block's, for the cluster
  Alt<U> list[kList];       // candidates
  Alt<U> best[kMaxTop];     // the block's alternatives in order
  alignas(16) U tops[kThreads];  // every lane's largest value
  int lanes[kThreads];      // those that reach the bound
  U bound;                  // no entry below it is an alternative
  int count, lane_count;
};

// The alternatives of values [0, n) one by one: each round takes the first one after the last
// found. Always right and slow: for rows that have too many equal entries to list.
template <typename T>
__device__ void select_rounds(const T* __restrict__ x, int n, int first, int top_k,
                              Shared<T>& sh) {
  using U = typename OrderKey<T>::U;
  Alt<U> last{std::numeric_limits<U>::max(), -1};
  for (int k = 0; k < top_k; ++k) {
    Alt<U> mine{0, std::numeric_limits<int>::max()};
    for (int c = threadIdx.x; c < n; c += kThreads) {
      const Alt<U> a{OrderKey<T>::of(x[c]), first + c};
      if (before(last, a) && before(a, mine)) mine = a;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Alt<U> other{__shfl_xor_sync(0xffffffffu, mine.key, o),
                         __shfl_xor_sync(0xffffffffu, mine.id, o)};
      if (before(other, mine)) mine = other;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh.list[threadIdx.x >> 5] = mine;
    __syncthreads();
    last = sh.list[0];
    for (int i = 1; i < kThreads / 32; ++i)
      if (before(sh.list[i], last)) last = sh.list[i];
    if (threadIdx.x == 0) sh.best[k] = last;
  }
  __syncthreads();
}

// The first top_k of n listed entries in order: an entry's place is how many come before it.
template <typename T, typename F>
__device__ __forceinline__ void rank_list(int n, int top_k, const Shared<T>& sh, F place) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const auto a = sh.list[i];
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += before(sh.list[j], a);
    if (rank < top_k) place(rank, a);
  }
}

// The block's alternatives into sh.best, from every lane's largest value. The top_k-th largest of
// those bounds the top_k-th largest value from below, and only lanes that reach it have entries
// to look at again: about top_k of the row's kThreads-th parts are read twice.
template <typename T, int VE>
__device__ void select_top(const T* __restrict__ x, int n, int first, int top_k, T lane_top,
                           Shared<T>& sh) {
  using U = typename OrderKey<T>::U;
  constexpr U most = std::numeric_limits<U>::max();
  const U key = OrderKey<T>::of(lane_top), none = OrderKey<T>::of(kLowest<T>);
  sh.tops[threadIdx.x] = key;
  if (threadIdx.x == 0) {
    sh.count = sh.lane_count = 0;
    sh.bound = most;
  }
  __syncthreads();
  // The top_k-th largest: the smallest that fewer than top_k others exceed.
  int larger = 0;
  const Vec<U, 16 / sizeof(U)>* tops = reinterpret_cast<const Vec<U, 16 / sizeof(U)>*>(sh.tops);
#pragma unroll 8
  for (int i = 0; i < kThreads * (int)sizeof(U) / 16; ++i) {
    const auto others = tops[i];
#pragma unroll
    for (int e = 0; e < 16 / (int)sizeof(U); ++e) larger += others.v[e] > key;
  }
  if (larger < top_k) atomicMin(&sh.bound, key);
  __syncthreads();
  U bound = sh.bound;
  if (bound <= none) {
    // Fewer lanes than alternatives have a value: list everything, or go the slow way.
    if (n > kList) {
      select_rounds(x, n, first, top_k, sh);
      return;
    }
    bound = 0;
  }
  if (key >= bound) sh.lanes[atomicAdd(&sh.lane_count, 1)] = threadIdx.x;
  __syncthreads();
  const int units = n / VE, each = (units + kThreads - 1) / kThreads, lanes = sh.lane_count;
  for (int i = threadIdx.x; i < lanes * each; i += kThreads) {
    const int c = sh.lanes[i / each] + i % each * kThreads;
    if (c >= units) continue;
    const Vec<T, VE> v = reinterpret_cast<const Vec<T, VE>*>(x)[c];
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const U k = OrderKey<T>::of(v.v[e]);
      if (k < bound) continue;
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = {k, first + c * VE + e};
    }
  }
  __syncthreads();
  const int found = sh.count;
  if (found > kList) {
    select_rounds(x, n, first, top_k, sh);
    return;
  }
  rank_list(found, top_k, sh, [&](int rank, Alt<U> a) { sh.best[rank] = a; });
  __syncthreads();
}

// The block's statistics from its lanes'. A lane's s holds its maximum's own 1, which rounds what
// is small beside it away; that matters in the lane that holds the block's maximum alone, so the
// block reads that lane's values (a kThreads-th of the row) once more and sums them without it,
// with full exponentials: beside the maximum they may all be far below it.
template <typename T, int VE>
__device__ Stats<T> block_stats(Seen<T> a, const Vec<T, VE>* __restrict__ xv, int units,
                                Shared<T>& sh) {
  static_assert(kThreads / 32 == 8, "one lane of a group of eight to a warp");
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const T top = warp_max(a.m);
  if (lane == 0) sh.tops_of[w] = top;
  if (threadIdx.x == 0) sh.holder = kThreads;
  __syncthreads();
  T m = sh.tops_of[lane & 7];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (a.m == m && a.s != T(0)) atomicMin(&sh.holder, (int)threadIdx.x);
  __syncthreads();
  const int holder = sh.holder;
  T rest = T(0), rest_u = T(0);
  int equal = 0;  // entries equal to the maximum, one of them the maximum itself
  if (holder < kThreads) {
    for (int c = holder + threadIdx.x * kThreads; c < units; c += kThreads * kThreads) {
      const Vec<T, VE> y = xv[c];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const T z = y.v[e] - m, t = y.v[e] == m ? T(0) : dev_exp(z);
        equal += y.v[e] == m;
        rest += t;
        rest_u += t * fmax(z, kLowest<T>);
      }
    }
  }
  equal = __reduce_add_sync(0xffffffffu, equal);
  rest = warp_sum(rest);
  rest_u = warp_sum(rest_u);
  Stats<T> mine{a.m, a.s == T(0) ? T(-1) : a.s - T(1), a.u};
  if ((int)threadIdx.x == holder && a.s == a.s) mine.r = mine.u = T(0);
  mine = lanes_join<32>(mine);
  if (lane == 0) {
    sh.stats[w] = mine;
    sh.rest[w] = rest;
    sh.rest_u[w] = rest_u;
    sh.equal[w] = equal;
  }
  __syncthreads();
  mine = lanes_join<8>(sh.stats[lane & 7]);
  rest = sh.rest[lane & 7];
  rest_u = sh.rest_u[lane & 7];
  equal = sh.equal[lane & 7];
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    rest += __shfl_xor_sync(0xffffffffu, rest, o);
    rest_u += __shfl_xor_sync(0xffffffffu, rest_u, o);
    equal += __shfl_xor_sync(0xffffffffu, equal, o);
  }
  if (holder < kThreads) {
    mine.r += rest + (T)(equal - 1);
    mine.u += rest_u;
  }
  return mine;
}

template <typename T>
struct ScoreArgs {
  const T* logits;
  const int64_t* targets;
  T* stats;
  T* log_probs;
  T* entropy;
  T* top;
  int64_t* ids;
  int classes, top_k, splits, part;  // part: classes of a split, a multiple of VE
  int64_t ignore_index;
  int* bad_target;
};

// The target's log probability; 0 without one.
template <typename T>
__device__ __forceinline__ T target_log_prob(const ScoreArgs<T>& a, int64_t r, const T* row, T m,
                                             T ls) {
  const int64_t t = a.targets[r];
  if (t == a.ignore_index) return T(0);
  if (t < 0 || t >= a.classes) {
    if (a.bad_target) *a.bad_target = 1;
    return T(0);
  }
  return (row[t] - m) - ls;
}

// A row's part of the VJP: dx_j = direct_j - p_j (total + g_ent (log p_j + H)), with direct_j what
// comes in at class j alone (g_log at the target, g_top at the alternatives) and total their sum.
// Built by whole warps.
template <typename T>
struct Pull {
  T m, r, inv, total, shift, slope, log;  // shift = H - log s, slope = g_ent, log = g_log
  int64_t target;                         // -1 without one
  __device__ Pull(int64_t row, int classes, const int64_t* targets, const T* stats,
                  const T* entropy, const T* g_log, const T* g_ent, const T* g_top, int top_k,
                  int64_t ignore_index) {
    m = stats[2 * row];
    r = stats[2 * row + 1];
    inv = T(1) / (T(1) + r);
    target = targets[row];
    if (target == ignore_index || target < 0 || target >= classes) target = -1;
    log = target >= 0 && g_log ? g_log[row] : T(0);
    slope = g_ent ? g_ent[row] : T(0);
    shift = g_ent ? entropy[row] - log_1p(r) : T(0);
    T tops = T(0);
    for (int k = threadIdx.x & 31; k < top_k; k += 32) tops += g_top[row * top_k + k];
    if (top_k > 0) tops = warp_sum(tops);
    total = log + tops;
  }
  // A class at which nothing comes in alone.
  __device__ __forceinline__ T spread(T x) const {
    const T z = x - m, p = dev_exp(z) * inv;
    // Nothing is left where log p may be -inf.
    return p == T(0) ? T(0) : -p * (total + slope * (z + shift));
  }
  // One at which `direct` does: direct (1 - p) - p (the rest), with 1 - p = r / (1 + r) at the
  // maximum, so that a nearly certain token's gradient keeps its digits.
  __device__ __forceinline__ T single(T x, T direct) const {
    const T z = x - m, p = dev_exp(z) * inv, q = z == T(0) ? r * inv : T(1) - p;
    return direct * q - (p == T(0) ? T(0) : p * ((total - direct) + slope * (z + shift)));
  }
};

// One block a row, or a cluster of `splits` blocks with a part of its classes each. HBM-bound: one
// read of the logits, VE of them to a load; 8 instructions and one exponential a value.
template <typename T, int VE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 5 : 4)
scores_fwd_kernel(ScoreArgs<T> a) {
  using U = typename OrderKey<T>::U;
  constexpr int N = 4;  // loads in a step
  __shared__ Shared<T> sh;
  pdl_trigger();
  pdl_wait();
  const int split = blockIdx.x % a.splits;
  const int64_t r = blockIdx.x / a.splits;
  const int first = split * a.part;
  const int n = a.classes - first < a.part ? a.classes - first : a.part;
  const T* row = a.logits + r * a.classes;
  const T* x = row + first;
  Seen<T> seen{kLowest<T>, T(0), T(0)};
  const int units = n / VE;  // parts are multiples of VE
  const Vec<T, VE>* xv = reinterpret_cast<const Vec<T, VE>*>(x);
  int c = threadIdx.x;
#pragma unroll 1
  for (; c + (N - 1) * kThreads < units; c += N * kThreads) {
    T v[N * VE];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Vec<T, VE> y = xv[c + i * kThreads];
#pragma unroll
      for (int e = 0; e < VE; ++e) v[i * VE + e] = y.v[e];
    }
    push(seen, v);
  }
  for (; c < units; c += kThreads) {
    const Vec<T, VE> y = xv[c];
    push(seen, y.v);
  }
  Stats<T> mine = block_stats<T, VE>(seen, xv, units, sh);
  if (a.top_k > 0) select_top<T, VE>(x, n, first, a.top_k, seen.m, sh);
  if (a.splits > 1) {
    const auto cluster = cooperative_groups::this_cluster();
    if (threadIdx.x == 0) sh.mine = mine;
    cluster.sync();
    const int other = threadIdx.x & 7;
    mine = lanes_join<8>(other < a.splits ? *cluster.map_shared_rank(&sh.mine, other)
                                          : no_stats<T>());
    if (split == 0) {
      for (int i = threadIdx.x; i < a.splits * a.top_k; i += kThreads)
        sh.list[i] = cluster.map_shared_rank(sh.best, i / a.top_k)[i % a.top_k];
    }
    cluster.sync();  // the others' results have been read
  }
  if (split != 0) return;
  const T ls = log_1p(mine.r);
  const T m = mine.r != T(-1) ? mine.m : T(-INFINITY);  // a closed row has no log probabilities
  auto place = [&](int rank, Alt<U> e) {
    a.top[r * a.top_k + rank] = (row[e.id] - m) - ls;
    a.ids[r * a.top_k + rank] = e.id;
  };
  if (a.splits > 1) {
    rank_list(a.splits * a.top_k, a.top_k, sh, place);
  } else {
    for (int k = threadIdx.x; k < a.top_k; k += kThreads) place(k, sh.best[k]);
  }
  if (threadIdx.x == 0) {
    a.stats[2 * r] = m;
    a.stats[2 * r + 1] = mine.r;
    a.entropy[r] = ls - mine.u / (T(1) + mine.r);
    a.log_probs[r] = target_log_prob(a, r, row, m, ls);
  }
}

// Block (row, part of the classes); one read of the logits, one write.
template <typename T, int VE>
__global__ void __launch_bounds__(kThreads)
scores_bwd_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets,
                  const T* __restrict__ stats, const T* __restrict__ entropy,
                  const int64_t* __restrict__ ids, const T* __restrict__ g_log,
                  const T* __restrict__ g_ent, const T* __restrict__ g_top, T* __restrict__ grad,
                  int classes, int part, int top_k, int64_t ignore_index) {
  pdl_trigger();
  pdl_wait();
  const int first = blockIdx.y * part;
  const int n = classes - first < part ? classes - first : part;
  const int64_t r = blockIdx.x;
  const Pull<T> p(r, classes, targets, stats, entropy, g_log, g_ent, g_top, top_k, ignore_index);
  T* d = grad + r * classes + first;
  const int units = n / VE;
  const Vec<T, VE>* xv = reinterpret_cast<const Vec<T, VE>*>(logits + r * classes + first);
  Vec<T, VE>* dv = reinterpret_cast<Vec<T, VE>*>(d);
#pragma unroll 4
  for (int c = threadIdx.x; c < units; c += kThreads) {
    Vec<T, VE> v = xv[c];
#pragma unroll
    for (int e = 0; e < VE; ++e) v.v[e] = p.spread(v.v[e]);
    dv[c] = v;
  }
  // The single classes again, by one lane each: the alternatives are distinct, the target may be
  // one of them.
  const T* x = logits + r * classes + first;
  bool hit = false;
  const int64_t at = p.target >= 0 ? p.target - first : -1;
  __syncthreads();
  for (int k = threadIdx.x; k < top_k; k += kThreads) {
    const int64_t i = ids[r * top_k + k] - first;
    if (i < 0 || i >= n) continue;
    hit |= i == at;
    d[i] = p.single(x[i], g_top[r * top_k + k] + (i == at ? p.log : T(0)));
  }
  hit = __syncthreads_or(hit);
  if (threadIdx.x == 0 && !hit && at >= 0 && at < n) d[at] = p.single(x[at], p.log);
}

// Rows of up to kWarpRow classes: a warp a row, its values in registers (NV of them to a lane). A
// block a row leaves most of its lanes idle there (8192 rows of 65 classes forward and backward:
// 42.5 us, with a warp a row 8.1). Alternatives by bisecting their keys cost the same for any
// number of them (8192 x 1000: 5 of them 59 us, 100 of them 90; one by one about 54 and 600).
constexpr int kWarpRow = 1024;

template <typename T, int NV>
__global__ void __launch_bounds__(kThreads)
scores_fwd_warp_kernel(ScoreArgs<T> a, int64_t rows) {
  using U = typename OrderKey<T>::U;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= rows) return;
  const T* row = a.logits + r * a.classes;
  T v[NV], m = kLowest<T>, rest = T(0), u = T(0);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = lane + 32 * i;
    v[i] = c < a.classes ? row[c] : T(-INFINITY);
    m = fmax(m, v[i]);
  }
  m = warp_max(m);
  bool has = false;
#pragma unroll
  for (int i = 0; i < NV; ++i) has |= v[i] == m;
  const unsigned holders = __ballot_sync(0xffffffffu, has);
  bool out = lane == __ffs(holders) - 1;  // this lane leaves the maximum's own 1 out, once
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const T z = v[i] - m, e = out && v[i] == m ? T(0) : dev_exp(z);
    out = out && v[i] != m;
    rest += e;
    u += e * fmax(z, kLowest<T>);
  }
  rest = holders == 0 ? T(-1) : warp_sum(rest);
  if (m == T(INFINITY)) rest = T(NAN);
  u = warp_sum(u);
  const T ls = log_1p(rest);
  if (rest == T(-1)) m = T(-INFINITY);  // a closed row has no log probabilities
  if (a.top_k > 0) {
    // The top_k-th key, bit by bit: the largest that at least top_k entries reach. Entries above
    // it and the first ones equal to it are the alternatives; their order is by rank.
    U key[NV], kth = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) key[i] = OrderKey<T>::of(v[i]);
    for (int bit = 8 * (int)sizeof(U) - 1; bit >= 0; --bit) {
      const U next = kth | (U)1 << bit;
      int reach = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i) reach += lane + 32 * i < a.classes && key[i] >= next;
      if (__reduce_add_sync(0xffffffffu, reach) >= a.top_k) kth = next;
    }
    __shared__ Alt<U> lists[kThreads / 32][kMaxTop];
    Alt<U>* list = lists[threadIdx.x >> 5];
    int above = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) above += lane + 32 * i < a.classes && key[i] > kth;
    int ties = __reduce_add_sync(0xffffffffu, above);
    above = 0;
    const unsigned before_me = (1u << lane) - 1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const bool in = lane + 32 * i < a.classes;
      const unsigned more = __ballot_sync(0xffffffffu, in && key[i] > kth);
      const unsigned same = __ballot_sync(0xffffffffu, in && key[i] == kth);
      if (more >> lane & 1) list[above + __popc(more & before_me)] = {key[i], lane + 32 * i};
      const int at = ties + __popc(same & before_me);
      if ((same >> lane & 1) && at < a.top_k) list[at] = {key[i], lane + 32 * i};
      above += __popc(more);
      ties += __popc(same);
    }
    __syncwarp();
    for (int k = lane; k < a.top_k; k += 32) {
      const Alt<U> mine = list[k];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < a.top_k; ++j) rank += before(list[j], mine);
      a.top[r * a.top_k + rank] = (row[mine.id] - m) - ls;
      a.ids[r * a.top_k + rank] = mine.id;
    }
  }
  if (lane == 0) {
    a.stats[2 * r] = m;
    a.stats[2 * r + 1] = rest;
    a.entropy[r] = ls - u / (T(1) + rest);
    a.log_probs[r] = target_log_prob(a, r, row, m, ls);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
scores_bwd_warp_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets,
                       const T* __restrict__ stats, const T* __restrict__ entropy,
                       const int64_t* __restrict__ ids, const T* __restrict__ g_log,
                       const T* __restrict__ g_ent, const T* __restrict__ g_top,
                       T* __restrict__ grad, int64_t rows, int classes, int top_k,
                       int64_t ignore_index) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (r >= rows) return;
  const Pull<T> p(r, classes, targets, stats, entropy, g_log, g_ent, g_top, top_k, ignore_index);
  const T* x = logits + r * classes;
  T* d = grad + r * classes;
#pragma unroll 8
  for (int c = lane; c < classes; c += 32)
    d[c] = c == p.target ? p.single(x[c], p.log) : p.spread(x[c]);
  __syncwarp();
  for (int k = lane; k < top_k; k += 32) {
    const int64_t i = ids[r * top_k + k];
    d[i] = p.single(x[i], g_top[r * top_k + k] + (i == p.target ? p.log : T(0)));
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int sm_count() {
  static int n = 0;
  if (!n) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
  }
  return n;
}

// Parts of a row where the rows alone leave multiprocessors empty: up to 8 (a cluster), none
// shorter than about 2048 classes, so that a part has more classes than alternatives are asked for.
int row_splits(int64_t rows, int64_t classes) {
  int s = 1;
  while (s < 8 && rows * s < 2 * sm_count() && classes >= 2 * s * 2048) s *= 2;
  return s;
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" {

int tg_token_log_probs_max_top(void) { return kMaxTop; }

int tg_token_log_probs_forward(int dtype, const void* logits, const int64_t* targets, void* stats,
                               void* log_probs, void* entropy, void* top_log_probs,
                               int64_t* top_ids, int64_t rows, int64_t classes, int64_t top_k,
                               int64_t ignore_index, int* bad_target_dev, void* stream) {
  TG_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && classes > 0 && classes <= kMaxClasses,
               "token_log_probs: bad shape");
  TG_CHECK_ARG(top_k >= 0 && top_k <= kMaxTop && top_k <= classes,
               "token_log_probs: top_k %lld (at most %d and the %lld classes)", (long long)top_k,
               kMaxTop, (long long)classes);
  TG_CHECK_ARG(top_k == 0 || (top_log_probs && top_ids), "token_log_probs: no room for top_k");
  if (rows == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    constexpr int VE = 16 / sizeof(T);
    ScoreArgs<T> a{(const T*)logits, targets, (T*)stats, (T*)log_probs, (T*)entropy,
                   (T*)top_log_probs, top_ids, (int)classes, (int)top_k, 1, (int)classes,
                   ignore_index, bad_target_dev};
    if (classes <= kWarpRow) {
      const dim3 grid((unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32)));
      TG_CUDA_TRY(launch_pdl(classes <= 128 ? scores_fwd_warp_kernel<T, 4>
                                            : scores_fwd_warp_kernel<T, kWarpRow / 32>,
                             grid, dim3(kThreads), 0, s, a, rows));
      return check_launch("token_log_probs");
    }
    a.splits = row_splits(rows, classes);
    if (a.splits > 1) a.part = (int)((classes + a.splits * VE - 1) / (a.splits * VE) * VE);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * a.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned)a.splits, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 2;
    const bool vec = classes % VE == 0 && aligned16(logits);
    TG_CUDA_TRY(vec ? cudaLaunchKernelEx(&cfg, scores_fwd_kernel<T, VE>, a)
                    : cudaLaunchKernelEx(&cfg, scores_fwd_kernel<T, 1>, a));
    return check_launch("token_log_probs");
  });
}

int tg_token_log_probs_backward(int dtype, const void* logits, const int64_t* targets,
                                const void* stats, const void* entropy, const int64_t* top_ids,
                                const void* g_log, const void* g_ent, const void* g_top,
                                void* grad, int64_t rows, int64_t classes, int64_t top_k,
                                int64_t ignore_index, void* stream) {
  TG_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && classes > 0 && classes <= kMaxClasses &&
                   top_k >= 0 && top_k <= kMaxTop, "token_log_probs backward: bad shape");
  if (rows == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    constexpr int VE = 16 / sizeof(T);
    if (!g_top) top_k = 0;  // no gradient comes in through the alternatives
    if (classes <= kWarpRow) {
      const dim3 grid((unsigned)((rows + kThreads / 32 - 1) / (kThreads / 32)));
      TG_CUDA_TRY(launch_pdl(scores_bwd_warp_kernel<T>, grid, dim3(kThreads), 0, s,
                             (const T*)logits, targets, (const T*)stats, (const T*)entropy,
                             top_ids, (const T*)g_log, (const T*)g_ent, (const T*)g_top, (T*)grad,
                             rows, (int)classes, (int)top_k, ignore_index));
      return check_launch("token_log_probs backward");
    }
    const int parts = row_splits(rows, classes);
    const int part = (int)((classes + parts * VE - 1) / (parts * VE) * VE);
    const dim3 grid((unsigned)rows, (unsigned)parts);
    const bool vec = classes % VE == 0 && aligned16(logits) && aligned16(grad);
    TG_CUDA_TRY(launch_pdl(vec ? scores_bwd_kernel<T, VE> : scores_bwd_kernel<T, 1>, grid,
                           dim3(kThreads), 0, s, (const T*)logits, targets, (const T*)stats,
                           (const T*)entropy, top_ids, (const T*)g_log, (const T*)g_ent,
                           (const T*)g_top, (T*)grad, (int)classes, part, (int)top_k,
                           ignore_index));
    return check_launch("token_log_probs backward");
  });
}

}  // extern "C"
