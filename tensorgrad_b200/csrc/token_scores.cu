// Scores of tokens under a language model's logits, class axis last (no reference counterpart;
// next to the cross entropy of ops/loss.py:23-97): per row x with m = max x, s = sum e^(x - m)
//   log p_t  = (x_t - m) - log s                     the given token
//   H        = log s - (1 / s) sum e^(x - m) (x - m) the entropy of the whole distribution
//   (log p_i, i) of the k largest x_i, equal ones by ascending i
// and their VJP. Row statistics m and s are kept apart for the VJP (p = e^(x - m) / s): folding
// them into one log-sum-exp would round p to that sum's spacing.
#include <limits>

#include "common.cuh"

namespace tg {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 128;

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
// Running maximum m, s = sum e^(x - m) and u = sum e^(x - m) (x - m).
template <typename T>
struct Stats {
  T m, s, u;
};

// The statistics of two sets of values as one. Shifting a maximum from m to m' >= m scales
// every e^(x - m) by c = e^(m - m') and moves every x - m by m - m'.
template <typename T>
__device__ __forceinline__ Stats<T> join(Stats<T> a, Stats<T> b) {
  const T m = fmax(a.m, b.m);
  if (m == T(-INFINITY)) return {m, a.s + b.s, a.u + b.u};
  Stats<T> r{m, T(0), T(0)};
  const T da = a.m - m, db = b.m - m;
  if (a.s != T(0)) {
    const T c = dev_exp<T>(da);
    r.s += a.s * c;
    r.u += c * (a.u + (da == T(-INFINITY) ? T(0) : a.s * da));
  }
  if (b.s != T(0)) {
    const T c = dev_exp<T>(db);
    r.s += b.s * c;
    r.u += c * (b.u + (db == T(-INFINITY) ? T(0) : b.s * db));
  }
  return r;
}

// One more value. A value of -inf adds nothing; NaN and +inf make s and u NaN.
template <typename T>
__device__ __forceinline__ void push(Stats<T>& a, T x) {
  if (x == T(-INFINITY)) return;
  a = join(a, Stats<T>{x, x - x + T(1), x - x});
}

template <typename T>
__device__ __forceinline__ Stats<T> block_join(Stats<T> a, Stats<T>* sh) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    a = join(a, Stats<T>{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                         __shfl_xor_sync(0xffffffffu, a.u, o)});
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  Stats<T> r = sh[0];
  for (int i = 1; i < kThreads / 32; ++i) r = join(r, sh[i]);
  __syncthreads();
  return r;
}

// The alternatives of a row one by one: each round takes the first one after the last found.
template <typename T>
__device__ void select_rounds(const T* __restrict__ x, int64_t classes, int top_k, T m, T ls,
                              T* __restrict__ top, int64_t* __restrict__ ids) {
  using U = typename OrderKey<T>::U;
  __shared__ Alt<U> best[kThreads / 32];
  Alt<U> last{std::numeric_limits<U>::max(), -1};
  for (int k = 0; k < top_k; ++k) {
    Alt<U> mine{0, std::numeric_limits<int>::max()};
    for (int64_t c = threadIdx.x; c < classes; c += kThreads) {
      const Alt<U> a{OrderKey<T>::of(x[c]), (int)c};
      if (before(last, a) && before(a, mine)) mine = a;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Alt<U> other{__shfl_xor_sync(0xffffffffu, mine.key, o),
                         __shfl_xor_sync(0xffffffffu, mine.id, o)};
      if (before(other, mine)) mine = other;
    }
    if ((threadIdx.x & 31) == 0) best[threadIdx.x >> 5] = mine;
    __syncthreads();
    last = best[0];
    for (int i = 1; i < kThreads / 32; ++i)
      if (before(best[i], last)) last = best[i];
    __syncthreads();
    if (threadIdx.x == 0) {
      top[k] = (x[last.id] - m) - ls;
      ids[k] = last.id;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
scores_fwd_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets,
                  T* __restrict__ stats, T* __restrict__ log_probs, T* __restrict__ entropy,
                  T* __restrict__ top, int64_t* __restrict__ ids, int64_t rows, int64_t classes,
                  int top_k, int64_t ignore_index, int* __restrict__ bad_target) {
  __shared__ Stats<T> sh[kThreads / 32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* x = logits + r * classes;
    Stats<T> a{T(-INFINITY), T(0), T(0)};
    for (int64_t c = threadIdx.x; c < classes; c += kThreads) push(a, x[c]);
    a = block_join(a, sh);
    const T ls = dev_log<T>(a.s);
    if (threadIdx.x == 0) {
      stats[2 * r] = a.m;
      stats[2 * r + 1] = a.s;
      entropy[r] = ls - a.u / a.s;
      const int64_t t = targets[r];
      T lp = T(0);
      if (t != ignore_index) {
        if (t < 0 || t >= classes) {
          if (bad_target) *bad_target = 1;
        } else {
          lp = (x[t] - a.m) - ls;
        }
      }
      log_probs[r] = lp;
    }
    if (top_k > 0)
      select_rounds<T>(x, classes, top_k, a.m, ls, top + r * top_k, ids + r * top_k);
  }
}

// dx_j = -p_j (g_log + sum g_top + g_ent (log p_j + H)), then g_log at the target and g_top at
// the alternatives.
template <typename T>
__global__ void __launch_bounds__(kThreads)
scores_bwd_kernel(const T* __restrict__ logits, const int64_t* __restrict__ targets,
                  const T* __restrict__ stats, const T* __restrict__ entropy,
                  const int64_t* __restrict__ ids, const T* __restrict__ g_log,
                  const T* __restrict__ g_ent, const T* __restrict__ g_top, T* __restrict__ grad,
                  int64_t rows, int64_t classes, int top_k, int64_t ignore_index) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* x = logits + r * classes;
    T* d = grad + r * classes;
    const T m = stats[2 * r], s = stats[2 * r + 1];
    const T inv = T(1) / s, ls = dev_log<T>(s);
    const int64_t t = targets[r];
    const bool given = t != ignore_index && t >= 0 && t < classes;
    const T gl = given ? g_log[r] : T(0), ge = g_ent[r], shift = entropy[r] - ls;
    T push_all = gl;
    for (int k = 0; k < top_k; ++k) push_all += g_top[r * top_k + k];
    for (int64_t c = threadIdx.x; c < classes; c += kThreads) {
      const T z = x[c] - m, p = dev_exp<T>(z) * inv;
      // p = 0 leaves nothing, also where log p is -inf.
      d[c] = p == T(0) ? T(0) : -p * (push_all + ge * (z + shift));
    }
    __syncthreads();
    if (threadIdx.x == 0 && given) d[t] += gl;
    __syncthreads();
    for (int k = threadIdx.x; k < top_k; k += kThreads) d[ids[r * top_k + k]] += g_top[r * top_k + k];
  }
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" {

int tg_token_log_probs_max_top(void) { return kMaxTop; }

size_t tg_token_log_probs_scratch_bytes(int dtype, int64_t rows, int64_t classes, int64_t top_k) {
  return 16;
}

int tg_token_log_probs_forward(int dtype, const void* logits, const int64_t* targets, void* stats,
                               void* log_probs, void* entropy, void* top_log_probs,
                               int64_t* top_ids, int64_t rows, int64_t classes, int64_t top_k,
                               int64_t ignore_index, int* bad_target_dev, void* scratch,
                               void* stream) {
  (void)scratch;
  TG_CHECK_ARG(rows >= 0 && classes > 0 && classes <= INT32_MAX, "token_log_probs: bad shape");
  TG_CHECK_ARG(top_k >= 0 && top_k <= kMaxTop && top_k <= classes,
               "token_log_probs: top_k %lld (at most %d and the %lld classes)", (long long)top_k,
               kMaxTop, (long long)classes);
  TG_CHECK_ARG(top_k == 0 || (top_log_probs && top_ids), "token_log_probs: no room for top_k");
  if (rows == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    const unsigned grid = (unsigned)(rows < 148 * 16 ? rows : 148 * 16);
    scores_fwd_kernel<T><<<grid, kThreads, 0, s>>>(
        (const T*)logits, targets, (T*)stats, (T*)log_probs, (T*)entropy, (T*)top_log_probs,
        top_ids, rows, classes, (int)top_k, ignore_index, bad_target_dev);
    return check_launch("token_log_probs");
  });
}

int tg_token_log_probs_backward(int dtype, const void* logits, const int64_t* targets,
                                const void* stats, const void* entropy, const int64_t* top_ids,
                                const void* g_log, const void* g_ent, const void* g_top,
                                void* grad, int64_t rows, int64_t classes, int64_t top_k,
                                int64_t ignore_index, void* stream) {
  TG_CHECK_ARG(rows >= 0 && classes > 0 && classes <= INT32_MAX && top_k >= 0 && top_k <= kMaxTop,
               "token_log_probs backward: bad shape");
  if (rows == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    const unsigned grid = (unsigned)(rows < 148 * 16 ? rows : 148 * 16);
    scores_bwd_kernel<T><<<grid, kThreads, 0, s>>>(
        (const T*)logits, targets, (const T*)stats, (const T*)entropy, top_ids, (const T*)g_log,
        (const T*)g_ent, (const T*)g_top, (T*)grad, rows, classes, (int)top_k, ignore_index);
    return check_launch("token_log_probs backward");
  });
}

}  // extern "C"
