// A key-value cache in pages and the attention of one new token over it (no reference
// counterpart; the paged form of the cache that nn/attention.py:27-111 of the reference keeps
// contiguous). A pool holds pages of `page_size` positions, (num_pages, kv_heads, page_size,
// head_dim) for the keys and as much for the values; a sequence's positions lie on the pages
// that its row of the page table names, in order.
//
// Page ids and lengths live on the device and are checked where they are read: an id outside
// [0, num_pages) reads page 0 or writes nothing, a length beyond the table counts as the
// table's end, and either sets *bad, which the host reads at its next synchronisation.
#include <cooperative_groups.h>

#include <limits>
#include <type_traits>

#include "common.cuh"

namespace tg {
namespace {

constexpr int kThreads = 256;

// n / d for 0 <= n < 2^31 by a multiplication (d fixed for a launch; Granlund and Montgomery,
// "Division by invariant integers using multiplication", 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};
FastDiv make_div(int64_t d) {
  uint32_t l = 0;
  while (((int64_t)1 << l) < d) ++l;
  return {(uint32_t)d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << l) - d)) / d + 1), l};
}
__device__ __forceinline__ int div_by(int n, FastDiv f) {
  return (int)((__umulhi((uint32_t)n, f.mul) + (uint32_t)n) >> f.shift);
}

struct Pool {
  int64_t num_pages, kv_heads, page_size, head_dim;  // head_dim in units of what is moved
  const int64_t* table;                              // (batch, max_pages)
  int64_t max_pages;
  int* bad;
};

// The position's row of one head in a pool, or -1 behind a bad id or off the table.
__device__ __forceinline__ int64_t row_of(const Pool& p, FastDiv size, int64_t b, int h,
                                          int64_t at) {
  if (at < 0 || at >= p.max_pages * p.page_size) {
    if (p.bad) *p.bad = 1;
    return -1;
  }
  const int slot = div_by((int)at, size);
  const int64_t page = p.table[b * p.max_pages + slot];
  if (page < 0 || page >= p.num_pages) {
    if (p.bad) *p.bad = 1;
    return -1;
  }
  return ((page * p.kv_heads + h) * p.page_size + ((int)at - slot * (int)size.d)) * p.head_dim;
}

__device__ __forceinline__ int64_t length_of(const Pool& p, const int64_t* lengths, int64_t b) {
  const int64_t n = lengths[b], most = p.max_pages * p.page_size;
  if (n < 0 || n > most) {
    if (p.bad) *p.bad = 1;
    return n < 0 ? 0 : most;
  }
  return n;
}

// ---------------------------------------------------------------- append, gather, copy
// V: the unit moved (an element, or 16 bytes where widths, strides and addresses allow). LPR lanes
// share a (sequence, head, position) row, its place is worked out once. HBM-bound: 16 x 12 heads
// of 64 over 1024 positions appended at 5.3 TB/s, one sequence of 65536 gathered at 5.7.
struct Rows {
  int64_t sb, sh, st;  // strides of (batch, head, position) in units
};

struct Moves {
  Pool pool;
  int rows;                       // batch * heads * positions
  FastDiv heads, positions, size;
  const int64_t* lengths;
};

template <int LPR, typename F>
__device__ __forceinline__ void each_row(const Moves& m, F body) {
  const int lane = threadIdx.x % LPR;
  const int step = (int)gridDim.x * (kThreads / LPR);
  for (int r = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR; r < m.rows; r += step) {
    const int bh = div_by(r, m.positions), t = r - bh * (int)m.positions.d;
    const int b = div_by(bh, m.heads), h = bh - b * (int)m.heads.d;
    body(b, h, t, lane);
  }
}

template <typename V, int LPR>
__global__ void __launch_bounds__(kThreads)
append_kernel(Moves m, const V* __restrict__ k, Rows ks, const V* __restrict__ v, Rows vs,
              V* __restrict__ keys, V* __restrict__ values) {
  each_row<LPR>(m, [&](int b, int h, int t, int lane) {
    const int64_t start = m.lengths[b];
    const int64_t to = row_of(m.pool, m.size, b, h, start < 0 ? -1 : start + t);
    if (to < 0) return;
    const V* a = k + b * ks.sb + h * ks.sh + t * ks.st;
    const V* c = v + b * vs.sb + h * vs.sh + t * vs.st;
    for (int i = lane; i < (int)m.pool.head_dim; i += LPR) {
      keys[to + i] = a[i];
      values[to + i] = c[i];
    }
  });
}

template <typename V, int LPR>
__global__ void __launch_bounds__(kThreads)
gather_kernel(Moves m, const V* __restrict__ keys, const V* __restrict__ values,
              V* __restrict__ k, V* __restrict__ v) {
  const int d = (int)m.pool.head_dim;
  each_row<LPR>(m, [&](int b, int h, int t, int lane) {
    const int64_t from =
        t < length_of(m.pool, m.lengths, b) ? row_of(m.pool, m.size, b, h, t) : -1;
    const int64_t to = (((int64_t)b * m.heads.d + h) * m.positions.d + t) * d;
    for (int i = lane; i < d; i += LPR) {
      k[to + i] = from < 0 ? V{} : keys[from + i];
      v[to + i] = from < 0 ? V{} : values[from + i];
    }
  });
}

// Pages src[i] to dst[i] in every layer of both pools; `units` of V to a page. Pages of 256 units
// and more take a block or several (1024 pages of 48 KB in 12 layers: 6.1 TB/s), shorter ones share
// one.
// Up to kInline pairs travel with the launch, more of them lie on the device.
constexpr int kInline = 64;

struct Pairs {
  const int64_t* src;
  const int64_t* dst;
  __device__ __forceinline__ int64_t from(int64_t i) const { return src[i]; }
  __device__ __forceinline__ int64_t to(int64_t i) const { return dst[i]; }
};
struct InlinePairs {
  int src[kInline], dst[kInline];
  __device__ __forceinline__ int64_t from(int64_t i) const { return src[i]; }
  __device__ __forceinline__ int64_t to(int64_t i) const { return dst[i]; }
};

template <typename V, typename P>
struct Copies {
  V* keys;
  V* values;
  int64_t layers, num_pages, units;
  P ids;
  int64_t pairs;
  int* bad;
};

// Where copy e of 2 layers pairs reads and writes; false behind a bad id.
template <typename V, typename P>
__device__ __forceinline__ bool place_of(const Copies<V, P>& c, int64_t l, int64_t i,
                                         const V*& from, V*& to) {
  const int64_t a = c.ids.from(i), b = c.ids.to(i);
  if (a < 0 || a >= c.num_pages || b < 0 || b >= c.num_pages) {
    if (c.bad) *c.bad = 1;
    return false;
  }
  V* pool = l < c.layers ? c.keys + l * c.num_pages * c.units
                         : c.values + (l - c.layers) * c.num_pages * c.units;
  from = pool + a * c.units;
  to = pool + b * c.units;
  return true;
}

template <typename V, typename P>
__global__ void __launch_bounds__(kThreads)
page_copy_kernel(const __grid_constant__ Copies<V, P> c, int parts, int64_t part) {
  const int64_t total = 2 * c.layers * c.pairs * parts;
  for (int64_t e = blockIdx.x; e < total; e += gridDim.x) {
    const int64_t p = e / parts, first = e % parts * part;
    const int64_t end = first + part < c.units ? first + part : c.units;
    const V* from;
    V* to;
    if (!place_of(c, p / c.pairs, p % c.pairs, from, to)) continue;
#pragma unroll 4
    for (int64_t i = first + threadIdx.x; i < end; i += kThreads) to[i] = from[i];
  }
}

template <typename V, typename P>
__global__ void __launch_bounds__(kThreads)
page_copy_short_kernel(const __grid_constant__ Copies<V, P> c, int total, FastDiv units, FastDiv pairs) {
  for (int e = blockIdx.x * kThreads + threadIdx.x; e < total; e += (int)gridDim.x * kThreads) {
    const int p = div_by(e, units), l = div_by(p, pairs);
    const V* from;
    V* to;
    if (!place_of(c, l, p - l * (int)pairs.d, from, to)) continue;
    const int i = e - p * (int)units.d;
    to[i] = from[i];
  }
}

// ---------------------------------------------------------------- attention of one token
constexpr int kMaxHead = 256;
constexpr int kAttend = 128;        // threads of an attention block
constexpr int kWarps = kAttend / 32;
constexpr int kLaneDims = 8;        // features of a position that one lane holds
constexpr int kTable = 512;        // pages named in shared memory at a time
constexpr int kMinSplit = 128;      // positions that a block has at least, if there are as many
constexpr int kMaxSplits = 512;
constexpr int kMaxCluster = 8;      // splits that join through their cluster's shared memory

// e^x on scores that carry the factor `unit`: float scores are in base 2 (one instruction less
// per weight), double ones in base e.
template <typename T>
struct Base;
template <>
struct Base<float> {
  static constexpr double unit = 1.4426950408889634;  // log2 e
  static __device__ __forceinline__ float exp_(float x) { return exp2f(x); }
  static __device__ __forceinline__ float natural(float x) { return x * 0.6931471805599453f; }
};
template <>
struct Base<double> {
  static constexpr double unit = 1.0;
  static __device__ __forceinline__ double exp_(double x) { return exp(x); }
  static __device__ __forceinline__ double natural(double x) { return x; }
};

// A lane's 8 features. Floats are kept and multiplied two to an instruction (fma.rn.f32x2: half the
// issue slots, the same roundings).
template <typename T>
struct Eight {
  T v[kLaneDims];
  __device__ __forceinline__ void set(const T (&x)[kLaneDims]) {
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) v[i] = x[i];
  }
  __device__ __forceinline__ T get(int i) const { return v[i]; }
  __device__ __forceinline__ T dot(const Eight& o) const {
    T s = v[0] * o.v[0];
#pragma unroll
    for (int i = 1; i < kLaneDims; ++i) s += v[i] * o.v[i];
    return s;
  }
  __device__ __forceinline__ void add(T f, const Eight& o) {
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) v[i] += f * o.v[i];
  }
  __device__ __forceinline__ void scale(T f) {
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) v[i] *= f;
  }
};

template <>
struct Eight<float> {
  using Two = unsigned long long;
  Two p[kLaneDims / 2];
  static __device__ __forceinline__ Two pack(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
  }
  static __device__ __forceinline__ float2 unpack(Two x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
  }
  static __device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
  }
  static __device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
  }
  __device__ __forceinline__ void set(const float (&x)[kLaneDims]) {
#pragma unroll
    for (int i = 0; i < kLaneDims / 2; ++i) p[i] = pack(x[2 * i], x[2 * i + 1]);
  }
  __device__ __forceinline__ float get(int i) const {
    const float2 x = unpack(p[i / 2]);
    return i % 2 ? x.y : x.x;
  }
  __device__ __forceinline__ float dot(const Eight& o) const {
    Two s = mul2(p[0], o.p[0]);
#pragma unroll
    for (int i = 1; i < kLaneDims / 2; ++i) s = fma2(p[i], o.p[i], s);
    const float2 x = unpack(s);
    return x.x + x.y;
  }
  __device__ __forceinline__ void add(float f, const Eight& o) {
    const Two both = pack(f, f);
#pragma unroll
    for (int i = 0; i < kLaneDims / 2; ++i) p[i] = fma2(both, o.p[i], p[i]);
  }
  __device__ __forceinline__ void scale(float f) {
    const Two both = pack(f, f);
#pragma unroll
    for (int i = 0; i < kLaneDims / 2; ++i) p[i] = mul2(p[i], both);
  }
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool live) {
  const int n = live ? BYTES : 0;  // nothing read, zeros written
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n));
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES),
                 "r"(n));
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

struct AttendArgs {
  Pool pool;
  int64_t heads, group, head_groups;  // query heads; to a key head; blocks that share one
  int64_t q_sb, q_sh;
  const int64_t* lengths;
  int64_t batch_heads;  // sequences times query heads
  int splits;
  bool clustered;       // a sequence's splits are one cluster
  FastDiv size;
  double scale;
};

// Positions to a split of a sequence of n: as even as `splits` makes them, but no fewer than
// kMinSplit, in multiples of 32.
__device__ __forceinline__ int split_length(int n, int splits) {
  const int even = (n + splits - 1) / splits;
  const int c = even > kMinSplit ? even : kMinSplit;
  return (c + 31) / 32 * 32;
}

// One block per (sequence, key head, split of its positions, group of GH query heads). LPT lanes
// share a position, each with 8 of its features; a lane group takes U positions at a time and runs
// its own softmax, a warp has 32 / LPT groups, queries and outputs of GH heads stay in registers.
// Each lane copies its features of the next positions' keys and values into shared memory itself
// (cp.async, VE elements at a time) and is the only one to read them: no barrier in the loop.
// The U GH scores of a group are reduced by halving: at each of the first levels a lane keeps
// half of its partial scores and hands the other half over, so that a score is finished, and its
// exponential taken, in one lane (LPT / (U GH) lanes), and is then dealt out to the group.
// What bounds it: reading keys and values once (6.5 to 6.8 TB/s up to 4 heads of 128 to a key
// head), behind that the issue slots (8 heads: 4.9 TB/s).
constexpr int U = 2;

// The maximum that weights are taken against follows only when a score is above it by more than
// this (a weight is then at most 2^4, in double e^4, and the sum keeps its digits): a warp with
// several heads would else scale its outputs in most of its first rounds (9 sequences of 10 heads
// on 5 of 40 in double, 64 of them up to 4096 positions: 143 -> 137 us).
constexpr int kSlack = 4;

constexpr int log2_of(int x) { return x <= 1 ? 0 : 1 + log2_of(x / 2); }

template <typename T, int VE, int LPT, int GH>
struct Attend {
  static constexpr int NVEC = kLaneDims / VE;
  static constexpr int VB = VE * (int)sizeof(T);
  static constexpr int ROW = 2 * NVEC * VB * kAttend;  // one position per lane group
  static constexpr int STAGE = U * ROW;
  static constexpr int ST = sizeof(T) == 4 ? 3 : 2;
  static constexpr int WIDTH = LPT * kLaneDims;  // features covered
  static constexpr int RING = ST * STAGE;
  // The warps' results and the block's, with a maximum and a sum each.
  static constexpr int JOIN = (kWarps + 1) * GH * (WIDTH + 2) * (int)sizeof(T);
  static constexpr int SMEM = (RING > JOIN ? RING : JOIN) + kTable * 8;
  // The scores of a group: value v = u GH + g ends in the lane of the group whose top LEVELS bits
  // are v's top bits, as its (v % KEPT)-th.
  static constexpr int V = U * GH;
  static constexpr int LEVELS = log2_of(LPT) < log2_of(V) ? log2_of(LPT) : log2_of(V);
  static constexpr int KEPT = V >> LEVELS;
  static constexpr int lane_of(int v) { return (v / KEPT) << (log2_of(LPT) - LEVELS); }
};

template <typename T, int VE, int LPT, int GH>
__global__ void __launch_bounds__(kAttend, 4)
paged_attention_kernel(AttendArgs a, const T* __restrict__ q, const T* __restrict__ keys,
                       const T* __restrict__ values, T* __restrict__ out, T* __restrict__ lse,
                       T* __restrict__ part) {
  using A = Attend<T, VE, LPT, GH>;
  constexpr int NVEC = A::NVEC, ST = A::ST, TPW = 32 / LPT, ROWS = kWarps * TPW, STEP = U * ROWS;
  constexpr int V = A::V, KEPT = A::KEPT;
  constexpr T kLowest = std::numeric_limits<T>::lowest();
  struct alignas(A::VB) Held {
    T v[VE];
  };
  extern __shared__ __align__(16) uint8_t smem[];
  int64_t* table = reinterpret_cast<int64_t*>(smem + A::SMEM - kTable * 8);
  pdl_trigger();
  pdl_wait();
  int64_t e = blockIdx.x;
  const int split = (int)(e % a.splits);
  e /= a.splits;
  const int64_t g0 = (e % a.head_groups) * GH;
  e /= a.head_groups;
  const int64_t kh = e % a.pool.kv_heads, b = e / a.pool.kv_heads;
  const int d = (int)a.pool.head_dim;
  const int n = (int)length_of(a.pool, a.lengths, b);
  const int len = split_length(n, a.splits);
  const int begin = split * len, end = begin + len < n ? begin + len : n;
  if (begin >= n && split > 0 && !a.clustered) return;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int sub = lane / LPT, j = lane % LPT;
  const int64_t h0 = kh * a.group + g0;
  const int live_heads = (int)(a.group - g0 < GH ? a.group - g0 : GH);

  // m and l belong to the KEPT scores that this lane finishes: the running maximum of that
  // score's head (the same in every lane of the group that has the head) and the sum over the
  // positions that came to this lane.
  Eight<T> qr[GH], acc[GH];
  T m[KEPT], l[KEPT];
#pragma unroll
  for (int g = 0; g < GH; ++g) {
    T x[kLaneDims], zero[kLaneDims] = {};
#pragma unroll
    for (int i = 0; i < kLaneDims; ++i) {
      const int c = ((i / VE) * LPT + j) * VE + i % VE;
      x[i] = g < live_heads && c < d
                 ? q[b * a.q_sb + (h0 + g) * a.q_sh + c] * (T)(a.scale * Base<T>::unit)
                 : T(0);
    }
    qr[g].set(x);
    acc[g].set(zero);
  }
#pragma unroll
  for (int r = 0; r < KEPT; ++r) {
    m[r] = kLowest;
    l[r] = T(0);
  }
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * A::VB;
  const uint8_t* mine = smem + threadIdx.x * A::VB;
  // Features behind the head's width are never copied: they stay zero.
  for (int i = 0; i < ST * U * 2 * NVEC; ++i) {
    if (((i % NVEC) * LPT + j) * VE < d) continue;
    T* z = reinterpret_cast<T*>(smem + threadIdx.x * A::VB + i * (A::VB * kAttend));
#pragma unroll
    for (int v = 0; v < VE; ++v) z[v] = T(0);
  }
  const int my_row = w * TPW + sub;  // of the ROWS positions of a round
  for (int t0 = begin; t0 < end;) {
    // Where the pages of the next positions start, as many as the table holds.
    const int p0 = div_by(t0, a.size);
    const int64_t stop = (int64_t)(p0 + kTable) * a.size.d;
    const int t1 = stop < end ? (int)stop : end;
    const int used = div_by(t1 - 1, a.size) - p0 + 1;
    __syncthreads();
    for (int i = threadIdx.x; i < used; i += kAttend) {
      int64_t page = a.pool.table[b * a.pool.max_pages + p0 + i];
      if (page < 0 || page >= a.pool.num_pages) {
        if (a.pool.bad) *a.pool.bad = 1;
        page = 0;
      }
      table[i] = (page * a.pool.kv_heads + kh) * a.pool.page_size * d;
    }
    __syncthreads();
    const int steps = (t1 - t0 + STEP - 1) / STEP;
    // Each lane of a group looks up the group's positions of one of the next LPT rounds, and hands
    // them out when their round comes: in every lane for every round it was a sixth of all
    // instructions (8 heads of 128 to a key head, 4 x 8 of them up to 65536 positions: 345 -> 315
    // us; the double case above: 137 -> 128 us).
    int64_t where[U];
    auto issue = [&](int i) {
      if (i % LPT == 0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = t0 + (i + j) * STEP + u * ROWS + my_row;
          where[u] = -1;
          if (t < t1) {
            const int p = div_by(t, a.size);
            where[u] = table[p - p0] + (int64_t)(t - p * (int)a.size.d) * d;
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = __shfl_sync(0xffffffffu, where[u], sub * LPT + i % LPT);
        const bool live = row >= 0;
        const int64_t at = (live ? row : 0) + j * VE;
        const uint32_t to = ring + (i % ST) * A::STAGE + u * A::ROW;
        const T* k = keys + at;
        const T* v = values + at;
#pragma unroll
        for (int x = 0; x < NVEC; ++x)
          if ((x * LPT + j) * VE < d) {
            copy_async<A::VB>(to + x * (A::VB * kAttend), k + x * (LPT * VE), live);
            copy_async<A::VB>(to + (NVEC + x) * (A::VB * kAttend), v + x * (LPT * VE), live);
          }
      }
    };
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      if (i < steps) issue(i);
      copy_commit();
    }
    for (int i = 0; i < steps; ++i) {
      copy_wait<ST - 2>();
      const uint8_t* from = mine + (i % ST) * A::STAGE;
      auto load = [&](const uint8_t* row) {
        T x[kLaneDims];
#pragma unroll
        for (int v = 0; v < NVEC; ++v) {
          const Held y = *reinterpret_cast<const Held*>(row + v * (A::VB * kAttend));
#pragma unroll
          for (int c = 0; c < VE; ++c) x[v * VE + c] = y.v[c];
        }
        Eight<T> e;
        e.set(x);
        return e;
      };
      T s[V];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Eight<T> x = load(from + u * A::ROW);
#pragma unroll
        for (int g = 0; g < GH; ++g) s[u * GH + g] = qr[g].dot(x);
      }
#pragma unroll
      for (int k = 0; k < log2_of(LPT); ++k) {
        const int o = LPT >> (k + 1);
        if (k < A::LEVELS) {
          const int half = V >> (k + 1);
          const bool upper = j & o;
#pragma unroll
          for (int v = 0; v < half; ++v) {
            const T give = upper ? s[v] : s[v + half], keep = upper ? s[v + half] : s[v];
            s[v] = keep + __shfl_xor_sync(0xffffffffu, give, o);
          }
        } else {
#pragma unroll
          for (int v = 0; v < KEPT; ++v) s[v] += __shfl_xor_sync(0xffffffffu, s[v], o);
        }
      }
      // s[0..KEPT): this lane's finished scores; its position is the first or second of the
      // group's two by its top bit.
      const int left = t1 - (t0 + i * STEP + my_row);
      const bool live = left > (j & (LPT / 2) ? ROWS : 0);
      bool grows = false;
#pragma unroll
      for (int r = 0; r < KEPT; ++r) {
        if (!live) s[r] = T(-INFINITY);
        grows |= s[r] > m[r] + kSlack;
      }
      if (__any_sync(0xffffffffu, grows)) {
        T c[KEPT];
#pragma unroll
        for (int r = 0; r < KEPT; ++r) {
          const T other = __shfl_xor_sync(0xffffffffu, s[r], LPT / 2);
          const T top = fmax(m[r], fmax(s[r], other));
          c[r] = Base<T>::exp_(m[r] - top);
          m[r] = top;
          l[r] *= c[r];
        }
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          acc[g].scale(__shfl_sync(0xffffffffu, c[g % KEPT], sub * LPT + A::lane_of(g)));
        }
      }
#pragma unroll
      for (int r = 0; r < KEPT; ++r) {
        s[r] = Base<T>::exp_(s[r] - m[r]);
        l[r] += s[r];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const Eight<T> x = load(from + u * A::ROW + NVEC * (A::VB * kAttend));
#pragma unroll
        for (int g = 0; g < GH; ++g) {
          const int v = u * GH + g;
          acc[g].add(__shfl_sync(0xffffffffu, s[v % KEPT], sub * LPT + A::lane_of(v)), x);
        }
      }
      if (i + ST - 1 < steps) issue(i + ST - 1);
      copy_commit();
    }
    copy_wait<0>();
    t0 = t1;
  }

  // Every lane learns its heads' maxima and sums, then the warp's lane groups join, then the
  // block's warps.
  T mg[GH], lg[GH], og[GH][kLaneDims];
#pragma unroll
  for (int g = 0; g < GH; ++g) {
#pragma unroll
    for (int k = 0; k < kLaneDims; ++k) og[g][k] = acc[g].get(k);
    mg[g] = __shfl_sync(0xffffffffu, m[g % KEPT], sub * LPT + A::lane_of(g));
    lg[g] = T(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
      lg[g] += __shfl_sync(0xffffffffu, l[g % KEPT], sub * LPT + A::lane_of(u * GH + g));
  }
#pragma unroll
  for (int o = LPT; o < 32; o <<= 1)
#pragma unroll
    for (int g = 0; g < GH; ++g) {
      const T top = fmax(mg[g], __shfl_xor_sync(0xffffffffu, mg[g], o));
      const T c = lg[g] == T(0) ? T(0) : Base<T>::exp_(mg[g] - top);
      lg[g] *= c;
      lg[g] += __shfl_xor_sync(0xffffffffu, lg[g], o);
      mg[g] = top;
#pragma unroll
      for (int k = 0; k < kLaneDims; ++k) {
        og[g][k] *= c;
        og[g][k] += __shfl_xor_sync(0xffffffffu, og[g][k], o);
      }
    }
  __syncthreads();
  T* sacc = reinterpret_cast<T*>(smem);                // [warp][GH][WIDTH]
  T* sm = sacc + kWarps * GH * A::WIDTH;               // [warp][GH]
  T* sl = sm + kWarps * GH;
  if (sub == 0) {
#pragma unroll
    for (int g = 0; g < GH; ++g) {
#pragma unroll
      for (int k = 0; k < kLaneDims; ++k)
        sacc[(w * GH + g) * A::WIDTH + ((k / VE) * LPT + j) * VE + k % VE] = og[g][k];
      if (j == 0) {
        sm[w * GH + g] = mg[g];
        sl[w * GH + g] = lg[g];
      }
    }
  }
  __syncthreads();
  const bool whole = n <= len;  // no other split of this sequence
  T* rt = sl + kWarps * GH;     // [GH], the block's maxima, sums and outputs
  T* rs = rt + GH;
  T* rv = rs + GH;
  for (int i = threadIdx.x; i < live_heads * d; i += kAttend) {
    const int g = i / d, c = i % d;
    T top = kLowest, sum = T(0), v = T(0);
#pragma unroll
    for (int k = 0; k < kWarps; ++k) top = fmax(top, sm[k * GH + g]);
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
      const T ls = sl[k * GH + g];
      const T f = ls == T(0) ? T(0) : Base<T>::exp_(sm[k * GH + g] - top);
      sum += ls * f;
      v += (ls == T(0) ? T(0) : sacc[(k * GH + g) * A::WIDTH + c]) * f;
    }
    const int64_t head = b * a.heads + h0 + g;
    if (a.clustered) {
      rv[g * d + c] = v;
      if (c == 0) {
        rt[g] = top;
        rs[g] = sum;
      }
    } else if (whole) {
      out[head * d + c] = n == 0 ? T(0) : v / sum;
      if (c == 0 && lse)
        lse[head] = n == 0 ? T(-INFINITY) : Base<T>::natural(top) + dev_log<T>(sum);
    } else {
      T* ml = part + (head * a.splits + split) * 2;
      part[a.batch_heads * a.splits * 2 + (head * a.splits + split) * d + c] = v;
      if (c == 0) {
        ml[0] = top;
        ml[1] = sum;
      }
    }
  }
  if (!a.clustered) return;
  // The splits of this sequence are this cluster's blocks: each joins a share of the outputs.
  const auto cluster = cooperative_groups::this_cluster();
  cluster.sync();
  for (int i = split * kAttend + threadIdx.x; i < live_heads * d; i += a.splits * kAttend) {
    const int g = i / d, c = i % d;
    T top = kLowest, sum = T(0), v = T(0);
    for (int r = 0; r < a.splits; ++r) top = fmax(top, cluster.map_shared_rank(rt, r)[g]);
    for (int r = 0; r < a.splits; ++r) {
      const T ls = cluster.map_shared_rank(rs, r)[g];
      const T f = ls == T(0) ? T(0) : Base<T>::exp_(cluster.map_shared_rank(rt, r)[g] - top);
      sum += ls * f;
      v += (ls == T(0) ? T(0) : cluster.map_shared_rank(rv, r)[i]) * f;
    }
    const int64_t head = b * a.heads + h0 + g;
    out[head * d + c] = n == 0 ? T(0) : v / sum;
    if (c == 0 && lse)
      lse[head] = n == 0 ? T(-INFINITY) : Base<T>::natural(top) + dev_log<T>(sum);
  }
  cluster.sync();  // the others may still read this block's results
}

// The splits of a sequence's head as one: block per (sequence, head), their weights found once,
// their outputs dealt to the warps.
constexpr int kJoinWarps = kThreads / 32;

template <typename T>
__global__ void __launch_bounds__(kThreads)
paged_join_kernel(AttendArgs a, const T* __restrict__ part, T* __restrict__ out,
                  T* __restrict__ lse) {
  __shared__ T weight[kMaxSplits], red[32], sacc[kJoinWarps][kMaxHead];
  pdl_wait();
  const int64_t head = blockIdx.x, b = head / a.heads;
  const int d = (int)a.pool.head_dim, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = (int)length_of(a.pool, a.lengths, b);
  const int len = split_length(n, a.splits);
  if (n <= len) return;  // written by its only block
  const int live = (n + len - 1) / len;
  const T* ml = part + head * a.splits * 2;
  T top = std::numeric_limits<T>::lowest(), sum = T(0);
  for (int i = threadIdx.x; i < live; i += kThreads) top = fmax(top, ml[2 * i]);
  top = block_max(top, red);
  for (int i = threadIdx.x; i < live; i += kThreads) {
    const T ls = ml[2 * i + 1], f = ls == T(0) ? T(0) : Base<T>::exp_(ml[2 * i] - top);
    weight[i] = f;
    sum += ls * f;
  }
  sum = block_sum(sum, red);  // its barriers also publish the weights
  const T* from = part + a.batch_heads * a.splits * 2 + head * a.splits * d;
  for (int c = lane; c < d; c += 32) {
    T v = T(0);
#pragma unroll 4
    for (int i = w; i < live; i += kJoinWarps) v += from[(int64_t)i * d + c] * weight[i];
    sacc[w][c] = v;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < d; c += kThreads) {
    T v = T(0);
#pragma unroll
    for (int i = 0; i < kJoinWarps; ++i) v += sacc[i][c];
    out[head * d + c] = v / sum;
  }
  if (threadIdx.x == 0 && lse) lse[head] = Base<T>::natural(top) + dev_log<T>(sum);
}

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

// Query heads that one block takes: the group of a key head, rounded up to a power of two, at
// most 4 (2 where the lanes hold double): 8 leave half as many warps for the registers, and two
// blocks that share keys and values through the L2 are faster (8 heads of 64 to a key head, 64 x 4
// of them up to 4096 positions: 190 us with 8, 116 with 4 a block; 96 since positions are looked up
// once for many rounds).
int heads_per_block(int dtype, int64_t group) {
  const int most = dtype == TG_F64 ? 2 : 4;
  int g = 1;
  while (g < group && g < most) g *= 2;
  return g;
}

// Splits of the longest sequence: none where the sequences and heads alone give every
// multiprocessor its 4 blocks (768 of them, up to 1024 positions of 64: 45.5 us unsplit, 47.0 in
// halves), else about twice that many blocks (32 of them, up to 65536 positions of 128: 252, 236
// and 250 us with 1, 2 and 3 times), none shorter than kMinSplit (one sequence of 1024 positions
// on 12 heads: 8.4, 7.1 and 8.4 us with 64, 128 and 256).
int split_count(int dtype, int64_t batch, int64_t heads, int64_t kv_heads, int64_t longest) {
  const int gh = heads_per_block(dtype, heads / kv_heads);
  const int64_t groups = (heads / kv_heads + gh - 1) / gh;
  const int64_t blocks = batch * kv_heads * groups, slots = 4 * (int64_t)sm_count();
  if (blocks >= slots) return 1;
  const int64_t want = (2 * slots + blocks - 1) / blocks;
  const int64_t most = (longest + kMinSplit - 1) / kMinSplit;
  const int64_t n = want < most ? want : most;
  if (n > kMaxCluster) return (int)(n > kMaxSplits ? kMaxSplits : n);
  int c = 1;  // clusters of 1, 2, 4 and 8
  while (c < n) c *= 2;
  return c;
}

template <typename T, int VE, int LPT, int GH>
int launch_attend(const AttendArgs& a, int64_t blocks, const T* q, const T* keys, const T* values,
                  T* out, T* lse, T* part, cudaStream_t s) {
  using A = Attend<T, VE, LPT, GH>;
  TG_CUDA_TRY(cudaFuncSetAttribute(paged_attention_kernel<T, VE, LPT, GH>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, A::SMEM));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kAttend);
  cfg.dynamicSmemBytes = A::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {(unsigned)(a.clustered ? a.splits : 1), 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 2;
  TG_CUDA_TRY(cudaLaunchKernelEx(&cfg, paged_attention_kernel<T, VE, LPT, GH>, a, q, keys, values,
                                 out, lse, part));
  return check_launch("paged_attention");
}

template <typename T, int VE, int LPT>
int attend_heads(int gh, const AttendArgs& a, int64_t blocks, const T* q, const T* keys,
                 const T* values, T* out, T* lse, T* part, cudaStream_t s) {
  switch (gh) {
    case 1: return launch_attend<T, VE, LPT, 1>(a, blocks, q, keys, values, out, lse, part, s);
    case 2: return launch_attend<T, VE, LPT, 2>(a, blocks, q, keys, values, out, lse, part, s);
  }
  if constexpr (sizeof(T) == 4)
    return launch_attend<T, VE, LPT, 4>(a, blocks, q, keys, values, out, lse, part, s);
  return set_error(TG_ERR_UNSUPPORTED, "paged_attention: %d heads to a block", gh);
}

template <typename T, int VE>
int attend_width(int gh, const AttendArgs& a, int64_t blocks, const T* q, const T* keys,
                 const T* values, T* out, T* lse, T* part, cudaStream_t s) {
  const int64_t d = a.pool.head_dim;
  if (d <= 32) return attend_heads<T, VE, 4>(gh, a, blocks, q, keys, values, out, lse, part, s);
  if (d <= 64) return attend_heads<T, VE, 8>(gh, a, blocks, q, keys, values, out, lse, part, s);
  if (d <= 128) return attend_heads<T, VE, 16>(gh, a, blocks, q, keys, values, out, lse, part, s);
  return attend_heads<T, VE, 32>(gh, a, blocks, q, keys, values, out, lse, part, s);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct alignas(16) Unit16 {
  uint32_t w[4];
};

int check_pool(const char* what, int64_t num_pages, int64_t kv_heads, int64_t page_size,
               int64_t head_dim, int64_t max_pages) {
  TG_CHECK_ARG(num_pages > 0 && kv_heads > 0 && page_size > 0 && head_dim > 0 && max_pages > 0,
               "%s: pool of %lld pages of (%lld heads, %lld positions, %lld features), table of "
               "%lld", what, (long long)num_pages, (long long)kv_heads, (long long)page_size,
               (long long)head_dim, (long long)max_pages);
  TG_CHECK_ARG(num_pages <= INT32_MAX && kv_heads <= INT32_MAX && head_dim <= INT32_MAX &&
                   max_pages <= (INT32_MAX - (1 << 16)) / page_size,
               "%s: positions up to 2^31 (table of %lld pages of %lld)", what,
               (long long)max_pages, (long long)page_size);
  return TG_OK;
}

// The rows of (batch, heads, positions), and how many blocks of LPR lanes a row they make.
int make_moves(const char* what, const Pool& pool, int64_t batch, int64_t positions,
               const int64_t* lengths, Moves& m) {
  // Half the range: a lane's next row is worked out before it is compared.
  TG_CHECK_ARG(batch <= INT32_MAX / 2 / pool.kv_heads / positions,
               "%s: %lld x %lld x %lld rows", what, (long long)batch, (long long)pool.kv_heads,
               (long long)positions);
  m.pool = pool;
  m.rows = (int)(batch * pool.kv_heads * positions);
  m.heads = make_div(pool.kv_heads);
  m.positions = make_div(positions);
  m.size = make_div(pool.page_size);
  m.lengths = lengths;
  return TG_OK;
}

// Calls f with the lanes to a row of `units`: a power of two up to a warp.
template <typename F>
int with_lanes(int64_t units, F f) {
  if (units <= 4) return f(std::integral_constant<int, 4>{});
  if (units <= 8) return f(std::integral_constant<int, 8>{});
  if (units <= 16) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 32>{});
}

template <typename V>
int launch_append(const Moves& m, const V* k, Rows ks, const V* v, Rows vs, V* keys, V* values,
                  cudaStream_t s) {
  return with_lanes(m.pool.head_dim, [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    append_kernel<V, LPR><<<grid_for((int64_t)m.rows * LPR, kThreads), kThreads, 0, s>>>(
        m, k, ks, v, vs, keys, values);
    return check_launch("paged_append");
  });
}

template <typename V>
int launch_gather(const Moves& m, const V* keys, const V* values, V* k, V* v, cudaStream_t s) {
  return with_lanes(m.pool.head_dim, [&](auto lanes) {
    constexpr int LPR = decltype(lanes)::value;
    gather_kernel<V, LPR><<<grid_for((int64_t)m.rows * LPR, kThreads), kThreads, 0, s>>>(
        m, keys, values, k, v);
    return check_launch("paged_gather");
  });
}

template <typename V, typename P>
int launch_copies(const Copies<V, P>& c, cudaStream_t s) {
  const int64_t pages = 2 * c.layers * c.pairs;
  if (c.units < kThreads && pages * c.units <= INT32_MAX / 2)
    page_copy_short_kernel<<<grid_for(pages * c.units, kThreads), kThreads, 0, s>>>(
        c, (int)(pages * c.units), make_div(c.units), make_div(c.pairs));
  else {
    // Few pages are cut into parts of at least 4 units a lane.
    const int64_t most = (c.units + 4 * kThreads - 1) / (4 * kThreads);
    const int64_t want = (148 * 8 + pages - 1) / pages;
    const int64_t parts = want < most ? want : most, part = (c.units + parts - 1) / parts;
    page_copy_kernel<<<grid_for(pages * parts, 1), kThreads, 0, s>>>(c, (int)parts, part);
  }
  return check_launch("page_copy");
}

template <typename P>
int copy_pages(int64_t page_bytes, int64_t layers, int64_t num_pages, void* key_pages,
               void* value_pages, const P& ids, int64_t pairs, int* bad, cudaStream_t s) {
  if (page_bytes % 16 == 0 && aligned16(key_pages) && aligned16(value_pages))
    return launch_copies(Copies<Unit16, P>{(Unit16*)key_pages, (Unit16*)value_pages, layers,
                                           num_pages, page_bytes / 16, ids, pairs, bad}, s);
  return launch_copies(Copies<uint32_t, P>{(uint32_t*)key_pages, (uint32_t*)value_pages, layers,
                                           num_pages, page_bytes / 4, ids, pairs, bad}, s);
}

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" {

int tg_paged_append(int dtype, int64_t batch, int64_t tokens, int64_t kv_heads, int64_t head_dim,
                    const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void* v,
                    int64_t v_sb, int64_t v_sh, int64_t v_st, void* key_pages, void* value_pages,
                    int64_t num_pages, int64_t page_size, const int64_t* pages, int64_t max_pages,
                    const int64_t* lengths, int* bad_page_dev, void* stream) {
  const int rc = check_pool("paged_append", num_pages, kv_heads, page_size, head_dim, max_pages);
  if (rc) return rc;
  TG_CHECK_ARG(batch >= 0 && tokens >= 0, "paged_append: bad sizes");
  if (batch == 0 || tokens == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    constexpr int64_t U = 16 / sizeof(T);
    Moves m;
    const Pool p{num_pages, kv_heads, page_size, head_dim, pages, max_pages, bad_page_dev};
    const int r = make_moves("paged_append", p, batch, tokens, lengths, m);
    if (r) return r;
    const int64_t strides = k_sb | k_sh | k_st | v_sb | v_sh | v_st;
    if (head_dim % U == 0 && strides % U == 0 && aligned16(k) && aligned16(v) &&
        aligned16(key_pages) && aligned16(value_pages)) {
      m.pool.head_dim /= U;
      return launch_append(m, (const Unit16*)k, Rows{k_sb / U, k_sh / U, k_st / U},
                           (const Unit16*)v, Rows{v_sb / U, v_sh / U, v_st / U},
                           (Unit16*)key_pages, (Unit16*)value_pages, s);
    }
    return launch_append(m, (const T*)k, Rows{k_sb, k_sh, k_st}, (const T*)v,
                         Rows{v_sb, v_sh, v_st}, (T*)key_pages, (T*)value_pages, s);
  });
}

int tg_paged_gather(int dtype, int64_t batch, int64_t longest, int64_t kv_heads, int64_t head_dim,
                    const void* key_pages, const void* value_pages, int64_t num_pages,
                    int64_t page_size, const int64_t* pages, int64_t max_pages,
                    const int64_t* lengths, void* k, void* v, int* bad_page_dev, void* stream) {
  const int rc = check_pool("paged_gather", num_pages, kv_heads, page_size, head_dim, max_pages);
  if (rc) return rc;
  TG_CHECK_ARG(batch >= 0 && longest >= 0, "paged_gather: bad sizes");
  if (batch == 0 || longest == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    constexpr int64_t U = 16 / sizeof(T);
    Moves m;
    const Pool p{num_pages, kv_heads, page_size, head_dim, pages, max_pages, bad_page_dev};
    const int r = make_moves("paged_gather", p, batch, longest, lengths, m);
    if (r) return r;
    if (head_dim % U == 0 && aligned16(k) && aligned16(v) && aligned16(key_pages) &&
        aligned16(value_pages)) {
      m.pool.head_dim /= U;
      return launch_gather(m, (const Unit16*)key_pages, (const Unit16*)value_pages, (Unit16*)k,
                           (Unit16*)v, s);
    }
    return launch_gather(m, (const T*)key_pages, (const T*)value_pages, (T*)k, (T*)v, s);
  });
}

int tg_page_copy(int64_t page_bytes, int64_t layers, int64_t num_pages, void* key_pages,
                 void* value_pages, const int64_t* src, const int64_t* dst, int64_t pairs,
                 int* bad_page_dev, void* stream) {
  TG_CHECK_ARG(page_bytes > 0 && page_bytes % 4 == 0 && layers > 0 && num_pages > 0 && pairs >= 0,
               "page_copy: bad sizes");
  if (pairs == 0) return TG_OK;
  return copy_pages(page_bytes, layers, num_pages, key_pages, value_pages, Pairs{src, dst}, pairs,
                    bad_page_dev, as_stream(stream));
}

int tg_page_copy_few_max(void) { return kInline; }

int tg_page_copy_few(int64_t page_bytes, int64_t layers, int64_t num_pages, void* key_pages,
                     void* value_pages, const int64_t* src_host, const int64_t* dst_host,
                     int64_t pairs, void* stream) {
  TG_CHECK_ARG(page_bytes > 0 && page_bytes % 4 == 0 && layers > 0 && num_pages > 0 &&
                   num_pages <= INT32_MAX && pairs >= 0 && pairs <= kInline,
               "page_copy_few: bad sizes");
  if (pairs == 0) return TG_OK;
  InlinePairs ids;
  for (int64_t i = 0; i < pairs; ++i) {
    if (src_host[i] < 0 || src_host[i] >= num_pages || dst_host[i] < 0 ||
        dst_host[i] >= num_pages)
      return set_error(TG_ERR_INDEX, "page_copy_few: pages %lld and %lld of %lld",
                       (long long)src_host[i], (long long)dst_host[i], (long long)num_pages);
    ids.src[i] = (int)src_host[i];
    ids.dst[i] = (int)dst_host[i];
  }
  return copy_pages(page_bytes, layers, num_pages, key_pages, value_pages, ids, pairs, nullptr,
                    as_stream(stream));
}

size_t tg_paged_attention_scratch_bytes(int dtype, int64_t batch, int64_t heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t longest) {
  if (batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 16;
  const int splits = split_count(dtype, batch, heads, kv_heads, longest);
  if (splits <= kMaxCluster) return 16;
  return (size_t)(batch * heads * splits * (head_dim + 2)) * (dtype == TG_F64 ? 8 : 4);
}

int tg_paged_attention(int dtype, int64_t batch, int64_t heads, int64_t kv_heads,
                       int64_t head_dim, const void* q, int64_t q_sb, int64_t q_sh,
                       const void* key_pages, const void* value_pages, int64_t num_pages,
                       int64_t page_size, const int64_t* pages, int64_t max_pages,
                       const int64_t* lengths, int64_t longest, void* out, void* lse,
                       int* bad_page_dev, void* scratch, void* stream) {
  const int rc = check_pool("paged_attention", num_pages, kv_heads, page_size, head_dim,
                            max_pages);
  if (rc) return rc;
  TG_CHECK_ARG(batch >= 0 && heads > 0 && heads % kv_heads == 0,
               "paged_attention: %lld query heads over %lld key heads", (long long)heads,
               (long long)kv_heads);
  if (head_dim > kMaxHead)
    return set_error(TG_ERR_UNSUPPORTED, "paged_attention: head_dim %lld (at most %d)",
                     (long long)head_dim, kMaxHead);
  TG_CHECK_ARG(batch <= INT32_MAX / (heads * kMaxSplits), "paged_attention: batch too large");
  if (batch == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    constexpr int VE = 16 / sizeof(T);
    AttendArgs a{};
    a.pool = {num_pages, kv_heads, page_size, head_dim, pages, max_pages, bad_page_dev};
    a.heads = heads;
    a.group = heads / kv_heads;
    const int gh = heads_per_block(dtype, a.group);
    a.head_groups = (a.group + gh - 1) / gh;
    a.batch_heads = batch * heads;
    a.q_sb = q_sb;
    a.q_sh = q_sh;
    a.lengths = lengths;
    a.splits = split_count(dtype, batch, heads, kv_heads, longest);
    a.clustered = a.splits > 1 && a.splits <= kMaxCluster;
    a.size = make_div(page_size);
    a.scale = 1.0 / sqrt((double)head_dim);
    const bool joins = a.splits > kMaxCluster;
    TG_CHECK_ARG(!joins || scratch, "paged_attention: no scratch");
    const int64_t blocks = batch * kv_heads * a.head_groups * a.splits;
    const int r = head_dim % VE == 0 && aligned16(key_pages) && aligned16(value_pages)
                      ? attend_width<T, VE>(gh, a, blocks, (const T*)q, (const T*)key_pages,
                                            (const T*)value_pages, (T*)out, (T*)lse, (T*)scratch,
                                            s)
                      : attend_width<T, 1>(gh, a, blocks, (const T*)q, (const T*)key_pages,
                                           (const T*)value_pages, (T*)out, (T*)lse, (T*)scratch,
                                           s);
    if (r || !joins) return r;
    TG_CUDA_TRY(launch_pdl(paged_join_kernel<T>, dim3((unsigned)(batch * heads)), dim3(kThreads),
                           0, s, a, (const T*)scratch, (T*)out, (T*)lse));
    return check_launch("paged_attention(join)");
  });
}

}  // extern "C"
