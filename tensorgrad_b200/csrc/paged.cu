// A key-value cache in pages and the attention of one new token over it (no reference
// counterpart; the paged form of the cache that nn/attention.py:27-111 of the reference keeps
// contiguous). A pool holds pages of `page_size` positions, (num_pages, kv_heads, page_size,
// head_dim) for the keys and as much for the values; a sequence's positions lie on the pages
// that its row of the page table names, in order.
//
// Page ids and lengths live on the device and are checked where they are read: an id outside
// [0, num_pages) reads page 0 or writes nothing, a length beyond the table counts as the
// table's end, and either sets *bad, which the host reads at its next synchronisation.
#include "common.cuh"

namespace tg {
namespace {

constexpr int kThreads = 256;

struct Pool {
  int64_t num_pages, kv_heads, page_size, head_dim;  // head_dim in units of the element moved
  const int64_t* table;                              // (batch, max_pages)
  int64_t max_pages;
  int* bad;
};

// The position's row of one head in a pool, or -1 behind a bad id or off the table.
__device__ __forceinline__ int64_t row_of(const Pool& p, int64_t b, int64_t h, int64_t at) {
  const int64_t slot = at / p.page_size;
  if (at < 0 || slot >= p.max_pages) {
    if (p.bad) *p.bad = 1;
    return -1;
  }
  const int64_t page = p.table[b * p.max_pages + slot];
  if (page < 0 || page >= p.num_pages) {
    if (p.bad) *p.bad = 1;
    return -1;
  }
  return ((page * p.kv_heads + h) * p.page_size + at % p.page_size) * p.head_dim;
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
// V: the unit moved (an element, or 16 bytes where widths, strides and addresses allow).
struct Rows {
  int64_t sb, sh, st;  // strides of (batch, head, position) in units
};

template <typename V>
__global__ void __launch_bounds__(kThreads)
append_kernel(Pool p, int64_t batch, int64_t tokens, const V* __restrict__ k, Rows ks,
              const V* __restrict__ v, Rows vs, const int64_t* __restrict__ start,
              V* __restrict__ keys, V* __restrict__ values) {
  const int64_t total = batch * tokens * p.kv_heads * p.head_dim;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
       e += (int64_t)gridDim.x * kThreads) {
    const int64_t c = e % p.head_dim, r = e / p.head_dim;
    const int64_t t = r % tokens, bh = r / tokens, h = bh % p.kv_heads, b = bh / p.kv_heads;
    const int64_t to = start[b] < 0 ? row_of(p, b, h, -1) : row_of(p, b, h, start[b] + t);
    if (to < 0) continue;
    keys[to + c] = k[b * ks.sb + h * ks.sh + t * ks.st + c];
    values[to + c] = v[b * vs.sb + h * vs.sh + t * vs.st + c];
  }
}

template <typename V>
__global__ void __launch_bounds__(kThreads)
gather_kernel(Pool p, int64_t batch, int64_t longest, const V* __restrict__ keys,
              const V* __restrict__ values, const int64_t* __restrict__ lengths,
              V* __restrict__ k, V* __restrict__ v) {
  const int64_t total = batch * p.kv_heads * longest * p.head_dim;
  for (int64_t e = (int64_t)blockIdx.x * kThreads + threadIdx.x; e < total;
       e += (int64_t)gridDim.x * kThreads) {
    const int64_t c = e % p.head_dim, r = e / p.head_dim;
    const int64_t t = r % longest, bh = r / longest, h = bh % p.kv_heads, b = bh / p.kv_heads;
    const int64_t from = t < length_of(p, lengths, b) ? row_of(p, b, h, t) : -1;
    k[e] = from < 0 ? V{} : keys[from + c];
    v[e] = from < 0 ? V{} : values[from + c];
  }
}

// Pages src[i] to dst[i] in every layer of both pools; `units` of V to a page.
template <typename V>
__global__ void __launch_bounds__(kThreads)
page_copy_kernel(V* keys, V* values, int64_t layers, int64_t num_pages, int64_t units,
                 const int64_t* __restrict__ src, const int64_t* __restrict__ dst, int64_t pairs,
                 int* __restrict__ bad) {
  const int64_t total = 2 * layers * pairs;
  for (int64_t e = blockIdx.x; e < total; e += gridDim.x) {
    const int64_t i = e % pairs, l = e / pairs;
    const int64_t from = src[i], to = dst[i];
    if (from < 0 || from >= num_pages || to < 0 || to >= num_pages) {
      if (bad && threadIdx.x == 0) *bad = 1;
      continue;
    }
    V* pool = (l < layers ? keys : values) + (l % layers) * num_pages * units;
    const V* a = pool + from * units;
    V* b = pool + to * units;
    for (int64_t c = threadIdx.x; c < units; c += kThreads) b[c] = a[c];
  }
}

// ---------------------------------------------------------------- attention of one token
constexpr int kMaxHead = 256;

// One block per (sequence, query head): each warp walks every eighth position with its own
// running maximum, sum and output, the eight are joined at the end.
template <typename T>
__global__ void __launch_bounds__(kThreads)
paged_attention_kernel(Pool p, int64_t heads, const T* __restrict__ q, int64_t q_sb, int64_t q_sh,
                       const T* __restrict__ keys, const T* __restrict__ values,
                       const int64_t* __restrict__ lengths, T scale, T* __restrict__ out,
                       T* __restrict__ lse) {
  constexpr int W = kThreads / 32, N = kMaxHead / 32;
  __shared__ T sm[W], sl[W], sa[W][kMaxHead];
  const int64_t b = blockIdx.x / heads, h = blockIdx.x % heads;
  const int64_t kh = h / (heads / p.kv_heads);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int d = (int)p.head_dim;
  const int64_t n = length_of(p, lengths, b);
  T qr[N], acc[N], m = T(-INFINITY), l = T(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    qr[i] = lane + 32 * i < d ? q[b * q_sb + h * q_sh + lane + 32 * i] * scale : T(0);
    acc[i] = T(0);
  }
  for (int64_t t = w; t < n; t += W) {
    int64_t at = row_of(p, b, kh, t);
    if (at < 0) at = kh * p.page_size * p.head_dim;
    T s = T(0);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < d) s += qr[i] * keys[at + lane + 32 * i];
    s = warp_sum(s);
    const T mn = fmax(m, s), c = m == mn ? T(1) : dev_exp<T>(m - mn);
    const T e = s == T(-INFINITY) ? T(0) : dev_exp<T>(s - mn);
    l = l * c + e;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 32 * i < d) acc[i] = acc[i] * c + e * values[at + lane + 32 * i];
    m = mn;
  }
  if (lane == 0) { sm[w] = m; sl[w] = l; }
#pragma unroll
  for (int i = 0; i < N; ++i) sa[w][lane + 32 * i] = acc[i];
  __syncthreads();
  T mx = T(-INFINITY), sum = T(0);
  for (int i = 0; i < W; ++i) mx = fmax(mx, sm[i]);
  for (int i = 0; i < W; ++i) sum += sl[i] == T(0) ? T(0) : sl[i] * dev_exp<T>(sm[i] - mx);
  for (int c = threadIdx.x; c < d; c += kThreads) {
    T a = T(0);
    for (int i = 0; i < W; ++i) a += sl[i] == T(0) ? T(0) : sa[i][c] * dev_exp<T>(sm[i] - mx);
    out[(b * heads + h) * d + c] = n == 0 ? T(0) : a / sum;
  }
  if (threadIdx.x == 0 && lse) lse[b * heads + h] = n == 0 ? T(-INFINITY) : mx + dev_log<T>(sum);
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
  return TG_OK;
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
    const Pool p{num_pages, kv_heads, page_size, head_dim, pages, max_pages, bad_page_dev};
    const int64_t strides = k_sb | k_sh | k_st | v_sb | v_sh | v_st;
    const int64_t total = batch * tokens * kv_heads * head_dim;
    if (head_dim % U == 0 && strides % U == 0 && aligned16(k) && aligned16(v) &&
        aligned16(key_pages) && aligned16(value_pages)) {
      Pool pu = p;
      pu.head_dim /= U;
      append_kernel<Unit16><<<grid_for(total / U, kThreads), kThreads, 0, s>>>(
          pu, batch, tokens, (const Unit16*)k, Rows{k_sb / U, k_sh / U, k_st / U},
          (const Unit16*)v, Rows{v_sb / U, v_sh / U, v_st / U}, lengths, (Unit16*)key_pages,
          (Unit16*)value_pages);
    } else {
      append_kernel<T><<<grid_for(total, kThreads), kThreads, 0, s>>>(
          p, batch, tokens, (const T*)k, Rows{k_sb, k_sh, k_st}, (const T*)v,
          Rows{v_sb, v_sh, v_st}, lengths, (T*)key_pages, (T*)value_pages);
    }
    return check_launch("paged_append");
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
    const Pool p{num_pages, kv_heads, page_size, head_dim, pages, max_pages, bad_page_dev};
    const int64_t total = batch * longest * kv_heads * head_dim;
    if (head_dim % U == 0 && aligned16(k) && aligned16(v) && aligned16(key_pages) &&
        aligned16(value_pages)) {
      Pool pu = p;
      pu.head_dim /= U;
      gather_kernel<Unit16><<<grid_for(total / U, kThreads), kThreads, 0, s>>>(
          pu, batch, longest, (const Unit16*)key_pages, (const Unit16*)value_pages, lengths,
          (Unit16*)k, (Unit16*)v);
    } else {
      gather_kernel<T><<<grid_for(total, kThreads), kThreads, 0, s>>>(
          p, batch, longest, (const T*)key_pages, (const T*)value_pages, lengths, (T*)k, (T*)v);
    }
    return check_launch("paged_gather");
  });
}

int tg_page_copy(int64_t page_bytes, int64_t layers, int64_t num_pages, void* key_pages,
                 void* value_pages, const int64_t* src, const int64_t* dst, int64_t pairs,
                 int* bad_page_dev, void* stream) {
  TG_CHECK_ARG(page_bytes > 0 && page_bytes % 4 == 0 && layers > 0 && num_pages > 0 && pairs >= 0,
               "page_copy: bad sizes");
  if (pairs == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  const unsigned grid = grid_for(2 * layers * pairs, 1);
  if (page_bytes % 16 == 0 && aligned16(key_pages) && aligned16(value_pages))
    page_copy_kernel<Unit16><<<grid, kThreads, 0, s>>>(
        (Unit16*)key_pages, (Unit16*)value_pages, layers, num_pages, page_bytes / 16, src, dst,
        pairs, bad_page_dev);
  else
    page_copy_kernel<uint32_t><<<grid, kThreads, 0, s>>>(
        (uint32_t*)key_pages, (uint32_t*)value_pages, layers, num_pages, page_bytes / 4, src, dst,
        pairs, bad_page_dev);
  return check_launch("page_copy");
}

size_t tg_paged_attention_scratch_bytes(int dtype, int64_t batch, int64_t heads, int64_t kv_heads,
                                        int64_t head_dim, int64_t longest) {
  return 16;
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
  TG_CHECK_ARG(batch * heads <= INT32_MAX, "paged_attention: batch too large");
  if (head_dim > kMaxHead)
    return set_error(TG_ERR_UNSUPPORTED, "paged_attention: head_dim %lld (at most %d)",
                     (long long)head_dim, kMaxHead);
  if (batch == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  (void)scratch;
  (void)longest;
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    const Pool p{num_pages, kv_heads, page_size, head_dim, pages, max_pages, bad_page_dev};
    paged_attention_kernel<T><<<(unsigned)(batch * heads), kThreads, 0, s>>>(
        p, heads, (const T*)q, q_sb, q_sh, (const T*)key_pages, (const T*)value_pages, lengths,
        (T)(1.0 / sqrt((double)head_dim)), (T*)out, (T*)lse);
    return check_launch("paged_attention");
  });
}

}  // extern "C"
