// Linear layers in 8-bit integers (no reference counterpart; the inference form of
// ops/layers.py:22-62): a scale for each token and each output channel,
//   s_m = max_k |x_mk| / 127,  q_mk = rint(x_mk / s_m),
//   y_mn = (sum_k q_mk w_nk) (s_m s_n) + bias_n,
// the sums exact in 32-bit integers (at most 127 * 128 * 131072 < 2^31). A row of zeros has scale
// 0 and integers 0; a row with a NaN or an infinity has scale NaN, so its outputs are NaN.
#include "common.cuh"

namespace tg {
namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxInner = 131072;

__host__ __device__ constexpr int64_t padded(int64_t inner) { return (inner + 15) / 16 * 16; }

// The integer of one value: the quotient rounds to the type first, then to the nearest integer
// (ties to even). The clamp only acts where a scale below the type's normal range lost bits.
template <typename T>
__device__ __forceinline__ int quantize(T x, T scale) {
  const T r = rint(x / scale);
  return (int)fmin(fmax(r, T(-127)), T(127));
}

// Row scales and integers; integer rows are ld bytes long, zero beyond the row's values.
template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int64_t inner, int8_t* __restrict__ q,
                     int64_t ld, T* __restrict__ scales) {
  __shared__ T sh[32];
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* a = x + r * inner;
    T top = T(0), odd = T(0);
    for (int64_t c = threadIdx.x; c < inner; c += kThreads) {
      const T v = fabs(a[c]);
      top = fmax(top, v);
      odd += v - v;  // NaN from a NaN or an infinity, else 0
    }
    top = block_max(top, sh);
    odd = block_sum(odd, sh);
    const T scale = top / T(127) + odd;
    const bool live = scale > T(0);
    for (int64_t c = threadIdx.x; c < ld; c += kThreads)
      q[r * ld + c] = (int8_t)(live && c < inner ? quantize(a[c], scale) : 0);
    if (threadIdx.x == 0) scales[r] = scale;
    __syncthreads();
  }
}

// A 64 x 64 tile of outputs to a block, 4 x 4 to a thread, 64 bytes of the reduction at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads)
int8_tile_kernel(const int8_t* __restrict__ a, const int8_t* __restrict__ b, int64_t ld,
                 int64_t b_ld, const T* __restrict__ a_scale, const T* __restrict__ b_scale,
                 const T* __restrict__ bias, T* __restrict__ y, int64_t rows, int64_t outer) {
  __shared__ int as[64][17], bs[64][17];
  const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  int acc[4][4] = {};
  const int lr = threadIdx.x >> 2, lc = (threadIdx.x & 3) * 4;  // this thread's 16 bytes
  for (int64_t k = 0; k < ld; k += 64) {
    int4 va = {}, vb = {};
    if (k + lc * 4 < ld) {
      if (m0 + lr < rows) va = *reinterpret_cast<const int4*>(a + (m0 + lr) * ld + k + lc * 4);
      if (n0 + lr < outer) vb = *reinterpret_cast<const int4*>(b + (n0 + lr) * b_ld + k + lc * 4);
    }
    __syncthreads();
    as[lr][lc] = va.x; as[lr][lc + 1] = va.y; as[lr][lc + 2] = va.z; as[lr][lc + 3] = va.w;
    bs[lr][lc] = vb.x; bs[lr][lc + 1] = vb.y; bs[lr][lc + 2] = vb.z; bs[lr][lc + 3] = vb.w;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      int av[4], bv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) { av[i] = as[ty + 16 * i][w]; bv[i] = bs[tx + 16 * i][w]; }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(av[i], bv[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + ty + 16 * i;
    if (m >= rows) continue;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= outer) continue;
      const T v = (T)acc[i][j] * (a_scale[m] * b_scale[n]);
      y[m * outer + n] = bias ? v + bias[n] : v;
    }
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" {

int tg_int8_quantize_rows(int dtype, const void* x, int64_t rows, int64_t inner, int8_t* q,
                          int64_t ld, void* scales, void* stream) {
  TG_CHECK_ARG(rows >= 0 && inner >= 0 && ld >= inner, "int8_quantize_rows: bad sizes");
  if (rows == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    quantize_rows_kernel<T><<<grid_for(rows, 1), kThreads, 0, s>>>((const T*)x, rows, inner, q,
                                                                  ld, (T*)scales);
    return check_launch("int8_quantize_rows");
  });
}

size_t tg_int8_linear_scratch_bytes(int dtype, int64_t rows, int64_t inner, int64_t outer) {
  (void)outer;
  const size_t es = dtype == TG_F64 ? 8 : 4;
  if (rows <= 0 || inner < 0) return 16;
  return (size_t)(rows * padded(inner) + 255) / 256 * 256 + (size_t)rows * es + 256;
}

int tg_int8_linear(int dtype, const void* x, int64_t rows, int64_t inner, const int8_t* weight,
                   int64_t ld, const void* scales, const void* bias, void* y, int64_t outer,
                   void* scratch, void* stream) {
  TG_CHECK_ARG(rows >= 0 && inner > 0 && outer >= 0 && ld % 16 == 0 && ld >= inner,
               "int8_linear: rows %lld, inner %lld, outer %lld, weight rows of %lld bytes",
               (long long)rows, (long long)inner, (long long)outer, (long long)ld);
  if (inner > kMaxInner)
    return set_error(TG_ERR_UNSUPPORTED, "int8_linear: inner %lld (at most %lld, so that the "
                     "integer sums fit 32 bits)", (long long)inner, (long long)kMaxInner);
  if (rows == 0 || outer == 0) return TG_OK;
  TG_CHECK_ARG(scratch && aligned16(scratch) && aligned16(weight),
               "int8_linear: scratch and weight start on 16-byte boundaries");
  cudaStream_t s = as_stream(stream);
  const int64_t k = padded(inner);
  int8_t* q = reinterpret_cast<int8_t*>(scratch);
  uint8_t* after = reinterpret_cast<uint8_t*>(scratch) + (rows * k + 255) / 256 * 256;
  const int rc = tg_int8_quantize_rows(dtype, x, rows, inner, q, k, after, stream);
  if (rc) return rc;
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    TG_CHECK_ARG((rows + 63) / 64 <= 65535, "int8_linear: too many rows");
    const dim3 grid((unsigned)((outer + 63) / 64), (unsigned)((rows + 63) / 64));
    int8_tile_kernel<T><<<grid, kThreads, 0, s>>>(q, weight, k, ld, (const T*)after,
                                                  (const T*)scales, (const T*)bias, (T*)y, rows,
                                                  outer);
    return check_launch("int8_linear");
  });
}

}  // extern "C"
