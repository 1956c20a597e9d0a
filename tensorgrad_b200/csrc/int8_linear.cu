// Linear layers in 8-bit integers (no reference counterpart; the inference form of
// ops/layers.py:22-62): a scale for each token and each output channel,
//   s_m = max_k |x_mk| * (1 / 127),  q_mk = rint(x_mk / s_m),
//   y_mn = (sum_k q_mk w_nk) (s_m s_n) + bias_n,
// the sums exact in 32-bit integers (at most 127 * 128 * 131072 < 2^31). A row of zeros has scale
// 0 and integers 0; a row with a NaN or an infinity has scale NaN, so its outputs are NaN.
#include "common.cuh"

namespace tg {

// The product on the tensor cores (int8_tc.cu): q (rows, padded inner), float scales and outputs.
int int8_gemm_tc(const int8_t* q, const int8_t* weight, int64_t ld, const float* row_scales,
                 const float* scales, const float* bias, float* y, int64_t rows, int64_t inner,
                 int64_t outer, cudaStream_t stream);

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

// The same by the scale's reciprocal: x * (1 / scale) is off the quotient by less than 2^-15 (two
// roundings at a size of at most 127 in float), so wherever it is not within 2^-13 of a half both
// have the same nearest integer; there, and for scales whose reciprocal may overflow, the
// division decides. 8192 x 4096 values: 59 us with a division each, 31 us with the reciprocal.
template <typename T>
struct Reciprocal {
  T scale, inv;
  __device__ explicit Reciprocal(T s) : scale(s), inv(s > T(1e-30) ? T(1) / s : T(NAN)) {}
  __device__ __forceinline__ int of(T x) const {
    const T q = x * inv, r = rint(q);
    if (fabs(fabs(q - r) - T(0.5)) > T(0.0001220703125)) return (int)r;
    return quantize(x, scale);  // also where inv is NaN: no comparison holds
  }
  // Four values, one test for all: a division anywhere is a matter of one in a thousand.
  __device__ __forceinline__ char4 of4(float4 x) const {
    const float a = x.x * inv, b = x.y * inv, c = x.z * inv, d = x.w * inv;
    const float ra = rint(a), rb = rint(b), rc = rint(c), rd = rint(d);
    const float off = fmaxf(fmaxf(fabsf(a - ra), fabsf(b - rb)), fmaxf(fabsf(c - rc), fabsf(d - rd)));
    if (off < 0.5f - 0.0001220703125f)
      return make_char4((signed char)(int)ra, (signed char)(int)rb, (signed char)(int)rc,
                        (signed char)(int)rd);
    return make_char4((signed char)quantize(x.x, scale), (signed char)quantize(x.y, scale),
                      (signed char)quantize(x.z, scale), (signed char)quantize(x.w, scale));
  }
};

// A row's scale from its largest magnitude, times 1 / 127 as the type rounds it; `odd` is NaN if
// the row has a NaN or an infinity.
template <typename T>
__device__ __forceinline__ T scale_of(T top, T odd) {
  return top * T(1.0 / 127) + odd;
}

// Row scales and integers; integer rows are ld bytes long, zero beyond the row's values.
template <typename T>
__global__ void __launch_bounds__(kThreads)
quantize_rows_kernel(const T* __restrict__ x, int64_t rows, int64_t inner, int8_t* __restrict__ q,
                     int64_t ld, T* __restrict__ scales) {
  __shared__ T sh[32];
  pdl_trigger();
  pdl_wait();
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
    const T scale = scale_of(top, odd);
    const bool live = scale > T(0);
    const Reciprocal<T> by(scale);
    for (int64_t c = threadIdx.x; c < ld; c += kThreads)
      q[r * ld + c] = (int8_t)(live && c < inner ? by.of(a[c]) : 0);
    if (threadIdx.x == 0) scales[r] = scale;
    __syncthreads();
  }
}

// Float rows of 16-byte groups, at most N of them to a thread: one read of the row, which stays
// in registers between its maximum and its integers. HBM-bound: 5 bytes a value.
template <int N>
__global__ void __launch_bounds__(kThreads)
quantize_rows_vec4_kernel(const float4* __restrict__ x, int groups,
                          char4* __restrict__ q, int64_t ld4, float* __restrict__ scales) {
  __shared__ float sh[2][kThreads / 32];
  pdl_trigger();
  pdl_wait();
  const int64_t r = blockIdx.x;
  float4 v[N];
  float top = 0.f, odd = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = threadIdx.x + i * kThreads;
    v[i] = c < groups ? x[r * groups + c] : make_float4(0.f, 0.f, 0.f, 0.f);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    top = fmaxf(top, fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w))));
    // NaN from a NaN or an infinity, else 0.
    odd = fmaf(v[i].x, 0.f, fmaf(v[i].y, 0.f, fmaf(v[i].z, 0.f, fmaf(v[i].w, 0.f, odd))));
  }
  top = warp_max(top);
  odd = warp_sum(odd);
  if ((threadIdx.x & 31) == 0) {
    sh[0][threadIdx.x >> 5] = top;
    sh[1][threadIdx.x >> 5] = odd;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    top = fmaxf(top, sh[0][i]);
    odd += sh[1][i];
  }
  const float scale = scale_of(top, odd);
  const bool live = scale > 0.f;
  const Reciprocal<float> by(scale);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int c = threadIdx.x + i * kThreads;
    if (c >= ld4) continue;
    q[r * ld4 + c] = live ? by.of4(v[i]) : make_char4(0, 0, 0, 0);
  }
  if (threadIdx.x == 0) scales[r] = scale;
}

// Up to R rows of input: every block quantises them into shared memory itself, then its warps
// walk the output channels, CH at a time, each lane with NV 16-byte groups of every one's weights
// in flight and the next ones' behind them; the first are on their way before the input is
// quantised. One launch. What bounds it is reading the weights once, and for small layers the
// chain of launch, input, weights.
template <typename T, int R, int CH, int NV, int FEW>
__global__ void __launch_bounds__(FEW)
few_rows_kernel(const T* __restrict__ x, int rows, int inner, const int8_t* __restrict__ weight,
                int64_t ld, const T* __restrict__ scales, const T* __restrict__ bias,
                T* __restrict__ y, int64_t outer) {
  constexpr int W = FEW / 32, PER = W >= R ? W / R : 1;  // warps to a row
  static_assert(W >= R, "a warp to a row");
  extern __shared__ __align__(16) int8_t xs[];  // [R][padded inner]
  __shared__ T sh[2][W], sx[R];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int k = (inner + 15) / 16 * 16, vecs = k / 16;
  const int chunks = (vecs + 32 * NV - 1) / (32 * NV);
  const int64_t stride = (int64_t)gridDim.x * W * CH;
  int64_t c0 = ((int64_t)blockIdx.x * W + w) * CH;
  auto load = [&](int4 (&to)[CH][NV], int64_t from, int chunk) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = (chunk * NV + i) * 32 + lane;
        to[c][i] = v < vecs && from + c < outer
                       ? __ldg(reinterpret_cast<const int4*>(weight + (from + c) * ld) + v)
                       : int4{};
      }
  };
  int4 wv[CH][NV];
  load(wv, c0, 0);
  {
    const int r = w / PER, t = threadIdx.x - r * PER * 32;
    const T* a = x + (int64_t)r * inner;
    T top = T(0), odd = T(0);
    // Float rows of 16-byte groups go four values at a time.
    const bool quads = sizeof(T) == 4 && inner % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    if (r < rows && quads) {
      const float4* a4 = reinterpret_cast<const float4*>(a);
#pragma unroll 4
      for (int c = t; c < inner / 4; c += PER * 32) {
        const float4 v = a4[c];
        top = fmax(top, (T)fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        odd += (T)fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, v.w * 0.f)));
      }
    } else if (r < rows) {
#pragma unroll 4
      for (int c = t; c < inner; c += PER * 32) {
        const T v = fabs(a[c]);
        top = fmax(top, v);
        odd += v - v;
      }
    }
    top = warp_max(top);
    odd = warp_sum(odd);
    if (lane == 0) {
      sh[0][w] = top;
      sh[1][w] = odd;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      top = fmax(top, sh[0][r * PER + i]);
      odd += sh[1][r * PER + i];
    }
    const T scale = scale_of(top, odd);
    const bool live = r < rows && scale > T(0);
    if (quads) {
      const Reciprocal<float> by((float)scale);
      const float4* a4 = reinterpret_cast<const float4*>(a);
#pragma unroll 4
      for (int c = t; c < k / 4; c += PER * 32)
        reinterpret_cast<char4*>(xs + r * k)[c] =
            live && c < inner / 4 ? by.of4(a4[c]) : make_char4(0, 0, 0, 0);
    } else {
      const Reciprocal<T> by(scale);
#pragma unroll 4
      for (int c = t; c < k; c += PER * 32)
        xs[r * k + c] = (int8_t)(live && c < inner ? by.of(a[c]) : 0);
    }
    if (t == 0) sx[r] = scale;
    __syncthreads();
  }
  const int4* xv = reinterpret_cast<const int4*>(xs);
  int acc[CH][R] = {};
  for (int chunk = 0; c0 < outer;) {
    int4 next[CH][NV];
    const bool last = chunk + 1 == chunks;
    load(next, last ? c0 + stride : c0, last ? 0 : chunk + 1);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = (chunk * NV + i) * 32 + lane;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int4 a = v < vecs ? xv[r * vecs + v] : int4{};
#pragma unroll
        for (int c = 0; c < CH; ++c)
          acc[c][r] = __dp4a(a.x, wv[c][i].x, __dp4a(a.y, wv[c][i].y, __dp4a(a.z, wv[c][i].z,
                      __dp4a(a.w, wv[c][i].w, acc[c][r]))));
      }
    }
    if (last) {
      int mine = 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const int total = __reduce_add_sync(0xffffffffu, acc[c][r]);
          if (lane == r * CH + c) mine = total;
          acc[c][r] = 0;
        }
      const int r = lane / CH;
      const int64_t c = c0 + lane % CH;
      if (lane < R * CH && r < rows && c < outer) {
        const T v = (T)mine * (sx[r] * scales[c]);
        y[r * outer + c] = bias ? v + bias[c] : v;
      }
      c0 += stride;
      chunk = 0;
    } else {
      ++chunk;
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < NV; ++i) wv[c][i] = next[c][i];
  }
}

// A 64 x 64 tile of outputs to a block, 4 x 4 to a thread, 64 bytes of the reduction at a time.
template <typename T>
__global__ void __launch_bounds__(kThreads)
int8_tile_kernel(const int8_t* __restrict__ a, const int8_t* __restrict__ b, int64_t ld,
                 int64_t b_ld, const T* __restrict__ a_scale, const T* __restrict__ b_scale,
                 const T* __restrict__ bias, T* __restrict__ y, int64_t rows, int64_t outer,
                 unsigned tiles_n) {
  __shared__ int as[64][17], bs[64][17];
  const int64_t m0 = (int64_t)(blockIdx.x / tiles_n) * 64;
  const int64_t n0 = (int64_t)(blockIdx.x % tiles_n) * 64;
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

// Shared memory for the rows' integers: what a launch has without asking, less 1 KB for the rest.
constexpr int64_t kFewBytes = 47 * 1024;

// Up to 8 rows take the one-launch kernel, more than 2 of them only below 16384 channels: there its
// multiplications cost more than the tensor cores' second launch (8 rows of 4096 through 4096
// channels 12.2 us against 15.5, 6 of 2048 through 8192 8.2 against 10.5, 8 of 768 through 50304
// 23.2 against 16.9; 2 rows 11.4 against 16.4).
bool takes_few(int64_t rows, int64_t inner, int64_t outer) {
  return rows <= 8 && (rows <= 2 || outer < 16384) &&
         (rows > 4 ? 8 : (rows > 2 ? 4 : rows)) * padded(inner) <= kFewBytes;
}

template <typename T, int R, int CH, int NV>
int launch_few_as(const T* x, int rows, int inner, const int8_t* weight, int64_t ld,
                  const T* scales, const T* bias, T* y, int64_t outer, cudaStream_t s) {
  // Every block quantises the input: short rows in many small blocks, long ones in few large.
  constexpr int FEW = NV > 2 ? 512 : (R <= 4 ? 128 : 256), W = FEW / 32;
  constexpr int64_t MOST = 148 * (NV <= 2 ? 6 : 1);
  const int64_t blocks = (outer + W * CH - 1) / (W * CH);
  const dim3 grid((unsigned)(blocks < MOST ? blocks : MOST));
  TG_CUDA_TRY(launch_pdl(few_rows_kernel<T, R, CH, NV, FEW>, grid, dim3(FEW),
                         (size_t)(R * padded(inner)), s, x, rows, inner, weight, ld, scales, bias,
                         y, outer));
  return check_launch("int8_linear(few rows)");
}

// Channels to a warp at a time: 8 loads in flight if the channels are many enough to give every
// multiprocessor 8 warps all the same.
template <typename T, int R, int NV>
int launch_few_rows(const T* x, int rows, int inner, const int8_t* weight, int64_t ld,
                    const T* scales, const T* bias, T* y, int64_t outer, cudaStream_t s) {
  if constexpr (NV <= 2)
    if (outer >= 4 * 148 * 8)
      return launch_few_as<T, R, 4, NV>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  if constexpr (NV <= 4)
    if (outer >= 2 * 148 * 8)
      return launch_few_as<T, R, 2, NV>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  return launch_few_as<T, R, 1, NV>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
}

template <typename T, int R>
int launch_few_inner(const T* x, int rows, int inner, const int8_t* weight, int64_t ld,
                     const T* scales, const T* bias, T* y, int64_t outer, cudaStream_t s) {
  if (inner <= 1024)
    return launch_few_rows<T, R, 2>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  if (inner <= 2048)
    return launch_few_rows<T, R, 4>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  return launch_few_rows<T, R, 8>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
}

template <typename T>
int launch_few(const T* x, int rows, int inner, const int8_t* weight, int64_t ld, const T* scales,
               const T* bias, T* y, int64_t outer, cudaStream_t s) {
  if (rows == 1) return launch_few_inner<T, 1>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  if (rows == 2) return launch_few_inner<T, 2>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  if (rows <= 4) return launch_few_inner<T, 4>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
  return launch_few_inner<T, 8>(x, rows, inner, weight, ld, scales, bias, y, outer, s);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace tg

using namespace tg;

extern "C" {

int tg_int8_quantize_rows(int dtype, const void* x, int64_t rows, int64_t inner, int8_t* q,
                          int64_t ld, void* scales, void* stream) {
  TG_CHECK_ARG(rows >= 0 && rows <= INT32_MAX && inner >= 0 && ld >= inner,
               "int8_quantize_rows: bad sizes");
  if (rows == 0) return TG_OK;
  cudaStream_t s = as_stream(stream);
  const dim3 grid(grid_for(rows, 1));
  if (dtype == TG_F32 && inner % 4 == 0 && ld % 4 == 0 && ld - inner < 16 && ld <= 8192 &&
      aligned16(x) && (reinterpret_cast<uintptr_t>(q) & 3) == 0) {
    const int groups = (int)(inner / 4);
    const int64_t ld4 = ld / 4;
    auto go = [&](auto kernel) {
      launch_pdl(kernel, dim3((unsigned)rows), dim3(kThreads), 0, s, (const float4*)x, groups,
                 (char4*)q, ld4, (float*)scales);
      return check_launch("int8_quantize_rows");
    };
    if (ld4 <= kThreads) return go(quantize_rows_vec4_kernel<1>);
    if (ld4 <= 2 * kThreads) return go(quantize_rows_vec4_kernel<2>);
    if (ld4 <= 4 * kThreads) return go(quantize_rows_vec4_kernel<4>);
    return go(quantize_rows_vec4_kernel<8>);
  }
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    launch_pdl(quantize_rows_kernel<T>, grid, dim3(kThreads), 0, s, (const T*)x, rows, inner, q,
               ld, (T*)scales);
    return check_launch("int8_quantize_rows");
  });
}

size_t tg_int8_linear_scratch_bytes(int dtype, int64_t rows, int64_t inner, int64_t outer) {
  const size_t es = dtype == TG_F64 ? 8 : 4;
  if (rows <= 0 || inner <= 0 || takes_few(rows, inner, outer)) return 16;
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
  TG_CHECK_ARG(weight && aligned16(weight), "int8_linear: the weight starts on a 16-byte boundary");
  cudaStream_t s = as_stream(stream);
  if (takes_few(rows, inner, outer))
    return TG_DISPATCH_FLOAT(dtype, T, [&] {
      return launch_few<T>((const T*)x, (int)rows, (int)inner, weight, ld, (const T*)scales,
                           (const T*)bias, (T*)y, outer, s);
    });
  TG_CHECK_ARG(scratch && aligned16(scratch), "int8_linear: no scratch");
  const int64_t k = padded(inner);
  int8_t* q = reinterpret_cast<int8_t*>(scratch);
  uint8_t* after = reinterpret_cast<uint8_t*>(scratch) + (rows * k + 255) / 256 * 256;
  const int rc = tg_int8_quantize_rows(dtype, x, rows, inner, q, k, after, stream);
  if (rc) return rc;
  if (dtype == TG_F32)
    return int8_gemm_tc(q, weight, ld, (const float*)after, (const float*)scales,
                        (const float*)bias, (float*)y, rows, inner, outer, s);
  return TG_DISPATCH_FLOAT(dtype, T, [&] {
    const int64_t tiles_n = (outer + 63) / 64, tiles_m = (rows + 63) / 64;
    if (tiles_n > INT32_MAX / tiles_m)  // one axis of tiles: a grid's second one ends at 65535
      return set_error(TG_ERR_UNSUPPORTED, "int8_linear: %lld x %lld outputs", (long long)rows,
                       (long long)outer);
    int8_tile_kernel<T><<<dim3((unsigned)(tiles_m * tiles_n)), kThreads, 0, s>>>(
        q, weight, k, ld, (const T*)after, (const T*)scales, (const T*)bias, (T*)y, rows, outer,
        (unsigned)tiles_n);
    return check_launch("int8_linear");
  });
}

}  // extern "C"
