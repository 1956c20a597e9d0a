// The 8-bit integer product of a linear layer on the tensor cores: y = (q w^T) scaled by row and
// channel, plus a bias, q (rows, k) and w (outer, k) signed bytes with k contiguous, sums exact in
// 32-bit integers (tcgen05.mma kind::i8), fp32 scales and outputs.
//
// One persistent CTA per SM, or a pair of CTAs (cta_group::2) on one 256-row tile; 384 threads:
//   warp 0 (lane 0): TMA producer: k-blocks of 128 bytes of A (128 rows) and of B through a ring
//                    of ST stages, 128-byte swizzle.
//   warp 1 (lane 0): MMA issuer (the pair's even CTA): four 32-byte steps a k-block into one of
//                    two accumulators in tensor memory.
//   warps 4..11    : epilogue, lane = row, two warps per lane quarter (one per half of the
//                    columns): integers from tensor memory, scaled, through 32 x 32 boxes in
//                    shared memory to TMA stores (rows of a multiple of 16 bytes) or plain ones.
// Bytes that shared memory must be fed per product bound it: a 128 x 256 tile needs 384 bytes per
// 32768 products of a k column, a pair's 256 x 256 tile 256 bytes a CTA for the same.
// Every wait is bounded; on expiry the kernel records TG_ERR_TIMEOUT in this unit's status word,
// drains and frees its tensor memory.
#include <initializer_list>

#include "tc_ptx.cuh"

namespace tg {
namespace tc {
namespace {

constexpr int kI8Threads = 384;
constexpr int kBK = 128;  // bytes of k a stage
constexpr int kI8Epi0 = 4, kI8EpiWarps = 8;
constexpr uint32_t kI8Box = 32 * 32 * 4;
constexpr int kGroupM = 16;  // row tiles that share their column tiles' loads through the L2

// Set only by tg_int8_set_wait_test: the producers then issue no load, so the first wait for one
// runs out and the kernel's abort-and-drain path runs with nothing in flight.
__device__ int g_withhold_loads = 0;

template <int BN, bool PAIR>
struct I8Layout {
  static constexpr int TILE_M = PAIR ? 256 : 128;
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr uint32_t A_BYTES = 128 * kBK, B_BYTES = B_ROWS * kBK;
  static constexpr uint32_t STAGE = A_BYTES + B_BYTES;
  static constexpr int ST = (int)(196608 / STAGE) < 8 ? (int)(196608 / STAGE) : 8;
  static constexpr uint32_t STAGING = kI8EpiWarps * kI8Box;
  static constexpr uint32_t SMEM = ST * STAGE + STAGING + 1024 + 512;
  static constexpr uint32_t COLS = 2 * BN;  // two accumulators
};

struct I8Args {
  int64_t rows, outer;
  int kblocks, tiles_m, tiles_n;
  int a_rows;  // rows of A a copy brings: 128, or about the product's if it has fewer
  const float* row_scale;
  const float* scale;
  const float* bias;
  float* y;
  int tma_y;
};

// D s32, A and B signed bytes, both K-major.
__host__ __device__ constexpr uint32_t i8_instr(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

template <bool PAIR>
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                       uint32_t idesc, uint32_t accumulate) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tma_load_2d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y)
      : "memory");
}
// The same, counted on a barrier of either CTA of the pair (its cluster address).
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, uint32_t bar,
                                                 int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x,
                                             int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(smem_u32(src)), "r"(x), "r"(y)
      : "memory");
}

// Tile `t`: kGroupM row tiles at a time walk all column tiles, rows fastest.
__device__ __forceinline__ void i8_tile(const I8Args& a, int t, int& m, int& n) {
  const int group = t / (kGroupM * a.tiles_n), first = group * kGroupM;
  const int height = a.tiles_m - first < kGroupM ? a.tiles_m - first : kGroupM;
  const int r = t - group * kGroupM * a.tiles_n;
  m = first + r % height;
  n = r / height;
}

template <int BN, bool PAIR>
__global__ void __launch_bounds__(kI8Threads, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmY, I8Args a) {
  using L = I8Layout<BN, PAIR>;
  constexpr int ST = L::ST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* staging = smem + ST * L::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + L::STAGING);
  uint64_t* empty = full + ST;
  uint64_t* acc_full = empty + ST;    // [2]
  uint64_t* acc_empty = acc_full + 2;  // [2]
  uint64_t* drain = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int unit = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int units = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int tiles = a.tiles_m * a.tiles_n;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], (PAIR ? 2 : 1) * kI8EpiWarps);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if (PAIR) tmem_alloc2(tmem_slot, L::COLS);
    else tmem_alloc(tmem_slot, L::COLS);
  }
  tc_fence_before();
  __syncthreads();
  if (PAIR) cluster_sync();  // both CTAs' barriers exist before any arrival across
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool stop = *(volatile int*)&g_withhold_loads != 0;
      for (int t = unit; t < tiles && !stop; t += units) {
        int m, n;
        i8_tile(a, t, m, n);
        const int m0 = m * L::TILE_M + (int)rank * 128, n0 = n * BN + (int)rank * L::B_ROWS;
        for (int j = 0; j < a.kblocks; ++j, ++it) {
          const int s = it % ST, round = it / ST;
          if (round > 0 && !wait_bar(&empty[s], (round - 1) & 1, abort_flag)) { stop = true; break; }
          uint8_t* st = smem + s * L::STAGE;
          if constexpr (PAIR) {
            // Both CTAs' copies count on the even CTA's barrier.
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * L::STAGE);
            const uint32_t bar = map_to_rank(&full[s], 0);
            tma_load_2d_pair(st, &tmA, bar, j * kBK, m0);
            tma_load_2d_pair(st + L::A_BYTES, &tmB, bar, j * kBK, n0);
          } else {
            mbar_arrive_expect_tx(&full[s], (uint32_t)a.a_rows * kBK + L::B_BYTES);
            tma_load_2d(st, &tmA, &full[s], j * kBK, m0);
            tma_load_2d(st + L::A_BYTES, &tmB, &full[s], j * kBK, n0);
          }
        }
      }
      // The copies in flight land, and the MMAs' last releases of the stages arrive, before the
      // CTA may exit.
      const bool aborted = *abort_flag != 0;
      for (int j = it - ST; j < it; ++j) {
        if (j < 0) continue;
        if (aborted && rank == 0) wait_bar(&full[j % ST], (j / ST) & 1, abort_flag, false);
        else if (!aborted) wait_bar(&empty[j % ST], (j / ST) & 1, abort_flag);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = i8_instr(L::TILE_M, BN);
      int it = 0, tc = 0;
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units, ++tc) {
        const int buf = tc & 1;
        if (tc >= 2 && !wait_bar(&acc_empty[buf], ((tc >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
        tc_fence_after();
        const uint32_t acc = tmem + (uint32_t)(buf * BN);
        for (int j = 0; j < a.kblocks; ++j, ++it) {
          const int s = it % ST;
          const bool landed = PAIR ? wait_bar_cluster(&full[s], (it / ST) & 1, abort_flag)
                                   : wait_bar(&full[s], (it / ST) & 1, abort_flag);
          if (!landed) { ok = false; break; }
          tc_fence_after();
          const uint32_t as = smem_u32(smem + s * L::STAGE), bs = as + L::A_BYTES;
#pragma unroll
          for (int kk = 0; kk < kBK / 32; ++kk)
            mma_i8<PAIR>(acc, smem_desc(as + kk * 32, 16, 1024, 2),
                         smem_desc(bs + kk * 32, 16, 1024, 2), idesc, (j | kk) != 0);
          if (PAIR) mma_commit_pair_both(&empty[s]);
          else mma_commit(&empty[s]);
        }
        if (!ok) break;
        if (PAIR) mma_commit_pair_both(&acc_full[buf]);
        else mma_commit(&acc_full[buf]);
      }
      if (!ok) {
        if (PAIR) mma_commit_pair_local(drain);
        else mma_commit(drain);
        wait_bar(drain, 0, abort_flag, false);
      }
    }
  } else if (warp >= kI8Epi0) {
    const int quarter = warp & 3, half = (warp - kI8Epi0) >> 2;
    const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
    float4* box = reinterpret_cast<float4*>(staging + (warp - kI8Epi0) * kI8Box);
    // 32-column chunks of this warp's half (a 32-wide tile is the first half's).
    constexpr int CHUNKS = BN >= 64 ? BN / 64 : 1;
    int tc = 0;
    for (int t = unit; t < tiles; t += units, ++tc) {
      const int buf = tc & 1;
      int m, n;
      i8_tile(a, t, m, n);
      const int64_t row0 = (int64_t)m * L::TILE_M + rank * 128 + 32 * quarter;
      const int64_t row = row0 + lane;
      const float rs = row < a.rows ? a.row_scale[row] : 0.f;
      if (!__all_sync(0xffffffffu, wait_bar(&acc_full[buf], (tc >> 1) & 1, abort_flag))) break;
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < CHUNKS; ++c) {
        if (BN < 64 && half == 1) {
          if (lane == 0) mbar_arrive(&acc_empty[buf]);
          break;
        }
        const int col = (half * CHUNKS + c) * 32;
        const int64_t n0 = (int64_t)n * BN + col;
        uint32_t r[32];
        tmem_ld32(tmem + lanes + (uint32_t)(buf * BN + col), r);
        if (c == CHUNKS - 1) {  // the accumulator is read: the next tile may take it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (PAIR && rank == 1) mbar_arrive_remote(map_to_rank(&acc_empty[buf], 0));
            else mbar_arrive(&acc_empty[buf]);
          }
        }
        if (n0 >= a.outer || row0 >= a.rows) continue;
        const bool in = n0 + lane < a.outer;
        const float cs = in ? a.scale[n0 + lane] : 0.f;
        const float cb = in && a.bias ? a.bias[n0 + lane] : 0.f;
        if (lane == 0) bulk_wait_read<0>();  // the box's last store has read it
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float s = rs * __shfl_sync(0xffffffffu, cs, 4 * k + i);
            v[i] = (float)(int)r[4 * k + i] * s;
            // One rounding for the product and one for the sum, as without a bias.
            if (a.bias) v[i] = __fadd_rn(v[i], __shfl_sync(0xffffffffu, cb, 4 * k + i));
          }
          box[lane * 8 + (k ^ (lane & 7))] = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (a.tma_y) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmY, box, (int)n0, (int)row0);
            bulk_commit();
          }
        } else {
          __syncwarp();
          const float* flat = reinterpret_cast<const float*>(box);
          for (int i = 0; i < 32 && row0 + i < a.rows; ++i)
            if (in) a.y[(row0 + i) * a.outer + n0 + lane] =
                flat[(i * 8 + ((lane >> 2) ^ (i & 7))) * 4 + (lane & 3)];
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  // Neither CTA leaves while the pair's MMAs may read its shared memory, or the other may arrive
  // on its barriers.
  if (PAIR) cluster_sync();
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc2(tmem, L::COLS);
    else tmem_dealloc(tmem, L::COLS);
  }
}

// Row-major bytes or floats (rows x inner elements, ld bytes to a row), boxes of box_inner
// elements x box_rows, 128-byte swizzle.
int i8_map(CUtensorMap* map, CUtensorMapDataType type, const void* ptr, int64_t inner,
           int64_t rows, int64_t ld, uint32_t box_inner, uint32_t box_rows) {
  EncodeFn enc = get_encode();
  if (!enc) return set_error(TG_ERR_UNSUPPORTED, "int8_linear: cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {box_inner, box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(TG_ERR_UNSUPPORTED, "int8_linear: tensor map encode failed (%d)", (int)r);
  return TG_OK;
}

bool g_i8_launched = false;

template <int BN, bool PAIR>
int launch_i8(const int8_t* q, const int8_t* w, int64_t ld, I8Args a, int64_t k, cudaStream_t st) {
  using L = I8Layout<BN, PAIR>;
  CUtensorMap ma, mb, my;
  int rc;
  // A product of few rows leaves the rest of the tile's A rows as they are in shared memory: the
  // accumulator rows that they make are never read.
  a.a_rows = !PAIR && a.rows < 128 ? (int)((a.rows + 15) / 16 * 16) : 128;
  if ((rc = i8_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, q, k, a.rows, k, kBK, a.a_rows))) return rc;
  if ((rc = i8_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, w, k, a.outer, ld, kBK, L::B_ROWS)))
    return rc;
  a.tma_y = a.outer % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 15) == 0;
  if (a.tma_y) {
    if ((rc = i8_map(&my, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a.y, a.outer, a.rows, a.outer * 4, 32,
                     32)))
      return rc;
  } else {
    my = ma;
  }
  a.tiles_m = (int)((a.rows + L::TILE_M - 1) / L::TILE_M);
  a.tiles_n = (int)((a.outer + BN - 1) / BN);
  auto kernel = int8_gemm_kernel<BN, PAIR>;
  TG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)L::SMEM));
  const int tiles = a.tiles_m * a.tiles_n;
  const int most = PAIR ? sm_count() / 2 : sm_count();
  const int n = tiles < most ? tiles : most;
  g_i8_launched = true;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(PAIR ? 2 * n : n));
  cfg.blockDim = dim3(kI8Threads);
  cfg.dynamicSmemBytes = L::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim = {PAIR ? 2u : 1u, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 2;
  TG_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, ma, mb, my, a));
  return check_launch("int8_linear(tensor cores)");
}

}  // namespace
}  // namespace tc

int int8_gemm_tc(const int8_t* q, const int8_t* weight, int64_t ld, const float* row_scales,
                 const float* scales, const float* bias, float* y, int64_t rows, int64_t inner,
                 int64_t outer, cudaStream_t stream) {
  const int64_t k = (inner + 15) / 16 * 16;
  if (rows >= (int64_t)1 << 31 || outer >= (int64_t)1 << 31 ||
      ((rows + 127) / 128) * ((outer + 31) / 32) >= (int64_t)1 << 30)
    return set_error(TG_ERR_UNSUPPORTED, "int8_linear: %lld x %lld outputs", (long long)rows,
                     (long long)outer);
  tc::I8Args a{};
  a.rows = rows;
  a.outer = outer;
  a.kblocks = (int)((k + tc::kBK - 1) / tc::kBK);
  a.row_scale = row_scales;
  a.scale = scales;
  a.bias = bias;
  a.y = y;
  // What a multiprocessor is fed from the L2 a k-block decides (77 GB/s each, 11.4 TB/s together,
  // measured alike for all widths): (A rows + BN) * 128 bytes a tile and k-block, times the rounds
  // that the tiles take. Narrow tiles win where few would leave multiprocessors empty (512 x 768 x
  // 2304: 64 wide 8.6 us, 128 wide 9.7, 256 wide 11.5), wide ones otherwise (4096 x 768 x 50304:
  // 368, 268 and 255 us). A pair feeds 256 rows to a CTA for a 256-wide tile instead of 384, but
  // costs a round more at its start and end: it wins on long reductions of several rounds (8192 x
  // 4096 x 4096 130 against 142 us; 2048 x 768 x 2304 13.8 against 13.2). Fewer than 96 rows a tile
  // cost as much as 96: a round has its own latency, so 64 wide in 2 rounds beats 32 wide in 3 (16 x
  // 4096 x 12288: 16.3 against 33.7 us, 16 x 768 x 12288: 9.2 against 10.7).
  const int64_t tm = (rows + 127) / 128, sms = tc::sm_count();
  const int64_t pairs = (rows + 255) / 256 * ((outer + 255) / 256);
  if (a.kblocks >= 16 && pairs > sms / 2)
    return tc::launch_i8<256, true>(q, weight, ld, a, k, stream);
  const int64_t a_rows = rows < 128 ? (rows + 15) / 16 * 16 : 128;
  int best = 32;
  int64_t least = INT64_MAX;
  for (const int bn : {32, 64, 128, 256}) {
    const int64_t rounds = (tm * ((outer + bn - 1) / bn) + sms - 1) / sms;
    const int64_t cost = rounds * (a_rows + bn < 96 ? 96 : a_rows + bn);
    if (cost < least) {
      least = cost;
      best = bn;
    }
  }
  switch (best) {
    case 32: return tc::launch_i8<32, false>(q, weight, ld, a, k, stream);
    case 64: return tc::launch_i8<64, false>(q, weight, ld, a, k, stream);
    case 128: return tc::launch_i8<128, false>(q, weight, ld, a, k, stream);
  }
  return tc::launch_i8<256, false>(q, weight, ld, a, k, stream);
}

}  // namespace tg

// The timeout record of the 8-bit integer products (this unit's status word); reset when asked.
// Reads nothing before the first of them.
extern "C" int tg_int8_tc_status(int reset) {
  if (!tg::tc::g_i8_launched) return 0;
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, tg::tc::g_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset && v != 0) {
    const int z = 0;
    cudaMemcpyToSymbol(tg::tc::g_status, &z, sizeof(int));
  }
  return v;
}

// Test support for these bounded waits (no reference counterpart): a wait budget in clock cycles
// (<= 0 restores the default of about two seconds) and, with withhold_loads != 0, producers that
// issue no load. Synchronous; affects later launches of this unit's kernels only.
extern "C" int tg_int8_set_wait_test(int64_t budget_cycles, int withhold_loads) {
  const long long b = budget_cycles > 0 ? (long long)budget_cycles : tg::tc::kTimeoutCycles;
  const int w = withhold_loads ? 1 : 0;
  TG_CUDA_TRY(cudaMemcpyToSymbol(tg::tc::g_wait_budget, &b, sizeof(b)));
  TG_CUDA_TRY(cudaMemcpyToSymbol(tg::tc::g_withhold_loads, &w, sizeof(w)));
  return TG_OK;
}
