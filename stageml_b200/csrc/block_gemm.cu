// e4m3 x e4m3 matrix product with one fp32 scale per 128 values of K (and per 128
// output columns for the weights), plain or grouped by expert:
//
//   out[r, n] = sum_kb sa[r, kb] * sb[n / 128, kb] * (sum_{k in block kb} a[r, k] * b[n, k])
//
// The inner sum of one K block runs on the tensor cores (tcgen05.mma kind::f8f6f4,
// four K = 32 steps into a fresh fp32 accumulator in TMEM); eight warps then read it,
// multiply by the block's scale and add it to the tile's sums in their registers.
// Two TMEM accumulators alternate, so the next block's MMAs run during that read.
//
// Tile: 128 rows x 256 columns per CTA, persistent CTAs. Warp 0: TMA producer, warp 1:
// TMEM allocation and MMA issue, warps 2..9: scaling and epilogue (warp w owns TMEM
// lanes 32 * (w % 4) and half of the columns, 128 fp32 sums per thread).
//
// SwiGLU: the tile's columns are 128 gate rows and the matching 128 up rows of B; the
// epilogue forms h = silu(gate) * up in fp32 and writes it as e4m3 codes with one scale
// per (row, 128 columns), the next product's operand, so h never exists in 16 bits.
#include "block_fp8.h"
#include "common.cuh"
#include "grouped_gemm.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int BK = 128;                  // e4m3 values = one 128-byte swizzle row = one scale block
constexpr int A_BYTES = BM * BK;         // 16 KB
constexpr int B_BYTES = BN * BK;         // 32 KB
constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int STAGES = 4;
constexpr int THREADS = 320;
constexpr int MATH_WARPS = 8;
constexpr int TMEM_COLS = 512;           // two 256-column accumulators
constexpr int kBandTiles = 16;           // plain rows: row tiles that share a pass over the columns
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + 256 /*barriers*/ + 4 * BM * 4 /*row maxima*/;

struct Params {
  int K, N, kb;                 // kb = ceil(K / 128)
  int b_group_rows, b_blocks;   // rows and 128-row scale blocks of one weight group
  int n_tiles;
  const float* a_scale;
  const float* b_scale;
  const int32_t* tile_group;
  const int32_t* group_offsets;
  const int32_t* num_tiles_dev;
  int tiles_cap;
  int64_t rows;
  const float* row_scale;
  void* out;
  uint8_t* q_out;
  float* q_scale;
  int32_t* status;
};

__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of kind::f8f6f4: f32 accumulator, both operands e4m3 (format 0), K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

struct Unit {
  int m, n, group;
};

// Unit u -> (row tile, column tile). All column tiles of a weight group's row tiles (or of
// a band of plain row tiles) come before the next group, row tiles fastest, so that the
// CTAs at work at one time share weight tiles and the group's rows stay in L2.
__device__ __forceinline__ Unit unit_of(const Params& p, int u, int tiles) {
  Unit w;
  int first, cnt;
  if (p.tile_group) {
    w.group = p.tile_group[u / p.n_tiles];
    first = p.group_offsets[w.group] / BM;
    cnt = p.group_offsets[w.group + 1] / BM - first;
  } else {
    w.group = 0;
    first = u / (p.n_tiles * kBandTiles) * kBandTiles;
    cnt = min(kBandTiles, tiles - first);
  }
  const int local = u - first * p.n_tiles;
  w.n = local / cnt;
  w.m = first + local - w.n * cnt;
  return w;
}

template <typename T>
__device__ __forceinline__ void store_row16(T* dst, const float* v, int valid, bool vec) {
  if (vec && valid >= 16) {
    if (sizeof(T) == 2) {
      float lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) lo[i] = v[i], hi[i] = v[8 + i];
      reinterpret_cast<uint4*>(dst)[0] = pack8<T>(lo);
      reinterpret_cast<uint4*>(dst)[1] = pack8<T>(hi);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < valid) dst[i] = from_f32<T>(v[i]);
  }
}
template <>
__device__ __forceinline__ void store_row16<float>(float* dst, const float* v, int valid, bool vec) {
  if (vec && valid >= 16) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<float4*>(dst)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i < valid) dst[i] = v[i];
  }
}

// OutT: output element (plain); SWIGLU writes codes and ignores it.
template <typename OutT, bool SWIGLU>
__global__ void __launch_bounds__(THREADS, 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                      const Params p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 6);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* row_max = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(bars) + 256);  // [2][2][128]
  auto full_bar = [&](int s) { return smem_u32(&bars[s]); };
  auto empty_bar = [&](int s) { return smem_u32(&bars[STAGES + s]); };
  auto tfull_bar = [&](int i) { return smem_u32(&bars[2 * STAGES + i]); };
  auto tempty_bar = [&](int i) { return smem_u32(&bars[2 * STAGES + 2 + i]); };
  const uint32_t drain_bar = smem_u32(&bars[2 * STAGES + 4]);
  const uint32_t max_bar = smem_u32(&bars[2 * STAGES + 5]);  // the row maxima of a SwiGLU tile are written
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull_bar(i), 1);
      mbar_init(tempty_bar(i), MATH_WARPS);
    }
    mbar_init(drain_bar, 1);
    mbar_init(max_bar, MATH_WARPS);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  volatile int never_abort = 0;

  int tiles = p.tiles_cap;
  if (p.num_tiles_dev) tiles = min(tiles, *p.num_tiles_dev);
  const int units = tiles * p.n_tiles;

  if (threadIdx.x == 0) {
    // ------------------------------------------------------------ producer
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
    const uint64_t pol_a = l2_policy_evict_last(), pol_b = l2_policy_evict_normal();
    const uint32_t base = smem_u32(smem);
    int last_phase[STAGES];
    for (int s = 0; s < STAGES; ++s) last_phase[s] = -1;
    uint32_t it = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
      const Unit w = unit_of(p, u, tiles);
      const int n0 = w.n * (SWIGLU ? 128 : BN);
      const int b0 = w.group * p.b_group_rows + n0;
      const int b1 = SWIGLU ? b0 + p.N : b0 + 128;
      for (int kb = 0; kb < p.kb; ++kb, ++it) {
        const int s = it % STAGES;
        const uint32_t ph = (it / STAGES) & 1;
        if (!mbar_wait(empty_bar(s), ph ^ 1, abort_flag, p.status, kDefaultWaitNs, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        const uint32_t sa = base + s * STAGE_BYTES;
        mbar_arrive_expect_tx(full_bar(s), STAGE_BYTES);
        tma_load_2d(sa, &tm_a, full_bar(s), kb * BK, w.m * BM, pol_a);
        tma_load_2d(sa + A_BYTES, &tm_b, full_bar(s), kb * BK, b0, pol_b);
        tma_load_2d(sa + A_BYTES + B_BYTES / 2, &tm_b, full_bar(s), kb * BK, b1, pol_b);
        last_phase[s] = (int)ph;
      }
    }
    if (!ok) {  // let the copies in flight land before the CTA leaves
      for (int s = 0; s < STAGES; ++s)
        if (last_phase[s] >= 0)
          mbar_wait(full_bar(s), (uint32_t)last_phase[s], &never_abort, p.status, 200000000ull, kDevTimeoutDrain);
    }
  } else if (threadIdx.x == 32) {
    // ------------------------------------------------------------ MMA issuer
    constexpr uint32_t idesc = idesc_e4m3(BM, BN);
    const uint32_t base = smem_u32(smem);
    uint32_t it = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
      for (int kb = 0; kb < p.kb; ++kb, ++it) {
        const int s = it % STAGES, acc = it & 1;
        if (!mbar_wait(tempty_bar(acc), ((it >> 1) & 1) ^ 1, abort_flag, p.status, kDefaultWaitNs, kDevTimeoutMma) ||
            !mbar_wait(full_bar(s), (it / STAGES) & 1, abort_flag, p.status, kDefaultWaitNs, kDevTimeoutMma)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint64_t ad = smem_desc_sw128(base + s * STAGE_BYTES);
        const uint64_t bd = smem_desc_sw128(base + s * STAGE_BYTES + A_BYTES);
#pragma unroll
        for (int k = 0; k < BK / 32; ++k) mma_f8(tmem_base + acc * BN, ad + 2 * k, bd + 2 * k, idesc, k > 0 ? 1u : 0u);
        tc_commit(empty_bar(s));
        tc_commit(tfull_bar(acc));
      }
    }
    // every MMA has stopped reading shared memory before the CTA leaves
    tc_commit(drain_bar);
    mbar_wait(drain_bar, 0, &never_abort, p.status, 1000000000ull, kDevTimeoutDrain);
  } else if (warp >= 2) {
    // ------------------------------------------------------------ scaling and epilogue
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const int row_in_tile = quarter * 32 + lane;
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16);
    // TMEM column of this thread's 16-column chunk c. Plain: columns [128 half, 128 half + 128).
    // SwiGLU: chunks 0-3 gate columns [64 half, +64), chunks 4-7 the same up columns.
    auto col_of = [&](int c) { return SWIGLU ? (c & 4) * 32 + 64 * half + 16 * (c & 3) : 128 * half + 16 * c; };
    const bool vec = p.N % (16 / (int)sizeof(OutT)) == 0;
    uint32_t it = 0, tile = 0;
    bool ok = true;
    for (int u = blockIdx.x; ok && u < units; u += gridDim.x, ++tile) {
      const Unit w = unit_of(p, u, tiles);
      const int64_t row = (int64_t)w.m * BM + row_in_tile;
      const bool row_ok = row < p.rows;
      const float* sa = p.a_scale + (row_ok ? row : 0) * p.kb;
      // weight scales: one per tile half (plain), gate and up (SwiGLU). The up rows start at
      // N inside the group, so a tile's up columns can straddle two 128-row scale blocks:
      // columns below `cut` take the first, the others the second (N % 16 == 0).
      const float *sb0, *sb1, *sb2;
      int cut = 128;
      {
        const float* g = p.b_scale + (int64_t)w.group * p.b_blocks * p.kb;
        if (SWIGLU) {
          const int up = p.N + w.n * 128;
          cut = 128 - (up & 127);
          sb0 = g + (int64_t)w.n * p.kb;
          sb1 = g + (int64_t)min(up >> 7, p.b_blocks - 1) * p.kb;
          sb2 = g + (int64_t)min((up >> 7) + 1, p.b_blocks - 1) * p.kb;
        } else {
          sb0 = sb1 = sb2 = g + (int64_t)min(2 * w.n + half, p.b_blocks - 1) * p.kb;
        }
      }
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      for (int kb = 0; kb < p.kb; ++kb, ++it) {
        const float xa = row_ok ? __ldg(sa + kb) : 0.f;
        const float s0 = xa * __ldg(sb0 + kb);
        float s1 = s0, s2 = s0;
        if (SWIGLU) {
          s1 = xa * __ldg(sb1 + kb);
          s2 = xa * __ldg(sb2 + kb);
        }
        const int buf = it & 1;
        // the whole warp stays or leaves: tcgen05.ld is warp-collective
        ok = __all_sync(0xffffffffu, mbar_wait(tfull_bar(buf), (it >> 1) & 1, abort_flag, p.status, kDefaultWaitNs,
                                               kDevTimeoutEpilogue));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t t[16];
          tmem_ld_x16(t_lane + buf * BN + col_of(c), t);
          tmem_wait_ld();
          const float s = SWIGLU && c >= 4 ? (64 * half + 16 * (c - 4) < cut ? s1 : s2) : s0;
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[16 * c + i] = fmaf(s, __uint_as_float(t[i]), acc[16 * c + i]);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(tempty_bar(buf));
      }
      if (!ok) break;
      if (SWIGLU) {
        const int n0 = w.n * 128 + 64 * half;
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          acc[i] = n0 + i < p.N ? silu_f32(acc[i]) * acc[64 + i] : 0.f;
          m = max(m, __float_as_uint(acc[i]) & 0x7fffffffu);
        }
        // the row's maximum over both halves; two buffers, so that one barrier per tile is enough
        // (a warp writes a buffer again only after every warp has read it and come to the next tile)
        uint32_t* mine = row_max + (tile & 1) * 2 * BM;
        mine[half * BM + row_in_tile] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(max_bar);
        ok = __all_sync(0xffffffffu, mbar_wait(max_bar, tile & 1, abort_flag, p.status, kDefaultWaitNs,
                                               kDevTimeoutEpilogue));
        if (!ok) break;
        m = max(m, mine[(half ^ 1) * BM + row_in_tile]);
        float s = __uint_as_float(m) / 448.0f;
        s = s == 0.f ? 1.f : s;
        if (row_ok) {
          uint8_t* q = p.q_out + row * p.N + n0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if (n0 + 16 * c < p.N) {  // N % 16 == 0: a chunk is inside or outside
              uint32_t v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float* f = acc + 16 * c + 4 * i;
                const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0] / s, f[1] / s), __NV_SATFINITE, __NV_E4M3);
                const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2] / s, f[3] / s), __NV_SATFINITE, __NV_E4M3);
                v[i] = lo | hi << 16;
              }
              *reinterpret_cast<uint4*>(q + 16 * c) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
          if (half == 0) p.q_scale[row * ((p.N + 127) / 128) + w.n] = s;
        }
      } else if (row_ok) {
        const int n0 = w.n * BN + 128 * half;
        const float rs = p.row_scale ? p.row_scale[row] : 1.f;
        OutT* out = static_cast<OutT*>(p.out) + row * p.N + n0;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int valid = p.N - (n0 + 16 * c);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[16 * c + i] *= rs;
          if (valid > 0) store_row16<OutT>(out + 16 * c, acc + 16 * c, valid, vec);
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <typename OutT, bool SWIGLU>
int run(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int grid, bool pdl, cudaStream_t stream) {
  auto kernel = block_gemm_kernel<OutT, SWIGLU>;
  SB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  SB_CUDA_CHECK(launch_kernel(kernel, dim3((unsigned)grid), dim3(THREADS), SMEM_BYTES, stream, pdl, ta, tb, p));
  count_launch();
  return STAGEML_OK;
}

}  // namespace

int launch_block_gemm(const BlockGemmLaunch& g, cudaStream_t stream) {
  if (g.a_rows == 0 || g.N == 0) return STAGEML_OK;
  Params p{};
  p.K = g.K;
  p.N = g.N;
  p.kb = (int)scale_blocks(g.K);
  p.b_group_rows = g.swiglu ? 2 * g.N : g.N;
  p.b_blocks = (int)scale_blocks(p.b_group_rows);
  p.n_tiles = g.swiglu ? (int)scale_blocks(g.N) : (g.N + BN - 1) / BN;
  p.a_scale = g.a_scale;
  p.b_scale = g.b_scale;
  p.tile_group = g.tile_group;
  p.group_offsets = g.group_offsets;
  p.num_tiles_dev = g.num_tiles_dev;
  p.rows = g.a_rows;
  p.tiles_cap = g.tile_group ? g.tiles_cap : (int)((g.a_rows + BM - 1) / BM);
  p.row_scale = g.row_scale;
  p.out = g.out;
  p.q_out = g.q_out;
  p.q_scale = g.q_scale;
  p.status = g.status;
  CUtensorMap ta, tb;
  SB_TRY(make_tmap_2d(&ta, g.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)g.a_rows, (uint64_t)g.K, (uint64_t)g.K, BM,
                      BK, 128));
  SB_TRY(make_tmap_2d(&tb, g.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)g.groups * p.b_group_rows, (uint64_t)g.K,
                      (uint64_t)g.K, 128, BK, 128));
  const int64_t units = (int64_t)p.tiles_cap * p.n_tiles;
  SB_CHECK_ARG(units <= 0x7fffffff, "block_gemm: too many tiles");
  const int grid = (int)(units < sm_count() ? units : sm_count());
  if (g.swiglu) return run<bf16, true>(ta, tb, p, grid, g.pdl, stream);
  if (g.out_dtype == STAGEML_F32) return run<float, false>(ta, tb, p, grid, g.pdl, stream);
  if (g.out_dtype == STAGEML_BF16) return run<bf16, false>(ta, tb, p, grid, g.pdl, stream);
  return run<f16, false>(ta, tb, p, grid, g.pdl, stream);
}

}  // namespace sb
