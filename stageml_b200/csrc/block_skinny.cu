// The block-scaled e4m3 product for a few rows: one token of a decode step, or the expert rows of
// a small batch. It streams the weights, once per 8 or 16 rows of a weight group:
//
//   out[m, n] = row_scale[m] * sum_kb sx[m, kb] * sw[n / 128, kb] * (sum_{k in kb} x[m, k] w[n, k])
//
// Bound: the weights' bytes from HBM. A unit is 16 weight rows (SwiGLU: 16 gate rows and the
// matching 16 up rows) of one group; the eight warps of a CTA take its K blocks in turn and
// add their sums in warp order through shared memory. Per K block a lane loads 16-byte runs
// of weight rows g and g + 8 (g = lane / 4) straight into the A fragments of
// mma.m16n8k32 (e4m3, fp32 sums); the K order inside the block is the lanes' own, the same
// for both operands, so nothing is shuffled. Rows are the N side (8 or 16 of them). The
// matrix unit is far from its limit here; tcgen05 would only add its set-up time: the same
// 1 x 4096 x 4096 product took 18 us on the pair kernel, bound by one accumulator round trip
// per K block, and takes 5 here. Measured over 64 experts of 2048 x 1408 with six per token and two
// shared: 8, 16 and 21 tokens in 113, 149 and 170 us, weights at 3.5 to 4 TB/s. Loading the next unit's
// weights before the sums of this one meet was no faster (111 us, not 114, for 8 tokens at the time) and
// slowed long rows down (8 experts of 4096 x 14336, 8 tokens: 319 us, not 293).
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int kWarps = 8;
constexpr int kUnitRows = 16;

struct SkinnyParams {
  const uint8_t* x;           // [*, K] codes
  const float* x_scale;       // [*, kb]
  const int32_t* row_map;     // plan row -> row of x (null: itself)
  const uint8_t* w;
  const float* w_scale;
  int K, N, kb;
  int w_group_rows, w_blocks;
  int units_n;                // column units per group
  int rows;                   // plain rows; grouped: from the counts
  const int32_t* tile_group;  // grouped: 128-row tile -> group
  const int32_t* group_counts;
  const int32_t* group_offsets;  // first row of each group
  const int32_t* num_tiles;
  int tiles_cap;
  const float* row_scale;
  void* out;                  // [*, N]
};

__device__ __forceinline__ uint4 load_weights(const uint8_t* p, bool valid) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (valid)
    asm volatile("ld.global.nc.L1::no_allocate.L2::128B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
  return v;
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// c = the block's sums of 16 weight rows (lo: row g, hi: row g + 8) with 8 rows of x.
__device__ __forceinline__ void block_mma(float (&c)[4], const uint4 (&lo)[2], const uint4 (&hi)[2], const uint4 (&x)[2]) {
  c[0] = c[1] = c[2] = c[3] = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    mma_e4m3(c, lo[h].x, hi[h].x, lo[h].y, hi[h].y, x[h].x, x[h].y);
    mma_e4m3(c, lo[h].z, hi[h].z, lo[h].w, hi[h].w, x[h].z, x[h].w);
  }
}

// NT: groups of 8 rows. SWIGLU: fp32 h = silu(gate) * up; else OutT.
template <typename OutT, bool SWIGLU, int NT>
__global__ void __launch_bounds__(32 * kWarps, 2) block_skinny_kernel(const SkinnyParams p) {
  constexpr int PARTS = SWIGLU ? 2 : 1;
  __shared__ float red[kWarps][PARTS][NT * 8][kUnitRows + 1];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tiles = p.tile_group ? min(p.tiles_cap, *p.num_tiles) : 1;
  const int units = tiles * p.units_n;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int tile = u / p.units_n, n0 = (u - tile * p.units_n) * kUnitRows;
    const int group = p.tile_group ? p.tile_group[tile] : 0;
    const int all_rows =
        p.tile_group ? min(128, p.group_counts[group] - (tile * 128 - p.group_offsets[group])) : p.rows;
    for (int first = 0; first < all_rows; first += NT * 8) {
    const int rows = min(all_rows - first, NT * 8);
    const int64_t row0 = (int64_t)tile * 128 + first;
    // x rows of this lane's column (row 8 j + g) for the fragments, and of its sums (8 j + 2 t, + 1)
    const uint8_t* x[NT];
    const float* sx[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      auto source = [&](int r) { return p.row_map ? (int64_t)p.row_map[row0 + r] : row0 + r; };
      x[j] = 8 * j + g < rows ? p.x + source(8 * j + g) * p.K + 16 * t : nullptr;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        sx[j][i] = 8 * j + 2 * t + i < rows ? p.x_scale + source(8 * j + 2 * t + i) * p.kb : nullptr;
    }
    const uint8_t* w[PARTS][2];
    const float* sw[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      const int n = n0 + q * p.N;  // the up rows follow the N gate rows
      sw[q] = p.w_scale + ((int64_t)group * p.w_blocks + (n >> 7)) * p.kb;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[q][i] = n0 + g + 8 * i < p.N ? p.w + ((int64_t)group * p.w_group_rows + n + g + 8 * i) * p.K + 16 * t : nullptr;
    }
    float acc[PARTS][NT][4];
#pragma unroll
    for (int q = 0; q < PARTS; ++q)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[q][j][i] = 0.f;
    constexpr int UNROLL = 4 / (PARTS * NT);  // K blocks loaded at once: 64 registers of weights
    for (int kb0 = warp; kb0 < p.kb; kb0 += kWarps * UNROLL) {
      uint4 wv[UNROLL][PARTS][2][2];
      // all weight loads of the round first
#pragma unroll
      for (int r = 0; r < UNROLL; ++r) {
        const int k = (kb0 + r * kWarps) * 128;
#pragma unroll
        for (int q = 0; q < PARTS; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              wv[r][q][i][h] = load_weights(w[q][i] + k + 64 * h, w[q][i] && k + 64 * h + 16 * t < p.K);
      }
#pragma unroll
      for (int r = 0; r < UNROLL; ++r) {
        const int kb = kb0 + r * kWarps, k = kb * 128;
        if (kb >= p.kb) break;
        float s[PARTS];
#pragma unroll
        for (int q = 0; q < PARTS; ++q) s[q] = __ldg(sw[q] + kb);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint4 xv[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            xv[h] = x[j] && k + 64 * h + 16 * t < p.K ? __ldg(reinterpret_cast<const uint4*>(x[j] + k + 64 * h))
                                                       : make_uint4(0, 0, 0, 0);
          const float s0 = sx[j][0] ? __ldg(sx[j][0] + kb) : 0.f, s1 = sx[j][1] ? __ldg(sx[j][1] + kb) : 0.f;
#pragma unroll
          for (int q = 0; q < PARTS; ++q) {
            float c[4];
            block_mma(c, wv[r][q][0], wv[r][q][1], xv);
            acc[q][j][0] = fmaf(s0 * s[q], c[0], acc[q][j][0]);
            acc[q][j][1] = fmaf(s1 * s[q], c[1], acc[q][j][1]);
            acc[q][j][2] = fmaf(s0 * s[q], c[2], acc[q][j][2]);
            acc[q][j][3] = fmaf(s1 * s[q], c[3], acc[q][j][3]);
          }
        }
      }
    }
#pragma unroll
    for (int q = 0; q < PARTS; ++q)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][q][8 * j + 2 * t + (i & 1)][g + 8 * (i >> 1)] = acc[q][j][i];
    __syncthreads();
    for (int e = threadIdx.x; e < NT * 8 * kUnitRows; e += 32 * kWarps) {
      const int r = e / kUnitRows, c = e % kUnitRows;
      if (r < rows && n0 + c < p.N) {
        float v[PARTS];
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
          v[q] = 0.f;
#pragma unroll
          for (int i = 0; i < kWarps; ++i) v[q] += red[i][q][r][c];
        }
        const int64_t row = row0 + r;
        if (SWIGLU)
          static_cast<float*>(p.out)[row * p.N + n0 + c] = v[0] / (1.f + __expf(-v[0])) * v[PARTS - 1];
        else
          static_cast<OutT*>(p.out)[row * p.N + n0 + c] = from_f32<OutT>(p.row_scale ? v[0] * p.row_scale[row] : v[0]);
      }
    }
    __syncthreads();  // the next unit writes the sums again
    }
  }
}

template <typename OutT, bool SWIGLU, int NT>
int run(const SkinnyParams& p, int64_t units, bool pdl, cudaStream_t stream) {
  const int grid = (int)std::min<int64_t>(units, (int64_t)sm_count() * 2);
  SB_CUDA_CHECK(launch_kernel(block_skinny_kernel<OutT, SWIGLU, NT>, dim3((unsigned)grid), dim3(32 * kWarps), 0, stream,
                              pdl, p));
  count_launch();
  return STAGEML_OK;
}

template <typename OutT, bool SWIGLU>
int run_rows(const SkinnyParams& p, int max_rows, int64_t units, bool pdl, cudaStream_t stream) {
  return max_rows <= 8 ? run<OutT, SWIGLU, 1>(p, units, pdl, stream) : run<OutT, SWIGLU, 2>(p, units, pdl, stream);
}

}  // namespace

int launch_block_skinny(const BlockGemmLaunch& g, const BlockSkinny& s, cudaStream_t stream) {
  if (g.a_rows == 0 || g.N == 0) return STAGEML_OK;
  SkinnyParams p{};
  p.x = g.a;
  p.x_scale = g.a_scale;
  p.row_map = s.row_map;
  p.w = g.b;
  p.w_scale = g.b_scale;
  p.K = g.K;
  p.N = g.N;
  p.kb = (int)scale_blocks(g.K);
  p.w_group_rows = g.swiglu ? 2 * g.N : g.N;
  p.w_blocks = (int)scale_blocks(p.w_group_rows);
  p.units_n = (g.N + kUnitRows - 1) / kUnitRows;
  p.rows = s.max_rows;
  p.tile_group = s.tile_group;
  p.group_counts = g.group_counts;
  p.group_offsets = g.group_offsets;
  p.num_tiles = s.num_tiles;
  p.tiles_cap = s.tiles_cap;
  p.row_scale = g.row_scale;
  p.out = g.out;
  const int64_t units = (int64_t)(s.tile_group ? s.tiles_cap : 1) * p.units_n;
  SB_CHECK_ARG(units <= 0x7fffffff, "block_skinny: too many units");
  if (g.swiglu) return run_rows<float, true>(p, s.max_rows, units, g.pdl, stream);
  if (g.out_dtype == STAGEML_F32) return run_rows<float, false>(p, s.max_rows, units, g.pdl, stream);
  if (g.out_dtype == STAGEML_BF16) return run_rows<bf16, false>(p, s.max_rows, units, g.pdl, stream);
  return run_rows<f16, false>(p, s.max_rows, units, g.pdl, stream);
}

}  // namespace sb
