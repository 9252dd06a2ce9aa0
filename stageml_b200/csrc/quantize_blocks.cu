// e4m3 quantization with one fp32 scale per 128 values of a row (activations) or per
// 128 x 128 tile (weights):
//   scale = max|x| / 448 over the block (1 where that is 0),  q = e4m3(x / scale),
// correctly rounded division, round-to-nearest-even, saturated to +-448. A NaN or an
// infinity in a block reaches the scale (the maximum is taken on the bit patterns of
// |x|, in which NaN > infinity > every number), so it is never hidden.
//
// One pass: a block's values stay in registers between the maximum and the encoding.
// Rows: 8 or 16 lanes per block, the maximum by shuffles. Tiles: one CTA per tile, 64
// values per thread.
// Bound: HBM (2 or 4 bytes read and 1 written per value).
#include "block_codes.cuh"
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

// 8 values of one row at columns [c, c + 8), zeros past the end. VEC: cols % 8 == 0
// and the rows are aligned for 16-byte loads.
template <typename T, bool VEC>
__device__ __forceinline__ void load_cols(const T* row, int64_t c, int64_t cols, Vals8<T>& v) {
  if (VEC && c < cols) {
    v.load(row + c);
  } else {
    v.zero();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) v.set(i, row[c + i]);
  }
}

// The largest magnitude (bits) over the 16 lanes of a block.
__device__ __forceinline__ uint32_t block_max(uint32_t m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

template <bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* row, int64_t c, int64_t cols, uint2 u) {
  if (VEC) {
    if (c < cols) *reinterpret_cast<uint2*>(row + c) = u;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = (uint8_t)((i < 4 ? u.x : u.y) >> (8 * (i & 3)));
  }
}

// Rows of whole blocks, in place: block u of the flattened tensor starts at 128 u and no row
// index is needed. 8 lanes per block, 16 values each: the scale and the shuffles, which every
// lane pays for per block, weigh half of what they do with 16 lanes (8192 x 4096 bf16 values:
// 26.6 us with 16 lanes, 21 with 8, 4.8 TB/s; instructions bound the former, not HBM). All
// blocks of a round are loaded before the first is encoded.
constexpr int kFlat = 2;
template <typename T>
__global__ void __launch_bounds__(256) quantize_block_flat_kernel(const T* __restrict__ x, int64_t units,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  const int sub = threadIdx.x & 7;
  const int64_t step = (int64_t)gridDim.x * 32;
  for (int64_t u0 = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3); u0 - (threadIdx.x >> 3) < units; u0 += step * kFlat) {
    Vals8<T> v[kFlat][2];
#pragma unroll
    for (int i = 0; i < kFlat; ++i) {
      const int64_t u = u0 + i * step;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (u < units)
          v[i][h].load(x + u * 128 + sub * 16 + 8 * h);
        else
          v[i][h].zero();
      }
    }
#pragma unroll
    for (int i = 0; i < kFlat; ++i) {
      const int64_t u = u0 + i * step;
      uint32_t m = max(v[i][0].amax(), v[i][1].amax());
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (u >= units) continue;
      const BlockScale s(m);
      const uint2 lo = v[i][0].encode(s), hi = v[i][1].encode(s);
      *reinterpret_cast<uint4*>(q + u * 128 + sub * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
      if (sub == 0) scale[u] = s.s;
    }
  }
}

// Other rows, or rows that are written to other places (a MoE plan's): unit u is block u % nb of
// row u / nb, 16 lanes per block, kUnits blocks per half-warp and round.
constexpr int kUnits = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_block_rows_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                                  const int32_t* __restrict__ out_row, int slots,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  const uint32_t nb = (uint32_t)((cols + 127) / 128);
  const int64_t units = rows * nb;
  const int sub = threadIdx.x & 15, half = threadIdx.x >> 4;
  // unit i of a round: 16 neighbouring units per CTA, then the next 16
  const int64_t step = (int64_t)gridDim.x * 16;
  for (int64_t u0 = (int64_t)blockIdx.x * 16; u0 < units; u0 += step * kUnits) {
    Vals8<T> v[kUnits];
    uint32_t row[kUnits], blk[kUnits];  // the column, 128 blk + 8 sub, can pass 32 bits
    auto col = [&](int i) { return (int64_t)blk[i] * 128 + sub * 8; };
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int64_t u = u0 + i * step + half;
      v[i].zero();
      if (u >= units) continue;
      row[i] = (uint32_t)u / nb;
      blk[i] = (uint32_t)u - row[i] * nb;
      load_cols<T, VEC>(x + row[i] * cols, col(i), cols, v[i]);
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const uint32_t m = block_max(v[i].amax());
      if (u0 + i * step + half >= units) continue;
      const BlockScale s(m);
      const uint2 code = v[i].encode(s);
      if (slots == 0) {
        store_codes<VEC>(q + row[i] * cols, col(i), cols, code);
        if (sub == 0) scale[(int64_t)row[i] * nb + blk[i]] = s.s;
      } else {
        for (int j = 0; j < slots; ++j) {
          const int64_t d = out_row[(int64_t)row[i] * slots + j];
          if (d < 0) continue;
          store_codes<VEC>(q + d * cols, col(i), cols, code);
          if (sub == 0) scale[d * nb + blk[i]] = s.s;
        }
      }
    }
  }
}

// fp32 rows row[p] (skipped when negative) of x, encoded in place of their own row of q; cols % 8 == 0.
__global__ void __launch_bounds__(256) quantize_block_pairs_kernel(const float* __restrict__ x,
                                                                   const int32_t* __restrict__ row, int64_t pairs,
                                                                   int64_t cols, uint8_t* __restrict__ q,
                                                                   float* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  const int64_t nb = (cols + 127) / 128, units = pairs * nb;
  const int64_t u = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int sub = threadIdx.x & 15;
  const int64_t p = u / nb, c = (u - p * nb) * 128 + sub * 8;
  const int64_t r = u < units ? row[p] : -1;
  Vals8<float> v;
  v.zero();
  if (r >= 0) load_cols<float, true>(x + r * cols, c, cols, v);
  const BlockScale s(block_max(v.amax()));
  if (r < 0) return;
  store_codes<true>(q + r * cols, c, cols, v.encode(s));
  if (sub == 0) scale[r * nb + (c >> 7)] = s.s;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_block_tiles_kernel(const T* __restrict__ w, int64_t rows, int64_t cols,
                                                                   uint8_t* __restrict__ q, float* __restrict__ scale) {
  __shared__ uint32_t red[8];
  const int64_t nb = (cols + 127) / 128, rb = (rows + 127) / 128;
  const int64_t tile = blockIdx.x;
  const int64_t b = tile / (rb * nb), t = tile - b * rb * nb;
  const int64_t r0 = t / nb * 128, c = t % nb * 128 + (threadIdx.x & 15) * 8;
  const T* src = w + b * rows * cols;
  uint8_t* dst = q + b * rows * cols;
  Vals8<T> v[8];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = r0 + j * 16 + (threadIdx.x >> 4);
    if (r < rows)
      load_cols<T, VEC>(src + r * cols, c, cols, v[j]);
    else
      v[j].zero();
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, v[j].amax());
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const BlockScale s(m);
  if (threadIdx.x == 0) scale[tile] = s.s;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = r0 + j * 16 + (threadIdx.x >> 4);
    if (r < rows) store_codes<VEC>(dst + r * cols, c, cols, v[j].encode(s));
  }
}

template <typename T>
bool vector_ok(const T* x, const uint8_t* q, int64_t cols) {
  return cols % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 8 == 0;
}

template <typename T>
int run_rows(const void* xv, int64_t rows, int64_t cols, const int32_t* out_row, int slots, uint8_t* q, float* scale,
             cudaStream_t stream, bool pdl) {
  const T* x = static_cast<const T*>(xv);
  const int64_t units = rows * scale_blocks(cols);
  SB_CHECK_ARG(units <= 0x7fffffff, "quantize_e4m3_blocks: more than 2^31 blocks");
  const bool vec = vector_ok(x, q, cols);
  if (slots == 0 && cols % 128 == 0 && vec && reinterpret_cast<uintptr_t>(q) % 16 == 0) {
    const dim3 grid((unsigned)std::min<int64_t>((units + 31) / 32, (int64_t)sm_count() * 32));
    SB_CUDA_CHECK(launch_kernel(quantize_block_flat_kernel<T>, grid, dim3(256), 0, stream, pdl, x, units, q, scale));
  } else {
    const dim3 grid((unsigned)std::min<int64_t>((units + 15) / 16, (int64_t)sm_count() * 32));
    auto kernel = vec ? quantize_block_rows_kernel<T, true> : quantize_block_rows_kernel<T, false>;
    SB_CUDA_CHECK(launch_kernel(kernel, grid, dim3(256), 0, stream, pdl, x, rows, cols, out_row, slots, q, scale));
  }
  count_launch();
  return STAGEML_OK;
}

template <typename T>
int run_tiles(const void* wv, int64_t batch, int64_t rows, int64_t cols, uint8_t* q, float* scale,
              cudaStream_t stream) {
  const T* w = static_cast<const T*>(wv);
  const dim3 grid((unsigned)(batch * scale_blocks(rows) * scale_blocks(cols)));
  if (vector_ok(w, q, cols))
    SB_CUDA_CHECK(
        launch_kernel(quantize_block_tiles_kernel<T, true>, grid, dim3(256), 0, stream, false, w, rows, cols, q, scale));
  else
    SB_CUDA_CHECK(launch_kernel(quantize_block_tiles_kernel<T, false>, grid, dim3(256), 0, stream, false, w, rows, cols,
                                q, scale));
  count_launch();
  return STAGEML_OK;
}

}  // namespace

int launch_quantize_block_rows(const void* x, int dtype, int64_t rows, int64_t cols, const int32_t* out_row, int slots,
                               uint8_t* q, float* scale, cudaStream_t stream, bool pdl) {
  if (rows == 0 || cols == 0) return STAGEML_OK;
  if (dtype == STAGEML_F32) return run_rows<float>(x, rows, cols, out_row, slots, q, scale, stream, pdl);
  if (dtype == STAGEML_BF16) return run_rows<bf16>(x, rows, cols, out_row, slots, q, scale, stream, pdl);
  return run_rows<f16>(x, rows, cols, out_row, slots, q, scale, stream, pdl);
}

int launch_quantize_block_pairs(const float* x, const int32_t* row, int64_t pairs, int64_t cols, uint8_t* q,
                                float* scale, cudaStream_t stream, bool pdl) {
  if (pairs == 0 || cols == 0) return STAGEML_OK;
  const int64_t units = pairs * scale_blocks(cols);
  SB_CUDA_CHECK(launch_kernel(quantize_block_pairs_kernel, dim3((unsigned)((units + 15) / 16)), dim3(256), 0, stream,
                              pdl, x, row, pairs, cols, q, scale));
  count_launch();
  return STAGEML_OK;
}

int launch_quantize_block_tiles(const void* w, int dtype, int64_t batch, int64_t rows, int64_t cols, uint8_t* q,
                                float* scale, cudaStream_t stream) {
  if (batch == 0 || rows == 0 || cols == 0) return STAGEML_OK;
  if (dtype == STAGEML_F32) return run_tiles<float>(w, batch, rows, cols, q, scale, stream);
  if (dtype == STAGEML_BF16) return run_tiles<bf16>(w, batch, rows, cols, q, scale, stream);
  return run_tiles<f16>(w, batch, rows, cols, q, scale, stream);
}

}  // namespace sb
