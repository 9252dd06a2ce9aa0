// e4m3 quantization with one fp32 scale per 128 values of a row (activations) or per
// 128 x 128 tile (weights):
//   scale = max|x| / 448 over the block (1 where that is 0),  q = e4m3(x / scale),
// correctly rounded division, round-to-nearest-even, saturated to +-448. A NaN or an
// infinity in a block reaches the scale (the maximum is taken on the bit patterns of
// |x|, in which NaN > infinity > every number), so it is never hidden.
//
// One pass: a block's values stay in registers between the maximum and the encoding.
// Rows: 16 lanes per block, 8 values per lane (one 16-byte load for 16-bit inputs), the
// maximum by four shuffles. Tiles: one CTA per tile, 64 values per thread.
// Bound: HBM (2 or 4 bytes read and 1 written per value).
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

// |v| as an integer that orders like |v|, NaN above infinity.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  const float s = __uint_as_float(amax_bits) / 448.0f;
  return s == 0.f ? 1.f : s;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  unpack8<T>(__ldg(reinterpret_cast<const uint4*>(p)), f);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

// 8 values of one row at columns [c, c + 8), zeros past the end. VEC: cols % 8 == 0
// and the rows are aligned for 16-byte loads.
template <typename T, bool VEC>
__device__ __forceinline__ void load_cols(const T* row, int64_t c, int64_t cols, float (&f)[8]) {
  if (VEC && c < cols) {
    load8<T>(row + c, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = c + i < cols ? to_f32<T>(row[c + i]) : 0.f;
  }
}

__device__ __forceinline__ uint2 encode8(const float (&f)[8], float s) {
  uint2 u;
  uint16_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * i] / s, f[2 * i + 1] / s), __NV_SATFINITE, __NV_E4M3);
  u.x = h[0] | (uint32_t)h[1] << 16;
  u.y = h[2] | (uint32_t)h[3] << 16;
  return u;
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

// A half-warp takes kUnits neighbouring blocks of the flattened (row, block) list per round, all
// loaded before the first is encoded.
constexpr int kUnits = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quantize_block_rows_kernel(const T* __restrict__ x, int64_t rows, int64_t cols,
                                                                  const int32_t* __restrict__ out_row, int slots,
                                                                  uint8_t* __restrict__ q, float* __restrict__ scale) {
  pdl_wait();
  pdl_trigger();
  const int64_t nb = (cols + 127) / 128;
  const int64_t units = rows * nb;
  const int sub = threadIdx.x & 15, half = threadIdx.x >> 4;
  const int64_t step = (int64_t)gridDim.x * 16 * kUnits;
  // a warp's two halves go through the same rounds (the shuffles)
  for (int64_t u0 = ((int64_t)blockIdx.x * 16 + (half & ~1)) * kUnits; u0 < units; u0 += step) {
    float f[kUnits][8];
    int64_t row[kUnits];
    int64_t u = u0 + (half & 1) * kUnits;
    int64_t r = u / nb, kb = u - r * nb;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      row[i] = r * nb + kb < units ? r : -1;
      if (row[i] >= 0) {
        load_cols<T, VEC>(x + r * cols, kb * 128 + sub * 8, cols, f[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[i][e] = 0.f;
      }
      if (++kb == nb) kb = 0, ++r;
    }
    r = u / nb, kb = u - r * nb;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) m = max(m, abs_bits(f[i][e]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (row[i] >= 0) {
        const float s = scale_of(m);
        const uint2 code = encode8(f[i], s);
        if (slots == 0) {
          store_codes<VEC>(q + r * cols, kb * 128 + sub * 8, cols, code);
          if (sub == 0) scale[r * nb + kb] = s;
        } else {
          for (int j = 0; j < slots; ++j) {
            const int64_t d = out_row[r * slots + j];
            if (d < 0) continue;
            store_codes<VEC>(q + d * cols, kb * 128 + sub * 8, cols, code);
            if (sub == 0) scale[d * nb + kb] = s;
          }
        }
      }
      if (++kb == nb) kb = 0, ++r;
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
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = 0.f;
  if (r >= 0) load_cols<float, true>(x + r * cols, c, cols, f);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(f[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (r < 0) return;
  const float s = scale_of(m);
  store_codes<true>(q + r * cols, c, cols, encode8(f, s));
  if (sub == 0) scale[r * nb + (c >> 7)] = s;
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
  float f[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = r0 + j * 16 + (threadIdx.x >> 4);
    if (r < rows) {
      load_cols<T, VEC>(src + r * cols, c, cols, f[j]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[j][i] = 0.f;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(f[j][i]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, red[i]);
  const float s = scale_of(m);
  if (threadIdx.x == 0) scale[tile] = s;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int64_t r = r0 + j * 16 + (threadIdx.x >> 4);
    if (r < rows) store_codes<VEC>(dst + r * cols, c, cols, encode8(f[j], s));
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
  const int64_t groups = (rows * scale_blocks(cols) + 16 * kUnits - 1) / (16 * kUnits);
  const dim3 grid((unsigned)std::min<int64_t>(groups, (int64_t)sm_count() * 32));
  auto kernel = vector_ok(x, q, cols) ? quantize_block_rows_kernel<T, true> : quantize_block_rows_kernel<T, false>;
  SB_CUDA_CHECK(launch_kernel(kernel, grid, dim3(256), 0, stream, pdl, x, rows, cols, out_row, slots, q, scale));
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
