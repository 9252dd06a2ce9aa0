// The norms after and before a block, fused with its gate and the residual sum:
//
//   u  = w_post * y * rsqrt(mean(y^2) + eps)      (u = y without a post weight)
//   r' = a r + g u                                 (r' = a r without a block output)
//   z  = w_pre * r' * rsqrt(mean(r'^2) + eps)
//
// r, r' [T, H] in the residual dtype; y, z [T, H] in the block dtype; g per channel [H],
// per token [T] or full [T, H]. All arithmetic is fp32 from the loads to the one rounding
// of each output; z comes from the unrounded r'. z may instead leave as e4m3 codes with
// one scale per 128 columns, the operand of the block-scaled products.
//
// Gradients (dz of z, dr' of r'), with n = r', ^ the normalised value, dn = w_pre dz:
//   d  = dr' + rsqrt_n (dn - n^ mean(dn n^))       dr = a d,  dw_pre = sum_t dz n^
//   dg = d u (summed over what g was broadcast over),  du = g d,  dw_post = sum_t du y^
//   dy = rsqrt_y (w_post du - y^ mean(w_post du y^))
// The statistics are computed again from r and y, which the backward reads anyway, so the
// forward saves nothing.
//
// A row is held in the registers of one CTA (of one warp up to 256 columns) from its load
// to its store, 8 values per 16-byte load, or single values where the width or an address
// is not a multiple of 8 values.
//
// Long batches: persistent CTAs whose next row arrives in shared memory by bulk copies
// (two stages) while the current one is reduced, so HBM stays busy across the row sums.
//
// Weight gradients: with y^ normalised (or y), the post weight and a per-channel gate have
// gradients that are multiples, column by column, of the same sum over tokens
//   S[c] = sum_t s_t d y^,   dw_post = g S (s_t = 1, per-channel g) or S (s_t = g_t or g_tc),
//   dg = w_post S,
// so at most two sums per column (S and dw_pre's) are kept, in the registers of the thread
// that owns the column. Each CTA takes every gridDim-th row and writes its sums once; a second
// kernel adds them in CTA order: no atomics, the same bits on every run. Bound: HBM.
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxH = 16384;  // 512 threads x 32 values
constexpr size_t kMaxRing = 200 * 1024;  // shared memory of a CTA's row ring

template <int VEC, typename T>
__device__ __forceinline__ void load_vals(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    f[0] = to_f32<T>(*p);
  } else if constexpr (sizeof(T) == 2) {
    unpack8<T>(__ldg(reinterpret_cast<const uint4*>(p)), f);
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
}

template <int VEC, typename T>
__device__ __forceinline__ void store_vals(T* p, const float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    *p = from_f32<T>(f[0]);
  } else if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = pack8<T>(f);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}

// A parameter in its own type (fp32, bf16 or f16), at element i.
template <int VEC>
__device__ __forceinline__ void load_param(const void* p, int dtype, int64_t i, float (&f)[VEC]) {
  if (dtype == STAGEML_F32)
    load_vals<VEC>(static_cast<const float*>(p) + i, f);
  else if (dtype == STAGEML_BF16)
    load_vals<VEC>(static_cast<const bf16*>(p) + i, f);
  else
    load_vals<VEC>(static_cast<const f16*>(p) + i, f);
}
__device__ __forceinline__ float load_param1(const void* p, int dtype, int64_t i) {
  float f[1];
  load_param<1>(p, dtype, i, f);
  return f[0];
}
__device__ __forceinline__ void store_param1(void* p, int dtype, int64_t i, float v) {
  if (dtype == STAGEML_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == STAGEML_BF16)
    static_cast<bf16*>(p)[i] = from_f32<bf16>(v);
  else
    static_cast<f16*>(p)[i] = from_f32<f16>(v);
}

template <int VEC>
__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, const float (&f)[VEC]) {
  if (dtype == STAGEML_F32)
    store_vals<VEC>(static_cast<float*>(p) + i, f);
  else if (dtype == STAGEML_BF16)
    store_vals<VEC>(static_cast<bf16*>(p) + i, f);
  else
    store_vals<VEC>(static_cast<f16*>(p) + i, f);
}

// Sum of (a, b) over the row's threads: a warp (WARP) or the CTA. `red` has 64 floats;
// consecutive calls alternate between its halves, so one barrier per call is enough.
template <bool WARP>
__device__ __forceinline__ float2 row_sum(float a, float b, float2* red, int& phase) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if (WARP) return make_float2(a, b);
  float2* buf = red + (phase ^= 1) * 16;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s.x += buf[i].x, s.y += buf[i].y;
  return s;
}

// Values of a row, from global memory or from the row's copy in shared memory.
template <bool SMEM, int VEC, typename T>
__device__ __forceinline__ void row_vals(const T* p, float (&f)[VEC]) {
  if constexpr (!SMEM) {
    load_vals<VEC>(p, f);
  } else if constexpr (sizeof(T) == 2) {
    unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
}

// Two-stage ring of rows in dynamic shared memory, filled by bulk copies. Thread 0 issues
// the copies of row i + 2 once every thread has read row i.
constexpr int kStages = 2;
struct RowRing {
  uint8_t* base;
  uint32_t stage_bytes;
  uint64_t* full;          // [kStages]
  volatile int* abort_flag;
  int32_t* status;

  __device__ void init(uint8_t* smem, uint32_t bytes, uint64_t* bars, int* flag, int32_t* st) {
    base = smem, stage_bytes = bytes, full = bars, abort_flag = flag, status = st;
    if (threadIdx.x == 0) {
      for (int i = 0; i < kStages; ++i) mbar_init(smem_u32(&full[i]), 1);
      *flag = 0;
      fence_barrier_init();
    }
    __syncthreads();
  }
  // The copies of the n-th row of this CTA (thread 0); null sources are left out.
  __device__ void fill(uint32_t n, const void* const (&src)[4], const uint32_t (&bytes)[4]) {
    fence_proxy_async_smem();  // the stage's reads (ordered by the caller's barrier) come first
    const uint32_t bar = smem_u32(&full[n % kStages]);
    uint32_t dst = smem_u32(base) + n % kStages * stage_bytes, total = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) total += src[i] ? bytes[i] : 0;
    mbar_arrive_expect_tx(bar, total);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (src[i]) bulk_load_1d(dst, src[i], bytes[i], bar);
      dst += bytes[i];
    }
  }
  // An expired wait is recorded in the status word; the caller goes on (with wrong values),
  // so that the CTA's barriers still meet.
  __device__ const uint8_t* wait(uint32_t n) {
    mbar_wait(smem_u32(&full[n % kStages]), (n / kStages) & 1, abort_flag, status, kDefaultWaitNs,
              kDevTimeoutProducer);
    return base + n % kStages * stage_bytes;
  }
};

template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING>
__global__ void __launch_bounds__(kMaxThreads) norm_residual_kernel(const stageml_norm_args a, float* z32) {
  extern __shared__ __align__(128) uint8_t row_smem[];
  __shared__ float2 red[32];
  __shared__ uint64_t bars[kStages];
  __shared__ int flag;
  int phase = 0;
  const int nt = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int H = a.H;
  const float inv_h = 1.f / (float)H;
  const uint32_t r_bytes = (uint32_t)H * sizeof(TR), y_bytes = (uint32_t)H * sizeof(TY);
  const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  RowRing ring;
  auto fill = [&](uint32_t n) {
    const int64_t row = first + n * step;
    if (row >= a.T) return;
    const void* src[4] = {static_cast<const TR*>(a.residual) + row * H,
                          a.block_out ? static_cast<const TY*>(a.block_out) + row * H : nullptr, nullptr, nullptr};
    const uint32_t bytes[4] = {r_bytes, y_bytes, 0, 0};
    ring.fill(n, src, bytes);
  };
  if constexpr (RING) {
    ring.init(row_smem, r_bytes + y_bytes, bars, &flag, a.status);
    if (threadIdx.x == 0)
      for (int i = 0; i < kStages; ++i) fill(i);
  }
  uint32_t count = 0;
  for (int64_t row = first; row < a.T; row += step, ++count) {
    const int64_t base = row * H;
    const TR* r_row = static_cast<const TR*>(a.residual) + base;
    const TY* y_row = static_cast<const TY*>(a.block_out) + base;
    if constexpr (RING) {
      const uint8_t* stage = ring.wait(count);
      r_row = reinterpret_cast<const TR*>(stage);
      y_row = reinterpret_cast<const TY*>(stage + r_bytes);
    }
    float n[V][VEC];
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = 0.f;
      if (a.block_out && c < H) row_vals<RING, VEC>(y_row + c, n[v]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sq = fmaf(n[v][i], n[v][i], sq);
    }
    if (a.block_out) {
      float inv = 1.f;
      if (a.post_weight) inv = rsqrtf(row_sum<WARP>(sq, 0.f, red, phase).x * inv_h + a.eps);
      const float token_gate =
          a.gate_mode == STAGEML_GATE_TOKEN ? load_param1(a.gate, a.gate_dtype, row) : 1.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (v * nt + tid) * VEC;
        if (c >= H) continue;
        float w[VEC];
        if (a.post_weight) {
          load_param<VEC>(a.post_weight, a.post_dtype, c, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[v][i] = n[v][i] * inv * w[i];
        }
        if (a.gate_mode == STAGEML_GATE_CHANNEL || a.gate_mode == STAGEML_GATE_FULL) {
          load_param<VEC>(a.gate, a.gate_dtype, a.gate_mode == STAGEML_GATE_FULL ? base + c : c, w);
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[v][i] *= w[i];
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[v][i] *= token_gate;
        }
      }
    }
    sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      if (c >= H) continue;
      float r[VEC];
      row_vals<RING, VEC>(r_row + c, r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        n[v][i] = fmaf(a.residual_scale, r[i], n[v][i]);
        sq = fmaf(n[v][i], n[v][i], sq);
      }
      store_vals<VEC>(static_cast<TR*>(a.new_residual) + base + c, n[v]);
    }
    float inv = 0.f;
    if (a.pre_weight)
      inv = rsqrtf(row_sum<WARP>(sq, 0.f, red, phase).x * inv_h + a.eps);
    else if (RING)
      __syncthreads();
    // the row's copy has been read by every thread (the barrier above)
    if constexpr (RING)
      if (threadIdx.x == 0) fill(count + kStages);
    if (!a.pre_weight) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      float w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = 0.f;
      if (c < H) load_param<VEC>(a.pre_weight, a.pre_dtype, c, w);
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = n[v][i] * inv * w[i];
      if constexpr (VEC == 8) {
        if (a.codes) {
          // 16 neighbouring lanes hold one block of 128 columns
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = max(m, c < H ? __float_as_uint(w[i]) & 0x7fffffffu : 0u);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          float s = __uint_as_float(m) / 448.0f;
          s = s == 0.f ? 1.f : s;
          if (c < H) {
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              q[i] = __nv_cvt_float2_to_fp8x2(make_float2(w[2 * i] / s, w[2 * i + 1] / s), __NV_SATFINITE, __NV_E4M3);
            *reinterpret_cast<uint2*>(a.codes + base + c) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
            if ((c & 127) == 0) a.code_scale[row * ((H + 127) / 128) + (c >> 7)] = s;
          }
          continue;
        }
      }
      if (c < H) {
        if (z32)
          store_vals<VEC>(z32 + base + c, w);
        else
          store_vals<VEC>(static_cast<TY*>(a.normed) + base + c, w);
      }
    }
  }
}

// Column sums that the backward keeps: S (for the post weight and a per-channel gate), dw_pre.
__host__ __device__ inline bool has_block_sum(const stageml_norm_args& a) {
  return a.post_weight || a.gate_mode == STAGEML_GATE_CHANNEL;
}
__host__ __device__ inline int n_sums_of(const stageml_norm_args& a) {
  return (has_block_sum(a) ? 1 : 0) + (a.pre_weight ? 1 : 0);
}

template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING>
__global__ void __launch_bounds__(kMaxThreads, 1) norm_residual_backward_kernel(const stageml_norm_args a, float* partial) {
  extern __shared__ __align__(128) uint8_t row_smem[];
  __shared__ float2 red[32];
  __shared__ uint64_t bars[kStages];
  __shared__ int flag;
  int phase = 0;
  const int nt = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int H = a.H;
  const float inv_h = 1.f / (float)H;
  const bool post = a.post_weight != nullptr, pre = a.pre_weight != nullptr && a.grad_normed != nullptr;
  const bool channel = a.gate_mode == STAGEML_GATE_CHANNEL, has_y = a.block_out != nullptr;
  const uint32_t r_bytes = (uint32_t)H * sizeof(TR), y_bytes = (uint32_t)H * sizeof(TY);
  const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  RowRing ring;
  auto fill = [&](uint32_t n) {
    const int64_t row = first + n * step;
    if (row >= a.T) return;
    const void* src[4] = {static_cast<const TR*>(a.residual) + row * H,
                          a.grad_residual ? static_cast<const TR*>(a.grad_residual) + row * H : nullptr,
                          has_y ? static_cast<const TY*>(a.block_out) + row * H : nullptr,
                          pre ? static_cast<const TY*>(a.grad_normed) + row * H : nullptr};
    const uint32_t bytes[4] = {r_bytes, r_bytes, y_bytes, y_bytes};
    ring.fill(n, src, bytes);
  };
  if constexpr (RING) {
    ring.init(row_smem, 2 * (r_bytes + y_bytes), bars, &flag, a.status);
    if (threadIdx.x == 0)
      for (int i = 0; i < kStages; ++i) fill(i);
  }
  float sum_y[V][VEC], sum_z[V][VEC];  // this thread's columns: S and dw_pre
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum_y[v][i] = sum_z[v][i] = 0.f;
  uint32_t count = 0;
  for (int64_t row = first; row < a.T; row += step, ++count) {
    const int64_t base = row * H;
    const TR* r_row = static_cast<const TR*>(a.residual) + base;
    const TR* dr_row = static_cast<const TR*>(a.grad_residual) + base;
    const TY* y_row = static_cast<const TY*>(a.block_out) + base;
    const TY* dz_row = static_cast<const TY*>(a.grad_normed) + base;
    if constexpr (RING) {
      const uint8_t* stage = ring.wait(count);
      r_row = reinterpret_cast<const TR*>(stage);
      dr_row = reinterpret_cast<const TR*>(stage + r_bytes);
      y_row = reinterpret_cast<const TY*>(stage + 2 * r_bytes);
      dz_row = reinterpret_cast<const TY*>(stage + 2 * r_bytes + y_bytes);
    }
    float y[V][VEC], n[V][VEC], d[V][VEC];
    float inv_y = 1.f;
    const float token_gate =
        a.gate_mode == STAGEML_GATE_TOKEN ? load_param1(a.gate, a.gate_dtype, row) : 1.f;
    auto gate_of = [&](int c, float (&g)[VEC]) {
      if (channel || a.gate_mode == STAGEML_GATE_FULL) {
        load_param<VEC>(a.gate, a.gate_dtype, channel ? c : base + c, g);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[i] = token_gate;
      }
    };
    auto post_of = [&](int c, float (&w)[VEC]) {
      if (post) {
        load_param<VEC>(a.post_weight, a.post_dtype, c, w);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) w[i] = 1.f;
      }
    };
    // y^ (or y), then n = r'
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[v][i] = 0.f;
      if (c < H && has_y) row_vals<RING, VEC>(y_row + c, y[v]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sq = fmaf(y[v][i], y[v][i], sq);
    }
    if (post) inv_y = rsqrtf(row_sum<WARP>(sq, 0.f, red, phase).x * inv_h + a.eps);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = d[v][i] = 0.f;
      if (c >= H) continue;
      float r[VEC];
      row_vals<RING, VEC>(r_row + c, r);
      if (has_y) {
        float w[VEC], g[VEC];
        post_of(c, w);
        gate_of(c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y[v][i] *= inv_y;
          n[v][i] = g[i] * (y[v][i] * w[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = fmaf(a.residual_scale, r[i], n[v][i]);
      if (pre) {
        float w[VEC];
        row_vals<RING, VEC>(dz_row + c, d[v]);
        load_param<VEC>(a.pre_weight, a.pre_dtype, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s1 = fmaf(n[v][i], n[v][i], s1);
          s2 = fmaf(d[v][i] * w[i], n[v][i], s2);
        }
      }
    }
    float inv_n = 0.f, mean = 0.f;
    if (pre) {
      const float2 s = row_sum<WARP>(s1, s2, red, phase);
      inv_n = rsqrtf(s.x * inv_h + a.eps);
      mean = s.y * inv_n * inv_h;  // mean(dn n^)
    }
    // d, then the gradients that need no further row sum
    float s3 = 0.f, s4 = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      if (c >= H) continue;
      if (pre) {
        float w[VEC];
        load_param<VEC>(a.pre_weight, a.pre_dtype, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float nh = n[v][i] * inv_n;
          sum_z[v][i] = fmaf(d[v][i], nh, sum_z[v][i]);
          d[v][i] = inv_n * (d[v][i] * w[i] - nh * mean);
        }
      }
      if (a.grad_residual) {
        float dr[VEC];
        row_vals<RING, VEC>(dr_row + c, dr);
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[v][i] += dr[i];
      }
      float t[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = a.residual_scale * d[v][i];
      store_vals<VEC>(static_cast<TR*>(a.d_residual) + base + c, t);
      if (!has_y) continue;
      float w[VEC], g[VEC];
      post_of(c, w);
      gate_of(c, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = d[v][i] * y[v][i];  // dg = w_post t
      if (a.gate_mode == STAGEML_GATE_FULL) {
        float dg[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) dg[i] = w[i] * t[i];
        store_param<VEC>(a.d_gate, a.gate_dtype, base + c, dg);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        s4 = fmaf(w[i], t[i], s4);
        sum_y[v][i] += channel ? t[i] : g[i] * t[i];
        d[v][i] *= g[i] * w[i];  // the gradient of y^
        s3 = fmaf(d[v][i], y[v][i], s3);
      }
    }
    if (has_y && (post || a.gate_mode == STAGEML_GATE_TOKEN)) {
      const float2 s = row_sum<WARP>(s3, s4, red, phase);
      s3 = s.x * inv_h;
      if (a.gate_mode == STAGEML_GATE_TOKEN && tid == 0) store_param1(a.d_gate, a.gate_dtype, row, s.y);
    } else if (RING) {
      __syncthreads();
    }
    // the row's copies have been read by every thread (the barrier above)
    if constexpr (RING)
      if (threadIdx.x == 0) fill(count + kStages);
    if (!has_y) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      if (c >= H) continue;
      float t[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = post ? inv_y * (d[v][i] - y[v][i] * s3) : d[v][i];
      store_vals<VEC>(static_cast<TY*>(a.d_block_out) + base + c, t);
    }
  }
  if (n_sums_of(a) == 0) return;
  // one row of sums per CTA, or per warp of a CTA of warp rows
  const int64_t owner = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  float* out = partial + owner * n_sums_of(a) * H;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * nt + tid) * VEC;
    if (c >= H) continue;
    if (has_block_sum(a)) store_vals<VEC>(out + c, sum_y[v]);
    if (a.pre_weight) store_vals<VEC>(out + (has_block_sum(a) ? H : 0) + c, sum_z[v]);
  }
}

// The weights' gradients: the column sums over all owners, in a fixed order (16 strands of
// every 16th owner, then the strands), times what the column's gradient is a multiple by.
constexpr int kStrands = 16;
__global__ void __launch_bounds__(32 * kStrands)
    norm_weight_sums_kernel(const stageml_norm_args a, const float* __restrict__ partial, int owners, int n_sums) {
  __shared__ float part[kStrands][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int64_t width = (int64_t)n_sums * a.H, i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < width) {
#pragma unroll 8
    for (int c = strand; c < owners; c += kStrands) s += __ldg(partial + c * width + i);
  }
  part[strand][lane] = s;
  __syncthreads();
  if (strand != 0 || i >= width) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < kStrands; ++w) s += part[w][lane];
  if (has_block_sum(a) && i < a.H) {
    const bool channel = a.gate_mode == STAGEML_GATE_CHANNEL;
    if (a.post_weight) store_param1(a.d_post, a.post_dtype, i, channel ? s * load_param1(a.gate, a.gate_dtype, i) : s);
    if (channel)
      store_param1(a.d_gate, a.gate_dtype, i, a.post_weight ? s * load_param1(a.post_weight, a.post_dtype, i) : s);
  } else {
    store_param1(a.d_pre, a.pre_dtype, i - (has_block_sum(a) ? a.H : 0), s);
  }
}

struct Shape {
  int threads, rows_per_cta;
};

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

bool vectors(const stageml_norm_args& a) {
  return a.H % 8 == 0 && aligned(a.residual) && aligned(a.block_out) && aligned(a.post_weight) && aligned(a.gate) &&
         aligned(a.pre_weight) && aligned(a.new_residual) && aligned(a.normed) && aligned(a.codes) &&
         aligned(a.grad_residual) && aligned(a.grad_normed) && aligned(a.d_residual) && aligned(a.d_block_out) &&
         (a.gate_mode != STAGEML_GATE_FULL || aligned(a.d_gate));
}

// Threads for `units` loads per row, `per` of them per thread.
Shape shape_of(int units, int per, bool warp) {
  if (warp) return {256, 8};
  return {std::min(kMaxThreads, ((units + per - 1) / per + 31) / 32 * 32), 1};
}

// Persistent CTAs of a kernel of `threads` threads and `smem` bytes: as many as fit in an SM's
// registers and shared memory, at most `rows`.
template <typename K>
int resident_ctas(K kernel, int threads, size_t smem, int64_t rows) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem) != cudaSuccess || per_sm < 1)
    per_sm = 1;
  return (int)std::min<int64_t>(rows, (int64_t)sm_count() * per_sm);
}

// The most owners of column sums (workspace): 2048 threads per SM.
int max_owners(const stageml_norm_args& a) {
  const int rows_per_sm = a.H <= 256 ? 64 : 32;  // warps of warp rows; CTAs of at least 64 threads
  return (int)std::min<int64_t>(a.T + 7, (int64_t)sm_count() * rows_per_sm);
}

template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING>
int run_forward(const stageml_norm_args& a, const Shape& s, float* z32, cudaStream_t stream) {
  auto kernel = norm_residual_kernel<TR, TY, VEC, V, WARP, RING>;
  int64_t grid = (a.T + s.rows_per_cta - 1) / s.rows_per_cta;
  size_t smem = 0;
  if (RING) {
    smem = (size_t)kStages * a.H * (sizeof(TR) + sizeof(TY));
    SB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    grid = resident_ctas(kernel, s.threads, smem, a.T);
  }
  SB_CUDA_CHECK(launch_kernel(kernel, dim3((unsigned)grid), dim3(s.threads), smem, stream, false, a, z32));
  count_launch();
  return STAGEML_OK;
}

template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING>
int run_backward(const stageml_norm_args& a, const Shape& s, float* partial, cudaStream_t stream) {
  auto kernel = norm_residual_backward_kernel<TR, TY, VEC, V, WARP, RING>;
  const int n_sums = n_sums_of(a);
  size_t smem = 0;
  if (RING) {
    smem = (size_t)kStages * a.H * 2 * (sizeof(TR) + sizeof(TY));
    SB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  }
  const int grid = resident_ctas(kernel, s.threads, smem, (a.T + s.rows_per_cta - 1) / s.rows_per_cta);
  SB_CUDA_CHECK(launch_kernel(kernel, dim3((unsigned)grid), dim3(s.threads), smem, stream, false, a, partial));
  count_launch();
  if (n_sums) {
    const int64_t width = (int64_t)n_sums * a.H;
    SB_CUDA_CHECK(launch_kernel(norm_weight_sums_kernel, dim3((unsigned)((width + 31) / 32)), dim3(32 * kStrands), 0,
                                stream, false, a, (const float*)partial, grid * s.rows_per_cta, n_sums));
    count_launch();
  }
  return STAGEML_OK;
}

template <typename TR, typename TY>
int dispatch(const stageml_norm_args& a, bool backward, float* scratch, cudaStream_t stream) {
#define SB_NORM(VEC, V, WARP, RING, units) \
  (backward ? run_backward<TR, TY, VEC, V, WARP, RING>(a, shape_of(units, V, WARP), scratch, stream) \
            : run_forward<TR, TY, VEC, V, WARP, RING>(a, shape_of(units, V, WARP), scratch, stream))
  if (vectors(a)) {
    const int units = a.H / 8;
    if (units <= 32) return SB_NORM(8, 1, true, false, units);
    // few rows: as many threads per row as possible, straight from global memory
    const size_t stages = (size_t)kStages * a.H * (sizeof(TR) + sizeof(TY)) * (backward ? 2 : 1);
    if (a.T <= sm_count() || stages > kMaxRing) {
      if (units <= kMaxThreads) return SB_NORM(8, 1, false, false, units);
      if (units <= 2 * kMaxThreads) return SB_NORM(8, 2, false, false, units);
      return SB_NORM(8, 4, false, false, units);
    }
    if (units <= 2 * kMaxThreads) return SB_NORM(8, 2, false, true, units);
    return SB_NORM(8, 4, false, true, units);
  }
  if (a.H <= 256) return SB_NORM(1, 8, true, false, a.H);
  if (a.H <= 8 * kMaxThreads) return SB_NORM(1, 8, false, false, a.H);
  return SB_NORM(1, 32, false, false, a.H);
#undef SB_NORM
}

int launch_any(const stageml_norm_args& a, bool backward, float* scratch, cudaStream_t stream) {
  if (a.resid_dtype == STAGEML_BF16) return dispatch<bf16, bf16>(a, backward, scratch, stream);
  if (a.resid_dtype == STAGEML_F16) return dispatch<f16, f16>(a, backward, scratch, stream);
  if (a.block_dtype == STAGEML_BF16) return dispatch<float, bf16>(a, backward, scratch, stream);
  if (a.block_dtype == STAGEML_F16) return dispatch<float, f16>(a, backward, scratch, stream);
  return dispatch<float, float>(a, backward, scratch, stream);
}

}  // namespace

int norm_max_width() { return kMaxH; }

size_t norm_residual_scratch(const stageml_norm_args& a) {
  // codes of a width or address without vector loads: z in fp32, quantized by a second kernel
  return a.codes && !vectors(a) ? (size_t)a.T * a.H * 4 : 0;
}

int launch_norm_residual(const stageml_norm_args& a, void* scratch, cudaStream_t stream) {
  if (a.T == 0) return STAGEML_OK;
  const bool two_step = a.codes && !vectors(a);
  SB_TRY(launch_any(a, false, two_step ? static_cast<float*>(scratch) : nullptr, stream));
  if (two_step)
    return launch_quantize_block_rows(scratch, STAGEML_F32, a.T, a.H, nullptr, 0, a.codes, a.code_scale, stream);
  return STAGEML_OK;
}

size_t norm_residual_backward_scratch(const stageml_norm_args& a) {
  return (size_t)max_owners(a) * n_sums_of(a) * a.H * 4;
}

int launch_norm_residual_backward(const stageml_norm_args& a, void* scratch, cudaStream_t stream) {
  if (a.T == 0) {
    // no tokens: the weights' gradients are zero
    const size_t es[3] = {4, 2, 2};
    if (a.post_weight) SB_CUDA_CHECK(cudaMemsetAsync(a.d_post, 0, a.H * es[a.post_dtype], stream));
    if (a.gate_mode == STAGEML_GATE_CHANNEL) SB_CUDA_CHECK(cudaMemsetAsync(a.d_gate, 0, a.H * es[a.gate_dtype], stream));
    if (a.pre_weight) SB_CUDA_CHECK(cudaMemsetAsync(a.d_pre, 0, a.H * es[a.pre_dtype], stream));
    return STAGEML_OK;
  }
  return launch_any(a, true, static_cast<float*>(scratch), stream);
}

}  // namespace sb
