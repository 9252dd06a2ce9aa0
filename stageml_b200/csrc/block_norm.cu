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
// is not a multiple of 8 values. The gradients of weights summed over tokens go through
// per-CTA sums (each CTA takes every gridDim-th row) and a second kernel that adds them in
// CTA order: no atomics, the same bits on every run. Bound: HBM.
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kMaxH = 16384;  // 512 threads x 32 values

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

template <typename TR, typename TY, int VEC, int V, bool WARP>
__global__ void __launch_bounds__(kMaxThreads) norm_residual_kernel(const stageml_norm_args a, float* z32) {
  __shared__ float2 red[32];
  int phase = 0;
  const int nt = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.T) return;  // whole warps
  const int H = a.H;
  const int64_t base = row * H;
  const float inv_h = 1.f / (float)H;
  float n[V][VEC];
  if (a.block_out) {
    const TY* y = static_cast<const TY*>(a.block_out) + base;
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = 0.f;
      if (c < H) load_vals<VEC>(y + c, n[v]);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sq = fmaf(n[v][i], n[v][i], sq);
    }
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
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = 0.f;
  }
  float sq = 0.f;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * nt + tid) * VEC;
    if (c >= H) continue;
    float r[VEC];
    load_vals<VEC>(static_cast<const TR*>(a.residual) + base + c, r);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      n[v][i] = fmaf(a.residual_scale, r[i], n[v][i]);
      sq = fmaf(n[v][i], n[v][i], sq);
    }
    store_vals<VEC>(static_cast<TR*>(a.new_residual) + base + c, n[v]);
  }
  if (!a.pre_weight) return;
  const float inv = rsqrtf(row_sum<WARP>(sq, 0.f, red, phase).x * inv_h + a.eps);
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

// Column sums kept per CTA in shared memory: [post | gate (per channel) | pre], H floats each.
template <typename TR, typename TY, int VEC, int V, bool WARP>
__global__ void __launch_bounds__(kMaxThreads) norm_residual_backward_kernel(const stageml_norm_args a, float* partial) {
  extern __shared__ float sums[];
  __shared__ float2 red[32];
  int phase = 0;
  const int nt = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int H = a.H;
  const float inv_h = 1.f / (float)H;
  const bool post = a.post_weight != nullptr, pre = a.pre_weight != nullptr;
  const bool channel = a.gate_mode == STAGEML_GATE_CHANNEL;
  const int n_sums = (int)post + (int)channel + (int)pre;
  const int warps = blockDim.x >> 5;
  // one set of sums per CTA, or per warp of a CTA of warp rows
  float* mine = sums + (WARP ? (size_t)(threadIdx.x >> 5) * n_sums * H : 0);
  float* s_post = mine;
  float* s_gate = s_post + (post ? H : 0);
  float* s_pre = s_gate + (channel ? H : 0);
  for (int i = tid; i < n_sums * H; i += nt) mine[i] = 0.f;
  if (WARP)
    __syncwarp();
  else
    __syncthreads();

  const int64_t row0 = WARP ? (int64_t)blockIdx.x * warps + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = (int64_t)gridDim.x * (WARP ? warps : 1);
  for (int64_t row = row0; row < a.T; row += step) {
    const int64_t base = row * H;
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
      if (c < H && a.block_out) load_vals<VEC>(static_cast<const TY*>(a.block_out) + base + c, y[v]);
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
      load_vals<VEC>(static_cast<const TR*>(a.residual) + base + c, r);
      if (a.block_out) {
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
      if (pre && a.grad_normed) {
        float w[VEC];
        load_vals<VEC>(static_cast<const TY*>(a.grad_normed) + base + c, d[v]);
        load_param<VEC>(a.pre_weight, a.pre_dtype, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s1 = fmaf(n[v][i], n[v][i], s1);
          s2 = fmaf(d[v][i] * w[i], n[v][i], s2);
        }
      }
    }
    float inv_n = 0.f, mean = 0.f;
    if (pre && a.grad_normed) {
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
      if (pre && a.grad_normed) {
        float w[VEC];
        load_param<VEC>(a.pre_weight, a.pre_dtype, c, w);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float nh = n[v][i] * inv_n;
          s_pre[c + i] += d[v][i] * nh;
          d[v][i] = inv_n * (d[v][i] * w[i] - nh * mean);
        }
      }
      if (a.grad_residual) {
        float dr[VEC];
        load_vals<VEC>(static_cast<const TR*>(a.grad_residual) + base + c, dr);
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[v][i] += dr[i];
      }
      float t[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = a.residual_scale * d[v][i];
      store_vals<VEC>(static_cast<TR*>(a.d_residual) + base + c, t);
      if (!a.block_out) continue;
      float w[VEC], g[VEC];
      post_of(c, w);
      gate_of(c, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = d[v][i] * (y[v][i] * w[i]);  // d u
      if (channel) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s_gate[c + i] += t[i];
      } else if (a.gate_mode == STAGEML_GATE_FULL) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) store_param1(a.d_gate, a.gate_dtype, base + c + i, t[i]);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s4 += t[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        d[v][i] *= g[i];  // du
        if (post) {
          s_post[c + i] += d[v][i] * y[v][i];
          d[v][i] *= w[i];
          s3 = fmaf(d[v][i], y[v][i], s3);
        }
      }
    }
    if (!a.block_out) continue;
    if (post || a.gate_mode == STAGEML_GATE_TOKEN) {
      const float2 s = row_sum<WARP>(s3, s4, red, phase);
      s3 = s.x * inv_h;
      if (a.gate_mode == STAGEML_GATE_TOKEN && tid == 0) store_param1(a.d_gate, a.gate_dtype, row, s.y);
    }
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
  if (n_sums == 0) return;
  __syncthreads();
  float* out = partial + (size_t)blockIdx.x * n_sums * H;
  for (int i = threadIdx.x; i < n_sums * H; i += blockDim.x) {
    float s = 0.f;
    for (int w = 0; w < (WARP ? warps : 1); ++w) s += sums[(size_t)w * n_sums * H + i];
    out[i] = s;
  }
}

// d_weight[c] = sum over CTAs of partial[cta][c], in CTA order within each of 8 fixed strands.
__global__ void __launch_bounds__(256) norm_weight_sums_kernel(const stageml_norm_args a, const float* partial, int ctas,
                                                               int n_sums) {
  __shared__ float part[8][33];
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int64_t width = (int64_t)n_sums * a.H, i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < width)
    for (int c = strand; c < ctas; c += 8) s += partial[c * width + i];
  part[strand][lane] = s;
  __syncthreads();
  if (strand != 0 || i >= width) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) s += part[w][lane];
  int which = (int)(i / a.H);
  const int col = (int)(i - (int64_t)which * a.H);
  if (a.post_weight) {
    if (which == 0) return store_param1(a.d_post, a.post_dtype, col, s);
    --which;
  }
  if (a.gate_mode == STAGEML_GATE_CHANNEL) {
    if (which == 0) return store_param1(a.d_gate, a.gate_dtype, col, s);
    --which;
  }
  store_param1(a.d_pre, a.pre_dtype, col, s);
}

struct Shape {
  int threads, rows_per_cta;
  bool warp;
};

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

bool vectors(const stageml_norm_args& a) {
  return a.H % 8 == 0 && aligned(a.residual) && aligned(a.block_out) && aligned(a.post_weight) && aligned(a.gate) &&
         aligned(a.pre_weight) && aligned(a.new_residual) && aligned(a.normed) && aligned(a.codes) &&
         aligned(a.grad_residual) && aligned(a.grad_normed) && aligned(a.d_residual) && aligned(a.d_block_out);
}

// Threads for `units` loads per row, `per` of them per thread.
Shape shape_of(int units, int per, bool warp_ok) {
  Shape s;
  s.warp = warp_ok && units <= 32 * per;
  if (s.warp) {
    s.threads = 256, s.rows_per_cta = 8;
  } else {
    s.threads = std::min(kMaxThreads, ((units + per - 1) / per + 31) / 32 * 32);
    s.rows_per_cta = 1;
  }
  return s;
}

int n_sums_of(const stageml_norm_args& a) {
  return (a.post_weight ? 1 : 0) + (a.gate_mode == STAGEML_GATE_CHANNEL ? 1 : 0) + (a.pre_weight ? 1 : 0);
}

// CTAs of the backward: enough for every SM, no more than rows.
int backward_ctas(const stageml_norm_args& a, int rows_per_cta, int per_sm) {
  return (int)std::min<int64_t>((a.T + rows_per_cta - 1) / rows_per_cta, (int64_t)sm_count() * per_sm);
}
constexpr int kBackwardCtasPerSm = 4;

template <typename TR, typename TY, int VEC, int V, bool WARP>
int run_forward(const stageml_norm_args& a, const Shape& s, float* z32, cudaStream_t stream) {
  const int64_t grid = (a.T + s.rows_per_cta - 1) / s.rows_per_cta;
  SB_CUDA_CHECK(launch_kernel(norm_residual_kernel<TR, TY, VEC, V, WARP>, dim3((unsigned)grid), dim3(s.threads), 0,
                              stream, false, a, z32));
  count_launch();
  return STAGEML_OK;
}

template <typename TR, typename TY, int VEC, int V, bool WARP>
int run_backward(const stageml_norm_args& a, const Shape& s, float* partial, cudaStream_t stream) {
  auto kernel = norm_residual_backward_kernel<TR, TY, VEC, V, WARP>;
  const int n_sums = n_sums_of(a);
  const size_t smem = (size_t)n_sums * a.H * 4 * (WARP ? s.threads / 32 : 1);
  SB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const int grid = backward_ctas(a, s.rows_per_cta, kBackwardCtasPerSm);
  SB_CUDA_CHECK(launch_kernel(kernel, dim3((unsigned)grid), dim3(s.threads), smem, stream, false, a, partial));
  count_launch();
  if (n_sums) {
    const int64_t width = (int64_t)n_sums * a.H;
    SB_CUDA_CHECK(launch_kernel(norm_weight_sums_kernel, dim3((unsigned)((width + 31) / 32)), dim3(256), 0, stream,
                                false, a, (const float*)partial, grid, n_sums));
    count_launch();
  }
  return STAGEML_OK;
}

template <typename TR, typename TY>
int dispatch(const stageml_norm_args& a, bool backward, float* scratch, cudaStream_t stream) {
#define SB_NORM(VEC, V, WARP, shape) \
  (backward ? run_backward<TR, TY, VEC, V, WARP>(a, shape, scratch, stream) \
            : run_forward<TR, TY, VEC, V, WARP>(a, shape, scratch, stream))
  if (vectors(a)) {
    const int units = a.H / 8;
    if (units <= 32) return SB_NORM(8, 1, true, shape_of(units, 1, true));
    if (units <= kMaxThreads) return SB_NORM(8, 1, false, shape_of(units, 1, false));
    if (units <= 2 * kMaxThreads) return SB_NORM(8, 2, false, shape_of(units, 2, false));
    return SB_NORM(8, 4, false, shape_of(units, 4, false));
  }
  if (a.H <= 256) return SB_NORM(1, 8, true, shape_of(a.H, 8, true));
  if (a.H <= 8 * kMaxThreads) return SB_NORM(1, 8, false, shape_of(a.H, 8, false));
  return SB_NORM(1, 32, false, shape_of(a.H, 32, false));
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
    return launch_quantize_block_rows(scratch, STAGEML_F32, a.T, a.H, nullptr, nullptr, a.codes, a.code_scale, stream);
  return STAGEML_OK;
}

size_t norm_residual_backward_scratch(const stageml_norm_args& a) {
  return (size_t)sm_count() * kBackwardCtasPerSm * n_sums_of(a) * a.H * 4;
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
