// The router's balance loss, its per-expert counts and the logits' gradient.
//
//   p[t, :] = softmax(logits[t, :])          over the tokens t with valid[t], n of them
//   counts[e] = number of their chosen slots (t, j) with ids[t, j] = e
//   f[e] = counts[e] / (n k),  P[e] = (1/n) sum_t p[t, e]
//   loss = c E sum_e f[e] P[e]
//   dlogits[t, e] = dloss c E / n * p[t, e] (f[e] - sum_i f[i] p[t, i])   (0 where not valid)
//
// f is a count and carries no gradient. ids < 0 are slots without an expert; an id >= E
// goes to the status word and is skipped. A token whose logits are all -infinity has no
// softmax: its p and its gradient are 0. n = 0 gives loss 0.
//
// Forward: lanes of a warp own experts (groups of 2..32 lanes per token, up to 8 experts
// per lane); each warp sums its tokens' p in registers, each CTA writes one partial sum per
// expert, and a second kernel adds the partials in CTA order: no floating-point atomics,
// the same bits on every run. Counts are integer atomics in shared memory. Backward: the
// softmax again from the logits, one pass. Bound: HBM for long batches (logits read twice,
// gradient written once), launches for short ones.
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// The token's softmax over `LANES` lanes, NJ experts per lane (expert lane + LANES j),
// from its logits in x; 0 everywhere when no logit is above -infinity.
template <int LANES, int NJ>
__device__ __forceinline__ void softmax_lanes(float (&x)[NJ]) {
  float m = x[0];
#pragma unroll
  for (int j = 1; j < NJ; ++j) m = fmaxf(m, x[j]);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const bool none = m == -INFINITY;
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    x[j] = none && x[j] == -INFINITY ? 0.f : expf(x[j] - m);
    s += x[j];
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const float inv = none && s == 0.f ? 0.f : 1.f / s;
#pragma unroll
  for (int j = 0; j < NJ; ++j) x[j] *= inv;
}

template <typename T, int LANES, int NJ>
__device__ __forceinline__ void load_logits(const T* __restrict__ logits, int64_t t, bool live, int E, int lane,
                                            float (&x)[NJ]) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + LANES * j;
    x[j] = live && e < E ? to_f32<T>(logits[t * E + e]) : -INFINITY;
  }
}

template <typename T, int LANES, int NJ>
__global__ void __launch_bounds__(kThreads)
    balance_sums_kernel(const T* __restrict__ logits, const void* __restrict__ ids, int ids_i64,
                        const uint8_t* __restrict__ valid, int64_t T_, int E, int k, float* __restrict__ psum,
                        int32_t* __restrict__ pcount, int32_t* status) {
  constexpr int PER_WARP = 32 / LANES;
  __shared__ float sums[kWarps][LANES * NJ];
  __shared__ int32_t counts[LANES * NJ + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1), sub = (threadIdx.x & 31) / LANES;
  for (int i = threadIdx.x; i <= LANES * NJ; i += kThreads) counts[i] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * kWarps * PER_WARP, step = (int64_t)gridDim.x * kWarps * PER_WARP;
  float acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = 0.f;
  int tokens = 0;
  for (int64_t t0 = first + warp * PER_WARP; t0 < T_; t0 += step) {
    const int64_t t = t0 + sub;
    const bool live = t < T_ && (!valid || valid[t]);
    float x[NJ];
    load_logits<T, LANES, NJ>(logits, t, live, E, lane, x);
    softmax_lanes<LANES, NJ>(x);
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] += x[j];
    if (live) {
      for (int j = lane; j < k; j += LANES) {
        const int64_t i = t * k + j;
        const int64_t e = ids_i64 ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
        if (e >= E) {
          if (status) atomicCAS(status, 0, (int)kDevBadIndex);
        } else if (e >= 0) {
          atomicAdd(&counts[e], 1);
        }
      }
      tokens += lane == 0;
    }
  }
#pragma unroll
  for (int o = LANES; o < 32; o <<= 1)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
  if (tokens) atomicAdd(&counts[LANES * NJ], tokens);
  if (sub == 0)
#pragma unroll
    for (int j = 0; j < NJ; ++j) sums[warp][lane + LANES * j] = acc[j];
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sums[w][e];
    psum[(int64_t)blockIdx.x * E + e] = s;
    pcount[(int64_t)blockIdx.x * (E + 1) + e] = counts[e];
  }
  if (threadIdx.x == 0) pcount[(int64_t)blockIdx.x * (E + 1) + E] = counts[LANES * NJ];
}

// One CTA: totals over the CTAs of the first kernel in a fixed order, then the loss.
__global__ void __launch_bounds__(1024) balance_loss_kernel(const float* __restrict__ psum,
                                                            const int32_t* __restrict__ pcount, int ctas, int E, int k,
                                                            float coefficient, float* loss, int32_t* counts,
                                                            int32_t* tokens) {
  __shared__ float fsum[1024];
  __shared__ int32_t isum[1024];
  __shared__ int32_t n_tokens;
  const int strands = 1024 / (E + 1);  // E <= 256
  const int e = threadIdx.x % (E + 1), strand = threadIdx.x / (E + 1);
  float s = 0.f;
  int c = 0;
  if (strand < strands)
    for (int i = strand; i < ctas; i += strands) {
      if (e < E) s += psum[(int64_t)i * E + e];
      c += pcount[(int64_t)i * (E + 1) + e];
    }
  fsum[threadIdx.x] = s;
  isum[threadIdx.x] = c;
  __syncthreads();
  if (strand == 0) {
    for (int w = 1; w < strands; ++w) {
      s += fsum[w * (E + 1) + e];
      c += isum[w * (E + 1) + e];
    }
    if (e == E) {
      n_tokens = c;
      *tokens = c;
    } else {
      counts[e] = c;
    }
  }
  __syncthreads();
  const float n = fmaxf((float)n_tokens, 1.f);
  fsum[threadIdx.x] = strand == 0 && e < E ? (float)c / (n * (float)k) * (s / n) : 0.f;
  __syncthreads();
  if (threadIdx.x < 32) {
    float t = 0.f;
    for (int i = threadIdx.x; i < E; i += 32) t += fsum[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (threadIdx.x == 0) *loss = coefficient * (float)E * t;
  }
}

template <typename T, int LANES, int NJ>
__global__ void __launch_bounds__(kThreads)
    balance_backward_kernel(const float* __restrict__ grad_loss, const T* __restrict__ logits,
                            const int32_t* __restrict__ counts, const int32_t* __restrict__ tokens,
                            const uint8_t* __restrict__ valid, int64_t T_, int E, int k, float coefficient,
                            T* __restrict__ grad) {
  constexpr int PER_WARP = 32 / LANES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (LANES - 1), sub = (threadIdx.x & 31) / LANES;
  const float n = fmaxf((float)*tokens, 1.f);
  const float scale = *grad_loss * coefficient * (float)E / n;
  float f[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const int e = lane + LANES * j;
    f[j] = e < E ? (float)counts[e] / (n * (float)k) : 0.f;
  }
  const int64_t first = (int64_t)blockIdx.x * kWarps * PER_WARP, step = (int64_t)gridDim.x * kWarps * PER_WARP;
  for (int64_t t0 = first + warp * PER_WARP; t0 < T_; t0 += step) {
    const int64_t t = t0 + sub;
    const bool live = t < T_ && (!valid || valid[t]);
    float x[NJ];
    load_logits<T, LANES, NJ>(logits, t, live, E, lane, x);
    softmax_lanes<LANES, NJ>(x);
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) dot = fmaf(x[j], f[j], dot);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (t < T_) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int e = lane + LANES * j;
        if (e < E) grad[t * E + e] = from_f32<T>(live ? scale * x[j] * (f[j] - dot) : 0.f);
      }
    }
  }
}

constexpr int kCtasPerSm = 4;

int ctas_for(int64_t T, int E) {
  int lanes = 2;
  while (lanes < 32 && lanes < E) lanes <<= 1;
  const int64_t per_cta = (int64_t)kWarps * (32 / lanes);
  return (int)std::min<int64_t>((T + per_cta - 1) / per_cta, (int64_t)sm_count() * kCtasPerSm);
}

// Calls f(lanes, experts per lane) as compile-time constants for E experts (E <= 256).
template <typename F>
int with_layout(int E, F&& f) {
  using std::integral_constant;
#define SB_LAYOUT(L, J) return f(integral_constant<int, L>{}, integral_constant<int, J>{})
  if (E <= 2) SB_LAYOUT(2, 1);
  if (E <= 4) SB_LAYOUT(4, 1);
  if (E <= 8) SB_LAYOUT(8, 1);
  if (E <= 16) SB_LAYOUT(16, 1);
  if (E <= 32) SB_LAYOUT(32, 1);
  if (E <= 64) SB_LAYOUT(32, 2);
  if (E <= 128) SB_LAYOUT(32, 4);
  SB_LAYOUT(32, 8);
#undef SB_LAYOUT
}

template <typename T>
int forward(const void* logits, const void* ids, int ids_i64, const uint8_t* valid, int64_t T_, int E, int k,
            float* psum, int32_t* pcount, int grid, int32_t* status, cudaStream_t stream) {
  return with_layout(E, [&](auto lanes, auto nj) {
    SB_CUDA_CHECK(launch_kernel(balance_sums_kernel<T, decltype(lanes)::value, decltype(nj)::value>,
                                dim3((unsigned)grid), dim3(kThreads), 0, stream, false, static_cast<const T*>(logits),
                                ids, ids_i64, valid, T_, E, k, psum, pcount, status));
    count_launch();
    return (int)STAGEML_OK;
  });
}

template <typename T>
int backward(const float* grad_loss, const void* logits, const int32_t* counts, const int32_t* tokens,
             const uint8_t* valid, int64_t T_, int E, int k, float coefficient, void* grad, int grid,
             cudaStream_t stream) {
  return with_layout(E, [&](auto lanes, auto nj) {
    SB_CUDA_CHECK(launch_kernel(balance_backward_kernel<T, decltype(lanes)::value, decltype(nj)::value>,
                                dim3((unsigned)grid), dim3(kThreads), 0, stream, false, grad_loss,
                                static_cast<const T*>(logits), counts, tokens, valid, T_, E, k, coefficient,
                                static_cast<T*>(grad)));
    count_launch();
    return (int)STAGEML_OK;
  });
}

}  // namespace

size_t balance_scratch_bytes(int64_t T, int E) { return (size_t)std::max(ctas_for(T, E), 1) * (2 * E + 1) * 4; }

int launch_balance_loss(const void* logits, int dtype, const void* ids, int ids_i64, const uint8_t* valid, int64_t T,
                        int E, int k, float coefficient, float* loss, int32_t* counts, int32_t* tokens,
                        int32_t* status, void* scratch, cudaStream_t stream) {
  const int grid = ctas_for(T, E);
  float* psum = static_cast<float*>(scratch);
  int32_t* pcount = reinterpret_cast<int32_t*>(psum + (size_t)grid * E);
  if (grid > 0) {
    if (dtype == STAGEML_F32)
      SB_TRY(forward<float>(logits, ids, ids_i64, valid, T, E, k, psum, pcount, grid, status, stream));
    else if (dtype == STAGEML_BF16)
      SB_TRY(forward<bf16>(logits, ids, ids_i64, valid, T, E, k, psum, pcount, grid, status, stream));
    else
      SB_TRY(forward<f16>(logits, ids, ids_i64, valid, T, E, k, psum, pcount, grid, status, stream));
  }
  SB_CUDA_CHECK(launch_kernel(balance_loss_kernel, dim3(1), dim3(1024), 0, stream, false, (const float*)psum,
                              (const int32_t*)pcount, grid, E, k, coefficient, loss, counts, tokens));
  count_launch();
  return STAGEML_OK;
}

int launch_balance_loss_backward(const float* grad_loss, const void* logits, int dtype, const int32_t* counts,
                                 const int32_t* tokens, const uint8_t* valid, int64_t T, int E, int k,
                                 float coefficient, void* grad_logits, cudaStream_t stream) {
  const int grid = ctas_for(T, E);
  if (grid == 0) return STAGEML_OK;
  if (dtype == STAGEML_F32)
    return backward<float>(grad_loss, logits, counts, tokens, valid, T, E, k, coefficient, grad_logits, grid, stream);
  if (dtype == STAGEML_BF16)
    return backward<bf16>(grad_loss, logits, counts, tokens, valid, T, E, k, coefficient, grad_logits, grid, stream);
  return backward<f16>(grad_loss, logits, counts, tokens, valid, T, E, k, coefficient, grad_logits, grid, stream);
}

}  // namespace sb
