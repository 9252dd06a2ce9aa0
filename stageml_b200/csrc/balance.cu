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
// A token's experts lie on 1..8 lanes, 4 consecutive experts per 16-byte load and up to 32
// per lane, so a warp works on 4 to 32 tokens at once and a softmax costs few shuffles.
// Each lane sums its experts' p over its tokens in registers; a CTA adds them in a fixed
// order in shared memory. Counts are integer atomics in shared memory. Batches of up to
// kClusterValues logits and kClusterTokens tokens run as one cluster whose first CTA adds the
// others' sums over distributed shared memory and writes the loss: one launch. Longer ones run as many clusters,
// each leaving one partial, which a second kernel adds in cluster order (one partial per CTA
// made that kernel 32 us, now 6). No floating-point atomics: the same bits
// on every run. Backward: the softmax again from the logits, one pass. Bound: HBM for long
// batches (logits read twice, gradient written once), launches for short ones. 65536 x 256 fp32
// logits with eight ids each: 34 us forward, 24 us backward; 256 x 8: 7 us both ways.
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxE = 256;
constexpr int kClusterCtas = 8;                // portable cluster size
// A one-launch batch: its logits, and its tokens, whose ids eight CTAs count one by one (20000 x 5, five
// ids: 30 us in one cluster, 10 in several).
constexpr int64_t kClusterValues = 256 * 1024, kClusterTokens = 4096;
inline bool one_launch(int64_t T, int E) { return T * E <= kClusterValues && T <= kClusterTokens; }

// Lanes per token and 4-expert groups per lane: expert (lane + LANES * j) * 4 + i.
template <int LANES, int NV>
struct Layout {
  static constexpr int lanes = LANES, groups = NV, per_warp = 32 / LANES, experts = LANES * NV * 4;
};

template <typename T, bool VEC>
__device__ __forceinline__ void load4(const T* p, int e, int E, bool live, float (&f)[4]) {
  if (!live || e >= E) {
    f[0] = f[1] = f[2] = f[3] = -INFINITY;
  } else if constexpr (VEC && sizeof(T) == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p + e));
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  } else if constexpr (VEC) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + e));
    const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f32<T>(h[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = e + i < E ? to_f32<T>(p[e + i]) : -INFINITY;
  }
}

// The token's logits on its lanes (-infinity when the token does not count), and its softmax, 0
// everywhere when no logit is above -infinity.
template <typename T, typename L, bool VEC>
__device__ __forceinline__ void load_logits(const T* __restrict__ logits, int64_t t, bool live, int E, int lane,
                                            float (&x)[L::groups][4]) {
  const T* row = logits + t * E;
#pragma unroll
  for (int j = 0; j < L::groups; ++j) load4<T, VEC>(row, (lane + L::lanes * j) * 4, E, live, x[j]);
}

// Sum over the token's experts. Up to 8 of them, every expert may be a chosen one (k = E); the
// gradient then vanishes but for the rounding of these sums, so they are taken pairwise by expert
// index (e with e + 4, then + 2, + 1) over separately rounded terms, as elementwise code takes them.
template <typename L>
__device__ __forceinline__ float token_sum(float (&v)[L::groups][4]) {
  if constexpr (L::lanes <= 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (L::lanes == 2) v[0][i] = __fadd_rn(v[0][i], __shfl_xor_sync(0xffffffffu, v[0][i], 1));
    return __fadd_rn(__fadd_rn(v[0][0], v[0][2]), __fadd_rn(v[0][1], v[0][3]));
  } else {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < L::groups; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s += v[j][i];
#pragma unroll
    for (int o = L::lanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
}

// Above 8 experts the fast exponential and one reciprocal per token: a gradient within 1.0e-7 (relative L2) of the
// definition's, where expf and a division per value give 0.9e-7 and take half as long again (65536 x 256 both ways:
// 93 us, from 61). Up to 8 experts those cost nothing that shows, and the cancellation above needs them.
template <typename L>
__device__ __forceinline__ void softmax(float (&x)[L::groups][4]) {
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < L::groups; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, x[j][i]);
#pragma unroll
  for (int o = L::lanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float shift = m == -INFINITY ? 0.f : m;
  float v[L::groups][4];
#pragma unroll
  for (int j = 0; j < L::groups; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) v[j][i] = x[j][i] = L::lanes <= 2 ? expf(x[j][i] - shift) : __expf(x[j][i] - shift);
  const float s = token_sum<L>(v);
  const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
  for (int j = 0; j < L::groups; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[j][i] = L::lanes <= 2 && s != 0.f ? x[j][i] / s : x[j][i] * inv;
}

struct BalanceIn {
  const void* ids;
  int ids_i64;
  const uint8_t* valid;
  int64_t T;
  int E, k;
  int32_t* status;
};

// This CTA's tokens (cta of ctas): sums[e] = sum of p, counts[e], counts[E] = tokens.
template <typename T, typename L, bool VEC>
__device__ __forceinline__ void cta_sums(const T* __restrict__ logits, const BalanceIn& in, int cta, int ctas,
                                         float (*warp_sums)[kMaxE], float* sums, int32_t* counts) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (L::lanes - 1), sub = (threadIdx.x & 31) / L::lanes;
  for (int i = threadIdx.x; i <= kMaxE; i += kThreads) counts[i] = 0;
  __syncthreads();
  // the slots of all tokens, apart from the softmax loop, whose loads they would hold up
  const int64_t slots = in.T * in.k;
  for (int64_t i = (int64_t)cta * kThreads + threadIdx.x; i < slots; i += (int64_t)ctas * kThreads) {
    const int64_t e = in.ids_i64 ? static_cast<const int64_t*>(in.ids)[i] : static_cast<const int32_t*>(in.ids)[i];
    if (in.valid && !in.valid[(uint32_t)i / (uint32_t)in.k]) continue;
    if (e >= in.E) {
      if (in.status) atomicCAS(in.status, 0, (int)kDevBadIndex);
    } else if (e >= 0) {
      atomicAdd(&counts[e], 1);
    }
  }
  float acc[L::groups][4];
#pragma unroll
  for (int j = 0; j < L::groups; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
  int tokens = 0;
  const int64_t step = (int64_t)ctas * kWarps * L::per_warp;
  auto counted = [&](int64_t t) { return t < in.T && (!in.valid || in.valid[t]); };
  // the next tokens' logits are read while these are worked on
  const int64_t t_first = ((int64_t)cta * kWarps + warp) * L::per_warp;
  float next[L::groups][4];
  bool next_live = counted(t_first + sub);
  load_logits<T, L, VEC>(logits, t_first + sub, next_live, in.E, lane, next);
  for (int64_t t0 = t_first; t0 < in.T; t0 += step) {
    const bool live = next_live;
    float x[L::groups][4];
#pragma unroll
    for (int j = 0; j < L::groups; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) x[j][i] = next[j][i];
    next_live = counted(t0 + step + sub);
    load_logits<T, L, VEC>(logits, t0 + step + sub, next_live, in.E, lane, next);
    softmax<L>(x);
#pragma unroll
    for (int j = 0; j < L::groups; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] += x[j][i];
    tokens += live && lane == 0;
  }
#pragma unroll
  for (int o = L::lanes; o < 32; o <<= 1)
#pragma unroll
    for (int j = 0; j < L::groups; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] += __shfl_xor_sync(0xffffffffu, acc[j][i], o);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
  if ((threadIdx.x & 31) == 0 && tokens) atomicAdd(&counts[in.E], tokens);
  if (sub == 0)
#pragma unroll
    for (int j = 0; j < L::groups; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) warp_sums[warp][(lane + L::lanes * j) * 4 + i] = acc[j][i];
  __syncthreads();
  for (int e = threadIdx.x; e < in.E; e += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += warp_sums[w][e];
    sums[e] = s;
  }
  __syncthreads();
}

// From the totals in shared memory (counts[E] = tokens): loss, counts, tokens. One CTA.
__device__ __forceinline__ void write_loss(const float* sums, const int32_t* counts, int E, int k, float coefficient,
                                           float* loss, int32_t* counts_out, int32_t* tokens_out) {
  for (int e = threadIdx.x; e < E; e += blockDim.x) counts_out[e] = counts[e];
  if (threadIdx.x < 32) {
    const float n = fmaxf((float)counts[E], 1.f);
    float t = 0.f;
    for (int e = threadIdx.x; e < E; e += 32) t += (float)counts[e] / (n * (float)k) * (sums[e] / n);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    if (threadIdx.x == 0) {
      *loss = coefficient * (float)E * t;
      *tokens_out = counts[E];
    }
  }
}

// Every CTA its sums, the first CTA of a cluster their totals in CTA order; one cluster: then the
// loss, several: one partial each (psum [clusters][E], pcount [clusters][E + 1]).
template <typename T, typename L, bool VEC>
__global__ void __launch_bounds__(kThreads, 3)
    balance_sums_kernel(const T* __restrict__ logits, const BalanceIn in, float coefficient, float* loss,
                        int32_t* counts_out, int32_t* tokens_out, float* __restrict__ psum,
                        int32_t* __restrict__ pcount, int cluster_ctas) {
  __shared__ float warp_sums[kWarps][kMaxE];
  __shared__ float sums[kMaxE];
  __shared__ int32_t counts[kMaxE + 1];
  cta_sums<T, L, VEC>(logits, in, blockIdx.x, gridDim.x, warp_sums, sums, counts);
  const bool leader = cluster_ctas == 1 || cluster_ctarank() == 0;
  if (cluster_ctas > 1) {
    cluster_sync_all();
    if (leader) {
      for (int e = threadIdx.x; e <= in.E; e += kThreads) {
        float s = e < in.E ? sums[e] : 0.f;
        int c = counts[e];
        for (int r = 1; r < cluster_ctas; ++r) {
          uint32_t v;
          if (e < in.E) {
            asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(&sums[e]), r)) : "memory");
            s += __uint_as_float(v);
          }
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(&counts[e]), r)) : "memory");
          c += (int)v;
        }
        if (e < in.E) sums[e] = s;
        counts[e] = c;
      }
    }
    cluster_sync_all();  // the others stay until their sums have been read
  }
  if (!leader) return;
  if ((int)gridDim.x == cluster_ctas) {
    write_loss(sums, counts, in.E, in.k, coefficient, loss, counts_out, tokens_out);
    return;
  }
  const int64_t cluster = blockIdx.x / cluster_ctas;
  for (int e = threadIdx.x; e <= in.E; e += kThreads) {
    if (e < in.E) psum[cluster * in.E + e] = sums[e];
    pcount[cluster * (in.E + 1) + e] = counts[e];
  }
}

// One CTA: totals over the partials in a fixed order (strands of every n-th CTA, then the
// strands), then the loss.
__global__ void __launch_bounds__(1024) balance_loss_kernel(const float* __restrict__ psum,
                                                            const int32_t* __restrict__ pcount, int ctas, int E, int k,
                                                            float coefficient, float* loss, int32_t* counts_out,
                                                            int32_t* tokens_out) {
  __shared__ float fsum[1024];
  __shared__ int32_t isum[1024];
  __shared__ float sums[kMaxE];
  __shared__ int32_t counts[kMaxE + 1];
  pdl_wait();
  const int strands = 1024 / (E + 1);
  const int e = threadIdx.x % (E + 1), strand = threadIdx.x / (E + 1);
  float s = 0.f;
  int c = 0;
  if (strand < strands) {
    // eight partials' loads at a time, the last turn's too
    for (int at = strand; at < ctas; at += 8 * strands) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t i = at + j * strands;
        s += i < ctas && e < E ? psum[i * E + e] : 0.f;
        c += i < ctas ? pcount[i * (E + 1) + e] : 0;
      }
    }
  }
  fsum[threadIdx.x] = s;
  isum[threadIdx.x] = c;
  __syncthreads();
  if (strand == 0) {
    for (int w = 1; w < strands; ++w) {
      s += fsum[w * (E + 1) + e];
      c += isum[w * (E + 1) + e];
    }
    if (e < E) sums[e] = s;
    counts[e] = c;
  }
  __syncthreads();
  write_loss(sums, counts, E, k, coefficient, loss, counts_out, tokens_out);
}

template <typename T, typename L, bool VEC>
__global__ void __launch_bounds__(kThreads)
    balance_backward_kernel(const float* __restrict__ grad_loss, const T* __restrict__ logits,
                            const int32_t* __restrict__ counts, const int32_t* __restrict__ tokens,
                            const uint8_t* __restrict__ valid, int64_t T_, int E, int k, float coefficient,
                            T* __restrict__ grad) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & (L::lanes - 1), sub = (threadIdx.x & 31) / L::lanes;
  const float n = fmaxf((float)*tokens, 1.f);
  const float scale = *grad_loss * coefficient * (float)E / n;
  float f[L::groups][4];
#pragma unroll
  for (int j = 0; j < L::groups; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = (lane + L::lanes * j) * 4 + i;
      f[j][i] = e < E ? (float)counts[e] / (n * (float)k) : 0.f;
    }
  const int64_t step = (int64_t)gridDim.x * kWarps * L::per_warp;
  for (int64_t t0 = ((int64_t)blockIdx.x * kWarps + warp) * L::per_warp; t0 < T_; t0 += step) {
    const int64_t t = t0 + sub;
    const bool live = t < T_ && (!valid || valid[t]);
    float x[L::groups][4];
    load_logits<T, L, VEC>(logits, t, live, E, lane, x);
    softmax<L>(x);
    float v[L::groups][4];
#pragma unroll
    for (int j = 0; j < L::groups; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) v[j][i] = __fmul_rn(x[j][i], f[j][i]);
    const float dot = token_sum<L>(v);
    if (t >= T_) continue;
    T* out = grad + t * E;
#pragma unroll
    for (int j = 0; j < L::groups; ++j) {
      const int e = (lane + L::lanes * j) * 4;
      if (e >= E) continue;
      float g[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) g[i] = scale * x[j][i] * (f[j][i] - dot);
      if constexpr (VEC && sizeof(T) == 4) {
        *reinterpret_cast<float4*>(out + e) = make_float4(g[0], g[1], g[2], g[3]);
      } else if constexpr (VEC) {
        T h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = from_f32<T>(g[i]);
        *reinterpret_cast<uint2*>(out + e) = *reinterpret_cast<const uint2*>(h);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (e + i < E) out[e + i] = from_f32<T>(g[i]);
      }
    }
  }
}

constexpr int kCtasPerSm = 3;

// Calls f with the layout for E experts as a type.
template <typename F>
int with_layout(int E, F&& f) {
  if (E <= 4) return f(Layout<1, 1>{});
  if (E <= 8) return f(Layout<2, 1>{});
  if (E <= 16) return f(Layout<4, 1>{});
  if (E <= 32) return f(Layout<8, 1>{});
  if (E <= 64) return f(Layout<8, 2>{});
  if (E <= 128) return f(Layout<16, 2>{});
  return f(Layout<16, 4>{});
}

int ctas_for(int64_t T, int E, int64_t most) {
  int per_warp = 0;
  with_layout(E, [&](auto l) { return per_warp = decltype(l)::per_warp; });
  const int64_t per_cta = (int64_t)kWarps * per_warp;
  return (int)std::min<int64_t>((T + per_cta - 1) / per_cta, most);
}
// CTAs of a long batch, in whole clusters (at least two).
int long_ctas(int64_t T, int E) {
  const int n = ctas_for(T, E, (int64_t)sm_count() * kCtasPerSm);
  return std::max(2, n / kClusterCtas) * kClusterCtas;
}

// 4 logits per load: E % 4 == 0 and the rows aligned to it.
template <typename T>
bool vectors(const void* logits, const void* grad, int E) {
  const uintptr_t mask = 4 * sizeof(T) - 1;
  return E % 4 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(grad)) & mask) == 0;
}

struct ForwardOut {
  float* loss;
  int32_t* counts;
  int32_t* tokens;
};

template <typename T, typename L, bool VEC>
int forward_layout(const T* logits, const BalanceIn& in, float coefficient, const ForwardOut& o, void* scratch,
                   cudaStream_t stream) {
  const bool one = one_launch(in.T, in.E);
  int cluster = kClusterCtas, grid = 0;
  if (one) {  // a power of two of CTAs with a token group per warp, at least one
    for (cluster = 1; cluster < kClusterCtas && cluster < ctas_for(in.T, in.E, kClusterCtas);) cluster <<= 1;
    grid = cluster;
  } else {
    grid = long_ctas(in.T, in.E);
  }
  const int clusters = grid / cluster;
  float* psum = static_cast<float*>(scratch);
  int32_t* pcount = reinterpret_cast<int32_t*>(psum + (size_t)clusters * in.E);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, balance_sums_kernel<T, L, VEC>, logits, in, coefficient, o.loss, o.counts,
                                   o.tokens, psum, pcount, cluster));
  count_launch();
  if (one) return STAGEML_OK;
  SB_CUDA_CHECK(launch_kernel(balance_loss_kernel, dim3(1), dim3(1024), 0, stream, true, (const float*)psum,
                              (const int32_t*)pcount, clusters, in.E, in.k, coefficient, o.loss, o.counts, o.tokens));
  count_launch();
  return STAGEML_OK;
}

template <typename T>
int forward(const void* logits, const BalanceIn& in, float coefficient, const ForwardOut& o, void* scratch,
            cudaStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  return with_layout(in.E, [&](auto l) {
    using L = decltype(l);
    return vectors<T>(x, nullptr, in.E) ? forward_layout<T, L, true>(x, in, coefficient, o, scratch, stream)
                                        : forward_layout<T, L, false>(x, in, coefficient, o, scratch, stream);
  });
}

template <typename T>
int backward(const float* grad_loss, const void* logits, const int32_t* counts, const int32_t* tokens,
             const uint8_t* valid, int64_t T_, int E, int k, float coefficient, void* grad, cudaStream_t stream) {
  const int grid = ctas_for(T_, E, (int64_t)sm_count() * 4);
  const bool vec = vectors<T>(logits, grad, E);
  return with_layout(E, [&](auto l) {
    using L = decltype(l);
    SB_CUDA_CHECK(launch_kernel(vec ? balance_backward_kernel<T, L, true> : balance_backward_kernel<T, L, false>,
                                dim3((unsigned)grid), dim3(kThreads), 0, stream, false, grad_loss,
                                static_cast<const T*>(logits), counts, tokens, valid, T_, E, k, coefficient,
                                static_cast<T*>(grad)));
    count_launch();
    return (int)STAGEML_OK;
  });
}

}  // namespace

size_t balance_scratch_bytes(int64_t T, int E) {
  return one_launch(T, E) ? 0 : (size_t)(long_ctas(T, E) / kClusterCtas) * (2 * E + 1) * 4;
}

int launch_balance_loss(const void* logits, int dtype, const void* ids, int ids_i64, const uint8_t* valid, int64_t T,
                        int E, int k, float coefficient, float* loss, int32_t* counts, int32_t* tokens,
                        int32_t* status, void* scratch, cudaStream_t stream) {
  const BalanceIn in = {ids, ids_i64, valid, T, E, k, status};
  const ForwardOut o = {loss, counts, tokens};
  if (dtype == STAGEML_F32) return forward<float>(logits, in, coefficient, o, scratch, stream);
  if (dtype == STAGEML_BF16) return forward<bf16>(logits, in, coefficient, o, scratch, stream);
  return forward<f16>(logits, in, coefficient, o, scratch, stream);
}

int launch_balance_loss_backward(const float* grad_loss, const void* logits, int dtype, const int32_t* counts,
                                 const int32_t* tokens, const uint8_t* valid, int64_t T, int E, int k,
                                 float coefficient, void* grad, cudaStream_t stream) {
  if (T == 0) return STAGEML_OK;
  if (dtype == STAGEML_F32)
    return backward<float>(grad_loss, logits, counts, tokens, valid, T, E, k, coefficient, grad, stream);
  if (dtype == STAGEML_BF16)
    return backward<bf16>(grad_loss, logits, counts, tokens, valid, T, E, k, coefficient, grad, stream);
  return backward<f16>(grad_loss, logits, counts, tokens, valid, T, E, k, coefficient, grad, stream);
}

}  // namespace sb
