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
// Long batches: persistent CTAs that keep the channels' factors as fp32 (w_post times a
// per-channel gate in one array, w_pre in another), the forward in the registers of the
// columns' threads, the backward, whose column sums are there, in shared memory; read in their
// own types every row, their loads, branches and conversions were half of the instructions.
// The next rows arrive in shared memory by bulk copies (a ring of rows) while the current one
// is reduced, so HBM stays busy across the row sums.
//
// Weight gradients: with y^ normalised (or y), the post weight and a per-channel gate have
// gradients that are multiples, column by column, of the same sum over tokens
//   S[c] = sum_t s_t d y^,   dw_post = g S (s_t = 1, per-channel g) or S (s_t = g_t or g_tc),
//   dg = w_post S,
// so at most two sums per column (S and dw_pre's) are kept, in the registers of the thread
// that owns the column. Each CTA takes every gridDim-th row and writes its sums once; a second
// kernel adds them in CTA order: no atomics, the same bits on every run.
//
// Bound: HBM for the forward (8192 x 4096 bf16 in 45 us, 268 MB: 6.0 TB/s); the backward (109 us,
// 336 MB, 3.1 TB/s) by the issue slots, 70 % of which its arithmetic takes: two norms recomputed and
// two differentiated per element. Widths that are not multiples of 8 take scalar loads (777 x 2047,
// fp32 stream: forward 8, backward 19 us) and beyond 4096 columns more registers than there are.
#include <atomic>

#include "block_codes.cuh"
#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int kMaxThreads = 512;
constexpr int kWarpRows = 8, kWarpWidth = 256;  // rows of a warp each: per CTA, and up to this width
constexpr int kMaxH = 16384;  // 512 threads x 32 values
constexpr size_t kMaxSmem = 224 * 1024;  // dynamic shared memory of a CTA

template <int VEC, typename T>
__device__ __forceinline__ void load_vals(const T* p, float (&f)[VEC]) {
  if constexpr (VEC == 1) {
    // read-only as the vectors: a plain load would wait for the stores before it. By its bits: the
    // 16-bit types' own __ldg is a pure expression to the compiler, which may run it where the branch
    // around it (a null parameter, a column past the end) says not to.
    if constexpr (sizeof(T) == 2) {
      const unsigned short u = __ldg(reinterpret_cast<const unsigned short*>(p));
      f[0] = to_f32<T>(*reinterpret_cast<const T*>(&u));
    } else {
      f[0] = __ldg(p);
    }
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

// A thread's columns of a parameter, (v nt + tid) VEC and on for each v, 0 past the row's end. The
// branch on the type stands outside the loads: a branch per load made each wait for the one before
// (a row of 13831 columns in 26 us).
template <int VEC, int V, typename T>
__device__ __forceinline__ void load_columns(const T* p, int tid, int nt, int H, float (&f)[V][VEC]) {
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int c = (v * nt + tid) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[v][i] = 0.f;
    if (c < H) load_vals<VEC>(p + c, f[v]);
  }
}
template <int VEC, int V>
__device__ __forceinline__ void load_columns(const void* p, int dtype, int64_t base, int tid, int nt, int H,
                                             float (&f)[V][VEC]) {
  if (dtype == STAGEML_F32)
    load_columns<VEC, V>(static_cast<const float*>(p) + base, tid, nt, H, f);
  else if (dtype == STAGEML_BF16)
    load_columns<VEC, V>(static_cast<const bf16*>(p) + base, tid, nt, H, f);
  else
    load_columns<VEC, V>(static_cast<const f16*>(p) + base, tid, nt, H, f);
}

// The channels' factors of a thread's columns: w_post times a per-channel gate (1 where neither is
// given) and w_pre (0 without).
template <int VEC, int V>
__device__ __forceinline__ void load_y_factors(const stageml_norm_args& a, int tid, int nt, int H, float (&f)[V][VEC]) {
  if (a.post_weight) {
    load_columns<VEC, V>(a.post_weight, a.post_dtype, 0, tid, nt, H, f);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[v][i] = 1.f;
  }
  if (a.gate_mode == STAGEML_GATE_CHANNEL) {
    float g[V][VEC];
    load_columns<VEC, V>(a.gate, a.gate_dtype, 0, tid, nt, H, g);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[v][i] *= g[v][i];
  }
}
template <int VEC, int V>
__device__ __forceinline__ void load_z_factors(const stageml_norm_args& a, int tid, int nt, int H, float (&f)[V][VEC]) {
  if (a.pre_weight) {
    load_columns<VEC, V>(a.pre_weight, a.pre_dtype, 0, tid, nt, H, f);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[v][i] = 0.f;
  }
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

// Sums over the row's threads: a warp (WARP) or the CTA. `red` has 2 x 16 places; consecutive
// calls alternate between its halves, so one barrier per call is enough.
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
  const int lane = threadIdx.x & 15;
  float2 s = lane < (int)(blockDim.x >> 5) ? buf[lane] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
    s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
  }
  return s;
}
template <bool WARP>
__device__ __forceinline__ float row_sum(float a, float2* red, int& phase) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (WARP) return a;
  float2* buf = red + (phase ^= 1) * 16;
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5].x = a;
  __syncthreads();
  const int lane = threadIdx.x & 15;
  float s = lane < (int)(blockDim.x >> 5) ? buf[lane].x : 0.f;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// Values of a row: from global memory, or (SMEM) from the row's copy at a shared-memory address.
// The address is a 32-bit one, so that the loads are shared-memory loads (through a pointer
// they were generic ones).
__device__ __forceinline__ uint4 shared16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
template <typename T>
struct RowIn {
  const T* global;
  uint32_t shared;
};
template <bool SMEM, int VEC, typename T>
__device__ __forceinline__ void row_vals(const RowIn<T>& row, int c, float (&f)[VEC]) {
  if constexpr (!SMEM) {
    load_vals<VEC>(row.global + c, f);
  } else if constexpr (sizeof(T) == 2) {
    unpack8<T>(shared16(row.shared + 2 * c), f);
  } else {
    const uint4 a = shared16(row.shared + 4 * c), b = shared16(row.shared + 4 * c + 16);
    f[0] = __uint_as_float(a.x), f[1] = __uint_as_float(a.y), f[2] = __uint_as_float(a.z), f[3] = __uint_as_float(a.w);
    f[4] = __uint_as_float(b.x), f[5] = __uint_as_float(b.y), f[6] = __uint_as_float(b.z), f[7] = __uint_as_float(b.w);
  }
}

// A row's values held as they were loaded: eight 16-bit values take four registers, and the
// kernels that hold several rows' worth run out of registers before anything else.
template <int VEC, typename T>
struct Held {
  float f[VEC];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 0.f;
  }
  template <bool SMEM>
  __device__ __forceinline__ void load(const RowIn<T>& row, int c) {
    row_vals<SMEM, VEC>(row, c, f);
  }
  __device__ __forceinline__ void floats(float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = f[i];
  }
};
template <typename T>
struct Held16 {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  template <bool SMEM>
  __device__ __forceinline__ void load(const RowIn<T>& row, int c) {
    if constexpr (SMEM)
      u = shared16(row.shared + 2 * c);
    else
      u = __ldg(reinterpret_cast<const uint4*>(row.global + c));
  }
  __device__ __forceinline__ void floats(float (&v)[8]) const { unpack8<T>(u, v); }
};
template <>
struct Held<8, bf16> : Held16<bf16> {};
template <>
struct Held<8, f16> : Held16<f16> {};

// The channels' factors: w_post times a per-channel gate (1 where neither is given) and w_pre,
// from fp32 arrays in shared memory (STAGED) or from the parameters themselves.
// Vectors of 8: the first four values of every eight in one plane, the others in a second, so that
// the lanes of a 16-byte read are 16 bytes apart (32 apart they take two passes).
template <bool STAGED>
struct Factors {
  const stageml_norm_args& a;
  uint32_t y_at, z_at;
  bool has_y;
  template <int VEC>
  __device__ __forceinline__ static int place(int c, int H) {
    return VEC == 1 ? c : (c >> 3) * 4 + (c & 3) + (c & 4 ? H / 2 : 0);
  }
  template <int VEC>
  __device__ __forceinline__ void stage(float* smem) {
    has_y = a.post_weight || a.gate_mode == STAGEML_GATE_CHANNEL;
    y_at = smem_u32(smem);
    z_at = y_at + (has_y ? 4 * a.H : 0);
    if (!STAGED) return;
    float* z_factor = smem + (has_y ? a.H : 0);
    constexpr int V = 8 / VEC;  // 8 values per thread and turn
    for (int at = 0; at < a.H; at += 8 * blockDim.x) {
      const int tid = at / VEC + threadIdx.x;
      float fy[V][VEC], fz[V][VEC];
      if (has_y) load_y_factors<VEC, V>(a, tid, blockDim.x, a.H, fy);
      if (a.pre_weight) load_z_factors<VEC, V>(a, tid, blockDim.x, a.H, fz);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (v * blockDim.x + tid) * VEC;
        if (c >= a.H) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          if (has_y) smem[place<VEC>(c + i, a.H)] = fy[v][i];
          if (a.pre_weight) z_factor[place<VEC>(c + i, a.H)] = fz[v][i];
        }
      }
    }
    __syncthreads();
  }
  template <int VEC>
  __device__ __forceinline__ void read(uint32_t at, int c, float (&f)[VEC]) const {
    if constexpr (VEC == 1) {
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f[0]) : "r"(at + 4 * c));
    } else {
      const uint4 lo = shared16(at + 2 * c), hi = shared16(at + 2 * a.H + 2 * c);
      f[0] = __uint_as_float(lo.x), f[1] = __uint_as_float(lo.y), f[2] = __uint_as_float(lo.z), f[3] = __uint_as_float(lo.w);
      f[4] = __uint_as_float(hi.x), f[5] = __uint_as_float(hi.y), f[6] = __uint_as_float(hi.z), f[7] = __uint_as_float(hi.w);
    }
  }
  template <int VEC>
  __device__ __forceinline__ void y(int c, float (&f)[VEC]) const {
    if (STAGED && has_y) {
      read<VEC>(y_at, c, f);
      return;
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 1.f;
    if (STAGED) return;
    if (a.post_weight) load_param<VEC>(a.post_weight, a.post_dtype, c, f);
    if (a.gate_mode == STAGEML_GATE_CHANNEL) {
      float g[VEC];
      load_param<VEC>(a.gate, a.gate_dtype, c, g);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f[i] *= g[i];
    }
  }
  template <int VEC>
  __device__ __forceinline__ void z(int c, float (&f)[VEC]) const {
    if (STAGED)
      read<VEC>(z_at, c, f);
    else
      load_param<VEC>(a.pre_weight, a.pre_dtype, c, f);
  }
};
size_t factor_bytes(const stageml_norm_args& a) {
  return ((a.post_weight || a.gate_mode == STAGEML_GATE_CHANNEL ? 1 : 0) + (a.pre_weight ? 1 : 0)) * (size_t)a.H * 4;
}

// Ring of rows in dynamic shared memory, filled by bulk copies. Thread 0 issues the copies of
// row i + STAGES once every thread has read row i.
constexpr int kForwardStages = 3, kBackwardStages = 2;
template <int STAGES>
struct RowRing {
  uint8_t* base;
  uint32_t stage_bytes;
  uint64_t* full;          // [STAGES]
  volatile int* abort_flag;  // [2]: a wait has run out; rows whose copies have been issued
  int32_t* status;

  __device__ void init(uint8_t* smem, uint32_t bytes, uint64_t* bars, int* flag, int32_t* st) {
    base = smem, stage_bytes = bytes, full = bars, abort_flag = flag, status = st;
    if (threadIdx.x == 0) {
      for (int i = 0; i < STAGES; ++i) mbar_init(smem_u32(&full[i]), 1);
      flag[0] = flag[1] = 0;
      fence_barrier_init();
    }
    __syncthreads();
  }
  // The copies of the n-th row of this CTA (thread 0); null sources are left out. None after a wait has run out:
  // the stage may still be the target of earlier ones.
  __device__ void fill(uint32_t n, const void* const (&src)[4], const uint32_t (&bytes)[4]) {
    if (abort_flag[0]) return;
    abort_flag[1] = (int)n + 1;
    fence_proxy_async_smem();  // the stage's reads (ordered by the caller's barrier) come first
    const uint32_t bar = smem_u32(&full[n % STAGES]);
    uint32_t dst = smem_u32(base) + n % STAGES * stage_bytes, total = 0;
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
  __device__ uint32_t wait(uint32_t n) {
    mbar_wait(smem_u32(&full[n % STAGES]), (n / STAGES) & 1, abort_flag, status, kDefaultWaitNs,
              kDevTimeoutProducer);
    return smem_u32(base) + n % STAGES * stage_bytes;
  }
  // After the last row (thread 0): if a wait has run out, copies may still be on their way into this CTA's shared
  // memory; it does not leave before they have landed, or as much time has passed again.
  __device__ void drain() {
    if (!abort_flag[0]) return;
    volatile int never = 0;
    const uint32_t issued = (uint32_t)abort_flag[1];
    for (uint32_t n = issued > STAGES ? issued - STAGES : 0; n < issued; ++n)
      mbar_wait(smem_u32(&full[n % STAGES]), (n / STAGES) & 1, &never, status, kDefaultWaitNs, kDevTimeoutDrain);
  }
};

// Without a ring every input of a row is loaded before its first sum, while the values fit in
// registers: one memory latency per row instead of one per phase.
__host__ __device__ constexpr bool eager_loads(bool ring, int values) { return !ring && values <= 8; }

// HELD: persistent CTAs, the factors of a thread's columns in its registers.
template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING, bool HELD>
__global__ void __launch_bounds__(kMaxThreads) norm_residual_kernel(const stageml_norm_args a, float* z32) {
  constexpr int STAGES = kForwardStages;
  constexpr bool EAGER = eager_loads(RING, V * VEC);
  extern __shared__ __align__(128) uint8_t row_smem[];
  __shared__ float2 red[32];
  __shared__ uint64_t bars[STAGES];
  __shared__ int flag[2];
  int phase = 0;
  const int nt = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int H = a.H;
  const float inv_h = 1.f / (float)H;
  const uint32_t r_bytes = (uint32_t)H * sizeof(TR), y_bytes = (uint32_t)H * sizeof(TY);
  const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  RowRing<STAGES> ring;
  auto fill = [&](uint32_t n) {
    const int64_t row = first + n * step;
    if (row >= a.T) return;
    const void* src[4] = {static_cast<const TR*>(a.residual) + row * H,
                          a.block_out ? static_cast<const TY*>(a.block_out) + row * H : nullptr, nullptr, nullptr};
    const uint32_t bytes[4] = {r_bytes, y_bytes, 0, 0};
    ring.fill(n, src, bytes);
  };
  if constexpr (RING) {
    ring.init(row_smem, r_bytes + y_bytes, bars, flag, a.status);
    if (threadIdx.x == 0)
      for (int i = 0; i < STAGES; ++i) fill(i);
  }
  float fy[V][VEC], fz[V][VEC];
  if constexpr (HELD) {
    load_y_factors<VEC, V>(a, tid, nt, H, fy);
    load_z_factors<VEC, V>(a, tid, nt, H, fz);
  }
  uint32_t count = 0;
  for (int64_t row = first; row < a.T; row += step, ++count) {
    const int64_t base = row * H;
    RowIn<TR> r_row{static_cast<const TR*>(a.residual) + base, 0};
    RowIn<TY> y_row{static_cast<const TY*>(a.block_out) + base, 0};
    if constexpr (RING) {
      r_row.shared = ring.wait(count);
      y_row.shared = r_row.shared + r_bytes;
    }
    float n[V][VEC];
    Held<VEC, TR> r_in[EAGER ? V : 1];
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = 0.f;
      if (a.block_out && c < H) row_vals<RING, VEC>(y_row, c, n[v]);
      if constexpr (EAGER)
        if (c < H) r_in[v].template load<false>(r_row, c);
    }
    if constexpr (!HELD) {
      load_y_factors<VEC, V>(a, tid, nt, H, fy);
      if constexpr (EAGER) load_z_factors<VEC, V>(a, tid, nt, H, fz);
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sq = fmaf(n[v][i], n[v][i], sq);
    // with held factors the full gate's few vectors are loaded one by one below: together they take the
    // registers of a third CTA per SM (8192 x 4096 in 51 us, not 45)
    if (!(HELD && VEC == 8) && a.block_out && a.gate_mode == STAGEML_GATE_FULL) {
      float g[V][VEC];
      load_columns<VEC, V>(a.gate, a.gate_dtype, base, tid, nt, H, g);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[v][i] *= g[v][i];
    }
    float scale = a.gate_mode == STAGEML_GATE_TOKEN ? load_param1(a.gate, a.gate_dtype, row) : 1.f;
    if (a.post_weight) scale *= rsqrtf(row_sum<WARP>(sq, red, phase) * inv_h + a.eps);
    sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      if (c >= H) continue;
      if (a.block_out) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[v][i] *= fy[v][i];
        if (HELD && VEC == 8 && a.gate_mode == STAGEML_GATE_FULL) {
          float g[VEC];
          load_param<VEC>(a.gate, a.gate_dtype, base + c, g);
#pragma unroll
          for (int i = 0; i < VEC; ++i) n[v][i] *= g[i];
        }
      }
      float r[VEC];
      if constexpr (EAGER)
        r_in[v].floats(r);
      else
        row_vals<RING, VEC>(r_row, c, r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        n[v][i] = fmaf(n[v][i], scale, a.residual_scale * r[i]);
        sq = fmaf(n[v][i], n[v][i], sq);
      }
      store_vals<VEC>(static_cast<TR*>(a.new_residual) + base + c, n[v]);
    }
    float inv = 0.f;
    if (a.pre_weight)
      inv = rsqrtf(row_sum<WARP>(sq, red, phase) * inv_h + a.eps);
    else if (RING)
      __syncthreads();
    // the row's copy has been read by every thread (the barrier above)
    if constexpr (RING)
      if (threadIdx.x == 0) fill(count + STAGES);
    if (!a.pre_weight) continue;
    if constexpr (!HELD && !EAGER) load_z_factors<VEC, V>(a, tid, nt, H, fz);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      float w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = n[v][i] * inv * fz[v][i];
      if constexpr (VEC == 8) {
        if (a.codes) {
          // 16 neighbouring lanes hold one block of 128 columns
          uint32_t m = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) m = max(m, c < H ? abs_bits(w[i]) : 0u);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
          const BlockScale s(m);
          if (c < H) {
            *reinterpret_cast<uint2*>(a.codes + base + c) = s.encode_signed8(w);
            if ((c & 127) == 0) a.code_scale[row * ((H + 127) / 128) + (c >> 7)] = s.s;
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
  if constexpr (RING)
    if (threadIdx.x == 0) ring.drain();
}

// Column sums that the backward keeps: S (for the post weight and a per-channel gate), dw_pre.
__host__ __device__ inline bool has_block_sum(const stageml_norm_args& a) {
  return a.post_weight || a.gate_mode == STAGEML_GATE_CHANNEL;
}
__host__ __device__ inline int n_sums_of(const stageml_norm_args& a) {
  return (has_block_sum(a) ? 1 : 0) + (a.pre_weight ? 1 : 0);
}

template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING, bool STAGED>
__global__ void __launch_bounds__(kMaxThreads, (RING && V == 1) || (!RING && V * VEC <= 4) ? 2 : 1)
    norm_residual_backward_kernel(const stageml_norm_args a, float* partial) {
  constexpr int STAGES = kBackwardStages;
  constexpr bool EAGER = eager_loads(RING, V * VEC);
  extern __shared__ __align__(128) uint8_t row_smem[];
  __shared__ float2 red[32];
  __shared__ uint64_t bars[STAGES];
  __shared__ int flag[2];
  int phase = 0;
  const int nt = WARP ? 32 : blockDim.x, tid = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int H = a.H;
  const float inv_h = 1.f / (float)H;
  const bool post = a.post_weight != nullptr, pre = a.pre_weight != nullptr && a.grad_normed != nullptr;
  const bool has_y = a.block_out != nullptr;
  const uint32_t r_bytes = (uint32_t)H * sizeof(TR), y_bytes = (uint32_t)H * sizeof(TY);
  const int64_t first = WARP ? (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? (int64_t)gridDim.x * (blockDim.x >> 5) : gridDim.x;
  RowRing<STAGES> ring;
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
    ring.init(row_smem, 2 * (r_bytes + y_bytes), bars, flag, a.status);
    if (threadIdx.x == 0)
      for (int i = 0; i < STAGES; ++i) fill(i);
  }
  Factors<STAGED> factors{a};
  factors.template stage<VEC>(reinterpret_cast<float*>(row_smem + (RING ? 2 * STAGES * (r_bytes + y_bytes) : 0)));
  float sum_y[V][VEC], sum_z[V][VEC];  // this thread's columns: S and dw_pre
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum_y[v][i] = sum_z[v][i] = 0.f;
  uint32_t count = 0;
  for (int64_t row = first; row < a.T; row += step, ++count) {
    const int64_t base = row * H;
    RowIn<TR> r_row{static_cast<const TR*>(a.residual) + base, 0}, dr_row{static_cast<const TR*>(a.grad_residual) + base, 0};
    RowIn<TY> y_row{static_cast<const TY*>(a.block_out) + base, 0}, dz_row{static_cast<const TY*>(a.grad_normed) + base, 0};
    if constexpr (RING) {
      r_row.shared = ring.wait(count);
      dr_row.shared = r_row.shared + r_bytes;
      y_row.shared = dr_row.shared + r_bytes;
      dz_row.shared = y_row.shared + y_bytes;
    }
    Held<VEC, TY> y_in[V], dz_in[V];
    Held<VEC, TR> r_in[EAGER ? V : 1], dr_in[EAGER ? V : 1];
    float n[V][VEC], d[V][VEC];
    // With f the channel's factor and g a gate that is not part of it: n = a r + f g y inv_y.
    const bool full = has_y && a.gate_mode == STAGEML_GATE_FULL;
    const float token_gate = a.gate_mode == STAGEML_GATE_TOKEN ? load_param1(a.gate, a.gate_dtype, row) : 1.f;
    float inv_y = 1.f;
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      y_in[v].zero();
      if (c < H && has_y) y_in[v].template load<RING>(y_row, c);
      if constexpr (EAGER) {
        dz_in[v].zero(), dr_in[v].zero();
        if (c < H) {
          r_in[v].template load<false>(r_row, c);
          if (pre) dz_in[v].template load<false>(dz_row, c);
          if (a.grad_residual) dr_in[v].template load<false>(dr_row, c);
        }
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float y[VEC];
      y_in[v].floats(y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) sq = fmaf(y[i], y[i], sq);
    }
    if (full) {
      load_columns<VEC, V>(a.gate, a.gate_dtype, base, tid, nt, H, n);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[v][i] = has_y ? 1.f : 0.f;
    }
    if (post) inv_y = rsqrtf(row_sum<WARP>(sq, red, phase) * inv_h + a.eps);
    const float y_scale = inv_y * token_gate;
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      if constexpr (!EAGER) dz_in[v].zero();
      if (c >= H) continue;
      if (has_y) {
        float f[VEC], y[VEC];
        factors.template y<VEC>(c, f);
        y_in[v].floats(y);
#pragma unroll
        for (int i = 0; i < VEC; ++i) n[v][i] *= y[i] * f[i];
      }
      float r[VEC];
      if constexpr (EAGER)
        r_in[v].floats(r);
      else
        row_vals<RING, VEC>(r_row, c, r);
#pragma unroll
      for (int i = 0; i < VEC; ++i) n[v][i] = fmaf(n[v][i], y_scale, a.residual_scale * r[i]);
      if (pre) {
        float f[VEC], dz[VEC];
        if constexpr (!EAGER) dz_in[v].template load<RING>(dz_row, c);
        dz_in[v].floats(dz);
        factors.template z<VEC>(c, f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          s1 = fmaf(n[v][i], n[v][i], s1);
          s2 = fmaf(dz[i] * f[i], n[v][i], s2);
        }
      }
    }
    float inv_n = 0.f, c_n = 0.f;
    if (pre) {
      const float2 s = row_sum<WARP>(s1, s2, red, phase);
      inv_n = rsqrtf(s.x * inv_h + a.eps);
      c_n = s.y * inv_h * inv_n * inv_n * inv_n;  // n^ mean(dn n^) inv_n = n c_n
    }
    // d, dr and the column sums; then d becomes p = f g d inv_y, the part of dy that needs no
    // further row sum: dy = p - y inv_y^2 mean(p y)
    float s3 = 0.f;
    float gates[VEC == 1 ? V : 1][VEC];
    if constexpr (VEC == 1)
      if (full) load_columns<VEC, V>(a.gate, a.gate_dtype, base, tid, nt, H, gates);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[v][i] = 0.f;
      if (c >= H) continue;
      float t[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = 0.f;
      if constexpr (EAGER)
        dr_in[v].floats(t);
      else if (a.grad_residual)
        row_vals<RING, VEC>(dr_row, c, t);
      if (pre) {
        float f[VEC], dz[VEC];
        factors.template z<VEC>(c, f);
        dz_in[v].floats(dz);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float e = dz[i] * inv_n;
          sum_z[v][i] = fmaf(e, n[v][i], sum_z[v][i]);
          d[v][i] = fmaf(e, f[i], fmaf(-c_n, n[v][i], t[i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) d[v][i] = t[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = a.residual_scale * d[v][i];
      store_vals<VEC>(static_cast<TR*>(a.d_residual) + base + c, t);
      if (!has_y) continue;
      float f[VEC], y[VEC];
      factors.template y<VEC>(c, f);
      y_in[v].floats(y);
      if (full) {
        float g[VEC];
        if constexpr (VEC == 1)
          g[0] = gates[v][0];
        else
          load_param<VEC>(a.gate, a.gate_dtype, base + c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float e = d[v][i] * inv_y, p = e * f[i];
          t[i] = p * y[i];  // dg
          sum_y[v][i] = fmaf(e * g[i], y[i], sum_y[v][i]);
          d[v][i] = p * g[i];
          s3 = fmaf(d[v][i], y[i], s3);
        }
        store_param<VEC>(a.d_gate, a.gate_dtype, base + c, t);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {  // without the token's gate, which multiplies the sums
          const float e = d[v][i] * inv_y;
          sum_y[v][i] = fmaf(e * token_gate, y[i], sum_y[v][i]);
          d[v][i] = e * f[i];
          s3 = fmaf(d[v][i], y[i], s3);
        }
      }
    }
    float c_y = 0.f;
    if (has_y && (post || a.gate_mode == STAGEML_GATE_TOKEN)) {
      s3 = row_sum<WARP>(s3, red, phase);
      if (a.gate_mode == STAGEML_GATE_TOKEN && tid == 0) store_param1(a.d_gate, a.gate_dtype, row, s3);
      if (post) c_y = s3 * token_gate * inv_h * inv_y * inv_y;
    } else if (RING) {
      __syncthreads();
    }
    // the row's copies have been read by every thread (the barrier above)
    if constexpr (RING)
      if (threadIdx.x == 0) fill(count + STAGES);
    if (!has_y) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * nt + tid) * VEC;
      if (c >= H) continue;
      float t[VEC], y[VEC];
      y_in[v].floats(y);
#pragma unroll
      for (int i = 0; i < VEC; ++i) t[i] = fmaf(-c_y, y[i], token_gate * d[v][i]);
      store_vals<VEC>(static_cast<TY*>(a.d_block_out) + base + c, t);
    }
  }
  if constexpr (RING)
    if (threadIdx.x == 0) ring.drain();
  if (n_sums_of(a) == 0) return;
  float* out = partial + (int64_t)blockIdx.x * n_sums_of(a) * H;
  if constexpr (WARP) {
    // the warps' sums are added first: an owner per warp left the second kernel thousands of rows
    __shared__ float warps[kWarpRows][kWarpWidth];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      if (which == 0 ? !has_block_sum(a) : !a.pre_weight) continue;
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (v * nt + tid) * VEC;
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (c < H) warps[threadIdx.x >> 5][c + i] = which == 0 ? sum_y[v][i] : sum_z[v][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < H; c += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kWarpRows; ++w) s += warps[w][c];
        out[(which == 1 && has_block_sum(a) ? H : 0) + c] = s;
      }
    }
    return;
  }
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
  pdl_wait();
  const int lane = threadIdx.x & 31, strand = threadIdx.x >> 5;
  const int64_t width = (int64_t)n_sums * a.H, i = (int64_t)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (i < width) {
    for (int at = strand; at < owners; at += 8 * kStrands) {  // eight loads at a time, the last turn's too
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int c = at + j * kStrands;
        s += c < owners ? __ldg(partial + c * width + i) : 0.f;
      }
    }
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
  if (warp) return {32 * kWarpRows, kWarpRows};
  return {std::min(kMaxThreads, ((units + per - 1) / per + 31) / 32 * 32), 1};
}

// Persistent CTAs of a kernel of `threads` threads and `smem` bytes: as many as fit in an SM's
// registers and shared memory, at most `rows`. The kernel may then be launched with up to kMaxSmem.
// The two calls cost 2 to 3 us; `last` keeps the kernel's latest answer with the device, threads and
// bytes that it is for.
template <typename K>
int resident_ctas(std::atomic<uint64_t>& last, K kernel, int threads, size_t smem, int64_t rows, int* grid) {
  int dev = 0, per_sm = 0;
  SB_CUDA_CHECK(cudaGetDevice(&dev));
  const uint64_t key = (uint64_t)(dev + 1) << 48 | (uint64_t)threads << 32 | (uint64_t)smem << 8;
  const uint64_t known = last.load(std::memory_order_relaxed);
  if ((known & ~uint64_t(0xff)) == key) {
    per_sm = (int)(known & 0xff);
  } else {
    if (smem > 40 * 1024)  // 48 KB with the static part need no leave
      SB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem));
    SB_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem));
    per_sm = std::max(per_sm, 1);
    last.store(key | (uint64_t)per_sm, std::memory_order_relaxed);
  }
  *grid = (int)std::min<int64_t>(rows, (int64_t)sm_count() * per_sm);
  return STAGEML_OK;
}

template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING, bool STAGED>
int run_forward(const stageml_norm_args& a, const Shape& s, float* z32, cudaStream_t stream) {
  auto kernel = norm_residual_kernel<TR, TY, VEC, V, WARP, RING, STAGED>;
  static std::atomic<uint64_t> resident{0};
  int grid = (int)((a.T + s.rows_per_cta - 1) / s.rows_per_cta);
  size_t smem = 0;
  if (STAGED) {
    smem = RING ? (size_t)kForwardStages * a.H * (sizeof(TR) + sizeof(TY)) : 0;
    SB_TRY(resident_ctas(resident, kernel, s.threads, smem, a.T, &grid));
  }
  SB_CUDA_CHECK(launch_kernel(kernel, dim3((unsigned)grid), dim3(s.threads), smem, stream, false, a, z32));
  count_launch();
  return STAGEML_OK;
}

// With `owners` only its grid, the number of CTAs that each leave a row of column sums.
template <typename TR, typename TY, int VEC, int V, bool WARP, bool RING, bool STAGED>
int run_backward(const stageml_norm_args& a, const Shape& s, float* partial, int* owners, cudaStream_t stream) {
  auto kernel = norm_residual_backward_kernel<TR, TY, VEC, V, WARP, RING, STAGED>;
  const int n_sums = n_sums_of(a);
  size_t smem = 0;
  if (STAGED)
    smem = (RING ? (size_t)kBackwardStages * a.H * 2 * (sizeof(TR) + sizeof(TY)) : 0) + factor_bytes(a);
  static std::atomic<uint64_t> resident{0};
  int grid = 0;
  // a warp takes four rows or more, for fewer rows of sums
  const int64_t ctas = WARP ? (a.T + 4 * kWarpRows - 1) / (4 * kWarpRows) : a.T;
  SB_TRY(resident_ctas(resident, kernel, s.threads, smem, ctas, &grid));
  if (owners) {
    *owners = grid;
    return STAGEML_OK;
  }
  SB_CUDA_CHECK(launch_kernel(kernel, dim3((unsigned)grid), dim3(s.threads), smem, stream, false, a, partial));
  count_launch();
  if (n_sums) {
    const int64_t width = (int64_t)n_sums * a.H;
    SB_CUDA_CHECK(launch_kernel(norm_weight_sums_kernel, dim3((unsigned)((width + 31) / 32)), dim3(32 * kStrands), 0,
                                stream, true, a, (const float*)partial, grid, n_sums));
    count_launch();
  }
  return STAGEML_OK;
}

template <typename TR, typename TY>
int dispatch(const stageml_norm_args& a, bool backward, float* scratch, int* owners, cudaStream_t stream) {
#define SB_NORM(VEC, V, WARP, RING, STAGED, units) \
  (backward ? run_backward<TR, TY, VEC, V, WARP, RING, STAGED>(a, shape_of(units, V, WARP), scratch, owners, stream) \
            : run_forward<TR, TY, VEC, V, WARP, RING, STAGED>(a, shape_of(units, V, WARP), scratch, stream))
  // Few rows run straight from global memory with as many threads per row as possible; more
  // than two rows per SM are worth a CTA's staged factors, and so is one row of the scalar backward,
  // which reads them three times.
  const bool many = a.T > 2 * (int64_t)sm_count();
  if (vectors(a)) {
    const int units = a.H / 8;
    if (a.H <= kWarpWidth) return SB_NORM(8, 1, true, false, false, units);
    const size_t row = a.H * (sizeof(TR) + sizeof(TY));
    const size_t ring = backward ? 2 * kBackwardStages * row + factor_bytes(a) : kForwardStages * row;
    if (!many || ring > kMaxSmem) {
      if (units <= kMaxThreads) return SB_NORM(8, 1, false, false, false, units);
      if (units <= 2 * kMaxThreads) return SB_NORM(8, 2, false, false, false, units);
      return SB_NORM(8, 4, false, false, false, units);
    }
    if (units <= (backward ? kMaxThreads : 256)) return SB_NORM(8, 1, false, true, true, units);
    if (units <= 2 * kMaxThreads) return SB_NORM(8, 2, false, true, true, units);
    return SB_NORM(8, 4, false, true, true, units);
  }
  if (a.H <= kWarpWidth) return SB_NORM(1, 8, true, false, false, a.H);
#define SB_NORM_SCALAR(V) \
  (many || backward ? SB_NORM(1, V, false, false, true, a.H) \
                    : run_forward<TR, TY, 1, V, false, false, false>(a, shape_of(a.H, V, false), scratch, stream))
  if (a.H <= 4 * kMaxThreads) return SB_NORM_SCALAR(4);
  if (a.H <= 8 * kMaxThreads) return SB_NORM_SCALAR(8);
  return SB_NORM_SCALAR(32);
#undef SB_NORM_SCALAR
#undef SB_NORM
}

int launch_any(const stageml_norm_args& a, bool backward, float* scratch, int* owners, cudaStream_t stream) {
  if (a.resid_dtype == STAGEML_BF16) return dispatch<bf16, bf16>(a, backward, scratch, owners, stream);
  if (a.resid_dtype == STAGEML_F16) return dispatch<f16, f16>(a, backward, scratch, owners, stream);
  if (a.block_dtype == STAGEML_BF16) return dispatch<float, bf16>(a, backward, scratch, owners, stream);
  if (a.block_dtype == STAGEML_F16) return dispatch<float, f16>(a, backward, scratch, owners, stream);
  return dispatch<float, float>(a, backward, scratch, owners, stream);
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
  SB_TRY(launch_any(a, false, two_step ? static_cast<float*>(scratch) : nullptr, nullptr, stream));
  if (two_step)
    return launch_quantize_block_rows(scratch, STAGEML_F32, a.T, a.H, nullptr, 0, a.codes, a.code_scale, stream);
  return STAGEML_OK;
}

size_t norm_residual_backward_scratch(const stageml_norm_args& a) {
  if (a.T == 0 || n_sums_of(a) == 0) return 0;
  int owners = 0;
  if (launch_any(a, true, nullptr, &owners, nullptr) != STAGEML_OK) {
    // no device to ask: 32 CTAs of 64 threads fill an SM
    clear_error();
    owners = (int)std::min<int64_t>(a.T, (int64_t)sm_count() * 32);
  }
  return (size_t)owners * n_sums_of(a) * a.H * 4;
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
  return launch_any(a, true, static_cast<float*>(scratch), nullptr, stream);
}

}  // namespace sb
