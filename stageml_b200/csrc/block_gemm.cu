// e4m3 x e4m3 matrix product with one fp32 scale per 128 values of K (and per 128
// output columns for the weights), plain or grouped by expert:
//
//   out[r, n] = sum_kb sa[r, kb] * sb[n / 128, kb] * (sum_{k in block kb} a[r, k] * b[n, k])
//
// The inner sum of one K block runs on the tensor cores (tcgen05.mma kind::f8f6f4,
// K = 32 per instruction) into a fresh fp32 accumulator in TMEM; math warps then read it,
// multiply by the block's scale and add it to the tile's sums in their registers. What
// bounds such a kernel is the round trip of an accumulator (MMAs, signal, TMEM read,
// signal), so the 512 TMEM columns are four accumulators of 128 columns in rotation: with
// two of 256 columns the same tile ran at 1250 to 1700 clocks per K block instead of 512.
//
// Pair kernel: a two-CTA cluster computes 256 rows x 256 columns with cta_group::2 MMAs of
// M = 256, N = 128 (two halves per K block); each CTA stages its own 128 rows of A and
// half of the B rows (32 KB per K block instead of 48), six stages. Per CTA: warp 0 TMA
// producer, warps 1 and 3 (even CTA) MMA issue, one half each, warp 2 the K blocks' scales
// (asynchronous copies to shared memory), warps 4..11 scaling and epilogue: a warp owns 32
// TMEM lanes of one half, 128 fp32 sums per thread, and reads the next 16 columns while it
// adds the last 16. Eight warps of 128 sums, not sixteen of 64: a scheduler's budget is 512
// issue slots per K block, 256 of them the additions, and every warp pays its own waits.
// The control warps give registers to the math warps. Persistent clusters.
//
// A unit of one row tile (a short batch, the odd last tile of an expert) is narrow: 64 rows per CTA,
// MMAs of M = 128, whose accumulators hold columns [0, 64) of a half in lanes 0..63 and [64, 128) in
// lanes 64..127: 64 sums per thread, half the work of a pair with an idle CTA. 64 experts of 2048 x
// 1408 with at most 128 rows each in 195 us (two CTAs per tile: 250); 64 x 4096 x 4096 in 11.5 us.
//
// SwiGLU: half h of a tile is 64 gate rows and the matching 64 up rows of B, so a thread
// holds the gate and up values of the same columns; the epilogue forms
// h = silu(gate) * up in fp32 and writes it as e4m3 codes with one scale per (row, 128
// columns), the next product's operand, so h never exists in 16 bits.
//
// Measured: 2048 x 11008 x 4096 in 103 to 109 us (1.7 to 1.8 PFLOP/s) in a run of calls, where the board's
// 1 kW holds the clock at 1.65 GHz, 92 us (2.0) in short ones; the accumulator round trip and then power bound
// it, the tensor pipe is active half of the time.
//
// Plain products of few tiles: clusters of two or four pairs, each with its share of a tile's K blocks;
// the sums meet over distributed shared memory, in a fixed order, and each pair stores its share of
// the columns.
//
// Every wait is bounded. No load is multicast.
#include <atomic>

#include "block_fp8.h"
#include "common.cuh"
#include "host_util.h"

namespace sb {
namespace {

constexpr int BM = 128;                  // rows per CTA
constexpr int BN = 256;                  // columns of a pair tile
constexpr int BK = 128;                  // e4m3 values = one 128-byte swizzle row = one scale block
constexpr int NACC = 128;                // columns of one accumulator
constexpr int A_BYTES = BM * BK;         // 16 KB
constexpr int B_HALF_BYTES = 64 * BK;    // this CTA's 64 rows of one half: 8 KB
constexpr int STAGE_BYTES = A_BYTES + 2 * B_HALF_BYTES;
constexpr int STAGES = 6;
constexpr int BUFS = 4;                  // TMEM accumulators
constexpr int TMEM_COLS = BUFS * NACC;
constexpr int MATH_WARP0 = 4;
constexpr int HALF_WARPS = 4;            // math warps per half
constexpr int THREADS = 32 * (MATH_WARP0 + 2 * HALF_WARPS);
// 384 threads are launched with 168 registers each; 128 x 80 + 256 x 208 is less than the total.
constexpr int CONTROL_REGS = 80, MATH_REGS = 208;
static_assert(128 * CONTROL_REGS + 256 * MATH_REGS <= THREADS * 168, "register split");
// Scales come in groups of four K blocks, so that the math warps wait for them once in four:
// [128 rows of A][4], then [3 weight scales][4].
constexpr int GROUP = 4;
constexpr int SLOTS = 3;
constexpr int SLOT_FLOATS = (BM + 4) * GROUP;
constexpr int MAX_GROUPS = 1024;
constexpr int kBandUnits = 8;            // plain rows: row units that share a pass over the columns
constexpr int BAR_BYTES = 512;
constexpr int TURN_PITCH = 17;           // floats per row of a math warp's 32 x 16 turning area
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 /*align*/ + BAR_BYTES + 2 * 2 * BM * 4 /*row maxima*/ +
                           SLOTS * SLOT_FLOATS * 4 + 2 * HALF_WARPS * 32 * TURN_PITCH * 4 + 2 * (MAX_GROUPS + 1) * 4;
static_assert(BUFS == 4, "two halves, two K blocks in flight");
static_assert(SMEM_BYTES <= 232448, "shared memory per block");
static_assert((2 * STAGES + 2 * BUFS + 2 + 2 * SLOTS) * 8 + 16 <= BAR_BYTES, "barrier area");

struct Params {
  int K, N, kb;                 // kb = ceil(K / 128)
  int b_group_rows, b_blocks;   // rows and 128-row scale blocks of one weight group
  int n_tiles;
  const float* a_scale;
  const float* b_scale;
  int vec_scales;               // four scales of a row are one aligned 16-byte load
  const int32_t* group_offsets; // grouped rows: [groups + 1] padded row offsets; null: plain rows
  const int32_t* group_counts;  // grouped rows: [groups] rows without the padding
  int groups;
  int64_t rows;
  const float* row_scale;
  void* out;
  uint8_t* q_out;
  float* q_scale;
  int32_t* status;
};

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void mma_f8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of kind::f8f6f4: f32 accumulator, both operands e4m3 (format 0), K-major.
__host__ __device__ constexpr uint32_t idesc_e4m3(int M, int N) {
  return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// Asynchronous copy of BYTES (4 or 16) global -> shared, zeros when not valid.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const float* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(valid ? BYTES : 0)
               : "memory");
}
// This thread's arrival on `bar` (counted at its initialisation) once its copies so far have landed.
__device__ __forceinline__ void copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// The wait of a whole warp, which then stays or leaves together. Every lane polls (one
// instruction for the warp); nothing but the poll and a vote lies on the path of a wait that is
// already over. Bounded by the SM's clock.
constexpr uint32_t kWaitClocks = 2000000000u;  // about 1 s
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint32_t abort_flag, int* err, int code) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const uint32_t t0 = (uint32_t)clock();
#pragma unroll 1
  while (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
    uint32_t gone;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(gone) : "r"(abort_flag) : "memory");
    const bool late = (uint32_t)clock() - t0 > kWaitClocks;
    if (__any_sync(0xffffffffu, gone || late)) {
      if (late) {
        asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort_flag), "r"(1) : "memory");
        if (err) atomicCAS(err, 0, code);
      }
      __syncwarp();
      return false;
    }
  }
  return true;
}

// The same for a role of one thread; `also` is a second barrier waited for at the same time, so
// that the polls' latencies overlap.
__device__ __forceinline__ bool lane_wait(uint32_t bar, uint32_t parity, uint32_t also, uint32_t also_parity,
                                          uint32_t abort_flag, int* err, int code) {
  bool a = mbar_try_wait(bar, parity), b = mbar_try_wait(also, also_parity);
  if (a && b) return true;
  const uint32_t t0 = (uint32_t)clock();
#pragma unroll 1
  while (true) {
    if (!a) a = mbar_try_wait(bar, parity);
    if (!b) b = mbar_try_wait(also, also_parity);
    if (a && b) return true;
    uint32_t gone;
    asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(gone) : "r"(abort_flag) : "memory");
    if (gone) return false;
    if ((uint32_t)clock() - t0 > kWaitClocks) {
      asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(abort_flag), "r"(1) : "memory");
      if (err) atomicCAS(err, 0, code);
      return false;
    }
  }
}

// Arrive on a barrier of either CTA where no memory is handed over (tensor-memory reads are
// ordered by the tcgen05 fences around it): no cluster-scope release, whose flush every K block of every warp would pay for.
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// A work unit: up to `step` consecutive row tiles of one weight group, one column tile.
struct Unit {
  int m, n, group;  // m = first row tile
  int tiles;        // row tiles of the unit
  int rows;         // grouped rows: without the padding of the group's last tile
};

// first[g] = row units of the groups before g, begin[g] = 128 times their row tiles, plus the rows of padding
// that end group g (less than 128; grouped rows), in shared memory: read from global memory for each unit,
// they were 0.7 us of every role's unit. One warp.
__device__ __forceinline__ void group_units(const Params& p, int step, int32_t* first, int32_t* begin) {
  const int lane = threadIdx.x & 31;
  for (int g = lane; g <= p.groups; g += 32)
    begin[g] = g < p.groups ? p.group_offsets[g + 1] - p.group_counts[g] : p.group_offsets[g];
  __syncwarp();
  int base = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    int c = 0;
    if (g < p.groups) c = (begin[g + 1] / BM - begin[g] / BM + step - 1) / step;
    int s = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += v;
    }
    if (g < p.groups) first[g] = base + s - c;
    base += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) first[p.groups] = base;
}

// Unit u -> row tiles and column tile. All column tiles of a weight group's row units (or of
// a band of plain row units) come before the next group, row units fastest, so that the
// CTAs at work at one time share weight tiles and the group's rows stay in L2.
template <bool GROUPED>
__device__ __forceinline__ Unit unit_of(const Params& p, int u, int step, const int32_t* first, const int32_t* begins) {
  Unit w;
  // the pointer is always there for grouped rows; without the test the SwiGLU kernel is allocated otherwise and
  // spills (64 experts of 2048 x 1408, 43 tokens: 206 us)
  if (GROUPED && p.group_offsets) {
    const int r = u / p.n_tiles;
    int lo = 0, hi = p.groups - 1;  // the last group with first[g] <= r (empty groups are passed over)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first[mid] <= r)
        lo = mid;
      else
        hi = mid - 1;
    }
    const int begin = begins[lo] / BM, tiles = begins[lo + 1] / BM - begin;
    const int cnt = first[lo + 1] - first[lo], local = u - first[lo] * p.n_tiles;
    w.group = lo;
    w.n = local / cnt;
    const int m = (local - w.n * cnt) * step;
    w.m = begin + m;
    w.tiles = min(step, tiles - m);
    w.rows = w.tiles * BM - (m + w.tiles == tiles ? begins[lo] % BM : 0);
  } else {
    const int tiles = (int)((p.rows + BM - 1) / BM), all = (tiles + step - 1) / step;
    const int band = u / (p.n_tiles * kBandUnits) * kBandUnits;
    const int cnt = min(kBandUnits, all - band), local = u - band * p.n_tiles;
    w.group = 0;
    w.n = local / cnt;
    const int m = (band + local - w.n * cnt) * step;
    w.m = m;
    w.tiles = min(step, tiles - m);
    w.rows = 0;
  }
  return w;
}

// Four lanes hold a row each, in four pieces of 16 bytes; afterwards lane i of the four holds piece
// i of the four rows (v[r] of row r). A thread of the epilogue owns a row, and a warp's store of one
// piece per row touches 32 lines, one per clock; transposed it touches 8 (64 bytes of each row).
__device__ __forceinline__ void transpose_pieces(uint4 (&v)[4]) {
  const bool hi = threadIdx.x & 2, odd = threadIdx.x & 1;
  auto swap = [](uint4& a, uint4& b, bool up, int mask) {  // up: a goes, else b
    uint4 t = up ? a : b;
    t.x = __shfl_xor_sync(0xffffffffu, t.x, mask);
    t.y = __shfl_xor_sync(0xffffffffu, t.y, mask);
    t.z = __shfl_xor_sync(0xffffffffu, t.z, mask);
    t.w = __shfl_xor_sync(0xffffffffu, t.w, mask);
    (up ? a : b) = t;
  };
  swap(v[0], v[2], hi, 2);
  swap(v[1], v[3], hi, 2);
  swap(v[0], v[1], odd, 1);
  swap(v[2], v[3], odd, 1);
}

// 16 bytes of outputs from the sums.
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* f) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f[i];
    return pack8<T>(v);
  }
}

// Stores W columns of a row per thread, the warp's 32 rows four by four (rows4 of `row`'s four exist);
// where the rows do not start at 16 bytes, 16 columns at a time through `turn`, so that a warp's store
// is of two rows' 16 columns (a thread storing its own row: 300 x 500 x 1536 in 44 us).
template <typename OutT, int W>
__device__ __forceinline__ void store_columns(const Params& p, float* v, float factor, int64_t row, int rows4, int n0,
                                              float* turn) {
  constexpr int PIECE = 16 / (int)sizeof(OutT);
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] *= factor;
  const int mine = threadIdx.x & 3;
  if (W < 4 * PIECE && p.N % PIECE == 0) {
    OutT* out = static_cast<OutT*>(p.out) + row * p.N + n0;
#pragma unroll
    for (int c = 0; c < W; c += PIECE)
      if (rows4 > mine && n0 + c < p.N) *reinterpret_cast<uint4*>(out + c) = pack16<OutT>(v + c);
  } else if (p.N % PIECE == 0) {
    OutT* out = static_cast<OutT*>(p.out) + (row - mine) * p.N + n0 + PIECE * mine;
#pragma unroll
    for (int c = 0; c + 4 * PIECE <= W; c += 4 * PIECE) {
      if (n0 + c >= p.N) break;
      uint4 u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = pack16<OutT>(v + c + PIECE * i);
      transpose_pieces(u);
      if (n0 + c + PIECE * mine < p.N) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < rows4) *reinterpret_cast<uint4*>(out + (int64_t)r * p.N + c) = u[r];
      }
    }
  } else {
    const int lane = threadIdx.x & 31;
    const int64_t row0 = row - lane;
#pragma unroll
    for (int c = 0; c < W; c += 16) {
      if (n0 + c >= p.N) break;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 16; ++i) turn[lane * TURN_PITCH + i] = v[c + i];
      __syncwarp();
      const int n = n0 + c + (lane & 15);
      OutT* out = static_cast<OutT*>(p.out) + (row0 + (lane >> 4)) * p.N + n;
#pragma unroll 4
      for (int r = 0; r < 32; r += 2, out += 2 * (int64_t)p.N) {
        const float f = turn[(r + (lane >> 4)) * TURN_PITCH + (lane & 15)];
        // rows4 of the lane that owns this row tells whether it exists
        const int there = __shfl_sync(0xffffffffu, rows4, r + (lane >> 4));
        if (n < p.N && there > ((r + (lane >> 4)) & 3)) *out = from_f32<OutT>(f);
      }
    }
  }
}

// The sums of a cluster's S pairs, each over its share of K: pair q ends with the tile's q-th 128 / S
// columns of each half. The others' sums of them arrive in the operand stages, which nothing reads
// any more once every pair has come to the first barrier ([pair][half][4 columns][row] in 16 bytes,
// so that a warp writes 512 bytes in a row). Its own sums first, then the others' in their order: the same
// bits every time.
template <int S, int COLS>
__device__ __forceinline__ void join_splits(const float* acc, float* own, uint32_t stage, int rank, int split, int half,
                                            int row) {
  constexpr int W = COLS / S;
  static_assert(S * 2 * W * BM * 4 <= STAGES * STAGE_BYTES, "exchange area");
  auto place = [&](int from, int c) { return (uint32_t)((((from * 2 + half) * (W / 4) + c / 4) * BM + row) * 16); };
  __syncwarp();
  cluster_sync_all();
#pragma unroll
  for (int q = 0; q < S; ++q) {
    if (q == split) continue;
    const uint32_t dst = mapa_shared(stage, 2 * q + rank);
#pragma unroll
    for (int c = 0; c < W; c += 4)
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + place(split, c)),
                   "f"(acc[q * W + c]), "f"(acc[q * W + c + 1]), "f"(acc[q * W + c + 2]), "f"(acc[q * W + c + 3])
                   : "memory");
  }
#pragma unroll
  for (int c = 0; c < W; ++c) {
    own[c] = acc[c];
#pragma unroll
    for (int q = 1; q < S; ++q) own[c] = split == q ? acc[q * W + c] : own[c];
  }
  __syncwarp();
  cluster_sync_all();
#pragma unroll
  for (int q = 0; q < S; ++q) {
    if (q == split) continue;
#pragma unroll
    for (int c = 0; c < W; c += 4) {
      float f[4];
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(f[0]), "=f"(f[1]), "=f"(f[2]), "=f"(f[3])
                   : "r"(stage + place(q, c))
                   : "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) own[c + i] += f[i];
    }
  }
}

template <int N>
struct Columns {
  static constexpr int value = N;
};

// OutT: output element (plain); SWIGLU writes codes and ignores it. GROUPED rows or plain ones. SPLITS pairs
// of a cluster share a tile's K blocks; a cluster then has one tile.
template <typename OutT, bool SWIGLU, bool GROUPED, int SPLITS>
__global__ void __launch_bounds__(THREADS, 1)
    block_gemm_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                           const __grid_constant__ CUtensorMap tm_b32, const Params p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * STAGE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 2 * BUFS + 2 + 2 * SLOTS);
  const uint32_t abort_flag = smem_u32(tmem_slot + 1);
  uint32_t* row_max = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(bars) + BAR_BYTES);  // [2][2][128]
  float* scales = reinterpret_cast<float*>(row_max + 2 * 2 * BM);                                 // [SLOTS][SLOT_FLOATS]
  float* turns = scales + SLOTS * SLOT_FLOATS;                                                    // [math warps][32][17]
  int32_t* first = reinterpret_cast<int32_t*>(turns + 2 * HALF_WARPS * 32 * TURN_PITCH);          // [groups + 1]
  int32_t* begins = first + MAX_GROUPS + 1;                                                       // [groups + 1]
  auto full_bar = [&](int s) { return smem_u32(&bars[s]); };                // both CTAs' copies (even CTA)
  auto empty_bar = [&](int s) { return smem_u32(&bars[STAGES + s]); };
  auto tfull_bar = [&](int i) { return smem_u32(&bars[2 * STAGES + i]); };
  auto tempty_bar = [&](int i) { return smem_u32(&bars[2 * STAGES + BUFS + i]); };  // both CTAs' math (even CTA)
  const uint32_t drain_bar = smem_u32(&bars[2 * STAGES + 2 * BUFS]);
  const uint32_t max_bar = smem_u32(&bars[2 * STAGES + 2 * BUFS + 1]);  // the row maxima of a SwiGLU tile are written
  auto sfull_bar = [&](uint32_t i) { return smem_u32(&bars[2 * STAGES + 2 * BUFS + 2 + i]); };
  auto sempty_bar = [&](uint32_t i) { return smem_u32(&bars[2 * STAGES + 2 * BUFS + 2 + SLOTS + i]); };
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int cta = (int)cluster_ctarank(), rank = SPLITS == 1 ? cta : cta & 1;
  const int lead = SPLITS == 1 ? 0 : cta - rank, split = SPLITS == 1 ? 0 : cta >> 1;
  const int cluster = blockIdx.x / (2 * SPLITS), clusters = gridDim.x / (2 * SPLITS);
  const int kb_begin = SPLITS == 1 ? 0 : p.kb * split / SPLITS;
  const int kb_count = SPLITS == 1 ? p.kb : p.kb * (split + 1) / SPLITS - kb_begin;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 2);  // each half's MMAs
    }
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(tfull_bar(i), 1);
      mbar_init(tempty_bar(i), 2 * HALF_WARPS);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(sfull_bar(i), 32);  // the copies of every lane of the scale warp
      mbar_init(sempty_bar(i), 2 * HALF_WARPS);
    }
    mbar_init(drain_bar, 2);
    mbar_init(max_bar, 2 * HALF_WARPS);
    tmem_slot[1] = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish_pair();
  }
  if (GROUPED && warp == 2) group_units(p, 2, first, begins);
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  volatile int never_abort = 0;

  const int row_units = GROUPED ? first[p.groups] : (int)((p.rows + 2 * BM - 1) / (2 * BM));
  const int units = row_units * p.n_tiles;

  if (warp >= MATH_WARP0) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MATH_REGS));
    // ------------------------------------------------------------ scaling and epilogue
    const int quarter = warp & 3, half = (warp - MATH_WARP0) / HALF_WARPS;
    const int row_in_tile = quarter * 32 + lane;
    // this thread's lane of its half's accumulator: all 128 columns (SwiGLU: 64 gate, the same 64 up)
    const uint32_t t_lane = tmem_base + ((uint32_t)(quarter * 32) << 16) + half * NACC;
    const uint32_t lead_tempty = mapa_shared(tempty_bar(0), lead);
    uint32_t it = 0, grp = 0, tile = 0;
    bool ok = true, joined = false;
    for (int u = cluster; ok && u < units; u += clusters, ++tile) {
      const Unit w = unit_of<GROUPED>(p, u, 2, first, begins);
      // One row tile: 64 rows per CTA, lanes 64..127 the same rows' later columns (`side`).
      const bool narrow = w.tiles == 1;
      const int side = narrow ? quarter >> 1 : 0;
      // The up rows start at N inside the group, so a tile's up columns can straddle two 128-row
      // scale blocks: the columns below `cut` take the first, the others the second. N % 16 == 0,
      // so 16 columns share a scale.
      const int cut = SWIGLU ? 128 - ((p.N + w.n * 128) & 127) - 64 * half - 32 * side : 0;
      float acc[128];
#pragma unroll
      for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      // Runs of 16 and 32 columns in turn: one is read while the other is added. The first run of
      // the next K block is read before the last one of this block is added, so that neither its
      // wait nor its latency lies between two K blocks that are both there.
      auto sum_blocks = [&](auto width) {
        constexpr int COLS = decltype(width)::value;  // of this thread: 128, or 64 of a narrow unit
        uint32_t t[32], v[16];
        auto scale_for = [&](int col, float c0, float c1, float c2) {
          return SWIGLU && col >= COLS / 2 ? (col - COLS / 2 < cut ? c1 : c2) : c0;
        };
        auto add16 = [&](int col, const uint32_t* r, float sc) {
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[col + i] = fmaf(sc, __uint_as_float(r[i]), acc[col + i]);
        };
        if (!warp_wait(tfull_bar((it & 1) * 2 + half), (it >> 1) & 1, abort_flag, p.status, kDevTimeoutEpilogue)) return false;
        tc_fence_after();
        tmem_ld_x16(t_lane + (it & 1) * 2 * NACC, v);
        for (int kb0 = 0; kb0 < kb_count; kb0 += GROUP) {
          const uint32_t sl = grp % SLOTS;
          if (!warp_wait(sfull_bar(sl), (grp / SLOTS) & 1, abort_flag, p.status, kDevTimeoutEpilogue)) return false;
          const float* slot = scales + sl * SLOT_FLOATS;
          float s0[GROUP], s1[GROUP], s2[GROUP];
          {
            const float4 xa = *reinterpret_cast<const float4*>(slot + row_in_tile * GROUP);
            const float4* wb = reinterpret_cast<const float4*>(slot + BM * GROUP);
            const float4 w0 = wb[SWIGLU ? 0 : half];
            s0[0] = xa.x * w0.x, s0[1] = xa.y * w0.y, s0[2] = xa.z * w0.z, s0[3] = xa.w * w0.w;
            if (SWIGLU) {
              const float4 w1 = wb[1], w2 = wb[2];
              s1[0] = xa.x * w1.x, s1[1] = xa.y * w1.y, s1[2] = xa.z * w1.z, s1[3] = xa.w * w1.w;
              s2[0] = xa.x * w2.x, s2[1] = xa.y * w2.y, s2[2] = xa.z * w2.z, s2[3] = xa.w * w2.w;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(sempty_bar(sl));
          ++grp;
#pragma unroll
          for (int j = 0; j < GROUP; ++j) {
            if (kb0 + j >= kb_count) break;
            const uint32_t buf = (it & 1) * 2 + half;
            const uint32_t src = t_lane + (it & 1) * 2 * NACC;
            auto add = [&](int col, const uint32_t* r) {
              add16(col, r, scale_for(col, s0[j], SWIGLU ? s1[j] : 0.f, SWIGLU ? s2[j] : 0.f));
            };
            uint32_t last[16];
            tmem_wait_ld();
            tmem_ld_x32(src + 16, t);
            add(0, v);
            tmem_wait_ld();
            if constexpr (COLS == 128) {
              tmem_ld_x16(src + 48, v);
              add(16, t), add(32, t + 16);
              tmem_wait_ld();
              tmem_ld_x32(src + 64, t);
              add(48, v);
              tmem_wait_ld();
              tmem_ld_x16(src + 96, v);
              add(64, t), add(80, t + 16);
              tmem_wait_ld();
              tmem_ld_x16(src + 112, last);
              add(96, v);
            } else {
              tmem_ld_x16(src + 48, last);
              add(16, t), add(32, t + 16);
            }
            tmem_wait_ld();
            tc_fence_before();
            if (lane == 0) arrive_remote(lead_tempty + 8u * buf);
            ++it;
            if (kb0 + j + 1 < kb_count) {
              if (!warp_wait(tfull_bar(buf ^ 2), (it >> 1) & 1, abort_flag, p.status, kDevTimeoutEpilogue)) return false;
              tc_fence_after();
              tmem_ld_x16(t_lane + (it & 1) * 2 * NACC, v);
            }
            add(COLS - 16, last);
          }
        }
        return true;
      };
      ok = narrow ? sum_blocks(Columns<64>{}) : sum_blocks(Columns<128>{});
      if (!ok) break;
      const int64_t row = narrow ? (int64_t)w.m * BM + 64 * rank + (row_in_tile & 63)
                                 : (int64_t)(w.m + rank) * BM + row_in_tile;
      // The padding of fp32 rows is not stored (64 experts of 2048 x 1408, 128 tokens: 7 of 8 rows of the tiles);
      // that of the codes is, a byte per value: their kernel has no register left for the row count.
      const int64_t end = SWIGLU || !GROUPED ? p.rows : (int64_t)w.m * BM + w.rows;
      const bool row_ok = row < end;
      const int64_t row4 = row - (lane & 3);  // the first of the four rows that four lanes store together
      const int rows4 = (int)max((int64_t)0, min((int64_t)4, end - row4));
      if (SWIGLU) {
        // a thread's 64 columns of h from its 64 gate and 64 up sums, or 32 of a narrow unit
        const int n0 = w.n * 128 + 64 * half + 32 * side;
        uint32_t m = 0;
        // h takes the gate values' place. The quotient within 2 ulp of fp32, 2^-18 of the e4m3 step that follows: the
        // correctly rounded division, which the streaming kernel has, spills here (Mixtral-shape layer, 2048 tokens:
        // 1.28 ms, from 1.13). Below gate = -87.3 it gives 0 for less than 1.1e-36 of up.
        auto activate = [&](auto width) {
          constexpr int COLS = decltype(width)::value / 2;
#pragma unroll
          for (int i = 0; i < COLS; ++i) {
            acc[i] = n0 + i < p.N ? __fdividef(acc[i], 1.f + __expf(-acc[i])) * acc[COLS + i] : 0.f;
            m = max(m, __float_as_uint(acc[i]) & 0x7fffffffu);
          }
        };
        if (narrow)
          activate(Columns<64>{});
        else
          activate(Columns<128>{});
        // the row's maximum over its two (narrow: four) threads; two buffers, so that one barrier per
        // tile is enough (a warp writes a buffer again only after every warp has read it and come to
        // the next tile)
        uint32_t* maxima = row_max + (tile & 1) * 2 * BM;
        maxima[half * BM + row_in_tile] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(max_bar);
        ok = warp_wait(max_bar, tile & 1, abort_flag, p.status, kDevTimeoutEpilogue);
        if (!ok) break;
        m = max(m, maxima[(half ^ 1) * BM + row_in_tile]);
        if (narrow) m = max(m, max(maxima[row_in_tile ^ 64], maxima[BM + (row_in_tile ^ 64)]));
        // h never leaves in another form, so its codes may come from the reciprocal: the quotient is within
        // 2 ulp of fp32, 2^-19 of an e4m3 step. A scale without a finite or normal reciprocal (rows of small
        // numbers) is moved by a power of two, with its row, first.
        float s = __uint_as_float(m) / 448.0f;
        s = s == 0.f ? 1.f : s;
        const float shift = s < 0x1p-100f ? 0x1p100f : s > 0x1p100f ? 0x1p-100f : 1.f;
        if (shift != 1.f) {
#pragma unroll
          for (int i = 0; i < 64; ++i) acc[i] *= shift;
        }
        const float inv = 1.f / (s * shift);
        uint4 codes[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* f = acc + 16 * c + 4 * i;
            const uint32_t lo =
                __nv_cvt_float2_to_fp8x2(make_float2(f[0] * inv, f[1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi =
                __nv_cvt_float2_to_fp8x2(make_float2(f[2] * inv, f[3] * inv), __NV_SATFINITE, __NV_E4M3);
            v[i] = lo | hi << 16;
          }
          codes[c] = make_uint4(v[0], v[1], v[2], v[3]);
        }
        if (narrow) {
          if (row_ok) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (n0 + 16 * c < p.N) *reinterpret_cast<uint4*>(p.q_out + row * p.N + n0 + 16 * c) = codes[c];
          }
        } else {
          transpose_pieces(codes);
          const int n = n0 + 16 * (lane & 3);
          if (n < p.N) {  // N % 16 == 0: 16 columns are inside or outside
            uint8_t* q = p.q_out + row4 * p.N + n;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (r < rows4) *reinterpret_cast<uint4*>(q + (int64_t)r * p.N) = codes[r];
          }
        }
        if (row_ok && half == 0 && side == 0) p.q_scale[row * ((p.N + 127) / 128) + w.n] = s;
      } else {
        const int n0 = w.n * BN + 128 * half + 64 * side;
        float* turn = turns + (warp - MATH_WARP0) * 32 * TURN_PITCH;
        const float rs = row_ok && p.row_scale ? p.row_scale[row] : 1.f;
        joined = true;
        auto store = [&](auto width) {
          constexpr int COLS = decltype(width)::value, W = COLS / SPLITS;
          if constexpr (SPLITS == 1) {
            store_columns<OutT, COLS>(p, acc, rs, row, rows4, n0, turn);
          } else {
            float own[W];
            join_splits<SPLITS, COLS>(acc, own, smem_u32(smem), rank, split, half, row_in_tile);
            store_columns<OutT, W>(p, own, rs, row, rows4, n0 + W * split, turn);
          }
        };
        if (narrow)
          store(Columns<64>{});
        else
          store(Columns<128>{});
      }
    }
    if (SPLITS > 1 && !joined) {  // an expired wait: the other pairs still meet this one
      __syncwarp();
      cluster_sync_all();
      cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CONTROL_REGS));
  if (warp == 0) {
    // ------------------------------------------------------------ producer (one thread)
    if (elect_one()) {
      tma_prefetch_desc(&tm_a);
      tma_prefetch_desc(&tm_b);
      const uint64_t pol_a = l2_policy_evict_last(), pol_b = l2_policy_evict_normal();
      const uint32_t base = smem_u32(smem);
      const uint32_t lead_full = mapa_shared(full_bar(0), lead);
      uint32_t s = 0, phase = 0, filled = 0;  // filled: bit i = stage i has been filled
      bool ok = true;
      for (int u = cluster; ok && u < units; u += clusters) {
        const Unit w = unit_of<GROUPED>(p, u, 2, first, begins);
        const int n0 = w.n * (SWIGLU ? 128 : BN);
        // B rows of half 0; half 1 is `next` rows on
        const int b0 = w.group * p.b_group_rows + n0 + rank * (SWIGLU ? p.N : 64);
        const int next = SWIGLU ? 64 : 128;
        const bool narrow = w.tiles == 1;  // 64 of the copied 128 rows per CTA
        const int a0 = narrow ? w.m * BM + 64 * rank : (w.m + rank) * BM;
        const int b32 = w.group * p.b_group_rows + n0 + rank * 32;  // narrow SwiGLU: 32 gate and up rows per half
        const uint32_t bytes = 2 * A_BYTES + 4 * B_HALF_BYTES;  // of both CTAs
        for (int kb = kb_begin; kb < kb_begin + kb_count; ++kb) {
          ok = lane_wait(empty_bar(s), phase ^ 1, empty_bar(s), phase ^ 1, abort_flag, p.status, kDevTimeoutProducer);
          if (!ok) break;
          const uint32_t dst = base + s * STAGE_BYTES, bar = lead_full + 8u * s;
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), bytes);
          tma_load_2d_pair(dst, &tm_a, bar, kb * BK, a0, pol_a);
          if (SWIGLU && narrow) {
#pragma unroll
            for (int i = 0; i < 4; ++i)  // gate and up rows of half 0, then of half 1
              tma_load_2d_pair(dst + A_BYTES + i * (B_HALF_BYTES / 2), &tm_b32, bar, kb * BK,
                               b32 + 64 * (i >> 1) + (i & 1) * p.N, pol_b);
          } else {
            tma_load_2d_pair(dst + A_BYTES, &tm_b, bar, kb * BK, b0, pol_b);
            tma_load_2d_pair(dst + A_BYTES + B_HALF_BYTES, &tm_b, bar, kb * BK, b0 + next, pol_b);
          }
          filled |= 1u << s;
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
      if (!ok) {
        // Let the copies in flight land before the CTA pair leaves. The odd CTA's complete on the
        // even CTA's barrier; it waits a fixed, ample time.
        if (rank == 0) {
          for (uint32_t i = 0; i < STAGES; ++i)  // stages before s were filled in this phase, the others in the last
            if (filled >> i & 1)
              mbar_wait(full_bar(i), i < s ? phase : phase ^ 1, &never_abort, p.status, 200000000ull, kDevTimeoutDrain);
        } else {
          const unsigned long long t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 200000ull) {
          }
        }
      }
    }
  } else if (warp == 1 || warp == 3) {
    // ------------------------------------------------------------ MMA issue, one half (one thread)
    if (rank == 0 && elect_one()) {
      const uint32_t half = warp >> 1;
      const uint16_t both = (uint16_t)(3 << lead);
      const uint64_t desc0 = smem_desc_sw128(smem_u32(smem));
      const uint32_t b_off = (A_BYTES + half * B_HALF_BYTES) >> 4;
      uint32_t s = 0, phase = 0, it = 0;
      bool ok = true;
      for (int u = cluster; ok && u < units; u += clusters) {
        const uint32_t idesc = unit_of<GROUPED>(p, u, 2, first, begins).tiles == 1 ? idesc_e4m3(BM, NACC) : idesc_e4m3(2 * BM, NACC);
        for (int kb = 0; kb < kb_count; ++kb, ++it) {
          const uint32_t buf = (it & 1) * 2 + half;
          ok = lane_wait(tempty_bar(buf), ((it >> 1) & 1) ^ 1, full_bar(s), phase, abort_flag, p.status, kDevTimeoutMma);
          if (!ok) break;
          tc_fence_after();
          const uint64_t ad = desc0 + (uint64_t)(s * (STAGE_BYTES >> 4)), bd = ad + b_off;
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_f8_pair(tmem_base + buf * NACC, ad + 2 * k, bd + 2 * k, idesc, k > 0 ? 1u : 0u);
          tc_commit_pair_both(tfull_bar(buf), both);
          tc_commit_pair_both(empty_bar(s), both);
          if (++s == STAGES) s = 0, phase ^= 1;
        }
      }
      // every MMA of this thread has stopped reading shared memory before the CTAs leave
      tc_commit_pair(drain_bar);
      mbar_wait(drain_bar, 0, &never_abort, p.status, 1000000000ull, kDevTimeoutDrain);
    }
  } else if (warp == 2) {
    // ------------------------------------------------------------ scales
    // Every lane copies the scales of four rows (32 i + lane), lanes 0..2 also one weight scale
    // each: plain, the tile's two halves; SwiGLU, gate, then the one or two 128-row blocks that
    // the up rows touch. 16-byte copies where a row's scales allow them.
    const uint32_t slots = smem_u32(scales);
    uint32_t grp = 0;
    bool ok = true;
    for (int u = cluster; ok && u < units; u += clusters) {
      const Unit w = unit_of<GROUPED>(p, u, 2, first, begins);
      // slots 32 i + lane: the CTA's rows in order, or a narrow unit's 64 rows twice
      const bool narrow = w.tiles == 1;
      const int64_t row0 = (narrow ? (int64_t)w.m * BM + 64 * rank : (int64_t)(w.m + rank) * BM) + lane;
      const int valid = (int)max((int64_t)0, min((int64_t)BM, p.rows - row0));  // the i-th row: from(i) < valid
      auto from = [&](int i) { return 32 * (narrow ? i & 1 : i); };
      const float* sa = p.a_scale + (valid > 0 ? row0 : 0) * p.kb;
      int block = 2 * w.n + (lane & 1);
      if (SWIGLU) block = lane == 0 ? w.n : ((p.N + w.n * 128) >> 7) + (lane == 2);
      const float* sb = p.b_scale + ((int64_t)w.group * p.b_blocks + min(block, p.b_blocks - 1)) * p.kb;
      for (int kb = kb_begin; kb < kb_begin + kb_count; kb += GROUP, ++grp) {
        const uint32_t sl = grp % SLOTS;
        ok = warp_wait(sempty_bar(sl), ((grp / SLOTS) & 1) ^ 1, abort_flag, p.status, kDevTimeoutProducer);
        if (!ok) break;
        const uint32_t dst = slots + sl * (SLOT_FLOATS * 4) + 16 * lane;
        if (p.vec_scales) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            copy_async<16>(dst + 512 * i, from(i) < valid ? sa + (int64_t)from(i) * p.kb + kb : p.a_scale,
                           from(i) < valid);
          if (lane < 3) copy_async<16>(dst + 16 * BM, sb + kb, true);
        } else {
#pragma unroll 1
          for (int j = 0; j < GROUP && kb + j < kb_begin + kb_count; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              copy_async<4>(dst + 512 * i + 4 * j, from(i) < valid ? sa + (int64_t)from(i) * p.kb + kb + j : p.a_scale,
                            from(i) < valid);
            if (lane < 3) copy_async<4>(dst + 16 * BM + 4 * j, sb + kb + j, true);
          }
        }
        copies_arrive(sfull_bar(sl));
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  if (SPLITS > 1) {  // the math warps' exchange
    __syncwarp();
    cluster_sync_all();
    cluster_sync_all();
  }
  }
  __syncwarp();
  tc_fence_before();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, TMEM_COLS);
  }
}

template <typename OutT, bool SWIGLU, bool GROUPED, int SPLITS = 1>
int run_pair(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tb32, const Params& p, int clusters, bool pdl,
             cudaStream_t stream) {
  auto kernel = block_gemm_pair_kernel<OutT, SWIGLU, GROUPED, SPLITS>;
  SB_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * SPLITS * clusters);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * SPLITS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  SB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tb32, p));
  count_launch();
  return STAGEML_OK;
}

template <typename OutT>
int run_plain(const CUtensorMap& ta, const CUtensorMap& tb, const Params& p, int clusters, int splits, bool pdl,
              cudaStream_t stream) {
  if (splits == 4) return run_pair<OutT, false, false, 4>(ta, tb, tb, p, clusters, pdl, stream);
  if (splits == 2) return run_pair<OutT, false, false, 2>(ta, tb, tb, p, clusters, pdl, stream);
  return run_pair<OutT, false, false>(ta, tb, tb, p, clusters, pdl, stream);
}

// Clusters of SPLITS pairs that the device runs at one time (not all of its SMs: a cluster lies in
// one of its processing clusters). Asked for once per device.
template <int SPLITS>
int resident_clusters() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if ((n = known[dev].load(std::memory_order_relaxed)) != 0) return n;
  auto kernel = block_gemm_pair_kernel<bf16, false, false, SPLITS>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * SPLITS);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM_BYTES;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * SPLITS;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess)
    return 0;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Pairs per tile: where the tiles leave SMs idle, several pairs share a tile's K blocks. A K block
// takes a pair 0.25 (narrow units) to 0.4 us on an idle device and the exchange 1.5 to 2 us, so two pairs
// pay from 12 blocks on (64 x 4096 outputs over 8, 12, 32, 112 blocks: 7.5, 8.9, 14.7, 38.6 us alone, 7.6,
// 8.5, 11.5, 23.9 in two) and four from 24 (300 x 1000 over 16, 24, 32: 11.2, 12.8, 14.5 in two, 11.6,
// 12.6, 13.3 in four), while all clusters run at one time (64 x 4096 in 16 clusters of eight CTAs took two
// turns: 25 us, not 15).
int splits_for(int64_t units, int kb) {
  if (kb >= 24 && units <= resident_clusters<4>()) return 4;
  if (kb >= 12 && units <= resident_clusters<2>()) return 2;
  return 1;
}

}  // namespace

int block_gemm_max_groups() { return MAX_GROUPS; }

int launch_block_gemm(const BlockGemmLaunch& g, cudaStream_t stream) {
  if (g.a_rows == 0 || g.N == 0) return STAGEML_OK;
  SB_CHECK_ARG(!g.swiglu || g.group_offsets, "block_gemm: SwiGLU rows are grouped");
  SB_CHECK_ARG(g.swiglu || !g.group_offsets || g.out_dtype == STAGEML_F32, "block_gemm: grouped rows leave in fp32");
  Params p{};
  p.K = g.K;
  p.N = g.N;
  p.kb = (int)scale_blocks(g.K);
  p.b_group_rows = g.swiglu ? 2 * g.N : g.N;
  p.b_blocks = (int)scale_blocks(p.b_group_rows);
  p.n_tiles = g.swiglu ? (int)scale_blocks(g.N) : (g.N + BN - 1) / BN;
  p.a_scale = g.a_scale;
  p.b_scale = g.b_scale;
  p.group_offsets = g.group_offsets;
  p.group_counts = g.group_counts;
  p.groups = g.groups;
  p.rows = g.a_rows;
  p.row_scale = g.row_scale;
  p.out = g.out;
  p.q_out = g.q_out;
  p.q_scale = g.q_scale;
  p.status = g.status;
  // row units: every group can end in a unit of one tile
  const int64_t tiles = (g.a_rows + BM - 1) / BM;
  const int64_t row_units = g.group_offsets ? std::min<int64_t>(tiles, tiles / 2 + g.groups) : (tiles + 1) / 2;
  const int64_t units = row_units * p.n_tiles;
  SB_CHECK_ARG(units <= 0x7fffffff, "block_gemm: too many tiles");
  const int pairs = sm_count() / 2;
  const int splits = g.group_offsets || g.swiglu ? 1 : splits_for(units, p.kb);
  p.vec_scales = p.kb % (GROUP * splits) == 0 &&
                 (reinterpret_cast<uintptr_t>(g.a_scale) | reinterpret_cast<uintptr_t>(g.b_scale)) % 16 == 0;
  CUtensorMap ta, tb;
  SB_TRY(make_tmap_2d(&ta, g.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)g.a_rows, (uint64_t)g.K, (uint64_t)g.K, BM,
                      BK, 128));
  SB_TRY(make_tmap_2d(&tb, g.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)g.groups * p.b_group_rows, (uint64_t)g.K,
                      (uint64_t)g.K, 64, BK, 128));
  const int clusters = (int)std::min<int64_t>(units, pairs);
  if (g.swiglu) {
    CUtensorMap tb32;  // a narrow unit's runs of 32 gate or up rows
    SB_TRY(make_tmap_2d(&tb32, g.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, (uint64_t)g.groups * p.b_group_rows, (uint64_t)g.K,
                        (uint64_t)g.K, 32, BK, 128));
    return run_pair<bf16, true, true>(ta, tb, tb32, p, clusters, g.pdl, stream);
  }
  if (g.group_offsets) return run_pair<float, false, true>(ta, tb, tb, p, clusters, g.pdl, stream);
  if (g.out_dtype == STAGEML_F32) return run_plain<float>(ta, tb, p, clusters, splits, g.pdl, stream);
  if (g.out_dtype == STAGEML_BF16) return run_plain<bf16>(ta, tb, p, clusters, splits, g.pdl, stream);
  return run_plain<f16>(ta, tb, p, clusters, splits, g.pdl, stream);
}

}  // namespace sb
