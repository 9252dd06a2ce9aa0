// Launchers of the block-scaled FP8 operators, the block norm and the router balance loss.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/stageml_b200.h"

namespace sb {

constexpr int kScaleBlock = 128;  // values per scale along K (and along N for weights)
inline int64_t scale_blocks(int64_t n) { return (n + kScaleBlock - 1) / kScaleBlock; }

// quantize_blocks.cu: e4m3 codes with one fp32 scale per 128 values of a row
// (scale [rows, ceil(cols/128)]) or per 128 x 128 tile of each of `batch` matrices
// (scale [batch, ceil(rows/128), ceil(cols/128)]).
// slots > 0: source row r is written to the output rows out_row[slots * r + j], j < slots (a MoE
// plan's pair_row; negative ones are left out).
int launch_quantize_block_rows(const void* x, int dtype, int64_t rows, int64_t cols, const int32_t* out_row, int slots,
                               uint8_t* q, float* scale, cudaStream_t stream, bool pdl = false);
// fp32 rows row[p] of x (negative: skipped) to the same rows of q and scale; cols % 8 == 0.
int launch_quantize_block_pairs(const float* x, const int32_t* row, int64_t pairs, int64_t cols, uint8_t* q,
                                float* scale, cudaStream_t stream, bool pdl);
int launch_quantize_block_tiles(const void* w, int dtype, int64_t batch, int64_t rows, int64_t cols, uint8_t* q,
                                float* scale, cudaStream_t stream);

// block_gemm.cu: out[r, n] = row_scale[r] * sum_kb a_scale[r, kb] * b_scale[g, n / 128, kb]
//                                         * sum_{k in block kb} a[r, k] * b[g, n, k]
// with g = the weight group of row r (0 for plain rows). swiglu: B holds 2N rows per
// group ([gate; up]) and the output is silu(gate) * up in e4m3 codes with one scale
// per (row, 128 columns).
struct BlockGemmLaunch {
  const uint8_t* a = nullptr;      // [a_rows, K] e4m3
  const float* a_scale = nullptr;  // [a_rows, ceil(K/128)]
  int64_t a_rows = 0;
  const uint8_t* b = nullptr;      // [groups, b_group_rows, K] e4m3
  const float* b_scale = nullptr;  // [groups, ceil(b_group_rows/128), ceil(K/128)]
  int groups = 1;
  int K = 0;
  int N = 0;                       // output columns
  bool swiglu = false;
  // grouped rows (a MoE plan's padded rows): [groups + 1] row offsets, multiples of 128, and [groups] rows without
  // the padding; at most block_gemm_max_groups() groups. Null: plain rows, all of group 0
  const int32_t* group_offsets = nullptr;
  const int32_t* group_counts = nullptr;
  const float* row_scale = nullptr;
  void* out = nullptr;             // [rows, N] out_dtype (plain)
  int out_dtype = STAGEML_BF16;    // F32, BF16 or F16; grouped rows of block_gemm.cu: F32
  uint8_t* q_out = nullptr;        // [rows, N] e4m3 (swiglu)
  float* q_scale = nullptr;        // [rows, ceil(N/128)] (swiglu)
  int32_t* status = nullptr;
  bool pdl = false;
};
// block_skinny.cu: the same product for few rows per weight group, streaming the weights once per 8 or
// 16 rows. swiglu: writes silu(gate) * up in fp32 to g.out. Grouped rows need the plan's tiles and
// offsets; row_map (optional) names the row of `a` of each plan row.
constexpr int kSkinnyRows = 16;
struct BlockSkinny {
  int max_rows = 0;  // plain rows: their number, at most kSkinnyRows; grouped: up to 8 or more per group expected
  const int32_t* row_map = nullptr;
  const int32_t* tile_group = nullptr;
  const int32_t* num_tiles = nullptr;
  int tiles_cap = 0;
};
int launch_block_skinny(const BlockGemmLaunch& g, const BlockSkinny& s, cudaStream_t stream);
int block_gemm_max_groups();
int launch_block_gemm(const BlockGemmLaunch& g, cudaStream_t stream);

// block_norm.cu (a.T > 0 rows or none; arguments checked by the C ABI)
int norm_max_width();
size_t norm_residual_scratch(const stageml_norm_args& a);
int launch_norm_residual(const stageml_norm_args& a, void* scratch, cudaStream_t stream);
size_t norm_residual_backward_scratch(const stageml_norm_args& a);
int launch_norm_residual_backward(const stageml_norm_args& a, void* scratch, cudaStream_t stream);

// balance.cu
size_t balance_scratch_bytes(int64_t T, int E);
int launch_balance_loss(const void* logits, int dtype, const void* ids, int ids_i64, const uint8_t* valid, int64_t T,
                        int E, int k, float coefficient, float* loss, int32_t* counts, int32_t* tokens,
                        int32_t* status, void* scratch, cudaStream_t stream);
int launch_balance_loss_backward(const float* grad_loss, const void* logits, int dtype, const int32_t* counts,
                                 const int32_t* tokens, const uint8_t* valid, int64_t T, int E, int k,
                                 float coefficient, void* grad_logits, cudaStream_t stream);

}  // namespace sb
