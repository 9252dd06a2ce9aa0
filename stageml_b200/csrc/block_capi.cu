// extern "C" entry points of the block-scaled FP8 products, the block norm and the
// router balance loss (include/stageml_b200.h): host-side argument checks, workspace
// carving, launches on the caller's stream.
#include "block_fp8.h"
#include "capi_util.h"
#include "kernels.h"

namespace sb {
namespace {

inline bool is_float(int dtype) { return dtype == STAGEML_F32 || is16(dtype); }

// The products round M and N up to whole tiles, and K up to a whole turn of a CTA's warps (4096 values), in 32 bits.
constexpr int kMaxSize = 0x7fffffff - 8191;

// ------------------------------------------------------------------ MoE layer
struct MoeBlocksBuffers {
  stageml_moe_plan plan{};
  void* perm = nullptr;
  uint8_t* xq = nullptr;     // [rows_cap, H] codes of the permuted rows
  float* xs = nullptr;       // [rows_cap, ceil(H/128)]
  float* h = nullptr;        // few rows: [rows_cap, I] silu(gate) * up in fp32
  uint8_t* hq = nullptr;     // [rows_cap, I] codes of silu(gate) * up
  float* hs = nullptr;       // [rows_cap, ceil(I/128)]
  float* y = nullptr;        // [rows_cap, H] weighted rows of the down projection, not rounded before the slots' sum
  int32_t* status = nullptr;
  size_t bytes = 0;
};

// Streaming products take 8 or 16 rows of a weight group per pass over its weights. 8: four routed rows per
// expert or fewer, few experts have more than eight (64 experts, six of them and two shared, 16 tokens: 148 us
// in passes of 8, 169 in passes of 16). Shared experts alone have one row per token: 16.
bool moe_blocks_sparse(const stageml_moe_blocks_args* a) { return a->k > 0 && (int64_t)a->T * a->k <= 4 * (int64_t)a->E; }

// Streaming products instead of tensor-core tiles, whose time is the same for any number of rows up to
// 128 per expert: up to kSkinnyRows tokens, and up to 128 routed rows, two per expert. Streamed and in tiles, us:
//   64 experts of 2048 x 1408, two of them, 17, 32, 48, 64 tokens      88, 137, 147, 162    110, 144, 158, 173
//   128 of 2048 x 768, four of them, 17, 32, 64                        107, 161, 212        123, 161, 208
//   256 of 2048 x 768, eight of them, 16, 17, 32                       197, 205, 287        200, 202, 267
// A shared expert has a row per token, and its passes come one after the other:
//   64 experts as above and one shared, 17, 24, 32, 64                 100, 110, 146, 191   116, 120, 144, 175
//   and four shared                                                    113, 139, 152, 236   119, 136, 143, 179
//   one shared of 4096 x 14336 alone, 8, 16, 17, 32                    60, 76, 108, 119     96, 97, 97, 96
// so 24 tokens are the most beside shared experts, and 16 without routed ones.
bool moe_blocks_skinny(const stageml_moe_blocks_args* a) {
  if (a->T <= kSkinnyRows) return true;
  return a->k > 0 && (a->n_shared == 0 || a->T <= 24) && (int64_t)a->T * a->k <= std::min<int64_t>(128, 2 * (int64_t)a->E);
}

void moe_blocks_carve(const stageml_moe_blocks_args* a, void* ws, MoeBlocksBuffers* b) {
  Carver c(ws);
  const int E_tot = a->E + a->n_shared;
  const int64_t P = (int64_t)a->T * (a->k + a->n_shared);
  carve_plan(c, P, E_tot, &b->plan);
  const size_t rows = (size_t)b->plan.rows_cap;
  b->perm = c.take_bytes(permute_scratch_bytes(P, permute_num_keys(0, 0, 0, E_tot)));
  b->xq = c.take<uint8_t>(rows * a->H);
  b->xs = c.take<float>(rows * scale_blocks(a->H));
  if (moe_blocks_skinny(a)) b->h = c.take<float>(rows * a->I);
  b->hq = c.take<uint8_t>(rows * a->I);
  b->hs = c.take<float>(rows * scale_blocks(a->I));
  b->y = c.take<float>(rows * a->H);
  b->status = c.take<int32_t>(1);
  b->bytes = c.off;
}

int moe_blocks_validate(const stageml_moe_blocks_args* a, bool check_ptrs) {
  SB_CHECK_ARG(a, "moe_blocks: null args");
  SB_CHECK_ARG(a->T >= 0 && a->H > 0 && a->I > 0 && a->E >= 0 && a->k >= 0 && a->n_shared >= 0,
               "moe_blocks: bad sizes T=%d H=%d I=%d E=%d k=%d n_shared=%d", a->T, a->H, a->I, a->E, a->k, a->n_shared);
  SB_CHECK_ARG(a->k + a->n_shared >= 1, "moe_blocks: need k + n_shared >= 1");
  SB_CHECK_ARG(a->k <= a->E && a->k <= 8, "moe_blocks: k=%d must be <= min(E, 8)", a->k);
  SB_CHECK_ARG(a->k > 0 || a->E == 0, "moe_blocks: E=%d routed experts with k = 0", a->E);
  SB_CHECK_ARG(a->H % 16 == 0 && a->I % 16 == 0, "moe_blocks: H=%d and I=%d must be multiples of 16", a->H, a->I);
  SB_CHECK_ARG(a->H <= kMaxSize && a->I <= kMaxSize, "moe_blocks: H=%d and I=%d: at most 2^31 - 8192", a->H, a->I);
  SB_CHECK_ARG((int64_t)(a->E + a->n_shared) * 2 * a->I <= 0x7fffffff && (int64_t)(a->E + a->n_shared) * a->H <= 0x7fffffff,
               "moe_blocks: too many weight rows");
  SB_CHECK_ARG(a->E + a->n_shared <= block_gemm_max_groups(), "moe_blocks: %d experts exceed %d", a->E + a->n_shared,
               block_gemm_max_groups());
  SB_CHECK_ARG(is16(a->act_dtype), "moe_blocks: act_dtype must be BF16 or F16");
  if (a->k > 0) {
    SB_CHECK_ARG(a->ids_dtype == STAGEML_I32 || a->ids_dtype == STAGEML_I64, "moe_blocks: ids must be int32 or int64");
    SB_CHECK_ARG(is_float(a->weights_dtype), "moe_blocks: weights must be F32, BF16 or F16");
  }
  if (a->T > 0 && check_ptrs) {
    SB_CHECK_ARG(a->x && a->gate_up && a->gate_up_scale && a->down && a->down_scale && a->out,
                 "moe_blocks: null tensor");
    SB_CHECK_ARG(a->k == 0 || (a->topk_ids && a->topk_weights), "moe_blocks: topk_ids and topk_weights are required");
    SB_CHECK_ARG(aligned16(a->x) && aligned16(a->gate_up) && aligned16(a->down) && aligned16(a->out),
                 "moe_blocks: x, gate_up, down and out must be 16-byte aligned");
  }
  return STAGEML_OK;
}

int moe_blocks_impl(const stageml_moe_blocks_args* a, void* ws, size_t ws_bytes, cudaStream_t st) {
  SB_TRY(moe_blocks_validate(a, true));
  if (a->T == 0) return STAGEML_OK;
  MoeBlocksBuffers b;
  moe_blocks_carve(a, nullptr, &b);
  if (!ws || ws_bytes < b.bytes)
    return set_error(STAGEML_ERR_WORKSPACE, "moe_blocks: workspace of %zu bytes < required %zu", ws_bytes, b.bytes);
  moe_blocks_carve(a, ws, &b);
  const int E_tot = a->E + a->n_shared;
  const int64_t P = (int64_t)a->T * (a->k + a->n_shared);
  int32_t* status = a->status ? a->status : b.status;
  PermuteScratch scr;
  permute_carve(b.perm, P, permute_num_keys(0, 0, 0, E_tot), &scr);
  const int slots = a->k + a->n_shared;
  const bool skinny = moe_blocks_skinny(a), pdl = pdl_enabled();
  SB_STAGE(STAGEML_STAGE_PERMUTE,
           launch_permute(a->topk_ids, a->ids_dtype, a->topk_weights, a->weights_dtype, nullptr, a->T, a->k,
                          a->n_shared, E_tot, 0, 0, b.plan, status, scr, st, nullptr, pdl));
  // few rows: codes by token, the product finds a plan row's token; else by plan row
  SB_STAGE(STAGEML_STAGE_GATHER_SHRINK,
           launch_quantize_block_rows(a->x, a->act_dtype, a->T, a->H, skinny ? nullptr : b.plan.pair_row,
                                      skinny ? 0 : slots, b.xq, b.xs, st, pdl));
  BlockGemmLaunch g;
  g.a = b.xq;
  g.a_scale = b.xs;
  g.a_rows = b.plan.rows_cap;
  g.b = a->gate_up;
  g.b_scale = a->gate_up_scale;
  g.groups = E_tot;
  g.K = a->H;
  g.N = a->I;
  g.swiglu = true;
  g.group_offsets = b.plan.group_offsets;
  g.group_counts = b.plan.group_counts;
  g.q_out = b.hq;
  g.q_scale = b.hs;
  g.status = status;
  g.pdl = pdl;
  BlockSkinny sk;
  if (skinny) {
    sk.max_rows = moe_blocks_sparse(a) ? std::min(a->T, 8) : a->T;
    sk.row_map = b.plan.row_token;
    sk.tile_group = b.plan.tile_group;
    sk.num_tiles = b.plan.num_tiles;
    sk.tiles_cap = (int)(b.plan.rows_cap / 128);
    g.out = b.h;
    SB_STAGE(STAGEML_STAGE_GEMM_GATE_UP, launch_block_skinny(g, sk, st));
    SB_STAGE(STAGEML_STAGE_SHRINK_H, launch_quantize_block_pairs(b.h, b.plan.pair_row, P, a->I, b.hq, b.hs, st, pdl));
    sk.row_map = nullptr;
  } else {
    SB_STAGE(STAGEML_STAGE_GEMM_GATE_UP, launch_block_gemm(g, st));
  }
  g.a = b.hq;
  g.a_scale = b.hs;
  g.b = a->down;
  g.b_scale = a->down_scale;
  g.K = a->I;
  g.N = a->H;
  g.swiglu = false;
  g.row_scale = b.plan.row_weight;
  g.out = b.y;
  g.out_dtype = STAGEML_F32;
  SB_STAGE(STAGEML_STAGE_GEMM_DOWN, skinny ? launch_block_skinny(g, sk, st) : launch_block_gemm(g, st));
  SB_STAGE(STAGEML_STAGE_COMBINE, launch_combine_f32(b.y, b.plan.pair_row, a->T, slots, a->H,
                                                     a->act_dtype == STAGEML_BF16, a->out, st, pdl));
  return STAGEML_OK;
}

// ------------------------------------------------------------------ block norm
int norm_validate(const stageml_norm_args* a, bool backward, bool check_ptrs) {
  SB_CHECK_ARG(a, "norm_residual: null args");
  SB_CHECK_ARG(a->T >= 0 && a->H > 0, "norm_residual: bad sizes T=%lld H=%d", (long long)a->T, a->H);
  SB_CHECK_ARG(a->H <= norm_max_width(), "norm_residual: H=%d exceeds %d", a->H, norm_max_width());
  SB_CHECK_ARG(a->T <= 0x7fffffff, "norm_residual: too many rows");
  SB_CHECK_ARG(is_float(a->resid_dtype) && is_float(a->block_dtype), "norm_residual: dtypes must be F32, BF16 or F16");
  SB_CHECK_ARG(a->resid_dtype == STAGEML_F32 || a->block_dtype == a->resid_dtype,
               "norm_residual: a 16-bit residual needs block rows of its own dtype");
  SB_CHECK_ARG(a->block_out || a->T == 0 || (!a->post_weight && a->gate_mode == STAGEML_GATE_NONE),
               "norm_residual: post_weight and gate need block_out");
  SB_CHECK_ARG(a->gate_mode >= STAGEML_GATE_NONE && a->gate_mode <= STAGEML_GATE_FULL, "norm_residual: gate mode %d",
               a->gate_mode);
  SB_CHECK_ARG(a->T == 0 || (a->gate_mode == STAGEML_GATE_NONE) == (a->gate == nullptr), "norm_residual: gate and gate_mode disagree");
  SB_CHECK_ARG((!a->post_weight || is_float(a->post_dtype)) && (!a->gate || is_float(a->gate_dtype)) &&
                   (!a->pre_weight || is_float(a->pre_dtype)),
               "norm_residual: weights must be F32, BF16 or F16");
  SB_CHECK_ARG(!a->codes || (a->pre_weight && a->code_scale), "norm_residual: codes need pre_weight and code_scale");
  if (a->T == 0 || !check_ptrs) return STAGEML_OK;
  SB_CHECK_ARG(a->residual, "norm_residual: null residual");
  if (!backward) {
    SB_CHECK_ARG(a->new_residual, "norm_residual: null output");
    SB_CHECK_ARG(!a->pre_weight || a->normed || a->codes, "norm_residual: pre_weight without normed or codes");
  } else {
    SB_CHECK_ARG(a->d_residual && (!a->block_out || a->d_block_out) && (!a->post_weight || a->d_post) &&
                     (!a->gate || a->d_gate) && (!a->pre_weight || a->d_pre),
                 "norm_residual_backward: a gradient output is missing");
    SB_CHECK_ARG(a->pre_weight || !a->grad_normed, "norm_residual_backward: grad_normed without pre_weight");
  }
  return STAGEML_OK;
}

size_t norm_scratch(const stageml_norm_args* a, bool backward) {
  return backward ? norm_residual_backward_scratch(*a) : norm_residual_scratch(*a);
}

int norm_call(const stageml_norm_args* a, bool backward, void* ws, size_t ws_bytes, cudaStream_t st) {
  SB_TRY(norm_validate(a, backward, true));
  const size_t need = a->T > 0 ? norm_scratch(a, backward) : 0;
  if (need > 0 && (!ws || ws_bytes < need))
    return set_error(STAGEML_ERR_WORKSPACE, "norm_residual: workspace of %zu bytes < required %zu", ws_bytes, need);
  SB_CHECK_ARG(need == 0 || aligned16(ws), "norm_residual: workspace must be 16-byte aligned");
  return backward ? launch_norm_residual_backward(*a, ws, st) : launch_norm_residual(*a, ws, st);
}

int balance_validate(const void* logits, int dtype, int64_t T, int E, int k) {
  SB_CHECK_ARG(T >= 0 && E >= 1 && E <= 256, "balance_loss: T=%lld, E=%d (at most 256)", (long long)T, E);
  SB_CHECK_ARG(k >= 1 && k <= 8, "balance_loss: k=%d must be in 1..8", k);
  SB_CHECK_ARG(is_float(dtype), "balance_loss: logits must be F32, BF16 or F16");
  SB_CHECK_ARG(T * k < (int64_t(1) << 31), "balance_loss: too many slots");
  SB_CHECK_ARG(T == 0 || logits, "balance_loss: null logits");
  return STAGEML_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" {

int stageml_quantize_e4m3_blocks(const void* x, int dtype, int64_t batch, int64_t rows, int64_t cols, int tiles,
                                 uint8_t* q_out, float* scale_out, stageml_stream_t stream) {
  clear_error();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SB_CHECK_ARG(batch >= 0 && rows >= 0 && cols >= 0, "quantize_e4m3_blocks: negative size");
  SB_CHECK_ARG(is_float(dtype), "quantize_e4m3_blocks: x must be F32, BF16 or F16");
  if (batch == 0 || rows == 0 || cols == 0) return STAGEML_OK;
  SB_CHECK_ARG(x && q_out && scale_out, "quantize_e4m3_blocks: null pointer");
  if (!tiles) return launch_quantize_block_rows(x, dtype, batch * rows, cols, nullptr, 0, q_out, scale_out, st);
  SB_CHECK_ARG(batch * scale_blocks(rows) * scale_blocks(cols) <= 0x7fffffff, "quantize_e4m3_blocks: too many tiles");
  return launch_quantize_block_tiles(x, dtype, batch, rows, cols, q_out, scale_out, st);
}

int stageml_block_matmul(const uint8_t* x, const float* x_scale, const uint8_t* w, const float* w_scale, int M, int N,
                         int K, int out_dtype, void* out, int32_t* status, stageml_stream_t stream) {
  clear_error();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  SB_CHECK_ARG(M >= 0 && N >= 0 && K >= 1, "block_matmul: bad sizes M=%d N=%d K=%d", M, N, K);
  SB_CHECK_ARG(K % 16 == 0, "block_matmul: K=%d must be a multiple of 16", K);
  SB_CHECK_ARG(M <= kMaxSize && N <= kMaxSize && K <= kMaxSize, "block_matmul: M=%d, N=%d, K=%d: at most 2^31 - 8192", M,
               N, K);
  SB_CHECK_ARG(is_float(out_dtype), "block_matmul: out_dtype must be F32, BF16 or F16");
  if (M == 0 || N == 0) return STAGEML_OK;
  SB_CHECK_ARG(x && x_scale && w && w_scale && out, "block_matmul: null pointer");
  SB_CHECK_ARG(aligned16(x) && aligned16(w) && aligned16(out), "block_matmul: x, w and out must be 16-byte aligned");
  BlockGemmLaunch g;
  g.a = x;
  g.a_scale = x_scale;
  g.a_rows = M;
  g.b = w;
  g.b_scale = w_scale;
  g.K = K;
  g.N = N;
  g.out = out;
  g.out_dtype = out_dtype;
  g.status = status;
  if (M <= kSkinnyRows) {
    BlockSkinny sk;
    sk.max_rows = M;
    SB_STAGE(STAGEML_STAGE_GEMM, launch_block_skinny(g, sk, st));
  } else {
    SB_STAGE(STAGEML_STAGE_GEMM, launch_block_gemm(g, st));
  }
  return STAGEML_OK;
}

size_t stageml_moe_blocks_workspace_bytes(const stageml_moe_blocks_args* args) {
  if (!args || moe_blocks_validate(args, false) != STAGEML_OK) return 0;
  MoeBlocksBuffers b;
  moe_blocks_carve(args, nullptr, &b);
  return b.bytes;
}

int stageml_moe_forward_blocks(const stageml_moe_blocks_args* args, void* workspace, size_t workspace_bytes,
                               stageml_stream_t stream) {
  clear_error();
  return moe_blocks_impl(args, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t stageml_norm_residual_workspace_bytes(const stageml_norm_args* args, int backward) {
  if (!args || norm_validate(args, backward != 0, false) != STAGEML_OK) return 0;
  return norm_scratch(args, backward != 0);
}

int stageml_norm_residual(const stageml_norm_args* args, void* workspace, size_t workspace_bytes,
                          stageml_stream_t stream) {
  clear_error();
  return norm_call(args, false, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int stageml_norm_residual_backward(const stageml_norm_args* args, void* workspace, size_t workspace_bytes,
                                   stageml_stream_t stream) {
  clear_error();
  return norm_call(args, true, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

size_t stageml_balance_workspace_bytes(int64_t T, int E) {
  return T >= 0 && E >= 1 && E <= 256 ? balance_scratch_bytes(T, E) : 0;
}

int stageml_balance_loss(const void* logits, int logits_dtype, const void* ids, int ids_dtype, const uint8_t* valid,
                         int64_t T, int E, int k, float coefficient, float* loss, int32_t* counts, int32_t* tokens,
                         int32_t* status, void* workspace, size_t workspace_bytes, stageml_stream_t stream) {
  clear_error();
  SB_TRY(balance_validate(logits, logits_dtype, T, E, k));
  SB_CHECK_ARG(ids_dtype == STAGEML_I32 || ids_dtype == STAGEML_I64, "balance_loss: ids must be int32 or int64");
  SB_CHECK_ARG((T == 0 || ids) && loss && counts && tokens, "balance_loss: null pointer");
  const size_t need = balance_scratch_bytes(T, E);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(STAGEML_ERR_WORKSPACE, "balance_loss: workspace of %zu bytes < required %zu", workspace_bytes, need);
  return launch_balance_loss(logits, logits_dtype, ids, ids_dtype == STAGEML_I64, valid, T, E, k, coefficient, loss,
                             counts, tokens, status, workspace, static_cast<cudaStream_t>(stream));
}

int stageml_balance_loss_backward(const float* grad_loss, const void* logits, int logits_dtype, const int32_t* counts,
                                  const int32_t* tokens, const uint8_t* valid, int64_t T, int E, int k,
                                  float coefficient, void* grad_logits, stageml_stream_t stream) {
  clear_error();
  SB_TRY(balance_validate(logits, logits_dtype, T, E, k));
  if (T == 0) return STAGEML_OK;
  SB_CHECK_ARG(grad_loss && counts && tokens && grad_logits, "balance_loss_backward: null pointer");
  return launch_balance_loss_backward(grad_loss, logits, logits_dtype, counts, tokens, valid, T, E, k, coefficient,
                                      grad_logits, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
