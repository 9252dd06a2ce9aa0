// PyTorch custom-op library for the StageML B200 residual path.
//
// Loading this library (torch.ops.load_library, e.g. through the
// STAGEML_CUSTOM_OP_LIB hook of stageml/custom_op_registry.py:40-48) registers
// the `stageml` namespace with the unchanged schema of the reference's
//   residual_moe(Tensor hidden, Tensor gate_up, Tensor down, Tensor topk_weights, Tensor topk_ids) -> Tensor
// (csrc/stageml_residual_op.cpp:17-19) plus the ops of the rest of the path.
// Only the CUDA dispatch key is implemented: a CPU tensor raises "no kernel
// for CPU" instead of silently running a slow fallback. Every op marshals its
// tensors into the C ABI of libstageml_b200.so (include/stageml_b200.h) on the
// current CUDA stream; workspaces come from the caching allocator.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <mutex>
#include <unordered_map>

#include "../../include/stageml_b200.h"

namespace {

using at::Tensor;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return STAGEML_F32;
    case at::kBFloat16:
      return STAGEML_BF16;
    case at::kHalf:
      return STAGEML_F16;
    case at::kFloat8_e4m3fn:
      return STAGEML_E4M3;
    case at::kInt:
      return STAGEML_I32;
    case at::kLong:
      return STAGEML_I64;
    default:
      TORCH_CHECK(false, "stageml: unsupported dtype ", t.scalar_type());
  }
  return -1;
}

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == STAGEML_OK, "stageml::", what, " failed (code ", rc, "): ", stageml_last_error());
}

void check_cuda(const Tensor& t, const char* name, const Tensor& ref) {
  TORCH_CHECK(t.is_cuda(), "stageml: ", name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == ref.device(), "stageml: ", name, " is on ", t.device(), " but expected ", ref.device());
  TORCH_CHECK(t.is_contiguous(), "stageml: ", name, " must be contiguous");
}

const void* opt_ptr(const c10::optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// An uninitialised contiguous tensor on ref's device, without the dispatcher's way there (0.5 us of a call
// whose kernel may take 3).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& ref) {
  return at::detail::empty_cuda(sizes, dtype, ref.device(), c10::nullopt);
}

Tensor workspace(size_t bytes, const Tensor& ref) {
  return fresh({(int64_t)std::max<size_t>(bytes, 16)}, at::kByte, ref);
}

// Per-device status word that kernels write data-dependent errors into.
int32_t* status_word(const Tensor& ref) {
  static std::mutex mu;
  static std::unordered_map<int, Tensor> words;
  std::lock_guard<std::mutex> lk(mu);
  const int dev = ref.device().index();
  auto it = words.find(dev);
  if (it == words.end()) {
    it = words.emplace(dev, at::zeros({1}, ref.options().dtype(at::kInt))).first;
  }
  return it->second.data_ptr<int32_t>();
}

stageml_stream_t cur_stream() { return static_cast<stageml_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }

// ------------------------------------------------------------------ ops
Tensor residual_moe(const Tensor& hidden, const Tensor& gate_up, const Tensor& down, const Tensor& topk_weights,
                    const Tensor& topk_ids) {
  TORCH_CHECK(hidden.dim() == 2 && gate_up.dim() == 3 && down.dim() == 3, "residual_moe: bad ranks");
  TORCH_CHECK(topk_ids.dim() == 2 && topk_weights.sizes() == topk_ids.sizes(), "residual_moe: bad top-k shapes");
  const int64_t T = hidden.size(0), H = hidden.size(1), E = gate_up.size(0), I2 = gate_up.size(1);
  TORCH_CHECK(I2 % 2 == 0 && gate_up.size(2) == H && down.size(0) == E && down.size(1) == H && down.size(2) == I2 / 2,
              "residual_moe: gate_up [E,2I,H] / down [E,H,I] do not match hidden [T,H]");
  TORCH_CHECK(topk_ids.size(0) == T, "residual_moe: topk_ids rows != tokens");
  TORCH_CHECK(gate_up.scalar_type() == hidden.scalar_type() && down.scalar_type() == hidden.scalar_type(),
              "residual_moe: gate_up and down must have hidden's dtype");
  for (auto* p : {&hidden, &gate_up, &down, &topk_weights, &topk_ids}) check_cuda(*p, "input", hidden);
  c10::cuda::CUDAGuard guard(hidden.device());
  auto out = at::empty({T, H}, hidden.options());
  const int k = (int)topk_ids.size(1);
  const size_t ws = stageml_residual_moe_workspace_bytes((int)T, (int)H, (int)(I2 / 2), (int)E, k);
  auto w = workspace(ws, hidden);
  check_rc(stageml_residual_moe(hidden.data_ptr(), gate_up.data_ptr(), down.data_ptr(), topk_weights.data_ptr(),
                                dtype_code(topk_weights), topk_ids.data_ptr(), dtype_code(topk_ids), (int)T, (int)H,
                                (int)(I2 / 2), (int)E, k, dtype_code(hidden), out.data_ptr(), status_word(hidden),
                                w.data_ptr(), (size_t)w.numel(), cur_stream()),
           "residual_moe");
  return out;
}

Tensor moe_forward(const Tensor& x, const Tensor& gate_up, const Tensor& down, const c10::optional<Tensor>& topk_weights,
                   const c10::optional<Tensor>& topk_ids, const c10::optional<Tensor>& router_w, int64_t k,
                   int64_t n_shared, bool renormalize, const c10::optional<Tensor>& tenant_ids, int64_t n_tenants,
                   int64_t rank, const c10::optional<Tensor>& lora_a13, const c10::optional<Tensor>& lora_b13,
                   const c10::optional<Tensor>& lora_a2, const c10::optional<Tensor>& lora_b2,
                   const c10::optional<Tensor>& lora_scale, const c10::optional<Tensor>& gate_up_scale,
                   const c10::optional<Tensor>& down_scale, const c10::optional<Tensor>& T_dev,
                   const c10::optional<Tensor>& fold_slot, int64_t n_fold,
                   const c10::optional<Tensor>& down_group) {
  TORCH_CHECK(x.dim() == 2 && gate_up.dim() == 3 && down.dim() == 3, "moe_forward: bad ranks");
  if (T_dev.has_value())
    TORCH_CHECK(T_dev->is_cuda() && T_dev->scalar_type() == at::kInt && T_dev->numel() >= 1,
                "moe_forward: T_dev must be a CUDA int32 tensor");
  TORCH_CHECK(n_fold >= 0 && n_fold < gate_up.size(0), "moe_forward: n_fold out of range");
  if (!fold_slot.has_value()) TORCH_CHECK(n_fold == 0, "moe_forward: n_fold > 0 needs fold_slot");
  // gate_up / down hold the E_tot base experts, then the n_fold folded weight groups
  const int64_t T = x.size(0), H = x.size(1), E_tot = gate_up.size(0) - n_fold, I = gate_up.size(1) / 2;
  const int64_t down_groups = down_group.has_value() ? E_tot : E_tot + n_fold;
  TORCH_CHECK(gate_up.size(2) == H && down.size(0) == down_groups && down.size(1) == H && down.size(2) == I,
              "moe_forward: weight shapes do not match x");
  if (down_group.has_value()) {
    check_cuda(*down_group, "down_group", x);
    TORCH_CHECK(down_group->scalar_type() == at::kInt && down_group->is_contiguous() &&
                    down_group->numel() == E_tot + n_fold,
                "moe_forward: down_group must be contiguous int32 [E_tot + n_fold]");
  }
  if (fold_slot.has_value()) {
    check_cuda(*fold_slot, "fold_slot", x);
    TORCH_CHECK(fold_slot->scalar_type() == at::kInt && fold_slot->is_contiguous() &&
                    fold_slot->numel() == n_tenants * E_tot,
                "moe_forward: fold_slot must be contiguous int32 [n_tenants, E_tot]");
  }
  check_cuda(x, "x", x);
  check_cuda(gate_up, "gate_up", x);
  check_cuda(down, "down", x);
  for (const auto* o : {&topk_weights, &topk_ids, &router_w, &tenant_ids, &lora_a13, &lora_b13, &lora_a2, &lora_b2,
                        &lora_scale, &gate_up_scale, &down_scale})
    if (o->has_value()) check_cuda(**o, "optional input", x);
  if (tenant_ids.has_value())
    TORCH_CHECK(tenant_ids->scalar_type() == at::kInt && tenant_ids->numel() == T,
                "moe_forward: tenant_ids must be int32 [T]");
  if (lora_scale.has_value()) TORCH_CHECK(lora_scale->scalar_type() == at::kFloat, "moe_forward: lora_scale fp32");
  if (router_w.has_value()) TORCH_CHECK(router_w->scalar_type() == at::kFloat, "moe_forward: router_w must be fp32");
  TORCH_CHECK(gate_up.scalar_type() == down.scalar_type(), "moe_forward: gate_up and down must share a dtype");
  if (gate_up.scalar_type() == at::kFloat8_e4m3fn) {
    TORCH_CHECK(gate_up_scale.has_value() && down_scale.has_value(),
                "moe_forward: e4m3 weights need gate_up_scale and down_scale");
    TORCH_CHECK(gate_up_scale->scalar_type() == at::kFloat && gate_up_scale->numel() == E_tot * 2 * I &&
                    gate_up_scale->is_contiguous(),
                "moe_forward: gate_up_scale must be contiguous fp32 [E_tot, 2I]");
    TORCH_CHECK(down_scale->scalar_type() == at::kFloat && down_scale->numel() == E_tot * H &&
                    down_scale->is_contiguous(),
                "moe_forward: down_scale must be contiguous fp32 [E_tot, H]");
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto out = at::empty({T, H}, x.options());
  stageml_moe_args a{};
  a.T = (int)T;
  a.H = (int)H;
  a.I = (int)I;
  a.n_shared = (int)n_shared;
  a.E = (int)(E_tot - n_shared);
  a.k = (int)k;
  a.act_dtype = dtype_code(x);
  a.weight_dtype = dtype_code(gate_up);
  a.x = x.data_ptr();
  a.topk_ids = opt_ptr(topk_ids);
  a.ids_dtype = topk_ids.has_value() ? dtype_code(*topk_ids) : STAGEML_I32;
  a.topk_weights = opt_ptr(topk_weights);
  a.weights_dtype = topk_weights.has_value() ? dtype_code(*topk_weights) : STAGEML_F32;
  a.router_w = static_cast<const float*>(opt_ptr(router_w));
  a.renormalize = renormalize ? 1 : 0;
  a.tenant_ids = static_cast<const int32_t*>(opt_ptr(tenant_ids));
  a.n_tenants = (int)n_tenants;
  a.rank = (int)rank;
  a.gate_up = gate_up.data_ptr();
  a.down = down.data_ptr();
  a.gate_up_scale = static_cast<const float*>(opt_ptr(gate_up_scale));
  a.down_scale = static_cast<const float*>(opt_ptr(down_scale));
  a.lora_a13 = opt_ptr(lora_a13);
  a.lora_b13 = opt_ptr(lora_b13);
  a.lora_a2 = opt_ptr(lora_a2);
  a.lora_b2 = opt_ptr(lora_b2);
  a.lora_scale = static_cast<const float*>(opt_ptr(lora_scale));
  a.out = out.data_ptr();
  a.status = status_word(x);
  a.T_dev = static_cast<const int32_t*>(opt_ptr(T_dev));
  a.fold_slot = static_cast<const int32_t*>(opt_ptr(fold_slot));
  a.n_fold = (int)n_fold;
  a.down_group = static_cast<const int32_t*>(opt_ptr(down_group));
  const size_t ws = stageml_moe_workspace_bytes(&a);
  TORCH_CHECK(ws > 0 || T == 0, "moe_forward: invalid arguments: ", stageml_last_error());
  auto w = workspace(ws, x);
  check_rc(stageml_moe_forward(&a, w.data_ptr(), (size_t)w.numel(), cur_stream()), "moe_forward");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> route_topk(const Tensor& x, const Tensor& gate_w, int64_t k, bool renormalize) {
  check_cuda(x, "x", x);
  check_cuda(gate_w, "gate_w", x);
  TORCH_CHECK(gate_w.scalar_type() == at::kFloat && gate_w.dim() == 2 && gate_w.size(1) == x.size(1),
              "route_topk: gate_w must be fp32 [E, H]");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), E = gate_w.size(0);
  auto ids = at::empty({T, k}, x.options().dtype(at::kInt));
  auto w = at::empty({T, k}, x.options().dtype(at::kFloat));
  auto logits = at::empty({T, E}, x.options().dtype(at::kFloat));
  check_rc(stageml_route_topk(x.data_ptr(), dtype_code(x), gate_w.data_ptr<float>(), (int)T, (int)x.size(1), (int)E,
                              (int)k, renormalize ? 1 : 0, logits.data_ptr<float>(), ids.data_ptr<int32_t>(),
                              w.data_ptr<float>(), cur_stream()),
           "route_topk");
  return {ids, w, logits};
}

std::tuple<Tensor, Tensor> topk_from_logits(const Tensor& logits, int64_t k, bool renormalize) {
  check_cuda(logits, "logits", logits);
  TORCH_CHECK(logits.scalar_type() == at::kFloat && logits.dim() == 2, "topk_from_logits: fp32 [T, E] logits");
  c10::cuda::CUDAGuard guard(logits.device());
  const int64_t T = logits.size(0);
  auto ids = at::empty({T, k}, logits.options().dtype(at::kInt));
  auto w = at::empty({T, k}, logits.options().dtype(at::kFloat));
  check_rc(stageml_topk_from_logits(logits.data_ptr<float>(), (int)T, (int)logits.size(1), (int)k, renormalize ? 1 : 0,
                                    ids.data_ptr<int32_t>(), w.data_ptr<float>(), cur_stream()),
           "topk_from_logits");
  return {ids, w};
}

std::vector<Tensor> permute(const Tensor& ids, const c10::optional<Tensor>& weights,
                            const c10::optional<Tensor>& tenant_ids, int64_t n_experts_total, int64_t n_shared,
                            int64_t n_tenants, bool group_by_tenant) {
  check_cuda(ids, "ids", ids);
  TORCH_CHECK(ids.dim() == 2, "permute: ids must be [T, k]");
  if (weights.has_value()) check_cuda(*weights, "weights", ids);
  if (tenant_ids.has_value()) {
    check_cuda(*tenant_ids, "tenant_ids", ids);
    TORCH_CHECK(tenant_ids->scalar_type() == at::kInt && tenant_ids->numel() == ids.size(0), "permute: tenant_ids");
  }
  c10::cuda::CUDAGuard guard(ids.device());
  const int T = (int)ids.size(0), k = (int)ids.size(1);
  const int64_t P = (int64_t)T * (k + n_shared);
  const int n_groups = group_by_tenant ? (int)(n_tenants * n_experts_total) : (int)n_experts_total;
  const int64_t rows_cap = stageml_plan_rows_cap(P, n_groups);
  auto io = ids.options().dtype(at::kInt);
  Tensor row_token = at::empty({rows_cap}, io), row_tenant = at::empty({rows_cap}, io),
         row_weight = at::empty({rows_cap}, io.dtype(at::kFloat)), row_pair = at::empty({rows_cap}, io),
         pair_row = at::empty({std::max<int64_t>(P, 1)}, io), tile_group = at::empty({rows_cap / 128}, io),
         group_offsets = at::empty({n_groups + 1}, io), group_counts = at::empty({n_groups}, io),
         num_tiles = at::empty({1}, io);
  stageml_moe_plan plan;
  plan.row_token = row_token.data_ptr<int32_t>();
  plan.row_tenant = row_tenant.data_ptr<int32_t>();
  plan.row_weight = row_weight.data_ptr<float>();
  plan.row_pair = row_pair.data_ptr<int32_t>();
  plan.pair_row = pair_row.data_ptr<int32_t>();
  plan.tile_group = tile_group.data_ptr<int32_t>();
  plan.group_offsets = group_offsets.data_ptr<int32_t>();
  plan.group_counts = group_counts.data_ptr<int32_t>();
  plan.num_tiles = num_tiles.data_ptr<int32_t>();
  plan.rows_cap = rows_cap;
  const size_t ws = stageml_permute_workspace_bytes(T, k, (int)n_shared, (int)n_experts_total, (int)n_tenants,
                                                    group_by_tenant ? 1 : 0);
  auto w = workspace(ws, ids);
  check_rc(stageml_permute(ids.data_ptr(), dtype_code(ids), opt_ptr(weights),
                           weights.has_value() ? dtype_code(*weights) : STAGEML_F32,
                           static_cast<const int32_t*>(opt_ptr(tenant_ids)), T, k, (int)n_shared, (int)n_experts_total,
                           (int)n_tenants, group_by_tenant ? 1 : 0, &plan, status_word(ids), w.data_ptr(),
                           (size_t)w.numel(), cur_stream()),
           "permute");
  return {row_token, row_tenant, row_weight, row_pair, pair_row, tile_group, group_offsets, group_counts, num_tiles};
}

// W: [rows, cols] (broadcast over the batch) or [batch, rows, cols]; A/B: [batch, ...] or unbatched.
Tensor lora_fold(const Tensor& W, const Tensor& A, const Tensor& B, const Tensor& scale, int64_t layout) {
  check_cuda(W, "W", W);
  check_cuda(A, "A", W);
  check_cuda(B, "B", W);
  check_cuda(scale, "scale", W);
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "lora_fold: scale must be fp32 [batch]");
  TORCH_CHECK(A.scalar_type() == W.scalar_type() && B.scalar_type() == W.scalar_type(), "lora_fold: dtype mismatch");
  const bool batched = A.dim() == 3;
  TORCH_CHECK((batched && B.dim() == 3) || (!batched && A.dim() == 2 && B.dim() == 2), "lora_fold: A/B ranks");
  const int64_t batch = batched ? A.size(0) : 1;
  TORCH_CHECK(W.dim() == 2 || (W.dim() == 3 && W.size(0) == batch), "lora_fold: W must be [rows, cols] or [batch, ...]");
  const int64_t rows = W.size(-2), cols = W.size(-1);
  const int64_t rank = layout == 0 ? A.size(-2) : A.size(-1);
  if (layout == 0) {
    TORCH_CHECK(A.size(-1) == cols && B.size(-2) == rows && B.size(-1) == rank, "lora_fold: [out,in] shapes");
  } else {
    TORCH_CHECK(A.size(-2) == rows && B.size(-2) == rank && B.size(-1) == cols, "lora_fold: [in,out] shapes");
  }
  TORCH_CHECK(scale.numel() == batch, "lora_fold: one scale per matrix");
  c10::cuda::CUDAGuard guard(W.device());
  auto out = batched ? at::empty({batch, rows, cols}, W.options()) : at::empty({rows, cols}, W.options());
  check_rc(stageml_lora_fold(W.data_ptr(), A.data_ptr(), B.data_ptr(), scale.data_ptr<float>(), (int)batch, (int)rows,
                             (int)cols, (int)rank, (int)layout, W.dim() == 3 ? rows * cols : 0,
                             batched ? A.stride(0) : 0, batched ? B.stride(0) : 0, dtype_code(W), out.data_ptr(),
                             cur_stream()),
           "lora_fold");
  return out;
}

Tensor lora_linear(const Tensor& x, const Tensor& w_bank, const c10::optional<Tensor>& bias,
                   const c10::optional<Tensor>& row_group, const c10::optional<Tensor>& row_tenant, int64_t n_tenants,
                   int64_t rank, const c10::optional<Tensor>& lora_a, const c10::optional<Tensor>& lora_b,
                   const c10::optional<Tensor>& lora_scale) {
  check_cuda(x, "x", x);
  check_cuda(w_bank, "w_bank", x);
  TORCH_CHECK(x.dim() == 2 && w_bank.dim() == 3 && w_bank.size(2) == x.size(1), "lora_linear: shapes");
  TORCH_CHECK(w_bank.scalar_type() == x.scalar_type(), "lora_linear: dtype mismatch");
  for (const auto* o : {&bias, &row_group, &row_tenant, &lora_a, &lora_b, &lora_scale})
    if (o->has_value()) check_cuda(**o, "optional input", x);
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w_bank.size(1);
  auto y = at::empty({M, N}, x.options());
  stageml_lora_linear_args a{};
  a.M = (int)M;
  a.K = (int)K;
  a.N = (int)N;
  a.dtype = dtype_code(x);
  a.x = x.data_ptr();
  a.w_bank = w_bank.data_ptr();
  a.n_groups = (int)w_bank.size(0);
  a.bias = opt_ptr(bias);
  a.row_group = static_cast<const int32_t*>(opt_ptr(row_group));
  a.row_tenant = static_cast<const int32_t*>(opt_ptr(row_tenant));
  a.n_tenants = (int)n_tenants;
  a.rank = (int)rank;
  a.lora_a = opt_ptr(lora_a);
  a.lora_b = opt_ptr(lora_b);
  a.lora_scale = static_cast<const float*>(opt_ptr(lora_scale));
  a.y = y.data_ptr();
  a.status = status_word(x);
  auto w = workspace(stageml_lora_linear_workspace_bytes(&a), x);
  check_rc(stageml_lora_linear(&a, w.data_ptr(), (size_t)w.numel(), cur_stream()), "lora_linear");
  return y;
}

Tensor moe_linear(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias, const Tensor& topk_ids,
                  const Tensor& topk_weights, const c10::optional<Tensor>& tenant_ids, int64_t n_experts,
                  bool group_by_tenant, int64_t n_tenants, int64_t rank, const c10::optional<Tensor>& lora_a,
                  const c10::optional<Tensor>& lora_b, const c10::optional<Tensor>& lora_scale) {
  check_cuda(x, "x", x);
  check_cuda(weight, "weight", x);
  check_cuda(topk_ids, "topk_ids", x);
  check_cuda(topk_weights, "topk_weights", x);
  for (const auto* o : {&bias, &tenant_ids, &lora_a, &lora_b, &lora_scale})
    if (o->has_value()) check_cuda(**o, "optional input", x);
  TORCH_CHECK(weight.dim() == 3 && weight.size(2) == x.size(1), "moe_linear: weight [G, N, K]");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t T = x.size(0), K = x.size(1), N = weight.size(1);
  auto out = at::empty({T, N}, x.options());
  const int k = (int)topk_ids.size(1);
  const size_t ws = stageml_moe_linear_workspace_bytes((int)T, (int)K, (int)N, (int)n_experts, k, group_by_tenant ? 1 : 0,
                                                       (int)n_tenants, (int)rank);
  auto w = workspace(ws, x);
  check_rc(stageml_moe_linear(x.data_ptr(), weight.data_ptr(), opt_ptr(bias), topk_ids.data_ptr(), dtype_code(topk_ids),
                              topk_weights.data_ptr(), dtype_code(topk_weights),
                              static_cast<const int32_t*>(opt_ptr(tenant_ids)), (int)T, (int)K, (int)N, (int)n_experts,
                              k, group_by_tenant ? 1 : 0, (int)n_tenants, (int)rank, opt_ptr(lora_a), opt_ptr(lora_b),
                              static_cast<const float*>(opt_ptr(lora_scale)), dtype_code(x), out.data_ptr(),
                              status_word(x), w.data_ptr(), (size_t)w.numel(), cur_stream()),
           "moe_linear");
  return out;
}

Tensor lora_gemv_f32(const Tensor& x, const Tensor& W, const c10::optional<Tensor>& A, const c10::optional<Tensor>& B,
                     double scale) {
  check_cuda(x, "x", x);
  check_cuda(W, "W", x);
  TORCH_CHECK(x.scalar_type() == at::kFloat && W.scalar_type() == at::kFloat, "lora_gemv_f32: fp32 only");
  TORCH_CHECK(x.dim() == 2 && W.dim() == 2 && W.size(0) == x.size(1), "lora_gemv_f32: x [M,in], W [in,out]");
  const int64_t M = x.size(0), in_f = x.size(1), out_f = W.size(1);
  int64_t rank = 0;
  if (A.has_value()) {
    check_cuda(*A, "A", x);
    TORCH_CHECK(B.has_value(), "lora_gemv_f32: A without B");
    check_cuda(*B, "B", x);
    rank = A->size(1);
    TORCH_CHECK(A->size(0) == in_f && B->size(0) == rank && B->size(1) == out_f, "lora_gemv_f32: A [in,r], B [r,out]");
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto y = at::empty({M, out_f}, x.options());
  auto w = workspace(stageml_lora_gemv_f32_workspace_bytes((int)M, (int)in_f, (int)out_f, (int)rank), x);
  check_rc(stageml_lora_gemv_f32(x.data_ptr<float>(), W.data_ptr<float>(),
                                 A.has_value() ? A->data_ptr<float>() : nullptr,
                                 B.has_value() ? B->data_ptr<float>() : nullptr, (float)scale, (int)M, (int)in_f,
                                 (int)out_f, (int)rank, y.data_ptr<float>(), w.data_ptr(), (size_t)w.numel(),
                                 cur_stream()),
           "lora_gemv_f32");
  return y;
}

std::tuple<Tensor, Tensor> quantize_e4m3_rows(const Tensor& w) {
  check_cuda(w, "w", w);
  TORCH_CHECK(w.dim() >= 1, "quantize_e4m3_rows: need at least one dim");
  c10::cuda::CUDAGuard guard(w.device());
  const int64_t cols = w.size(-1), rows = w.numel() / std::max<int64_t>(cols, 1);
  auto q = at::empty(w.sizes(), w.options().dtype(at::kFloat8_e4m3fn));
  auto sizes = w.sizes().vec();
  sizes.pop_back();
  auto s = at::empty(sizes, w.options().dtype(at::kFloat));
  check_rc(stageml_quantize_e4m3_rows(w.data_ptr(), dtype_code(w), rows, cols, static_cast<uint8_t*>(q.data_ptr()),
                                      s.data_ptr<float>(), cur_stream()),
           "quantize_e4m3_rows");
  return {q, s};
}

Tensor combine_rows(const Tensor& y, const Tensor& pair_row, int64_t T, int64_t kk) {
  check_cuda(y, "y", y);
  check_cuda(pair_row, "pair_row", y);
  TORCH_CHECK(y.dim() == 2 && pair_row.scalar_type() == at::kInt && pair_row.numel() >= T * kk,
              "combine_rows: y [rows, H], pair_row int32 [T*kk]");
  c10::cuda::CUDAGuard guard(y.device());
  auto out = at::empty({T, y.size(1)}, y.options());
  check_rc(stageml_combine_rows(y.data_ptr(), pair_row.data_ptr<int32_t>(), (int)T, (int)kk, (int)y.size(1),
                                dtype_code(y), out.data_ptr(), cur_stream()),
           "combine_rows");
  return out;
}

// ------------------------------------------------ block-scaled FP8, block norm, balance loss
void check_e4m3(const Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn, "stageml: ", what, " must be float8_e4m3fn, got ", t.scalar_type());
}
void check_float_dtype(const Tensor& t, const char* what) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, "stageml: ",
              what, " must be float32, bfloat16 or float16, got ", t.scalar_type());
}
int64_t blocks128(int64_t n) { return (n + 127) / 128; }

// These operators have no autograd kernel (below), so a gradient or a tangent that an input asks for would be dropped
// without a word. The differentiable ones are called under their autograd functions, where grad mode is off.
void refuse_gradient(const char* op, const Tensor& t) {
  if (!t.defined()) return;
  const bool asks = (c10::GradMode::is_enabled() && t.requires_grad()) ||
                    (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined());
  TORCH_CHECK(!asks, op, " has no gradient for its inputs here: call it under torch.no_grad() or on detached tensors, or "
              "the differentiable function of stageml_b200.ops");
}
void refuse_gradient(const char* op, const c10::optional<Tensor>& t) {
  if (t.has_value()) refuse_gradient(op, *t);
}
template <typename... Ts>
void refuse_gradients(const char* op, const Ts&... tensors) {
  (refuse_gradient(op, tensors), ...);
}

std::tuple<Tensor, Tensor> quantize_e4m3_blocks(const Tensor& x, bool tiles) {
  refuse_gradients("quantize_e4m3_blocks", x);
  check_cuda(x, "x", x);
  check_float_dtype(x, "quantize_e4m3_blocks: x");
  TORCH_CHECK(x.dim() >= (tiles ? 2 : 1), "quantize_e4m3_blocks: x needs at least ", tiles ? 2 : 1, " dims");
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t cols = x.size(-1), rows = x.dim() >= 2 ? x.size(-2) : 1;
  int64_t batch = 1;
  for (int64_t d = 0; d + 2 < x.dim(); ++d) batch *= x.size(d);
  auto sizes = x.sizes().vec();
  sizes.back() = blocks128(cols);
  if (tiles) sizes[sizes.size() - 2] = blocks128(rows);
  auto q = fresh(x.sizes(), at::kFloat8_e4m3fn, x);
  auto s = fresh(sizes, at::kFloat, x);
  check_rc(stageml_quantize_e4m3_blocks(x.data_ptr(), dtype_code(x), batch, rows, cols, tiles ? 1 : 0,
                                        static_cast<uint8_t*>(q.data_ptr()), s.data_ptr<float>(), cur_stream()),
           "quantize_e4m3_blocks");
  return {q, s};
}

Tensor block_matmul(const Tensor& x, const Tensor& x_scale, const Tensor& w, const Tensor& w_scale,
                    at::ScalarType out_dtype) {
  refuse_gradients("block_matmul", x, x_scale, w, w_scale);
  check_cuda(x, "x", x);
  check_cuda(x_scale, "x_scale", x);
  check_cuda(w, "w", x);
  check_cuda(w_scale, "w_scale", x);
  check_e4m3(x, "block_matmul: x");
  check_e4m3(w, "block_matmul: w");
  TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && w.size(1) == x.size(1), "block_matmul: x [M, K] and w [N, K], got ",
              x.sizes(), " and ", w.sizes());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK(M <= INT32_MAX && N <= INT32_MAX && K <= INT32_MAX, "block_matmul: sizes past 2^31");
  TORCH_CHECK(x_scale.scalar_type() == at::kFloat && x_scale.dim() == 2 && x_scale.size(0) == M &&
                  x_scale.size(1) == blocks128(K),
              "block_matmul: x_scale must be fp32 [M, ceil(K/128)], got ", x_scale.sizes());
  TORCH_CHECK(w_scale.scalar_type() == at::kFloat && w_scale.dim() == 2 && w_scale.size(0) == blocks128(N) &&
                  w_scale.size(1) == blocks128(K),
              "block_matmul: w_scale must be fp32 [ceil(N/128), ceil(K/128)], got ", w_scale.sizes());
  c10::cuda::CUDAGuard guard(x.device());
  auto out = fresh({M, N}, out_dtype, x);
  check_float_dtype(out, "block_matmul: out_dtype");
  check_rc(stageml_block_matmul(static_cast<const uint8_t*>(x.data_ptr()), x_scale.data_ptr<float>(),
                                static_cast<const uint8_t*>(w.data_ptr()), w_scale.data_ptr<float>(), (int)M, (int)N,
                                (int)K, dtype_code(out), out.data_ptr(), status_word(x), cur_stream()),
           "block_matmul");
  return out;
}

Tensor moe_forward_blocks(const Tensor& x, const Tensor& gate_up, const Tensor& gate_up_scale, const Tensor& down,
                          const Tensor& down_scale, const c10::optional<Tensor>& topk_ids,
                          const c10::optional<Tensor>& topk_weights, int64_t n_shared) {
  refuse_gradients("moe_forward_blocks", x, gate_up, gate_up_scale, down, down_scale, topk_weights);
  TORCH_CHECK(x.dim() == 2 && gate_up.dim() == 3 && down.dim() == 3, "moe_forward_blocks: x [T, H], gate_up [E, 2I, H], ",
              "down [E, H, I]");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf,
              "moe_forward_blocks: x must be bfloat16 or float16");
  check_e4m3(gate_up, "moe_forward_blocks: gate_up");
  check_e4m3(down, "moe_forward_blocks: down");
  const int64_t T = x.size(0), H = x.size(1), E_tot = gate_up.size(0), I = gate_up.size(1) / 2;
  TORCH_CHECK(gate_up.size(1) % 2 == 0 && gate_up.size(2) == H && down.size(0) == E_tot && down.size(1) == H &&
                  down.size(2) == I,
              "moe_forward_blocks: weight shapes do not match x");
  TORCH_CHECK(T <= INT32_MAX && H <= INT32_MAX && I <= INT32_MAX && E_tot <= INT32_MAX,
              "moe_forward_blocks: sizes past 2^31");
  TORCH_CHECK(n_shared >= 0 && n_shared <= E_tot, "moe_forward_blocks: n_shared out of range");
  TORCH_CHECK(gate_up_scale.scalar_type() == at::kFloat &&
                  gate_up_scale.sizes() == at::IntArrayRef({E_tot, blocks128(2 * I), blocks128(H)}),
              "moe_forward_blocks: gate_up_scale must be fp32 [E, ceil(2I/128), ceil(H/128)], got ",
              gate_up_scale.sizes());
  TORCH_CHECK(down_scale.scalar_type() == at::kFloat &&
                  down_scale.sizes() == at::IntArrayRef({E_tot, blocks128(H), blocks128(I)}),
              "moe_forward_blocks: down_scale must be fp32 [E, ceil(H/128), ceil(I/128)], got ", down_scale.sizes());
  for (auto* t : {&x, &gate_up, &gate_up_scale, &down, &down_scale}) check_cuda(*t, "input", x);
  TORCH_CHECK(topk_ids.has_value() == topk_weights.has_value(), "moe_forward_blocks: topk_ids and topk_weights go together");
  int64_t k = 0;
  if (topk_ids.has_value()) {
    check_cuda(*topk_ids, "topk_ids", x);
    check_cuda(*topk_weights, "topk_weights", x);
    check_float_dtype(*topk_weights, "moe_forward_blocks: topk_weights");
    TORCH_CHECK(topk_ids->dim() == 2 && topk_ids->size(0) == T && topk_weights->sizes() == topk_ids->sizes(),
                "moe_forward_blocks: topk_ids and topk_weights must be [T, k]");
    k = topk_ids->size(1);
  }
  c10::cuda::CUDAGuard guard(x.device());
  auto out = fresh({T, H}, x.scalar_type(), x);
  stageml_moe_blocks_args a{};
  a.T = (int)T;
  a.H = (int)H;
  a.I = (int)I;
  a.E = (int)(E_tot - n_shared);
  a.k = (int)k;
  a.n_shared = (int)n_shared;
  a.act_dtype = dtype_code(x);
  a.x = x.data_ptr();
  a.topk_ids = opt_ptr(topk_ids);
  a.ids_dtype = topk_ids.has_value() ? dtype_code(*topk_ids) : STAGEML_I32;
  a.topk_weights = opt_ptr(topk_weights);
  a.weights_dtype = topk_weights.has_value() ? dtype_code(*topk_weights) : STAGEML_F32;
  a.gate_up = static_cast<const uint8_t*>(gate_up.data_ptr());
  a.gate_up_scale = gate_up_scale.data_ptr<float>();
  a.down = static_cast<const uint8_t*>(down.data_ptr());
  a.down_scale = down_scale.data_ptr<float>();
  a.out = out.data_ptr();
  a.status = status_word(x);
  const size_t ws = stageml_moe_blocks_workspace_bytes(&a);
  TORCH_CHECK(ws > 0, "moe_forward_blocks: invalid arguments: ", stageml_last_error());
  auto w = workspace(ws, x);
  check_rc(stageml_moe_forward_blocks(&a, w.data_ptr(), (size_t)w.numel(), cur_stream()), "moe_forward_blocks");
  return out;
}

// How a gate is broadcast over a residual [..., H]: per channel [H] (or [1, .., H]), per
// token [..., 1], or full.
int gate_mode_of(const Tensor& gate, const Tensor& residual) {
  const auto rs = residual.sizes(), gs = gate.sizes();
  if (gs == rs) return STAGEML_GATE_FULL;
  if (!gs.empty() && gs.back() == rs.back() && gate.numel() == rs.back()) return STAGEML_GATE_CHANNEL;
  if (gs.size() == rs.size() && gs.back() == 1 && gs.slice(0, gs.size() - 1) == rs.slice(0, rs.size() - 1))
    return STAGEML_GATE_TOKEN;
  TORCH_CHECK(false, "norm_residual: gate ", gs, " must be [H], [..., 1] or [..., H] for a residual ", rs);
  return -1;
}

// The inputs that the forward and the backward share, made contiguous, and their arguments.
struct NormInputs {
  c10::optional<Tensor> block_out, post, gate, pre;
  Tensor residual;
  stageml_norm_args a{};
};

c10::optional<Tensor> norm_input(const c10::optional<Tensor>& t, const Tensor& residual, const char* name) {
  if (!t.has_value()) return c10::nullopt;
  TORCH_CHECK(t->is_cuda() && t->device() == residual.device(), "norm_residual: ", name, " must be on ",
              residual.device(), ", got ", t->device());
  check_float_dtype(*t, name);
  return t->contiguous();
}

void norm_inputs(NormInputs* n, const c10::optional<Tensor>& block_out, const Tensor& residual,
                 const c10::optional<Tensor>& post_weight, const c10::optional<Tensor>& gate,
                 const c10::optional<Tensor>& pre_weight, double residual_scale, double eps,
                 at::ScalarType block_dtype) {
  TORCH_CHECK(residual.is_cuda(), "norm_residual: residual must be a CUDA tensor");
  TORCH_CHECK(residual.dim() >= 1, "norm_residual: residual must be [..., H]");
  check_float_dtype(residual, "norm_residual: residual");
  const int64_t H = residual.size(-1);
  TORCH_CHECK(H >= 1 && H <= INT32_MAX, "norm_residual: bad width ", H);
  n->residual = residual.contiguous();
  n->block_out = norm_input(block_out, residual, "block_out");
  n->post = norm_input(post_weight, residual, "post_weight");
  n->gate = norm_input(gate, residual, "gate");
  n->pre = norm_input(pre_weight, residual, "pre_weight");
  if (block_out.has_value()) {
    TORCH_CHECK(block_out->sizes() == residual.sizes(), "norm_residual: block_out must have residual's shape");
    TORCH_CHECK(block_out->scalar_type() == block_dtype, "norm_residual: block_out must be ", block_dtype);
  }
  for (const auto* w : {&n->post, &n->pre})
    if (w->has_value())
      TORCH_CHECK((*w)->dim() == 1 && (*w)->size(0) == H, "norm_residual: a norm weight must be [H], got ",
                  (*w)->sizes());
  stageml_norm_args& a = n->a;
  a.T = residual.numel() / H;
  a.H = (int)H;
  a.resid_dtype = dtype_code(residual);
  a.block_dtype = block_dtype == at::kFloat      ? STAGEML_F32
                  : block_dtype == at::kBFloat16 ? STAGEML_BF16
                  : block_dtype == at::kHalf     ? STAGEML_F16
                                                 : -1;
  a.residual = n->residual.data_ptr();
  a.block_out = opt_ptr(n->block_out);
  a.post_weight = opt_ptr(n->post);
  a.post_dtype = n->post.has_value() ? dtype_code(*n->post) : STAGEML_F32;
  a.gate = opt_ptr(n->gate);
  a.gate_mode = n->gate.has_value() ? gate_mode_of(*gate, residual) : STAGEML_GATE_NONE;
  a.gate_dtype = n->gate.has_value() ? dtype_code(*n->gate) : STAGEML_F32;
  a.pre_weight = opt_ptr(n->pre);
  a.pre_dtype = n->pre.has_value() ? dtype_code(*n->pre) : STAGEML_F32;
  a.residual_scale = (float)residual_scale;
  a.eps = (float)eps;
  a.status = status_word(residual);
}

// -> [new_residual], [new_residual, normed] or [new_residual, codes, scale]
std::vector<Tensor> norm_residual(const c10::optional<Tensor>& block_out, const Tensor& residual,
                                  const c10::optional<Tensor>& post_weight, const c10::optional<Tensor>& gate,
                                  const c10::optional<Tensor>& pre_weight, double residual_scale, double eps,
                                  bool quantize, c10::optional<at::ScalarType> normed_dtype) {
  refuse_gradients("norm_residual", block_out, residual, post_weight, gate, pre_weight);
  const at::ScalarType bd = block_out.has_value()      ? block_out->scalar_type()
                            : normed_dtype.has_value() ? *normed_dtype
                                                       : residual.scalar_type();
  TORCH_CHECK(!normed_dtype.has_value() || *normed_dtype == bd, "norm_residual: normed_dtype must be block_out's dtype");
  NormInputs n;
  norm_inputs(&n, block_out, residual, post_weight, gate, pre_weight, residual_scale, eps, bd);
  stageml_norm_args& a = n.a;
  TORCH_CHECK(!quantize || pre_weight.has_value(), "norm_residual: quantize needs pre_weight");
  c10::cuda::CUDAGuard guard(residual.device());
  std::vector<Tensor> out;
  out.reserve(3);
  out.push_back(fresh(residual.sizes(), residual.scalar_type(), residual));
  a.new_residual = out[0].data_ptr();
  if (quantize) {
    auto sizes = residual.sizes().vec();
    sizes.back() = blocks128(a.H);
    out.push_back(fresh(residual.sizes(), at::kFloat8_e4m3fn, residual));
    out.push_back(fresh(sizes, at::kFloat, residual));
    a.codes = static_cast<uint8_t*>(out[1].data_ptr());
    a.code_scale = out[2].data_ptr<float>();
  } else if (pre_weight.has_value()) {
    out.push_back(fresh(residual.sizes(), bd, residual));
    a.normed = out[1].data_ptr();
  }
  const size_t bytes = stageml_norm_residual_workspace_bytes(&a, 0);
  Tensor ws = bytes ? workspace(bytes, residual) : Tensor();
  check_rc(stageml_norm_residual(&a, bytes ? ws.data_ptr() : nullptr, bytes, cur_stream()), "norm_residual");
  return out;
}

// -> gradients of [residual, block_out?, post_weight?, gate?, pre_weight?] (those present, in this order)
std::vector<Tensor> norm_residual_backward(const c10::optional<Tensor>& grad_residual,
                                           const c10::optional<Tensor>& grad_normed,
                                           const c10::optional<Tensor>& block_out, const Tensor& residual,
                                           const c10::optional<Tensor>& post_weight, const c10::optional<Tensor>& gate,
                                           const c10::optional<Tensor>& pre_weight, double residual_scale, double eps) {
  refuse_gradients("norm_residual_backward", grad_residual, grad_normed, block_out, residual, post_weight, gate, pre_weight);
  TORCH_CHECK(grad_residual.has_value() || grad_normed.has_value(), "norm_residual_backward: no gradient given");
  const at::ScalarType bd = block_out.has_value()     ? block_out->scalar_type()
                            : grad_normed.has_value() ? grad_normed->scalar_type()
                                                      : residual.scalar_type();
  NormInputs n;
  norm_inputs(&n, block_out, residual, post_weight, gate, pre_weight, residual_scale, eps, bd);
  stageml_norm_args& a = n.a;
  const auto dr = norm_input(grad_residual, residual, "grad_residual");
  const auto dz = norm_input(grad_normed, residual, "grad_normed");
  TORCH_CHECK(!dr.has_value() || (dr->sizes() == residual.sizes() && dr->scalar_type() == residual.scalar_type()),
              "norm_residual_backward: grad_residual must match residual");
  TORCH_CHECK(!dz.has_value() || (dz->sizes() == residual.sizes() && dz->scalar_type() == bd),
              "norm_residual_backward: grad_normed must have residual's shape and the block dtype");
  TORCH_CHECK(!dz.has_value() || pre_weight.has_value(), "norm_residual_backward: grad_normed without pre_weight");
  c10::cuda::CUDAGuard guard(residual.device());
  a.grad_residual = opt_ptr(dr);
  a.grad_normed = opt_ptr(dz);
  std::vector<Tensor> out;
  out.reserve(5);
  auto add = [&](const Tensor& like) {
    out.push_back(fresh(like.sizes(), like.scalar_type(), like));
    return out.back().data_ptr();
  };
  a.d_residual = add(residual);
  if (block_out.has_value()) a.d_block_out = add(*block_out);
  if (post_weight.has_value()) a.d_post = add(*post_weight);
  if (gate.has_value()) a.d_gate = add(*gate);
  if (pre_weight.has_value()) a.d_pre = add(*pre_weight);
  const size_t bytes = stageml_norm_residual_workspace_bytes(&a, 1);
  Tensor ws = bytes ? workspace(bytes, residual) : Tensor();
  check_rc(stageml_norm_residual_backward(&a, bytes ? ws.data_ptr() : nullptr, bytes, cur_stream()),
           "norm_residual_backward");
  return out;
}

const uint8_t* valid_ptr(const c10::optional<Tensor>& valid, const Tensor& logits) {
  if (!valid.has_value()) return nullptr;
  check_cuda(*valid, "valid", logits);
  TORCH_CHECK((valid->scalar_type() == at::kBool || valid->scalar_type() == at::kByte) &&
                  valid->numel() == logits.size(0),
              "balance_loss: valid must be bool or uint8 [T]");
  return static_cast<const uint8_t*>(valid->data_ptr());
}

std::tuple<Tensor, Tensor, Tensor> balance_loss(const Tensor& logits, const Tensor& topk_ids, double coefficient,
                                                const c10::optional<Tensor>& valid) {
  refuse_gradients("balance_loss", logits);
  check_cuda(logits, "logits", logits);
  check_cuda(topk_ids, "topk_ids", logits);
  check_float_dtype(logits, "balance_loss: logits");
  TORCH_CHECK(logits.dim() == 2 && topk_ids.dim() == 2 && topk_ids.size(0) == logits.size(0),
              "balance_loss: logits [T, E] and topk_ids [T, k], got ", logits.sizes(), " and ", topk_ids.sizes());
  const int64_t T = logits.size(0), E = logits.size(1), k = topk_ids.size(1);
  TORCH_CHECK(E >= 1 && E <= 256 && k >= 1 && k <= 8, "balance_loss: E=", E, " must be in 1..256 and k=", k, " in 1..8");
  const uint8_t* v = valid_ptr(valid, logits);
  c10::cuda::CUDAGuard guard(logits.device());
  auto loss = fresh({}, at::kFloat, logits);
  auto counts = fresh({E}, at::kInt, logits);
  auto tokens = fresh({}, at::kInt, logits);
  const size_t bytes = stageml_balance_workspace_bytes(T, (int)E);
  Tensor w = bytes ? workspace(bytes, logits) : Tensor();
  check_rc(stageml_balance_loss(logits.data_ptr(), dtype_code(logits), topk_ids.data_ptr(), dtype_code(topk_ids), v, T,
                                (int)E, (int)k, (float)coefficient, loss.data_ptr<float>(), counts.data_ptr<int32_t>(),
                                tokens.data_ptr<int32_t>(), status_word(logits), bytes ? w.data_ptr() : nullptr, bytes,
                                cur_stream()),
           "balance_loss");
  return {loss, counts, tokens};
}

Tensor balance_loss_backward(const Tensor& grad_loss, const Tensor& logits, const Tensor& counts, const Tensor& tokens,
                             int64_t k, double coefficient, const c10::optional<Tensor>& valid) {
  refuse_gradients("balance_loss_backward", grad_loss, logits);
  check_cuda(logits, "logits", logits);
  check_float_dtype(logits, "balance_loss_backward: logits");
  TORCH_CHECK(logits.dim() == 2, "balance_loss_backward: logits must be [T, E]");
  for (auto* t : {&grad_loss, &counts, &tokens}) check_cuda(*t, "input", logits);
  TORCH_CHECK(grad_loss.scalar_type() == at::kFloat && grad_loss.numel() == 1, "balance_loss_backward: grad_loss fp32 [1]");
  TORCH_CHECK(counts.scalar_type() == at::kInt && counts.numel() == logits.size(1) &&
                  tokens.scalar_type() == at::kInt && tokens.numel() == 1,
              "balance_loss_backward: counts int32 [E] and tokens int32 [1] of the forward");
  TORCH_CHECK(k >= 1 && k <= 8, "balance_loss_backward: k=", k, " must be in 1..8");
  const uint8_t* v = valid_ptr(valid, logits);
  c10::cuda::CUDAGuard guard(logits.device());
  auto grad = fresh(logits.sizes(), logits.scalar_type(), logits);
  check_rc(stageml_balance_loss_backward(grad_loss.data_ptr<float>(), logits.data_ptr(), dtype_code(logits),
                                         counts.data_ptr<int32_t>(), tokens.data_ptr<int32_t>(), v, logits.size(0),
                                         (int)logits.size(1), (int)k, (float)coefficient, grad.data_ptr(), cur_stream()),
           "balance_loss_backward");
  return grad;
}

// Returns the device status word (synchronising on it) and clears it.
int64_t take_status(const Tensor& like) {
  c10::cuda::CUDAGuard guard(like.device());
  int32_t* p = status_word(like);
  auto t = at::from_blob(p, {1}, like.options().dtype(at::kInt));
  const int64_t v = t.item<int32_t>();
  t.zero_();
  return v;
}

}  // namespace

TORCH_LIBRARY(stageml, m) {
  m.def("residual_moe(Tensor hidden, Tensor gate_up, Tensor down, Tensor topk_weights, Tensor topk_ids) -> Tensor");
  m.def(
      "moe_forward(Tensor x, Tensor gate_up, Tensor down, Tensor? topk_weights, Tensor? topk_ids, Tensor? router_w, "
      "int k, int n_shared, bool renormalize, Tensor? tenant_ids, int n_tenants, int rank, Tensor? lora_a13, "
      "Tensor? lora_b13, Tensor? lora_a2, Tensor? lora_b2, Tensor? lora_scale, Tensor? gate_up_scale, "
      "Tensor? down_scale, Tensor? T_dev=None, Tensor? fold_slot=None, int n_fold=0, Tensor? down_group=None) "
      "-> Tensor");
  m.def("route_topk(Tensor x, Tensor gate_w, int k, bool renormalize) -> (Tensor, Tensor, Tensor)");
  m.def("topk_from_logits(Tensor logits, int k, bool renormalize) -> (Tensor, Tensor)");
  m.def(
      "permute(Tensor ids, Tensor? weights, Tensor? tenant_ids, int n_experts_total, int n_shared, int n_tenants, "
      "bool group_by_tenant) -> Tensor[]");
  m.def("lora_fold(Tensor W, Tensor A, Tensor B, Tensor scale, int layout) -> Tensor");
  m.def(
      "lora_linear(Tensor x, Tensor w_bank, Tensor? bias, Tensor? row_group, Tensor? row_tenant, int n_tenants, "
      "int rank, Tensor? lora_a, Tensor? lora_b, Tensor? lora_scale) -> Tensor");
  m.def(
      "moe_linear(Tensor x, Tensor weight, Tensor? bias, Tensor topk_ids, Tensor topk_weights, Tensor? tenant_ids, "
      "int n_experts, bool group_by_tenant, int n_tenants, int rank, Tensor? lora_a, Tensor? lora_b, "
      "Tensor? lora_scale) -> Tensor");
  m.def("lora_gemv_f32(Tensor x, Tensor W, Tensor? A, Tensor? B, float scale) -> Tensor");
  m.def("quantize_e4m3_rows(Tensor w) -> (Tensor, Tensor)");
  m.def("combine_rows(Tensor y, Tensor pair_row, int T, int kk) -> Tensor");
  m.def("take_status(Tensor like) -> int");
  m.def("quantize_e4m3_blocks(Tensor x, bool tiles) -> (Tensor, Tensor)");
  m.def("block_matmul(Tensor x, Tensor x_scale, Tensor w, Tensor w_scale, ScalarType out_dtype) -> Tensor");
  m.def(
      "moe_forward_blocks(Tensor x, Tensor gate_up, Tensor gate_up_scale, Tensor down, Tensor down_scale, "
      "Tensor? topk_ids, Tensor? topk_weights, int n_shared) -> Tensor");
  m.def(
      "norm_residual(Tensor? block_out, Tensor residual, Tensor? post_weight, Tensor? gate, "
      "Tensor? pre_weight, float residual_scale, float eps, bool quantize, ScalarType? normed_dtype) -> Tensor[]");
  m.def(
      "norm_residual_backward(Tensor? grad_residual, Tensor? grad_normed, Tensor? block_out, Tensor residual, "
      "Tensor? post_weight, Tensor? gate, Tensor? pre_weight, float residual_scale, float eps) "
      "-> Tensor[]");
  m.def("balance_loss(Tensor logits, Tensor topk_ids, float coefficient, Tensor? valid) -> (Tensor, Tensor, Tensor)");
  m.def(
      "balance_loss_backward(Tensor grad_loss, Tensor logits, Tensor counts, Tensor tokens, int k, "
      "float coefficient, Tensor? valid) -> Tensor");
}

TORCH_LIBRARY_IMPL(stageml, CUDA, m) {
  m.impl("residual_moe", &residual_moe);
  m.impl("moe_forward", &moe_forward);
  m.impl("route_topk", &route_topk);
  m.impl("topk_from_logits", &topk_from_logits);
  m.impl("permute", &permute);
  m.impl("lora_fold", &lora_fold);
  m.impl("lora_linear", &lora_linear);
  m.impl("moe_linear", &moe_linear);
  m.impl("lora_gemv_f32", &lora_gemv_f32);
  m.impl("quantize_e4m3_rows", &quantize_e4m3_rows);
  m.impl("combine_rows", &combine_rows);
  m.impl("take_status", &take_status);
  m.impl("quantize_e4m3_blocks", &quantize_e4m3_blocks);
  m.impl("block_matmul", &block_matmul);
  m.impl("moe_forward_blocks", &moe_forward_blocks);
  m.impl("norm_residual", &norm_residual);
  m.impl("norm_residual_backward", &norm_residual_backward);
  m.impl("balance_loss", &balance_loss);
  m.impl("balance_loss_backward", &balance_loss_backward);
}

// The operators above without an autograd formula of their own in the dispatcher: ops.py
// wraps the differentiable ones in autograd functions, and each refuses gradients and tangents
// itself, so the dispatcher's generic autograd kernel (several us per call) is passed by.
TORCH_LIBRARY_IMPL(stageml, Autograd, m) {
  for (const char* op : {"quantize_e4m3_blocks", "block_matmul", "moe_forward_blocks", "norm_residual",
                         "norm_residual_backward", "balance_loss", "balance_loss_backward"})
    m.impl(op, torch::CppFunction::makeFallthrough());
}
