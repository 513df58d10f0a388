// warp_route._C: the torch-op boundary (src/bindings.cpp:145-152 in the
// reference), implemented over the C-ABI of libwarp_route_hip.so.
//
// The three ops keep the reference's names and seven positional arguments
// (hidden, gate_w, weight_buf, num_experts, hidden_dim, intermediate_dim,
// top_k) and add trailing defaulted ones:
//   renormalize=False  divide the selected weights by their sum
//   topk_ids=None      optional int32 [k] / [B,k] output of selected experts
//   topk_weights=None  optional fp32 [k] / [B,k] output of their weights
// Differences from the reference, all compatible with its call forms:
//   * weight_buf may be float32 (the reference layout), float16, bfloat16,
//     float8_e4m3fn (codes plus fp32 row scales) or float4_e2m1fn_x2 (MXFP4
//     codes plus E8M0 block scales), laid out as wr_layout_dtype says; hidden
//     may be float32 or float16 and the output takes its dtype; gate_w is
//     float32.
//   * top_k may be 1..min(6, num_experts) on every op (the reference's fused
//     and batched ops accepted only 1 or 2, src/bindings.cpp:75,117).
//   * work is enqueued on the current HIP stream of hidden's device and the
//     device is not synchronised (the reference used stream 0 and
//     cudaDeviceSynchronize, src/bindings.cpp:54-55,93-94,137-140).
//   * scratch comes from the caching allocator; nothing calls hipMalloc per
//     call (the reference's naive op did, src/bindings.cpp:53-56).
// ROCm builds of torch report HIP tensors as device type "cuda"; the
// *MasqueradingAsCUDA guard and stream accessors accept that device type.
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <cstdlib>
#include <optional>

#include "warp_route.h"
#include "wr_ffn.h"

namespace {

// When set, fused_moe_forward reads the hand-off status of its call
// (wr_fused_moe_status, which synchronises the stream) and raises if a wait
// expired.  Off by default: the check costs a stream synchronisation and
// cannot run under graph capture.  WARP_ROUTE_CHECK_HANDOFF=1 in the
// environment turns it on at import.
std::atomic<bool> g_check_handoff{[] {
  const char* v = std::getenv("WARP_ROUTE_CHECK_HANDOFF");
  return v != nullptr && v[0] != '\0' && v[0] != '0';
}()};

#define WR_CHECK_DEVICE(t) TORCH_CHECK((t).is_cuda(), #t " must be a CUDA (HIP) tensor")
#define WR_CHECK_CONTIGUOUS(t) TORCH_CHECK((t).is_contiguous(), #t " must be contiguous")

int dtype_tag(const torch::Tensor& t, const char* name) {
  if (t.scalar_type() == torch::kFloat32) return WR_F32;
  if (t.scalar_type() == torch::kFloat16) return WR_F16;
  TORCH_CHECK(false, name, " must be float32 or float16, got ", t.scalar_type());
  return -1;
}

int weight_dtype_tag(const torch::Tensor& t) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return WR_F32;
    case torch::kFloat16: return WR_F16;
    case torch::kBFloat16: return WR_BF16;
    case torch::kFloat8_e4m3fn: return WR_FP8_E4M3;
    case torch::kFloat4_e2m1fn_x2: return WR_MXFP4;
    default:
      TORCH_CHECK(false,
                  "weight_buf must be float32, float16, bfloat16, float8_e4m3fn or "
                  "float4_e2m1fn_x2, got ",
                  t.scalar_type());
  }
  return -1;
}

void check_common(const torch::Tensor& gate_w, const torch::Tensor& weight_buf, int num_experts,
                  int hidden_dim, int intermediate_dim, int top_k,
                  const torch::Device& dev) {
  WR_CHECK_DEVICE(gate_w);
  WR_CHECK_CONTIGUOUS(gate_w);
  TORCH_CHECK(gate_w.scalar_type() == torch::kFloat32, "gate_w must be float32");
  TORCH_CHECK(gate_w.dim() == 2 && gate_w.size(0) == num_experts && gate_w.size(1) == hidden_dim,
              "gate_w must have shape [", num_experts, ", ", hidden_dim, "], got shape ",
              gate_w.sizes());
  WR_CHECK_DEVICE(weight_buf);
  WR_CHECK_CONTIGUOUS(weight_buf);
  const int wdt = weight_dtype_tag(weight_buf);
  TORCH_CHECK(gate_w.device() == dev && weight_buf.device() == dev,
              "hidden, gate_w and weight_buf must be on the same device");
  TORCH_CHECK(num_experts >= 1 && hidden_dim >= 1 && intermediate_dim >= 1,
              "num_experts, hidden_dim and intermediate_dim must be positive");
  TORCH_CHECK(num_experts <= WR_MAX_EXPERTS, "num_experts ", num_experts,
              " exceeds GATE_MAX_EXPERTS ", WR_MAX_EXPERTS);
  TORCH_CHECK(top_k >= 1 && top_k <= WR_MAX_TOPK && top_k <= num_experts,
              "top_k must be in [1, min(", WR_MAX_TOPK, ", num_experts)], got ", top_k);
  const int64_t es = weight_buf.element_size();
  TORCH_CHECK(wdt != WR_MXFP4 || (hidden_dim % 32 == 0 && intermediate_dim % 32 == 0),
              "MXFP4 weights need hidden_dim and intermediate_dim to be multiples of 32, got ",
              hidden_dim, " and ", intermediate_dim);
  const int64_t need = wr_weight_bytes(num_experts, hidden_dim, intermediate_dim, wdt);
  TORCH_CHECK(weight_buf.numel() * es >= need, "weight_buf too small: need ", need,
              " bytes, got ", weight_buf.numel() * es);
}

void check_topk_out(const std::optional<torch::Tensor>& t, c10::ScalarType st, int64_t n,
                    const torch::Device& dev, const char* name) {
  if (!t.has_value()) return;
  const torch::Tensor& v = *t;
  WR_CHECK_DEVICE(v);
  WR_CHECK_CONTIGUOUS(v);
  TORCH_CHECK(v.scalar_type() == st, name, " must be ", st);
  TORCH_CHECK(v.device() == dev, name, " must be on hidden's device");
  TORCH_CHECK(v.numel() == n, name, " must hold ", n, " elements, got ", v.numel());
}

wr_moe_args make_args(const torch::Tensor& hidden, const torch::Tensor& gate_w,
                      const torch::Tensor& weight_buf, int E, int h, int I, int k, bool renorm,
                      int B, torch::Tensor& out, const std::optional<torch::Tensor>& ids,
                      const std::optional<torch::Tensor>& ws_out) {
  wr_moe_args a{};
  a.gate_w = gate_w.data_ptr<float>();
  a.weight_buf = weight_buf.data_ptr();
  a.weight_bytes = weight_buf.numel() * (int64_t)weight_buf.element_size();
  a.weight_dtype = weight_dtype_tag(weight_buf);
  a.num_experts = E;
  a.hidden_dim = h;
  a.intermediate_dim = I;
  a.top_k = k;
  a.renormalize = renorm ? 1 : 0;
  a.batch_size = B;
  a.act_dtype = dtype_tag(hidden, "hidden");
  a.x = hidden.data_ptr();
  a.out = out.data_ptr();
  a.topk_ids = ids.has_value() ? ids->data_ptr<int32_t>() : nullptr;
  a.topk_weights = ws_out.has_value() ? ws_out->data_ptr<float>() : nullptr;
  return a;
}

torch::Tensor alloc_workspace(int kind, int E, int h, int I, int k, int B,
                              const torch::Device& dev) {
  const size_t n = wr_workspace_bytes(kind, E, h, I, k, B);
  TORCH_CHECK(n > 0, "invalid MoE shape for workspace sizing");
  return torch::empty({(int64_t)n}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
}

void check_status(int st, const char* op) {
  TORCH_CHECK(st == WR_OK, op, " failed: ", wr_status_str(st), " (status ", st, ")");
}

// Expiries of single-token hand-off waits, read from the library's
// host-visible word without a synchronisation: this reports the expiries of
// every single-token call whose kernel has run by now (this one or an
// earlier one), once each.
void check_expired(const char* op) {
  TORCH_CHECK(wr_fused_moe_expired(1) == 0, op,
              " failed: a single-token fused call's hand-off wait expired (that call's output "
              "rows are NaN); seen after its kernel ran, so it may have been an earlier call");
}

torch::Tensor single_token_op(int kind, torch::Tensor hidden, torch::Tensor gate_w,
                              torch::Tensor weight_buf, int num_experts, int hidden_dim,
                              int intermediate_dim, int top_k, bool renormalize,
                              std::optional<torch::Tensor> topk_ids,
                              std::optional<torch::Tensor> topk_weights) {
  WR_CHECK_DEVICE(hidden);
  WR_CHECK_CONTIGUOUS(hidden);
  dtype_tag(hidden, "hidden");
  TORCH_CHECK(hidden.dim() == 1 && hidden.size(0) == hidden_dim, "hidden must have shape [",
              hidden_dim, "], got shape ", hidden.sizes());
  const torch::Device dev = hidden.device();
  check_common(gate_w, weight_buf, num_experts, hidden_dim, intermediate_dim, top_k, dev);
  check_topk_out(topk_ids, torch::kInt32, top_k, dev, "topk_ids");
  check_topk_out(topk_weights, torch::kFloat32, top_k, dev, "topk_weights");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  torch::Tensor out = torch::empty_like(hidden);
  torch::Tensor ws = alloc_workspace(kind, num_experts, hidden_dim, intermediate_dim, top_k, 1, dev);
  wr_moe_args a = make_args(hidden, gate_w, weight_buf, num_experts, hidden_dim,
                            intermediate_dim, top_k, renormalize, 1, out, topk_ids, topk_weights);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = (size_t)ws.numel();
  void* stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  if (kind == WR_KIND_FUSED) {
    check_status(wr_fused_moe(&a, stream), "fused_moe_forward");
    if (g_check_handoff.load(std::memory_order_relaxed)) {
      const int st = wr_fused_moe_status(a.workspace, a.workspace_bytes, stream);
      if (st == WR_ETIMEOUT) (void)wr_fused_moe_expired(1);  // reported here, not again
      check_status(st, "fused_moe_forward");
    }
    check_expired("fused_moe_forward");
  } else
    check_status(wr_naive_moe(&a, stream), "naive_moe_forward");
  return out;
}

// fused_moe_forward(hidden, gate_w, weight_buf, num_experts, hidden_dim,
// intermediate_dim, top_k) -- src/bindings.cpp:62-97.
torch::Tensor fused_moe_forward(torch::Tensor hidden, torch::Tensor gate_w,
                                torch::Tensor weight_buf, int num_experts, int hidden_dim,
                                int intermediate_dim, int top_k, bool renormalize,
                                std::optional<torch::Tensor> topk_ids,
                                std::optional<torch::Tensor> topk_weights) {
  return single_token_op(WR_KIND_FUSED, hidden, gate_w, weight_buf, num_experts, hidden_dim,
                         intermediate_dim, top_k, renormalize, topk_ids, topk_weights);
}

// naive_moe_forward(...) -- src/bindings.cpp:26-59.
torch::Tensor naive_moe_forward(torch::Tensor hidden, torch::Tensor gate_w,
                                torch::Tensor weight_buf, int num_experts, int hidden_dim,
                                int intermediate_dim, int top_k, bool renormalize,
                                std::optional<torch::Tensor> topk_ids,
                                std::optional<torch::Tensor> topk_weights) {
  return single_token_op(WR_KIND_NAIVE, hidden, gate_w, weight_buf, num_experts, hidden_dim,
                         intermediate_dim, top_k, renormalize, topk_ids, topk_weights);
}

// batched_fused_moe_forward(hidden_batch [B,h], ...) -> [B,h] --
// src/bindings.cpp:101-143.
torch::Tensor batched_fused_moe_forward(torch::Tensor hidden_batch, torch::Tensor gate_w,
                                        torch::Tensor weight_buf, int num_experts, int hidden_dim,
                                        int intermediate_dim, int top_k, bool renormalize,
                                        std::optional<torch::Tensor> topk_ids,
                                        std::optional<torch::Tensor> topk_weights) {
  WR_CHECK_DEVICE(hidden_batch);
  WR_CHECK_CONTIGUOUS(hidden_batch);
  dtype_tag(hidden_batch, "hidden_batch");
  TORCH_CHECK(hidden_batch.dim() == 2 && hidden_batch.size(1) == hidden_dim,
              "hidden_batch must have shape [batch_size, ", hidden_dim, "], got shape ",
              hidden_batch.sizes());
  const torch::Device dev = hidden_batch.device();
  check_common(gate_w, weight_buf, num_experts, hidden_dim, intermediate_dim, top_k, dev);
  const int B = (int)hidden_batch.size(0);
  check_topk_out(topk_ids, torch::kInt32, (int64_t)B * top_k, dev, "topk_ids");
  check_topk_out(topk_weights, torch::kFloat32, (int64_t)B * top_k, dev, "topk_weights");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  torch::Tensor out = torch::empty_like(hidden_batch);
  if (B == 0) return out;
  torch::Tensor ws =
      alloc_workspace(WR_KIND_BATCHED, num_experts, hidden_dim, intermediate_dim, top_k, B, dev);
  wr_moe_args a = make_args(hidden_batch, gate_w, weight_buf, num_experts, hidden_dim,
                            intermediate_dim, top_k, renormalize, B, out, topk_ids, topk_weights);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = (size_t)ws.numel();
  void* stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_status(wr_batched_fused_moe(&a, stream), "batched_fused_moe_forward");
  check_expired("batched_fused_moe_forward");
  return out;
}

// gate_topk(hidden [h] or [B,h], gate_w, num_experts, hidden_dim, top_k,
// renormalize=False) -> (ids int32, weights fp32), shaped like hidden's batch
// dims + [k].  Router logits, softmax and top-K only (src/gate.cu:103-116).
std::tuple<torch::Tensor, torch::Tensor> gate_topk(torch::Tensor hidden, torch::Tensor gate_w,
                                                   int num_experts, int hidden_dim, int top_k,
                                                   bool renormalize) {
  WR_CHECK_DEVICE(hidden);
  WR_CHECK_CONTIGUOUS(hidden);
  dtype_tag(hidden, "hidden");
  TORCH_CHECK((hidden.dim() == 1 || hidden.dim() == 2) && hidden.size(-1) == hidden_dim,
              "hidden must have shape [", hidden_dim, "] or [batch_size, ", hidden_dim,
              "], got shape ", hidden.sizes());
  WR_CHECK_DEVICE(gate_w);
  WR_CHECK_CONTIGUOUS(gate_w);
  TORCH_CHECK(gate_w.scalar_type() == torch::kFloat32, "gate_w must be float32");
  TORCH_CHECK(gate_w.dim() == 2 && gate_w.size(0) == num_experts && gate_w.size(1) == hidden_dim,
              "gate_w must have shape [", num_experts, ", ", hidden_dim, "], got shape ",
              gate_w.sizes());
  TORCH_CHECK(gate_w.device() == hidden.device(), "hidden and gate_w must be on the same device");
  TORCH_CHECK(num_experts <= WR_MAX_EXPERTS, "num_experts ", num_experts,
              " exceeds GATE_MAX_EXPERTS ", WR_MAX_EXPERTS);
  TORCH_CHECK(top_k >= 1 && top_k <= WR_MAX_TOPK && top_k <= num_experts,
              "top_k must be in [1, min(", WR_MAX_TOPK, ", num_experts)], got ", top_k);
  const torch::Device dev = hidden.device();
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  const int B = hidden.dim() == 2 ? (int)hidden.size(0) : 1;
  std::vector<int64_t> shape;
  if (hidden.dim() == 2) shape.push_back(B);
  shape.push_back(top_k);
  torch::Tensor ids = torch::empty(shape, torch::TensorOptions().dtype(torch::kInt32).device(dev));
  torch::Tensor ws = torch::empty(shape, torch::TensorOptions().dtype(torch::kFloat32).device(dev));
  if (B == 0) return {ids, ws};
  wr_moe_args a{};
  a.gate_w = gate_w.data_ptr<float>();
  a.weight_dtype = WR_F32;
  a.num_experts = num_experts;
  a.hidden_dim = hidden_dim;
  a.intermediate_dim = 1;
  a.top_k = top_k;
  a.renormalize = renormalize ? 1 : 0;
  a.batch_size = B;
  a.act_dtype = dtype_tag(hidden, "hidden");
  a.x = hidden.data_ptr();
  a.topk_ids = ids.data_ptr<int32_t>();
  a.topk_weights = ws.data_ptr<float>();
  void* stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
  check_status(wr_gate_topk(&a, stream), "gate_topk");
  return {ids, ws};
}

// ---- dense gated FFN and int8 products (include/wr_ffn.h) -------------------
int float_tag(const torch::Tensor& t, const char* name) {
  if (t.scalar_type() == torch::kBFloat16) return WR_BF16;
  if (t.scalar_type() == torch::kFloat32) return WR_F32;
  if (t.scalar_type() == torch::kFloat16) return WR_F16;
  TORCH_CHECK(false, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  return -1;
}

void check_operand(const torch::Tensor& t, const char* name, c10::ScalarType st,
                   const torch::Device& dev, at::IntArrayRef shape) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA (HIP) tensor");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.scalar_type() == st, name, " must be ", st, ", got ", t.scalar_type());
  TORCH_CHECK(t.device() == dev, name, " must be on the device of the first argument");
  TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape, ", got shape ", t.sizes());
}

void check_tokens(const torch::Tensor& x, const char* name) {
  TORCH_CHECK(x.is_cuda(), name, " must be a CUDA (HIP) tensor");
  TORCH_CHECK(x.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(x.dim() == 2, name, " must have shape [rows, columns], got shape ", x.sizes());
  TORCH_CHECK(x.size(0) <= WR_FFN_MAX_ROWS && x.size(1) >= 1, name, " has an unsupported shape ",
              x.sizes());
}

void check_dims(int64_t h, int64_t I, int64_t most) {
  TORCH_CHECK(h >= 1 && I >= 1 && h <= most && I <= most,
              "dimensions must be in [1, ", most, "], got ", h, " and ", I);
}

// The C-ABI takes 16-byte aligned pointers: a view that starts elsewhere is copied.
torch::Tensor aligned16(const torch::Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone();
}

torch::Tensor scratch(size_t bytes, const torch::Device& dev) {
  TORCH_CHECK(bytes > 0, "invalid shape for workspace sizing");
  return torch::empty({(int64_t)bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
}

void* stream_of(const torch::Device& dev) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
}

wr_ffn_args ffn_args(const torch::Tensor& x, const torch::Tensor& wg, const torch::Tensor& wu,
                     const torch::Tensor& wd) {
  wr_ffn_args a{};
  a.x = x.data_ptr();
  a.w_gate = wg.data_ptr();
  a.w_up = wu.data_ptr();
  a.w_down = wd.data_ptr();
  a.dtype = float_tag(x, "x");
  a.batch_size = (int32_t)x.size(0);
  a.hidden_dim = (int32_t)x.size(1);
  a.intermediate_dim = (int32_t)wg.size(0);
  return a;
}

void check_ffn(const torch::Tensor& x, const torch::Tensor& w_gate, const torch::Tensor& w_up,
               const torch::Tensor& w_down) {
  check_tokens(x, "x");
  float_tag(x, "x");
  TORCH_CHECK(w_gate.dim() == 2, "w_gate must have shape [intermediate_dim, hidden_dim], got shape ",
              w_gate.sizes());
  const int64_t h = x.size(1), I = w_gate.size(0);
  check_dims(h, I, WR_FFN_MAX_DIM);
  check_operand(w_gate, "w_gate", x.scalar_type(), x.device(), {I, h});
  check_operand(w_up, "w_up", x.scalar_type(), x.device(), {I, h});
  check_operand(w_down, "w_down", x.scalar_type(), x.device(), {h, I});
}

// gated_ffn_forward(x [T,h], w_gate [I,h], w_up [I,h], w_down [h,I], keep) -> [y], or
// [y, g, u, a] with keep: what gated_ffn_backward reads.
std::vector<torch::Tensor> gated_ffn_forward(torch::Tensor x, torch::Tensor w_gate,
                                             torch::Tensor w_up, torch::Tensor w_down, bool keep) {
  check_ffn(x, w_gate, w_up, w_down);
  const torch::Device dev = x.device();
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  x = aligned16(x);
  w_gate = aligned16(w_gate);
  w_up = aligned16(w_up);
  w_down = aligned16(w_down);
  std::vector<torch::Tensor> out{torch::empty_like(x)};
  wr_ffn_args a = ffn_args(x, w_gate, w_up, w_down);
  if (keep) {
    for (int i = 0; i < 3; ++i)
      out.push_back(torch::empty({x.size(0), wr_ffn_saved_row(a.intermediate_dim)},
                                 i < 2 ? x.options().dtype(torch::kFloat32) : x.options()));
    if (x.size(0) > 0) {
      a.saved_gate = out[1].data_ptr<float>();
      a.saved_up = out[2].data_ptr<float>();
      a.saved_act = out[3].data_ptr();
    }
  }
  if (x.size(0) == 0) return out;
  a.out = out[0].data_ptr();
  torch::Tensor ws = scratch(
      wr_ffn_workspace_bytes(0, a.dtype, a.hidden_dim, a.intermediate_dim, a.batch_size), dev);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = (size_t)ws.numel();
  check_status(wr_ffn_forward(&a, stream_of(dev)), "gated_ffn_forward");
  return out;
}

// gated_ffn_backward(dy, x, w_gate, w_up, w_down, g, u, a, need [4]) -> [dx, dw_gate,
// dw_up, dw_down], those not needed undefined.
std::vector<std::optional<torch::Tensor>> gated_ffn_backward(
    torch::Tensor dy, torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up,
    torch::Tensor w_down, torch::Tensor g, torch::Tensor u, torch::Tensor act,
    std::vector<bool> need) {
  check_ffn(x, w_gate, w_up, w_down);
  const torch::Device dev = x.device();
  check_operand(dy, "dy", x.scalar_type(), dev, x.sizes());
  const int64_t row = wr_ffn_saved_row((int)w_gate.size(0));
  check_operand(g, "g", torch::kFloat32, dev, {x.size(0), row});
  check_operand(u, "u", torch::kFloat32, dev, {x.size(0), row});
  check_operand(act, "a", x.scalar_type(), dev, {x.size(0), row});
  TORCH_CHECK(need.size() == 4, "need must hold 4 truth values, got ", need.size());
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  dy = aligned16(dy);
  x = aligned16(x);
  w_gate = aligned16(w_gate);
  w_up = aligned16(w_up);
  w_down = aligned16(w_down);
  g = aligned16(g);
  u = aligned16(u);
  act = aligned16(act);
  wr_ffn_args a = ffn_args(x, w_gate, w_up, w_down);
  const torch::Tensor* like[4] = {&x, &w_gate, &w_up, &w_down};
  void** slot[4] = {&a.dx, &a.dw_gate, &a.dw_up, &a.dw_down};
  std::vector<std::optional<torch::Tensor>> out(4);
  bool any = false;
  for (int i = 0; i < 4; ++i) {
    if (!need[i]) continue;
    out[i] = torch::empty_like(*like[i]);
    *slot[i] = out[i]->data_ptr();
    any = true;
  }
  if (!any) return out;
  a.dout = dy.data_ptr();
  a.saved_gate = g.data_ptr<float>();
  a.saved_up = u.data_ptr<float>();
  a.saved_act = act.data_ptr();
  torch::Tensor ws = scratch(
      wr_ffn_workspace_bytes(1, a.dtype, a.hidden_dim, a.intermediate_dim, a.batch_size), dev);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = (size_t)ws.numel();
  check_status(wr_ffn_backward(&a, stream_of(dev)), "gated_ffn_backward");
  return out;
}

// The differentiable form: y, with what the backward pass reads kept when a gradient is
// needed.  Differentiable once: the gradients of a backward pass that builds a graph
// raise when they are differentiated themselves.
class GatedFfn : public torch::autograd::Function<GatedFfn> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x,
                               const torch::Tensor& w_gate, const torch::Tensor& w_up,
                               const torch::Tensor& w_down) {
    std::vector<torch::Tensor> r = gated_ffn_forward(x, w_gate, w_up, w_down, true);
    ctx->save_for_backward({x, w_gate, w_up, w_down, r[1], r[2], r[3]});
    return r[0];
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const torch::autograd::variable_list s = ctx->get_saved_variables();
    std::vector<bool> need(4);
    for (int i = 0; i < 4; ++i) need[i] = ctx->needs_input_grad(i);
    torch::autograd::variable_list out(4);
    {
      const at::AutoGradMode off(false);
      const auto got = gated_ffn_backward(grads[0].contiguous(), s[0], s[1], s[2], s[3], s[4], s[5],
                                          s[6], need);
      for (int i = 0; i < 4; ++i)
        if (got[i].has_value()) out[i] = *got[i];
    }
    if (at::GradMode::is_enabled()) {
      auto once = std::make_shared<torch::autograd::DelayedError>(
          "gated_ffn is differentiable once: its gradients cannot be differentiated", 1);
      for (torch::Tensor& t : out) {
        if (!t.defined()) continue;
        t.set_requires_grad(true);
        t = (*once)({t})[0];
      }
    }
    return out;
  }
};

// Under graph capture, gradient accumulators of leaves that an eager graph keeps alive
// belong to that graph's stream.  A captured backward pass would wait for it, which
// torch does not survive: refused here.
void check_capture(const std::array<torch::Tensor, 4>& leaves, const torch::Device& dev) {
  const auto stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index());
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(stream.stream(), &status) != hipSuccess ||
      status == hipStreamCaptureStatusNone)
    return;
  for (const torch::Tensor& t : leaves) {
    if (!t.requires_grad() || !t.is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto home = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!home.has_value() || *home == stream.unwrap(),
                "gated_ffn is captured into a graph while an eager autograd graph of the same "
                "tensors is alive: drop its outputs before the capture");
  }
}

// gated_ffn(x [.., h], w_gate, w_up, w_down) -> y, differentiable where a gradient is asked for.
torch::Tensor gated_ffn(const torch::Tensor& x, const torch::Tensor& w_gate,
                        const torch::Tensor& w_up, const torch::Tensor& w_down) {
  TORCH_CHECK(x.dim() >= 1, "x must have at least one dimension");
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA (HIP) tensor");
  TORCH_CHECK(x.is_contiguous(), "x must be contiguous");
  const int64_t h = x.size(-1);
  const torch::Tensor rows =
      x.dim() == 2 ? x : x.reshape({h > 0 ? x.numel() / h : x.numel(), h});
  torch::Tensor y;
  const std::array<torch::Tensor, 4> leaves{x, w_gate, w_up, w_down};
  bool grad = false;
  for (const torch::Tensor& t : leaves) grad = grad || t.requires_grad();
  if (grad && at::GradMode::is_enabled()) {
    check_capture(leaves, x.device());
    y = GatedFfn::apply(rows, w_gate, w_up, w_down);
  } else {
    y = gated_ffn_forward(rows, w_gate, w_up, w_down, false)[0];
  }
  return x.dim() == 2 ? y : y.reshape(x.sizes());
}

// quantize_int8(x [rows, cols]) -> (codes int8, scales fp32 [rows]).
std::tuple<torch::Tensor, torch::Tensor> quantize_int8(torch::Tensor x) {
  check_tokens(x, "x");
  const int tag = float_tag(x, "x");
  TORCH_CHECK(x.size(1) <= WR_INT8_MAX_COLS, "x has an unsupported shape ", x.sizes());
  const torch::Device dev = x.device();
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  x = aligned16(x);
  torch::Tensor q = torch::empty_like(x, x.options().dtype(torch::kInt8));
  torch::Tensor s = torch::empty({x.size(0)}, x.options().dtype(torch::kFloat32));
  if (x.size(0) == 0) return {q, s};
  check_status(wr_quantize_int8(x.data_ptr(), tag, (int)x.size(0), (int)x.size(1),
                                q.data_ptr<int8_t>(), s.data_ptr<float>(), stream_of(dev)),
               "quantize_int8");
  return {q, s};
}

// int8_matmul(x int8 [M,K], x_scale [M], w int8 [N,K], w_scale [N], out_dtype) -> [M,N].
torch::Tensor int8_matmul(torch::Tensor x, torch::Tensor x_scale, torch::Tensor w,
                          torch::Tensor w_scale, py::object out_dtype) {
  check_tokens(x, "x");
  const torch::Device dev = x.device();
  TORCH_CHECK(w.dim() == 2, "w must have shape [out_features, in_features], got shape ", w.sizes());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  check_operand(x, "x", torch::kInt8, dev, {M, K});
  check_operand(x_scale, "x_scale", torch::kFloat32, dev, {M});
  check_operand(w, "w", torch::kInt8, dev, {N, K});
  check_operand(w_scale, "w_scale", torch::kFloat32, dev, {N});
  TORCH_CHECK(K <= WR_INT8_MAX_K && N >= 1 && N <= WR_FFN_MAX_DIM, "in_features must be in [1, ",
              WR_INT8_MAX_K, "] and out_features in [1, ", WR_FFN_MAX_DIM, "], got ", K, " and ", N);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  x = aligned16(x);
  w = aligned16(w);
  torch::Tensor out = torch::empty(
      {M, N}, torch::TensorOptions().dtype(torch::python::detail::py_object_to_dtype(out_dtype)).device(dev));
  wr_int8_args a{};
  a.out_dtype = float_tag(out, "out_dtype");
  if (M == 0) return out;
  a.x = x.data_ptr<int8_t>();
  a.x_scale = x_scale.data_ptr<float>();
  a.w = w.data_ptr<int8_t>();
  a.w_scale = w_scale.data_ptr<float>();
  a.out = out.data_ptr();
  a.rows = (int32_t)M;
  a.out_features = (int32_t)N;
  a.in_features = (int32_t)K;
  torch::Tensor ws = scratch(wr_int8_workspace_bytes(a.rows, a.out_features, a.in_features), dev);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = (size_t)ws.numel();
  check_status(wr_int8_matmul(&a, stream_of(dev)), "int8_matmul");
  return out;
}

// gated_ffn_int8(x [T,h], w_gate int8 [I,h], s_gate [I], w_up, s_up, w_down int8 [h,I],
// s_down [h]) -> [T,h] in x's dtype.
torch::Tensor gated_ffn_int8(torch::Tensor x, torch::Tensor w_gate, torch::Tensor s_gate,
                             torch::Tensor w_up, torch::Tensor s_up, torch::Tensor w_down,
                             torch::Tensor s_down) {
  check_tokens(x, "x");
  const int tag = float_tag(x, "x");
  const torch::Device dev = x.device();
  TORCH_CHECK(w_gate.dim() == 2, "w_gate must have shape [intermediate_dim, hidden_dim], got shape ",
              w_gate.sizes());
  const int64_t h = x.size(1), I = w_gate.size(0);
  check_dims(h, I, WR_INT8_MAX_K);
  check_operand(w_gate, "w_gate", torch::kInt8, dev, {I, h});
  check_operand(s_gate, "s_gate", torch::kFloat32, dev, {I});
  check_operand(w_up, "w_up", torch::kInt8, dev, {I, h});
  check_operand(s_up, "s_up", torch::kFloat32, dev, {I});
  check_operand(w_down, "w_down", torch::kInt8, dev, {h, I});
  check_operand(s_down, "s_down", torch::kFloat32, dev, {h});
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dev);
  x = aligned16(x);
  w_gate = aligned16(w_gate);
  w_up = aligned16(w_up);
  w_down = aligned16(w_down);
  torch::Tensor out = torch::empty_like(x);
  if (x.size(0) == 0) return out;
  wr_ffn_int8_args a{};
  a.x = x.data_ptr();
  a.w_gate = w_gate.data_ptr<int8_t>();
  a.s_gate = s_gate.data_ptr<float>();
  a.w_up = w_up.data_ptr<int8_t>();
  a.s_up = s_up.data_ptr<float>();
  a.w_down = w_down.data_ptr<int8_t>();
  a.s_down = s_down.data_ptr<float>();
  a.out = out.data_ptr();
  a.dtype = tag;
  a.batch_size = (int32_t)x.size(0);
  a.hidden_dim = (int32_t)h;
  a.intermediate_dim = (int32_t)I;
  torch::Tensor ws = scratch(
      wr_ffn_int8_workspace_bytes(a.hidden_dim, a.intermediate_dim, a.batch_size), dev);
  a.workspace = ws.data_ptr();
  a.workspace_bytes = (size_t)ws.numel();
  check_status(wr_ffn_int8(&a, stream_of(dev)), "gated_ffn_int8");
  return out;
}

void set_handoff_check(bool enabled) { g_check_handoff.store(enabled); }
bool handoff_check() { return g_check_handoff.load(); }

py::dict layout(int num_experts, int hidden_dim, int intermediate_dim, int elem_bytes) {
  wr_offsets o;
  check_status(wr_layout(num_experts, hidden_dim, intermediate_dim, elem_bytes, &o), "layout");
  py::dict d;
  d["gate_proj_offset"] = o.gate_proj_offset;
  d["up_proj_offset"] = o.up_proj_offset;
  d["down_proj_offset"] = o.down_proj_offset;
  d["expert_stride"] = o.expert_stride;
  return d;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  const auto opt = py::arg("topk_ids") = py::none();
  const auto optw = py::arg("topk_weights") = py::none();
  m.def("naive_moe_forward", &naive_moe_forward,
        "Naive multi-kernel MoE forward (host top-K; fp32, fp16, bf16, fp8 e4m3 or mxfp4 "
        "weights)",
        py::arg("hidden"),
        py::arg("gate_w"), py::arg("weight_buf"), py::arg("num_experts"), py::arg("hidden_dim"),
        py::arg("intermediate_dim"), py::arg("top_k"), py::arg("renormalize") = false, opt, optw);
  m.def("fused_moe_forward", &fused_moe_forward,
        "Fused decode MoE forward for one token (fp32, fp16, bf16, fp8 e4m3 or mxfp4 weights)",
        py::arg("hidden"),
        py::arg("gate_w"), py::arg("weight_buf"), py::arg("num_experts"), py::arg("hidden_dim"),
        py::arg("intermediate_dim"), py::arg("top_k"), py::arg("renormalize") = false, opt, optw);
  m.def("batched_fused_moe_forward", &batched_fused_moe_forward,
        "Batched fused MoE forward for B tokens (fp32, fp16, bf16, fp8 e4m3 or mxfp4 weights)",
        py::arg("hidden_batch"),
        py::arg("gate_w"), py::arg("weight_buf"), py::arg("num_experts"), py::arg("hidden_dim"),
        py::arg("intermediate_dim"), py::arg("top_k"), py::arg("renormalize") = false, opt, optw);
  m.def("gate_topk", &gate_topk, "Router logits, softmax and top-K", py::arg("hidden"),
        py::arg("gate_w"), py::arg("num_experts"), py::arg("hidden_dim"), py::arg("top_k"),
        py::arg("renormalize") = false);
  m.def("gated_ffn", &gated_ffn, "Dense gated FFN (fp32, fp16 or bf16), differentiable",
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"));
  m.def("gated_ffn_forward", &gated_ffn_forward,
        "Dense gated FFN (fp32, fp16 or bf16); with keep also what its backward pass reads",
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"),
        py::arg("keep") = false);
  m.def("gated_ffn_backward", &gated_ffn_backward, "Gradients of gated_ffn_forward", py::arg("dy"),
        py::arg("x"), py::arg("w_gate"), py::arg("w_up"), py::arg("w_down"), py::arg("g"),
        py::arg("u"), py::arg("a"), py::arg("need"));
  m.def("quantize_int8", &quantize_int8, "int8 codes and fp32 scales of rows", py::arg("x"));
  m.def("int8_matmul", &int8_matmul, "Product of int8 codes, scaled per row and column",
        py::arg("x"), py::arg("x_scale"), py::arg("w"), py::arg("w_scale"), py::arg("out_dtype"));
  m.def("gated_ffn_int8", &gated_ffn_int8, "Dense gated FFN on int8 weights", py::arg("x"),
        py::arg("w_gate"), py::arg("s_gate"), py::arg("w_up"), py::arg("s_up"), py::arg("w_down"),
        py::arg("s_down"));
  m.def("set_handoff_check", &set_handoff_check,
        "Make fused_moe_forward synchronise and raise if its hand-off wait expired",
        py::arg("enabled"));
  m.def("handoff_check", &handoff_check, "Whether fused_moe_forward checks its hand-off");
  m.def("layout", &layout, "Packed expert layout offsets in bytes", py::arg("num_experts"),
        py::arg("hidden_dim"), py::arg("intermediate_dim"), py::arg("elem_bytes"));
  m.def("total_weight_bytes", &wr_total_weight_bytes, "Packed layout size in bytes (-1 if invalid)",
        py::arg("num_experts"), py::arg("hidden_dim"), py::arg("intermediate_dim"),
        py::arg("elem_bytes"));
  m.def("weight_bytes", &wr_weight_bytes,
        "Packed layout size in bytes for a wr_dtype tag (-1 if invalid)", py::arg("num_experts"),
        py::arg("hidden_dim"), py::arg("intermediate_dim"), py::arg("weight_dtype"));
}
