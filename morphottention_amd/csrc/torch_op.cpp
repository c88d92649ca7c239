// torch.ops.morphottention.{forward, backward}: the reference op schemas
// (packages/morphottention/csrc/cuda/binder.cpp:6-15) registered on the CUDA
// dispatch key, which PyTorch-ROCm uses for HIP tensors, plus two ops used by
// the autograd Function that carry the forward projection to the backward and
// take the variant bits (masked diagonal, cube projection).
//
// Checks and messages follow packages/morphottention/csrc/cuda/attention/attention.cpp:9-38,64-91.
// Unlike the reference this layer sets a device guard (the reference launches
// on whatever device is current) and honours `causal`.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <optional>
#include <utility>
#include <vector>

#include "../../include/morphottention.h"

namespace {

void check(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kHalf, name, " must be float16");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

struct Shape {
  int64_t B, N, D, H, M;
};

Shape check_inputs(const at::Tensor& X, const at::Tensor& W_phi, const at::Tensor& gate_q, const at::Tensor& gate_k,
                   const at::Tensor& W_V, int64_t H, int64_t cube_m) {
  check(X, "X");
  check(W_phi, "W_phi");
  check(gate_q, "gate_q");
  check(gate_k, "gate_k");
  check(W_V, "W_V");
  TORCH_CHECK(X.dim() == 3, "X must be [B, N, D]");
  const int64_t B = X.size(0), N = X.size(1), D = X.size(2);
  TORCH_CHECK(H > 0 && D % H == 0, "D must be divisible by H");
  const int64_t head_dim_v = D / H;
  TORCH_CHECK(W_phi.dim() == 2 && W_phi.size(0) == D && W_phi.size(1) == H * cube_m, "W_phi must be [D, H*cube_m]");
  TORCH_CHECK(W_V.dim() == 2 && W_V.size(0) == D && W_V.size(1) == H * head_dim_v, "W_V must be [D, H*head_dim_v]");
  TORCH_CHECK(gate_q.dim() == 2 && gate_q.size(0) == H && gate_q.size(1) == cube_m, "gate_q must be [H, cube_m]");
  TORCH_CHECK(gate_k.dim() == 2 && gate_k.size(0) == H && gate_k.size(1) == cube_m, "gate_k must be [H, cube_m]");
  for (const at::Tensor* t : {&W_phi, &gate_q, &gate_k, &W_V})
    TORCH_CHECK(t->device() == X.device(), "all tensors must be on the same device as X");
  return {B, N, D, H, cube_m};
}

morpho_stream_t current_stream(const at::Tensor& X) {
  return reinterpret_cast<morpho_stream_t>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(X.device().index()).stream());
}

// The ABI's mode word: bit 0 causal, the other bits the variant
// (MORPHO_MODE_MASK_DIAG, MORPHO_MODE_PROJ_*, MORPHO_MODE_DETERMINISTIC), which
// only the *_train ops take.
int mode_of(bool causal, int64_t variant) {
  TORCH_CHECK((variant & ~(int64_t)(MORPHO_MODE_MASK_DIAG | MORPHO_MODE_PROJ_HARDTANH01 | MORPHO_MODE_PROJ_IDENTITY |
                                    MORPHO_MODE_DETERMINISTIC)) == 0 &&
                  (variant & (MORPHO_MODE_PROJ_HARDTANH01 | MORPHO_MODE_PROJ_IDENTITY)) !=
                      (MORPHO_MODE_PROJ_HARDTANH01 | MORPHO_MODE_PROJ_IDENTITY),
              "variant must combine MORPHO_MODE_MASK_DIAG (2) and MORPHO_MODE_DETERMINISTIC (32) with at most one "
              "of MORPHO_MODE_PROJ_HARDTANH01 (4) and MORPHO_MODE_PROJ_IDENTITY (8), got ", variant);
  return (causal ? MORPHO_MODE_CAUSAL : 0) | (int)variant;
}

void raise_on(int status, const char* what) {
  TORCH_CHECK(status == MORPHO_OK, "morphottention ", what, " failed (", morpho_status_string(status),
              "): ", morpho_last_error());
}

// A workspace size of 0 means the sizes fail the ABI's validation; report its
// reason (empty dimension, unsupported cube_m or head width, problem too
// large). morpho_forward validates the sizes before it looks at any pointer
// or touches the device, so a call without buffers only returns that error.
void raise_size_error(int64_t B, int64_t N, int64_t D, int64_t H, int64_t M, int mode, const char* what) {
  const int st = morpho_forward(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, B, N, D, H, M, 1.0f,
                                mode, nullptr, 0, nullptr);
  raise_on(st == MORPHO_OK ? MORPHO_ERR_INVALID_ARGUMENT : st, what);
}

std::vector<at::Tensor> forward_impl(const at::Tensor& X, const at::Tensor& W_phi, const at::Tensor& gate_q,
                                     const at::Tensor& gate_k, const at::Tensor& W_V, int64_t H, int64_t cube_m,
                                     double scale, bool causal, int64_t variant, bool keep_workspace) {
  const int mode = mode_of(causal, variant);
  const Shape s = check_inputs(X, W_phi, gate_q, gate_k, W_V, H, cube_m);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(X.device());
  auto out = at::empty_like(X);
  auto lse = at::empty({s.B * H, s.N}, X.options().dtype(at::kFloat));
  const size_t ws_bytes = morpho_forward_workspace_size(s.B, s.N, s.D, s.H, s.M);
  if (ws_bytes == 0) raise_size_error(s.B, s.N, s.D, s.H, s.M, mode, "forward");
  auto ws = at::empty({(int64_t)ws_bytes}, X.options().dtype(at::kByte));
  raise_on(morpho_forward(X.data_ptr(), W_phi.data_ptr(), gate_q.data_ptr(), gate_k.data_ptr(), W_V.data_ptr(),
                          out.data_ptr(), lse.data_ptr<float>(), s.B, s.N, s.D, s.H, s.M, (float)scale, mode,
                          ws.data_ptr(), ws_bytes, current_stream(X)),
           "forward");
  if (keep_workspace) return {out, lse, ws};
  return {out, lse};
}

std::vector<at::Tensor> backward_impl(const at::Tensor& grad_out, const at::Tensor& X, const at::Tensor& W_phi,
                                      const at::Tensor& gate_q, const at::Tensor& gate_k, const at::Tensor& W_V,
                                      const at::Tensor& out, const at::Tensor& lse, const at::Tensor* fwd_ws,
                                      int64_t H, int64_t cube_m, double scale, bool causal, int64_t variant) {
  const int mode = mode_of(causal, variant);
  check(grad_out, "grad_out");
  const Shape s = check_inputs(X, W_phi, gate_q, gate_k, W_V, H, cube_m);
  check(out, "out");
  TORCH_CHECK(lse.is_cuda(), "lse must be a CUDA tensor");
  TORCH_CHECK(lse.scalar_type() == at::kFloat, "lse must be float32");
  TORCH_CHECK(lse.is_contiguous(), "lse must be contiguous");
  TORCH_CHECK(grad_out.sizes() == X.sizes(), "grad_out must match X shape [B, N, D]");
  TORCH_CHECK(out.sizes() == X.sizes(), "out must match X shape [B, N, D]");
  TORCH_CHECK(lse.dim() == 2 && lse.size(0) == s.B * H && lse.size(1) == s.N, "lse must be [B*H, N]");
  TORCH_CHECK(grad_out.device() == X.device() && out.device() == X.device() && lse.device() == X.device() &&
                  (!fwd_ws || fwd_ws->device() == X.device()),
              "all tensors must be on the same device as X");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(X.device());
  const void* fwd_ptr = nullptr;
  if (fwd_ws) {
    const size_t need = morpho_forward_workspace_size(s.B, s.N, s.D, s.H, s.M);
    TORCH_CHECK(fwd_ws->is_cuda() && fwd_ws->scalar_type() == at::kByte && fwd_ws->is_contiguous() &&
                    (size_t)fwd_ws->numel() >= need,
                "workspace must be the uint8 CUDA tensor returned by forward_train for these sizes");
    fwd_ptr = fwd_ws->data_ptr();
  }
  auto dX = at::empty_like(X);
  auto dW_phi = at::empty_like(W_phi);
  auto d_gate_q = at::empty_like(gate_q);
  auto d_gate_k = at::empty_like(gate_k);
  auto dW_V = at::empty_like(W_V);
  const size_t ws_bytes = morpho_backward_workspace_size_for_mode(s.B, s.N, s.D, s.H, s.M, fwd_ptr != nullptr, mode);
  if (ws_bytes == 0) raise_size_error(s.B, s.N, s.D, s.H, s.M, mode, "backward");
  auto ws = at::empty({(int64_t)ws_bytes}, X.options().dtype(at::kByte));
  raise_on(morpho_backward(grad_out.data_ptr(), X.data_ptr(), W_phi.data_ptr(), gate_q.data_ptr(), gate_k.data_ptr(),
                           W_V.data_ptr(), out.data_ptr(), lse.data_ptr<float>(), dX.data_ptr(), dW_phi.data_ptr(),
                           d_gate_q.data_ptr(), d_gate_k.data_ptr(), dW_V.data_ptr(), s.B, s.N, s.D, s.H, s.M,
                           (float)scale, mode, fwd_ptr, ws.data_ptr(), ws_bytes, current_stream(X)),
           "backward");
  return {dX, dW_phi, d_gate_q, d_gate_k, dW_V};
}

std::vector<at::Tensor> op_forward(const at::Tensor& X, const at::Tensor& W_phi, const at::Tensor& gate_q,
                                   const at::Tensor& gate_k, const at::Tensor& W_V, int64_t H, int64_t cube_m,
                                   double scale, bool causal) {
  return forward_impl(X, W_phi, gate_q, gate_k, W_V, H, cube_m, scale, causal, 0, false);
}

std::vector<at::Tensor> op_forward_train(const at::Tensor& X, const at::Tensor& W_phi, const at::Tensor& gate_q,
                                         const at::Tensor& gate_k, const at::Tensor& W_V, int64_t H, int64_t cube_m,
                                         double scale, bool causal, int64_t variant) {
  return forward_impl(X, W_phi, gate_q, gate_k, W_V, H, cube_m, scale, causal, variant, true);
}

std::vector<at::Tensor> op_backward(const at::Tensor& grad_out, const at::Tensor& X, const at::Tensor& W_phi,
                                    const at::Tensor& gate_q, const at::Tensor& gate_k, const at::Tensor& W_V,
                                    const at::Tensor& out, const at::Tensor& lse, int64_t H, int64_t cube_m,
                                    double scale, bool causal) {
  return backward_impl(grad_out, X, W_phi, gate_q, gate_k, W_V, out, lse, nullptr, H, cube_m, scale, causal, 0);
}

std::vector<at::Tensor> op_backward_train(const at::Tensor& grad_out, const at::Tensor& X, const at::Tensor& W_phi,
                                          const at::Tensor& gate_q, const at::Tensor& gate_k, const at::Tensor& W_V,
                                          const at::Tensor& out, const at::Tensor& lse, const at::Tensor& workspace,
                                          int64_t H, int64_t cube_m, double scale, bool causal, int64_t variant) {
  return backward_impl(grad_out, X, W_phi, gate_q, gate_k, W_V, out, lse, &workspace, H, cube_m, scale, causal,
                       variant);
}

// ---- soft tropical aggregation (no reference op: the reference defines the
// accumulators of morfology/soft_morph.cuh but never wires them)
void check_tau(const at::Tensor& tau, const at::Tensor& X) {
  TORCH_CHECK(tau.is_cuda() && tau.device() == X.device(), "tau must be a CUDA tensor on the device of X");
  TORCH_CHECK(tau.scalar_type() == at::kFloat && tau.numel() == 1 && tau.is_contiguous(),
              "tau must be one contiguous float32 element");
}

// The soft ops also accept MORPHO_MODE_SOFT_EXACT (16) in `variant`.
int soft_mode_of(bool causal, int64_t variant) {
  TORCH_CHECK((variant & MORPHO_MODE_DETERMINISTIC) == 0,
              "MORPHO_MODE_DETERMINISTIC (32) applies to the softmax backward only");
  return mode_of(causal, variant & ~(int64_t)MORPHO_MODE_SOFT_EXACT) | (int)(variant & MORPHO_MODE_SOFT_EXACT);
}

int sgn_of(int64_t sgn) {
  TORCH_CHECK(sgn == 1 || sgn == -1, "sgn must be +1 (dilation) or -1 (erosion), got ", sgn);
  return (int)sgn;
}

std::vector<at::Tensor> op_soft_forward(const at::Tensor& X, const at::Tensor& W_phi, const at::Tensor& gate_q,
                                        const at::Tensor& gate_k, const at::Tensor& W_V, const at::Tensor& tau,
                                        int64_t H, int64_t cube_m, double scale, bool causal, int64_t sgn,
                                        int64_t variant) {
  const int mode = soft_mode_of(causal, variant);
  const int sg = sgn_of(sgn);
  const Shape s = check_inputs(X, W_phi, gate_q, gate_k, W_V, H, cube_m);
  check_tau(tau, X);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(X.device());
  auto out = at::empty_like(X);
  auto zb = at::empty({s.B * H, s.N, s.D / H}, X.options().dtype(at::kFloat));
  const size_t ws_bytes = morpho_soft_forward_workspace_size(s.B, s.N, s.D, s.H, s.M);
  if (ws_bytes == 0) raise_size_error(s.B, s.N, s.D, s.H, s.M, mode & ~MORPHO_MODE_SOFT_EXACT, "soft_forward");
  auto ws = at::empty({(int64_t)ws_bytes}, X.options().dtype(at::kByte));
  raise_on(morpho_soft_forward(X.data_ptr(), W_phi.data_ptr(), gate_q.data_ptr(), gate_k.data_ptr(), W_V.data_ptr(),
                               tau.data_ptr<float>(), out.data_ptr(), zb.data_ptr<float>(), s.B, s.N, s.D, s.H, s.M,
                               (float)scale, mode, sg, ws.data_ptr(), ws_bytes, current_stream(X)),
           "soft_forward");
  return {out, zb, ws};
}

std::vector<at::Tensor> op_soft_backward(const at::Tensor& grad_out, const at::Tensor& X, const at::Tensor& W_phi,
                                         const at::Tensor& gate_q, const at::Tensor& gate_k, const at::Tensor& W_V,
                                         const at::Tensor& tau, const at::Tensor& zb, const at::Tensor& workspace,
                                         int64_t H, int64_t cube_m, double scale, bool causal, int64_t sgn,
                                         int64_t variant) {
  const int mode = soft_mode_of(causal, variant);
  const int sg = sgn_of(sgn);
  check(grad_out, "grad_out");
  const Shape s = check_inputs(X, W_phi, gate_q, gate_k, W_V, H, cube_m);
  check_tau(tau, X);
  TORCH_CHECK(grad_out.sizes() == X.sizes(), "grad_out must match X shape [B, N, D]");
  TORCH_CHECK(zb.is_cuda() && zb.scalar_type() == at::kFloat && zb.is_contiguous() && zb.dim() == 3 &&
                  zb.size(0) == s.B * H && zb.size(1) == s.N && zb.size(2) == s.D / H,
              "zb must be the float32 [B*H, N, D/H] tensor of soft_forward");
  const size_t need = morpho_soft_forward_workspace_size(s.B, s.N, s.D, s.H, s.M);
  TORCH_CHECK(workspace.is_cuda() && workspace.scalar_type() == at::kByte && workspace.is_contiguous() &&
                  (size_t)workspace.numel() >= need,
              "workspace must be the uint8 CUDA tensor returned by soft_forward for these sizes");
  TORCH_CHECK(grad_out.device() == X.device() && zb.device() == X.device() && workspace.device() == X.device(),
              "all tensors must be on the same device as X");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(X.device());
  auto dX = at::empty_like(X);
  auto dW_phi = at::empty_like(W_phi);
  auto d_gate_q = at::empty_like(gate_q);
  auto d_gate_k = at::empty_like(gate_k);
  auto dW_V = at::empty_like(W_V);
  auto dtau = at::empty_like(tau);
  const size_t ws_bytes = morpho_soft_backward_workspace_size(s.B, s.N, s.D, s.H, s.M, 1);
  auto ws = at::empty({(int64_t)ws_bytes}, X.options().dtype(at::kByte));
  raise_on(morpho_soft_backward(grad_out.data_ptr(), X.data_ptr(), W_phi.data_ptr(), gate_q.data_ptr(),
                                gate_k.data_ptr(), W_V.data_ptr(), tau.data_ptr<float>(), zb.data_ptr<float>(),
                                dX.data_ptr(), dW_phi.data_ptr(), d_gate_q.data_ptr(), d_gate_k.data_ptr(),
                                dW_V.data_ptr(), dtau.data_ptr<float>(), s.B, s.N, s.D, s.H, s.M, (float)scale, mode,
                                sg, workspace.data_ptr(), ws.data_ptr(), ws_bytes, current_stream(X)),
           "soft_backward");
  return {dX, dW_phi, d_gate_q, d_gate_k, dW_V, dtau};
}

// ---- paged cache (no reference op: the reference computes whole sequences only)
void check_ints(const at::Tensor& t, const char* name, const at::Tensor& codes) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  TORCH_CHECK(t.device() == codes.device(), "all tensors must be on the same device as codes");
}

// The pool of one layer, or of several (codes then have 5 dimensions).
morpho_cache check_pool(const at::Tensor& codes, const at::Tensor& values, bool layers) {
  check(codes, "codes");
  check(values, "values");
  TORCH_CHECK(values.device() == codes.device(), "all tensors must be on the same device as codes");
  const int64_t k = codes.dim() - 4;
  if (layers) {
    TORCH_CHECK(k == 0 || k == 1, "codes must be [pages, H, page_size, cube_m] or [layers, pages, H, page_size, cube_m]");
  } else {
    TORCH_CHECK(k == 0, "codes must be [pages, H, page_size, cube_m]");
  }
  const int64_t L = k ? codes.size(0) : 1, pages = codes.size(k), H = codes.size(k + 1), P = codes.size(k + 2),
                M = codes.size(k + 3);
  TORCH_CHECK(values.dim() == k + 5 && (k == 0 || values.size(0) == L) && values.size(k) == pages &&
                  values.size(k + 1) == H && P % 8 == 0 && values.size(k + 2) == P / 8 && values.size(k + 4) == 8,
              "values must be [pages, H, page_size / 8, head_dim_v, 8] (with the layers of codes before)");
  return morpho_cache{codes.data_ptr(), values.data_ptr(), L, pages, H, M, values.size(k + 3), P};
}

struct CacheCall {
  const int32_t *table, *lens, *new_lens;
  int64_t seq_pages;
};
CacheCall check_cache_call(const at::Tensor& codes, const at::Tensor& table, const at::Tensor& lens,
                           const std::optional<at::Tensor>& new_lens, int64_t B) {
  check_ints(table, "table", codes);
  check_ints(lens, "lens", codes);
  TORCH_CHECK(table.dim() == 2 && table.size(0) == B, "table must be [B, seq_pages]");
  TORCH_CHECK(lens.dim() == 1 && lens.size(0) == B, "lens must be [B]");
  if (new_lens) {
    check_ints(*new_lens, "new_lens", codes);
    TORCH_CHECK(new_lens->dim() == 1 && new_lens->size(0) == B, "new_lens must be [B]");
  }
  return {table.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), new_lens ? new_lens->data_ptr<int32_t>() : nullptr,
          table.size(1)};
}

at::Tensor op_cache_append(const at::Tensor& X, const at::Tensor& weights, const at::Tensor& codes,
                           const at::Tensor& values, const at::Tensor& table, const at::Tensor& lens,
                           const std::optional<at::Tensor>& new_lens, int64_t variant) {
  const int mode = mode_of(false, variant);
  const morpho_cache c = check_pool(codes, values, false);
  check(X, "X");
  check(weights, "weights");
  TORCH_CHECK(X.dim() == 3, "X must be [B, n, D]");
  const int64_t B = X.size(0), n = X.size(1), D = c.H * c.head_dim_v;
  TORCH_CHECK(X.size(2) == D, "X must be [B, n, D] with D = H*head_dim_v of the cache (", D, ")");
  TORCH_CHECK(weights.dim() == 2 && weights.size(0) == c.H * c.cube_m + D && weights.size(1) == D,
              "weights must be [H*cube_m + D, D]");
  TORCH_CHECK(X.device() == codes.device() && weights.device() == codes.device(),
              "all tensors must be on the same device as codes");
  const CacheCall k = check_cache_call(codes, table, lens, new_lens, B);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
  auto phi = at::empty({B, n, c.H, c.cube_m}, X.options());
  raise_on(morpho_cache_append(X.data_ptr(), weights.data_ptr(), &c, k.table, k.lens, k.new_lens, phi.data_ptr(), B, n,
                               k.seq_pages, mode, current_stream(codes)),
           "cache_append");
  return phi;
}

struct AttentionCall {
  morpho_cache cache;
  CacheCall call;
  int64_t B, n;
};
AttentionCall check_attention_call(const at::Tensor& phi, const at::Tensor& gate_q, const at::Tensor& gate_k,
                                   const at::Tensor& codes, const at::Tensor& values, const at::Tensor& table,
                                   const at::Tensor& lens, const std::optional<at::Tensor>& new_lens,
                                   const std::optional<at::Tensor>& tree) {
  const morpho_cache c = check_pool(codes, values, false);
  check(phi, "phi");
  check(gate_q, "gate_q");
  check(gate_k, "gate_k");
  TORCH_CHECK(phi.dim() == 4 && phi.size(2) == c.H && phi.size(3) == c.cube_m,
              "phi must be [B, n, H, cube_m] with H and cube_m of the cache");
  const int64_t B = phi.size(0), n = phi.size(1);
  TORCH_CHECK(gate_q.dim() == 2 && gate_q.size(0) == c.H && gate_q.size(1) == c.cube_m, "gate_q must be [H, cube_m]");
  TORCH_CHECK(gate_k.dim() == 2 && gate_k.size(0) == c.H && gate_k.size(1) == c.cube_m, "gate_k must be [H, cube_m]");
  TORCH_CHECK(phi.device() == codes.device() && gate_q.device() == codes.device() && gate_k.device() == codes.device(),
              "all tensors must be on the same device as codes");
  const CacheCall k = check_cache_call(codes, table, lens, new_lens, B);
  if (tree) {
    TORCH_CHECK(tree->is_cuda() && tree->scalar_type() == at::kLong && tree->is_contiguous() && tree->dim() == 2 &&
                    tree->size(0) == B && tree->size(1) == n && tree->device() == codes.device(),
                "tree must be a contiguous int64 [B, n] CUDA tensor on the device of codes");
  }
  return {c, k, B, n};
}

std::vector<at::Tensor> op_cache_attention(const at::Tensor& phi, const at::Tensor& gate_q, const at::Tensor& gate_k,
                                           const at::Tensor& codes, const at::Tensor& values, const at::Tensor& table,
                                           const at::Tensor& lens, const std::optional<at::Tensor>& new_lens,
                                           const std::optional<at::Tensor>& tree, double scale, bool causal,
                                           int64_t variant, int64_t max_len) {
  const int mode = mode_of(causal, variant);
  const AttentionCall call = check_attention_call(phi, gate_q, gate_k, codes, values, table, lens, new_lens, tree);
  const morpho_cache& c = call.cache;
  const CacheCall& k = call.call;
  const int64_t B = call.B, n = call.n;
  TORCH_CHECK(max_len >= 0, "max_len must not be negative (0: the table's length), got ", max_len);
  if (max_len == 0) max_len = k.seq_pages * c.page_size;
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
  auto out = at::empty({B, n, c.H * c.head_dim_v}, phi.options());
  auto lse = at::empty({B * c.H, n}, phi.options().dtype(at::kFloat));
  const size_t ws_bytes = morpho_cache_attention_workspace_size(&c, B, n, k.seq_pages, max_len);
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, phi.options().dtype(at::kByte));
  raise_on(morpho_cache_attention(phi.data_ptr(), gate_q.data_ptr(), gate_k.data_ptr(), &c, k.table, k.lens,
                                  k.new_lens, tree ? tree->data_ptr<int64_t>() : nullptr, out.data_ptr(),
                                  lse.data_ptr<float>(), B, n, k.seq_pages, max_len, (float)scale, mode,
                                  ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, current_stream(codes)),
           "cache_attention");
  return {out, lse};
}

void op_cache_copy_pages(const at::Tensor& codes, const at::Tensor& values, const at::Tensor& src,
                         const at::Tensor& dst) {
  const morpho_cache c = check_pool(codes, values, true);
  check_ints(src, "src", codes);
  check_ints(dst, "dst", codes);
  TORCH_CHECK(src.dim() == 1 && dst.dim() == 1 && src.size(0) == dst.size(0), "src and dst must be [pairs]");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
  raise_on(morpho_cache_copy_pages(&c, src.data_ptr<int32_t>(), dst.data_ptr<int32_t>(), src.size(0),
                                   current_stream(codes)),
           "cache_copy_pages");
}

void op_cache_compact(const at::Tensor& codes, const at::Tensor& values, const at::Tensor& table,
                      const at::Tensor& lens, const at::Tensor& keep, const std::optional<at::Tensor>& keep_lens) {
  const morpho_cache c = check_pool(codes, values, true);
  check_ints(keep, "keep", codes);
  TORCH_CHECK(keep.dim() == 2, "keep must be [B, kept]");
  const int64_t B = keep.size(0);
  if (keep_lens) {
    check_ints(*keep_lens, "keep_lens", codes);
    TORCH_CHECK(keep_lens->dim() == 1 && keep_lens->size(0) == B, "keep_lens must be [B]");
  }
  const CacheCall k = check_cache_call(codes, table, lens, std::nullopt, B);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
  raise_on(morpho_cache_compact(&c, k.table, k.lens, keep.data_ptr<int32_t>(),
                                keep_lens ? keep_lens->data_ptr<int32_t>() : nullptr, B, keep.size(1), k.seq_pages,
                                current_stream(codes)),
           "cache_compact");
}

// ---- a decoding loop on the device (no reference op)
std::vector<at::Tensor> op_cache_shared_attention(const at::Tensor& phi, const at::Tensor& gate_q,
                                                  const at::Tensor& gate_k, const at::Tensor& codes,
                                                  const at::Tensor& values, const at::Tensor& table,
                                                  const at::Tensor& lens, const std::optional<at::Tensor>& new_lens,
                                                  const std::optional<at::Tensor>& tree, const at::Tensor& members,
                                                  const at::Tensor& starts, const at::Tensor& group,
                                                  const at::Tensor& pages, int64_t max_prefix, int64_t max_rest,
                                                  double scale, bool causal, int64_t variant) {
  const int mode = mode_of(causal, variant);
  const AttentionCall k = check_attention_call(phi, gate_q, gate_k, codes, values, table, lens, new_lens, tree);
  for (const auto& [t, name] : {std::pair<const at::Tensor&, const char*>(members, "members"),
                                {starts, "starts"}, {group, "group"}, {pages, "pages"}}) {
    check_ints(t, name, codes);
    TORCH_CHECK(t.dim() == 1, name, " must have one dimension");
  }
  TORCH_CHECK(group.size(0) == k.B, "group must be [B]");
  TORCH_CHECK(pages.size(0) > 0 && starts.size(0) == pages.size(0) + 1, "starts must be [groups + 1], pages [groups]");
  const int64_t cap = k.call.seq_pages * k.cache.page_size;
  TORCH_CHECK(max_prefix >= 0 && max_rest >= 0, "max_prefix and max_rest must not be negative (0: the table's length)");
  const morpho_shared_prefix shared{members.data_ptr<int32_t>(), starts.data_ptr<int32_t>(),
                                    group.data_ptr<int32_t>(),   pages.data_ptr<int32_t>(),
                                    members.size(0),             pages.size(0),
                                    max_prefix ? max_prefix : cap, max_rest ? max_rest : cap};
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(codes.device());
  auto out = at::empty({k.B, k.n, k.cache.H * k.cache.head_dim_v}, phi.options());
  auto lse = at::empty({k.B * k.cache.H, k.n}, phi.options().dtype(at::kFloat));
  const size_t ws_bytes = morpho_cache_shared_attention_workspace_size(
      &k.cache, k.B, k.n, k.call.seq_pages, shared.members_count, shared.groups, shared.max_prefix, shared.max_rest);
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, phi.options().dtype(at::kByte));
  raise_on(morpho_cache_shared_attention(phi.data_ptr(), gate_q.data_ptr(), gate_k.data_ptr(), &k.cache, k.call.table,
                                         k.call.lens, k.call.new_lens, tree ? tree->data_ptr<int64_t>() : nullptr,
                                         &shared, out.data_ptr(), lse.data_ptr<float>(), k.B, k.n, k.call.seq_pages,
                                         (float)scale, mode, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes,
                                         current_stream(codes)),
           "cache_shared_attention");
  return {out, lse};
}

std::vector<at::Tensor> op_cache_plan(const at::Tensor& table, const at::Tensor& held, const at::Tensor& lens,
                                      const at::Tensor& free_pages, const at::Tensor& free_count, int64_t n,
                                      const std::optional<at::Tensor>& new_lens, int64_t page_size) {
  check_ints(table, "table", table);
  check_ints(held, "held", table);
  check_ints(lens, "lens", table);
  check_ints(free_pages, "free_pages", table);
  check_ints(free_count, "free_count", table);
  TORCH_CHECK(table.dim() == 2, "table must be [B, seq_pages]");
  const int64_t B = table.size(0);
  TORCH_CHECK(held.dim() == 1 && held.size(0) == B, "held must be [B]");
  TORCH_CHECK(lens.dim() == 1 && lens.size(0) == B, "lens must be [B]");
  TORCH_CHECK(free_pages.dim() == 1, "free_pages must have one dimension");
  TORCH_CHECK(free_count.numel() == 1, "free_count must be one number");
  if (new_lens) {
    check_ints(*new_lens, "new_lens", table);
    TORCH_CHECK(new_lens->dim() == 1 && new_lens->size(0) == B, "new_lens must be [B]");
  }
  TORCH_CHECK(n > 0 && n <= (1 << 22), "n must be 1 to 2^22, got ", n);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(table.device());
  auto granted = at::empty({B}, table.options());
  auto slots = at::empty({B, n}, table.options().dtype(at::kLong));
  const size_t ws_bytes = morpho_cache_plan_workspace_size(B, n);
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, table.options().dtype(at::kByte));
  raise_on(morpho_cache_plan(table.data_ptr<int32_t>(), held.data_ptr<int32_t>(), lens.data_ptr<int32_t>(),
                             new_lens ? new_lens->data_ptr<int32_t>() : nullptr, free_pages.data_ptr<int32_t>(),
                             free_count.data_ptr<int32_t>(), free_pages.size(0), granted.data_ptr<int32_t>(),
                             slots.data_ptr<int64_t>(), B, n, table.size(1), page_size,
                             ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, current_stream(table)),
           "cache_plan");
  return {granted, slots};
}

// The rows of a tensor of logits: any strides but the last one's.
morpho_logits check_logits(const at::Tensor& t, const char* name, const at::Tensor& logits, int64_t B, int64_t rows,
                           int64_t vocab) {
  TORCH_CHECK(t.is_cuda() && t.device() == logits.device(), name, " must be a CUDA tensor on the device of logits");
  TORCH_CHECK(t.scalar_type() == logits.scalar_type(), name, " must have the type of logits");
  TORCH_CHECK(t.dim() == 3 && t.size(0) == B && t.size(1) == rows && t.size(2) == vocab, name, " must be [", B, ", ",
              rows, ", ", vocab, "]");
  TORCH_CHECK(vocab == 1 || t.stride(2) == 1, name, " must be contiguous along the vocabulary");
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

std::vector<at::Tensor> op_verify_drafts(const at::Tensor& logits, const at::Tensor& tokens, const at::Tensor& uniform,
                                         const std::optional<at::Tensor>& tree,
                                         const std::optional<at::Tensor>& new_lens,
                                         const std::optional<at::Tensor>& draft_logits, double temperature) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  const auto st = logits.scalar_type();
  TORCH_CHECK(st == at::kHalf || st == at::kBFloat16 || st == at::kFloat,
              "logits must be float16, bfloat16 or float32");
  TORCH_CHECK(logits.dim() == 3, "logits must be [B, n, vocab]");
  const int64_t B = logits.size(0), n = logits.size(1), V = logits.size(2);
  const morpho_logits p = check_logits(logits, "logits", logits, B, n, V);
  morpho_logits q{nullptr, 0, 0};
  if (draft_logits && n > 1) q = check_logits(*draft_logits, "draft_logits", logits, B, n - 1, V);
  auto flat = [&](const at::Tensor& t, at::ScalarType type, const char* name, const char* type_name) {
    TORCH_CHECK(t.is_cuda() && t.device() == logits.device(), name, " must be a CUDA tensor on the device of logits");
    TORCH_CHECK(t.scalar_type() == type && t.is_contiguous() && t.dim() == 2 && t.size(0) == B && t.size(1) == n, name,
                " must be a contiguous ", type_name, " [B, n] tensor");
  };
  flat(tokens, at::kLong, "tokens", "int64");
  flat(uniform, at::kFloat, "uniform", "float32");
  if (tree) flat(*tree, at::kLong, "tree", "int64");
  if (new_lens) {
    check_ints(*new_lens, "new_lens", logits);
    TORCH_CHECK(new_lens->dim() == 1 && new_lens->size(0) == B, "new_lens must be [B]");
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  const int type = st == at::kHalf ? MORPHO_FLOAT16 : st == at::kBFloat16 ? MORPHO_BFLOAT16 : MORPHO_FLOAT32;
  auto keep = at::empty({B, n}, logits.options().dtype(at::kInt));
  auto keep_lens = at::empty({B}, logits.options().dtype(at::kInt));
  auto token = at::empty({B}, logits.options().dtype(at::kLong));
  const size_t ws_bytes = morpho_verify_workspace_size(B, n, V, type, q.data != nullptr, tree.has_value(), temperature);
  at::Tensor ws;
  if (ws_bytes) ws = at::empty({(int64_t)ws_bytes}, logits.options().dtype(at::kByte));
  raise_on(morpho_verify_drafts(&p, &q, type, tokens.data_ptr<int64_t>(), uniform.data_ptr<float>(),
                                tree ? tree->data_ptr<int64_t>() : nullptr,
                                new_lens ? new_lens->data_ptr<int32_t>() : nullptr, keep.data_ptr<int32_t>(),
                                keep_lens.data_ptr<int32_t>(), token.data_ptr<int64_t>(), B, n, V, temperature,
                                ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, current_stream(logits)),
           "verify_drafts");
  return {keep, keep_lens, token};
}

}  // namespace

TORCH_LIBRARY(morphottention, m) {
  m.def("forward(Tensor X, Tensor W_phi, Tensor gate_q, Tensor gate_k, Tensor W_V, "
        "int H, int cube_m, float scale, bool causal) -> Tensor[]");
  m.def("backward(Tensor grad_out, Tensor X, Tensor W_phi, Tensor gate_q, Tensor gate_k, "
        "Tensor W_V, Tensor out, Tensor lse, int H, int cube_m, float scale, bool causal) -> Tensor[]");
  m.def("forward_train(Tensor X, Tensor W_phi, Tensor gate_q, Tensor gate_k, Tensor W_V, "
        "int H, int cube_m, float scale, bool causal, int variant=0) -> Tensor[]");
  m.def("backward_train(Tensor grad_out, Tensor X, Tensor W_phi, Tensor gate_q, Tensor gate_k, "
        "Tensor W_V, Tensor out, Tensor lse, Tensor workspace, int H, int cube_m, float scale, bool causal, "
        "int variant=0) -> Tensor[]");
  m.def("soft_forward(Tensor X, Tensor W_phi, Tensor gate_q, Tensor gate_k, Tensor W_V, Tensor tau, "
        "int H, int cube_m, float scale, bool causal, int sgn, int variant=0) -> Tensor[]");
  m.def("soft_backward(Tensor grad_out, Tensor X, Tensor W_phi, Tensor gate_q, Tensor gate_k, Tensor W_V, "
        "Tensor tau, Tensor zb, Tensor workspace, int H, int cube_m, float scale, bool causal, int sgn, "
        "int variant=0) -> Tensor[]");
  m.def("cache_append(Tensor X, Tensor weights, Tensor(a!) codes, Tensor(b!) values, Tensor table, Tensor lens, "
        "Tensor? new_lens=None, int variant=0) -> Tensor");
  m.def("cache_attention(Tensor phi, Tensor gate_q, Tensor gate_k, Tensor codes, Tensor values, Tensor table, "
        "Tensor lens, Tensor? new_lens, Tensor? tree, float scale, bool causal, int variant=0, int max_len=0) "
        "-> Tensor[]");
  m.def("cache_copy_pages(Tensor(a!) codes, Tensor(b!) values, Tensor src, Tensor dst) -> ()");
  m.def("cache_compact(Tensor(a!) codes, Tensor(b!) values, Tensor table, Tensor lens, Tensor keep, "
        "Tensor? keep_lens=None) -> ()");
  m.def("cache_shared_attention(Tensor phi, Tensor gate_q, Tensor gate_k, Tensor codes, Tensor values, Tensor table, "
        "Tensor lens, Tensor? new_lens, Tensor? tree, Tensor members, Tensor starts, Tensor group, Tensor pages, "
        "int max_prefix, int max_rest, float scale, bool causal, int variant=0) -> Tensor[]");
  m.def("cache_plan(Tensor(a!) table, Tensor(b!) held, Tensor lens, Tensor(c!) free_pages, Tensor(d!) free_count, "
        "int n, Tensor? new_lens, int page_size) -> Tensor[]");
  m.def("verify_drafts(Tensor logits, Tensor tokens, Tensor uniform, Tensor? tree, Tensor? new_lens, "
        "Tensor? draft_logits, float temperature) -> Tensor[]");
}

TORCH_LIBRARY_IMPL(morphottention, CUDA, m) {
  m.impl("forward", &op_forward);
  m.impl("backward", &op_backward);
  m.impl("forward_train", &op_forward_train);
  m.impl("backward_train", &op_backward_train);
  m.impl("soft_forward", &op_soft_forward);
  m.impl("soft_backward", &op_soft_backward);
  m.impl("cache_append", &op_cache_append);
  m.impl("cache_attention", &op_cache_attention);
  m.impl("cache_copy_pages", &op_cache_copy_pages);
  m.impl("cache_compact", &op_cache_compact);
  m.impl("cache_shared_attention", &op_cache_shared_attention);
  m.impl("cache_plan", &op_cache_plan);
  m.impl("verify_drafts", &op_verify_drafts);
}
