// The operators' host path in C++: argument checks, allocations, launch and, where there is one, the autograd node.
//
// A call on small tensors is bound by the host.  Through a Python autograd function and ctypes a forward + backward pass of
// simplicial attention on one small molecule took 171 us of which the kernels are 15; the backward node additionally
// competes for the interpreter lock with the thread that waits for it.  A block list (two launches of 17 us together) took 27 us
// that way and takes 20.  These functions serve calls whose operands are
// ready as they are (contiguous, on one device, of the types the kernels take) and return None for every other call, which
// then takes the Python path with its conversions and error messages.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <mutex>

#include "../../include/matterformer_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;
using torch::autograd::Variable;
using OptTensor = std::optional<Tensor>;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MF_DTYPE_F32;
    case at::kBFloat16: return MF_DTYPE_BF16;
    case at::kHalf: return MF_DTYPE_F16;
    default: return -1;
  }
}

void check(int rc) {
  if (rc == MF_OK) return;
  char msg[512];
  mf_last_error(msg, sizeof(msg));
  if (rc == MF_ERR_INVALID_ARGUMENT) throw py::value_error(msg);
  throw std::runtime_error(msg);
}

// The status word of the most recent call on kernels that keep one (see simplicial.py).
std::mutex g_status_mutex;
OptTensor g_status;
void remember_status(OptTensor workspace) {
  OptTensor word;
  if (workspace) word = at::narrow_copy(*workspace, 0, 0, 4);
  std::lock_guard<std::mutex> lock(g_status_mutex);
  g_status = std::move(word);
}
OptTensor last_status() {
  std::lock_guard<std::mutex> lock(g_status_mutex);
  return g_status;
}

const float* fptr(const Tensor& t) { return t.defined() && t.numel() ? t.const_data_ptr<float>() : nullptr; }
float* grad_ptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
Tensor bytes(int64_t n, const Tensor& like) { return n ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor(); }

// The workspace that a call asks for.  On tensor-core kernels without a status word it only holds the list of heavy molecules, which
// the caller may not want.
size_t workspace_bytes(const MfSimplicialFwdArgs& a, bool heavy_first) {
  const bool leave_out = !heavy_first && mf_simplicial_fwd_backend(&a) == MF_BACKEND_TCGEN05 && !mf_simplicial_fwd_keeps_status(&a);
  return leave_out ? 0 : mf_simplicial_fwd_workspace_bytes(&a);
}
size_t workspace_bytes(const MfSimplicialBwdArgs& a, bool heavy_first) {
  const bool leave_out = !heavy_first && mf_simplicial_bwd_backend(&a) == MF_BACKEND_TCGEN05 && !mf_simplicial_bwd_keeps_status(&a);
  return leave_out ? 0 : mf_simplicial_bwd_workspace_bytes(&a);
}

// ---------------------------------------------------------------------------------------------------------------------
// 2-simplicial attention
// ---------------------------------------------------------------------------------------------------------------------
// inputs: q k1 v1 k2 v2 | query_valid key_valid pair_valid | u v w gate | al ar agate | ml mr basis   (undefined when absent)
enum { Q, K1, V1, K2, V2, QV, KV, PV, U, V, W, GATE, AL, AR, AG, ML, MR, BASIS, kInputs };

template <typename Args>
void fill_common(Args& a, const std::array<Tensor, kInputs>& t, int precision, int backend) {
  const Tensor& q = t[Q];
  a.batch = q.size(0), a.heads = q.size(1), a.tokens = q.size(2), a.head_dim = q.size(3);
  a.dtype = dtype_code(q), a.precision = precision, a.backend = backend;
  a.q = q.const_data_ptr(), a.k1 = t[K1].const_data_ptr(), a.v1 = t[V1].const_data_ptr(), a.k2 = t[K2].const_data_ptr(),
  a.v2 = t[V2].const_data_ptr();
  a.query_valid = static_cast<const uint8_t*>(t[QV].const_data_ptr());
  a.pair_key_valid = static_cast<const uint8_t*>(t[KV].const_data_ptr());
  a.pair_valid = t[PV].defined() ? static_cast<const uint8_t*>(t[PV].const_data_ptr()) : nullptr;
  a.u = fptr(t[U]), a.v_bias = fptr(t[V]), a.w = fptr(t[W]), a.gate = fptr(t[GATE]);
  a.angle_left = fptr(t[AL]), a.angle_right = fptr(t[AR]), a.angle_gate = fptr(t[AG]);
  a.message_left = fptr(t[ML]), a.message_right = fptr(t[MR]), a.message_basis = fptr(t[BASIS]);
  a.angle_rank = t[AL].defined() ? t[AL].size(4) : 0, a.message_rank = t[ML].defined() ? t[ML].size(4) : 0;
}

struct SimplicialAttention : torch::autograd::Function<SimplicialAttention> {
  static Variable forward(AutogradContext* ctx, const Tensor& q, const Tensor& k1, const Tensor& v1, const Tensor& k2,
                          const Tensor& v2, const Tensor& qv, const Tensor& kv, const OptTensor& pv, const OptTensor& u,
                          const OptTensor& v, const OptTensor& w, const OptTensor& gate, const OptTensor& al, const OptTensor& ar,
                          const OptTensor& ag, const OptTensor& ml, const OptTensor& mr, const OptTensor& basis, int64_t precision,
                          int64_t backend, bool heavy_first) {
    auto or_none = [](const OptTensor& t) { return t ? *t : Tensor(); };
    const std::array<Tensor, kInputs> t = {q, k1, v1, k2, v2, qv, kv, or_none(pv), or_none(u), or_none(v), or_none(w), or_none(gate),
                                           or_none(al), or_none(ar), or_none(ag), or_none(ml), or_none(mr), or_none(basis)};
    const c10::cuda::CUDAGuard guard(q.device());
    MfSimplicialFwdArgs a{};
    fill_common(a, t, precision, backend);
    const Tensor out32 = at::empty(q.sizes(), q.options().dtype(at::kFloat));
    const Tensor lse = at::empty(q.sizes().slice(0, 3), out32.options());
    const Tensor out = q.scalar_type() == at::kFloat ? out32 : at::empty_like(q);
    a.out = out32.data_ptr<float>(), a.lse = lse.data_ptr<float>();
    a.out_cast = out.is_same(out32) ? nullptr : out.data_ptr();
    const Tensor ws = bytes(workspace_bytes(a, heavy_first), q);
    if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    check(mf_simplicial_fwd(&a, c10::cuda::getCurrentCUDAStream().stream()));
    if (mf_simplicial_fwd_backend(&a) == MF_BACKEND_TCGEN05)
      remember_status(ws.defined() && mf_simplicial_fwd_keeps_status(&a) ? OptTensor(ws) : std::nullopt);
    ctx->saved_data["call"] = precision | backend << 8 | (int64_t)heavy_first << 16;
    tensor_list saved(t.begin(), t.end());
    saved.push_back(out32);
    saved.push_back(lse);
    ctx->save_for_backward(std::move(saved));
    return out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grad_out) {
    const tensor_list saved = ctx->get_saved_variables();
    std::array<Tensor, kInputs> t;
    std::copy(saved.begin(), saved.begin() + kInputs, t.begin());
    const Tensor &q = t[Q], &out32 = saved[kInputs], &lse = saved[kInputs + 1];
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor go = grad_out[0].to(q.scalar_type()).contiguous();
    MfSimplicialBwdArgs a{};
    const int64_t call = ctx->saved_data["call"].toInt();
    fill_common(a, t, call & 255, call >> 8 & 255);
    a.grad_out = go.const_data_ptr(), a.out = out32.const_data_ptr<float>(), a.lse = lse.const_data_ptr<float>();
    tensor_list g(kInputs + 3);  // (one for each argument of forward)
    for (int i = Q; i <= V2; ++i) g[i] = at::empty_like(q);
    a.dq = g[Q].data_ptr(), a.dk1 = g[K1].data_ptr(), a.dv1 = g[V1].data_ptr(), a.dk2 = g[K2].data_ptr(), a.dv2 = g[V2].data_ptr();
    // edges of the node are counted over the tensors that were given
    auto wanted = [&](int i) {
      if (!t[i].defined()) return false;
      size_t edge = 0;
      for (int j = 0; j < i; ++j) edge += t[j].defined();
      return ctx->needs_input_grad(edge);
    };
    Tensor coeff;
    if (t[U].defined() || t[AL].defined() || t[ML].defined()) {
      const bool zeros = mf_simplicial_bwd_needs_zeros(&a) != 0;
      auto make = [&](const Tensor& like) { return zeros ? at::zeros_like(like) : at::empty_like(like); };
      for (int i = U; i <= MR; ++i)
        if (wanted(i)) g[i] = make(t[i]);
      a.du = grad_ptr(g[U]), a.dv_bias = grad_ptr(g[V]), a.dw = grad_ptr(g[W]), a.dgate = grad_ptr(g[GATE]);
      a.dangle_left = grad_ptr(g[AL]), a.dangle_right = grad_ptr(g[AR]), a.dangle_gate = grad_ptr(g[AG]);
      a.dmessage_left = grad_ptr(g[ML]), a.dmessage_right = grad_ptr(g[MR]);
      if (wanted(BASIS)) {
        const std::vector<int64_t> shape = {a.batch, a.heads, a.tokens, a.message_rank};
        coeff = zeros ? at::zeros(shape, lse.options()) : at::empty(shape, lse.options());
        a.message_coeff = coeff.data_ptr<float>();
      }
    }
    const Tensor ws = bytes(workspace_bytes(a, call >> 16), q);
    if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
    check(mf_simplicial_bwd(&a, stream));
    if (mf_simplicial_bwd_backend(&a) == MF_BACKEND_TCGEN05)
      remember_status(ws.defined() && mf_simplicial_bwd_keeps_status(&a) ? OptTensor(ws) : std::nullopt);
    if (coeff.defined()) {
      g[BASIS] = at::empty_like(t[BASIS]);
      check(mf_simplicial_basis_grad(a.message_coeff, a.grad_out, a.dtype, a.batch, a.heads, a.tokens, a.message_rank, a.head_dim,
                                     g[BASIS].data_ptr<float>(), stream));
    }
    return g;
  }
};

bool ready(const Tensor& t, const Tensor& like, at::ScalarType type, at::IntArrayRef shape) {
  return t.device() == like.device() && t.scalar_type() == type && t.sizes() == shape && t.is_contiguous();
}

std::optional<Tensor> simplicial_attention(const Tensor& q, const Tensor& k1, const Tensor& v1, const Tensor& k2, const Tensor& v2,
                                           const Tensor& qv, const Tensor& kv, const OptTensor& pv, std::vector<OptTensor> bias,
                                           std::vector<OptTensor> angle, std::vector<OptTensor> message, int64_t precision,
                                           int64_t backend, int64_t max_rank, bool heavy_first) {
  if (!q.is_cuda() || q.dim() != 4 || dtype_code(q) < 0 || !q.is_contiguous()) return std::nullopt;
  for (const Tensor* t : {&k1, &v1, &k2, &v2})
    if (!ready(*t, q, q.scalar_type(), q.sizes())) return std::nullopt;
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  if (!ready(qv, q, at::kBool, {B, N}) || !ready(kv, q, at::kBool, {B, N})) return std::nullopt;
  if (pv && !ready(*pv, q, at::kBool, {B, N, N})) return std::nullopt;
  auto complete = [](const std::vector<OptTensor>& g, size_t n) {
    if (g.size() != n) return false;
    for (const OptTensor& t : g)
      if (!t || !t->defined()) return false;
    return true;
  };
  if (!bias.empty()) {
    if (!complete(bias, 4)) return std::nullopt;
    for (int i = 0; i < 3; ++i)
      if (!ready(*bias[i], q, at::kFloat, {B, H, N, N})) return std::nullopt;
    if (!ready(*bias[3], q, at::kFloat, {B, H, N})) return std::nullopt;
  }
  if (!angle.empty()) {
    if (!complete(angle, 3) || angle[0]->dim() != 5) return std::nullopt;
    const int64_t R = angle[0]->size(4);
    if (R < 1 || R > max_rank || !ready(*angle[0], q, at::kFloat, {B, H, N, N, R}) || !ready(*angle[1], q, at::kFloat, {B, H, N, N, R}) ||
        !ready(*angle[2], q, at::kFloat, {B, H, N}))
      return std::nullopt;
  }
  if (!message.empty()) {
    if (!complete(message, 3) || message[0]->dim() != 5) return std::nullopt;
    const int64_t R = message[0]->size(4);
    if (R < 1 || R > max_rank || !ready(*message[0], q, at::kFloat, {B, H, N, N, R}) ||
        !ready(*message[1], q, at::kFloat, {B, H, N, N, R}) || !ready(*message[2], q, at::kFloat, {H, R, D}))
      return std::nullopt;
  }
  bias.resize(4), angle.resize(3), message.resize(3);
  return SimplicialAttention::apply(q, k1, v1, k2, v2, qv, kv, pv, bias[0], bias[1], bias[2], bias[3], angle[0], angle[1], angle[2],
                                    message[0], message[1], message[2], precision, backend, heavy_first);
}

// ---------------------------------------------------------------------------------------------------------------------
// Radius block-sparse and local-window attention
// ---------------------------------------------------------------------------------------------------------------------
struct SparseAttention : torch::autograd::Function<SparseAttention> {
  static void fill(MfSparseAttnArgs& a, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& n, const Tensor& count,
                   const Tensor& cols, const Tensor& mask, int64_t window, double scale, int64_t backend) {
    a.batch = q.size(0), a.heads = q.size(1), a.tokens = q.size(2), a.head_dim = q.size(3);
    a.dtype = dtype_code(q), a.window = window, a.scale = scale, a.backend = a.dtype == MF_DTYPE_BF16 ? backend : 0;
    a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr();
    a.num_atoms = n.const_data_ptr<int32_t>();
    if (window == 0) {
      a.block_count = count.const_data_ptr<int32_t>(), a.block_cols = cols.const_data_ptr<int32_t>();
      a.block_mask = reinterpret_cast<const uint32_t*>(mask.const_data_ptr<int32_t>());
    }
  }

  static Variable forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& n, const Tensor& count,
                          const Tensor& cols, const Tensor& mask, int64_t window, double scale, int64_t backend) {
    const c10::cuda::CUDAGuard guard(q.device());
    MfSparseAttnArgs a{};
    fill(a, q, k, v, n, count, cols, mask, window, scale, backend);
    const Tensor out = at::empty_like(q), lse = at::empty(q.sizes().slice(0, 3), q.options().dtype(at::kFloat));
    a.out = out.data_ptr(), a.lse = lse.data_ptr<float>();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
    check(window ? mf_local_attn_fwd(&a, stream) : mf_radius_attn_fwd(&a, stream));
    ctx->saved_data["window"] = window;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["backend"] = backend;
    ctx->save_for_backward({q, k, v, n, count, cols, mask, out, lse});
    return out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grad_out) {
    const tensor_list s = ctx->get_saved_variables();
    const Tensor& q = s[0];
    const c10::cuda::CUDAGuard guard(q.device());
    const int64_t window = ctx->saved_data["window"].toInt();
    MfSparseAttnArgs a{};
    fill(a, q, s[1], s[2], s[3], s[4], s[5], s[6], window, ctx->saved_data["scale"].toDouble(), ctx->saved_data["backend"].toInt());
    const Tensor go = grad_out[0].to(q.scalar_type()).contiguous();
    a.out = s[7].data_ptr(), a.lse = s[8].data_ptr<float>(), a.grad_out = go.const_data_ptr();
    tensor_list g(10);
    for (int i = 0; i < 3; ++i) g[i] = at::empty_like(q);
    a.dq = g[0].data_ptr(), a.dk = g[1].data_ptr(), a.dv = g[2].data_ptr();
    const Tensor ws = bytes(mf_sparse_attn_bwd_workspace_bytes(&a), q);
    if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    const cudaStream_t stream = c10::cuda::getCurrentCUDAStream().stream();
    check(window ? mf_local_attn_bwd(&a, stream) : mf_radius_attn_bwd(&a, stream));
    return g;
  }
};

// window 0: the block list; otherwise the band.  `n` (B) int32; the caller has checked shapes and types of q, k, v.
std::optional<Tensor> sparse_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& n, const Tensor& count,
                                       const Tensor& cols, const Tensor& mask, int64_t window, double scale, int64_t backend) {
  for (const Tensor* t : {&q, &k, &v})
    if (!ready(*t, q, q.scalar_type(), q.sizes())) return std::nullopt;
  if (!ready(n, q, at::kInt, {q.size(0)})) return std::nullopt;
  if (window == 0)
    for (const Tensor* t : {&count, &cols, &mask})
      if (t->device() != q.device() || t->scalar_type() != at::kInt || !t->is_contiguous()) return std::nullopt;
  return SparseAttention::apply(q, k, v, n, count, cols, mask, window, scale, backend);
}

// ---------------------------------------------------------------------------------------------------------------------
// Neighbour lists and block lists
// ---------------------------------------------------------------------------------------------------------------------
// Positions (B, N, 3), latents (B, 6) or cells (B, 3, 3) and, if given, counts of the types and on the device that the kernels take.
bool structures_ready(const Tensor& pos, const Tensor& lattice, const OptTensor& n) {
  if (!pos.is_cuda() || pos.dim() != 3 || pos.size(2) != 3 || pos.numel() == 0 || !ready(pos, pos, at::kFloat, pos.sizes())) return false;
  const int64_t B = pos.size(0);
  if (!ready(lattice, pos, at::kFloat, {B, 6}) && !ready(lattice, pos, at::kFloat, {B, 3, 3})) return false;
  return !n || (n->numel() == B && ready(*n, pos, at::kInt, n->sizes()));
}
Tensor counts(const OptTensor& n, const Tensor& pos, const at::TensorOptions& ints) {
  return n ? *n : at::full({pos.size(0)}, pos.size(1), ints);
}

// perm, block_count, block_cols, block_mask, num_atoms
std::optional<std::array<Tensor, 5>> radius_blocks(const Tensor& pos, const Tensor& lattice, const OptTensor& num_atoms, double cutoff) {
  if (!structures_ready(pos, lattice, num_atoms)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(pos.device());
  const int64_t B = pos.size(0), N = pos.size(1), T = (N + 31) / 32;
  const auto ints = at::TensorOptions(pos.device()).dtype(at::kInt);
  const Tensor n = counts(num_atoms, pos, ints);
  const Tensor perm = at::empty({B, N}, ints), count = at::empty({B, T}, ints), cols = at::empty({B, T, T}, ints);
  const Tensor mask = at::empty({B, T, T, 32}, ints), ws = bytes(mf_radius_blocks_workspace_bytes(B, N), pos);
  check(mf_radius_blocks(pos.const_data_ptr<float>(), lattice.const_data_ptr<float>(), lattice.dim() == 3, n.const_data_ptr<int32_t>(), B, N,
                         cutoff, perm.data_ptr<int32_t>(), count.data_ptr<int32_t>(), cols.data_ptr<int32_t>(),
                         reinterpret_cast<uint32_t*>(mask.data_ptr<int32_t>()), ws.data_ptr(), ws.numel(),
                         c10::cuda::getCurrentCUDAStream().stream()));
  return std::array<Tensor, 5>{perm, count, cols, mask, n};
}

std::optional<std::array<Tensor, 2>> knn_topk(const Tensor& pos, const Tensor& lattice, const OptTensor& num_atoms, int64_t k,
                                              bool include_self) {
  if (k < 1 || k > 32 || !structures_ready(pos, lattice, num_atoms)) return std::nullopt;
  const c10::cuda::CUDAGuard guard(pos.device());
  const int64_t B = pos.size(0), N = pos.size(1);
  const auto ints = at::TensorOptions(pos.device()).dtype(at::kInt);
  const Tensor n = counts(num_atoms, pos, ints);
  const Tensor idx = at::empty({B, N, k}, ints), d2 = at::empty({B, N, k}, ints.dtype(at::kFloat));
  const Tensor ws = bytes(mf_knn_cells_workspace_bytes(B, N), pos);
  check(mf_knn_topk_lattice(pos.const_data_ptr<float>(), lattice.const_data_ptr<float>(), lattice.dim() == 3, n.const_data_ptr<int32_t>(), B,
                            N, k, include_self, idx.data_ptr<int32_t>(), d2.data_ptr<float>(), ws.data_ptr(), ws.numel(),
                            c10::cuda::getCurrentCUDAStream().stream()));
  return std::array<Tensor, 2>{idx, d2};
}

// ---------------------------------------------------------------------------------------------------------------------
// A backward pass under capture
// ---------------------------------------------------------------------------------------------------------------------
// A leaf has one node that takes its gradients, on the stream on which the first graph that is still alive made it.  The engine joins
// that stream with the one of a backward pass.  While the latter is being captured another stream joins the capture, but the default stream
// cannot: that ends the capture with an error of the runtime which names nothing.  The operators below say so instead: noted when
// their forward pass is captured, raised by its backward pass.
bool foreign_leaf(const Tensor& t) {
  if (!t.defined() || !t.is_cuda() || !t.requires_grad() || !t.is_leaf()) return false;
  const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
  if (!node) return false;
  const auto stream = node->stream();
  return stream && *stream == c10::cuda::getDefaultCUDAStream(t.device().index()).unwrap();
}
// Whether something follows the operations of this thread and would not see a kernel launched past them: a trace, a dispatch mode, a
// transform of torch.func.  (What matterformer_b200.fused.watched asks, without its microsecond.)
bool watched() {
  return torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::stack_len() > 0 ||
         c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}
bool capturing() { return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; }
bool foreign_leaves(std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled() || !capturing()) return false;
  for (const Tensor* t : inputs)
    if (foreign_leaf(*t)) return true;
  return false;
}
void refuse_foreign(bool foreign, const char* name) {
  if (foreign && capturing())
    throw std::runtime_error(std::string(name) + ": a backward pass cannot be captured while a graph of the same leaf from the default stream is alive; "
                             "release that graph (the outputs that hold it) before the capture");
}

// ---------------------------------------------------------------------------------------------------------------------
// Gated feed-forward block
// ---------------------------------------------------------------------------------------------------------------------
// A contiguous tensor without the way through the dispatcher, which takes as long again as the allocation.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), at::MemoryFormat::Contiguous));
}
Tensor fresh_bytes(int64_t n, const Tensor& like) { return n ? fresh({n}, at::kByte, like) : Tensor(); }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

struct GatedMlp : torch::autograd::Function<GatedMlp> {
  static void fill(MfGatedMlpArgs& a, const Tensor& x, const Tensor& w_in, const Tensor& w_out, const Tensor& b_in, const Tensor& b_out, int64_t activation) {
    a.dim = x.size(-1), a.hidden = w_out.size(1), a.dim_out = w_out.size(0), a.rows = x.numel() / a.dim;
    a.dtype = a.grad_dtype = dtype_code(x), a.activation = activation;
    a.x = x.const_data_ptr(), a.w_in = w_in.const_data_ptr(), a.w_out = w_out.const_data_ptr();
    a.b_in = b_in.defined() ? b_in.const_data_ptr() : nullptr, a.b_out = b_out.defined() ? b_out.const_data_ptr() : nullptr;
  }

  struct Made {
    Tensor y, pre, act;
  };
  static Made block(const Tensor& x, const Tensor& w_in, const Tensor& w_out, const Tensor& bi, const Tensor& bo, int64_t activation, bool keep) {
    const c10::cuda::CUDAGuard guard(x.device());
    MfGatedMlpArgs a{};
    fill(a, x, w_in, w_out, bi, bo, activation);
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = a.dim_out;
    const Tensor y = fresh(shape, x.scalar_type(), x), act = fresh({a.rows, a.hidden}, x.scalar_type(), x);
    const Tensor pre = keep ? fresh_bytes((int64_t)mf_gated_mlp_pre_bytes(a.rows, a.hidden), x) : Tensor();
    a.y = y.data_ptr(), a.act = act.data_ptr(), a.pre = keep ? pre.data_ptr() : nullptr;
    const Tensor ws = fresh_bytes(mf_gated_mlp_fwd_workspace_bytes(&a), x);
    if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    check(mf_gated_mlp_fwd(&a, c10::cuda::getCurrentCUDAStream().stream()));
    return {y, pre, act};
  }

  static Variable forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_in, const Tensor& w_out, const OptTensor& b_in, const OptTensor& b_out,
                          int64_t activation, bool foreign) {
    const Tensor bi = b_in ? *b_in : Tensor(), bo = b_out ? *b_out : Tensor();
    const Made made = block(x, w_in, w_out, bi, bo, activation, true);
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["foreign"] = foreign;
    ctx->save_for_backward({x, w_in, w_out, bi, bo, made.pre, made.act});
    return made.y;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grad_y) {
    const tensor_list s = ctx->get_saved_variables();
    const Tensor& x = s[0];
    const c10::cuda::CUDAGuard guard(x.device());
    MfGatedMlpArgs a{};
    tensor_list g(7);  // (one for each argument of forward)
    refuse_foreign(ctx->saved_data["foreign"].toBool(), "gated_mlp");
    {
      const at::NoGradGuard no_grad;
      fill(a, x, s[1], s[2], s[3], s[4], ctx->saved_data["activation"].toInt());
      Tensor gy = grad_y[0].to(x.scalar_type()).contiguous();
      if (!aligned(gy)) gy = gy.clone();
      a.pre = s[5].data_ptr(), a.act = s[6].data_ptr(), a.grad_y = gy.const_data_ptr();
      size_t edge = 0;  // edges of the node are counted over the tensors that were given
      for (int i = 0; i < 5; ++i)
        if (s[i].defined() && ctx->needs_input_grad(edge++)) g[i] = fresh(s[i].sizes(), s[i].scalar_type(), s[i]);
      auto ptr = [&](int i) { return g[i].defined() ? g[i].data_ptr() : nullptr; };
      a.grad_x = ptr(0), a.grad_w_in = ptr(1), a.grad_w_out = ptr(2), a.grad_b_in = ptr(3), a.grad_b_out = ptr(4);
      const Tensor ws = fresh_bytes(mf_gated_mlp_bwd_workspace_bytes(&a), x);
      if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
      check(mf_gated_mlp_bwd(&a, c10::cuda::getCurrentCUDAStream().stream()));
    }
    if (at::GradMode::is_enabled()) {  // create_graph: an error for who differentiates again, as torch's once_differentiable has it
      tensor_list given;
      for (int i = 0; i < 5; ++i)
        if (g[i].defined()) given.push_back(g[i].set_requires_grad(true));
      const auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable",
                                                                        (int64_t)given.size());
      const tensor_list out = (*node)(std::move(given));
      for (int i = 0, j = 0; i < 5; ++i)
        if (g[i].defined()) g[i] = out[j++];
    }
    return g;
  }
};

// Parameters in the type of x, everything contiguous and aligned, nothing that watches.
std::optional<Tensor> gated_mlp(const Tensor& x, const Tensor& w_in, const Tensor& w_out, const OptTensor& b_in, const OptTensor& b_out, int64_t activation) {
  if (watched() || !x.is_cuda() || x.dim() < 1 || (x.scalar_type() != at::kBFloat16 && x.scalar_type() != at::kHalf) || !x.is_contiguous() || x.numel() == 0) return std::nullopt;
  if (w_out.dim() != 2) return std::nullopt;
  const int64_t C = x.size(-1), O = w_out.size(0), F = w_out.size(1);
  if (C % 8 || O % 8 || F % 8 || C < 8 || O < 8 || F < 8 || std::max({C, O, F}) > 1 << 28) return std::nullopt;
  const at::ScalarType type = x.scalar_type();
  if (!ready(w_in, x, type, {2 * F, C}) || !ready(w_out, x, type, {O, F}) || (b_in && !ready(*b_in, x, type, {2 * F})) ||
      (b_out && !ready(*b_out, x, type, {O})))
    return std::nullopt;
  bool keep = false;
  for (const Tensor* t : {&x, &w_in, &w_out, b_in ? &*b_in : &x, b_out ? &*b_out : &x}) {
    if (!aligned(*t) || t->_fw_grad(0).defined()) return std::nullopt;
    keep = keep || t->requires_grad();
  }
  const Tensor none;
  const Tensor &bi = b_in ? *b_in : none, &bo = b_out ? *b_out : none;
  if (!keep || !at::GradMode::is_enabled()) return GatedMlp::block(x, w_in, w_out, bi, bo, activation, false).y;
  const c10::cuda::CUDAGuard guard(x.device());
  return GatedMlp::apply(x, w_in, w_out, b_in, b_out, activation, foreign_leaves({&x, &w_in, &w_out, &bi, &bo}));
}

// ---------------------------------------------------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------------------------------------------------
// What a call turns by; `table` (axes, pairs), or (pairs) where `flat`, is the caller's.
struct Turning {
  const double* table;
  int64_t axes, pairs;
  bool flat;
  int64_t heads, layout;  // heads 0: one or two head-major tensors; otherwise a packed projection with that many heads
  double amplitude;
  bool inverse;
};
// The same for the backward pass, with a copy of the table, which may have changed by then.
struct SavedTurning : torch::CustomClassHolder {
  Turning turning;
  std::array<double, 128> table;
  bool foreign;
  SavedTurning(const Turning& t, bool foreign_) : turning(t), foreign(foreign_) {
    std::copy_n(t.table, t.axes * t.pairs, table.begin());
    turning.table = table.data();
    turning.inverse = !t.inverse;
  }
};

struct Rotary : torch::autograd::Function<Rotary> {
  static tensor_list turn(const Tensor& first, const OptTensor& second, const Tensor& positions, const Turning& by) {
    const c10::cuda::CUDAGuard guard(first.device());
    const int64_t heads = by.heads;
    auto adjacent = [](const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); };
    const Tensor x[2] = {adjacent(first), second ? adjacent(*second) : Tensor()};
    tensor_list out;
    MfRotaryArgs a{};
    auto add = [&](const Tensor& t, const Tensor& o, int64_t at, int64_t n, bool rotates, int token, int64_t head_in, int64_t head_out) {
      const int64_t bytes = at * (int64_t)t.element_size();
      a.tensor[a.tensors++] = {static_cast<const char*>(t.const_data_ptr()) + bytes, static_cast<char*>(o.data_ptr()) + bytes, (int32_t)n, rotates,
                               t.stride(0), t.stride(token), head_in, o.stride(0), o.stride(token), head_out};
    };
    for (const Tensor& t : x) {
      if (!t.defined()) continue;
      out.push_back(t.is_contiguous() ? fresh(t.sizes(), t.scalar_type(), t) : at::empty_like(t));
      if (out.back().stride(-1) != 1) out.back() = at::empty(t.sizes(), t.options());  // (overlapping inputs may have another order)
      const Tensor& o = out.back();
      a.batch = t.size(0), a.tokens = t.size(heads ? 1 : 2), a.head_dim = heads ? t.size(2) / (3 * heads) : t.size(3);
      if (heads)
        for (int i = 0; i < 3; ++i) add(t, o, i * heads * a.head_dim, heads, i < 2, 1, a.head_dim, a.head_dim);
      else add(t, o, 0, t.size(1), true, 2, t.stride(1), o.stride(1));
    }
    a.axes = by.axes, a.pairs = by.pairs;
    a.dtype = dtype_code(first), a.layout = by.layout, a.inverse = by.inverse, a.amplitude = by.amplitude;
    a.position_type = positions.scalar_type() == at::kInt    ? MF_POSITION_I32
                      : positions.scalar_type() == at::kLong ? MF_POSITION_I64
                      : positions.scalar_type() == at::kFloat ? MF_POSITION_F32
                                                             : MF_POSITION_F64;
    a.positions = positions.const_data_ptr(), a.position_batch = positions.dim() == (by.flat ? 2 : 3) ? positions.stride(0) : 0;
    a.frequencies = by.table;
    check(mf_rotary(&a, c10::cuda::getCurrentCUDAStream().stream()));
    return out;
  }

  static tensor_list forward(AutogradContext* ctx, const Tensor& first, const OptTensor& second, const Tensor& positions, const Turning& by, bool foreign) {
    const tensor_list out = turn(first, second, positions, by);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions.is_inference() ? positions.clone() : positions});
    ctx->saved_data["turning"] = c10::IValue::make_capsule(c10::make_intrusive<SavedTurning>(by, foreign));
    return out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list given, g(5);  // (one for each argument of forward)
    const auto held = ctx->saved_data["turning"].toCapsule();
    const SavedTurning& saved = static_cast<const SavedTurning&>(*held);
    refuse_foreign(saved.foreign, "rotary_embedding");
    bool keep = false;
    for (const Tensor& t : grads)
      if (t.defined()) given.push_back(t), keep = keep || (at::GradMode::is_enabled() && t.requires_grad());
    if (given.empty()) return g;
    const Tensor positions = ctx->get_saved_variables()[0];
    const OptTensor second = given.size() > 1 ? OptTensor(given[1]) : std::nullopt;
    const tensor_list turned = keep ? Rotary::apply(given[0], second, positions, saved.turning, false) : turn(given[0], second, positions, saved.turning);
    for (size_t i = 0, j = 0; i < grads.size(); ++i)
      if (grads[i].defined()) g[i] = turned[j++];
    return g;
  }
};

std::optional<tensor_list> rotary(const Tensor& first, const OptTensor& second, const Tensor& positions, const Tensor& table, int64_t heads, int64_t layout,
                                  double amplitude) {
  if (watched() || !first.is_cuda() || dtype_code(first) < 0 || first.dim() != (heads ? 3 : 4) || first.numel() == 0 || !std::isfinite(amplitude)) return std::nullopt;
  if (heads < 0 || (heads && first.size(2) % (3 * heads))) return std::nullopt;
  const int64_t B = first.size(0), N = first.size(heads ? 1 : 2), D = heads ? first.size(2) / (3 * heads) : first.size(3);
  if (second && (second->dim() != 4 || second->scalar_type() != first.scalar_type() || second->device() != first.device() || second->numel() == 0 ||
                 second->size(0) != B || second->size(2) != N || second->size(3) != D))
    return std::nullopt;
  if (B >= 1ll << 31 || N >= 1ll << 31 || (heads ? heads : std::max(first.size(1), second ? second->size(1) : 0)) * D > 1 << 27) return std::nullopt;
  if (!table.device().is_cpu() || table.scalar_type() != at::kDouble || !table.is_contiguous() || table.dim() < 1 || table.dim() > 2 || table.requires_grad() ||
      table.numel() < 1 || table.numel() > 128 || 2 * table.numel() > D)
    return std::nullopt;
  const at::ScalarType type = positions.scalar_type();
  std::vector<int64_t> shape = {B, N};
  if (table.dim() == 2) shape.push_back(table.size(0));
  if (positions.device() != first.device() || !positions.is_contiguous() || positions.requires_grad() ||
      (type != at::kInt && type != at::kLong && type != at::kFloat && type != at::kDouble) ||
      (positions.sizes() != at::IntArrayRef(shape) && positions.sizes() != at::IntArrayRef(shape).slice(1)))
    return std::nullopt;
  if (first._fw_grad(0).defined() || (second && second->_fw_grad(0).defined())) return std::nullopt;
  const bool keep = at::GradMode::is_enabled() && (first.requires_grad() || (second && second->requires_grad()));
  const Turning by = {table.const_data_ptr<double>(), table.dim() == 1 ? 1 : table.size(0), table.size(-1), table.dim() == 1, heads, layout, amplitude, false};
  if (!keep) return Rotary::turn(first, second, positions, by);  // (past autograd: 9.1 -> 6.9 us a call)
  const Tensor none;
  const c10::cuda::CUDAGuard guard(first.device());
  return Rotary::apply(first, second, positions, by, foreign_leaves({&first, second ? &*second : &none}));
}

// ---------------------------------------------------------------------------------------------------------------------
// Dense attention with a learned bias by buckets
// ---------------------------------------------------------------------------------------------------------------------
struct DenseCall : torch::CustomClassHolder {
  int64_t heads, backend;  // heads 0: head-major q, k, v; otherwise a packed projection with that many heads
  bool causal, foreign;
  double scale;
  DenseCall(int64_t heads_, int64_t backend_, bool causal_, bool foreign_, double scale_)
      : heads(heads_), backend(backend_), causal(causal_), foreign(foreign_), scale(scale_) {}
};

struct DenseAttention : torch::autograd::Function<DenseAttention> {
  enum { Q, K, V, BIAS, BUCKETS, NUM_Q, NUM_K, MASK, kOperands };
  using Operands = std::array<Tensor, kOperands>;

  static MfRows rows(const Tensor& t) {
    auto step = [&](int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
    return {step(0), step(1), step(2)};
  }
  // the third `i` of a packed (B, N, 3 H D), or all of a packed (B, N, H D)
  static MfRows packed_rows(const Tensor& t, int64_t D) { return {t.size(1) * t.size(2), D, t.size(2)}; }
  static const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

  static void fill(MfDenseAttnArgs& a, const Operands& t, const DenseCall& call) {
    const Tensor& q = t[Q];
    a.dtype = dtype_code(q), a.causal = call.causal, a.backend = call.backend, a.scale = call.scale;
    a.batch = q.size(0);
    if (call.heads) {
      const int64_t HD = q.size(2) / 3;
      a.heads = a.kv_heads = call.heads, a.queries = a.keys = q.size(1), a.head_dim = HD / call.heads;
      a.q = q.const_data_ptr(), a.k = static_cast<const char*>(a.q) + 2 * HD, a.v = static_cast<const char*>(a.q) + 4 * HD;
      a.q_rows = a.k_rows = a.v_rows = packed_rows(q, a.head_dim);
    } else {
      a.heads = q.size(1), a.queries = q.size(2), a.head_dim = q.size(3), a.kv_heads = t[K].size(1), a.keys = t[K].size(2);
      a.q = q.const_data_ptr(), a.k = t[K].const_data_ptr(), a.v = t[V].const_data_ptr();
      a.q_rows = rows(q), a.k_rows = rows(t[K]), a.v_rows = rows(t[V]);
    }
    a.num_queries = static_cast<const int32_t*>(ptr(t[NUM_Q])), a.num_keys = static_cast<const int32_t*>(ptr(t[NUM_K]));
    a.key_mask = static_cast<const uint8_t*>(ptr(t[MASK])), a.key_mask_batch = a.keys;
    if (t[BIAS].defined()) {
      const Tensor& buckets = t[BUCKETS];
      a.bias = t[BIAS].const_data_ptr(), a.bias_dtype = dtype_code(t[BIAS]), a.num_buckets = t[BIAS].size(0);
      a.buckets = static_cast<const uint8_t*>(buckets.const_data_ptr());
      if (buckets.dim() == 1) a.bucket_kind = MF_BUCKETS_OFFSET, a.reach = buckets.size(0) / 2;
      else a.bucket_kind = MF_BUCKETS_PAIR, a.bucket_batch = buckets.size(0) > 1 ? buckets.stride(0) : 0, a.bucket_row = buckets.stride(1);
    }
  }
  // A dense (B, H, N, D) tensor in the order of tokens and heads of t.
  static Tensor like(const Tensor& t) {
    const int64_t B = t.size(0), H = t.size(1), N = t.size(2), D = t.size(3);
    if (H > 1 && N > 1 && t.stride(1) < t.stride(2)) return fresh({B, N, H, D}, t.scalar_type(), t).transpose(1, 2);
    return fresh({B, H, N, D}, t.scalar_type(), t);
  }

  struct Made {
    Tensor out, lse;
  };
  static Made attend(const Operands& t, const DenseCall& call, bool keep) {
    const Tensor& q = t[Q];
    const c10::cuda::CUDAGuard guard(q.device());
    MfDenseAttnArgs a{};
    fill(a, t, call);
    const Tensor out = call.heads ? fresh({q.size(0), q.size(1), q.size(2) / 3}, q.scalar_type(), q) : like(q);
    a.out = out.data_ptr(), a.out_rows = call.heads ? packed_rows(out, a.head_dim) : rows(out);
    const Tensor lse = keep ? fresh({a.batch, a.heads, a.queries}, at::kFloat, q) : Tensor();
    a.lse = keep ? lse.data_ptr<float>() : nullptr;
    const Tensor ws = fresh_bytes(mf_dense_attn_fwd_workspace_bytes(&a), q);
    if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
    check(mf_dense_attn_fwd(&a, c10::cuda::getCurrentCUDAStream().stream()));
    return {out, lse};
  }

  static Variable forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& v, const OptTensor& bias, const Operands& t,
                          const c10::intrusive_ptr<DenseCall>& call) {
    const Made made = attend(t, *call, true);
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    tensor_list saved(t.begin(), t.end());
    saved.push_back(made.out);
    saved.push_back(made.lse);
    ctx->save_for_backward(std::move(saved));
    return made.out;
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grad_out) {
    const auto held = ctx->saved_data["call"].toCapsule();
    const DenseCall& call = static_cast<const DenseCall&>(*held);
    refuse_foreign(call.foreign, "dense_attention");
    const tensor_list s = ctx->get_saved_variables();
    Operands t;
    std::copy_n(s.begin(), (int)kOperands, t.begin());
    const Tensor &q = t[Q], &out = s[kOperands];
    const c10::cuda::CUDAGuard guard(q.device());
    tensor_list g(6);  // (one for each argument of forward)
    {
      const at::NoGradGuard no_grad;
      MfDenseAttnArgs a{};
      fill(a, t, call);
      Tensor go = grad_out[0].to(q.scalar_type());
      if (!(call.heads ? go.is_contiguous() && aligned(go) : rows_ready(go))) go = go.is_contiguous() ? go.clone() : go.contiguous();
      a.out = out.data_ptr(), a.lse = s[kOperands + 1].data_ptr<float>(), a.grad_out = go.const_data_ptr();
      a.out_rows = call.heads ? packed_rows(out, a.head_dim) : rows(out), a.grad_out_rows = call.heads ? packed_rows(go, a.head_dim) : rows(go);
      size_t edge = 0;  // edges of the node are counted over the tensors that were given
      bool wants[4];
      for (int i = Q; i <= BIAS; ++i) wants[i] = t[i].defined() && ctx->needs_input_grad(edge++);
      if (call.heads) {
        if (wants[Q]) {
          const int64_t HD = q.size(2) / 3;
          g[Q] = fresh(q.sizes(), q.scalar_type(), q);
          a.dq = g[Q].data_ptr(), a.dk = static_cast<char*>(a.dq) + 2 * HD, a.dv = static_cast<char*>(a.dq) + 4 * HD;
          a.dq_rows = a.dk_rows = a.dv_rows = packed_rows(q, a.head_dim);
        }
      } else {
        for (int i = Q; i <= V; ++i)
          if (wants[i]) g[i] = like(t[i]);
        if (wants[Q]) a.dq = g[Q].data_ptr(), a.dq_rows = rows(g[Q]);
        if (wants[K]) a.dk = g[K].data_ptr(), a.dk_rows = rows(g[K]);
        if (wants[V]) a.dv = g[V].data_ptr(), a.dv_rows = rows(g[V]);
      }
      if (wants[BIAS]) g[BIAS] = fresh(t[BIAS].sizes(), t[BIAS].scalar_type(), q), a.dbias = g[BIAS].data_ptr();
      const Tensor ws = fresh_bytes(mf_dense_attn_bwd_workspace_bytes(&a), q);
      if (ws.defined()) a.workspace = ws.data_ptr(), a.workspace_bytes = ws.numel();
      check(mf_dense_attn_bwd(&a, c10::cuda::getCurrentCUDAStream().stream()));
    }
    if (at::GradMode::is_enabled()) {  // create_graph: an error for who differentiates again
      tensor_list given;
      for (int i = Q; i <= BIAS; ++i)
        if (g[i].defined()) given.push_back(g[i].set_requires_grad(true));
      const auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that was marked with @once_differentiable",
                                                                        (int64_t)given.size());
      const tensor_list made = (*node)(std::move(given));
      for (int i = Q, j = 0; i <= BIAS; ++i)
        if (g[i].defined()) g[i] = made[j++];
    }
    return g;
  }

  static bool rows_ready(const Tensor& t) {
    if (t.stride(3) != 1 || !aligned(t)) return false;
    for (int d = 0; d < 3; ++d)
      if (t.size(d) > 1 && t.stride(d) % 8) return false;
    return true;
  }
};

// Operands that are ready as they are, nothing that watches; the C ABI checks sizes.
std::optional<Tensor> dense_attention(const Tensor& q, const OptTensor& k, const OptTensor& v, const OptTensor& bias, const OptTensor& buckets,
                                      const OptTensor& num_queries, const OptTensor& num_keys, const OptTensor& key_mask, int64_t heads, bool causal,
                                      std::optional<double> scale, int64_t backend) {
  using D = DenseAttention;
  if (watched() || !q.is_cuda() || (q.scalar_type() != at::kBFloat16 && q.scalar_type() != at::kHalf) || q.numel() == 0) return std::nullopt;
  int64_t B, M, N, H, C;
  if (heads) {
    if (heads < 1 || q.dim() != 3 || q.size(2) % (3 * heads) || !q.is_contiguous() || !aligned(q)) return std::nullopt;
    B = q.size(0), M = N = q.size(1), H = heads, C = q.size(2) / (3 * heads);
  } else {
    if (q.dim() != 4 || !k || !v || k->dim() != 4 || k->sizes() != v->sizes() || k->numel() == 0) return std::nullopt;
    B = q.size(0), M = q.size(2), N = k->size(2), H = q.size(1), C = q.size(3);
    if (k->size(0) != B || k->size(3) != C || H % k->size(1)) return std::nullopt;
    for (const Tensor* t : {&q, &*k, &*v})
      if (t->scalar_type() != q.scalar_type() || t->device() != q.device() || !D::rows_ready(*t)) return std::nullopt;
  }
  if (C != 32 && C != 64 && C != 128) return std::nullopt;
  if (bias.has_value() != buckets.has_value()) return std::nullopt;
  if (bias) {
    if (bias->dim() != 2 || bias->size(1) != H || bias->size(0) < 1 || bias->size(0) > 128 || dtype_code(*bias) < 0 || bias->device() != q.device() || !bias->is_contiguous())
      return std::nullopt;
    const Tensor& w = *buckets;
    if (w.scalar_type() != at::kByte || w.device() != q.device() || w.is_inference()) return std::nullopt;
    if (w.dim() == 1) {
      if (w.size(0) % 2 == 0 || !w.is_contiguous()) return std::nullopt;
    } else if (w.dim() != 3 || (w.size(0) != 1 && w.size(0) != B) || w.size(1) != M || w.size(2) != N || (N > 1 && w.stride(2) != 1)) {
      return std::nullopt;
    }
  }
  for (const OptTensor* n : {&num_queries, &num_keys})
    if (*n && ((*n)->dim() != 1 || (*n)->is_inference() || !ready(**n, q, at::kInt, {B}))) return std::nullopt;
  if (key_mask && (key_mask->is_inference() || !ready(*key_mask, q, at::kBool, {B, N}))) return std::nullopt;
  const double by = scale ? *scale : 1.0 / std::sqrt((double)C);
  if (!std::isfinite(by)) return std::nullopt;
  bool keep = false;
  for (const Tensor* t : {&q, k ? &*k : &q, v ? &*v : &q, bias ? &*bias : &q}) {
    if (t->_fw_grad(0).defined()) return std::nullopt;
    keep = keep || t->requires_grad();
  }
  const Tensor none;
  auto given = [&](const OptTensor& t) { return t ? *t : none; };
  const D::Operands t = {q, given(k), given(v), given(bias), given(buckets), given(num_queries), given(num_keys), given(key_mask)};
  if (!keep || !at::GradMode::is_enabled()) return D::attend(t, DenseCall(heads, backend, causal, false, by), false).out;
  const c10::cuda::CUDAGuard guard(q.device());
  return D::apply(q, k, v, bias, t, c10::make_intrusive<DenseCall>(heads, backend, causal, foreign_leaves({&q, &t[D::K], &t[D::V], &t[D::BIAS]}), by));
}

std::optional<Tensor> distance_buckets(const Tensor& coords, const Tensor& edges, const OptTensor& num_atoms) {
  if (watched() || !coords.is_cuda() || coords.dim() != 3 || coords.size(2) != 3 || coords.scalar_type() != at::kFloat || !coords.is_contiguous() || coords.numel() == 0 ||
      coords._fw_grad(0).defined())
    return std::nullopt;
  if (!edges.device().is_cpu() || edges.scalar_type() != at::kDouble || edges.dim() != 1 || !edges.is_contiguous() || edges.numel() > 127) return std::nullopt;
  const int64_t B = coords.size(0), N = coords.size(1), row = (N + 15) / 16 * 16;
  if (num_atoms && !ready(*num_atoms, coords, at::kInt, {B})) return std::nullopt;
  const c10::cuda::CUDAGuard guard(coords.device());
  const Tensor out = fresh({B, N, row}, at::kByte, coords);
  check(mf_distance_buckets(coords.const_data_ptr<float>(), num_atoms ? num_atoms->const_data_ptr<int32_t>() : nullptr, B, N, edges.const_data_ptr<double>(),
                            edges.numel(), static_cast<uint8_t*>(out.data_ptr()), N * row, row, c10::cuda::getCurrentCUDAStream().stream()));
  const at::AutoDispatchBelowADInplaceOrView guard_view;
  return out.as_strided({B, N, N}, {N * row, row, 1});
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("simplicial_attention", &simplicial_attention);
  m.def("sparse_attention", &sparse_attention);
  m.def("radius_blocks", &radius_blocks);
  m.def("knn_topk", &knn_topk);
  m.def("foreign_leaf", &foreign_leaf);
  m.def("gated_mlp", &gated_mlp);
  m.def("rotary", &rotary);
  m.def("dense_attention", &dense_attention);
  m.def("distance_buckets", &distance_buckets);
  m.def("remember_status", &remember_status);
  m.def("last_status", &last_status);
}
