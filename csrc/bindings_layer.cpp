// torch bindings of the layer operators: gated projection, embedding lookup, windowed attention.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "bindings.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients computed by kernels, for a backward pass that may itself be recorded: they carry an error for whoever
// differentiates them.
template <class Compute>
variable_list once_differentiable(const char* name, Compute compute) {
  const bool recorded = at::GradMode::is_enabled();
  variable_list grads;
  {
    const at::NoGradGuard off;
    grads = compute();
  }
  if (!recorded) return grads;
  variable_list given;
  for (const at::Tensor& t : grads)
    if (t.defined()) given.push_back(t.detach().set_requires_grad(true));
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " can be differentiated once only", (int64_t)given.size());
  const variable_list held = (*error)(std::move(given));
  size_t i = 0;
  for (at::Tensor& t : grads)
    if (t.defined()) t = held[i++];
  return grads;
}

// A pass captured into a CUDA graph cannot hand a gradient to a node of the default stream, and an eager graph that still
// lives keeps such a node for each of its leaves. Refused before anything is recorded: the engine would meet it inside the
// capture, where its failure ends the process.
void check_capture(const char* name, std::initializer_list<const at::Tensor*> inputs) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  for (const at::Tensor* t : inputs) {
    if (!t->requires_grad()) continue;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::impl::gradient_edge(*t).function;
    const auto stream = node ? node->stream() : std::nullopt;
    TORCH_CHECK(!stream || stream->id() != 0, name, ": an eager graph on the default stream still holds an input of this captured pass; "
                "release it (or build it on a stream of its own) before the capture");
  }
}

// Rows that the copy engine can address: unit inner stride, 16-byte aligned rows; anything else is laid out anew.
at::Tensor rows16(const at::Tensor& t) {
  const bool fits = t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1) &&
                    (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1))) &&  // (rows that overlap do not fit)
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
long long row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? (t.size(1) + 7) / 8 * 8 : t.stride(0); }

bool is16(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }

// ---------------------------------------------------------------- gated projection
// x as rows [M, K] that the copy engine can address.
at::Tensor rows_of(const at::Tensor& x, int64_t M, int64_t K) { return rows16(x.dim() == 2 ? x : x.reshape({M, K})); }

// x [..., K], wg / wu [F, K] of one 16-bit type -> h [..., F]; kept: where the projections are wanted for the gradients,
// f32 [2, M, F] with padded rows.
at::Tensor gated_forward(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, int64_t act, at::Tensor* kept) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1 && wg.dim() == 2 && wu.dim() == 2, "x [..., K] and weights [F, K] must be CUDA tensors");
  TORCH_CHECK_VALUE(is16(x), "gated_linear runs in bfloat16 or float16 on CUDA, got ", x.scalar_type());
  for (const at::Tensor* t : {&wg, &wu})
    TORCH_CHECK_VALUE(t->device() == x.device() && t->scalar_type() == x.scalar_type(), "x and the weights must share type and device");
  const int64_t K = x.size(-1), F = wg.size(0);
  TORCH_CHECK_VALUE(wg.size(1) == K && wu.sizes() == wg.sizes(), "weights ", wg.sizes(), " and ", wu.sizes(), " must both be [F, ", K, "]");
  TORCH_CHECK_VALUE(K > 0 && K % 8 == 0 && K < (1 << 30) && F < (1 << 30), "K must be a multiple of 8, got ", K);
  TORCH_CHECK_VALUE(act >= kGluSilu && act <= kGluGeluErf, "unknown activation");
  const c10::cuda::CUDAGuard guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = F;
  at::Tensor h = new_like(x, shape, x.scalar_type());
  const int64_t M = x.numel() / K, Fp = (F + 7) / 8 * 8;
  TORCH_CHECK_VALUE(M < (1ll << 30), "too many rows");
  GluArgs a{};
  if (kept) *kept = new_like(x, {2, M, Fp}, at::kFloat);
  if (M == 0 || F == 0) return h;
  const at::Tensor x2 = rows_of(x, M, K), g2 = rows16(wg), u2 = rows16(wu);
  a.x = x2.data_ptr(), a.ldx = row_stride(x2);
  a.wg = g2.data_ptr(), a.ldwg = row_stride(g2);
  a.wu = u2.data_ptr(), a.ldwu = row_stride(u2);
  a.h = h.data_ptr(), a.ldh = F;
  if (kept) a.g = kept->data_ptr<float>(), a.u = a.g + M * Fp, a.lds = Fp;
  a.M = (int)M, a.K = (int)K, a.F = (int)F, a.act = (int)act;
  a.f16 = x.scalar_type() == at::kHalf;
  a.err = err_ptr();
  at::Tensor ws;
  a.ws_floats = dfl_glu_ws(0, a.M, a.K, a.F);
  if (a.ws_floats) ws = new_like(x, {a.ws_floats}, at::kFloat), a.ws = ws.data_ptr<float>();
  DFL_CHECK_RC(dfl_glu(&a, cur_stream()), "gated_linear");
  return h;
}

// Gradients of gated_linear: {dx, dwg, dwu} (undefined where not needed) from dh and what the forward kept.
variable_list gated_backward(const at::Tensor& dh, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, const at::Tensor& kept,
                             int64_t act, bool need_dx, bool need_dwg, bool need_dwu) {
  const int64_t K = x.size(-1), F = wg.size(0), M = x.numel() / K, Fp = (F + 7) / 8 * 8;
  TORCH_CHECK(dh.device() == x.device() && dh.scalar_type() == x.scalar_type() && dh.numel() == M * F, "the gradient ", dh.sizes(), " ",
              dh.scalar_type(), " does not match the output");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor dx, dwg, dwu;
  if (need_dx) dx = new_like(x, x.sizes(), x.scalar_type());
  if (need_dwg) dwg = new_like(wg, wg.sizes(), x.scalar_type());
  if (need_dwu) dwu = new_like(wu, wu.sizes(), x.scalar_type());
  if (M == 0 || F == 0) {
    for (at::Tensor* t : {&dx, &dwg, &dwu})
      if (t->defined()) t->zero_();
    return {dx, dwg, dwu};
  }
  at::Tensor d2 = dh.dim() == 2 ? dh : dh.reshape({M, F});
  if (F > 1 && (d2.stride(1) != 1 || (M > 1 && d2.stride(0) < F))) d2 = d2.contiguous();
  const at::Tensor dgu = new_like(x, {2, M, Fp}, x.scalar_type());
  GluGradArgs e{};
  e.dh = d2.data_ptr(), e.lddh = M > 1 ? d2.stride(0) : F;
  e.g = kept.data_ptr<float>(), e.u = e.g + M * Fp, e.lds = Fp;
  e.dg = dgu.data_ptr(), e.du = reinterpret_cast<uint16_t*>(e.dg) + M * Fp;
  e.M = M, e.F = (int)F, e.act = (int)act, e.f16 = x.scalar_type() == at::kHalf;
  DFL_CHECK_RC(dfl_glu_grad(&e, cur_stream()), "gated_linear (gradient of the product)");
  const at::Tensor x2 = rows_of(x, M, K), g2 = rows16(wg), u2 = rows16(wu);
  GluGemmArgs a{};
  a.dg = e.dg, a.du = e.du, a.lds = Fp;
  a.x = x2.data_ptr(), a.ldx = row_stride(x2);
  a.wg = g2.data_ptr(), a.ldwg = row_stride(g2);
  a.wu = u2.data_ptr(), a.ldwu = row_stride(u2);
  a.M = (int)M, a.K = (int)K, a.F = (int)F, a.f16 = e.f16;
  a.err = err_ptr();
  at::Tensor ws;  // (one for both products, which run one after the other)
  const int dw = need_dwg && need_dwu ? 2 : 3;
  a.ws_floats = std::max(need_dx ? dfl_glu_ws(1, a.M, a.K, a.F) : 0, need_dwg || need_dwu ? dfl_glu_ws(dw, a.M, a.K, a.F) : 0);
  if (a.ws_floats) ws = new_like(x, {a.ws_floats}, at::kFloat), a.ws = ws.data_ptr<float>();
  if (need_dx) {
    a.dx = dx.data_ptr();
    DFL_CHECK_RC(dfl_glu_dx(&a, cur_stream()), "gated_linear (gradient of x)");
  }
  if (need_dwg || need_dwu) {
    a.dwg = need_dwg ? dwg.data_ptr() : nullptr;
    a.dwu = need_dwu ? dwu.data_ptr() : nullptr;
    DFL_CHECK_RC(dfl_glu_dw(&a, cur_stream()), "gated_linear (gradients of the weights)");
  }
  return {dx, dwg, dwu};
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, int64_t act) {
    at::Tensor kept;
    const at::Tensor h = gated_forward(x, wg, wu, act, &kept);
    ctx->save_for_backward({x, wg, wu, kept});
    ctx->saved_data["act"] = act;
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dh) {
    return once_differentiable("gated_linear", [&]() -> variable_list {
      const variable_list s = ctx->get_saved_variables();
      variable_list d = gated_backward(dh[0], s[0], s[1], s[2], s[3], ctx->saved_data["act"].toInt(), ctx->needs_input_grad(0),
                                       ctx->needs_input_grad(1), ctx->needs_input_grad(2));
      d.emplace_back();
      return d;
    });
  }
};

at::Tensor gated_linear(const at::Tensor& x, const at::Tensor& wg, const at::Tensor& wu, int64_t act) {
  TORCH_CHECK_VALUE(plain_tensors({&x, &wg, &wu}), "the kernel takes no wrapped tensors and no tangents");
  if (at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad())) {
    check_capture("gated_linear", {&x, &wg, &wu});
    return GatedLinear::apply(x, wg, wu, act);
  }
  return gated_forward(x, wg, wu, act, nullptr);
}

// ---------------------------------------------------------------- embedding lookup
at::Tensor integer_ids(const at::Tensor& ids) {  // contiguous int32 or int64
  const bool as_is = ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong;
  return (as_is ? ids : ids.to(at::kLong)).contiguous();
}

// scale * w[ids]: ids of any shape, w [V, D] -> [..., D].
at::Tensor embedding_forward(const at::Tensor& ids, const at::Tensor& w, double scale) {
  TORCH_CHECK_VALUE(w.is_cuda() && w.dim() == 2 && ids.device() == w.device(), "ids and weight [V, D] must be on one CUDA device");
  TORCH_CHECK_VALUE(at::isIntegralType(ids.scalar_type(), false), "ids must be integers, got ", ids.scalar_type());
  EmbedArgs a{};
  a.dtype = dtype_code(w, "weight");
  a.V = w.size(0);
  TORCH_CHECK_VALUE(w.size(1) < (1 << 30), "the rows are too long");
  a.D = (int)w.size(1);
  const c10::cuda::CUDAGuard guard(w.device());
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(a.D);
  at::Tensor y = new_like(w, shape, w.scalar_type());
  if (y.numel() == 0) return y;
  const at::Tensor i = integer_ids(ids), t = w.stride(1) == 1 || a.D == 1 ? w : w.contiguous();
  a.ids = i.data_ptr(), a.id_bytes = (int)i.element_size();
  a.w = t.data_ptr(), a.ldw = t.stride(0);
  a.y = y.data_ptr();
  a.n = i.numel();
  a.scale = (float)scale;
  a.err = err_ptr();
  DFL_CHECK_RC(dfl_embed(&a, cur_stream()), "embedding");
  return y;
}

// Gradient of the above: dy [..., D] for ids -> [V, D]; pad: the row that gets none (-1: every row gets its own).
at::Tensor embedding_grad(const at::Tensor& dy, const at::Tensor& ids, int64_t V, double scale, int64_t pad) {
  TORCH_CHECK_VALUE(dy.is_cuda() && dy.dim() >= 1 && ids.device() == dy.device() && at::isIntegralType(ids.scalar_type(), false),
                    "dy [..., D] and integer ids must be on one CUDA device");
  EmbedGradArgs a{};
  a.dtype = dtype_code(dy, "dy");
  a.n = ids.numel(), a.V = V;
  TORCH_CHECK_VALUE(dy.size(-1) < (1 << 30) && a.n < (1ll << 30) && V < (1ll << 30), "too many ids or rows");
  a.D = (int)dy.size(-1);
  TORCH_CHECK_VALUE(dy.numel() == a.n * a.D, "dy ", dy.sizes(), " does not match ", a.n, " ids");
  const c10::cuda::CUDAGuard guard(dy.device());
  at::Tensor dw = new_like(dy, {V, a.D}, dy.scalar_type());
  if (dw.numel() == 0) return dw;
  if (a.n == 0) return dw.zero_();
  const at::Tensor i = integer_ids(ids), d = dy.contiguous();
  a.ids = i.data_ptr(), a.id_bytes = (int)i.element_size();
  a.dy = d.data_ptr(), a.dw = dw.data_ptr();
  a.scale = (float)scale;
  a.pad = pad;
  a.ws_bytes = dfl_embed_grad_ws(a.n, a.V, a.D);
  const at::Tensor ws = new_like(dy, {a.ws_bytes}, at::kByte);
  a.ws = ws.data_ptr();
  DFL_CHECK_RC(dfl_embed_grad(&a, cur_stream()), "embedding (gradient)");
  return dw;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& ids, const at::Tensor& w, double scale, int64_t pad) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = w.size(0);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["pad"] = pad;
    return embedding_forward(ids, w, scale);
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    return once_differentiable("embedding", [&]() -> variable_list {
      return {at::Tensor(), embedding_grad(dy[0], ctx->get_saved_variables()[0], ctx->saved_data["rows"].toInt(),
                                           ctx->saved_data["scale"].toDouble(), ctx->saved_data["pad"].toInt()), at::Tensor(), at::Tensor()};
    });
  }
};

at::Tensor embedding(const at::Tensor& ids, const at::Tensor& w, double scale, const c10::optional<int64_t>& padding_idx) {
  TORCH_CHECK_VALUE(plain_tensors({&ids, &w}), "the kernel takes no wrapped tensors and no tangents");
  TORCH_CHECK_VALUE(w.dim() == 2, "weight must be [V, D], got ", w.sizes());
  int64_t pad = -1;
  if (padding_idx.has_value()) {
    pad = *padding_idx + (*padding_idx < 0 ? w.size(0) : 0);
    TORCH_CHECK_VALUE(pad >= 0 && pad < w.size(0), "padding_idx ", *padding_idx, " is not a row of ", w.size(0));
  }
  if (at::GradMode::is_enabled() && w.requires_grad()) {
    check_capture("embedding", {&w});
    return Embedding::apply(ids, w, scale, pad);
  }
  return embedding_forward(ids, w, scale);
}

}  // namespace

void bind_layer(py::module_& m) {
  m.def("gated_linear", &gated_linear, py::arg("x"), py::arg("wg"), py::arg("wu"), py::arg("act"));
  m.def("embedding", &embedding, py::arg("ids"), py::arg("w"), py::arg("scale"), py::arg("padding_idx") = py::none());
  m.def("embedding_grad", &embedding_grad, py::arg("dy"), py::arg("ids"), py::arg("V"), py::arg("scale"), py::arg("pad"));
}
