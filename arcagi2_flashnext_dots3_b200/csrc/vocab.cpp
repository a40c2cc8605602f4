// torch bindings of the vocabulary-row kernels (k_vocab.cu): argument checks, outputs, autograd, and one launch call on the
// current stream. Autograd is done here, not in Python, where a small loss with its gradient took 95 us of host time.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include "vocab.h"

namespace {

namespace v = fw::vocab;

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Logits as the kernels take them: unit stride along the vocabulary.
torch::Tensor check_rows(const torch::Tensor& t, const char* name, int64_t dim) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.dim() == dim, name, " must be a CUDA tensor of ", dim, " dimensions");
  TORCH_CHECK_VALUE(t.scalar_type() == torch::kFloat || t.scalar_type() == torch::kHalf ||
                    t.scalar_type() == torch::kBFloat16, name, " must be fp32, fp16 or bf16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.size(-1) >= 1 && t.size(-1) <= v::kMaxV, name, " must have 1 to ", v::kMaxV, " columns, got ",
                    t.sizes());
  TORCH_CHECK_VALUE(t.size(0) <= (1 << 26), name, " must have at most 2^26 rows");
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
void check_out(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && t.device() == like.device() &&
                    (t.size(1) == 1 || t.stride(1) == 1), name,
                    " must have the logits' shape, type and device and unit stride along the vocabulary");
  TORCH_CHECK_VALUE(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must not have overlapping rows");
  // out may be the logits themselves or lie beside them (also between their rows), not shifted over them
  const int64_t n = t.size(0), V = t.size(1), es = t.element_size();
  if (!n || (t.data_ptr() == like.data_ptr() && (n == 1 || t.stride(0) == like.stride(0)))) return;
  const int64_t d = ((intptr_t)t.data_ptr() - (intptr_t)like.data_ptr()) / es;
  const int64_t span = (n - 1) * t.stride(0) + V, like_span = (n - 1) * like.stride(0) + V;
  bool apart = d >= like_span || -d >= span;
  if (!apart && n > 1 && t.stride(0) == like.stride(0)) {
    const int64_t ld = t.stride(0), r = ((d % ld) + ld) % ld;
    apart = r >= V && ld - r >= V;
  }
  TORCH_CHECK_VALUE(apart, name, " overlaps the logits without being the same rows");
}
torch::Tensor check_vec(const torch::Tensor& t, const torch::Tensor& like, int64_t n, torch::ScalarType ty,
                        const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device() && t.scalar_type() == ty && t.dim() == 1 && t.numel() == n, name,
                    " must be ", ty, " [", n, "] on the logits' device, got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}
torch::Tensor check_ids(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.device() == like.device() && t.dim() == 2 && t.size(0) == like.size(0) &&
                    (t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64), name, " must be int32 or int64 [",
                    like.size(0), ", ...] on the logits' device, got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}
float check_temp(double t) {
  TORCH_CHECK_VALUE(t >= 1e-6 && t <= 1e6, "temperature must be in [1e-6, 1e6], got ", t);
  return (float)t;
}
void launched(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, what, " launch failed: ", cudaGetErrorString(e));
}
v::Type type_of(const torch::Tensor& t) {
  return t.scalar_type() == torch::kFloat ? v::F32 : t.scalar_type() == torch::kHalf ? v::F16 : v::BF16;
}
v::Logits rows_of(const torch::Tensor& t) { return {t.data_ptr(), t.stride(0)}; }
torch::Tensor bytes_like(const torch::Tensor& t, size_t n) {
  return torch::empty({(int64_t)n}, t.options().dtype(torch::kUInt8));
}
torch::Tensor floats_like(const torch::Tensor& t, torch::IntArrayRef shape) {
  return torch::empty(shape, t.options().dtype(torch::kFloat));
}
// What a backward pass returns for an input, with an error in place of its own derivative.
torch::Tensor once(const torch::Tensor& d) {
  if (!torch::GradMode::is_enabled()) return d;
  auto error = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that was marked with once_differentiable", 1);
  return (*error)({d.detach().requires_grad_()})[0];
}

std::tuple<torch::Tensor, torch::Tensor> teacher_topk(torch::Tensor logits, int64_t k, double temp) {
  const torch::NoGradGuard no_grad;
  logits = check_rows(logits, "logits", 2);
  TORCH_CHECK_VALUE(k >= 1 && k <= v::kMaxK, "k must be in [1, ", v::kMaxK, "], got ", k);
  const int64_t n = logits.size(0), V = logits.size(1);
  const float t = check_temp(temp);
  const torch::Tensor ids = torch::empty({n, k}, logits.options().dtype(torch::kInt32)), lp = floats_like(logits, {n, k});
  if (!n) return {ids, lp};
  const c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor ws = bytes_like(logits, v::teacher_topk_workspace(type_of(logits), rows_of(logits), n, V));
  launched(v::teacher_topk(type_of(logits), rows_of(logits), n, V, k, t, ids.data_ptr<int32_t>(), lp.data_ptr<float>(),
                           ws.data_ptr(), at::cuda::getCurrentCUDAStream()),
           "teacher_topk");
  return {ids, lp};
}

// Teacher ids and log-probabilities as the kernels take them
v::Teacher check_kd(const torch::Tensor& logits, torch::Tensor& t_ids, torch::Tensor& t_lp) {
  t_ids = check_ids(t_ids, logits, "teacher ids");
  TORCH_CHECK_VALUE(t_lp.sizes() == t_ids.sizes() && t_lp.device() == logits.device(), "teacher ids ", t_ids.sizes(),
                    " and log-probabilities ", t_lp.sizes(), " must agree in shape and device");
  TORCH_CHECK_VALUE(t_ids.size(1) >= 1 && t_ids.size(1) <= v::kMaxK, "1 to ", v::kMaxK, " teacher tokens per row, got ",
                    t_ids.size(1));
  t_lp = t_lp.detach().to(torch::kFloat).contiguous();
  return {t_ids.data_ptr(), t_ids.scalar_type() == torch::kInt64, t_lp.data_ptr<float>(), (int)t_ids.size(1)};
}
torch::Tensor kd_loss(const torch::Tensor& logits, const v::Teacher& teacher, float t, float* stats) {
  const int64_t n = logits.size(0), V = logits.size(1);
  const torch::Tensor loss = floats_like(logits, {n});
  if (!n) return loss;
  const c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor ws = bytes_like(logits, v::kd_topk_loss_workspace(type_of(logits), rows_of(logits), n, V));
  launched(v::kd_topk_loss(type_of(logits), rows_of(logits), n, V, teacher, t, loss.data_ptr<float>(), stats,
                           ws.data_ptr(), at::cuda::getCurrentCUDAStream()), "kd_topk");
  return loss;
}

struct KdTopK : torch::autograd::Function<KdTopK> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& logits_, torch::Tensor t_ids, torch::Tensor t_lp,
                               double temp) {
    const torch::Tensor logits = check_rows(logits_, "logits", 2);
    const v::Teacher teacher = check_kd(logits, t_ids, t_lp);
    const float t = check_temp(temp);
    const torch::Tensor stats = floats_like(logits, {logits.size(0), v::kKdStats});
    ctx->saved_data["t"] = temp;
    // a copy made for its strides has no gradient of its own, so it may be saved like an input
    ctx->save_for_backward({logits, t_ids, t_lp, stats});
    return kd_loss(logits, teacher, t, stats.data_ptr<float>());
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    torch::Tensor out;
    {
      const torch::NoGradGuard no_grad;
      const torch::Tensor logits = s[0].detach(), weight = g[0].to(torch::kFloat).contiguous();
      const int64_t n = logits.size(0), V = logits.size(1);
      out = torch::empty(logits.sizes(), logits.options());
      if (n) {
        const v::Teacher teacher{s[1].data_ptr(), s[1].scalar_type() == torch::kInt64, s[2].data_ptr<float>(),
                                 (int)s[1].size(1)};
        const c10::cuda::CUDAGuard guard(logits.device());
        launched(v::kd_topk_bwd(type_of(logits), rows_of(logits), n, V, teacher, (float)ctx->saved_data["t"].toDouble(),
                                weight.data_ptr<float>(), s[3].data_ptr<float>(), out.data_ptr(), out.stride(0),
                                at::cuda::getCurrentCUDAStream()), "kd_topk backward");
      }
    }
    return {once(out), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};
torch::Tensor kd_topk(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp, double temp) {
  if (logits.requires_grad() && torch::GradMode::is_enabled()) return KdTopK::apply(logits, t_ids, t_lp, temp);
  const torch::NoGradGuard no_grad;
  logits = check_rows(logits, "logits", 2);
  const v::Teacher teacher = check_kd(logits, t_ids, t_lp);
  return kd_loss(logits, teacher, check_temp(temp), nullptr);
}

// loss of each row and d sum(weight * loss) / d logits, to `out` if given; that may be the logits themselves
std::tuple<torch::Tensor, torch::Tensor> kd_topk_grad(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp,
                                                      torch::Tensor weight, double temp,
                                                      c10::optional<torch::Tensor> out_) {
  const torch::NoGradGuard no_grad;
  logits = check_rows(logits, "logits", 2);
  const v::Teacher teacher = check_kd(logits, t_ids, t_lp);
  const int64_t n = logits.size(0), V = logits.size(1);
  weight = check_vec(weight.to(torch::kFloat), logits, n, torch::kFloat, "weight");
  const torch::Tensor out = out_ ? *out_ : torch::empty(logits.sizes(), logits.options());
  check_out(out, logits, "out");
  const float t = check_temp(temp);
  const torch::Tensor loss = floats_like(logits, {n});
  if (!n) return {loss, out};
  const c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor ws =
      bytes_like(logits, v::kd_topk_grad_workspace(type_of(logits), rows_of(logits), n, V, teacher.k));
  launched(v::kd_topk_grad(type_of(logits), rows_of(logits), n, V, teacher, t, weight.data_ptr<float>(),
                           loss.data_ptr<float>(), out.data_ptr(), out.stride(0), ws.data_ptr(),
                           at::cuda::getCurrentCUDAStream()), "kd_topk_grad");
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();    // what was saved of it is gone
  return {loss, out};
}

void check_pair(torch::Tensor& draft, torch::Tensor& target) {
  TORCH_CHECK_VALUE(draft.sizes() == target.sizes() && draft.scalar_type() == target.scalar_type() &&
                    draft.device() == target.device(), "draft and target logits must agree in shape, type and device: ",
                    draft.sizes(), " ", draft.scalar_type(), " ", draft.device(), " and ", target.sizes(), " ",
                    target.scalar_type(), " ", target.device());
  draft = check_rows(draft, "draft logits", 2);
  target = check_rows(target, "target logits", 2);
}
variable_list accept_rows(const torch::Tensor& draft, const torch::Tensor& target, float t, float* stats) {
  const int64_t n = draft.size(0);
  const torch::Tensor alpha = floats_like(draft, {n}), kl = floats_like(draft, {n});
  if (!n) return {alpha, kl};
  const c10::cuda::CUDAGuard guard(draft.device());
  launched(v::accept_kl(type_of(draft), rows_of(draft), rows_of(target), n, draft.size(1), t, alpha.data_ptr<float>(),
                        kl.data_ptr<float>(), stats, at::cuda::getCurrentCUDAStream()), "accept_kl");
  return {alpha, kl};
}

struct AcceptKl : torch::autograd::Function<AcceptKl> {
  static variable_list forward(AutogradContext* ctx, torch::Tensor draft, torch::Tensor target, double temp) {
    check_pair(draft, target);
    const float t = check_temp(temp);
    const torch::Tensor stats = floats_like(draft, {draft.size(0), v::kAcceptStats});
    ctx->saved_data["t"] = temp;
    ctx->save_for_backward({draft, target, stats});
    return accept_rows(draft, target, t, stats.data_ptr<float>());
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    torch::Tensor out;
    {
      const torch::NoGradGuard no_grad;
      const torch::Tensor draft = s[0].detach(), target = s[1].detach();
      const torch::Tensor g_alpha = g[0].to(torch::kFloat).contiguous(), g_kl = g[1].to(torch::kFloat).contiguous();
      const int64_t n = draft.size(0);
      out = torch::empty(draft.sizes(), draft.options());
      if (n) {
        const c10::cuda::CUDAGuard guard(draft.device());
        launched(v::accept_kl_bwd(type_of(draft), rows_of(draft), rows_of(target), n, draft.size(1),
                                  (float)ctx->saved_data["t"].toDouble(), s[2].data_ptr<float>(), g_alpha.data_ptr<float>(),
                                  g_kl.data_ptr<float>(), out.data_ptr(), out.stride(0),
                                  at::cuda::getCurrentCUDAStream()), "accept_kl backward");
      }
    }
    return {once(out), torch::Tensor(), torch::Tensor()};
  }
};
std::tuple<torch::Tensor, torch::Tensor> accept_kl(torch::Tensor draft, torch::Tensor target, double temp) {
  target = target.detach();
  variable_list r;
  if (draft.requires_grad() && torch::GradMode::is_enabled()) {
    r = AcceptKl::apply(draft, target, temp);
  } else {
    const torch::NoGradGuard no_grad;
    check_pair(draft, target);
    r = accept_rows(draft, target, check_temp(temp), nullptr);
  }
  return {r[0], r[1]};
}

std::tuple<torch::Tensor, torch::Tensor> spec_verify(torch::Tensor logits, torch::Tensor drafts, torch::Tensor temps,
                                                     torch::Tensor seeds, torch::Tensor steps,
                                                     c10::optional<torch::Tensor> draft_logits,
                                                     c10::optional<torch::Tensor> n_draft) {
  const torch::NoGradGuard no_grad;
  logits = check_rows(logits, "logits", 3);
  const int64_t B = logits.size(0), k = logits.size(1) - 1;
  TORCH_CHECK_VALUE(k >= 0 && k <= v::kMaxK, "drafts per sequence must be in [0, ", v::kMaxK, "], got ", k);
  drafts = check_ids(drafts, logits, "drafts");
  TORCH_CHECK_VALUE(drafts.size(1) == k, "drafts must be [B, ", k, "] for logits of ", k + 1, " positions");
  temps = check_vec(temps, logits, B, torch::kFloat, "temps");
  seeds = check_vec(seeds, logits, B, torch::kInt64, "seeds");
  steps = check_vec(steps, logits, B, torch::kInt64, "steps");
  if (n_draft) n_draft = check_vec(*n_draft, logits, B, torch::kInt32, "n_draft");
  if (draft_logits) {
    TORCH_CHECK_VALUE(draft_logits->dim() == 3 && draft_logits->size(0) == B && draft_logits->size(1) == k &&
                      draft_logits->size(2) == logits.size(2) && draft_logits->scalar_type() == logits.scalar_type() &&
                      draft_logits->device() == logits.device(), "draft_logits must be [", B, ", ", k, ", ",
                      logits.size(2), "] in the logits' type and device, got ", draft_logits->scalar_type(), " ",
                      draft_logits->sizes());
    draft_logits = check_rows(*draft_logits, "draft_logits", 3);
  }
  const torch::Tensor accepted = torch::empty({B}, logits.options().dtype(torch::kInt32));
  const torch::Tensor next = torch::empty({B}, logits.options().dtype(torch::kInt32));
  if (!B) return {accepted, next};
  const c10::cuda::CUDAGuard guard(logits.device());
  v::Verify a{};
  a.type = type_of(logits);
  a.batch = B;
  a.V = logits.size(2);
  a.k = k;
  a.logits = logits.data_ptr();
  a.logits_b = logits.stride(0);
  a.logits_j = logits.stride(1);
  if (draft_logits && k) {
    a.draft_logits = draft_logits->data_ptr();
    a.draft_b = draft_logits->stride(0);
    a.draft_j = draft_logits->stride(1);
  }
  a.drafts = drafts.data_ptr();
  a.wide = drafts.scalar_type() == torch::kInt64;
  a.temps = temps.data_ptr<float>();
  a.seeds = seeds.data_ptr<int64_t>();
  a.steps = steps.data_ptr<int64_t>();
  a.n_draft = n_draft ? n_draft->data_ptr<int32_t>() : nullptr;
  a.accepted = accepted.data_ptr<int32_t>();
  a.next = next.data_ptr<int32_t>();
  const torch::Tensor ws = bytes_like(logits, v::spec_verify_workspace(a));
  a.workspace = ws.data_ptr();
  launched(v::spec_verify(a, at::cuda::getCurrentCUDAStream()), "spec_verify");
  return {accepted, next};
}

}  // namespace

void register_vocab(pybind11::module& m) {
  m.def("teacher_topk", &teacher_topk);
  m.def("kd_topk", &kd_topk);
  m.def("kd_topk_grad", &kd_topk_grad);
  m.def("accept_kl", &accept_kl);
  m.def("spec_verify", &spec_verify);
}
