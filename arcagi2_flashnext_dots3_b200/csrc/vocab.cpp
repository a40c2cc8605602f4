// torch bindings of the vocabulary-row kernels (k_vocab.cu): argument checks, then one launch call on the current stream.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include "vocab.h"

namespace {

namespace v = fw::vocab;

void check_rows(const torch::Tensor& t, const char* name, int64_t dim) {
  TORCH_CHECK(t.is_cuda() && t.dim() == dim, name, " must be a CUDA tensor of ", dim, " dimensions");
  TORCH_CHECK(t.scalar_type() == torch::kFloat || t.scalar_type() == torch::kHalf || t.scalar_type() == torch::kBFloat16,
              name, " must be fp32, fp16 or bf16");
  TORCH_CHECK(t.size(-1) >= 1 && t.size(-1) <= v::kMaxV, name, " must have 1 to ", v::kMaxV, " columns");
  TORCH_CHECK(t.size(-1) == 1 || t.stride(-1) == 1, name, " must have unit stride along the vocabulary");
  TORCH_CHECK(t.size(0) <= (1 << 26), name, " must have at most 2^26 rows");
}
void check_out(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  check_rows(t, name, 2);
  TORCH_CHECK(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && t.device() == like.device(), name,
              " must have the logits' shape, type and device");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must not have overlapping rows");
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
  TORCH_CHECK(apart, name, " overlaps the logits without being the same rows");
}
void check_vec(const torch::Tensor& t, const torch::Tensor& like, int64_t n, torch::ScalarType ty, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == ty && t.is_contiguous() && t.numel() == n, name,
              " must be a contiguous ", ty, " tensor of ", n, " values on the logits' device");
}
bool check_ids(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.is_contiguous() && t.dim() == 2 && t.size(0) == like.size(0) &&
              (t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64), name,
              " must be contiguous int32 / int64 [rows, ...] on the logits' device");
  return t.scalar_type() == torch::kInt64;
}
float check_temp(double t) {
  TORCH_CHECK(t >= 1e-6 && t <= 1e6, "temperature must be in [1e-6, 1e6], got ", t);
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
float* opt(const c10::optional<torch::Tensor>& t) { return t ? t->data_ptr<float>() : nullptr; }

void teacher_topk(torch::Tensor logits, double temp, torch::Tensor ids, torch::Tensor lp) {
  check_rows(logits, "logits", 2);
  TORCH_CHECK(ids.dim() == 2 && ids.size(1) >= 1 && ids.size(1) <= v::kMaxK, "k must be in [1, ", v::kMaxK, "]");
  const int64_t n = logits.size(0), k = ids.size(1);
  check_vec(ids, logits, n * k, torch::kInt32, "ids");
  check_vec(lp, logits, n * k, torch::kFloat, "lp");
  const float t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor ws = bytes_like(logits, v::teacher_topk_workspace(type_of(logits), rows_of(logits), n, logits.size(1)));
  launched(v::teacher_topk(type_of(logits), rows_of(logits), n, logits.size(1), k, t, ids.data_ptr<int32_t>(),
                           lp.data_ptr<float>(), ws.data_ptr(), at::cuda::getCurrentCUDAStream()),
           "teacher_topk");
}

v::Teacher check_kd(const torch::Tensor& logits, const torch::Tensor& t_ids, const torch::Tensor& t_lp) {
  check_rows(logits, "logits", 2);
  const bool wide = check_ids(t_ids, logits, "t_ids");
  TORCH_CHECK(t_ids.size(1) >= 1 && t_ids.size(1) <= v::kMaxK, "teacher tokens per row must be in [1, ", v::kMaxK, "]");
  check_vec(t_lp, logits, t_ids.numel(), torch::kFloat, "t_lp");
  return {t_ids.data_ptr(), wide, t_lp.data_ptr<float>(), (int)t_ids.size(1)};
}
// loss of each row; with stats what kd_topk_bwd needs
void kd_topk_loss(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp, double temp, torch::Tensor loss,
                  c10::optional<torch::Tensor> stats) {
  const v::Teacher teacher = check_kd(logits, t_ids, t_lp);
  const int64_t n = logits.size(0);
  check_vec(loss, logits, n, torch::kFloat, "loss");
  if (stats) check_vec(*stats, logits, n * v::kKdStats, torch::kFloat, "stats");
  const float t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor ws = bytes_like(logits, v::kd_topk_loss_workspace(type_of(logits), rows_of(logits), n, logits.size(1)));
  launched(v::kd_topk_loss(type_of(logits), rows_of(logits), n, logits.size(1), teacher, t, loss.data_ptr<float>(),
                           opt(stats), ws.data_ptr(), at::cuda::getCurrentCUDAStream()), "kd_topk_loss");
}

// loss of each row and out = d sum(weight * loss) / d logits; out may be the logits themselves
void kd_topk_grad(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp, double temp, torch::Tensor weight,
                  torch::Tensor loss, torch::Tensor out) {
  const v::Teacher teacher = check_kd(logits, t_ids, t_lp);
  const int64_t n = logits.size(0);
  check_vec(loss, logits, n, torch::kFloat, "loss");
  check_vec(weight, logits, n, torch::kFloat, "weight");
  check_out(out, logits, "out");
  const float t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  const torch::Tensor ws = bytes_like(
      logits, v::kd_topk_grad_workspace(type_of(logits), rows_of(logits), n, logits.size(1), teacher.k));
  launched(v::kd_topk_grad(type_of(logits), rows_of(logits), n, logits.size(1), teacher, t, weight.data_ptr<float>(),
                           loss.data_ptr<float>(), out.data_ptr(), out.stride(0), ws.data_ptr(),
                           at::cuda::getCurrentCUDAStream()), "kd_topk_grad");
}

void kd_topk_bwd(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp, double temp, torch::Tensor stats,
                 torch::Tensor weight, torch::Tensor out) {
  const v::Teacher teacher = check_kd(logits, t_ids, t_lp);
  const int64_t n = logits.size(0);
  check_vec(stats, logits, n * v::kKdStats, torch::kFloat, "stats");
  check_vec(weight, logits, n, torch::kFloat, "weight");
  check_out(out, logits, "out");
  const float t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  launched(v::kd_topk_bwd(type_of(logits), rows_of(logits), n, logits.size(1), teacher, t,
                          weight.data_ptr<float>(), stats.data_ptr<float>(), out.data_ptr(), out.stride(0),
                          at::cuda::getCurrentCUDAStream()), "kd_topk_bwd");
}

void check_pair(const torch::Tensor& draft, const torch::Tensor& target) {
  check_rows(draft, "draft logits", 2);
  check_rows(target, "target logits", 2);
  TORCH_CHECK(draft.sizes() == target.sizes() && draft.scalar_type() == target.scalar_type() &&
              draft.device() == target.device(), "draft and target logits must have one shape, type and device");
}

void accept_kl(torch::Tensor draft, torch::Tensor target, double temp, torch::Tensor alpha, torch::Tensor kl,
               c10::optional<torch::Tensor> stats) {
  check_pair(draft, target);
  const int64_t n = draft.size(0);
  check_vec(alpha, draft, n, torch::kFloat, "alpha");
  check_vec(kl, draft, n, torch::kFloat, "kl");
  if (stats) check_vec(*stats, draft, n * v::kAcceptStats, torch::kFloat, "stats");
  const float t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(draft.device());
  launched(v::accept_kl(type_of(draft), rows_of(draft), rows_of(target), n, draft.size(1), t,
                        alpha.data_ptr<float>(), kl.data_ptr<float>(), opt(stats), at::cuda::getCurrentCUDAStream()),
           "accept_kl");
}

void accept_kl_bwd(torch::Tensor draft, torch::Tensor target, double temp, torch::Tensor stats, torch::Tensor g_alpha,
                   torch::Tensor g_kl, torch::Tensor out) {
  check_pair(draft, target);
  const int64_t n = draft.size(0);
  check_vec(stats, draft, n * v::kAcceptStats, torch::kFloat, "stats");
  check_vec(g_alpha, draft, n, torch::kFloat, "g_alpha");
  check_vec(g_kl, draft, n, torch::kFloat, "g_kl");
  check_out(out, draft, "out");
  const float t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(draft.device());
  launched(v::accept_kl_bwd(type_of(draft), rows_of(draft), rows_of(target), n, draft.size(1), t,
                            stats.data_ptr<float>(), g_alpha.data_ptr<float>(), g_kl.data_ptr<float>(), out.data_ptr(),
                            out.stride(0), at::cuda::getCurrentCUDAStream()), "accept_kl_bwd");
}

void spec_verify(torch::Tensor logits, torch::Tensor drafts, torch::Tensor temps, torch::Tensor seeds,
                 torch::Tensor steps, c10::optional<torch::Tensor> draft_logits, c10::optional<torch::Tensor> n_draft,
                 torch::Tensor accepted, torch::Tensor next) {
  check_rows(logits, "logits", 3);
  const int64_t B = logits.size(0), k = logits.size(1) - 1;
  TORCH_CHECK(k >= 0 && k <= v::kMaxK, "drafts per sequence must be in [0, ", v::kMaxK, "]");
  const bool wide = check_ids(drafts, logits, "drafts");
  TORCH_CHECK(drafts.size(1) == k, "drafts must be [B, ", k, "] for logits of ", k + 1, " positions");
  check_vec(temps, logits, B, torch::kFloat, "temps");
  check_vec(seeds, logits, B, torch::kInt64, "seeds");
  check_vec(steps, logits, B, torch::kInt64, "steps");
  if (n_draft) check_vec(*n_draft, logits, B, torch::kInt32, "n_draft");
  if (draft_logits) {
    check_rows(*draft_logits, "draft_logits", 3);
    TORCH_CHECK(draft_logits->size(0) == B && draft_logits->size(1) == k && draft_logits->size(2) == logits.size(2) &&
                draft_logits->scalar_type() == logits.scalar_type() && draft_logits->device() == logits.device(),
                "draft_logits must be [B, k, V] in the logits' type and device");
  }
  check_vec(accepted, logits, B, torch::kInt32, "accepted");
  check_vec(next, logits, B, torch::kInt32, "next");
  if (!B) return;
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
  a.wide = wide;
  a.temps = temps.data_ptr<float>();
  a.seeds = seeds.data_ptr<int64_t>();
  a.steps = steps.data_ptr<int64_t>();
  a.n_draft = n_draft ? n_draft->data_ptr<int32_t>() : nullptr;
  a.accepted = accepted.data_ptr<int32_t>();
  a.next = next.data_ptr<int32_t>();
  const torch::Tensor ws = bytes_like(logits, v::spec_verify_workspace(a));
  a.workspace = ws.data_ptr();
  launched(v::spec_verify(a, at::cuda::getCurrentCUDAStream()), "spec_verify");
}

}  // namespace

void register_vocab(pybind11::module& m) {
  m.attr("kd_stats") = v::kKdStats;
  m.attr("accept_stats") = v::kAcceptStats;
  m.def("teacher_topk", &teacher_topk);
  m.def("kd_topk_loss", &kd_topk_loss);
  m.def("kd_topk_grad", &kd_topk_grad);
  m.def("kd_topk_bwd", &kd_topk_bwd);
  m.def("accept_kl", &accept_kl);
  m.def("accept_kl_bwd", &accept_kl_bwd);
  m.def("spec_verify", &spec_verify);
}
