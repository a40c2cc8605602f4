// Launch interface of the vocabulary-row kernels (k_vocab.cu), bound to torch in vocab.cpp. Every function enqueues on
// `stream` and returns the launch status. Row strides count elements; `type` is the logits' type.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace fw {
namespace vocab {

enum Type { F32 = 0, F16 = 1, BF16 = 2 };

constexpr int kMaxK = 128;       // teacher tokens per row, drafts per sequence
constexpr int kMaxV = 1 << 20;
constexpr int kKdStats = 4;      // floats of per-row state between kd_topk and kd_topk_bwd
constexpr int kAcceptStats = 7;  // floats of per-row state between accept_kl and accept_kl_bwd

struct Logits {
  const void* p;
  int64_t ld;
};

struct Teacher {                 // [rows, k] ids (int32 or int64) and fp32 log-probabilities
  const void* ids;
  bool wide;
  const float* lp;
  int k;
};

// A workspace has the bytes that its ..._workspace() says.
size_t teacher_topk_workspace(Type type, Logits z, int64_t rows, int V);
cudaError_t teacher_topk(Type type, Logits z, int64_t rows, int V, int k, float temp, int32_t* ids, float* lp,
                         void* workspace, cudaStream_t stream);

// stats may be null
size_t kd_topk_loss_workspace(Type type, Logits z, int64_t rows, int V);
cudaError_t kd_topk_loss(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, float* loss, float* stats,
                         void* workspace, cudaStream_t stream);
// loss, and out = d sum(weight loss) / d logits; out may be the logits
size_t kd_topk_grad_workspace(Type type, Logits z, int64_t rows, int V, int k);
cudaError_t kd_topk_grad(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, const float* weight,
                         float* loss, void* out, int64_t out_ld, void* workspace, cudaStream_t stream);
cudaError_t kd_topk_bwd(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, const float* weight,
                        const float* stats, void* out, int64_t out_ld, cudaStream_t stream);

cudaError_t accept_kl(Type type, Logits draft, Logits target, int64_t rows, int V, float temp, float* alpha, float* kl,
                      float* stats, cudaStream_t stream);
cudaError_t accept_kl_bwd(Type type, Logits draft, Logits target, int64_t rows, int V, float temp, const float* stats,
                          const float* g_alpha, const float* g_kl, void* out, int64_t out_ld, cudaStream_t stream);

struct Verify {
  Type type;
  int64_t batch;
  int V, k;
  const void* logits;            // [batch, k + 1, V], strides in elements
  int64_t logits_b, logits_j;
  const void* draft_logits;      // [batch, k, V] or null: point-mass drafts
  int64_t draft_b, draft_j;
  const void* drafts;            // [batch, k]
  bool wide;
  const float* temps;
  const int64_t *seeds, *steps;
  const int32_t* n_draft;        // [batch] or null: k everywhere
  int32_t *accepted, *next;
  void* workspace;               // spec_verify_workspace() bytes
};
size_t spec_verify_workspace(const Verify& a);
cudaError_t spec_verify(const Verify& a, cudaStream_t stream);

}  // namespace vocab
}  // namespace fw
