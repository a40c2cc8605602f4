// Operators over rows of vocabulary logits: recording a teacher's top tokens, distilling from them, the acceptance /
// KL objective of a draft head, and verifying drafted tokens. z is a row of V logits (fp32, fp16 or bf16), T the
// temperature, p = softmax(z / T).
//
//   teacher_topk : the k largest logits of a row (ties: lowest id) with their log p.
//   kd_topk      : KL(teacher || student) over the teacher's K tokens and one bin for all others. With pt_k the
//                  teacher's probabilities, ps_k the student's, tt = max(1 - sum pt, 1e-8) and ts = max(student mass
//                  outside the K tokens, 1e-8):
//                    loss = sum_k pt_k (log pt_k - log ps_k) + tt (log tt - log ts)
//                    d loss / d z_v = ([v = id_k] c_k - p_v sum c) / T,  c_k = -pt_k + ps_k tt / ts
//                  (the second term of c_k is 0 where ts sits at its floor). The tail mass is summed over the tokens
//                  outside the K, not taken as 1 - sum ps: a confident student would lose it to cancellation.
//   accept_kl    : q = softmax(draft / T), p = softmax(target / T): alpha = sum_v min(q_v, p_v) (the probability that
//                  a token drawn from q is accepted), kl = KL(p || q);
//                    d alpha / d zq_v = q_v ([q_v <= p_v] - A) / T, A = sum_v q_v [q_v <= p_v]
//                    d kl / d zq_v = (q_v - p_v) / T
//   spec_verify  : draft j of a sequence is accepted while u q_j(d) < p_j(d); at the first rejection the next token
//                  is drawn from the residual max(p - q, 0) (a point-mass draft: p without d), after the last draft
//                  from p. The draw is the exponential race argmin_v -log(u_v) / r_v, which picks the same token as
//                  argmax_v log r_v - log(-log u_v) and needs no normalization of r. Uniforms are the sampler's
//                  counter hash (k_sample.cu). The reference verifies with vLLM's rejection sampler.
//
// A logit at or below -1e30 (-inf, the lowest fp32 / bf16 value) is masked: probability 0. A row with nothing left has
// no distribution: its losses and gradients are 0, its recorded ids -1, its next token -1. Sums, maxima and all
// statistics are fp32 (the teacher's tail mass, a difference from 1, in fp64).
//
// This is the plain form of the kernels: one block per row, one pass over the row per statistic.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace {

#define STREAM at::cuda::getCurrentCUDAStream()

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxK = 128;          // teacher tokens per row
constexpr float kMasked = -1e30f;   // logits at or below are masked
constexpr float kTailFloor = 1e-8f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float masked(float z) { return z <= kMasked ? -INFINITY : z; }

// Block-wide reduction; the result reaches every thread. `sm` holds kWarps values.
template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* sm, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sm[0];
  for (int w = 1; w < kWarps; ++w) v = op(v, sm[w]);
  return v;
}
struct Add { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct MinU64 {
  __device__ unsigned long long operator()(unsigned long long a, unsigned long long b) const { return a < b ? a : b; }
};

// Largest logit of a row (-inf when everything is masked) and sum exp((z - m) / T).
template <typename T>
__device__ float row_max(const T* x, int V, float* sm) {
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += kThreads) m = fmaxf(m, masked(to_f(x[i])));
  return block_reduce(m, sm, Max());
}
template <typename T>
__device__ float row_sum(const T* x, int V, float m, float inv_t, float* sm) {
  float s = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) s += expf((masked(to_f(x[i])) - m) * inv_t);
  return block_reduce(s, sm, Add());
}

// (value, index) pairs ordered by value descending, index ascending, as one increasing 64-bit key.
__device__ __forceinline__ unsigned long long rank_key(float v, uint32_t i) {
  const uint32_t u = __float_as_uint(v + 0.f);   // -0 ranks with +0
  const uint32_t ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)~ord << 32) | i;
}

__device__ __forceinline__ int64_t load_id(const void* ids, bool wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
}

// ------------------------------------------------------------------------------------------- teacher top-k
template <typename T>
__global__ void __launch_bounds__(kThreads) topk_kernel(const T* logits, int64_t ld, int V, int k, float inv_t,
                                                        int32_t* ids, float* lp) {
  __shared__ float sm[kWarps];
  __shared__ unsigned long long sk[kWarps];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  const float m = row_max(x, V, sm);
  const float lse = logf(row_sum(x, V, m, inv_t, sm));
  unsigned long long last = 0;      // keys are > 0: the complement of an ordered -inf is not reached
  for (int j = 0; j < k; ++j) {
    unsigned long long best = ~0ull;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float z = to_f(x[i]);
      const unsigned long long key = rank_key(z, i);
      if (z > kMasked && (j == 0 || key > last) && key < best) best = key;
    }
    best = block_reduce(best, sk, MinU64());
    if (threadIdx.x == 0) {
      const int id = best == ~0ull ? -1 : (int)(uint32_t)best;
      ids[row * k + j] = id;
      lp[row * k + j] = id < 0 ? -INFINITY : (to_f(x[id]) - m) * inv_t - lse;
    }
    if (best == ~0ull) last = ~0ull;
    else last = best;
  }
}

// ------------------------------------------------------------------------------------------- distillation
// Reads a row's teacher entries into shared memory: id (-1 where padded, out of range or repeated), teacher
// probability, student logit. Returns the teacher's tail mass.
template <typename T>
__device__ float load_teacher(const T* x, int V, const void* t_ids, bool wide, const float* t_lp, int64_t row, int K,
                              int* s_id, float* s_pt, float* s_lp, float* s_z, double* s_sum) {
  for (int i = threadIdx.x; i < K; i += kThreads) {
    const int64_t id = load_id(t_ids, wide, row * K + i);
    s_id[i] = id < 0 || id >= V ? -1 : (int)id;
  }
  __syncthreads();
  bool repeated = false;
  if (threadIdx.x < K) {
    const int id = s_id[threadIdx.x];
    for (int j = 0; j < (int)threadIdx.x; ++j) repeated |= s_id[j] == id;
  }
  __syncthreads();
  double pt = 0.0;
  if (threadIdx.x < K) {
    const int i = threadIdx.x;
    if (repeated) s_id[i] = -1;
    const bool ok = s_id[i] >= 0;
    s_lp[i] = ok ? t_lp[row * K + i] : -INFINITY;
    pt = ok ? exp((double)s_lp[i]) : 0.0;
    s_pt[i] = (float)pt;
    s_z[i] = ok ? masked(to_f(x[s_id[i]])) : -INFINITY;
  }
  const double sum = block_reduce(pt, s_sum, Add());
  return (float)fmax(1.0 - sum, (double)kTailFloor);
}

struct KdRow {
  float m, inv_s, ratio, csum;   // max logit, 1 / sum exp, tt / ts (0 at the floor), sum c
};

template <typename T, bool kGrad>
__global__ void __launch_bounds__(kThreads) kd_kernel(const T* logits, int64_t ld, int V, const void* t_ids, bool wide,
                                                      const float* t_lp, int K, float inv_t, const float* weight,
                                                      float* loss, KdRow* stats, T* out, int64_t out_ld) {
  extern __shared__ uint32_t bitmap[];
  __shared__ float sm[kWarps];
  __shared__ double sd[kWarps];
  __shared__ int s_id[kMaxK];
  __shared__ float s_pt[kMaxK], s_lp[kMaxK], s_z[kMaxK];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  for (int i = threadIdx.x; i < (V + 31) / 32; i += kThreads) bitmap[i] = 0;
  const float tt = load_teacher(x, V, t_ids, wide, t_lp, row, K, s_id, s_pt, s_lp, s_z, sd);
  if (threadIdx.x < K && s_id[threadIdx.x] >= 0) atomicOr(&bitmap[s_id[threadIdx.x] >> 5], 1u << (s_id[threadIdx.x] & 31));
  const float m = row_max(x, V, sm);   // ends behind a barrier: the bitmap is complete
  float tail = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads)
    if (!(bitmap[i >> 5] >> (i & 31) & 1)) tail += expf((masked(to_f(x[i])) - m) * inv_t);
  tail = block_reduce(tail, sm, Add());
  float e = 0.f;
  if (threadIdx.x < K) e = expf((s_z[threadIdx.x] - m) * inv_t);
  const float total = tail + block_reduce(e, sm, Add());
  const float inv_s = 1.f / total, ps = e * inv_s;
  const float ts = fmaxf(tail * inv_s, kTailFloor);
  const float ratio = tail * inv_s >= kTailFloor ? tt / ts : 0.f;
  float term = 0.f, c = 0.f;
  if (threadIdx.x < K && s_id[threadIdx.x] >= 0) {
    const float s = (s_z[threadIdx.x] - m) * inv_t - logf(total), pt = s_pt[threadIdx.x];
    term = pt == 0.f ? 0.f : pt * (s_lp[threadIdx.x] - s);
    c = -pt + ratio * ps;
  }
  const float l = block_reduce(term, sm, Add()) + tt * (logf(tt) - logf(ts));
  const float csum = block_reduce(c, sm, Add());
  const bool nothing = m == -INFINITY;
  if (threadIdx.x == 0) {
    loss[row] = nothing ? 0.f : l;
    if (stats) stats[row] = nothing ? KdRow{0.f, 0.f, 0.f, 0.f} : KdRow{m, inv_s, ratio, csum};
  }
  if (!kGrad) return;
  const float w = weight[row] * inv_t;
  T* o = out + row * out_ld;
  for (int i = threadIdx.x; i < V; i += kThreads)
    o[i] = from_f<T>(nothing ? 0.f : -csum * inv_s * w * expf((masked(to_f(x[i])) - m) * inv_t));
  __syncthreads();
  if (threadIdx.x < K && s_id[threadIdx.x] >= 0)
    o[s_id[threadIdx.x]] = from_f<T>(nothing ? 0.f : w * (c - csum * ps));
}

template <typename T>
__global__ void __launch_bounds__(kThreads) kd_bwd_kernel(const T* logits, int64_t ld, int V, const void* t_ids,
                                                          bool wide, const float* t_lp, int K, float inv_t,
                                                          const float* weight, const KdRow* stats, T* out,
                                                          int64_t out_ld) {
  __shared__ double sd[kWarps];
  __shared__ int s_id[kMaxK];
  __shared__ float s_pt[kMaxK], s_lp[kMaxK], s_z[kMaxK];
  const int64_t row = blockIdx.x;
  const T* x = logits + row * ld;
  T* o = out + row * out_ld;
  load_teacher(x, V, t_ids, wide, t_lp, row, K, s_id, s_pt, s_lp, s_z, sd);
  const KdRow st = stats[row];
  const float w = weight[row] * inv_t;
  const bool nothing = st.inv_s == 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads)
    o[i] = from_f<T>(nothing ? 0.f : -st.csum * st.inv_s * w * expf((masked(to_f(x[i])) - st.m) * inv_t));
  __syncthreads();
  if (threadIdx.x < K && s_id[threadIdx.x] >= 0) {
    const float ps = expf((s_z[threadIdx.x] - st.m) * inv_t) * st.inv_s;
    o[s_id[threadIdx.x]] = from_f<T>(nothing ? 0.f : w * (-s_pt[threadIdx.x] + (st.ratio - st.csum) * ps));
  }
}

// ------------------------------------------------------------------------------------------- acceptance and KL
struct AcceptRow {
  float mq, lq, mp, lp, a;       // max and log-sum of both sides, A; lq = -inf marks a row with nothing to compare
};

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_kernel(const T* draft, int64_t ldq, const T* target, int64_t ldp,
                                                          int V, float inv_t, float* alpha, float* kl,
                                                          AcceptRow* stats) {
  __shared__ float sm[kWarps];
  const int64_t row = blockIdx.x;
  const T *xq = draft + row * ldq, *xp = target + row * ldp;
  const float mq = row_max(xq, V, sm), mp = row_max(xp, V, sm);
  const float lq = logf(row_sum(xq, V, mq, inv_t, sm)), lp = logf(row_sum(xp, V, mp, inv_t, sm));
  float a = 0.f, s = 0.f, d = 0.f;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float q = (masked(to_f(xq[i])) - mq) * inv_t - lq, p = (masked(to_f(xp[i])) - mp) * inv_t - lp;
    const float e = expf(fminf(q, p)), ep = expf(p);
    s += e;
    if (q <= p) a += e;
    if (ep != 0.f) d += ep * (p - q);
  }
  s = block_reduce(s, sm, Add());
  a = block_reduce(a, sm, Add());
  d = block_reduce(d, sm, Add());
  const bool nothing = mq == -INFINITY || mp == -INFINITY;
  if (threadIdx.x == 0) {
    alpha[row] = nothing ? 0.f : isnan(lq + lp) ? NAN : s;   // the minimum drops a NaN operand
    kl[row] = nothing ? 0.f : d;
    if (stats) stats[row] = nothing ? AcceptRow{0.f, -INFINITY, 0.f, 0.f, 0.f} : AcceptRow{mq, lq, mp, lp, a};
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_bwd_kernel(const T* draft, int64_t ldq, const T* target, int64_t ldp,
                                                              int V, float inv_t, const AcceptRow* stats,
                                                              const float* g_alpha, const float* g_kl, T* out,
                                                              int64_t out_ld) {
  const int64_t row = blockIdx.x;
  const T *xq = draft + row * ldq, *xp = target + row * ldp;
  T* o = out + row * out_ld;
  const AcceptRow st = stats[row];
  const float ga = g_alpha[row] * inv_t, gk = g_kl[row] * inv_t;
  for (int i = threadIdx.x; i < V; i += kThreads) {
    const float q = (masked(to_f(xq[i])) - st.mq) * inv_t - st.lq, p = (masked(to_f(xp[i])) - st.mp) * inv_t - st.lp;
    const float g = expf(q) * (ga * ((q <= p ? 1.f : 0.f) - st.a) + gk) - gk * expf(p);
    o[i] = from_f<T>(st.lq == -INFINITY ? 0.f : g);
  }
}

// ------------------------------------------------------------------------------------------- draft verification
__device__ __forceinline__ uint32_t hash23(uint64_t base, uint64_t i) {   // the sampler's 23 random bits at index i
  uint64_t z = base + i * 0x8CB92BA72F3D8DD7ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return (uint32_t)((z ^ (z >> 31)) >> 41);
}
__device__ __forceinline__ float unit(uint32_t h) { return ((float)h + 0.5f) * (1.0f / 8388608.0f); }

template <typename T>
__global__ void __launch_bounds__(kThreads) verify_kernel(const T* logits, int64_t lb, int64_t lj, int V, int k,
                                                          const void* drafts, bool wide, const float* temps,
                                                          const int64_t* seeds, const int64_t* steps, const T* draft,
                                                          int64_t qb, int64_t qj, const int32_t* n_draft,
                                                          int32_t* accepted, int32_t* next) {
  __shared__ float sm[kWarps];
  __shared__ unsigned long long sk[kWarps];
  const int64_t b = blockIdx.x;
  const float temp = temps[b];
  const int n = n_draft ? min(max(n_draft[b], 0), k) : k;
  for (int j = 0;; ++j) {
    const T* x = logits + b * lb + j * lj;
    const T* y = draft && j < n ? draft + b * qb + j * qj : nullptr;
    const int64_t d = j < n ? load_id(drafts, wide, b * k + j) : -1;
    const bool known = d >= 0 && d < V;
    if (!(temp > 0.f)) {
      unsigned long long best = ~0ull;
      for (int i = threadIdx.x; i < V; i += kThreads)
        if (to_f(x[i]) > kMasked) best = min(best, rank_key(to_f(x[i]), i));
      best = block_reduce(best, sk, MinU64());
      const int id = best == ~0ull ? -1 : (int)(uint32_t)best;
      if (j < n && known && d == id) continue;
      if (threadIdx.x == 0) {
        accepted[b] = j;
        next[b] = id;
      }
      return;
    }
    const float inv_t = 1.f / temp;
    const uint64_t base = (uint64_t)seeds[b] * 0x9E3779B97F4A7C15ull + (uint64_t)(steps[b] + j) * 0xD1B54A32D192ED03ull + 1ull;
    const float m = row_max(x, V, sm), s = row_sum(x, V, m, inv_t, sm);
    float mq = 0.f, sq = 1.f;
    if (y) {
      mq = row_max(y, V, sm);
      sq = row_sum(y, V, mq, inv_t, sm);
    }
    if (j < n && known) {
      const float u = unit(hash23(base, ~0ull));
      const float pd = expf((masked(to_f(x[d])) - m) * inv_t) / s;
      const float qd = y ? expf((masked(to_f(y[d])) - mq) * inv_t) / sq : 1.f;
      if (u * qd < pd) continue;
    }
    unsigned long long best = ~0ull;
    for (int whole = 0; whole < 2 && best == ~0ull; ++whole) {   // an empty residual leaves p itself
      for (int i = threadIdx.x; i < V; i += kThreads) {
        float r = expf((masked(to_f(x[i])) - m) * inv_t) / s;
        if (!whole && y) r -= expf((masked(to_f(y[i])) - mq) * inv_t) / sq;
        if (!whole && !y && i == d) r = 0.f;
        if (r > 0.f)
          best = min(best, (unsigned long long)__float_as_uint(-logf(unit(hash23(base, i))) / r) << 32 | (uint32_t)i);
      }
      best = block_reduce(best, sk, MinU64());
    }
    if (threadIdx.x == 0) {
      accepted[b] = j;
      next[b] = best == ~0ull ? -1 : (int)(uint32_t)best;
    }
    return;
  }
}

// ------------------------------------------------------------------------------------------- entry points
void check_rows(const torch::Tensor& t, const char* name, int64_t dim) {
  TORCH_CHECK(t.is_cuda() && t.dim() == dim, name, " must be a CUDA tensor of ", dim, " dimensions");
  TORCH_CHECK(t.scalar_type() == torch::kFloat || t.scalar_type() == torch::kHalf || t.scalar_type() == torch::kBFloat16,
              name, " must be fp32, fp16 or bf16");
  TORCH_CHECK(t.size(-1) >= 1 && t.size(-1) <= (1 << 20), name, " must have 1 to 2^20 columns");
  TORCH_CHECK(t.size(-1) == 1 || t.stride(-1) == 1, name, " must have unit stride along the vocabulary");
}
void check_out(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  check_rows(t, name, 2);
  TORCH_CHECK(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && t.device() == like.device(), name,
              " must have the logits' shape, type and device");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must not have overlapping rows");
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
  return (float)(1.0 / t);
}
void launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  TORCH_CHECK(e == cudaSuccess, what, " launch failed: ", cudaGetErrorString(e));
}
template <typename T> const T* cptr(const torch::Tensor& t) { return reinterpret_cast<const T*>(t.data_ptr()); }
template <typename T> T* ptr(const torch::Tensor& t) { return reinterpret_cast<T*>(t.data_ptr()); }

template <typename F>
void by_type(torch::ScalarType ty, F&& f) {
  if (ty == torch::kFloat) f(float());
  else if (ty == torch::kHalf) f(__half());
  else f(__nv_bfloat16());
}

void teacher_topk(torch::Tensor logits, double temp, torch::Tensor ids, torch::Tensor lp) {
  check_rows(logits, "logits", 2);
  TORCH_CHECK(ids.dim() == 2 && ids.size(1) >= 1 && ids.size(1) <= kMaxK, "k must be in [1, ", kMaxK, "]");
  const int64_t n = logits.size(0), k = ids.size(1);
  check_vec(ids, logits, n * k, torch::kInt32, "ids");
  check_vec(lp, logits, n * k, torch::kFloat, "lp");
  const float inv_t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  by_type(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    topk_kernel<T><<<n, kThreads, 0, STREAM>>>(cptr<T>(logits), logits.stride(0), logits.size(1), k, inv_t,
                                               ids.data_ptr<int32_t>(), lp.data_ptr<float>());
  });
  launched("teacher_topk");
}

bool check_kd(const torch::Tensor& logits, const torch::Tensor& t_ids, const torch::Tensor& t_lp) {
  check_rows(logits, "logits", 2);
  const bool wide = check_ids(t_ids, logits, "t_ids");
  TORCH_CHECK(t_ids.size(1) >= 1 && t_ids.size(1) <= kMaxK, "teacher tokens per row must be in [1, ", kMaxK, "]");
  check_vec(t_lp, logits, t_ids.numel(), torch::kFloat, "t_lp");
  return wide;
}
size_t kd_smem(int64_t V, const void* kernel) {
  const size_t bytes = (size_t)(V + 31) / 32 * 4;
  if (bytes > 32768) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    TORCH_CHECK(e == cudaSuccess, "kd_topk shared memory: ", cudaGetErrorString(e));
  }
  return bytes;
}

// loss of each row; with weight and out also out = d sum(weight * loss) / d logits (out may be the logits themselves);
// with stats what kd_topk_bwd needs.
void kd_topk(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp, double temp, torch::Tensor loss,
             c10::optional<torch::Tensor> stats, c10::optional<torch::Tensor> weight, c10::optional<torch::Tensor> out) {
  const bool wide = check_kd(logits, t_ids, t_lp);
  const int64_t n = logits.size(0);
  check_vec(loss, logits, n, torch::kFloat, "loss");
  if (stats) check_vec(*stats, logits, n * 4, torch::kFloat, "stats");
  TORCH_CHECK(weight.has_value() == out.has_value(), "the gradient form takes weight and out together");
  if (weight) check_vec(*weight, logits, n, torch::kFloat, "weight");
  if (out) check_out(*out, logits, "out");
  const float inv_t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  by_type(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    auto kernel = out ? kd_kernel<T, true> : kd_kernel<T, false>;
    const size_t smem = kd_smem(logits.size(1), (const void*)kernel);
    kernel<<<n, kThreads, smem, STREAM>>>(cptr<T>(logits), logits.stride(0), logits.size(1), t_ids.data_ptr(), wide,
                                          t_lp.data_ptr<float>(), t_ids.size(1), inv_t,
                                          weight ? weight->data_ptr<float>() : nullptr, loss.data_ptr<float>(),
                                          stats ? ptr<KdRow>(*stats) : nullptr, out ? ptr<T>(*out) : nullptr,
                                          out ? out->stride(0) : 0);
  });
  launched("kd_topk");
}

void kd_topk_bwd(torch::Tensor logits, torch::Tensor t_ids, torch::Tensor t_lp, double temp, torch::Tensor stats,
                 torch::Tensor weight, torch::Tensor out) {
  const bool wide = check_kd(logits, t_ids, t_lp);
  const int64_t n = logits.size(0);
  check_vec(stats, logits, n * 4, torch::kFloat, "stats");
  check_vec(weight, logits, n, torch::kFloat, "weight");
  check_out(out, logits, "out");
  const float inv_t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(logits.device());
  by_type(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    kd_bwd_kernel<T><<<n, kThreads, 0, STREAM>>>(cptr<T>(logits), logits.stride(0), logits.size(1), t_ids.data_ptr(),
                                                 wide, t_lp.data_ptr<float>(), t_ids.size(1), inv_t,
                                                 weight.data_ptr<float>(), cptr<KdRow>(stats), ptr<T>(out),
                                                 out.stride(0));
  });
  launched("kd_topk_bwd");
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
  if (stats) check_vec(*stats, draft, n * 5, torch::kFloat, "stats");
  const float inv_t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(draft.device());
  by_type(draft.scalar_type(), [&](auto t) {
    using T = decltype(t);
    accept_kernel<T><<<n, kThreads, 0, STREAM>>>(cptr<T>(draft), draft.stride(0), cptr<T>(target), target.stride(0),
                                                 draft.size(1), inv_t, alpha.data_ptr<float>(), kl.data_ptr<float>(),
                                                 stats ? ptr<AcceptRow>(*stats) : nullptr);
  });
  launched("accept_kl");
}

void accept_kl_bwd(torch::Tensor draft, torch::Tensor target, double temp, torch::Tensor stats, torch::Tensor g_alpha,
                   torch::Tensor g_kl, torch::Tensor out) {
  check_pair(draft, target);
  const int64_t n = draft.size(0);
  check_vec(stats, draft, n * 5, torch::kFloat, "stats");
  check_vec(g_alpha, draft, n, torch::kFloat, "g_alpha");
  check_vec(g_kl, draft, n, torch::kFloat, "g_kl");
  check_out(out, draft, "out");
  const float inv_t = check_temp(temp);
  if (!n) return;
  const c10::cuda::CUDAGuard guard(draft.device());
  by_type(draft.scalar_type(), [&](auto t) {
    using T = decltype(t);
    accept_bwd_kernel<T><<<n, kThreads, 0, STREAM>>>(cptr<T>(draft), draft.stride(0), cptr<T>(target), target.stride(0),
                                                     draft.size(1), inv_t, cptr<AcceptRow>(stats),
                                                     g_alpha.data_ptr<float>(), g_kl.data_ptr<float>(), ptr<T>(out),
                                                     out.stride(0));
  });
  launched("accept_kl_bwd");
}

void spec_verify(torch::Tensor logits, torch::Tensor drafts, torch::Tensor temps, torch::Tensor seeds,
                 torch::Tensor steps, c10::optional<torch::Tensor> draft_logits, c10::optional<torch::Tensor> n_draft,
                 torch::Tensor accepted, torch::Tensor next) {
  check_rows(logits, "logits", 3);
  const int64_t B = logits.size(0), k = logits.size(1) - 1;
  TORCH_CHECK(k >= 0 && k <= kMaxK, "drafts per sequence must be in [0, ", kMaxK, "]");
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
  by_type(logits.scalar_type(), [&](auto t) {
    using T = decltype(t);
    verify_kernel<T><<<B, kThreads, 0, STREAM>>>(
        cptr<T>(logits), logits.stride(0), logits.stride(1), logits.size(2), k, drafts.data_ptr(), wide,
        temps.data_ptr<float>(), seeds.data_ptr<int64_t>(), steps.data_ptr<int64_t>(),
        draft_logits && k ? cptr<T>(*draft_logits) : nullptr, draft_logits ? draft_logits->stride(0) : 0,
        draft_logits ? draft_logits->stride(1) : 0, n_draft ? n_draft->data_ptr<int32_t>() : nullptr,
        accepted.data_ptr<int32_t>(), next.data_ptr<int32_t>());
  });
  launched("spec_verify");
}

}  // namespace

void register_vocab(pybind11::module& m) {
  m.def("teacher_topk", &teacher_topk);
  m.def("kd_topk", &kd_topk);
  m.def("kd_topk_bwd", &kd_topk_bwd);
  m.def("accept_kl", &accept_kl);
  m.def("accept_kl_bwd", &accept_kl_bwd);
  m.def("spec_verify", &spec_verify);
}
