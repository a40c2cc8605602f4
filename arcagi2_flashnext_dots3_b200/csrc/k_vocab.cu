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
// Work split. Every operator reads its logits once and is bound by that stream (and the gradient's), so:
//   * a row is cut into 16-byte vectors over the C blocks of a thread-block cluster, C chosen so that a block's slice
//     fits a few times into an SM's shared memory and few rows still fill the GPU (see plan_of);
//   * a slice is copied asynchronously (cp.async) into shared memory; a thread reads back only the vectors that it
//     copied, so the statistics need no block barrier before them and a second pass over the row costs no memory
//     traffic;
//   * one pass takes the running maximum and sum of a softmax; the blocks of a cluster exchange their sums through
//     distributed shared memory (each writes its part into every peer, one cluster barrier) and each finishes the row
//     statistics by itself, in rank order: bits do not depend on timing;
//   * exp(x) is ex2(x log2 e / T - c) with c = m log2 e / T rounded once and used for the sum and for every
//     probability alike, so that rounding cancels; one FMA and one ex2 per element.
#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "ptx.cuh"
#include "vocab.h"

namespace fw {
namespace vocab {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 16;
constexpr float kTailFloor = 1e-8f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Smallest logit that is not masked, the float after -1e30, and the start of every running maximum: a masked logit's
// ex2 argument against it (or anything above) is hugely negative, so masked logits add exactly 0 and no test is needed.
constexpr float kFloor = -9.9999994e29f;

// ------------------------------------------------------------------------------------------- types
template <typename T> struct Vec;   // the 16-byte vector of T
template <> struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kPad = 0xFF800000u;   // -inf
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ float back(float x) { return x; }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t kPad = 0xFC00FC00u;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(u32_as_h2(w[i]));
      f[2 * i] = p.x;
      f[2 * i + 1] = p.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h2_as_u32(__floats2half2_rn(f[2 * i], f[2 * i + 1]));
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half back(float x) { return __float2half_rn(x); }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t kPad = 0xFF80FF80u;
  static __device__ __forceinline__ void unpack(const uint4& u, float (&f)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 back(float x) { return __float2bfloat16_rn(x); }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A block may write into a peer's shared memory once the peer runs: every block arrives when it starts and waits before
// its first such store.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_peers_run() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 8-byte store to this block's address `p` in the shared memory of cluster rank `rank`
__device__ __forceinline__ void st_peer(const void* p, uint32_t rank, unsigned long long v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned long long as_u64(float a, float b) {
  return (unsigned long long)__float_as_uint(b) << 32 | __float_as_uint(a);
}

// ------------------------------------------------------------------------------------------- slices
// A row seen as 16-byte vectors from the last 16-byte boundary at or before its start: element i is lane (i + phase) %
// N of vector (i + phase) / N. Block `rank` of the cluster owns vectors [first, first + count).
template <typename T>
struct Slice {
  const T* row;
  int V, phase, first, count;
  __device__ __forceinline__ Slice(const T* r, int V_, int per, uint32_t rank) : row(r), V(V_) {
    constexpr int N = Vec<T>::N;
    phase = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    const int total = (V + phase + N - 1) / N;
    first = min((int)rank * per, total);
    count = min(per, total - first);
  }
  __device__ __forceinline__ int start(int v) const { return (first + v) * Vec<T>::N - phase; }   // first element
  __device__ __forceinline__ bool full(int i0) const { return i0 >= 0 && i0 + Vec<T>::N <= V; }
  // the shared-memory place of element i when this block owns it, else -1
  __device__ __forceinline__ int place(int i) const {
    const int at = i + phase - first * Vec<T>::N;
    return at >= 0 && at < count * Vec<T>::N ? at : -1;
  }
};

// Starts the copy of this thread's vectors of elements laid out as in `s`, taken from `row` (the slice's own row or
// another one); out-of-row lanes become -inf. Vectors that `row` does not hold at a 16-byte boundary (the ends of a
// row, a second row with another phase) go through plain loads.
template <typename T>
__device__ __forceinline__ void load_slice(const Slice<T>& s, const T* row, uint4* sm) {
  constexpr int N = Vec<T>::N;
  const bool aligned = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
  for (int v = threadIdx.x; v < s.count; v += kThreads) {
    const int i0 = s.start(v);
    if (aligned && s.full(i0)) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(sm + v)), "l"(row + i0) : "memory");
    } else {
      T* d = reinterpret_cast<T*>(sm + v);
      const uint32_t pad = Vec<T>::kPad;
#pragma unroll
      for (int k = 0; k < N; ++k)
        d[k] = i0 + k >= 0 && i0 + k < s.V ? row[i0 + k] : *reinterpret_cast<const T*>(&pad);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
__device__ __forceinline__ void wait_slices() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// Stores a vector of results: whole when it lies inside the row on a 16-byte boundary of `out`, else by elements.
template <typename T>
__device__ __forceinline__ void store_vec(const Slice<T>& s, T* out, bool aligned, int i0, const float (&f)[Vec<T>::N]) {
  if (aligned && s.full(i0)) {
    *reinterpret_cast<uint4*>(out + i0) = Vec<T>::pack(f);
  } else {
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k)
      if (i0 + k >= 0 && i0 + k < s.V) out[i0 + k] = Vec<T>::back(f[k]);
  }
}

// ------------------------------------------------------------------------------------------- softmax statistics
// sum = sum over elements of 2^(z kl - c), c = (largest z so far) kl, kl = log2(e) / T
struct Soft {
  float c, sum;
};
__device__ __forceinline__ Soft join(Soft a, Soft b) {
  const float c = fmaxf(a.c, b.c);
  return {c, a.sum * ex2(a.c - c) + b.sum * ex2(b.c - c)};
}
__device__ __forceinline__ Soft shfl_xor(Soft a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.c, o), __shfl_xor_sync(0xffffffffu, a.sum, o)};
}

template <int N>
__device__ __forceinline__ float vec_max(const float (&f)[N]) {
  float m = fmaxf(f[0], f[1]);
#pragma unroll
  for (int k = 2; k < N; ++k) m = fmaxf(m, f[k]);
  return m;
}
template <int N>
__device__ __forceinline__ float vec_min(const float (&f)[N]) {
  float m = fminf(f[0], f[1]);
#pragma unroll
  for (int k = 2; k < N; ++k) m = fminf(m, f[k]);
  return m;
}
__device__ __forceinline__ float masked(float z) { return z < kFloor ? -INFINITY : z; }
template <int N>
__device__ __forceinline__ void add_soft(const float (&f)[N], float kl, float& m, Soft& s) {
  const float vm = vec_max(f);
  if (vm > m) {
    m = vm;
    const float c = vm * kl;
    s.sum *= ex2(s.c - c);
    s.c = c;
  }
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    a += ex2(fmaf(f[k], kl, -s.c));
    b += ex2(fmaf(f[k + 1], kl, -s.c));
  }
  s.sum += a + b;
}

template <typename V, typename Op>
__device__ __forceinline__ V warp_reduce(V v, Op op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
struct Add { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };
struct Max { __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct MinKey {
  __device__ __forceinline__ unsigned long long operator()(unsigned long long a, unsigned long long b) const {
    return a < b ? a : b;
  }
};

// (value, index) ordered by value descending, then index ascending, as an increasing 64-bit key; ~0 is no entry.
constexpr unsigned long long kNone = ~0ull;
__device__ __forceinline__ unsigned long long rank_key(float v, uint32_t i) {
  const uint32_t u = __float_as_uint(v + 0.f);   // -0 ranks with +0
  const uint32_t ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)~ord << 32) | i;
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t ord = ~(uint32_t)(key >> 32);
  return __uint_as_float((ord & 0x80000000u) ? (ord ^ 0x80000000u) : ~ord);
}

// The softmax of a whole row from the blocks' parts: block -> cluster. `warp_part` and `part` are this kernel's shared
// scratch ([kWarps], [kMaxCluster]); ends behind a cluster barrier.
__device__ __forceinline__ Soft row_soft(Soft s, uint32_t rank, uint32_t size, unsigned long long* warp_part,
                                         unsigned long long* part) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s = join(s, shfl_xor(s, o));
  if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = as_u64(s.c, s.sum);
  __syncthreads();
  if (threadIdx.x < 32) {
    const unsigned long long w = warp_part[threadIdx.x & (kWarps - 1)];
    s = {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))};
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) s = join(s, shfl_xor(s, o));
    if (threadIdx.x < size) st_peer(part + rank, threadIdx.x, as_u64(s.c, s.sum));
  }
  cluster_sync();
  Soft r{__uint_as_float((uint32_t)part[0]), __uint_as_float((uint32_t)(part[0] >> 32))};
  for (uint32_t i = 1; i < size; ++i)
    r = join(r, Soft{__uint_as_float((uint32_t)part[i]), __uint_as_float((uint32_t)(part[i] >> 32))});
  return r;
}

__device__ __forceinline__ int load_id(const Teacher& t, int64_t i, int V) {
  const int64_t id = t.wide ? static_cast<const int64_t*>(t.ids)[i] : (int64_t) static_cast<const int32_t*>(t.ids)[i];
  return id < 0 || id >= V ? -1 : (int)id;
}

// ------------------------------------------------------------------------------------------- teacher top-k
// Each block selects the k best of its slice, the first block of the cluster merges the k-lists. Selection: the k-th
// best of G >= k group maxima (a group: the vectors of kThreads / G threads) is a bound that at least k elements of
// the slice reach and few others do (with k = 20 of 32 groups about 31 of independent values); the elements that reach it
// are collected and ranked by counting. More than kCand of them (long runs of equal logits): k rounds of the smallest
// key above the last, which any input ends in.
constexpr int kCand = 512;

// entries of a sorted list of n keys that are smaller than `key`
__device__ __forceinline__ int below(const unsigned long long* list, int n, unsigned long long key) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] < key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) topk_kernel(const T* logits, int64_t ld, int V, int per, int k, int groups,
                                                        float kl, int32_t* ids, float* lp) {
  constexpr int N = Vec<T>::N;
  extern __shared__ uint4 dyn[];
  __shared__ unsigned long long warp_part[kWarps], part[kMaxCluster], cand[kCand];
  __shared__ float gmax[kThreads];
  __shared__ float s_bound;
  __shared__ int s_count;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t row = blockIdx.x / size;
  cluster_started();
  unsigned long long* mine = reinterpret_cast<unsigned long long*>(dyn + per);   // [k], then [size * k] received
  unsigned long long* recv = mine + k;
  const Slice<T> s(logits + row * ld, V, per, rank);
  load_slice(s, s.row, dyn);
  if (threadIdx.x == 0) s_count = 0;
  wait_slices();
  float m = kFloor;
  Soft soft{kFloor * kl, 0.f};
  float best = -INFINITY;                 // as m, but below kFloor when this thread has nothing
  for (int v = threadIdx.x; v < s.count; v += kThreads) {
    float f[N];
    Vec<T>::unpack(dyn[v], f);
    best = fmaxf(best, vec_max(f));
    add_soft(f, kl, m, soft);
  }
  float gm = best;
  for (int o = kThreads / groups / 2; o; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
  const int lanes = kThreads / groups;
  if (threadIdx.x % lanes == 0) gmax[threadIdx.x / lanes] = gm;
  __syncthreads();
  if (threadIdx.x < groups) {
    const float g = gmax[threadIdx.x];
    int r = 0;
    for (int j = 0; j < groups; ++j) r += gmax[j] > g || (gmax[j] == g && j < (int)threadIdx.x);
    if (r == k - 1) s_bound = fmaxf(g, kFloor);
  }
  __syncthreads();
  const float bound = s_bound;
  if (best >= bound) {
    for (int v = threadIdx.x; v < s.count; v += kThreads) {
      float f[N];
      Vec<T>::unpack(dyn[v], f);
      if (vec_max(f) >= bound) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (f[j] >= bound) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kCand) cand[at] = rank_key(f[j], s.start(v) + j);
          }
      }
    }
  }
  for (int i = threadIdx.x; i < k; i += kThreads) mine[i] = kNone;
  __syncthreads();
  const int n = s_count;
  if (n <= kCand) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned long long key = cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += cand[j] < key;
      if (r < k) mine[r] = key;
    }
  } else {
    unsigned long long last = 0;          // below every key of an unmasked logit
    for (int j = 0; j < k; ++j) {
      unsigned long long b = kNone;
      for (int v = threadIdx.x; v < s.count; v += kThreads) {
        float f[N];
        Vec<T>::unpack(dyn[v], f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const unsigned long long key = rank_key(f[i], s.start(v) + i);
          if (f[i] >= kFloor && key > last && key < b) b = key;
        }
      }
      b = warp_reduce(b, MinKey());
      __syncthreads();
      if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = b;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) b = min(b, warp_part[w]);
      if (threadIdx.x == 0) mine[j] = b;
      last = b;
    }
  }
  __syncthreads();
  cluster_peers_run();
  for (int i = threadIdx.x; i < k; i += kThreads) st_peer(recv + rank * k + i, 0, mine[i]);
  const Soft all = row_soft(soft, rank, size, warp_part, part);
  if (rank != 0) return;
  const float lse = log2f(all.sum);
  int total = 0;
  for (uint32_t l = 0; l < size; ++l) total += below(recv + l * k, k, kNone);
  for (int e = threadIdx.x; e < (int)size * k; e += kThreads) {
    const unsigned long long key = recv[e];
    if (key == kNone) continue;
    int r = 0;
    for (uint32_t l = 0; l < size; ++l) r += below(recv + l * k, k, key);
    if (r < k) {
      ids[row * k + r] = (int32_t)(uint32_t)key;
      lp[row * k + r] = kLn2 * (fmaf(key_value(key), kl, -all.c) - lse);
    }
  }
  for (int i = total + threadIdx.x; i < k; i += kThreads) {
    ids[row * k + i] = -1;
    lp[row * k + i] = -INFINITY;
  }
}

// ------------------------------------------------------------------------------------------- distillation
struct KdRow {
  float c, inv_s, ratio, csum;   // softmax offset and 1 / sum (0: nothing in the row), tt / ts (0 at the floor), sum c
};
static_assert(sizeof(KdRow) == kKdStats * 4, "KdRow is what callers allocate");

// Whether entry i of the row's teacher ids repeats an earlier one.
__device__ __forceinline__ bool repeats(const int* ids, int i) {
  bool r = false;
  for (int j = 0; j < i; ++j) r |= ids[j] == ids[i];
  return r;
}

// One cluster per row. The teacher's tokens are replaced by -inf in shared memory once the slice is in, so the pass over
// it sums the tail alone (a confident student's tail is lost in 1 - sum ps) and the gradient pass leaves zeros at them,
// which the owners of the tokens then overwrite. All reads of the row lie before the cluster barrier, all writes behind
// it: out may be the logits.
template <typename T, bool kGrad>
__global__ void __launch_bounds__(kThreads) kd_kernel(const T* logits, int64_t ld, int V, int per, Teacher t, float kl,
                                                      float inv_t, const float* weight, float* loss, KdRow* stats,
                                                      T* out, int64_t out_ld) {
  constexpr int N = Vec<T>::N;
  extern __shared__ uint4 dyn[];
  __shared__ unsigned long long warp_part[kWarps], part[kMaxCluster];
  __shared__ int s_id[kMaxK];
  __shared__ float s_red[3][kMaxK / 32];
  __shared__ double s_mass[kMaxK / 32];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t row = blockIdx.x / size;
  cluster_started();
  const Slice<T> s(logits + row * ld, V, per, rank);
  load_slice(s, s.row, dyn);
  // thread i < K holds teacher entry i
  const int K = t.k, tid = threadIdx.x;
  if (tid < K) s_id[tid] = load_id(t, row * K + tid, V);
  __syncthreads();
  int id = -1;
  float pt = 0.f, tlp = -INFINITY, z = -INFINITY;
  double mass = 0.0;
  if (tid < K && s_id[tid] >= 0 && !repeats(s_id, tid)) {
    id = s_id[tid];
    tlp = t.lp[row * K + tid];
    mass = exp((double)tlp);
    pt = (float)mass;
    z = masked(Vec<T>::one(s.row[id]));
  }
  wait_slices();
  __syncthreads();
  if (id >= 0 && s.place(id) >= 0) {
    const uint32_t pad = Vec<T>::kPad;
    reinterpret_cast<T*>(dyn)[s.place(id)] = *reinterpret_cast<const T*>(&pad);
  }
  if (tid < kMaxK) {
    mass = warp_reduce(mass, Add());
    if ((tid & 31) == 0) s_mass[tid >> 5] = mass;
  }
  __syncthreads();
  float m = kFloor;
  Soft soft{kFloor * kl, 0.f};
  for (int v = tid; v < s.count; v += kThreads) {
    float f[N];
    Vec<T>::unpack(dyn[v], f);
    add_soft(f, kl, m, soft);
  }
  cluster_peers_run();
  const Soft tail = row_soft(soft, rank, size, warp_part, part);
  // offset of the whole row: the teacher's tokens join here
  if (tid < kMaxK) {
    const float zc = warp_reduce(z, Max());
    if ((tid & 31) == 0) s_red[0][tid >> 5] = zc;
  }
  __syncthreads();
  float c = tail.c;
#pragma unroll
  for (int w = 0; w < kMaxK / 32; ++w) c = fmaxf(c, s_red[0][w] * kl);
  const float tail_sum = tail.sum * ex2(tail.c - c);
  const float e = ex2(fmaf(z, kl, -c));
  __syncthreads();
  if (tid < kMaxK) {
    const float es = warp_reduce(e, Add());
    if ((tid & 31) == 0) s_red[0][tid >> 5] = es;
  }
  __syncthreads();
  float total = tail_sum;
#pragma unroll
  for (int w = 0; w < kMaxK / 32; ++w) total += s_red[0][w];
  const bool nothing = total == 0.f;
  const float inv_s = 1.f / total, ps = e * inv_s, ts_raw = tail_sum * inv_s;
  const double tt_raw = 1.0 - (s_mass[0] + s_mass[1] + s_mass[2] + s_mass[3]);
  const float tt = (float)fmax(tt_raw, (double)kTailFloor), ts = ts_raw < kTailFloor ? kTailFloor : ts_raw;
  const float ratio = ts_raw < kTailFloor ? 0.f : tt / ts;
  const float cc = id >= 0 ? fmaf(ratio, ps, -pt) : 0.f;
  const float term = id >= 0 && pt != 0.f ? pt * (tlp - kLn2 * (fmaf(z, kl, -c) - log2f(total))) : 0.f;
  if (tid < kMaxK) {
    const float a = warp_reduce(cc, Add()), b = warp_reduce(term, Add());
    if ((tid & 31) == 0) {
      s_red[1][tid >> 5] = a;
      s_red[2][tid >> 5] = b;
    }
  }
  __syncthreads();
  float csum = 0.f, l = tt * (logf(tt) - logf(ts));
#pragma unroll
  for (int w = 0; w < kMaxK / 32; ++w) {
    csum += s_red[1][w];
    l += s_red[2][w];
  }
  if (rank == 0 && tid == 0) {
    loss[row] = nothing ? 0.f : l;
    if (stats) stats[row] = nothing ? KdRow{0.f, 0.f, 0.f, 0.f} : KdRow{c, inv_s, ratio, csum};
  }
  if (!kGrad) return;
  const float w = nothing ? 0.f : weight[row] * inv_t;
  const float scale = nothing ? 0.f : -csum * inv_s * w;
  T* o = out + row * out_ld;
  const bool aligned = ((reinterpret_cast<uintptr_t>(o) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
  for (int v = tid; v < s.count; v += kThreads) {
    float f[N];
    Vec<T>::unpack(dyn[v], f);
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = scale * ex2(fmaf(f[k], kl, -c));
    store_vec(s, o, aligned, s.start(v), f);
  }
  __syncthreads();
  if (id >= 0 && s.place(id) >= 0) o[id] = Vec<T>::back(nothing ? 0.f : w * fmaf(-csum, ps, cc));
}

// The gradient from saved statistics: nothing to reduce, so a row is cut over independent blocks of `per` vectors.
template <typename T>
__global__ void __launch_bounds__(kThreads) kd_bwd_kernel(const T* logits, int64_t ld, int V, int per, int splits,
                                                          Teacher t, float kl, float inv_t, const float* weight,
                                                          const KdRow* stats, T* out, int64_t out_ld) {
  constexpr int N = Vec<T>::N;
  __shared__ int s_id[kMaxK];
  const int64_t row = blockIdx.x / splits;
  const Slice<T> s(logits + row * ld, V, per, blockIdx.x % splits);
  const KdRow st = stats[row];
  const float w = st.inv_s == 0.f ? 0.f : weight[row] * inv_t, scale = -st.csum * st.inv_s * w;
  T* o = out + row * out_ld;
  const bool aligned = ((reinterpret_cast<uintptr_t>(o) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
  const int tid = threadIdx.x;
  if (tid < t.k) s_id[tid] = load_id(t, row * t.k + tid, V);
#pragma unroll 4
  for (int v = tid; v < s.count; v += kThreads) {
    const int i0 = s.start(v);
    float f[N];
    if (s.full(i0)) {
      Vec<T>::unpack(*reinterpret_cast<const uint4*>(s.row + i0), f);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) f[k] = i0 + k >= 0 && i0 + k < V ? Vec<T>::one(s.row[i0 + k]) : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) f[k] = st.inv_s == 0.f ? 0.f : scale * ex2(fmaf(f[k], kl, -st.c));
    store_vec(s, o, aligned, i0, f);
  }
  __syncthreads();
  if (tid < t.k && s_id[tid] >= 0 && s.place(s_id[tid]) >= 0 && !repeats(s_id, tid)) {
    const int id = s_id[tid];
    const float ps = ex2(fmaf(masked(Vec<T>::one(s.row[id])), kl, -st.c)) * st.inv_s;
    const float pt = (float)exp((double)t.lp[row * t.k + tid]);
    o[id] = Vec<T>::back(st.inv_s == 0.f ? 0.f : w * fmaf(st.ratio - st.csum, ps, -pt));
  }
}

// ------------------------------------------------------------------------------------------- acceptance and KL
// log2 q_v = zq_v kl - bq up to the rounding of bq, whose remainder is in fq = 2^(rounded - exact), and for p alike; a =
// sum_v q_v [q_v <= p_v]. fq = 0 marks a row with nothing to compare.
struct AcceptRow {
  float bq, fq, bp, fp, a;
};
static_assert(sizeof(AcceptRow) == kAcceptStats * 4, "AcceptRow is what callers allocate");

// Both softmaxes and d = sum 2^xp (xp - xq) with xq, xp the ex2 arguments of the elements: KL in bits is then
// d / sum_p + log2 sum_q - log2 sum_p, and no second pass needs the probabilities of p.
struct Pair {
  Soft q, p;
  float d;
};
__device__ __forceinline__ Pair join(const Pair& a, const Pair& b) {
  Pair r;
  r.q = join(a.q, b.q);
  r.p.c = fmaxf(a.p.c, b.p.c);
  const float ea = ex2(a.p.c - r.p.c), eb = ex2(b.p.c - r.p.c);
  r.p.sum = a.p.sum * ea + b.p.sum * eb;
  // the arguments move by the change of their offsets; a part whose weight vanishes adds nothing, even if infinite
  const float da = a.d + a.p.sum * ((a.p.c - r.p.c) - (a.q.c - r.q.c));
  const float db = b.d + b.p.sum * ((b.p.c - r.p.c) - (b.q.c - r.q.c));
  r.d = (ea == 0.f ? 0.f : ea * da) + (eb == 0.f ? 0.f : eb * db);
  return r;
}
__device__ __forceinline__ Pair shfl_xor(const Pair& a, int o) {
  return {shfl_xor(a.q, o), shfl_xor(a.p, o), __shfl_xor_sync(0xffffffffu, a.d, o)};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_kernel(const T* draft, int64_t ldq, const T* target, int64_t ldp,
                                                          int V, int per, float kl, float* alpha, float* out_kl,
                                                          AcceptRow* stats) {
  constexpr int N = Vec<T>::N;
  extern __shared__ uint4 dyn[];
  __shared__ unsigned long long part[kMaxCluster][3], sums[kMaxCluster];
  __shared__ Pair warp_pair[kWarps];
  __shared__ float2 warp_sum[kWarps];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t row = blockIdx.x / size;
  cluster_started();
  uint4* dp = dyn + per;
  const Slice<T> s(draft + row * ldq, V, per, rank);
  load_slice(s, s.row, dyn);
  load_slice(s, target + row * ldp, dp);
  wait_slices();
  const int tid = threadIdx.x;
  float mq = kFloor, mp = kFloor;
  Pair a{{kFloor * kl, 0.f}, {kFloor * kl, 0.f}, 0.f};
  for (int v = tid; v < s.count; v += kThreads) {
    float q[N], p[N];
    Vec<T>::unpack(dyn[v], q);
    Vec<T>::unpack(dp[v], p);
    const float vq = vec_max(q), vp = vec_max(p);
    if (vq > mq || vp > mp) {
      mq = fmaxf(mq, vq);
      mp = fmaxf(mp, vp);
      a = join(a, Pair{{mq * kl, 0.f}, {mp * kl, 0.f}, 0.f});
    }
    if (vec_min(q) < kFloor) {            // a token that only the draft masks makes KL infinite, whatever masks it
#pragma unroll
      for (int k = 0; k < N; ++k) q[k] = masked(q[k]);
    }
    float sq = 0.f, sp = 0.f, d = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float xq = fmaf(q[k], kl, -a.q.c), xp = fmaf(p[k], kl, -a.p.c), ep = ex2(xp);
      sq += ex2(xq);
      sp += ep;
      d += ep > 0.f ? ep * (xp - xq) : 0.f;
    }
    a.q.sum += sq;
    a.p.sum += sp;
    a.d += d;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) a = join(a, shfl_xor(a, o));
  if ((tid & 31) == 0) warp_pair[tid >> 5] = a;
  __syncthreads();
  cluster_peers_run();
  if (tid < 32) {
    a = warp_pair[tid & (kWarps - 1)];
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) a = join(a, shfl_xor(a, o));
    if (tid < (int)size) {
      st_peer(&part[rank][0], tid, as_u64(a.q.c, a.q.sum));
      st_peer(&part[rank][1], tid, as_u64(a.p.c, a.p.sum));
      st_peer(&part[rank][2], tid, as_u64(a.d, 0.f));
    }
  }
  cluster_sync();
  for (uint32_t i = 0; i < size; ++i) {
    const unsigned long long u = part[i][0], w = part[i][1];
    const Pair b{{__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32))},
                 {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))},
                 __uint_as_float((uint32_t)part[i][2])};
    a = i ? join(a, b) : b;
  }
  const double lq = log2((double)a.q.sum), lp = log2((double)a.p.sum);
  const double bq = a.q.c + lq, bp = a.p.c + lp;
  const float rq = (float)bq, rp = (float)bp;
  float below_p = 0.f, above = 0.f;        // sums of min(q, p) where q <= p and where q > p
  for (int v = tid; v < s.count; v += kThreads) {
    float q[N], p[N];
    Vec<T>::unpack(dyn[v], q);
    Vec<T>::unpack(dp[v], p);
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float xq = fmaf(q[k], kl, -rq), xp = fmaf(p[k], kl, -rp), e = ex2(fminf(xq, xp));
      x += xq <= xp ? e : 0.f;
      y += xq <= xp ? 0.f : e;
    }
    below_p += x;
    above += y;
  }
  below_p = warp_reduce(below_p, Add());
  above = warp_reduce(above, Add());
  if ((tid & 31) == 0) warp_sum[tid >> 5] = make_float2(below_p, above);
  __syncthreads();
  if (tid == 0) {
    float2 t = warp_sum[0];
    for (int w = 1; w < kWarps; ++w) {
      t.x += warp_sum[w].x;
      t.y += warp_sum[w].y;
    }
    st_peer(sums + rank, 0, as_u64(t.x, t.y));
  }
  cluster_sync();
  if (rank != 0 || tid != 0) return;
  float x = 0.f, y = 0.f;
  for (uint32_t i = 0; i < size; ++i) {
    x += __uint_as_float((uint32_t)sums[i]);
    y += __uint_as_float((uint32_t)(sums[i] >> 32));
  }
  const bool nothing = a.q.sum == 0.f || a.p.sum == 0.f;
  const float fq = exp2f((float)((double)rq - bq)), fp = exp2f((float)((double)rp - bp));
  const bool nan = isnan(a.q.sum) || isnan(a.p.sum);      // the minimum drops a NaN operand
  alpha[row] = nothing ? 0.f : nan ? NAN : fq * x + fp * y;
  out_kl[row] = nothing ? 0.f : (float)((double)kLn2 * ((double)a.d / a.p.sum + (lq - lp)));
  if (stats) stats[row] = nothing ? AcceptRow{0.f, 0.f, 0.f, 0.f, 0.f} : AcceptRow{rq, fq, rp, fp, fq * x};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) accept_bwd_kernel(const T* draft, int64_t ldq, const T* target, int64_t ldp,
                                                              int V, int per, int splits, float kl, float inv_t,
                                                              const AcceptRow* stats, const float* g_alpha,
                                                              const float* g_kl, T* out, int64_t out_ld) {
  constexpr int N = Vec<T>::N;
  const int64_t row = blockIdx.x / splits;
  const Slice<T> s(draft + row * ldq, V, per, blockIdx.x % splits);
  const T* xp_row = target + row * ldp;
  const AcceptRow st = stats[row];
  const bool nothing = st.fq == 0.f;
  const float ga = g_alpha[row] * inv_t, gk = g_kl[row] * inv_t;
  const float under = st.fq * (ga * (1.f - st.a) + gk), over = st.fq * (gk - ga * st.a), kp = gk * st.fp;
  T* o = out + row * out_ld;
  const bool aligned = ((reinterpret_cast<uintptr_t>(o) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
  const bool same = ((reinterpret_cast<uintptr_t>(xp_row) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
#pragma unroll 2
  for (int v = threadIdx.x; v < s.count; v += kThreads) {
    const int i0 = s.start(v);
    float q[N], p[N];
    if (same && s.full(i0)) {
      Vec<T>::unpack(*reinterpret_cast<const uint4*>(s.row + i0), q);
      Vec<T>::unpack(*reinterpret_cast<const uint4*>(xp_row + i0), p);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const bool in = i0 + k >= 0 && i0 + k < V;
        q[k] = in ? Vec<T>::one(s.row[i0 + k]) : -INFINITY;
        p[k] = in ? Vec<T>::one(xp_row[i0 + k]) : -INFINITY;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float xq = fmaf(q[k], kl, -st.bq), xp = fmaf(p[k], kl, -st.bp);
      q[k] = nothing ? 0.f : ex2(xq) * (xq <= xp ? under : over) - kp * ex2(xp);
    }
    store_vec(s, o, aligned, i0, q);
  }
}

// ------------------------------------------------------------------------------------------- draft verification
// Two launches. The first reduces every needed row of logits, cut over blocks, to softmax parts (T > 0) or to its best
// token (T <= 0). The second, one cluster per sequence and started early by programmatic launch, joins the parts, finds
// the first rejected draft and draws from that position alone: the race costs a hash per token and is run for one row
// of the k + 1. A draw needs -log(u) / r below the best so far; -log(u) >= 1 - u, which is the hash's integer, so the
// logarithm and the division are taken for the few tokens that can win.
constexpr int kDrawThreads = 512;
constexpr int kDrawWarps = kDrawThreads / 32;

__device__ __forceinline__ uint32_t hash23(uint64_t base, uint64_t i) {   // the sampler's 23 random bits at index i
  uint64_t z = base + i * 0x8CB92BA72F3D8DD7ull;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return (uint32_t)(z >> 41);     // the last step, z ^ (z >> 31), leaves bits 33 and up as they are
}
__device__ __forceinline__ float unit(uint32_t h) { return ((float)h + 0.5f) * (1.0f / 8388608.0f); }

__device__ __forceinline__ int drafts_of(const Verify& a, int64_t b) {
  return a.n_draft ? min(max(a.n_draft[b], 0), a.k) : a.k;
}

// parts [batch][2 k + 1 rows: k + 1 of the target, k of the draft][splits], 8 bytes: Soft, or a rank_key
template <typename T, int kUnroll>
__global__ void __launch_bounds__(kThreads) verify_parts_kernel(Verify a, int splits) {
  constexpr int N = Vec<T>::N;
  __shared__ unsigned long long warp_part[kWarps];
  const int rows = a.draft_logits ? 2 * a.k + 1 : a.k + 1;
  const int split = blockIdx.x % splits;
  const int j = (blockIdx.x / splits) % rows;
  const int64_t b = blockIdx.x / splits / rows;
  pdl_launch_dependents();
  const int n = drafts_of(a, b);
  const float temp = a.temps[b];
  const bool draft = j > a.k, greedy = !(temp > 0.f);
  if ((draft ? j - a.k - 1 >= n : j > n) || (draft && greedy)) return;
  const T* row = draft ? static_cast<const T*>(a.draft_logits) + b * a.draft_b + (j - a.k - 1) * a.draft_j
                       : static_cast<const T*>(a.logits) + b * a.logits_b + j * a.logits_j;
  const Slice<T> s(row, a.V, kUnroll * kThreads, split);
  uint4 u[kUnroll];
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const int v = threadIdx.x + i * kThreads, i0 = s.start(v);
    u[i] = make_uint4(Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad);
    if (v < s.count) {
      if (s.full(i0)) {
        u[i] = *reinterpret_cast<const uint4*>(row + i0);
      } else {
        float f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = i0 + k >= 0 && i0 + k < a.V ? Vec<T>::one(row[i0 + k]) : -INFINITY;
        u[i] = Vec<T>::pack(f);
      }
    }
  }
  unsigned long long res;
  if (greedy) {
    res = kNone;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      float f[N];
      Vec<T>::unpack(u[i], f);
      if (vec_max(f) > m) {
        m = vec_max(f);
#pragma unroll
        for (int k = 0; k < N; ++k)
          if (f[k] >= kFloor) res = min(res, rank_key(f[k], s.start(threadIdx.x + i * kThreads) + k));
      }
    }
    res = warp_reduce(res, MinKey());
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = res;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) res = min(res, warp_part[w]);
  } else {
    const float kl = kLog2e / temp;
    float m = kFloor;
    Soft soft{kFloor * kl, 0.f};
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      float f[N];
      Vec<T>::unpack(u[i], f);
      add_soft(f, kl, m, soft);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) soft = join(soft, shfl_xor(soft, o));
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = as_u64(soft.c, soft.sum);
    __syncthreads();
    const unsigned long long w = warp_part[threadIdx.x & (kWarps - 1)];
    soft = {__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))};
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) soft = join(soft, shfl_xor(soft, o));
    res = as_u64(soft.c, soft.sum);
  }
  if (threadIdx.x == 0) static_cast<unsigned long long*>(a.workspace)[blockIdx.x] = res;
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads) verify_draw_kernel(Verify a, int splits, int per) {
  constexpr int N = Vec<T>::N;
  __shared__ Soft s_p[kMaxK + 1], s_q[kMaxK];
  __shared__ unsigned long long s_best[kMaxK + 1];
  __shared__ int s_ok[kMaxK + 1];
  __shared__ unsigned long long warp_best[kDrawWarps], part[2][kMaxCluster];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t b = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31;
  const int rows = a.draft_logits ? 2 * a.k + 1 : a.k + 1;
  pdl_wait();
  const int n = drafts_of(a, b);
  const float temp = a.temps[b];
  const bool greedy = !(temp > 0.f);
  const float kl = greedy ? 1.f : kLog2e / temp;
  const uint64_t seed = (uint64_t)a.seeds[b] * 0x9E3779B97F4A7C15ull + 1ull, step = (uint64_t)a.steps[b];
  const unsigned long long* parts = static_cast<const unsigned long long*>(a.workspace) + b * rows * splits;
  for (int j = tid >> 5; j <= n; j += kDrawWarps) {     // one warp per position
    const int64_t id = j < n ? (a.wide ? static_cast<const int64_t*>(a.drafts)[b * a.k + j]
                                       : (int64_t) static_cast<const int32_t*>(a.drafts)[b * a.k + j])
                             : -1;
    const bool known = id >= 0 && id < a.V;
    if (greedy) {
      unsigned long long best = kNone;
      for (int i = lane; i < splits; i += 32) best = min(best, parts[j * splits + i]);
      best = warp_reduce(best, MinKey());
      if (lane == 0) {
        s_best[j] = best;
        s_ok[j] = known && best != kNone && (uint32_t)best == (uint32_t)id;
      }
      continue;
    }
    const auto whole = [&](int r) {
      Soft t{kFloor * kl, 0.f};
      for (int i = lane; i < splits; i += 32) {
        const unsigned long long w = parts[r * splits + i];
        t = join(t, Soft{__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32))});
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) t = join(t, shfl_xor(t, o));
      return t;
    };
    const Soft p = whole(j), q = a.draft_logits && j < n ? whole(a.k + 1 + j) : Soft{0.f, 1.f};
    if (lane == 0) {
      s_p[j] = p;
      if (j < n) s_q[j] = q;
      bool ok = false;
      if (known) {
        const float zp = Vec<T>::one(static_cast<const T*>(a.logits)[b * a.logits_b + j * a.logits_j + id]);
        const float pd = p.sum > 0.f ? ex2(fmaf(zp, kl, -p.c)) / p.sum : 0.f;
        float qd = 1.f;
        if (a.draft_logits) {
          const float zq = Vec<T>::one(static_cast<const T*>(a.draft_logits)[b * a.draft_b + j * a.draft_j + id]);
          qd = q.sum > 0.f ? ex2(fmaf(zq, kl, -q.c)) / q.sum : 0.f;
        }
        ok = unit(hash23(seed + (step + j) * 0xD1B54A32D192ED03ull, ~0ull)) * qd < pd;
      }
      s_ok[j] = ok;
    }
  }
  __syncthreads();
  int acc = 0;
  while (acc < n && s_ok[acc]) ++acc;
  if (greedy) {
    if (rank == 0 && tid == 0) {
      a.accepted[b] = acc;
      a.next[b] = s_best[acc] == kNone ? -1 : (int)(uint32_t)s_best[acc];
    }
    return;
  }
  cluster_started();
  const T* row = static_cast<const T*>(a.logits) + b * a.logits_b + acc * a.logits_j;
  const T* qrow = a.draft_logits && acc < n ? static_cast<const T*>(a.draft_logits) + b * a.draft_b + acc * a.draft_j : nullptr;
  const int64_t id = acc >= n ? -1 : a.wide ? static_cast<const int64_t*>(a.drafts)[b * a.k + acc]
                                            : (int64_t) static_cast<const int32_t*>(a.drafts)[b * a.k + acc];
  const Slice<T> s(row, a.V, per, rank);
  const Soft p = s_p[acc];
  const float ip = 1.f / p.sum, cq = qrow ? s_q[acc].c : 0.f, iq = qrow && s_q[acc].sum > 0.f ? 1.f / s_q[acc].sum : 0.f;
  const bool same = ((reinterpret_cast<uintptr_t>(qrow) ^ reinterpret_cast<uintptr_t>(row)) & 15) == 0;
  const uint64_t base = seed + (step + acc) * 0xD1B54A32D192ED03ull;
  unsigned long long best = kNone;
  cluster_peers_run();
  for (int whole = acc == n; whole < 2 && best == kNone; ++whole) {   // second round: an empty residual leaves p itself
    float bound = INFINITY;                                           // the best of this warp
    for (int v0 = tid - lane; v0 < s.count; v0 += kDrawThreads) {     // the same trip count for a whole warp
      const int v = v0 + lane, i0 = s.start(v);
      if (v < s.count) {
        float f[N], g[N];
        if (s.full(i0)) {
          Vec<T>::unpack(*reinterpret_cast<const uint4*>(row + i0), f);
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) f[k] = i0 + k >= 0 && i0 + k < a.V ? Vec<T>::one(row[i0 + k]) : -INFINITY;
        }
        if (qrow && !whole) {
          if (same && s.full(i0)) {
            Vec<T>::unpack(*reinterpret_cast<const uint4*>(qrow + i0), g);
          } else {
#pragma unroll
            for (int k = 0; k < N; ++k) g[k] = i0 + k >= 0 && i0 + k < a.V ? Vec<T>::one(qrow[i0 + k]) : -INFINITY;
          }
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
          float r = ex2(fmaf(f[k], kl, -p.c)) * ip;
          if (!whole) {
            if (qrow) r -= ex2(fmaf(g[k], kl, -cq)) * iq;
            else if (i0 + k == id) r = 0.f;
          }
          const uint32_t h = hash23(base, (uint64_t)(uint32_t)(i0 + k));
          const float miss = (float)(8388607u - h) + 0.5f;            // (1 - u) 2^23
          if (r > 0.f && miss * (0.999999f / 8388608.0f) <= bound * r) {
            const float e = -logf(unit(h)) / r;
            best = min(best, (unsigned long long)__float_as_uint(e) << 32 | (uint32_t)(i0 + k));
            bound = fminf(bound, e);
          }
        }
      }
      bound = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(bound)));
    }
    best = warp_reduce(best, MinKey());
    if (lane == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid < 32) {
      best = warp_reduce(warp_best[tid & (kDrawWarps - 1)], MinKey());
      if (tid < (int)size) st_peer(&part[whole][rank], tid, best);
    }
    cluster_sync();
    best = kNone;
    for (uint32_t i = 0; i < size; ++i) best = min(best, part[whole][i]);
  }
  if (rank == 0 && tid == 0) {
    a.accepted[b] = acc;
    a.next[b] = best == kNone ? -1 : (int)(uint32_t)best;
  }
}

// ------------------------------------------------------------------------------------------- launches
int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Blocks per row and vectors per block. `bytes`: of one vector position over all tensors that a block keeps.
struct Plan {
  int cluster, per;
};
Plan plan_of(int64_t rows, int V, int lanes, int bytes) {
  const int total = (V + lanes - 1) / lanes + 1;     // + 1: a row that starts off a boundary
  int c = 1;
  while (c < 8 && (int64_t)total * bytes > (int64_t)c * 40960) c *= 2;
  while (c < kMaxCluster && (int64_t)total * bytes > (int64_t)c * 204800) c *= 2;
  while (c < kMaxCluster && rows * c < sm_count() && total > 2 * kThreads * c) c *= 2;
  return {c, (total + c - 1) / c};
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), int64_t blocks, int threads, int cluster, size_t smem, bool early,
                   cudaStream_t stream, A... args) {
  const void* f = reinterpret_cast<const void*>(kernel);
  cudaError_t e;
  if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (smem > 32768 && (e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess)
    return e;
  if (cluster > 8 && (e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
    return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  attr[n].id = cudaLaunchAttributeClusterDimension;
  attr[n].val.clusterDim.x = cluster;
  attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
  ++n;
  if (early) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

template <typename F>
cudaError_t by_type(Type type, F&& f) {
  if (type == F32) return f(float());
  if (type == F16) return f(__half());
  return f(__nv_bfloat16());
}

constexpr int kBwdVectors = 8;       // vectors per thread of an elementwise gradient block

}  // namespace

cudaError_t teacher_topk(Type type, Logits z, int64_t rows, int V, int k, float inv_t, int32_t* ids, float* lp,
                         cudaStream_t stream) {
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    const Plan p = plan_of(rows, V, Vec<T>::N, 16);
    const int groups = k <= 24 ? 32 : k <= 48 ? 64 : k <= 96 ? 128 : 256;
    return launch(topk_kernel<T>, rows * p.cluster, kThreads, p.cluster, p.per * 16 + (p.cluster + 1) * k * 8, false,
                  stream, static_cast<const T*>(z.p), z.ld, V, p.per, k, groups, kLog2e * inv_t, ids, lp);
  });
}

cudaError_t kd_topk(Type type, Logits z, int64_t rows, int V, Teacher t, float inv_t, const float* weight, float* loss,
                    float* stats, void* out, int64_t out_ld, cudaStream_t stream) {
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    const Plan p = plan_of(rows, V, Vec<T>::N, 16);
    return launch(out ? kd_kernel<T, true> : kd_kernel<T, false>, rows * p.cluster, kThreads, p.cluster, p.per * 16,
                  false, stream, static_cast<const T*>(z.p), z.ld, V, p.per, t, kLog2e * inv_t, inv_t, weight, loss,
                  reinterpret_cast<KdRow*>(stats), static_cast<T*>(out), out_ld);
  });
}

cudaError_t kd_topk_bwd(Type type, Logits z, int64_t rows, int V, Teacher t, float inv_t, const float* weight,
                        const float* stats, void* out, int64_t out_ld, cudaStream_t stream) {
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    const int total = (V + Vec<T>::N - 1) / Vec<T>::N + 1, per = kBwdVectors * kThreads, splits = (total + per - 1) / per;
    return launch(kd_bwd_kernel<T>, rows * splits, kThreads, 1, 0, false, stream, static_cast<const T*>(z.p), z.ld, V,
                  per, splits, t, kLog2e * inv_t, inv_t, weight, reinterpret_cast<const KdRow*>(stats),
                  static_cast<T*>(out), out_ld);
  });
}

cudaError_t accept_kl(Type type, Logits draft, Logits target, int64_t rows, int V, float inv_t, float* alpha, float* kl,
                      float* stats, cudaStream_t stream) {
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    const Plan p = plan_of(rows, V, Vec<T>::N, 32);
    return launch(accept_kernel<T>, rows * p.cluster, kThreads, p.cluster, p.per * 32, false, stream,
                  static_cast<const T*>(draft.p), draft.ld, static_cast<const T*>(target.p), target.ld, V, p.per,
                  kLog2e * inv_t, alpha, kl, reinterpret_cast<AcceptRow*>(stats));
  });
}

cudaError_t accept_kl_bwd(Type type, Logits draft, Logits target, int64_t rows, int V, float inv_t, const float* stats,
                          const float* g_alpha, const float* g_kl, void* out, int64_t out_ld, cudaStream_t stream) {
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    const int total = (V + Vec<T>::N - 1) / Vec<T>::N + 1, per = kBwdVectors * kThreads, splits = (total + per - 1) / per;
    return launch(accept_bwd_kernel<T>, rows * splits, kThreads, 1, 0, false, stream, static_cast<const T*>(draft.p),
                  draft.ld, static_cast<const T*>(target.p), target.ld, V, per, splits, kLog2e * inv_t, inv_t,
                  reinterpret_cast<const AcceptRow*>(stats), g_alpha, g_kl, static_cast<T*>(out), out_ld);
  });
}

namespace {
struct VerifyPlan {
  int unroll, splits, rows;
};
VerifyPlan verify_plan(const Verify& a) {
  const int lanes = a.type == F32 ? 4 : 8, total = (a.V + lanes - 1) / lanes + 1;
  const int rows = a.draft_logits ? 2 * a.k + 1 : a.k + 1;
  const auto splits = [&](int unroll) { return (total + unroll * kThreads - 1) / (unroll * kThreads); };
  const int unroll = a.batch * rows * splits(8) >= 2 * sm_count() ? 8 : 2;
  return {unroll, splits(unroll), rows};
}
}  // namespace

size_t spec_verify_workspace(const Verify& a) {
  const VerifyPlan p = verify_plan(a);
  return (size_t)a.batch * p.rows * p.splits * 8;
}

cudaError_t spec_verify(const Verify& a, cudaStream_t stream) {
  const VerifyPlan p = verify_plan(a);
  return by_type(a.type, [&](auto x) {
    using T = decltype(x);
    cudaError_t e = launch(p.unroll == 8 ? verify_parts_kernel<T, 8> : verify_parts_kernel<T, 2>,
                           a.batch * p.rows * p.splits, kThreads, 1, 0, false, stream, a, p.splits);
    if (e != cudaSuccess) return e;
    const int total = (a.V + Vec<T>::N - 1) / Vec<T>::N + 1;
    int c = 1;
    while (c < kMaxCluster && total > kDrawThreads * c && (c < 8 || a.batch * c < sm_count())) c *= 2;
    return launch(verify_draw_kernel<T>, a.batch * c, kDrawThreads, c, 0, true, stream, a, p.splits, (total + c - 1) / c);
  });
}

}  // namespace vocab
}  // namespace fw
