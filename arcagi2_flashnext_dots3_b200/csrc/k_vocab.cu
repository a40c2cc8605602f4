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
//                    d alpha / d zq_v = q_v (h_v - A) / T, A = sum_v q_v h_v, h = 1 where q < p, 1/2 where q = p, else 0
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
// Work split. Every operator is bound by reading its logits once (and writing the gradient once), so a row is cut into
// units of a few 16-byte vectors per thread that spread over the whole GPU:
//   * forms with one look at the logits (top-k, the loss alone, verification) take a unit per block, straight into
//     registers; a second small kernel, started early, joins the units' parts of a row in order;
//   * gradients from saved statistics are elementwise: a unit per block;
//   * forms that look twice (loss with gradient of more logits than L2 holds, acceptance) give a row to one block, several of
//     which share an SM, or to a cluster of blocks. A block copies as much of its share as fits into shared memory
//     (cp.async, read back only by the thread that copied it) and streams the rest, once for each look: the second time it
//     comes from L2. Nothing is exchanged outside a cluster, whose blocks write their parts into each other's shared
//     memory and finish the row's statistics each by itself, in rank order. One kernel over both looks without clusters,
//     its blocks waiting for the other blocks of their row through global memory, took 276 us where this takes 239
//     (1024 x 151936 fp32), and a loss kernel followed by a gradient kernel 287;
//   * exp(x) is ex2(x log2 e / T - c) with c = m log2 e / T rounded once and used for the sum and for every
//     probability alike, so that rounding cancels; one FMA and one ex2 per element. The offset's rounding stays in range
//     while |z| / T is below 2^30, logits of 1000 at the smallest T (1e-6); verification, whose temperatures come with requests,
//     takes the largest logit off instead.
// Times below are of one B200, GPU time per call with inputs larger than L2, and "of the copy rate" is of 6551 GB/s.
#include <algorithm>
#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "ptx.cuh"
#include "vocab.h"

namespace fw {
namespace vocab {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// Vectors per thread and unit. 16 gained the loss 2% above 1000 rows of 16-bit logits and lost 7% at 333 x 151935; top-k lost
// 10% everywhere, and fp32 never gained.
constexpr int kUnit = 8;
constexpr int kMaxCluster = 16;
constexpr int kRowThreads = 256;     // of the kernels that look twice
constexpr int kRowWarps = kRowThreads / 32;
// Their blocks per SM, and the vectors that a block keeps in shared memory (32 KB over its tensors). One tensor: five blocks of
// 48 registers (three to six blocks are within 1%). Two tensors: four of 64 registers; five blocks spill (508 x 151936 bf16:
// 132 us instead of 118), three are too few to cover the loads (2044 x 32768 fp32: 150 us instead of 136).
constexpr int kRowBlocks = 5;
constexpr int kPairBlocks = 4;
constexpr int kKeep = 2048;
constexpr float kTailFloor = 1e-8f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLog2ed = 1.4426950408889634;
constexpr float kLn2 = 0.6931471805599453f;
constexpr double kLn2d = 0.6931471805599453;
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
  using Pair = __half2;
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
  using Pair = __nv_bfloat162;
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

// Two fp32 operations per instruction.
using Two = unsigned long long;
__device__ __forceinline__ Two two(float a, float b) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ Two two(float a) { return two(a, a); }
__device__ __forceinline__ float2 halves(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Two ex2_two(Two a) {
  const float2 f = halves(a);
  return two(ex2(f.x), ex2(f.y));
}
__device__ __forceinline__ float sum(Two a) {
  const float2 f = halves(a);
  return f.x + f.y;
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
  bool inside;                       // every vector lies whole in the row
  __device__ __forceinline__ Slice(const T* r, int V_, int per, uint32_t rank) : row(r), V(V_) {
    constexpr int N = Vec<T>::N;
    phase = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    const int total = (V + phase + N - 1) / N;
    first = min((int)rank * per, total);
    count = min(per, total - first);
    inside = start(0) >= 0 && start(per - 1) + N <= V;
  }   // rank * per stays below 2^31: V is at most kMaxV
  __device__ __forceinline__ int start(int v) const { return (first + v) * Vec<T>::N - phase; }   // first element
  __device__ __forceinline__ bool full(int i0) const { return i0 >= 0 && i0 + Vec<T>::N <= V; }
  // the place of element i in the slice, -1 when it is not in it
  __device__ __forceinline__ int place(int i) const {
    const int at = i + phase - first * Vec<T>::N;
    return at >= 0 && at < count * Vec<T>::N ? at : -1;
  }
};

// This thread's vectors of `row` at the places of slice `s` (of that row or another one) in registers, -inf where the row
// has no element. Ends of rows, and rows that start on different 16-byte boundaries, go element by element.
template <typename T>
__device__ __forceinline__ uint4 ragged_vec(const Slice<T>& s, const T* row, int i0) {
  constexpr int N = Vec<T>::N;
  float f[N];
#pragma unroll
  for (int k = 0; k < N; ++k) f[k] = i0 + k >= 0 && i0 + k < s.V ? Vec<T>::one(row[i0 + k]) : -INFINITY;
  return Vec<T>::pack(f);
}
template <typename T, int kVec>
__device__ __forceinline__ void load_unit(const Slice<T>& s, const T* row, uint4 (&x)[kVec]) {
  const bool same = ((reinterpret_cast<uintptr_t>(row) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
  const int v = threadIdx.x;
  if (same && s.inside) {
    const uint4* p = reinterpret_cast<const uint4*>(row + s.start(v));
#pragma unroll
    for (int i = 0; i < kVec; ++i) x[i] = __ldcs(p + i * kThreads);
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int i0 = s.start(v + i * kThreads);
    x[i] = same && s.full(i0) ? __ldcs(reinterpret_cast<const uint4*>(row + i0)) : ragged_vec(s, row, i0);
  }
}
template <typename T, int kVec>
__device__ __forceinline__ void load_unit(const Slice<T>& s, uint4 (&x)[kVec]) {
  load_unit(s, s.row, x);
}
// A block's share of a row in the kernels that look twice: `n` whole vectors from element `e0`, which lies on a 16-byte
// boundary, and the elements in front of the row's first boundary and behind its last, which the first and the last block
// of the cluster take one by one. `kept` of the vectors (whole rounds of the block) stay in shared memory.
constexpr int kRound = 4 * kRowThreads;
template <typename T>
struct Share {
  const T* row;
  int e0, n, kept, head, tail0, tail;   // head: [0, head), tail: [tail0, tail0 + tail)
  __device__ __forceinline__ Share(const T* r, int V, uint32_t rank, uint32_t size, int keep) : row(r) {
    constexpr int N = Vec<T>::N;
    const int phase = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    const int lead = min((N - phase) % N, V), all = (V - lead) / N, per = (all + size - 1) / size;
    const int first = min((int)rank * per, all);
    e0 = lead + first * N;
    n = min(per, all - first);
    kept = min(n, keep) / kRound * kRound;
    head = rank == 0 ? lead : 0;
    tail0 = lead + all * N;
    tail = rank == size - 1 ? V - tail0 : 0;
  }
  // the single element of this thread, -1 where it has none
  __device__ __forceinline__ int single() const {
    const int t = threadIdx.x;
    return t < head ? t : t >= 32 && t - 32 < tail ? tail0 + t - 32 : -1;
  }
  __device__ __forceinline__ bool holds(int id) const {
    return (id >= e0 && id < e0 + n * Vec<T>::N) || id < head || (id >= tail0 && id < tail0 + tail);
  }
  // whether element id, held by the block, is in one of this thread's vectors
  __device__ __forceinline__ bool owns(int id) const {
    return id >= e0 && id < e0 + n * Vec<T>::N && (id - e0) / Vec<T>::N % kRowThreads == (int)threadIdx.x;
  }
};
template <typename T>
__device__ __forceinline__ bool same_phase(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}
// Starts the copy of the kept vectors of `row` (the share's own or another one) to sm[v], by the thread that reads them.
template <typename T>
__device__ __forceinline__ void copy_kept(const Share<T>& s, const T* row, uint4* sm) {
  const T* p = row + s.e0 + threadIdx.x * Vec<T>::N;
  if (same_phase(row, s.row)) {
    const uint32_t d = smem_u32(sm + threadIdx.x);
    for (int v = 0; v < s.kept; v += kRound)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + (v + i * kRowThreads) * 16),
                     "l"(p + (v + i * kRowThreads) * Vec<T>::N) : "memory");
  } else {
    for (int v = 0; v < s.kept; v += kRowThreads) {
      T* d = reinterpret_cast<T*>(sm + v + threadIdx.x);
#pragma unroll
      for (int k = 0; k < Vec<T>::N; ++k) d[k] = p[v * Vec<T>::N + k];
    }
  }
}
// Vectors v, v + kRowThreads, .. of the share from memory; -inf past its end.
template <typename T, int kVec>
__device__ __forceinline__ void stream(const Share<T>& s, const T* row, bool same, int v, uint4 (&x)[kVec]) {
  constexpr int N = Vec<T>::N;
  const T* p = row + s.e0 + v * N;
  if (same && v + (kVec - 1) * kRowThreads < s.n) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) x[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i * kRowThreads);
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    x[i] = make_uint4(Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad);
    if (v + i * kRowThreads < s.n) {
      if (same) {
        x[i] = __ldcg(reinterpret_cast<const uint4*>(p) + i * kRowThreads);
      } else {
        T* e = reinterpret_cast<T*>(&x[i]);
#pragma unroll
        for (int k = 0; k < N; ++k) e[k] = p[i * kRowThreads * N + k];
      }
    }
  }
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ void store_ragged(const Slice<T>& s, T* out, int i0, const uint4& u) {
  const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
  for (int k = 0; k < Vec<T>::N; ++k)
    if (i0 + k >= 0 && i0 + k < s.V) out[i0 + k] = e[k];
}
// Stores this thread's vectors f(0), f(1), .. of a unit of results to `out`, laid out as slice `s`.
template <int kVec, typename T, typename F>
__device__ __forceinline__ void store_unit(const Slice<T>& s, T* out, F f) {
  const bool same = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(s.row)) & 15) == 0;
  if (same && s.inside) {
    uint4* p = reinterpret_cast<uint4*>(out + s.start(threadIdx.x));
#pragma unroll
    for (int i = 0; i < kVec; ++i) __stcs(p + i * kThreads, f(i));
    return;
  }
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    const int i0 = s.start(threadIdx.x + i * kThreads);
    if (same && s.full(i0)) *reinterpret_cast<uint4*>(out + i0) = f(i);
    else store_ragged(s, out, i0, f(i));
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
__device__ __forceinline__ Soft as_soft(unsigned long long u) {
  return {__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32))};
}
__device__ __forceinline__ Soft shfl_xor(Soft a, int o) {
  return {__shfl_xor_sync(0xffffffffu, a.c, o), __shfl_xor_sync(0xffffffffu, a.sum, o)};
}

// Extremes of a vector; 16-bit types take them in pairs.
template <typename T>
__device__ __forceinline__ float packed_max(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else {
    using T2 = typename Vec<T>::Pair;
    const T2* p = reinterpret_cast<const T2*>(&u);
    const T2 m = __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
    return fmaxf(Vec<T>::one(m.x), Vec<T>::one(m.y));
  }
}
template <typename T>
__device__ __forceinline__ float packed_min(const uint4& u) {
  if constexpr (sizeof(T) == 4) {
    return fminf(fminf(__uint_as_float(u.x), __uint_as_float(u.y)), fminf(__uint_as_float(u.z), __uint_as_float(u.w)));
  } else {
    using T2 = typename Vec<T>::Pair;
    const T2* p = reinterpret_cast<const T2*>(&u);
    const T2 m = __hmin2(__hmin2(p[0], p[1]), __hmin2(p[2], p[3]));
    return fminf(Vec<T>::one(m.x), Vec<T>::one(m.y));
  }
}
__device__ __forceinline__ float masked(float z) { return z < kFloor ? -INFINITY : z; }
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

// (value, index) ordered by value descending, then index ascending, as an increasing 64-bit key above 0; any NaN ranks above all
// numbers. ~0 is no entry, and key_value of it is a NaN.
constexpr unsigned long long kNone = ~0ull;
constexpr unsigned long long kNanKey = 1ull << 32;
__device__ __forceinline__ unsigned long long rank_key(float v, uint32_t i) {
  if (isnan(v)) return kNanKey | i;
  const uint32_t u = __float_as_uint(v + 0.f);   // -0 ranks with +0
  const uint32_t ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)~ord << 32) | i;
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t ord = ~(uint32_t)(key >> 32);
  return __uint_as_float((ord & 0x80000000u) ? (ord ^ 0x80000000u) : ~ord);
}

template <typename T, int kVec>
__device__ __forceinline__ float unit_max(const uint4 (&x)[kVec]) {
  if constexpr (sizeof(T) == 4) {
    float m = packed_max<T>(x[0]);
#pragma unroll
    for (int i = 1; i < kVec; ++i) m = fmaxf(m, packed_max<T>(x[i]));
    return m;
  } else {
    using T2 = typename Vec<T>::Pair;
    T2 m = *reinterpret_cast<const T2*>(&x[0]);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const T2* p = reinterpret_cast<const T2*>(&x[i]);
      m = __hmax2(m, __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3])));
    }
    return fmaxf(Vec<T>::one(m.x), Vec<T>::one(m.y));
  }
}
// Whether the vectors hold a NaN, which the maxima above drop.
template <typename T, int kVec>
__device__ __forceinline__ bool unit_nan(const uint4 (&x)[kVec]) {
  if constexpr (sizeof(T) == 4) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      float f[4];
      Vec<T>::unpack(x[i], f);
      nan |= isnan(f[0]) | isnan(f[1]) | isnan(f[2]) | isnan(f[3]);
    }
    return nan;
  } else {
    using T2 = typename Vec<T>::Pair;
    T2 m = *reinterpret_cast<const T2*>(&x[0]);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const T2* p = reinterpret_cast<const T2*>(&x[i]);
      m = __hmax2_nan(m, __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3])));
    }
    return isnan(Vec<T>::one(m.x)) || isnan(Vec<T>::one(m.y));
  }
}
// Adds vectors to a thread's running softmax with maximum m; returns their largest logit.
template <typename T, int kVec>
__device__ __forceinline__ float add_soft(const uint4 (&x)[kVec], float kl, float& m, Soft& s) {
  constexpr int N = Vec<T>::N;
  const float vm = unit_max<T>(x);
  if (vm > m) {
    m = vm;
    const float c = vm * kl;
    s.sum *= ex2(s.c - c);
    s.c = c;
  }
  const Two k2 = two(kl), c2 = two(-s.c);
  Two a = two(0.f), b = two(0.f);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    float f[N];
    Vec<T>::unpack(x[i], f);
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      a = add2(a, ex2_two(fma2(two(f[k], f[k + 1]), k2, c2)));
      b = add2(b, ex2_two(fma2(two(f[k + 2], f[k + 3]), k2, c2)));
    }
  }
  s.sum += sum(add2(a, b));
  return vm;
}
// Joins a list of parts over a warp, in an order that depends on their number alone: every lane gets the same bits.
template <typename Load>
__device__ __forceinline__ Soft join_parts(int n, float kl, Load load) {
  Soft t{kFloor * kl, 0.f};
  for (int i = threadIdx.x & 31; i < n; i += 32) t = join(t, as_soft(load(i)));
#pragma unroll
  for (int o = 16; o; o >>= 1) t = join(t, shfl_xor(t, o));
  return t;
}

// Kernels that look once: block (x, y, z) takes unit x of row y + z gridDim.y (neighbouring blocks in neighbouring memory:
// with the rows along x the gradients ran at 93% of the copy rate instead of 100%).
__device__ __forceinline__ int64_t unit_row() { return (int64_t)blockIdx.z * gridDim.y + blockIdx.y; }
__device__ __forceinline__ int64_t unit_index() { return unit_row() * gridDim.x + blockIdx.x; }

__device__ __forceinline__ int load_id(const Teacher& t, int64_t i, int V) {
  const int64_t id = t.wide ? static_cast<const int64_t*>(t.ids)[i] : (int64_t) static_cast<const int32_t*>(t.ids)[i];
  return id < 0 || id >= V ? -1 : (int)id;
}

// ------------------------------------------------------------------------------------------- teacher top-k
// The first kernel reads the logits: softmax parts, and the maximum of each thread's vectors. The second, one block per row,
// selects: the k-th largest of G >= k group maxima (a group: the logits of kThreads / G threads over all units) is a bound
// that at least k values reach and few others do (with k = 20 of 32 groups about 31 of independent values). The vectors
// of threads whose maximum reaches it are read again, one per thread; what reaches it is collected and ranked by counting.
// More than kCand (long runs of equal logits): k rounds of the smallest key above the last, which any input ends in.
// 104 us for 1024 x 151936 fp32 (91% of the copy rate), 119 us for 2048 x 152064 bf16 (80%): the first kernel reads at 106% and 93%
// of the copy rate (89 and 102 us), and the selection of the last rows runs behind it (18 and 23 us by itself). Few rows: 12 us for
// 8 x 151936 fp32, the two kernels' latencies. Selecting in each unit, and joining lists, took 133 and 317 us: the selection's
// barriers then stand between a block's loads and the next block's.
// The selection is held to six blocks per SM: with the registers it takes by itself (47) 2048 rows took 121 us; eight blocks
// spill, 117 us there and 13.8 instead of 12.0 at 8 rows.
constexpr int kCand = 512;

template <typename T>
__global__ void __launch_bounds__(kThreads) topk_units_kernel(const T* logits, int64_t ld, int64_t rows, int V, int width,
                                                              float kl, unsigned long long* parts, float* tops) {
  __shared__ unsigned long long warp_part[kWarps];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  const int64_t row = unit_row();
  if (row >= rows) return;
  const Slice<T> s(logits + row * ld, V, kUnit * kThreads, blockIdx.x);
  float m = kFloor;
  Soft soft{kFloor * kl, 0.f};
  uint4 x[kUnit];
  load_unit(s, x);
  const float top = add_soft<T>(x, kl, m, soft);
  // a NaN (or +inf) among them: to be looked at
  if (tid < width) tops[unit_index() * width + tid] = isnan(soft.sum) ? INFINITY : top;
#pragma unroll
  for (int o = 16; o; o >>= 1) soft = join(soft, shfl_xor(soft, o));
  if ((tid & 31) == 0) warp_part[tid >> 5] = as_u64(soft.c, soft.sum);
  __syncthreads();
  if (tid < 32) {
    const Soft t = join_parts(kWarps, kl, [&](int i) { return warp_part[i]; });
    if (tid == 0) parts[unit_index()] = as_u64(t.c, t.sum);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 6) topk_select_kernel(const T* logits, int64_t ld, int V, int units, int width,
                                                               int k, int groups, float kl, const unsigned long long* parts,
                                                               const float* tops, int32_t* ids, float* lp) {
  constexpr int N = Vec<T>::N;
  __shared__ unsigned long long cand[kCand], warp_key[kWarps];
  __shared__ float gmax[kThreads], s_bound, s_soft[2];
  __shared__ int list[kCand], s_listed, s_count;
  const int tid = threadIdx.x, shift = __ffs(kThreads / groups) - 1;
  const int64_t row = blockIdx.x;
  const Slice<T> s(logits + row * ld, V, V + N, 0);
  tops += row * units * width + tid;
  const int held = tid < width ? units : 0;        // rows of more than one unit have all threads' maxima
  pdl_wait();
  const auto each_top = [&](auto f) {              // f(unit, maximum) for this thread of every unit
    for (int u0 = 0; u0 < held; u0 += 8) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = u0 + i < held ? tops[(u0 + i) * kThreads] : -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) f(u0 + i, x[i]);
    }
  };
  float top = -INFINITY;
  each_top([&](int, float x) { top = fmaxf(top, x); });
  float g = top;
  for (int o = (1 << shift) >> 1; o; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  if ((tid & ((1 << shift) - 1)) == 0) gmax[tid >> shift] = g;
  if (tid == 0) s_listed = s_count = 0;
  __syncthreads();
  if (tid < groups) {
    g = gmax[tid];
    int r = 0;
    for (int j = 0; j < groups; ++j) r += gmax[j] > g || (gmax[j] == g && j < tid);
    if (r == k - 1) s_bound = fmaxf(g, kFloor);    // kFloor: fewer than k groups hold a value, and all are collected
  }
  if (tid >= kThreads - 32) {
    const Soft t = join_parts(units, kl, [&](int i) { return parts[row * units + i]; });
    if (tid == kThreads - 1) {
      s_soft[0] = t.c;
      s_soft[1] = log2f(t.sum);
    }
  }
  __syncthreads();
  const float bound = s_bound;
  if (top >= bound)
    each_top([&](int u, float x) {
      if (x >= bound) {
        const int at = atomicAdd(&s_listed, 1);
        if (at < kCand) list[at] = u << 8 | tid;
      }
    });
  __syncthreads();
  // visits the logits that reach the bound in vector i of the thread and unit `from`
  const auto look = [&](int from, int i, auto visit) {
    const int at = s.start(((from >> 8) * kUnit + i) * kThreads + (from & 255));
    const uint4 x = s.full(at) ? __ldcg(reinterpret_cast<const uint4*>(s.row + at)) : ragged_vec(s, s.row, at);
    float f[N];
    Vec<T>::unpack(x, f);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (!(f[j] < bound)) visit(rank_key(f[j], at + j));          // a NaN too
  };
  const int listed = s_listed;
  if (listed <= kCand)
    for (int i = tid; i < listed * kUnit; i += kThreads)
      look(list[i / kUnit], i % kUnit, [&](unsigned long long key) {
        const int at = atomicAdd(&s_count, 1);
        if (at < kCand) cand[at] = key;
      });
  __syncthreads();
  const auto write = [&](int r, unsigned long long key) {
    ids[row * k + r] = key == kNone ? -1 : (int32_t)(uint32_t)key;
    lp[row * k + r] = key == kNone ? -INFINITY : kLn2 * (fmaf(key_value(key), kl, -s_soft[0]) - s_soft[1]);
  };
  const int n = s_count;
  if (max(n, listed) <= kCand) {
    for (int i = tid; i < n; i += kThreads) {
      const unsigned long long key = cand[i];
      int r = 0;
      for (int j = 0; j < n; ++j) r += cand[j] < key;
      if (r < k) write(r, key);
    }
    for (int i = n + tid; i < k; i += kThreads) write(i, kNone);
    return;
  }
  unsigned long long last = 0;                     // below every key of an unmasked logit
  for (int r = 0; r < k; ++r) {
    unsigned long long b = kNone;
    each_top([&](int u, float x) {
      if (x >= bound)
        for (int i = 0; i < kUnit; ++i)
          look(u << 8 | tid, i, [&](unsigned long long key) {
            if (key > last && key < b) b = key;
          });
    });
    b = warp_reduce(b, MinKey());
    __syncthreads();
    if ((tid & 31) == 0) warp_key[tid >> 5] = b;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) b = min(b, warp_key[w]);
    if (tid == 0) write(r, b);
    last = b;
  }
}

// ------------------------------------------------------------------------------------------- distillation
struct KdRow {
  float c, inv_s, ratio, csum;   // softmax offset and 1 / sum (0: nothing in the row), tt / ts (0 at the floor), sum c
};
struct KdSaved {
  float c, inv_s, pull, csum;    // of a KdRow, and pull_of
};
static_assert(sizeof(KdSaved) == kKdStats * 4, "KdSaved is what callers allocate");

// Whether entry i of the row's teacher ids repeats an earlier one.
__device__ __forceinline__ bool repeats(const int* ids, int i) {
  bool r = false;
  for (int j = 0; j < i; ++j) r |= ids[j] == ids[i];
  return r;
}

constexpr int kE = kMaxK / 32;       // teacher entries per lane: entry lane + 32 i

// Lists the places in a slice of the tokens id[0 .. kE) over one warp; returns their number.
template <typename T>
__device__ __forceinline__ int list_places(const Slice<T>& s, const int (&id)[kE], int* places) {
  int n = 0;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const int place = id[i] < 0 ? -1 : s.place(id[i]);
    const unsigned in = __ballot_sync(0xffffffffu, place >= 0);
    if (place >= 0) places[n + __popc(in & ((1u << (threadIdx.x & 31)) - 1u))] = place;
    n += __popc(in);
  }
  return n;
}

__device__ __forceinline__ void load_ids(const Teacher& t, int64_t row, int V, int (&id)[kE]) {
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    const int j = (threadIdx.x & 31) + 32 * i;
    id[i] = j < t.k ? load_id(t, row * t.k + j, V) : -1;
  }
}

// A row's teacher entries over the lanes of a warp.
struct TeacherRow {
  float lp[kE], pt[kE], z[kE];       // log-probability, probability, student logit (-inf, 0 and -inf where left out)
  unsigned kept;                     // bit i: entry lane + 32 i is in the vocabulary and not repeated
};
template <typename T>
__device__ __forceinline__ void load_entries(const Teacher& t, int64_t row, const T* x, const int (&id)[kE],
                                             float (&lp)[kE], float (&z)[kE]) {
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    lp[i] = id[i] >= 0 ? t.lp[row * t.k + (threadIdx.x & 31) + 32 * i] : -INFINITY;
    z[i] = id[i] >= 0 ? Vec<T>::one(x[id[i]]) : -INFINITY;
  }
}
// `s_id`: kMaxK words of this warp's own.
__device__ __forceinline__ TeacherRow teacher_row(int k, const int (&id)[kE], const float (&lp)[kE], const float (&z)[kE],
                                                  int* s_id) {
  TeacherRow e;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kE; ++i) s_id[lane + 32 * i] = id[i];
  __syncwarp();
  e.kept = 0;
#pragma unroll
  for (int i = 0; i < kE; ++i) {
    e.lp[i] = e.z[i] = -INFINITY;
    e.pt[i] = 0.f;
    if (32 * i < k) {
      if (id[i] >= 0 && !repeats(s_id, lane + 32 * i)) {
        e.lp[i] = lp[i];
        e.z[i] = masked(z[i]);
        e.kept |= 1u << i;
      }
      e.pt[i] = expf(e.lp[i]);
    }
  }
  __syncwarp();
  return e;
}

// What does not depend on the tail: offset and sum of the softmax of the teacher's tokens, sum pt (log pt - log of their
// terms), sum pt, tt and its logarithm. Losses can be small differences of these (a flat teacher leaves nearly all mass in
// the tail), so what only they need is fp64.
struct TeacherSums {
  double l, mass, log_tt;
  float c, es, tt, w;                  // w: the row's weight / T
};
__device__ __forceinline__ TeacherSums teacher_sums(const TeacherRow& e, float kl, int k) {
  TeacherSums r;
  float zm = kFloor;
#pragma unroll
  for (int i = 0; i < kE; ++i) zm = fmaxf(zm, e.z[i]);
  r.c = warp_reduce(zm, Max()) * kl;
  r.es = 0.f;
  r.l = r.mass = 0.0;
#pragma unroll
  for (int i = 0; i < kE; ++i)
    if (32 * i < k) {
      const double pt = exp((double)e.lp[i]);
      r.es += ex2(fmaf(e.z[i], kl, -r.c));
      if (pt != 0.0) r.l += pt * ((double)e.lp[i] - kLn2d * ((double)e.z[i] * kl - r.c));
      r.mass += pt;
    }
  r.es = warp_reduce(r.es, Add());
  r.l = warp_reduce(r.l, Add());
  r.mass = warp_reduce(r.mass, Add());
  const bool floor = 1.0 - r.mass < (double)kTailFloor;
  r.tt = floor ? kTailFloor : (float)(1.0 - r.mass);
  r.log_tt = floor ? log((double)kTailFloor) : log1p(-r.mass);
  r.w = 0.f;
  return r;
}
// Statistics of a row from its tail, the softmax of all but the teacher's tokens.
__device__ __forceinline__ KdRow kd_finish(const TeacherSums& e, const Soft& tail) {
  const float c = fmaxf(tail.c, e.c);
  const float tail_sum = tail.sum * ex2(tail.c - c), es = e.es * ex2(e.c - c), total = tail_sum + es;
  if (total == 0.f) return KdRow{0.f, 0.f, 0.f, 0.f};      // nothing in the row
  const float inv_s = 1.f / total, ts = tail_sum * inv_s, ratio = ts < kTailFloor ? 0.f : e.tt / ts;
  return KdRow{c, inv_s, ratio, ratio * (es * inv_s) - (float)e.mass};
}
// sum pt (log pt - log ps) + tt (log tt - log ts); log ts = -log1p(teacher's / tail's sum) keeps its digits near ts = 1
__device__ __forceinline__ float kd_loss(const TeacherSums& e, const Soft& tail) {
  const float c = fmaxf(tail.c, e.c);
  const float tail_sum = tail.sum * ex2(tail.c - c), es = e.es * ex2(e.c - c);
  const double total = (double)tail_sum + es;
  if (total == 0.0) return 0.f;
  const double log_ts = tail_sum < kTailFloor * total ? log((double)kTailFloor) : -log1p((double)es / tail_sum);
  double l = e.l + e.tt * (e.log_tt - log_ts);
  if (e.mass != 0.0) l += e.mass * kLn2d * ((double)c - e.c + log2(total));
  return (float)l;
}
// The gradient at a teacher's token is w (c_k - ps sum c) = w (pull ps - pt) with pull = tt / ts - sum c = tt / ts (1 - sum ps) +
// sum pt, that is tt + sum pt, without tt at the floor. Formed as the difference it loses the tail of a sure student (ts = 1e-6:
// 0.06 of a gradient of 0.3).
__device__ __forceinline__ float pull_of(const TeacherSums& e, float ratio) {
  return (float)e.mass + (ratio > 0.f ? e.tt : 0.f);
}
__device__ __forceinline__ float kd_pull(float c, float inv_s, float pull, float w, float z, float pt, float kl) {
  const float ps = ex2(fmaf(z, kl, -c)) * inv_s;
  return inv_s == 0.f ? 0.f : w * fmaf(pull, ps, -pt);
}

// A vector with -inf in element j.
template <typename T>
__device__ __forceinline__ uint4 without(uint4 x, int j) {
  constexpr int N = Vec<T>::N;
  float f[N];
  Vec<T>::unpack(x, f);
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (k == j) f[k] = -INFINITY;
  return Vec<T>::pack(f);
}
// scale 2^(z kl - c) for the elements of a vector
template <typename T>
__device__ __forceinline__ uint4 scaled_exp(const uint4& x, Two scale, Two minus_c, Two k2) {
  constexpr int N = Vec<T>::N;
  float f[N];
  Vec<T>::unpack(x, f);
#pragma unroll
  for (int k = 0; k < N; k += 2) {
    const float2 g = halves(mul2(scale, ex2_two(fma2(two(f[k], f[k + 1]), k2, minus_c))));
    f[k] = g.x;
    f[k + 1] = g.y;
  }
  return Vec<T>::pack(f);
}

// The tail's part of one unit: vectors that hold a teacher's token give it up. With kd_loss_kernel behind it 92 us for 1024 x
// 151936 fp32 (103% of the copy rate), 236 us for 4096 x 152064 bf16 (80%), 6.5 us for 16 x 32000 fp32 (latency).
template <typename T>
__global__ void __launch_bounds__(kThreads) kd_parts_kernel(const T* logits, int64_t ld, int64_t rows, int V, Teacher t,
                                                            float kl, unsigned long long* parts) {
  constexpr int N = Vec<T>::N;
  __shared__ int places[kMaxK], s_listed;
  __shared__ unsigned long long warp_part[kWarps];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  const int64_t row = unit_row();
  if (row >= rows) return;
  const Slice<T> s(logits + row * ld, V, kUnit * kThreads, blockIdx.x);
  uint4 x[kUnit];
  load_unit(s, x);
  if (tid < 32) {
    int id[kE];
    load_ids(t, row, V, id);
    const int n = list_places(s, id, places);
    if (tid == 0) s_listed = n;
  }
  __syncthreads();
  const int listed = s_listed;
  float m = kFloor;
  Soft soft{kFloor * kl, 0.f};
  for (int j = 0; j < listed; ++j) {
    const int v = places[j] / N;
    if (v % kThreads == tid)
#pragma unroll
      for (int i = 0; i < kUnit; ++i)
        if (v == tid + i * kThreads) x[i] = without<T>(x[i], places[j] % N);
  }
  add_soft<T>(x, kl, m, soft);
#pragma unroll
  for (int o = 16; o; o >>= 1) soft = join(soft, shfl_xor(soft, o));
  if ((tid & 31) == 0) warp_part[tid >> 5] = as_u64(soft.c, soft.sum);
  __syncthreads();
  if (tid < 32) {
    const Soft r = join_parts(kWarps, kl, [&](int i) { return warp_part[i]; });
    if (tid == 0) parts[unit_index()] = as_u64(r.c, r.sum);
  }
}

template <typename T>
__global__ void __launch_bounds__(32) kd_loss_kernel(const T* logits, int64_t ld, int splits, int V, Teacher t, float kl,
                                                     const unsigned long long* parts, float* loss, KdSaved* stats) {
  __shared__ int s_id[kMaxK];
  const int64_t row = blockIdx.x;
  pdl_launch_dependents();
  int id[kE];
  load_ids(t, row, V, id);
  float lp[kE], z[kE];
  load_entries(t, row, logits + row * ld, id, lp, z);
  const TeacherSums sums = teacher_sums(teacher_row(t.k, id, lp, z, s_id), kl, t.k);
  pdl_wait();
  const Soft tail = join_parts(splits, kl, [&](int i) { return parts[row * splits + i]; });
  if (threadIdx.x == 0) {
    loss[row] = kd_loss(sums, tail);
    if (stats) {
      const KdRow f = kd_finish(sums, tail);
      stats[row] = KdSaved{f.c, f.inv_s, pull_of(sums, f.ratio), f.csum};
    }
  }
}

// What kd_grad_kernel needs of the rows' teachers, prepared by a small kernel before it: with the student's logits at the
// teacher's tokens read there, the gradient may go over the logits.
struct KdRows {
  int* id;                           // [rows, k], -1: left out
  float *z, *pt;                     // [rows, k]
  TeacherSums* sums;                 // [rows]
};
template <typename T>
__global__ void __launch_bounds__(32) kd_prepare_kernel(const T* logits, int64_t ld, int V, Teacher t, float kl, float inv_t,
                                                        const float* weight, KdRows r) {
  __shared__ int s_id[kMaxK];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  pdl_launch_dependents();
  int id[kE];
  float lp[kE], z[kE];
  load_ids(t, row, V, id);
  load_entries(t, row, logits + row * ld, id, lp, z);
  const TeacherRow e = teacher_row(t.k, id, lp, z, s_id);
#pragma unroll
  for (int i = 0; i < kE; ++i)
    if (lane + 32 * i < t.k) {
      const int64_t at = row * t.k + lane + 32 * i;
      r.id[at] = e.kept >> i & 1 ? id[i] : -1;
      r.z[at] = e.z[i];
      r.pt[at] = e.pt[i];
    }
  TeacherSums s = teacher_sums(e, kl, t.k);
  s.w = weight[row] * inv_t;
  if (lane == 0) r.sums[row] = s;
}

// The teacher's tokens in a block's share of a row.
struct ShareIds {
  int n, id[kMaxK];
  float z[kMaxK], pt[kMaxK];
};

// Loss and gradient of a row by one block or cluster. The owner of a teacher's token takes it out (-inf) before the first
// look, which so sums the tail alone (a confident student's tail is lost in 1 - sum ps); after the second look it writes
// the token's gradient. 239 us for 1024 x 151936 fp32 (80% of the copy rate for one read and one write), 521 us for 4096 x
// 152064 bf16 (73%). A block's phases (load, reduce, write) leave its share of the memory idle between them, which only the
// other blocks of the SM fill; in bf16 the two ex2 per 4 bytes take 60% of the time as well.
template <typename T>
__global__ void __launch_bounds__(kRowThreads, kRowBlocks) kd_grad_kernel(const T* logits, int64_t ld, int V, int keep,
                                                                          int k, float kl, float* loss, T* out,
                                                                          int64_t out_ld, KdRows r) {
  constexpr int N = Vec<T>::N;
  extern __shared__ uint4 dyn[];
  __shared__ unsigned long long warp_part[kRowWarps], part[kMaxCluster];
  __shared__ ShareIds list;
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t row = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31;
  const Share<T> s(logits + row * ld, V, rank, size, keep);
  cluster_started();
  copy_kept(s, s.row, dyn);
  pdl_wait();
  if (tid < 32) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kE; ++i) {
      const int64_t at = row * k + lane + 32 * i;
      const int id = lane + 32 * i < k ? r.id[at] : -1;
      const bool in = id >= 0 && s.holds(id);
      const unsigned all = __ballot_sync(0xffffffffu, in);
      if (in) {
        const int j = n + __popc(all & ((1u << lane) - 1u));
        list.id[j] = id;
        list.z[j] = r.z[at];
        list.pt[j] = r.pt[at];
      }
      n += __popc(all);
    }
    if (lane == 0) list.n = n;
  }
  __syncthreads();
  const int listed = list.n;
  int own = 0, own_v = 0;              // this thread's teacher tokens among the streamed vectors, the vector of one
  for (int j = 0; j < listed; ++j)
    if (s.owns(list.id[j]) && (list.id[j] - s.e0) / N >= s.kept) {
      ++own;
      own_v = (list.id[j] - s.e0) / N;
    }
  float m = kFloor;
  Soft soft{kFloor * kl, 0.f};
  for (int v = s.kept + tid; v < s.n; v += kRound) {
    uint4 x[4];
    stream(s, s.row, true, v, x);
    if (own > 1 || (own == 1 && own_v >= v && own_v < v + kRound))
      for (int j = 0; j < listed; ++j) {
        const int at = list.id[j] - s.e0;
        if (s.owns(list.id[j]))
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (at / N == v + i * kRowThreads) x[i] = without<T>(x[i], at % N);
      }
    add_soft<T>(x, kl, m, soft);
  }
  const int single = s.single();
  bool single_in = single >= 0;
  if (single_in) {
    for (int j = 0; j < listed; ++j) single_in &= list.id[j] != single;
    if (single_in) {
      uint4 x[1] = {make_uint4(Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad)};
      *reinterpret_cast<T*>(x) = s.row[single];
      add_soft<T>(x, kl, m, soft);
    }
  }
  wait_copies();
  for (int j = 0; j < listed; ++j) {
    const int at = list.id[j] - s.e0;
    if (s.owns(list.id[j]) && at / N < s.kept) dyn[at / N] = without<T>(dyn[at / N], at % N);
  }
  for (int v = tid; v < s.kept; v += kRound) {
    const uint4 x[4] = {dyn[v], dyn[v + kRowThreads], dyn[v + 2 * kRowThreads], dyn[v + 3 * kRowThreads]};
    add_soft<T>(x, kl, m, soft);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) soft = join(soft, shfl_xor(soft, o));
  if (lane == 0) warp_part[tid >> 5] = as_u64(soft.c, soft.sum);
  __syncthreads();
  cluster_peers_run();
  if (tid < 32) {
    const Soft b = join_parts(kRowWarps, kl, [&](int i) { return warp_part[i]; });
    if (lane < (int)size) st_peer(part + rank, lane, as_u64(b.c, b.sum));
  }
  cluster_sync();
  const Soft tail = join_parts(size, kl, [&](int i) { return part[i]; });
  const TeacherSums& e = r.sums[row];
  const KdRow f = kd_finish(e, tail);
  const float w = e.w;
  if (rank == 0 && tid == 0) loss[row] = kd_loss(e, tail);
  T* o = out + row * out_ld;
  const Two scale = two(f.inv_s == 0.f ? 0.f : -f.csum * f.inv_s * w), c2 = two(-f.c), k2 = two(kl);
  if (same_phase<T>(o, s.row)) {
    uint4* p = reinterpret_cast<uint4*>(o + s.e0);
    for (int v = s.kept + tid; v < s.n; v += kRound) {
      uint4 x[4];
      stream(s, s.row, true, v, x);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (v + i * kRowThreads < s.n) __stcs(p + v + i * kRowThreads, scaled_exp<T>(x[i], scale, c2, k2));
    }
    for (int v = tid; v < s.kept; v += kRound)
#pragma unroll
      for (int i = 0; i < 4; ++i) __stcs(p + v + i * kRowThreads, scaled_exp<T>(dyn[v + i * kRowThreads], scale, c2, k2));
  } else {
    for (int v = tid; v < s.n; v += kRowThreads) {
      const uint4 x = v < s.kept ? dyn[v] : __ldcg(reinterpret_cast<const uint4*>(s.row + s.e0) + v);
      const uint4 u = scaled_exp<T>(x, scale, c2, k2);
#pragma unroll
      for (int j = 0; j < N; ++j) o[s.e0 + v * N + j] = reinterpret_cast<const T*>(&u)[j];
    }
  }
  if (single_in) {
    uint4 x = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<T*>(&x) = s.row[single];
    x = scaled_exp<T>(x, scale, c2, k2);
    o[single] = *reinterpret_cast<const T*>(&x);
  }
  for (int j = 0; j < listed; ++j)
    if (s.owns(list.id[j]) || list.id[j] == single)
      o[list.id[j]] = Vec<T>::back(kd_pull(f.c, f.inv_s, pull_of(e, f.ratio), w, list.z[j], list.pt[j], kl));
}

// The gradient from statistics, elementwise; `out` may be the logits. 189 us for 1024 x 151936 fp32, 376 us for 4096 x 152064
// bf16 (both 101% of the copy rate).
template <typename T>
__global__ void __launch_bounds__(kThreads) kd_bwd_kernel(const T* logits, int64_t ld, int64_t rows, int V, Teacher t,
                                                          float kl, float inv_t, const float* weight,
                                                          const KdSaved* stats, T* out, int64_t out_ld) {
  const int64_t row = unit_row();
  if (row >= rows) return;
  const Slice<T> s(logits + row * ld, V, kUnit * kThreads, blockIdx.x);
  uint4 x[kUnit];
  load_unit(s, x);
  T* o = out + row * out_ld;
  const int tid = threadIdx.x;
  int id = tid < t.k ? load_id(t, row * t.k + tid, V) : -1;
  if (id >= 0 && s.place(id) < 0) id = -1;
  const float z = id >= 0 ? masked(Vec<T>::one(s.row[id])) : 0.f;
  pdl_wait();
  const KdSaved st = stats[row];
  const float w = st.inv_s == 0.f ? 0.f : weight[row] * inv_t;
  const Two scale = two(st.inv_s == 0.f ? 0.f : -st.csum * st.inv_s * w), c2 = two(-st.c), k2 = two(kl);
  __syncthreads();                                     // every z is read
  store_unit<kUnit>(s, o, [&](int i) { return scaled_exp<T>(x[i], scale, c2, k2); });
  __syncthreads();
  if (id >= 0) {
    bool repeated = false;
    for (int j = 0; j < tid; ++j) repeated |= load_id(t, row * t.k + j, V) == id;
    if (!repeated) o[id] = Vec<T>::back(kd_pull(st.c, st.inv_s, st.pull, w, z, expf(t.lp[row * t.k + tid]), kl));
  }
}

// ------------------------------------------------------------------------------------------- acceptance and KL
// log2 q_v = zq_v kl - bq up to the rounding of bq, whose remainder is in fq = 2^(rounded - exact), and for p alike. fq = 0 marks
// a row with nothing to compare. steep, middle: h_v = (zq_v - zp_v) steep + middle, held to [0, 1] (share2); a = sum_v q_v h_v.
struct AcceptRow {
  float bq, fq, bp, fp, steep, middle, a;
};
static_assert(sizeof(AcceptRow) == kAcceptStats * 4, "AcceptRow is what callers allocate");

// Both softmaxes, with their largest logits in place of the offsets, and d = sum 2^xp (xp - xq) with xq, xp the ex2 arguments
// of the elements: KL in bits is then d / sum_p + log2 sum_q - log2 sum_p, and no second look needs the probabilities of p.
struct Pair {
  float mq, sq, mp, sp, d;
};
// The rounded offset of a maximum: never contracted into an FMA, or its uses would differ.
__device__ __forceinline__ float offset(float m, float kl) { return __fmul_rn(m, kl); }
__device__ __forceinline__ Pair join(const Pair& a, const Pair& b, float kl) {
  Pair r;
  r.mq = fmaxf(a.mq, b.mq);
  r.mp = fmaxf(a.mp, b.mp);
  const float cq = offset(r.mq, kl), cp = offset(r.mp, kl);
  const float qa = offset(a.mq, kl) - cq, qb = offset(b.mq, kl) - cq, pa = offset(a.mp, kl) - cp, pb = offset(b.mp, kl) - cp;
  const float ea = ex2(pa), eb = ex2(pb);
  r.sq = fmaf(a.sq, ex2(qa), __fmul_rn(b.sq, ex2(qb)));    // one order for both: equal sides stay equal to the last bit
  r.sp = fmaf(a.sp, ea, __fmul_rn(b.sp, eb));
  // the arguments move by the change of their offsets; a part whose weight vanishes adds nothing, even if infinite
  const float da = a.d + a.sp * (pa - qa), db = b.d + b.sp * (pb - qb);
  r.d = (ea == 0.f ? 0.f : ea * da) + (eb == 0.f ? 0.f : eb * db);
  return r;
}
__device__ __forceinline__ Pair shfl_xor(const Pair& a, int o) {
  const auto x = [&](float f) { return __shfl_xor_sync(0xffffffffu, f, o); };
  return {x(a.mq), x(a.sq), x(a.mp), x(a.sp), x(a.d)};
}

constexpr int kPairVec = 4;          // vectors per thread, unit and side of the gradient

// h of two tokens: 1 where q < p, 0 where q > p, 1/2 where they are equal. With gap the log2 of the ratio of the sums, log2 q_v -
// log2 p_v = (zq_v - zp_v) kl - gap; the difference of the logits comes first and keeps the digits that the ex2 arguments
// lose to their offsets. Sums that differ by less than 2^-21 of themselves, a few roundings, count as equal, and within 2^-21 (1
// + |gap|) of equality, what gap itself may be off by, h goes from 1 to 0 in a line. A = sum q h must take each token's h as the
// token itself does, or a sure token gets a gradient of full size where 1 - q is all there is: so the forward and the backward
// form h by these operations alone. One FMA and one saturating FMA; a NaN (both masked by -inf) becomes 0, for tokens without mass.
__device__ __forceinline__ float2 share2(Two q, Two p, float steep, float middle) {
  const float2 d = halves(fma2(p, two(-1.f), q));
  return {__saturatef(fmaf(d.x, steep, middle)), __saturatef(fmaf(d.y, steep, middle))};
}

template <typename Load>
__device__ __forceinline__ Pair join_pairs(int n, float kl, Load load) {
  Pair t{kFloor, 0.f, kFloor, 0.f, 0.f};
  for (int i = threadIdx.x & 31; i < n; i += 32) t = join(t, load(i), kl);
#pragma unroll
  for (int o = 16; o; o >>= 1) t = join(t, shfl_xor(t, o), kl);
  return t;
}
// Adds pairs of vectors to a thread's running Pair.
template <typename T, int kVec>
__device__ __forceinline__ void add_pair(const uint4 (&xq)[kVec], const uint4 (&xp)[kVec], float kl, Pair& a) {
  constexpr int N = Vec<T>::N;
  const float vq = unit_max<T>(xq), vp = unit_max<T>(xp);
  float low = packed_min<T>(xq[0]);
#pragma unroll
  for (int i = 0; i < kVec; ++i) low = fminf(low, fminf(packed_min<T>(xq[i]), packed_min<T>(xp[i])));
  if (vq > a.mq || vp > a.mp) a = join(a, Pair{fmaxf(vq, kFloor), 0.f, fmaxf(vp, kFloor), 0.f, 0.f}, kl);
  const Two k2 = two(kl), cq = two(-offset(a.mq, kl)), cp = two(-offset(a.mp, kl)), minus = two(-1.f);
  Two sq = two(0.f), sp = two(0.f), d = two(0.f);
  const auto look = [&](auto guarded) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      float q[N], p[N];
      Vec<T>::unpack(xq[i], q);
      Vec<T>::unpack(xp[i], p);
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        if (guarded) {
          q[k] = masked(q[k]);
          q[k + 1] = masked(q[k + 1]);
        }
        const Two eq = fma2(two(q[k], q[k + 1]), k2, cq), ep = fma2(two(p[k], p[k + 1]), k2, cp), w = ex2_two(ep);
        sq = add2(sq, ex2_two(eq));
        sp = add2(sp, w);
        const Two gap = fma2(eq, minus, ep);
        if (guarded) {
          const float2 wf = halves(w), gf = halves(gap);
          d = add2(d, two(wf.x > 0.f ? wf.x * gf.x : 0.f, wf.y > 0.f ? wf.y * gf.y : 0.f));
        } else {
          d = fma2(w, gap, d);
        }
      }
    }
  };
  // masked logits: 0 times an infinite gap is 0, and a token that only the draft masks makes KL infinite, whatever masks it
  if (low >= kFloor) look(std::false_type());
  else look(std::true_type());
  a.sq += sum(sq);
  a.sp += sum(sp);
  a.d += sum(d);
}

// One row by one block or cluster. First look: both softmaxes and d; second look: the sums of min(q, p) and of q h. 137 us for 2044
// x 32768 fp32 (60% of the copy rate), 123 us for 508 x 151936 bf16 (38%): three ex2 per pair of logits (64 us of the 123) and
// some 34 instructions come near the time of the loads, and the two looks of a block do not overlap. h by comparisons, with the
// few equal tokens in a branch, took 143 and 129 us; with the mass of q on either side summed by itself (a fourth ex2) 144 and 133.
template <typename T>
__global__ void __launch_bounds__(kRowThreads, kPairBlocks) accept_kernel(const T* draft, int64_t ldq, const T* target,
                                                                         int64_t ldp, int V, int keep, float kl,
                                                                         float* alpha, float* out_kl, AcceptRow* stats) {
  constexpr int N = Vec<T>::N;
  extern __shared__ uint4 dyn[];
  __shared__ unsigned long long part[3][kMaxCluster], sums[kMaxCluster];
  __shared__ Pair warp_pair[kRowWarps];
  __shared__ float2 warp_sum[kRowWarps];
  const uint32_t rank = cluster_rank(), size = cluster_size();
  const int64_t row = blockIdx.x / size;
  const int tid = threadIdx.x, lane = tid & 31;
  const T* other = target + row * ldp;
  const Share<T> s(draft + row * ldq, V, rank, size, keep);
  const bool same = same_phase(other, s.row);
  const uint4 *dq = dyn, *dp = dyn + s.kept;
  cluster_started();
  copy_kept(s, s.row, dyn);
  copy_kept(s, other, dyn + s.kept);
  const int single = s.single();
  uint4 lone[2][1];
  if (single >= 0) {
    lone[0][0] = lone[1][0] = make_uint4(Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad);
    *reinterpret_cast<T*>(lone[0]) = s.row[single];
    *reinterpret_cast<T*>(lone[1]) = other[single];
  }
  Pair a{kFloor, 0.f, kFloor, 0.f, 0.f};
  for (int v = s.kept + tid; v < s.n; v += 2 * kRowThreads) {
    uint4 xq[2], xp[2];
    stream(s, s.row, true, v, xq);
    stream(s, other, same, v, xp);
    add_pair<T>(xq, xp, kl, a);
  }
  if (single >= 0) add_pair<T>(lone[0], lone[1], kl, a);
  wait_copies();
  for (int v = tid; v < s.kept; v += 2 * kRowThreads) {
    const uint4 xq[2] = {dq[v], dq[v + kRowThreads]}, xp[2] = {dp[v], dp[v + kRowThreads]};
    add_pair<T>(xq, xp, kl, a);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) a = join(a, shfl_xor(a, o), kl);
  if (lane == 0) warp_pair[tid >> 5] = a;
  __syncthreads();
  cluster_peers_run();
  if (tid < 32) {
    a = join_pairs(kRowWarps, kl, [&](int i) { return warp_pair[i]; });
    if (lane < (int)size) {
      st_peer(&part[0][rank], lane, as_u64(a.mq, a.sq));
      st_peer(&part[1][rank], lane, as_u64(a.mp, a.sp));
      st_peer(&part[2][rank], lane, as_u64(a.d, 0.f));
    }
  }
  cluster_sync();
  a = join_pairs(size, kl, [&](int i) {
    const Soft q = as_soft(part[0][i]), p = as_soft(part[1][i]);
    return Pair{q.c, q.sum, p.c, p.sum, as_soft(part[2][i]).c};
  });
  const float cq = offset(a.mq, kl), cp = offset(a.mp, kl), rq = cq + log2f(a.sq), rp = cp + log2f(a.sp);
  const float ratio = log2f(__fdiv_rn(a.sq, a.sp)), gap = (cq - cp) + (fabsf(ratio) < 0x1p-21f ? 0.f : ratio);
  const float per_tie = 0x1p20f / (1.f + fabsf(gap));
  const float steep = -kl * per_tie, middle = fmaf(gap, per_tie, 0.5f);
  Two least = two(0.f), held = two(0.f);     // sums of min(q, p), and of it times h: sum q h, as h = 0 where q > p
  // rq and rp are rounded: what they lose differs, and is given back to q before the two are compared
  const Two k2 = two(kl), bq = two(-rq), bp = two(-rp), to_p = two((rq - rp) - gap);
  const auto look = [&](const uint4& uq, const uint4& up) {
    float q[N], p[N];
    Vec<T>::unpack(uq, q);
    Vec<T>::unpack(up, p);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const Two zq = two(q[k], q[k + 1]), zp = two(p[k], p[k + 1]);
      const float2 eq = halves(add2(fma2(zq, k2, bq), to_p)), ep = halves(fma2(zp, k2, bp));
      const float2 h = share2(zq, zp, steep, middle);
      const Two e = two(ex2(fminf(eq.x, ep.x)), ex2(fminf(eq.y, ep.y)));
      least = add2(least, e);
      held = fma2(e, two(h.x, h.y), held);
    }
  };
  for (int v = s.kept + tid; v < s.n; v += 2 * kRowThreads) {
    uint4 xq[2], xp[2];
    stream(s, s.row, true, v, xq);
    stream(s, other, same, v, xp);
    look(xq[0], xp[0]);
    look(xq[1], xp[1]);                      // padding adds 0
  }
  if (single >= 0) look(lone[0][0], lone[1][0]);
#pragma unroll 2
  for (int v = tid; v < s.kept; v += kRowThreads) look(dq[v], dp[v]);
  const float x = warp_reduce(sum(least), Add()), y = warp_reduce(sum(held), Add());
  if (lane == 0) warp_sum[tid >> 5] = make_float2(x, y);
  __syncthreads();
  if (tid < 32) {
    float2 w = lane < kRowWarps ? warp_sum[lane] : make_float2(0.f, 0.f);
    w.x = warp_reduce(w.x, Add());
    w.y = warp_reduce(w.y, Add());
    if (lane == 0) st_peer(sums + rank, 0, as_u64(w.x, w.y));
  }
  cluster_sync();
  if (rank != 0 || tid != 0) return;
  float2 w = make_float2(0.f, 0.f);
  for (uint32_t i = 0; i < size; ++i) {
    w.x += as_soft(sums[i]).c;
    w.y += as_soft(sums[i]).sum;
  }
  const double lq = log2((double)a.sq), lp = log2((double)a.sp);
  const float fq = exp2f((float)((double)rq - (cq + lq))), fp = exp2f((float)((double)rp - (cp + lp)));
  const bool nothing = a.sq == 0.f || a.sp == 0.f;
  const bool nan = isnan(a.sq) || isnan(a.sp);            // the minimum drops a NaN operand
  alpha[row] = nothing ? 0.f : nan ? NAN : fp * w.x;
  out_kl[row] = nothing ? 0.f : (float)(kLn2d * ((double)a.d / a.sp + lq - lp));
  if (!stats) return;
  stats[row] = nothing ? AcceptRow{} : AcceptRow{rq, fq, rp, fp, steep, middle, fp * w.y};
}

// The gradient from the row's statistics, elementwise. 118 us for 2044 x 32768 fp32 (104% of the copy rate), 69 us for 508 x
// 151936 bf16 (101%).
template <typename T>
__global__ void __launch_bounds__(kThreads) accept_bwd_kernel(const T* draft, int64_t ldq, const T* target, int64_t ldp,
                                                              int64_t rows, int V, float kl, float inv_t,
                                                              const AcceptRow* stats, const float* g_alpha,
                                                              const float* g_kl, T* out, int64_t out_ld) {
  constexpr int N = Vec<T>::N;
  const int64_t row = unit_row();
  if (row >= rows) return;
  const Slice<T> s(draft + row * ldq, V, kPairVec * kThreads, blockIdx.x);
  uint4 xq[kPairVec], xp[kPairVec];
  load_unit(s, xq);
  load_unit(s, target + row * ldp, xp);
  const AcceptRow st = stats[row];
  const bool nothing = st.fq == 0.f;
  const float ga = g_alpha[row] * inv_t, gk = g_kl[row] * inv_t;
  const Two jump = two(st.fq * ga), rest = two(st.fq * (gk - ga * st.a)), kp = two(-gk * st.fp);
  const Two k2 = two(kl), bq = two(-st.bq), bp = two(-st.bp);
  store_unit<kPairVec>(s, out + row * out_ld, [&](int i) {
    float q[N], p[N];
    Vec<T>::unpack(xq[i], q);
    Vec<T>::unpack(xp[i], p);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      const Two zq = two(q[k], q[k + 1]), zp = two(p[k], p[k + 1]);
      const float2 h = share2(zq, zp, st.steep, st.middle);
      const float2 g = halves(fma2(ex2_two(fma2(zq, k2, bq)), fma2(two(h.x, h.y), jump, rest),
                                   mul2(kp, ex2_two(fma2(zp, k2, bp)))));
      q[k] = nothing ? 0.f : g.x;
      q[k + 1] = nothing ? 0.f : g.y;
    }
    return Vec<T>::pack(q);
  });
}

// ------------------------------------------------------------------------------------------- draft verification
// Two launches. The first reduces every needed row of logits, cut over blocks, to softmax parts (T > 0) or to its best
// token (T <= 0). The second, as many blocks per sequence as run at once, started early by programmatic launch, joins the
// parts, finds the first rejected draft and draws from that position alone: the race costs a hash per token and is run for
// one row of the k + 1. A draw needs -log(u) / r below the best so far; -log(u) >= 1 - u, which is the hash's integer, so
// the logarithm and the division are taken for the few tokens that can win.
// 55.5 us for 64 sequences of 3 soft drafts x 151936 bf16: 31 us the rows (68% of the copy rate), 24 us the draw, bound by the 51
// instructions per token, most of them the hash's 64-bit products. 34.9 us for 32 sequences of up to 7 point-mass drafts x
// 152064 fp32 (68% of the copy rate over both). One sequence of 3: 10 us, latency.
constexpr int kDrawThreads = 256;
constexpr int kDrawWarps = kDrawThreads / 32;
constexpr int kDrawVec = 2;          // vectors that a thread requests at once

// Temperatures come with requests, from next to nothing to infinity. kl stays finite; at T = 1e20 all logits weigh the same to
// fp32, and a masked one still nothing. The rounding of an offset m kl leaves fp32's range of exponents where |z| / T passes 2^30,
// so here the largest logit is taken off first and the rest scaled: one more operation per logit (54.0 -> 55.5 us for 64 sequences
// of 3 soft drafts x 151936 bf16).
__device__ __forceinline__ float scale_of(float temp) { return fminf(kLog2e / fminf(temp, 1e20f), 3e38f); }
// sum = sum over elements of 2^((z - m) kl), m the largest z or kFloor
struct Peak {
  float m, sum;
};
__device__ __forceinline__ Peak join(Peak a, Peak b, float kl) {
  const float m = fmaxf(a.m, b.m);
  return {m, a.sum * ex2((a.m - m) * kl) + b.sum * ex2((b.m - m) * kl)};
}
__device__ __forceinline__ Peak as_peak(unsigned long long u) {
  return {__uint_as_float((uint32_t)u), __uint_as_float((uint32_t)(u >> 32))};
}
// A warp's part of a unit: its threads share their maximum. `top`: the thread's largest logit.
template <typename T, int kVec>
__device__ __forceinline__ Peak warp_peak(const uint4 (&x)[kVec], float top, float kl) {
  constexpr int N = Vec<T>::N;
  const float m = warp_reduce(fmaxf(top, kFloor), Max());
  const Two k2 = two(kl), m2 = two(-m);
  Two a = two(0.f), b = two(0.f);
#pragma unroll
  for (int i = 0; i < kVec; ++i) {
    float f[N];
    Vec<T>::unpack(x[i], f);
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      a = add2(a, ex2_two(mul2(add2(two(f[k], f[k + 1]), m2), k2)));
      b = add2(b, ex2_two(mul2(add2(two(f[k + 2], f[k + 3]), m2), k2)));
    }
  }
  return {m, warp_reduce(sum(add2(a, b)), Add())};
}
// Joins a list of parts over a warp, as join_parts does.
template <typename Load>
__device__ __forceinline__ Peak join_peaks(int n, float kl, Load load) {
  Peak t{kFloor, 0.f};
  for (int i = threadIdx.x & 31; i < n; i += 32) t = join(t, as_peak(load(i)), kl);
#pragma unroll
  for (int o = 16; o; o >>= 1)
    t = join(t, Peak{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.sum, o)}, kl);
  return t;
}

constexpr uint64_t kIndexStep = 0x8CB92BA72F3D8DD7ull;
// x * c modulo 2^64 in 32-bit halves
__device__ __forceinline__ uint2 mul64(uint32_t lo, uint32_t hi, uint64_t c) {
  const uint64_t w = (uint64_t)lo * (uint32_t)c;
  return make_uint2((uint32_t)w, (uint32_t)(w >> 32) + lo * (uint32_t)(c >> 32) + hi * (uint32_t)c);
}
// The sampler's 23 random bits of counter base + index kIndexStep: z ^= z >> 30, z *= c1, z ^= z >> 27, z *= c2, and the top
// bits, which its last step, z ^ (z >> 31), leaves as they are.
__device__ __forceinline__ uint32_t random23(uint64_t counter) {
  uint32_t lo = (uint32_t)counter, hi = (uint32_t)(counter >> 32);
  lo ^= __funnelshift_r(lo, hi, 30);
  hi ^= hi >> 30;
  const uint2 y = mul64(lo, hi, 0xBF58476D1CE4E5B9ull);
  lo = y.x ^ __funnelshift_r(y.x, y.y, 27);
  hi = y.y ^ (y.y >> 27);
  return mul64(lo, hi, 0x94D049BB133111EBull).y >> 9;
}
__device__ __forceinline__ float unit(uint32_t h) { return ((float)h + 0.5f) * (1.0f / 8388608.0f); }

__device__ __forceinline__ int drafts_of(const Verify& a, int64_t b) {
  return a.n_draft ? min(max(a.n_draft[b], 0), a.k) : a.k;
}

// Workspace: best draw and arrivals of each sequence, then parts [batch][2 k + 1 rows: k + 1 of the target, k of the
// draft][splits], 8 bytes each: Peak, or a rank_key.
__device__ __forceinline__ unsigned long long* verify_best(const Verify& a) {
  return static_cast<unsigned long long*>(a.workspace);
}
__device__ __forceinline__ unsigned long long* verify_count(const Verify& a) { return verify_best(a) + a.batch; }
__device__ __forceinline__ unsigned long long* verify_parts(const Verify& a) { return verify_best(a) + 2 * a.batch; }

template <typename T>
__global__ void __launch_bounds__(kThreads, 5) verify_parts_kernel(Verify a, int splits) {
  constexpr int N = Vec<T>::N;
  __shared__ unsigned long long warp_part[kWarps];
  const int rows = a.draft_logits ? 2 * a.k + 1 : a.k + 1;
  const int split = blockIdx.x % splits;
  const int j = (blockIdx.x / splits) % rows;
  const int64_t b = blockIdx.x / splits / rows;
  pdl_launch_dependents();
  if (j == 0 && split == 0 && threadIdx.x == 0) {
    verify_best(a)[b] = kNone;
    verify_count(a)[b] = 0;
  }
  const int n = drafts_of(a, b);
  const float temp = a.temps[b];
  const bool draft = j > a.k, greedy = !(temp > 0.f);
  if ((draft ? j - a.k - 1 >= n : j > n) || (draft && greedy)) return;
  const T* row = draft ? static_cast<const T*>(a.draft_logits) + b * a.draft_b + (j - a.k - 1) * a.draft_j
                       : static_cast<const T*>(a.logits) + b * a.logits_b + j * a.logits_j;
  const Slice<T> s(row, a.V, kUnit * kThreads, split);
  uint4 x[kUnit];
  load_unit(s, x);
  const float top = unit_max<T>(x);
  unsigned long long res;
  if (greedy) {
    res = kNone;
    const float best = warp_reduce(top, Max());
    if (top == best && best >= kFloor) {
#pragma unroll
      for (int i = kUnit - 1; i >= 0; --i) {          // ends at the thread's first element of that value
        float f[N];
        Vec<T>::unpack(x[i], f);
#pragma unroll
        for (int k = N - 1; k >= 0; --k)
          if (f[k] == best) res = rank_key(best, s.start(threadIdx.x + i * kThreads) + k);
      }
    }
    if (unit_nan<T>(x)) res = kNanKey;
    res = warp_reduce(res, MinKey());
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = res;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) res = min(res, warp_part[w]);
  } else {
    const float kl = scale_of(temp);
    const Peak part = warp_peak<T>(x, top, kl);
    if ((threadIdx.x & 31) == 0) warp_part[threadIdx.x >> 5] = as_u64(part.m, part.sum);
    __syncthreads();
    if (threadIdx.x >= 32) return;
    const Peak t = join_peaks(kWarps, kl, [&](int i) { return warp_part[i]; });
    res = as_u64(t.m, t.sum);
  }
  if (threadIdx.x == 0) verify_parts(a)[blockIdx.x] = res;
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 5) verify_draw_kernel(Verify a, int splits, int blocks, int per) {
  constexpr int N = Vec<T>::N;
  __shared__ Peak s_p[kMaxK + 1], s_q[kMaxK];
  __shared__ unsigned long long s_best[kMaxK + 1];
  __shared__ int s_ok[kMaxK + 1];
  __shared__ unsigned long long warp_best[kDrawWarps];
  __shared__ bool s_again;
  const int rank = blockIdx.x % blocks;
  const int64_t b = blockIdx.x / blocks;
  const int tid = threadIdx.x, lane = tid & 31;
  const int rows = a.draft_logits ? 2 * a.k + 1 : a.k + 1;
  pdl_wait();
  const int n = drafts_of(a, b);
  const float temp = a.temps[b];
  const bool greedy = !(temp > 0.f);
  const float kl = greedy ? 1.f : scale_of(temp);
  const uint64_t seed = (uint64_t)a.seeds[b] * 0x9E3779B97F4A7C15ull + 1ull, step = (uint64_t)a.steps[b];
  const unsigned long long* parts = verify_parts(a) + b * rows * splits;
  for (int j = tid >> 5; j <= n; j += kDrawWarps) {     // one warp per position
    const int64_t id = j < n ? (a.wide ? static_cast<const int64_t*>(a.drafts)[b * a.k + j]
                                       : (int64_t) static_cast<const int32_t*>(a.drafts)[b * a.k + j])
                             : -1;
    const bool known = id >= 0 && id < a.V;
    if (greedy) {
      unsigned long long best = kNone;
      for (int i = lane; i < splits; i += 32) best = min(best, parts[j * splits + i]);
      best = warp_reduce(best, MinKey());
      if (isnan(key_value(best))) best = kNone;
      if (lane == 0) {
        s_best[j] = best;
        s_ok[j] = known && best != kNone && (uint32_t)best == (uint32_t)id;
      }
      continue;
    }
    const auto whole = [&](int r) { return join_peaks(splits, kl, [&](int i) { return parts[r * splits + i]; }); };
    const Peak p = whole(j), q = a.draft_logits && j < n ? whole(a.k + 1 + j) : Peak{0.f, 1.f};
    if (lane == 0) {
      s_p[j] = p;
      if (j < n) s_q[j] = q;
      bool ok = false;
      if (known) {
        const float zp = Vec<T>::one(static_cast<const T*>(a.logits)[b * a.logits_b + j * a.logits_j + id]);
        const float pd = p.sum > 0.f ? ex2((zp - p.m) * kl) / p.sum : 0.f;
        float qd = 1.f;
        if (a.draft_logits) {
          const float zq = Vec<T>::one(static_cast<const T*>(a.draft_logits)[b * a.draft_b + j * a.draft_j + id]);
          qd = q.sum == 0.f ? 0.f : ex2((zq - q.m) * kl) / q.sum;        // NaN in the row: NaN, and the draft is rejected
        }
        ok = unit(random23(seed + (step + j) * 0xD1B54A32D192ED03ull - kIndexStep)) * qd < pd;   // index -1
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
  const T* row = static_cast<const T*>(a.logits) + b * a.logits_b + acc * a.logits_j;
  const T* qrow = a.draft_logits && acc < n ? static_cast<const T*>(a.draft_logits) + b * a.draft_b + acc * a.draft_j : nullptr;
  const int64_t id = acc >= n ? -1 : a.wide ? static_cast<const int64_t*>(a.drafts)[b * a.k + acc]
                                            : (int64_t) static_cast<const int32_t*>(a.drafts)[b * a.k + acc];
  const Peak p = s_p[acc];
  const float ip = 1.f / p.sum, mq = qrow ? s_q[acc].m : 0.f, iq = qrow && s_q[acc].sum > 0.f ? 1.f / s_q[acc].sum : 0.f;
  const bool same = ((reinterpret_cast<uintptr_t>(qrow) ^ reinterpret_cast<uintptr_t>(row)) & 15) == 0;
  const uint64_t base = seed + (step + acc) * 0xD1B54A32D192ED03ull;
  // The earliest of all times is exponential with the rate sum r: 1 for p, 1 - p(d) beside a point mass. A draw that only
  // looks for times up to 24 / rate misses them in one of 2^34 cases, and saves the logarithms that each warp took until it
  // had a bound of its own. The rate of a residual is not known; 1024 covers all but rates of about 1/64 and below, which
  // are rejected as rarely. The block that completes a sequence without a token repeats the search alone, without the
  // limit, and, if the residual is empty, over p itself.
  float limit = 24.f;
  if (qrow) limit = 1024.f;
  else if (id >= 0 && id < a.V) limit = 24.f / fmaxf(1.f - ex2((Vec<T>::one(row[id]) - p.m) * kl) * ip, 1e-6f);
  for (int stage = 0;; ++stage) {
    const bool whole = acc == n || stage == 2 || (qrow && isnan(s_q[acc].sum));
    const Slice<T> s(row, a.V, stage ? a.V : per, stage ? 0 : rank);
    unsigned long long best = kNone;
    float bound = stage ? INFINITY : limit;                           // of this warp: the limit, then its best time
    const auto race = [&](auto residual) {                            // 0: p, 1: p without the draft, 2: p - q
      for (int v0 = tid; v0 - lane < s.count; v0 += kDrawVec * kDrawThreads) {   // the same trip count for a whole warp
        uint4 xp[kDrawVec], xq[kDrawVec];
#pragma unroll
        for (int i = 0; i < kDrawVec; ++i) {
          const int v = v0 + i * kDrawThreads, i0 = s.start(v);
          xp[i] = xq[i] = make_uint4(Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad, Vec<T>::kPad);
          if (v < s.count) {
            xp[i] = s.full(i0) ? __ldcs(reinterpret_cast<const uint4*>(row + i0)) : ragged_vec(s, row, i0);
            if (residual == 2)
              xq[i] = same && s.full(i0) ? __ldcs(reinterpret_cast<const uint4*>(qrow + i0)) : ragged_vec(s, qrow, i0);
          }
        }
#pragma unroll
        for (int i = 0; i < kDrawVec; ++i) {
          if (v0 - lane + i * kDrawThreads >= s.count) break;          // for the whole warp
          const int i0 = s.start(v0 + i * kDrawThreads);
          float f[N], g[N];
          Vec<T>::unpack(xp[i], f);
          Vec<T>::unpack(xq[i], g);
          uint64_t counter = base + (uint64_t)(int64_t)i0 * kIndexStep;
#pragma unroll
          for (int k0 = 0; k0 < N; k0 += 4) {                         // one branch for four tokens
            float r[4], ahead = 1.f;
            uint32_t h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k, counter += kIndexStep) {
              r[k] = ex2((f[k0 + k] - p.m) * kl) * ip;
              if (residual == 1 && i0 + k0 + k == id) r[k] = 0.f;
              if (residual == 2) r[k] = fmaf(ex2((g[k0 + k] - mq) * kl), -iq, r[k]);
              // u = (h + 1/2) 2^-23; -log(u) > 1 - u > 1 - (h + 1) 2^-23, exact from 1 + h 2^-23
              h[k] = random23(counter);
              const float miss = (2.f - 0x1p-23f) - __uint_as_float(0x3F800000u | h[k]);
              ahead = fminf(ahead, fmaf(-bound, r[k], miss));         // above 0 for r <= 0, no operand where it is NaN
            }
            if (ahead <= 0.f)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const float e = -logf(unit(h[k])) / r[k];
                if (r[k] > 0.f && e <= bound) {
                  best = min(best, (unsigned long long)__float_as_uint(e) << 32 | (uint32_t)(i0 + k0 + k));
                  bound = e * 1.000001f;                              // rounded up: ties stay in
                }
              }
          }
          bound = __uint_as_float(__reduce_min_sync(0xffffffffu, __float_as_uint(bound)));
        }
      }
    };
    if (whole) race(std::integral_constant<int, 0>());
    else if (qrow) race(std::integral_constant<int, 2>());
    else race(std::integral_constant<int, 1>());
    best = warp_reduce(best, MinKey());
    if (lane == 0) warp_best[tid >> 5] = best;
    __syncthreads();
    if (tid == 0) {
      for (int i = 1; i < kDrawWarps; ++i) best = min(best, warp_best[i]);
      s_again = false;
      bool last = stage > 0;
      if (!stage) {
        atomicMin(verify_best(a) + b, best);
        __threadfence();
        last = atomicAdd(verify_count(a) + b, 1ull) == (unsigned long long)(blocks - 1);
        if (last) best = atomicMin(verify_best(a) + b, kNone);
      }
      if (last) {
        s_again = best == kNone && stage < (acc == n ? 1 : 2) && p.sum > 0.f;
        a.accepted[b] = acc;
        a.next[b] = best == kNone ? -1 : (int)(uint32_t)best;
      }
    }
    __syncthreads();
    if (!s_again) return;
  }
}

// ------------------------------------------------------------------------------------------- launches
int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Vectors per row of `z`, one more where a row may start off a 16-byte boundary, and units per row.
int vectors_of(Type type, Logits z, int64_t rows, int V) {
  const int lanes = type == F32 ? 4 : 8;
  const bool aligned = (reinterpret_cast<uintptr_t>(z.p) & 15) == 0 && (rows == 1 || z.ld % lanes == 0);
  return (V + lanes - 1) / lanes + (aligned ? 0 : 1);
}
int splits_of(Type type, Logits z, int64_t rows, int V, int vec = kUnit) {
  return (vectors_of(type, z, rows, V) + vec * kThreads - 1) / (vec * kThreads);
}

// Blocks per row (a cluster) and vectors of each tensor that a block keeps, in the kernels that look twice; `sides` tensors
// share a block. A cluster costs its barriers, so it grows only
//   * until what all running blocks do not keep takes 72 MB of L2's 126, as the second look reads it there (clusters of 1, 2, 4, 8,
//     16: 1024 x 151936 fp32 with gradient 340, 300, 286, 250, 329 us, taken 8; 2048 x 152064 bf16 312, 283, 271, 353,
//     547 us, taken 4; acceptance of 2044 x 32768 fp32 159, 136, 167, 240, 479 us, taken 2);
//   * until one wave of blocks fills the GPU, as long as each thread has a vector (acceptance of 4 x 151936 bf16 46, 27, 18,
//     13, 11 us, taken 16; 64 x 151936 bf16 51, 30, 23, 23, 31 us, taken 8).
struct Plan {
  int cluster, keep, smem;
};
Plan plan_of(Type type, int64_t rows, int V, int sides) {
  const int total = V / (type == F32 ? 4 : 8) + 1;
  const int64_t slots = (sides == 1 ? kRowBlocks : kPairBlocks) * sm_count();
  int c = 1;
  while (c < kMaxCluster && (total * sides / c - kKeep) * 16ll * slots > 72 << 20) c *= 2;
  while (c < kMaxCluster && total * sides > kRowThreads * c && rows * c * 2 <= slots) c *= 2;
  const int per = (total + c - 1) / c, keep = std::min(per, kKeep / sides) / kRound * kRound;
  return {c, keep, keep * sides * 16};
}

struct Shape {
  int64_t blocks;
  int units = 0;               // per row: `blocks` rows of them
  int threads = kThreads, cluster = 1;
  size_t smem = 0;
  bool early = false;          // may start while the kernel before it runs (griddepcontrol.wait orders them)
};
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), const Shape& s, cudaStream_t stream, A... args) {
  if (s.cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  if (s.blocks < 1 || s.blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)s.blocks);
  if (s.units) {
    const unsigned y = (unsigned)std::min<int64_t>(s.blocks, 32768);
    cfg.gridDim = dim3(s.units, y, (unsigned)((s.blocks + y - 1) / y));
  }
  cfg.blockDim = dim3(s.threads);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[3];
  int n = 0;
  if (s.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = s.cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (s.early) {
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

// Hands out the workspace piece by piece, 16-byte aligned.
struct Carver {
  char* p;
  size_t used = 0;
  template <typename T> T* take(size_t n) {
    T* r = reinterpret_cast<T*>(p + used);
    used += (n * sizeof(T) + 15) & ~size_t(15);
    return r;
  }
};
struct TopWork {
  int splits, width;           // units per row, maxima per unit: of the threads that have a vector
  unsigned long long* parts;
  float* tops;
  size_t bytes;
};
TopWork carve_topk(Type type, Logits z, int64_t rows, int V, void* p) {
  Carver c{static_cast<char*>(p)};
  TopWork t{};
  t.splits = splits_of(type, z, rows, V);
  t.width = std::min(vectors_of(type, z, rows, V), kThreads);
  t.parts = c.take<unsigned long long>(rows * t.splits);
  t.tops = c.take<float>(rows * t.splits * t.width);
  t.bytes = c.used;
  return t;
}
KdRows carve_kd(int64_t rows, int k, void* p, size_t& bytes) {
  Carver c{static_cast<char*>(p)};
  KdRows r{};
  r.id = c.take<int>(rows * k);
  r.z = c.take<float>(rows * k);
  r.pt = c.take<float>(rows * k);
  r.sums = c.take<TeacherSums>(rows);
  bytes = c.used;
  return r;
}

}  // namespace

size_t teacher_topk_workspace(Type type, Logits z, int64_t rows, int V) {
  return carve_topk(type, z, rows, V, nullptr).bytes;
}
cudaError_t teacher_topk(Type type, Logits z, int64_t rows, int V, int k, float temp, int32_t* ids, float* lp,
                         void* workspace, cudaStream_t stream) {
  const TopWork w = carve_topk(type, z, rows, V, workspace);
  const int groups = k <= 24 ? 32 : k <= 48 ? 64 : k <= 96 ? 128 : 256;
  const float kl = (float)(kLog2ed / temp);
  Shape units, select;
  units.blocks = select.blocks = rows;
  units.units = w.splits;
  select.early = true;
  return by_type(type, [&](auto t) {
    using T = decltype(t);
    const T* p = static_cast<const T*>(z.p);
    const cudaError_t e = launch(topk_units_kernel<T>, units, stream, p, z.ld, rows, V, w.width, kl, w.parts, w.tops);
    if (e != cudaSuccess) return e;
    return launch(topk_select_kernel<T>, select, stream, p, z.ld, V, w.splits, w.width, k, groups, kl, w.parts, w.tops, ids, lp);
  });
}

size_t kd_topk_loss_workspace(Type type, Logits z, int64_t rows, int V) {
  return rows * splits_of(type, z, rows, V) * sizeof(unsigned long long);
}
cudaError_t kd_topk_loss(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, float* loss, float* stats,
                         void* workspace, cudaStream_t stream) {
  const int splits = splits_of(type, z, rows, V);
  unsigned long long* words = static_cast<unsigned long long*>(workspace);
  Shape parts, last;
  parts.blocks = last.blocks = rows;
  parts.units = splits;
  last.threads = 32;
  last.early = true;
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    const T* p = static_cast<const T*>(z.p);
    const cudaError_t e = launch(kd_parts_kernel<T>, parts, stream, p, z.ld, rows, V, t, (float)(kLog2ed / temp), words);
    if (e != cudaSuccess) return e;
    return launch(kd_loss_kernel<T>, last, stream, p, z.ld, splits, V, t, (float)(kLog2ed / temp), words, loss,
                  reinterpret_cast<KdSaved*>(stats));
  });
}

static cudaError_t kd_from_stats(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, const float* weight,
                                 const float* stats, void* out, int64_t out_ld, bool early, cudaStream_t stream) {
  Shape s;
  s.blocks = rows;
  s.units = splits_of(type, z, rows, V);
  s.early = early;
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    return launch(kd_bwd_kernel<T>, s, stream, static_cast<const T*>(z.p), z.ld, rows, V, t, (float)(kLog2ed / temp),
                  1.f / temp, weight, reinterpret_cast<const KdSaved*>(stats), static_cast<T*>(out), out_ld);
  });
}

// Logits that fit in L2 are read from there the second time whichever block does it, and two grids of units then beat one of
// clusters (192 x 151936 fp32, 117 MB: 62 us, 74 in clusters; 64 x 152064 bf16: 21 and 26 us); more come from memory again (256
// x 151936 fp32, 156 MB: 83 us, 77 in clusters).
static bool kd_in_l2(Type type, int64_t rows, int V) {
  int dev = 0, l2 = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&l2, cudaDevAttrL2CacheSize, dev);
  return rows * V * (type == F32 ? 4 : 2) <= l2;
}
size_t kd_topk_grad_workspace(Type type, Logits z, int64_t rows, int V, int k) {
  if (kd_in_l2(type, rows, V)) return rows * sizeof(KdSaved) + kd_topk_loss_workspace(type, z, rows, V);
  size_t bytes;
  carve_kd(rows, k, nullptr, bytes);
  return bytes;
}
cudaError_t kd_topk_grad(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, const float* weight,
                         float* loss, void* out, int64_t out_ld, void* workspace, cudaStream_t stream) {
  if (kd_in_l2(type, rows, V)) {
    float* stats = static_cast<float*>(workspace);
    const cudaError_t e = kd_topk_loss(type, z, rows, V, t, temp, loss, stats, stats + rows * kKdStats, stream);
    return e != cudaSuccess ? e : kd_from_stats(type, z, rows, V, t, temp, weight, stats, out, out_ld, true, stream);
  }
  size_t bytes;
  const KdRows r = carve_kd(rows, t.k, workspace, bytes);
  const Plan p = plan_of(type, rows, V, 1);
  Shape prepare, grad;
  prepare.blocks = rows;
  prepare.threads = 32;
  grad.blocks = rows * p.cluster;
  grad.threads = kRowThreads;
  grad.cluster = p.cluster;
  grad.smem = p.smem;
  grad.early = true;
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    const T* src = static_cast<const T*>(z.p);
    const float kl = (float)(kLog2ed / temp);
    const cudaError_t e = launch(kd_prepare_kernel<T>, prepare, stream, src, z.ld, V, t, kl, 1.f / temp, weight, r);
    if (e != cudaSuccess) return e;
    return launch(kd_grad_kernel<T>, grad, stream, src, z.ld, V, p.keep, t.k, kl, loss, static_cast<T*>(out), out_ld, r);
  });
}
cudaError_t kd_topk_bwd(Type type, Logits z, int64_t rows, int V, Teacher t, float temp, const float* weight,
                        const float* stats, void* out, int64_t out_ld, cudaStream_t stream) {
  return kd_from_stats(type, z, rows, V, t, temp, weight, stats, out, out_ld, false, stream);
}

cudaError_t accept_kl(Type type, Logits draft, Logits target, int64_t rows, int V, float temp, float* alpha, float* kl,
                      float* stats, cudaStream_t stream) {
  const Plan p = plan_of(type, rows, V, 2);
  Shape s;
  s.blocks = rows * p.cluster;
  s.threads = kRowThreads;
  s.cluster = p.cluster;
  s.smem = p.smem;
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    return launch(accept_kernel<T>, s, stream, static_cast<const T*>(draft.p), draft.ld, static_cast<const T*>(target.p),
                  target.ld, V, p.keep, (float)(kLog2ed / temp), alpha, kl, reinterpret_cast<AcceptRow*>(stats));
  });
}
cudaError_t accept_kl_bwd(Type type, Logits draft, Logits target, int64_t rows, int V, float temp, const float* stats,
                          const float* g_alpha, const float* g_kl, void* out, int64_t out_ld, cudaStream_t stream) {
  Shape s;
  s.blocks = rows;
  s.units = splits_of(type, draft, rows, V, kPairVec);
  return by_type(type, [&](auto x) {
    using T = decltype(x);
    return launch(accept_bwd_kernel<T>, s, stream, static_cast<const T*>(draft.p), draft.ld,
                  static_cast<const T*>(target.p), target.ld, rows, V, (float)(kLog2ed / temp), 1.f / temp,
                  reinterpret_cast<const AcceptRow*>(stats), g_alpha, g_kl, static_cast<T*>(out), out_ld);
  });
}

namespace {
struct VerifyPlan {
  int splits, rows;            // units per row; rows per sequence
};
VerifyPlan verify_plan(const Verify& a) {
  const int lanes = a.type == F32 ? 4 : 8, total = (a.V + lanes - 1) / lanes + 1;
  return {(total + kUnit * kThreads - 1) / (kUnit * kThreads), a.draft_logits ? 2 * a.k + 1 : a.k + 1};
}
}  // namespace

size_t spec_verify_workspace(const Verify& a) {
  const VerifyPlan p = verify_plan(a);
  return ((size_t)a.batch * p.rows * p.splits + 2 * a.batch) * 8;
}

cudaError_t spec_verify(const Verify& a, cudaStream_t stream) {
  const VerifyPlan p = verify_plan(a);
  return by_type(a.type, [&](auto x) {
    using T = decltype(x);
    Shape parts, draw;
    parts.blocks = a.batch * p.rows * p.splits;
    const cudaError_t e = launch(verify_parts_kernel<T>, parts, stream, a, p.splits);
    if (e != cudaSuccess) return e;
    // as many blocks as run at once over all sequences, each of at least one vector per thread
    const int total = (a.V + Vec<T>::N - 1) / Vec<T>::N + 1;
    const int64_t most = (total + kDrawThreads - 1) / kDrawThreads, want = std::max<int64_t>(1, (5 * sm_count()) / a.batch);
    const int c = (int)std::min(most, want);
    draw.blocks = a.batch * c;
    draw.threads = kDrawThreads;
    draw.early = true;
    return launch(verify_draw_kernel<T>, draw, stream, a, p.splits, c, (total + c - 1) / c);
  });
}

}  // namespace vocab
}  // namespace fw
