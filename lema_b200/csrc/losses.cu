// losses.cu — training losses over vocabulary logits and their gradients:
//
//   token_logprobs   lp_t = log softmax(x_t / tau)[l_t], and its backward
//                    dx_v = (g_t / tau) (1[v = l_t] - q_v),  q = softmax(x_t / tau)
//   preference       sequences 0..P-1 chosen, P..2P-1 rejected;
//                    R_b = sum_t (lp_bt - ref_bt), h_p = beta (R_p - R_{P+p}),
//                    L = mean_p (1 - e) softplus(-h_p) + e softplus(h_p)
//   policy           r = exp(lp - old), d = ref - lp,
//                    L = sum_t w_t [-min(r A, clip(r, 1 - lo, 1 + hi) A) + kl (e^d - 1 - d)],
//                    w = 1 / N over the counted tokens, or 1 / (B n_b) per sequence
//   distill          p = softmax(teacher_k / tau) over the teacher's K logits,
//                    L = tau^2 mean_t sum_k p_k (log p_k - log q_{id_k}),
//                    dx_v = (tau / N) (q_v - sum_{k: id_k = v} p_k)
//
// Every gradient row is a scalar times (softmax - a few point masses), so all four share one
// row pass: the row's maximum m and sum s of exp((x - m) / tau), the objective's few numbers,
// and the row of q = exp((x - m) / tau) / s written once. Rows that do not count (a target of
// ignore_index, a false mask) are not read; their gradient row is zero.
//
// Precision: exponentials and their sum in fp32; what is computed once per token (the
// log-probability, ratios, KL terms, sums over tokens) in fp64, since losses are differences
// of nearly equal log-probabilities; every output rounded once.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "internal.h"
#include "ptx.cuh"
#include "quant_core.cuh"

namespace lema {
namespace {

constexpr int kMaxTeacher = 1024;

// Rows of logits: row r starts (r / n1) * ld0 + (r % n1) * ld1 elements behind the base.
struct RowMap {
  int64_t n1, ld0, ld1;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return (r / n1) * ld0 + (r % n1) * ld1;
  }
};

// Workspace: head, counted rows of each sequence, partial sums of token_kernel's CTAs, what
// each row leaves for it.
struct WsHead {
  int64_t total;    // rows that count
  uint32_t ticket;  // CTAs of token_kernel / pair_kernel that are done
};
constexpr int64_t kWsHead = 256;
constexpr int kTokenThreads = 256;

// What one row leaves behind: its maximum m, s = sum exp((x - m) / tau), the target's logit
// (distill: the teacher's sum of exponentials), and for distill sum_k p'_k ((t_k - t_max) -
// (x_k - m)) over the unnormalised weights p'.
struct RowStat {
  float m, s, x, unused;
  double a;
};

struct RowArgs {
  const void* x;
  RowMap in;
  int64_t T;
  int32_t V;
  double inv_tau;                // 1 / tau
  float c;                       // log2(e) / tau
  const int64_t* targets;        // [T]; null for distill
  int64_t ignore;
  float* logps;                  // [T]
  float2* stats;                 // [T] (m, 1 / s), may be null
  float* coef;                   // [T], may be null: dL/dlp (policy), row weight (distill)
  RowStat* row;                  // [T]
  double* lp64;                  // [T] log-probabilities (preference)
  double2* part;                 // (loss, kl) of each CTA of token_kernel / of each pair
  void* dx;                      // null: no gradient
  RowMap out;
  float grad_scale;
  int32_t* err;
  WsHead* head;
  int32_t* seq_count;            // [n0] counted rows of each sequence
  float* loss;
  float* kl;
  // policy
  const float* old_logps;
  const float* adv;
  int64_t adv_s0, adv_s1;
  const float* ref_logps;
  double clip_lo, clip_hi, kl_coef;
  int32_t per_sequence;
  int64_t n0;
  // distill
  const void* teacher_ids;
  int32_t ids_i32;
  const void* teacher_logits;
  int32_t tl_f32;
  int32_t K;
  const uint8_t* mask;           // [T], may be null
  // backward from saved statistics
  const float* g;                // [T] gradient of each row's log-probability (or row weight)
  const float* upstream;         // scalar, may be null
};

enum Objective { kLogp = 0, kPolicy = 1, kDistill = 2 };

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// ---- 16-byte vectors of a row ---------------------------------------------------
// A row may start at any element. It is read as the aligned 16-byte vectors that hold it: the
// first and the last may also hold neighbours' elements, which are replaced by -inf (they
// share a 16-byte granule with the row, so the load stays inside the allocation's pages).

template <typename T>
struct Vec;
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kE = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {  // i < 4
    return f2_from_bf16x2(i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)));
  }
  static __device__ __forceinline__ float max(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 pack(const uint64_t (&p)[4]) {
    return make_uint4(bf16x2_from_f2(p[0]), bf16x2_from_f2(p[1]), bf16x2_from_f2(p[2]),
                      bf16x2_from_f2(p[3]));
  }
};
template <>
struct Vec<float> {
  static constexpr int kE = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {  // i < 2
    return i == 0 ? f2_pack(__uint_as_float(v.x), __uint_as_float(v.y))
                  : f2_pack(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ float max(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                 fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint4 pack(const uint64_t (&p)[2]) {
    float a, b, c, d;
    f2_unpack(p[0], a, b);
    f2_unpack(p[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c),
                      __float_as_uint(d));
  }
};

template <typename T>
struct Span {
  const uint4* v0;  // the row's first aligned vector
  int lead;         // elements in front of the row in it
  int nvec;
  int V;
  __device__ __forceinline__ Span(const T* x, int V_) : V(V_) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(x);
    v0 = reinterpret_cast<const uint4*>(p & ~uintptr_t{15});
    lead = static_cast<int>((p & 15u) / sizeof(T));
    nvec = (lead + V + Vec<T>::kE - 1) / Vec<T>::kE;
  }
  // Elements of vector v outside the row become -inf.
  __device__ __forceinline__ void clean(uint4& w, int v) const {
    if (v == 0 || v == nvec - 1) {
      T e[Vec<T>::kE];
      *reinterpret_cast<uint4*>(e) = w;
      const T neg_inf = static_cast<T>(-INFINITY);
#pragma unroll
      for (int j = 0; j < Vec<T>::kE; ++j) {
        const int i = v * Vec<T>::kE + j - lead;
        if (i < 0 || i >= V) e[j] = neg_inf;
      }
      w = *reinterpret_cast<const uint4*>(e);
    }
  }
};

__device__ __forceinline__ uint4 ld16(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// exp((x - m) / tau) of a vector's elements, as packed fp32 pairs: the maximum is taken off
// first, so that rows of the type's lowest value stay finite.
template <typename T>
__device__ __forceinline__ void exp_vec(const uint4& w, uint64_t neg_m2, uint64_t c2,
                                        uint64_t (&e)[Vec<T>::kE / 2]) {
#pragma unroll
  for (int i = 0; i < Vec<T>::kE / 2; ++i) {
    float lo, hi;
    f2_unpack(f2_mul(f2_add(Vec<T>::pair(w, i), neg_m2), c2), lo, hi);
    e[i] = f2_pack(ex2(lo), ex2(hi));
  }
}

// Writes vector v (elements of a row at `dst`, whose phase within 16 bytes is the input row's
// when SAME): whole vectors at once, the row's ends element by element.
template <typename T>
__device__ __forceinline__ void store_vec(T* dst, const Span<T>& sp, int v, const uint4& w,
                                          bool same) {
  const int i0 = v * Vec<T>::kE - sp.lead;
  if (same && i0 >= 0 && i0 + Vec<T>::kE <= sp.V) {
    *reinterpret_cast<uint4*>(dst + i0) = w;
  } else {
    T e[Vec<T>::kE];
    *reinterpret_cast<uint4*>(e) = w;
#pragma unroll
    for (int j = 0; j < Vec<T>::kE; ++j)
      if (i0 + j >= 0 && i0 + j < sp.V) dst[i0 + j] = e[j];
  }
}

template <typename T>
__device__ __forceinline__ bool same_phase(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15u) == 0;
}

// Adds k to element i of the row (a point mass) if vector v holds it.
template <typename T>
__device__ __forceinline__ void add_mass(uint64_t (&g)[Vec<T>::kE / 2], int at, float k) {
  // `at`: the element's place in the vector, outside [0, kE) for all but one vector
#pragma unroll
  for (int i = 0; i < Vec<T>::kE / 2; ++i) {
    float lo, hi;
    f2_unpack(g[i], lo, hi);
    lo += at == 2 * i ? k : 0.f;
    hi += at == 2 * i + 1 ? k : 0.f;
    g[i] = f2_pack(lo, hi);
  }
}

// ---- reductions ------------------------------------------------------------------

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ double block_sum_d(double v, double* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) r += red[w];
  return r;
}

// Maximum and sum of a row from each thread's (m, s); every thread gets both. The threads'
// sums are added in fp64.
template <int THREADS>
__device__ __forceinline__ void block_combine(float& m, double& s, float c, float* redf,
                                              double* redd) {
  const float mt = m;
  m = warp_max(m);
  if (THREADS > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) redf[threadIdx.x >> 5] = m;
    __syncthreads();
    m = redf[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) m = fmaxf(m, redf[w]);
  }
  // a thread that saw only -inf adds nothing; a row of -inf alone becomes NaN
  s *= static_cast<double>(ex2((mt - m) * c));
  s = warp_sum(s);
  if (THREADS > 32) {
    if ((threadIdx.x & 31) == 0) redd[threadIdx.x >> 5] = s;
    __syncthreads();
    s = redd[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) s += redd[w];
  }
}

// One thread's share of a row's maximum and sum: vectors tid, tid + STEP, ..., in one sweep with
// a running maximum, U loads in flight.
template <typename T, int STEP, int U>
__device__ __forceinline__ void thread_stats(const Span<T>& sp, int tid, float c, float& m,
                                             double& s) {
  m = -INFINITY;
  float sum = 0.f;
  const uint64_t c2 = f2_splat(c);
  for (int base = tid; base < sp.nvec; base += STEP * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = base + u * STEP;
      if (v < sp.nvec)
        w[u] = ld16(sp.v0 + v);
      else
        w[u] = make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
    }
    float mx = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      sp.clean(w[u], base + u * STEP);
      mx = fmaxf(mx, Vec<T>::max(w[u]));
    }
    const float mm = mx == -INFINITY ? 0.f : mx;
    sum *= ex2((m - mm) * c);
    m = mx;
    const uint64_t neg_m2 = f2_splat(-mm);
    uint64_t acc = f2_splat(0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint64_t e[Vec<T>::kE / 2];
      exp_vec<T>(w[u], neg_m2, c2, e);
#pragma unroll
      for (int i = 0; i < Vec<T>::kE / 2; ++i) acc = f2_add(acc, e[i]);
    }
    float lo, hi;
    f2_unpack(acc, lo, hi);
    sum += lo + hi;
  }
  s = static_cast<double>(sum);
}

__device__ __forceinline__ int64_t teacher_id(const RowArgs& a, int64_t i) {
  return a.ids_i32 ? static_cast<const int32_t*>(a.teacher_ids)[i]
                   : static_cast<const int64_t*>(a.teacher_ids)[i];
}
__device__ __forceinline__ float teacher_logit(const RowArgs& a, int64_t i) {
  return a.tl_f32 ? static_cast<const float*>(a.teacher_logits)[i]
                  : __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher_logits)[i]);
}

__device__ __forceinline__ bool row_counts(const RowArgs& a, int64_t r, int64_t& target) {
  if (a.targets == nullptr) return a.mask == nullptr || a.mask[r] != 0;
  target = a.targets[r];
  return target != a.ignore;
}

// log(1 + e^x) without overflow.
__device__ __forceinline__ double softplus(double x) {
  return fmax(x, 0.0) + log1p(exp(-fabs(x)));
}

// 1 / (the number of tokens a token's term is divided by).
__device__ __forceinline__ double token_weight(const RowArgs& a, int64_t r) {
  const int64_t n = a.per_sequence ? a.n0 * a.seq_count[r / a.in.n1] : a.head->total;
  return 1.0 / static_cast<double>(n);
}

// dL/dlp of one token of the clipped policy loss over its weight, and (LOSS) its loss and KL.
// F = double for what is returned, float for the gradient's coefficient.
template <typename F, bool LOSS>
__device__ __forceinline__ F policy_token(const RowArgs& a, int64_t r, F lp, F* loss, F* kl) {
  const int64_t b = r / a.in.n1, t = r % a.in.n1;
  const F A = a.adv[b * a.adv_s0 + t * a.adv_s1];
  // on-policy the ratio is 1, and NaN for a log-probability that is not finite
  const F ratio = exp(lp - (a.old_logps ? static_cast<F>(a.old_logps[r]) : lp));
  const F lo = static_cast<F>(1.0 - a.clip_lo), hi = static_cast<F>(1.0 + a.clip_hi);
  const F bent = ratio < lo ? lo : (ratio > hi ? hi : ratio);  // a NaN ratio stays NaN
  const F plain = ratio * A, clipped = bent * A;
  const bool use_plain = !(clipped < plain);
  F coef = use_plain ? -plain : F(0);
  F d_kl = F(0);
  if (a.ref_logps) {
    const F d = static_cast<F>(a.ref_logps[r]) - lp;
    const F e = expm1(d);
    d_kl = e - d;
    coef -= static_cast<F>(a.kl_coef) * e;
  }
  if (LOSS) {
    *kl = d_kl;
    *loss = static_cast<F>(a.kl_coef) * d_kl - (use_plain ? plain : clipped);
  }
  return coef;
}

// ---- kernels ---------------------------------------------------------------------

// Counts the rows that enter the loss: in all, and for each sequence of n1 rows. Clears the
// ticket.
__global__ void __launch_bounds__(1024) count_kernel(RowArgs a) {
  __shared__ double red[32];
  if (a.seq_count != nullptr && a.per_sequence)
    for (int64_t b = threadIdx.x; b < a.n0; b += blockDim.x) a.seq_count[b] = 0;
  if (threadIdx.x == 0) a.head->ticket = 0;
  __syncthreads();
  double n = 0;
  for (int64_t r0 = 0; r0 < a.T; r0 += blockDim.x) {
    const int64_t r = r0 + threadIdx.x;
    int64_t target;
    if (r < a.T && row_counts(a, r, target)) {
      n += 1;
      if (a.per_sequence) atomicAdd(&a.seq_count[r / a.in.n1], 1);
    }
  }
  const double total = block_sum_d(n, red);
  if (threadIdx.x == 0) a.head->total = static_cast<int64_t>(total);
}

// A row that does not count.
template <typename T, int THREADS>
__device__ __forceinline__ void zero_row(const RowArgs& a, int64_t r, int tid) {
  if (tid == 0) {
    if (a.logps) a.logps[r] = 0.f;
    if (a.stats) a.stats[r] = make_float2(0.f, 0.f);
    if (a.coef) a.coef[r] = 0.f;
  }
  if (a.dx == nullptr) return;
  T* dx = static_cast<T*>(a.dx) + a.out.at(r);
  const Span<T> so(dx, a.V);
  for (int v = tid; v < so.nvec; v += THREADS)
    store_vec<T>(dx, so, v, make_uint4(0u, 0u, 0u, 0u), true);
}

// token_logprobs: one CTA a row.
constexpr int kStatThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kStatThreads) logprobs_kernel(RowArgs a) {
  __shared__ float redf[kStatThreads / 32];
  __shared__ double redd[kStatThreads / 32];
  const int tid = threadIdx.x;
  for (int64_t r = blockIdx.x; r < a.T; r += gridDim.x) {
    int64_t target;
    if (!row_counts(a, r, target)) {
      zero_row<T, kStatThreads>(a, r, tid);
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    const bool ok = target >= 0 && target < a.V;
    const float xt = ok ? to_f(x[target]) : 0.f;
    const Span<T> sp(x, a.V);
    float m;
    double s;
    thread_stats<T, kStatThreads, 4>(sp, tid, a.c, m, s);
    block_combine<kStatThreads>(m, s, a.c, redf, redd);
    if (tid == 0) {
      const double lp = ok ? (static_cast<double>(xt) - m) * a.inv_tau - log(s) : NAN;
      if (!ok) atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
      a.logps[r] = static_cast<float>(lp);
      if (a.lp64) a.lp64[r] = lp;
      if (a.stats) a.stats[r] = make_float2(m, static_cast<float>(1.0 / s));
    }
  }
}

// The teacher's entries of a row: unnormalised weights, indices (-1: no weight) and the
// student's logits there. Returns the sum of the weights; *a_sum the row's share of
// RowStat::a, *any false for a row without an entry, *bad whether an index is outside the
// vocabulary.
template <typename T, int THREADS>
__device__ __forceinline__ double teacher_row(const RowArgs& a, int64_t r, const T* x, float m,
                                              int tid, float* s_p, int32_t* s_id, float* s_x,
                                              float* redf, double* redd, double* a_sum, bool* any,
                                              bool* bad) {
  float tm = -INFINITY;
  bool entry = false, wrong = false;
  for (int k = tid; k < a.K; k += THREADS) {
    const float t = teacher_logit(a, r * a.K + k);
    s_p[k] = t;
    entry |= t != -INFINITY;
    tm = fmaxf(tm, t);
  }
  tm = warp_max(tm);
  *any = __syncthreads_or(entry);
  if ((threadIdx.x & 31) == 0) redf[threadIdx.x >> 5] = tm;
  __syncthreads();
  tm = redf[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) tm = fmaxf(tm, redf[w]);
  double sum = 0.0, acc = 0.0;
  for (int k = tid; k < a.K; k += THREADS) {
    const float t = s_p[k];
    int32_t keep = -1;
    float p = 0.f;
    if (*any && t != -INFINITY) {
      const double d = static_cast<double>(t) - tm;
      p = static_cast<float>(exp(d * a.inv_tau));
      sum += static_cast<double>(p);
      const int64_t id = teacher_id(a, r * a.K + k);
      if (id < 0 || id >= a.V) {
        wrong = true;
      } else if (p != 0.f) {
        const float xv = to_f(x[id]);
        acc += static_cast<double>(p) * (d - (static_cast<double>(xv) - m));
        keep = static_cast<int32_t>(id);
        s_x[k] = xv;
      }
    }
    s_id[k] = keep;
    s_p[k] = p;
  }
  *bad = __syncthreads_or(wrong);
  *a_sum = block_sum_d(acc, redd);
  return block_sum_d(sum, redd);
}

// Adds the teacher's weights to a row whose k q has been written: entries that repeat an
// index write the same value, summed in the same order.
template <typename T, int THREADS>
__device__ __forceinline__ void teacher_masses(const RowArgs& a, T* dx, int tid, const float* s_p,
                                               const int32_t* s_id, const float* s_x, float m,
                                               float inv_s, float inv_t, float k) {
  for (int j = tid; j < a.K; j += THREADS) {
    const int32_t id = s_id[j];
    if (id < 0) continue;
    float p = 0.f;
    for (int i = 0; i < a.K; ++i) p += s_id[i] == id ? s_p[i] : 0.f;
    put(dx + id, k * (ex2((s_x[j] - m) * a.c) * inv_s - p * inv_t));
  }
}

// Gradient rows: k (1[v = target] - q_v), or for distill k (q_v - p_v). Rows are swept twice;
// the second sweep finds them in L2.
constexpr int kRowThreads = 512;
template <typename T, int OBJ>
__global__ void __launch_bounds__(kRowThreads) rows_kernel(RowArgs a) {
  __shared__ float redf[kRowThreads / 32];
  __shared__ double redd[kRowThreads / 32];
  __shared__ float s_p[OBJ == kDistill ? kMaxTeacher : 1];
  __shared__ int32_t s_id[OBJ == kDistill ? kMaxTeacher : 1];
  __shared__ float s_x[OBJ == kDistill ? kMaxTeacher : 1];
  const int tid = threadIdx.x;
  for (int64_t r = blockIdx.x; r < a.T; r += gridDim.x) {
    int64_t target = -1;
    if (!row_counts(a, r, target)) {
      zero_row<T, kRowThreads>(a, r, tid);
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    const Span<T> sp(x, a.V);
    const bool ok = OBJ == kDistill || (target >= 0 && target < a.V);
    const float xt = OBJ != kDistill && ok ? to_f(x[target]) : 0.f;
    float m;
    double s;
    thread_stats<T, kRowThreads, 4>(sp, tid, a.c, m, s);
    block_combine<kRowThreads>(m, s, a.c, redf, redd);
    const float inv_s = static_cast<float>(1.0 / s);
    float k, inv_t = 0.f;
    if (OBJ == kDistill) {
      bool any, bad;
      double acc;
      const double tsum = teacher_row<T, kRowThreads>(a, r, x, m, tid, s_p, s_id, s_x, redf, redd,
                                                      &acc, &any, &bad);
      inv_t = static_cast<float>(1.0 / tsum);
      const float w = any ? static_cast<float>(token_weight(a, r) / a.inv_tau) : 0.f;
      k = bad ? NAN : w;
      if (tid == 0) {
        if (bad) atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
        if (a.coef) a.coef[r] = k;
        a.row[r] = RowStat{m, static_cast<float>(s), any ? static_cast<float>(tsum) : 0.f, 0.f,
                           bad ? NAN : acc};
      }
    } else {
      const float lp = ok ? static_cast<float>((static_cast<double>(xt) - m) * a.inv_tau) -
                                logf(static_cast<float>(s))
                          : NAN;
      k = policy_token<float, false>(a, r, lp, nullptr, nullptr) *
          static_cast<float>(token_weight(a, r) * a.inv_tau);
      if (tid == 0) {
        if (!ok) atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
        a.row[r] = RowStat{m, static_cast<float>(s), ok ? xt : NAN, 0.f, 0.0};
      }
    }
    if (tid == 0 && a.stats) a.stats[r] = make_float2(m, inv_s);
    if (a.dx == nullptr) continue;
    k *= a.grad_scale;
    T* dx = static_cast<T*>(a.dx) + a.out.at(r);
    const bool same = same_phase<T>(x, dx);
    if (k == 0.f) {
      const Span<T> so(dx, a.V);
      for (int v = tid; v < so.nvec; v += kRowThreads)
        store_vec<T>(dx, so, v, make_uint4(0u, 0u, 0u, 0u), true);
      __syncthreads();
      continue;
    }
    const uint64_t neg_m2 = f2_splat(-m), c2 = f2_splat(a.c);
    const uint64_t kq2 = f2_splat(OBJ == kDistill ? k * inv_s : -k * inv_s);
    const int at = OBJ == kDistill ? -1 : static_cast<int>(target) + sp.lead;
    for (int v = tid; v < sp.nvec; v += kRowThreads) {
      const uint4 w = ld16(sp.v0 + v);
      uint64_t e[Vec<T>::kE / 2];
      exp_vec<T>(w, neg_m2, c2, e);
#pragma unroll
      for (int i = 0; i < Vec<T>::kE / 2; ++i) e[i] = f2_mul(e[i], kq2);
      if (OBJ != kDistill && at / Vec<T>::kE == v) add_mass<T>(e, at - v * Vec<T>::kE, k);
      store_vec<T>(dx, sp, v, Vec<T>::pack(e), same);
    }
    __syncthreads();
    if (OBJ == kDistill) {
      teacher_masses<T, kRowThreads>(a, dx, tid, s_p, s_id, s_x, m, inv_s, inv_t, k);
      __syncthreads();
    }
  }
}

// The tokens' terms in fp64, from what the rows left; the CTAs' sums are added in order by the
// CTA that ends last.
template <int OBJ>
__global__ void __launch_bounds__(kTokenThreads) token_kernel(RowArgs a) {
  __shared__ double red[kTokenThreads / 32];
  __shared__ bool s_last;
  const int64_t r = blockIdx.x * static_cast<int64_t>(kTokenThreads) + threadIdx.x;
  double loss = 0.0, kl = 0.0;
  int64_t target;
  if (r < a.T && row_counts(a, r, target)) {
    const RowStat st = a.row[r];
    const double w = token_weight(a, r);
    const double log_s = log(static_cast<double>(st.s));
    if (OBJ == kDistill) {
      // sum_k p_k (log p_k - log q_k), p_k = p'_k / t
      const double t = st.x;
      if (t != 0.0)
        loss = w / (a.inv_tau * a.inv_tau) * (st.a / t * a.inv_tau - log(t) + log_s);
    } else {
      const double lp = (static_cast<double>(st.x) - st.m) * a.inv_tau - log_s;
      a.logps[r] = static_cast<float>(lp);
      const double coef = policy_token<double, true>(a, r, lp, &loss, &kl);
      if (a.coef) a.coef[r] = static_cast<float>(w * coef);
      loss *= w;
      kl *= w;
    }
  }
  loss = block_sum_d(loss, red);
  kl = block_sum_d(kl, red);
  if (threadIdx.x == 0) {
    a.part[blockIdx.x] = make_double2(loss, kl);
    __threadfence();
    s_last = atomicAdd(&a.head->ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  loss = kl = 0.0;
  for (unsigned i = threadIdx.x; i < gridDim.x; i += kTokenThreads) {
    const double2 p = __ldcg(&a.part[i]);
    loss += p.x;
    kl += p.y;
  }
  loss = block_sum_d(loss, red);
  kl = block_sum_d(kl, red);
  if (threadIdx.x == 0) {
    *a.loss = static_cast<float>(loss);
    if (a.kl) *a.kl = static_cast<float>(kl);
  }
}

// One CTA per pair: the two sequences' summed log ratios, the pair's loss and dL/dlp of its
// tokens.
__global__ void __launch_bounds__(256) pair_kernel(RowArgs a, int64_t P, double beta,
                                                   double smooth, float* rewards) {
  __shared__ double red[8];
  const int64_t p = blockIdx.x, S = a.T / (2 * P);
  double R[2];
  for (int side = 0; side < 2; ++side) {
    const int64_t b = p + side * P;
    double sum = 0.0;
    for (int64_t t = threadIdx.x; t < S; t += blockDim.x) {
      const int64_t r = b * S + t;
      if (a.targets[r] == a.ignore) continue;
      sum += a.lp64[r] - (a.ref_logps ? static_cast<double>(a.ref_logps[r]) : 0.0);
    }
    R[side] = beta * block_sum_d(sum, red);
  }
  const double h = R[0] - R[1];
  // sigma(-h) = 1 / (1 + e^h)
  const double dh = (smooth / (1.0 + exp(-h)) - (1.0 - smooth) / (1.0 + exp(h))) * beta /
                    static_cast<double>(P);
  if (threadIdx.x == 0) {
    rewards[p] = static_cast<float>(R[0]);
    rewards[p + P] = static_cast<float>(R[1]);
    a.part[p] = make_double2(
        ((1.0 - smooth) * softplus(-h) + smooth * softplus(h)) / static_cast<double>(P), 0.0);
  }
  for (int side = 0; side < 2; ++side)
    for (int64_t t = threadIdx.x; t < S; t += blockDim.x) {
      const int64_t r = (p + side * P) * S + t;
      a.coef[r] = a.targets[r] == a.ignore ? 0.f : static_cast<float>(side ? -dh : dh);
    }
}

// The pairs' losses added in a fixed order.
__global__ void __launch_bounds__(256) pair_sum_kernel(const double2* part, int64_t n,
                                                       float* loss) {
  __shared__ double red[8];
  double l = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) l += part[i].x;
  l = block_sum_d(l, red);
  if (threadIdx.x == 0) *loss = static_cast<float>(l);
}

// Gradient rows from saved statistics: k (1[v = target] - q_v). A CTA takes kBwdVecs vectors
// of one row; nothing is reduced, so rows of any length keep every SM busy.
constexpr int kBwdThreads = 256;
constexpr int kBwdU = 4;
constexpr int kBwdVecs = kBwdThreads * kBwdU;
template <typename T>
__global__ void __launch_bounds__(kBwdThreads) logprobs_bwd_kernel(RowArgs a, int chunks) {
  const int tid = threadIdx.x;
  const int64_t units = a.T * chunks;
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const int64_t r = unit / chunks;
    const int v0 = static_cast<int>(unit - r * chunks) * kBwdVecs;
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    T* dx = static_cast<T*>(a.dx) + a.out.at(r);
    const Span<T> sp(x, a.V);
    const int64_t target = a.targets[r];
    const float k = target == a.ignore
                        ? 0.f
                        : a.g[r] * a.grad_scale * (a.upstream ? *a.upstream : 1.f) *
                              static_cast<float>(a.inv_tau);
    const bool same = same_phase<T>(x, dx);
    if (k == 0.f) {
      // zeros need no input: whole vectors of the output's own phase
      const Span<T> so(dx, a.V);
#pragma unroll
      for (int u = 0; u < kBwdU; ++u) {
        const int v = v0 + tid + u * kBwdThreads;
        if (v < so.nvec) store_vec<T>(dx, so, v, make_uint4(0u, 0u, 0u, 0u), true);
      }
      continue;
    }
    uint4 w[kBwdU];
#pragma unroll
    for (int u = 0; u < kBwdU; ++u) {
      const int v = v0 + tid + u * kBwdThreads;
      if (v < sp.nvec) w[u] = ld16(sp.v0 + v);
    }
    const float2 st = a.stats[r];
    const uint64_t neg_m2 = f2_splat(-st.x), c2 = f2_splat(a.c), kq2 = f2_splat(-k * st.y);
    const int64_t at = target + sp.lead;
#pragma unroll
    for (int u = 0; u < kBwdU; ++u) {
      const int v = v0 + tid + u * kBwdThreads;
      if (v >= sp.nvec) continue;
      uint64_t e[Vec<T>::kE / 2];
      exp_vec<T>(w[u], neg_m2, c2, e);
#pragma unroll
      for (int i = 0; i < Vec<T>::kE / 2; ++i) e[i] = f2_mul(e[i], kq2);
      if (at / Vec<T>::kE == v) add_mass<T>(e, static_cast<int>(at - v * Vec<T>::kE), k);
      store_vec<T>(dx, sp, v, Vec<T>::pack(e), same);
    }
  }
}

// distill's gradient rows from saved statistics.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) distill_bwd_kernel(RowArgs a) {
  __shared__ float redf[kRowThreads / 32];
  __shared__ double redd[kRowThreads / 32];
  __shared__ float s_p[kMaxTeacher];
  __shared__ int32_t s_id[kMaxTeacher];
  __shared__ float s_x[kMaxTeacher];
  const int tid = threadIdx.x;
  const float up = a.upstream ? *a.upstream : 1.f;
  for (int64_t r = blockIdx.x; r < a.T; r += gridDim.x) {
    int64_t target;
    const float k = row_counts(a, r, target) ? a.g[r] * up : 0.f;
    if (k == 0.f) {
      zero_row<T, kRowThreads>(a, r, tid);
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    T* dx = static_cast<T*>(a.dx) + a.out.at(r);
    const Span<T> sp(x, a.V);
    const bool same = same_phase<T>(x, dx);
    const float2 st = a.stats[r];
    bool any, bad;
    double acc;
    const double tsum = teacher_row<T, kRowThreads>(a, r, x, st.x, tid, s_p, s_id, s_x, redf, redd,
                                                    &acc, &any, &bad);
    const uint64_t neg_m2 = f2_splat(-st.x), c2 = f2_splat(a.c), kq2 = f2_splat(k * st.y);
    for (int v = tid; v < sp.nvec; v += kRowThreads) {
      const uint4 w = ld16(sp.v0 + v);
      uint64_t e[Vec<T>::kE / 2];
      exp_vec<T>(w, neg_m2, c2, e);
#pragma unroll
      for (int i = 0; i < Vec<T>::kE / 2; ++i) e[i] = f2_mul(e[i], kq2);
      store_vec<T>(dx, sp, v, Vec<T>::pack(e), same);
    }
    __syncthreads();
    teacher_masses<T, kRowThreads>(a, dx, tid, s_p, s_id, s_x, st.x, st.y,
                                   static_cast<float>(1.0 / tsum), k);
    __syncthreads();
  }
}

// ---- host side ----------------------------------------------------------------

int bad(const char* what) { return set_error(LEMA_ERR_INVALID_ARGUMENT, what); }

// Whether n rows `ld` elements apart stay inside 64-bit offsets.
bool span_ok(int64_t n, int64_t ld) {
  return ld >= 0 && ld <= (int64_t{1} << 60) / std::max<int64_t>(n, 1);
}

// Sizes, strides and temperature shared by every entry point; fills the common fields.
int make_rows(RowArgs& a, const void* x, int64_t n0, int64_t n1, int64_t ld0, int64_t ld1,
              int64_t V, double temperature) {
  a = RowArgs{};
  if (n0 < 0 || n1 < 0) return bad("negative row count");
  if (V <= 0 || V > (1 << 30)) return bad("vocabulary size must be in [1, 2^30]");
  if (!(temperature >= 1e-6 && temperature <= 1e6))
    return bad("temperature must be in [1e-6, 1e6]");
  if (n0 > 0 && n1 > INT32_MAX / n0)
    return set_error(LEMA_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  if (n0 * n1 > 0 && x == nullptr) return bad("null logits");
  if (!span_ok(n0, ld0) || !span_ok(n1, ld1)) return bad("row stride negative or past 64 bits");
  a.x = x;
  a.in = RowMap{std::max<int64_t>(n1, 1), ld0, ld1};
  a.out = a.in;
  a.n0 = n0;
  a.T = n0 * n1;
  a.V = static_cast<int32_t>(V);
  a.inv_tau = 1.0 / temperature;
  a.c = static_cast<float>(1.4426950408889634 / temperature);
  a.grad_scale = 1.f;
  return LEMA_OK;
}

int set_out(RowArgs& a, void* dx, int64_t ldd0, int64_t ldd1) {
  if (dx == nullptr) return LEMA_OK;
  if (!span_ok(a.n0, ldd0) || !span_ok(a.in.n1, ldd1))
    return bad("gradient row stride negative or past 64 bits");
  // rows inside a sequence and sequences, either of them outermost
  const int64_t n1 = a.in.n1, inner = (n1 - 1) * ldd1 + a.V, across = (a.n0 - 1) * ldd0 + a.V;
  const bool rows_in_seq = (n1 == 1 || ldd1 >= a.V) && (a.n0 <= 1 || ldd0 >= inner);
  const bool seqs_in_row = (a.n0 <= 1 || ldd0 >= a.V) && (n1 == 1 || ldd1 >= across);
  if (!rows_in_seq && !seqs_in_row) return bad("gradient rows overlap");
  a.dx = dx;
  a.out = RowMap{a.in.n1, ldd0, ldd1};
  return LEMA_OK;
}

int64_t round256(int64_t n) { return (n + 255) / 256 * 256; }

int64_t token_ctas(int64_t T) { return (T + kTokenThreads - 1) / kTokenThreads; }

// Partial sums: one for each CTA of token_kernel, or for each pair.
int64_t parts(int64_t n0, int64_t T) { return std::max(token_ctas(T), n0) + 1; }

int64_t ws_bytes_for(int64_t n0, int64_t T) {
  return kWsHead + round256(n0 * 4) + round256(parts(n0, T) * 16) +
         T * static_cast<int64_t>(sizeof(RowStat));
}

int set_ws(RowArgs& a, void* ws, int64_t ws_bytes) {
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0 ||
      ws_bytes < ws_bytes_for(a.n0, a.T))
    return bad("workspace: 16-byte aligned, at least lema_loss_workspace_bytes(n0, n1) bytes");
  char* p = static_cast<char*>(ws);
  a.head = reinterpret_cast<WsHead*>(p);
  p += kWsHead;
  a.seq_count = reinterpret_cast<int32_t*>(p);
  p += round256(a.n0 * 4);
  a.part = reinterpret_cast<double2*>(p);
  p += round256(parts(a.n0, a.T) * 16);
  a.row = reinterpret_cast<RowStat*>(p);
  a.lp64 = reinterpret_cast<double*>(p);
  return LEMA_OK;
}

unsigned rows_grid(const RowArgs& a) {
  return static_cast<unsigned>(std::min<int64_t>(a.T, 1 << 20));
}

int launch_logprobs(const RowArgs& a, int x_f32, cudaStream_t s) {
  if (x_f32)
    logprobs_kernel<float><<<rows_grid(a), kStatThreads, 0, s>>>(a);
  else
    logprobs_kernel<__nv_bfloat16><<<rows_grid(a), kStatThreads, 0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}

int launch_logprobs_bwd(const RowArgs& a, int x_f32, cudaStream_t s) {
  const int e = x_f32 ? 4 : 8;
  // a misaligned row spans up to one vector more
  const int chunks = static_cast<int>(((a.V + e - 1) / e + 1 + kBwdVecs - 1) / kBwdVecs);
  const int64_t grid = std::min<int64_t>(a.T * chunks, INT32_MAX);
  if (x_f32)
    logprobs_bwd_kernel<float><<<static_cast<unsigned>(grid), kBwdThreads, 0, s>>>(a, chunks);
  else
    logprobs_bwd_kernel<__nv_bfloat16><<<static_cast<unsigned>(grid), kBwdThreads, 0, s>>>(a,
                                                                                        chunks);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}

// Counts, the rows' statistics and gradients, the tokens' terms.
template <int OBJ>
int launch_loss(const RowArgs& a, int x_f32, cudaStream_t s) {
  count_kernel<<<1, 1024, 0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  if (a.T > 0) {
    if (x_f32)
      rows_kernel<float, OBJ><<<rows_grid(a), kRowThreads, 0, s>>>(a);
    else
      rows_kernel<__nv_bfloat16, OBJ><<<rows_grid(a), kRowThreads, 0, s>>>(a);
    LEMA_CUDA_TRY(cudaGetLastError());
  }
  token_kernel<OBJ><<<static_cast<unsigned>(std::max<int64_t>(1, token_ctas(a.T))), kTokenThreads,
                      0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}

// Statistics are read and written as pairs.
int set_stats(RowArgs& a, const float* stats) {
  if ((reinterpret_cast<uintptr_t>(stats) & 7u) != 0) return bad("stats: 8-byte alignment");
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  return LEMA_OK;
}

int need_err(RowArgs& a) {
  a.err = gemm_error_word();
  return a.err ? LEMA_OK : set_error(LEMA_ERR_CUDA, "cannot resolve device error word");
}

}  // namespace
}  // namespace lema

using namespace lema;

extern "C" int64_t lema_loss_workspace_bytes(int64_t n0, int64_t n1) {
  if (n0 < 0 || n1 < 0 || (n0 > 0 && n1 > INT32_MAX / n0)) return -1;
  return ws_bytes_for(n0, n0 * n1);
}

extern "C" int lema_token_logprobs(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                   int64_t ld0, int64_t ld1, int64_t V, const int64_t* targets,
                                   int64_t ignore_index, double temperature, float* logps,
                                   float* stats, void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (a.T == 0) return LEMA_OK;
  if (!targets || !logps) return bad("null targets or logps");
  if ((rc = need_err(a))) return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  a.logps = logps;
  if ((rc = set_stats(a, stats))) return rc;
  return launch_logprobs(a, x_f32, static_cast<cudaStream_t>(stream));
}

extern "C" int lema_token_logprobs_bwd(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                       int64_t ld0, int64_t ld1, int64_t V,
                                       const int64_t* targets, int64_t ignore_index,
                                       double temperature, const float* stats,
                                       const float* dlogps, const float* upstream, void* dx,
                                       int64_t ldd0, int64_t ldd1, void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (a.T == 0) return LEMA_OK;
  if (!targets || !stats || !dlogps || !dx) return bad("null pointer");
  if ((rc = set_out(a, dx, ldd0, ldd1))) return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  if ((rc = set_stats(a, stats))) return rc;
  a.g = dlogps;
  a.upstream = upstream;
  return launch_logprobs_bwd(a, x_f32, static_cast<cudaStream_t>(stream));
}

extern "C" int lema_preference_loss(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                    int64_t ld0, int64_t ld1, int64_t V, const int64_t* targets,
                                    int64_t ignore_index, const float* ref_logps, double beta,
                                    double label_smoothing, double grad_scale, void* ws,
                                    int64_t ws_bytes, float* logps, float* stats, float* coef,
                                    float* loss, float* rewards, void* dx, int64_t ldd0,
                                    int64_t ldd1, void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, n0, n1, ld0, ld1, V, 1.0);
  if (rc) return rc;
  if (n0 == 0 || n0 % 2 != 0) return bad("preference_loss needs chosen and rejected sequences");
  if (!(beta > 0.0) || !std::isfinite(beta)) return bad("beta must be positive");
  if (!(label_smoothing >= 0.0 && label_smoothing < 0.5))
    return bad("label_smoothing must be in [0, 0.5)");
  if (!loss || !rewards || (a.T > 0 && (!targets || !logps || !stats || !coef)))
    return bad("null pointer");
  if ((rc = set_ws(a, ws, ws_bytes)) || (rc = set_out(a, dx, ldd0, ldd1)) || (rc = need_err(a)))
    return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  a.ref_logps = ref_logps;
  a.logps = logps;
  if ((rc = set_stats(a, stats))) return rc;
  a.coef = coef;
  auto s = static_cast<cudaStream_t>(stream);
  if (a.T > 0 && (rc = launch_logprobs(a, x_f32, s))) return rc;
  pair_kernel<<<static_cast<unsigned>(n0 / 2), 256, 0, s>>>(a, n0 / 2, beta, label_smoothing,
                                                            rewards);
  LEMA_CUDA_TRY(cudaGetLastError());
  pair_sum_kernel<<<1, 256, 0, s>>>(a.part, n0 / 2, loss);
  LEMA_CUDA_TRY(cudaGetLastError());
  if (dx == nullptr || a.T == 0) return LEMA_OK;
  a.g = coef;
  a.grad_scale = static_cast<float>(grad_scale);
  return launch_logprobs_bwd(a, x_f32, s);
}

extern "C" int lema_policy_loss(const void* x, int32_t x_f32, int64_t n0, int64_t n1, int64_t ld0,
                                int64_t ld1, int64_t V, const int64_t* targets,
                                int64_t ignore_index, double temperature, const float* old_logps,
                                const float* advantages, int64_t adv_s0, int64_t adv_s1,
                                const float* ref_logps, double clip_lo,
                                double clip_hi, double kl_coef, int32_t per_sequence, double grad_scale, void* ws,
                                int64_t ws_bytes, float* logps, float* stats, float* coef,
                                float* loss, float* kl, void* dx, int64_t ldd0, int64_t ldd1,
                                void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (!(clip_lo >= 0.0 && clip_lo <= 1.0) || !(clip_hi >= 0.0) || !std::isfinite(clip_hi))
    return bad("clip must be in [0, 1] below and finite, >= 0 above");
  if (!(kl_coef >= 0.0) || !std::isfinite(kl_coef)) return bad("kl_coef must be >= 0");
  if (!loss || !kl || (a.T > 0 && (!targets || !advantages || !logps))) return bad("null pointer");
  if ((rc = set_ws(a, ws, ws_bytes)) || (rc = set_out(a, dx, ldd0, ldd1)) || (rc = need_err(a)))
    return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  a.old_logps = old_logps;
  a.adv = advantages;
  a.adv_s0 = adv_s0;
  a.adv_s1 = adv_s1;
  a.ref_logps = ref_logps;
  a.clip_lo = clip_lo;
  a.clip_hi = clip_hi;
  a.kl_coef = kl_coef;
  a.per_sequence = per_sequence;
  a.logps = logps;
  if ((rc = set_stats(a, stats))) return rc;
  a.coef = coef;
  a.grad_scale = static_cast<float>(grad_scale);
  a.loss = loss;
  a.kl = kl;
  return launch_loss<kPolicy>(a, x_f32, static_cast<cudaStream_t>(stream));
}

namespace lema {
namespace {
int set_teacher(RowArgs& a, const void* ids, int32_t ids_i32, const void* logits, int32_t tl_f32,
                int64_t K, const uint8_t* mask) {
  if (K < 1 || K > kMaxTeacher)
    return set_error(LEMA_ERR_UNSUPPORTED, "between 1 and 1024 teacher entries a row");
  if (a.T > 0 && (!ids || !logits)) return bad("null teacher indices or logits");
  a.teacher_ids = ids;
  a.ids_i32 = ids_i32;
  a.teacher_logits = logits;
  a.tl_f32 = tl_f32;
  a.K = static_cast<int32_t>(K);
  a.mask = mask;
  return LEMA_OK;
}
}  // namespace
}  // namespace lema

extern "C" int lema_distill_loss(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                 int64_t ld0, int64_t ld1, int64_t V, const void* teacher_ids,
                                 int32_t ids_i32, const void* teacher_logits, int32_t tl_f32,
                                 int64_t K, const uint8_t* mask, double temperature,
                                 double grad_scale, void* ws, int64_t ws_bytes, float* stats,
                                 float* coef, float* loss, void* dx, int64_t ldd0, int64_t ldd1,
                                 void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (!loss) return bad("null loss");
  if ((rc = set_teacher(a, teacher_ids, ids_i32, teacher_logits, tl_f32, K, mask)) ||
      (rc = set_ws(a, ws, ws_bytes)) || (rc = set_out(a, dx, ldd0, ldd1)) || (rc = need_err(a)))
    return rc;
  if ((rc = set_stats(a, stats))) return rc;
  a.coef = coef;
  a.grad_scale = static_cast<float>(grad_scale);
  a.loss = loss;
  return launch_loss<kDistill>(a, x_f32, static_cast<cudaStream_t>(stream));
}

extern "C" int lema_distill_loss_bwd(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                     int64_t ld0, int64_t ld1, int64_t V,
                                     const void* teacher_ids, int32_t ids_i32,
                                     const void* teacher_logits, int32_t tl_f32, int64_t K,
                                     const uint8_t* mask, double temperature, const float* stats,
                                     const float* coef, const float* upstream, void* dx,
                                     int64_t ldd0, int64_t ldd1, void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if ((rc = set_teacher(a, teacher_ids, ids_i32, teacher_logits, tl_f32, K, mask))) return rc;
  if (a.T == 0) return LEMA_OK;
  if (!stats || !coef || !dx) return bad("null pointer");
  if ((rc = set_out(a, dx, ldd0, ldd1))) return rc;
  if ((rc = set_stats(a, stats))) return rc;
  a.g = coef;
  a.upstream = upstream;
  auto s = static_cast<cudaStream_t>(stream);
  if (x_f32)
    distill_bwd_kernel<float><<<rows_grid(a), kRowThreads, 0, s>>>(a);
  else
    distill_bwd_kernel<__nv_bfloat16><<<rows_grid(a), kRowThreads, 0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}
