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

namespace lema {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTeacher = 1024;

// Rows of logits: row r starts (r / n1) * ld0 + (r % n1) * ld1 elements behind the base.
struct RowMap {
  int64_t n1, ld0, ld1;
  __device__ __forceinline__ int64_t at(int64_t r) const {
    return (r / n1) * ld0 + (r % n1) * ld1;
  }
};

// Workspace header, cleared by count_kernel.
struct WsHead {
  int64_t total;  // rows that count
};
constexpr int64_t kWsHead = 256;

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
  double2* part;                 // [T] (weighted loss, weighted kl) of each row
  void* dx;                      // null: no gradient
  RowMap out;
  float grad_scale;
  int32_t* err;
  const WsHead* head;
  const int32_t* seq_count;      // [n0] counted rows of each sequence
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

template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* red, F f) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) r = f(r, red[w]);
  return r;
}

__device__ __forceinline__ float block_max(float v, float* red) {
  return block_reduce(v, red, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  return block_reduce(v, red, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ double block_sum_d(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = red[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) r += red[w];
  return r;
}

__device__ __forceinline__ int64_t teacher_id(const RowArgs& a, int64_t i) {
  return a.ids_i32 ? static_cast<const int32_t*>(a.teacher_ids)[i]
                   : static_cast<const int64_t*>(a.teacher_ids)[i];
}
__device__ __forceinline__ float teacher_logit(const RowArgs& a, int64_t i) {
  return a.tl_f32 ? static_cast<const float*>(a.teacher_logits)[i]
                  : __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher_logits)[i]);
}

// log(1 + e^x) without overflow.
__device__ __forceinline__ double softplus(double x) {
  return fmax(x, 0.0) + log1p(exp(-fabs(x)));
}

// Weighted loss, weighted KL and dL/dlp of one token of the clipped policy loss.
__device__ __forceinline__ void policy_token(const RowArgs& a, int64_t r, double lp, double w,
                                             double& loss, double& kl, double& coef) {
  const int64_t b = r / a.in.n1, t = r % a.in.n1;
  const double A = a.adv[b * a.adv_s0 + t * a.adv_s1];
  // on-policy the ratio is 1, and NaN for a log-probability that is not finite
  const double ratio = exp(lp - (a.old_logps ? static_cast<double>(a.old_logps[r]) : lp));
  const double lo = 1.0 - a.clip_lo, hi = 1.0 + a.clip_hi;
  // a NaN ratio stays NaN (fmin / fmax would drop it)
  const double bent = ratio < lo ? lo : (ratio > hi ? hi : ratio);
  const double plain = ratio * A, clipped = bent * A;
  const bool use_plain = !(clipped < plain);
  loss = -(use_plain ? plain : clipped);
  coef = use_plain ? -plain : 0.0;
  kl = 0.0;
  if (a.ref_logps) {
    const double d = static_cast<double>(a.ref_logps[r]) - lp;
    const double e = expm1(d);
    kl = e - d;
    coef -= a.kl_coef * e;
  }
  loss = w * (loss + a.kl_coef * kl);
  kl *= w;
  coef *= w;
}

// Counts the rows that enter the loss: in all, and for each sequence of n1 rows.
__global__ void __launch_bounds__(1024) count_kernel(const int64_t* targets, int64_t ignore,
                                                     const uint8_t* mask, int64_t T, int64_t n1,
                                                     int64_t n0, int32_t* seq_count,
                                                     WsHead* head) {
  __shared__ double red[32];
  for (int64_t b = threadIdx.x; b < n0; b += blockDim.x) seq_count[b] = 0;
  __syncthreads();
  double n = 0;
  for (int64_t r0 = 0; r0 < T; r0 += blockDim.x) {
    const int64_t r = r0 + threadIdx.x;
    const bool in = r < T && (targets ? targets[r] != ignore : (!mask || mask[r]));
    if (in) {
      n += 1;
      atomicAdd(&seq_count[r / n1], 1);
    }
  }
  const double total = block_sum_d(n, red);
  if (threadIdx.x == 0) head->total = static_cast<int64_t>(total);
}

template <typename T, int OBJ>
__global__ void __launch_bounds__(kThreads) rows_kernel(RowArgs a) {
  __shared__ float red[kWarps];
  __shared__ double redd[kWarps];
  __shared__ float s_coef;
  __shared__ float s_p[OBJ == kDistill ? kMaxTeacher : 1];
  __shared__ int32_t s_id[OBJ == kDistill ? kMaxTeacher : 1];
  __shared__ float s_x[OBJ == kDistill ? kMaxTeacher : 1];
  const int tid = threadIdx.x;
  for (int64_t r = blockIdx.x; r < a.T; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    T* dx = a.dx ? static_cast<T*>(a.dx) + a.out.at(r) : nullptr;
    bool counts;
    int64_t target = -1;
    if (OBJ == kDistill) {
      counts = !a.mask || a.mask[r];
    } else {
      target = a.targets[r];
      counts = target != a.ignore;
    }
    if (!counts) {
      if (tid == 0) {
        if (a.logps) a.logps[r] = 0.f;
        if (a.stats) a.stats[r] = make_float2(0.f, 0.f);
        if (a.coef) a.coef[r] = 0.f;
        if (a.part) a.part[r] = make_double2(0.0, 0.0);
      }
      if (dx)
        for (int i = tid; i < a.V; i += kThreads) put(dx + i, 0.f);
      continue;
    }
    float m = -INFINITY;
    for (int i = tid; i < a.V; i += kThreads) m = fmaxf(m, to_f(x[i]));
    m = block_max(m, red);
    float s = 0.f;
    for (int i = tid; i < a.V; i += kThreads) s += ex2((to_f(x[i]) - m) * a.c);
    s = block_sum(s, red);
    const float inv_s = 1.f / s;
    if (OBJ == kDistill) {
      float tm = -INFINITY;
      bool bad = false, nan = false;
      for (int k = tid; k < a.K; k += kThreads) {
        const float t = teacher_logit(a, r * a.K + k);
        s_p[k] = t;
        nan |= t != t;
        tm = fmaxf(tm, t);
      }
      tm = block_max(tm, red);
      double tsum = 0.0;
      for (int k = tid; k < a.K; k += kThreads) {
        const double d = (static_cast<double>(s_p[k]) - tm) * a.inv_tau;
        tsum += exp(d);
      }
      tsum = block_sum_d(tsum, redd);
      const double log_t = log(tsum), log_s = log(static_cast<double>(s));
      double kl = 0.0;
      const bool empty = tm == -INFINITY;  // no teacher entry at all (a NaN entry is kept)
      const bool any_nan = __syncthreads_or(nan);
      const bool use = !empty || any_nan;
      for (int k = tid; k < a.K; k += kThreads) {
        const float t = s_p[k];
        const int64_t id = teacher_id(a, r * a.K + k);
        int32_t keep = -1;
        float p = 0.f;
        if (use && t != -INFINITY) {
          const double lt = (static_cast<double>(t) - tm) * a.inv_tau - log_t;
          const double pd = exp(lt);
          if (id < 0 || id >= a.V) {
            bad = true;
          } else if (pd != 0.0) {
            const float xv = to_f(x[id]);
            const double lq =
                (static_cast<double>(xv) - m) * a.inv_tau - log_s;
            kl += pd * (lt - lq);
            p = static_cast<float>(pd);
            keep = static_cast<int32_t>(id);
            s_x[k] = xv;
          }
        }
        s_id[k] = keep;
        s_p[k] = p;
      }
      const bool any_bad = __syncthreads_or(bad);
      kl = block_sum_d(kl, redd);
      if (any_bad) kl = NAN;
      if (tid == 0) {
        const double w = 1.0 / static_cast<double>(a.head->total);
        const double tau = 1.0 / a.inv_tau;
        if (any_bad && a.err) atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
        a.part[r] = make_double2(use ? w * tau * tau * kl : 0.0, 0.0);
        const float coef = any_bad ? NAN : (use ? static_cast<float>(w * tau) : 0.f);
        s_coef = coef;
        if (a.coef) a.coef[r] = coef;
        if (a.stats) a.stats[r] = make_float2(m, inv_s);
      }
    } else if (tid == 0) {
      double lp = NAN;
      if (target >= 0 && target < a.V)
        lp = (static_cast<double>(to_f(x[target])) - m) * a.inv_tau -
             log(static_cast<double>(s));
      else if (a.err)
        atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
      if (a.logps) a.logps[r] = static_cast<float>(lp);
      if (a.stats) a.stats[r] = make_float2(m, inv_s);
      if (OBJ == kPolicy) {
        const int64_t n = a.per_sequence ? a.n0 * a.seq_count[r / a.in.n1] : a.head->total;
        double loss, kl, coef;
        policy_token(a, r, lp, 1.0 / static_cast<double>(n), loss, kl, coef);
        a.part[r] = make_double2(loss, kl);
        if (a.coef) a.coef[r] = static_cast<float>(coef);
        s_coef = static_cast<float>(coef * a.inv_tau);
      }
    }
    if (OBJ == kLogp || dx == nullptr) {
      __syncthreads();
      continue;
    }
    __syncthreads();
    const float k = s_coef * a.grad_scale;
    if (OBJ == kPolicy) {
      // k (1[v = target] - q_v)
      const float kq = k * inv_s;
      for (int i = tid; i < a.V; i += kThreads) {
        const float q = ex2((to_f(x[i]) - m) * a.c) * kq;
        put(dx + i, k == 0.f ? 0.f : (i == target ? k - q : -q));
      }
    } else {
      const float kq = k * inv_s;
      for (int i = tid; i < a.V; i += kThreads)
        put(dx + i, k == 0.f ? 0.f : ex2((to_f(x[i]) - m) * a.c) * kq);
      __syncthreads();
      for (int j = tid; j < a.K; j += kThreads) {
        const int32_t id = s_id[j];
        if (id < 0) continue;
        // entries that repeat an index hold the same sum, added in the same order
        float p = 0.f;
        for (int i = 0; i < a.K; ++i) p += s_id[i] == id ? s_p[i] : 0.f;
        put(dx + id, k * (ex2((s_x[j] - m) * a.c) * inv_s - p));
      }
    }
    __syncthreads();
  }
}

// Loss and KL: the rows' terms added in fp64 in a fixed order.
__global__ void __launch_bounds__(1024) finish_kernel(const double2* part, int64_t n, float* loss,
                                                      float* kl) {
  __shared__ double red[32];
  double l = 0.0, k = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
    l += part[i].x;
    k += part[i].y;
  }
  l = block_sum_d(l, red);
  k = block_sum_d(k, red);
  if (threadIdx.x == 0) {
    *loss = static_cast<float>(l);
    if (kl) *kl = static_cast<float>(k);
  }
}

// One CTA per pair: the two sequences' summed log ratios, the pair's loss and dL/dlp of its
// tokens.
__global__ void __launch_bounds__(256) pair_kernel(RowArgs a, int64_t P, double beta,
                                                   double smooth, double2* part, float* rewards) {
  __shared__ double red[8];
  const int64_t p = blockIdx.x, S = a.T / (2 * P);
  double R[2];
  for (int side = 0; side < 2; ++side) {
    const int64_t b = p + side * P;
    double sum = 0.0;
    for (int64_t t = threadIdx.x; t < S; t += blockDim.x) {
      const int64_t r = b * S + t;
      if (a.targets[r] == a.ignore) continue;
      sum += static_cast<double>(a.logps[r]) -
             (a.ref_logps ? static_cast<double>(a.ref_logps[r]) : 0.0);
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
    part[p] = make_double2(
        ((1.0 - smooth) * softplus(-h) + smooth * softplus(h)) / static_cast<double>(P), 0.0);
  }
  for (int side = 0; side < 2; ++side)
    for (int64_t t = threadIdx.x; t < S; t += blockDim.x) {
      const int64_t r = (p + side * P) * S + t;
      a.coef[r] = a.targets[r] == a.ignore ? 0.f : static_cast<float>(side ? -dh : dh);
    }
}

// Gradient rows from saved statistics: k (1[v = target] - q_v), or k (q_v - sum p) for distill.
template <typename T, int OBJ>
__global__ void __launch_bounds__(kThreads) rows_bwd_kernel(RowArgs a) {
  __shared__ float red[kWarps];
  __shared__ double redd[kWarps];
  __shared__ float s_p[OBJ == kDistill ? kMaxTeacher : 1];
  __shared__ int32_t s_id[OBJ == kDistill ? kMaxTeacher : 1];
  __shared__ float s_x[OBJ == kDistill ? kMaxTeacher : 1];
  const int tid = threadIdx.x;
  const float up = a.grad_scale * (a.upstream ? *a.upstream : 1.f);
  for (int64_t r = blockIdx.x; r < a.T; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    T* dx = static_cast<T*>(a.dx) + a.out.at(r);
    bool counts;
    int64_t target = -1;
    if (OBJ == kDistill) {
      counts = !a.mask || a.mask[r];
    } else {
      target = a.targets[r];
      counts = target != a.ignore;
    }
    float k = counts ? a.g[r] * up : 0.f;
    if (OBJ != kDistill) k *= static_cast<float>(a.inv_tau);
    if (k == 0.f) {
      for (int i = tid; i < a.V; i += kThreads) put(dx + i, 0.f);
      continue;
    }
    const float2 st = a.stats[r];
    const float m = st.x, kq = k * st.y;
    if (OBJ != kDistill) {
      for (int i = tid; i < a.V; i += kThreads) {
        const float q = ex2((to_f(x[i]) - m) * a.c) * kq;
        put(dx + i, i == target ? k - q : -q);
      }
      continue;
    }
    float tm = -INFINITY;
    for (int j = tid; j < a.K; j += kThreads) {
      const float t = teacher_logit(a, r * a.K + j);
      s_p[j] = t;
      tm = fmaxf(tm, t);
    }
    tm = block_max(tm, red);
    double tsum = 0.0;
    for (int j = tid; j < a.K; j += kThreads)
      tsum += exp((static_cast<double>(s_p[j]) - tm) * a.inv_tau);
    tsum = block_sum_d(tsum, redd);
    for (int j = tid; j < a.K; j += kThreads) {
      const float t = s_p[j];
      const int64_t id = teacher_id(a, r * a.K + j);
      const bool keep = t != -INFINITY && id >= 0 && id < a.V;
      s_id[j] = keep ? static_cast<int32_t>(id) : -1;
      s_x[j] = keep ? to_f(x[id]) : 0.f;
      s_p[j] = static_cast<float>(
          exp((static_cast<double>(t) - tm) * a.inv_tau) / tsum);
    }
    __syncthreads();
    for (int i = tid; i < a.V; i += kThreads) put(dx + i, ex2((to_f(x[i]) - m) * a.c) * kq);
    __syncthreads();
    for (int j = tid; j < a.K; j += kThreads) {
      const int32_t id = s_id[j];
      if (id < 0) continue;
      float p = 0.f;
      for (int i = 0; i < a.K; ++i) p += s_id[i] == id ? s_p[i] : 0.f;
      put(dx + id, k * (ex2((s_x[j] - m) * a.c) * st.y - p));
    }
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

int64_t ws_bytes_for(int64_t n0, int64_t T) {
  return kWsHead + (n0 * 4 + 255) / 256 * 256 + T * static_cast<int64_t>(sizeof(double2));
}

// The workspace: head, counted rows of each sequence, partial sums.
int set_ws(RowArgs& a, void* ws, int64_t ws_bytes) {
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15u) != 0 ||
      ws_bytes < ws_bytes_for(a.n0, a.T))
    return bad("workspace: 16-byte aligned, at least lema_loss_workspace_bytes(n0, n1) bytes");
  char* p = static_cast<char*>(ws);
  a.head = reinterpret_cast<const WsHead*>(p);
  a.seq_count = reinterpret_cast<const int32_t*>(p + kWsHead);
  a.part = reinterpret_cast<double2*>(p + kWsHead + (a.n0 * 4 + 255) / 256 * 256);
  return LEMA_OK;
}

unsigned rows_grid(const RowArgs& a) {
  return static_cast<unsigned>(std::min<int64_t>(a.T, 1 << 20));
}

template <int OBJ>
int launch_rows(const RowArgs& a, int x_f32, cudaStream_t s) {
  if (x_f32)
    rows_kernel<float, OBJ><<<rows_grid(a), kThreads, 0, s>>>(a);
  else
    rows_kernel<__nv_bfloat16, OBJ><<<rows_grid(a), kThreads, 0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}

template <int OBJ>
int launch_bwd(const RowArgs& a, int x_f32, cudaStream_t s) {
  if (x_f32)
    rows_bwd_kernel<float, OBJ><<<rows_grid(a), kThreads, 0, s>>>(a);
  else
    rows_bwd_kernel<__nv_bfloat16, OBJ><<<rows_grid(a), kThreads, 0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}

int launch_count(const RowArgs& a, cudaStream_t s) {
  count_kernel<<<1, 1024, 0, s>>>(a.targets, a.ignore, a.mask, a.T, a.in.n1, a.n0,
                                  const_cast<int32_t*>(a.seq_count),
                                  const_cast<WsHead*>(a.head));
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
  return launch_rows<kLogp>(a, x_f32, static_cast<cudaStream_t>(stream));
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
  return launch_bwd<kLogp>(a, x_f32, static_cast<cudaStream_t>(stream));
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
  a.coef = nullptr;
  double2* part = a.part;
  a.part = nullptr;
  auto s = static_cast<cudaStream_t>(stream);
  if (a.T > 0 && (rc = launch_rows<kLogp>(a, x_f32, s))) return rc;
  a.coef = coef;
  pair_kernel<<<static_cast<unsigned>(n0 / 2), 256, 0, s>>>(a, n0 / 2, beta, label_smoothing,
                                                            part, rewards);
  LEMA_CUDA_TRY(cudaGetLastError());
  finish_kernel<<<1, 1024, 0, s>>>(part, n0 / 2, loss, nullptr);
  LEMA_CUDA_TRY(cudaGetLastError());
  if (dx == nullptr || a.T == 0) return LEMA_OK;
  a.g = coef;
  a.grad_scale = static_cast<float>(grad_scale);
  return launch_bwd<kLogp>(a, x_f32, s);
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
  auto s = static_cast<cudaStream_t>(stream);
  if ((rc = launch_count(a, s))) return rc;
  if (a.T > 0 && (rc = launch_rows<kPolicy>(a, x_f32, s))) return rc;
  finish_kernel<<<1, 1024, 0, s>>>(a.part, a.T, loss, kl);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
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
  auto s = static_cast<cudaStream_t>(stream);
  if ((rc = launch_count(a, s))) return rc;
  if (a.T > 0 && (rc = launch_rows<kDistill>(a, x_f32, s))) return rc;
  finish_kernel<<<1, 1024, 0, s>>>(a.part, a.T, loss, nullptr);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
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
  return launch_bwd<kDistill>(a, x_f32, static_cast<cudaStream_t>(stream));
}
