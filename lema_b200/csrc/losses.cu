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
// Precision: exponentials (ex2.approx, 2^-22) and their sum in fp32; what is computed once per
// token (the log-probability, its differences from the old and the reference one, the side of a
// clip end, sums over tokens) in fp64, since losses are differences of nearly equal log-
// probabilities, and with it ratios and KL terms where they are returned. A gradient row's
// coefficient takes their exponentials in fp32 (for bf16 rows approximate ones) of the same fp64
// differences. Every output is rounded once.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>

#include "internal.h"
#include "ptx.cuh"
#include "quant_core.cuh"

namespace lema {
namespace {

constexpr int kMaxTeacher = 1024;

// Rows of logits: row r starts (r / n1) * ld0 + (r % n1) * ld1 elements behind the base.
struct RowMap {
  int64_t n1, ld0, ld1;
  // Row numbers fit 32 bits, which divide several times faster than 64.
  __device__ __forceinline__ uint32_t seq(int64_t r) const {
    return static_cast<uint32_t>(r) / static_cast<uint32_t>(n1);
  }
  __device__ __forceinline__ int64_t at(int64_t r) const {
    const uint32_t b = seq(r);
    return b * ld0 + (r - b * n1) * ld1;
  }
};

// Workspace: head, counted rows of each sequence, the list of rows, partial sums, what each
// row leaves for its token's terms (preference: its log-probability).
struct WsHead {
  int64_t total;    // rows that count
  uint32_t ticket;  // CTAs of token_kernel or pair_kernel that are done
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
  double inv_tau, c_full;        // 1 / tau, log2(e) / tau
  float c, c_lo;                 // log2(e) / tau, rounded, and what the rounding left
  const int64_t* targets;        // [T]; null for distill
  int64_t ignore;
  float* logps;                  // [T]
  float2* stats;                 // [T] (m, 1 / s), may be null
  float* coef;                   // [T] dL/dlp, may be null
  RowStat* row;                  // [T]
  double* lp64;                  // [T] log-probabilities (preference)
  double2* part;                 // (loss, kl) of each CTA that adds tokens' terms, or pair
  void* dx;                      // null: no gradient
  RowMap out;
  float grad_scale;
  int32_t* err;
  WsHead* head;
  int32_t* seq_count;            // [n0] counted rows of each sequence (per_sequence only)
  int32_t* list;                 // [T] the rows that count, then the others
  float* loss;
  float* kl;
  // policy
  const float* old_logps;
  const float* adv;
  int64_t adv_s0, adv_s1;
  const float* ref_logps;
  double clip_lo, clip_hi, kl_coef;
  double log_lo, log_hi;         // log(1 - clip_lo), log(1 + clip_hi)
  int32_t per_sequence;
  int64_t n0;
  // distill
  const void* teacher_ids;
  int32_t ids_i32;
  const void* teacher_logits;
  int32_t tl_f32;
  int32_t K, K4;                 // entries a row, rounded up to four
  const uint8_t* mask;           // [T], may be null
  // backward from saved statistics
  const float* g;                // [T] gradient of each row's log-probability
  const float* upstream;         // scalar, may be null
  int32_t zeros_done;            // the rows of zeros are written
  int32_t self_count;            // no count_kernel ran: CTAs count for themselves
};

enum Objective { kPolicy = 1, kDistill = 2 };

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// The larger of two, NaN if either is.
__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- 16-byte vectors of a row ---------------------------------------------------
// A row may start at any element: its aligned 16-byte vectors are moved whole, the elements in
// front of the first and behind the last (its edges, fewer than a vector each) one by one, by
// the threads 0 .. kEdges - 1 of whoever holds the row.

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
  static __device__ __forceinline__ float max_nan(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    const float a = __low2float(m), b = __high2float(m);
    return max_or_nan(a, b);
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
  static __device__ __forceinline__ float max_nan(const uint4& v) {
    return max_or_nan(max_or_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                      max_or_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint4 pack(const uint64_t (&p)[2]) {
    float a, b, c, d;
    f2_unpack(p[0], a, b);
    f2_unpack(p[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c),
                      __float_as_uint(d));
  }
};

constexpr int kEdges = 16;  // edge e: element e of the head (e < 8), or e - 8 of the tail

template <typename T>
struct Span {
  int head, nvec, tail;  // elements, vectors, elements
  __device__ __forceinline__ Span(const T* x, int V) {
    const int to_go = static_cast<int>((16u - (reinterpret_cast<uintptr_t>(x) & 15u)) & 15u);
    head = min(V, to_go / static_cast<int>(sizeof(T)));
    nvec = (V - head) / Vec<T>::kE;
    tail = V - head - nvec * Vec<T>::kE;
  }
  __device__ __forceinline__ const uint4* vecs(const T* x) const {
    return reinterpret_cast<const uint4*>(x + head);
  }
  // The element that is edge e, or -1.
  __device__ __forceinline__ int edge(int e) const {
    if (e < 8) return e < head ? e : -1;
    return e - 8 < tail ? head + nvec * Vec<T>::kE + e - 8 : -1;
  }
  // Which thread of G holds element i (vectors are dealt round robin).
  __device__ __forceinline__ int owner(int i, int G) const {
    if (i < head) return i;
    const int v = (i - head) / Vec<T>::kE;
    return v < nvec ? v % G : i - head - nvec * Vec<T>::kE + 8;
  }
};

template <typename T>
__device__ __forceinline__ uint4 neg_inf_vec() {
  return make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
}

__device__ __forceinline__ uint4 ld16(const uint4* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// 2^((x - m) c), c = log2(e) / tau, for the elements of a vector as packed fp32 pairs, with one
// multiply-add each: x c - fl(m c). The rounding of m c is the same factor in every exponential of
// the row, at most 2^-13 from 1; `fix` takes it out. Rows with |m c| above 2048 (a row of the
// type's lowest value, for one) are shifted by their maximum first, see shift_vec.
struct ExpScale {
  uint64_t c, mc;
  float fix;  // sum of exp((x - m) / tau) = fix * sum of what exp_vec gives
  __device__ __forceinline__ ExpScale(float m, float c_) : c(f2_splat(c_)) {
    m = m == -INFINITY ? 0.f : m;
    const float p = m * c_;
    mc = f2_splat(-p);
    fix = 1.f - 0.69314718f * fmaf(m, c_, -p);  // 2^(p - m c)
  }
};
// The whole number nearest to m c (0 for a maximum without one).
__device__ __forceinline__ float whole_max(float m, float c) {
  return m == -INFINITY ? 0.f : rintf(m * c);
}
// 2^n for whole n <= 0.
__device__ __forceinline__ float exp2_whole(float n) {
  if (n < -126.f) return 0.f;
  return __uint_as_float(static_cast<uint32_t>(static_cast<int>(n) + 127) << 23);
}
__device__ __forceinline__ bool far_max(float m, float c) {
  return fabsf(m * c) > 2048.f && m != -INFINITY;
}
// What takes a partial sum of a row whose maximum is `from` to the larger maximum `to` (neither
// of them -inf). A sum is about its maximum; with WHOLE it is about whole_max while the maximum is
// near, and only a far one is about itself, so where one of the two is near the factor goes by
// the two references that the sums have: 2^(from c - n) or 2^(n - to c), c with what its rounding
// left, since 2048 times that is 2e-5.
__device__ __forceinline__ float rescale_far(float from, float to, float c, float c_lo) {
  if (!far_max(to, c)) return ex2(fmaf(from, c, -whole_max(to, c)) + from * c_lo);
  if (!far_max(from, c)) return ex2(fmaf(-to, c, whole_max(from, c)) - to * c_lo);
  return ex2((from - to) * c);
}
template <bool WHOLE>
__device__ __forceinline__ float rescale(float from, float to, float c, float c_lo) {
  if (!WHOLE) return ex2((from - to) * c);
  if (far_max(from, c) || far_max(to, c)) return rescale_far(from, to, c, c_lo);
  return exp2_whole(whole_max(from, c) - whole_max(to, c));
}
__device__ __forceinline__ uint64_t exp_pair(uint64_t x, const ExpScale& k) {
  float lo, hi;
  f2_unpack(f2_fma(x, k.c, k.mc), lo, hi);
  return f2_pack(ex2(lo), ex2(hi));
}
template <typename T>
__device__ __forceinline__ void exp_vec(const uint4& w, const ExpScale& k,
                                        uint64_t (&e)[Vec<T>::kE / 2]) {
#pragma unroll
  for (int i = 0; i < Vec<T>::kE / 2; ++i) e[i] = exp_pair(Vec<T>::pair(w, i), k);
}
// x - m in place of x, rounded to T. With |m c| above 2048 the elements whose exponential is not 0
// lie within 6 percent of m, where the difference is a small multiple of their last place: exact.
template <typename T>
__device__ __forceinline__ void shift_vec(uint4& w, float m) {
  uint64_t d[Vec<T>::kE / 2];
#pragma unroll
  for (int i = 0; i < Vec<T>::kE / 2; ++i) d[i] = f2_add(Vec<T>::pair(w, i), f2_splat(-m));
  w = Vec<T>::pack(d);
}

// The same about a whole n, sums about different n meeting exactly, for log-probabilities that are
// added up: a preference reward sums hundreds of them and keeps little, so what shifts them all
// the same way shows (it was 2e-5 off with exp_vec). That is c's own rounding, 1e-8 of x - m,
// added back here with a second multiply-add; and ex2.approx, which is 5e-8 low on average but 1e-8
// on [-1/2, 1/2], where its argument is brought here: Cody and Waite's reduction, by a constant in
// two parts. Elements are kept above n - 120, which is nothing beside the maximum. NaNs are
// looked for apart.
struct WholeScale {
  uint64_t c, c_lo, up;  // 1.5 * 2^23 - n, added and taken off: rounds to a whole number
  __device__ __forceinline__ WholeScale(float n, float c_, float c_lo_)
      : c(f2_splat(c_)), c_lo(f2_splat(c_lo_)), up(f2_splat(12582912.f - n)) {}
};
__device__ __forceinline__ uint64_t exp_pair_whole(uint64_t x, const WholeScale& k) {
  const uint64_t t = f2_fma(x, k.c, k.up);
  const uint64_t minus_u = f2_fma(t, f2_splat(-1.f), k.up);
  float f0, f1, t0, t1;
  f2_unpack(f2_fma(x, k.c_lo, f2_fma(x, k.c, minus_u)), f0, f1);
  f2_unpack(t, t0, t1);
  // times 2^(u - n): the low bits of t, into the exponent
  return f2_pack(__uint_as_float(__float_as_uint(ex2(f0)) + (__float_as_uint(t0) << 23)),
                 __uint_as_float(__float_as_uint(ex2(f1)) + (__float_as_uint(t1) << 23)));
}
__device__ __forceinline__ void keep_above(uint4& w, float low, __nv_bfloat16) {
  const __nv_bfloat162 l = __float2bfloat162_rn(low);
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], l);
}
__device__ __forceinline__ void keep_above(uint4& w, float low, float) {
  float* f = reinterpret_cast<float*>(&w);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = fmaxf(f[i], low);
}

// The logarithm of what exp_pair_whole gives for the target over what it should give: the sum of
// a row's exponentials is off alike on average, so adding this to the target's log-probability
// leaves what does not add up over a sequence.
__device__ __forceinline__ double ex2_error(float x, const RowArgs& a) {
  const double e = static_cast<double>(x) * a.c_full;
  const float f = static_cast<float>(e - rint(e));
  if (!(fabsf(f) <= 0.5f)) return 0.0;
  return log(static_cast<double>(ex2(f))) - 0.6931471805599453 * static_cast<double>(f);
}

template <typename T>
__device__ __forceinline__ bool same_phase(const T* a, const T* b) {
  return ((reinterpret_cast<uintptr_t>(a) ^ reinterpret_cast<uintptr_t>(b)) & 15u) == 0;
}

// A predicated store: no branch among a row's stores.
__device__ __forceinline__ void st16_if(uint4* p, const uint4& v, bool yes) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.u32 p, %5, 0;\n\t"
      "@p st.global.v4.u32 [%0], {%1, %2, %3, %4};\n\t}\n" ::"l"(p),
      "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(static_cast<uint32_t>(yes))
      : "memory");
}

// The vectors of a warp (one behind the other, those of the first lanes `in`) where the output row
// starts at another phase within 16 bytes than the input row, as after logits[:, :-1] over an odd
// vocabulary: each lane stores the aligned vector that its own and the next lane's make up, the
// first and last lane the elements around. 8 x 512 rows of 32000 bf16: the policy loss takes
// 230 us, with every element stored alone 378, at the same phase 124.
template <typename T>
__device__ __noinline__ void store_apart(T* dst, uint4 w, bool in) {
  const int lane = threadIdx.x & 31;
  const int gap = static_cast<int>(-reinterpret_cast<uintptr_t>(dst) & 15u);  // bytes to 16
  uint32_t a[8] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) a[4 + i] = __shfl_down_sync(0xffffffffu, a[i], 1);
  const bool next = __shfl_down_sync(0xffffffffu, in, 1) && lane < 31;
  if (gap & 4) {
#pragma unroll
    for (int i = 0; i < 7; ++i) a[i] = a[i + 1];
  }
  if (gap & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) a[i] = a[i + 2];
  }
  uint4 o;
  o.x = __funnelshift_r(a[0], a[1], (gap & 3) * 8);
  o.y = __funnelshift_r(a[1], a[2], (gap & 3) * 8);
  o.z = __funnelshift_r(a[2], a[3], (gap & 3) * 8);
  o.w = __funnelshift_r(a[3], a[4], (gap & 3) * 8);
  const int front = gap / static_cast<int>(sizeof(T));
  if (in && next) *reinterpret_cast<uint4*>(dst + front) = o;
  if (in && (lane == 0 || !next)) {
    const T* we = reinterpret_cast<const T*>(&w);
    const T* oe = reinterpret_cast<const T*>(&o);
#pragma unroll
    for (int j = 0; j < Vec<T>::kE; ++j) {
      if (lane == 0 && j < front) dst[j] = we[j];
      if (!next && j < Vec<T>::kE - front) dst[front + j] = oe[j];
    }
  }
  __syncwarp();  // an element that another lane has stored may be replaced behind this
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

// Barrier of a group of G threads: a warp, or the whole CTA.
template <int G>
__device__ __forceinline__ void group_sync() {
  if (G == 32)
    __syncwarp();
  else
    __syncthreads();
}

// Maximum of a row and sum of exp((x - m) / tau) from the (m, s) of a group's threads, for every
// thread. WHOLE: each sum is about the reference of its own maximum (rescale), the row's about
// that of the row's: see about_max. Sums meet in fp64.
template <int G, bool WHOLE>
__device__ __forceinline__ void group_combine(float& m, double& s, const RowArgs& a, float* redf,
                                              double* redd) {
  const float mt = m;
  const int warp = (threadIdx.x % G) >> 5;
  m = warp_max(m);
  if (G > 32) {
    group_sync<G>();
    if ((threadIdx.x & 31) == 0) redf[warp] = m;
    group_sync<G>();
    m = redf[0];
#pragma unroll
    for (int w = 1; w < G / 32; ++w) m = fmaxf(m, redf[w]);
  }
  // a thread that saw only -inf adds nothing
  s *= mt == -INFINITY ? 0.0 : static_cast<double>(rescale<WHOLE>(mt, m, a.c, a.c_lo));
  s = warp_sum(s);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) redd[warp] = s;
    group_sync<G>();
    s = redd[0];
#pragma unroll
    for (int w = 1; w < G / 32; ++w) s += redd[w];
  }
  if (m == -INFINITY) s = NAN;
}
// The logarithm that takes a sum about whole_max of m to one about m.
__device__ __forceinline__ double about_max(float m, const RowArgs& a) {
  if (far_max(m, a.c)) return 0.0;
  return (static_cast<double>(whole_max(m, a.c)) - static_cast<double>(m) * a.c_full) *
         0.6931471805599453;
}

// One thread's share of a row's maximum and sum: its edge and the vectors tid, tid + G, ..., in
// one sweep with a running maximum, U loads in flight.
template <typename T, int G, int U, bool WHOLE>
__device__ __forceinline__ void thread_stats(const T* x, const Span<T>& sp, int tid, float c,
                                             float c_lo, float& m, double& s) {
  const uint4* xv = sp.vecs(x);
  m = -INFINITY;
  float sum = 0.f;
  if (sp.head + sp.tail > 0 && tid < kEdges) {
    const int i = sp.edge(tid);
    const float xe = i >= 0 ? to_f(x[i]) : -INFINITY;
    if (xe != xe || xe == INFINITY) sum = NAN;
    if (fabsf(xe) < INFINITY)
      sum = WHOLE && !far_max(xe, c) ? ex2(fmaf(xe, c, -whole_max(xe, c)) + xe * c_lo) : 1.f;
    if (xe == xe) m = xe;
  }
  for (int base = tid; base < sp.nvec; base += G * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      w[u] = base + u * G < sp.nvec ? ld16(xv + base + u * G) : neg_inf_vec<T>();
    float mx = m;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float v = WHOLE ? Vec<T>::max_nan(w[u]) : Vec<T>::max(w[u]);
      if (WHOLE) nan |= v != v;
      mx = fmaxf(mx, v);
    }
    if (WHOLE && (nan || mx == INFINITY)) {
      sum = NAN;  // and stays so
      mx = m;
    }
    const bool far = far_max(mx, c);
    const float n = far ? 0.f : whole_max(mx, c);
    if (m != -INFINITY) sum *= rescale<WHOLE>(m, mx, c, c_lo);  // the sum so far
    m = mx;
    if (far) {
#pragma unroll
      for (int u = 0; u < U; ++u) shift_vec<T>(w[u], m);
    }
    const ExpScale k(far ? 0.f : m, c);
    const WholeScale kw(n, c, c_lo);
    const float low = (n - 120.f) / c;
    uint64_t acc[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (WHOLE) keep_above(w[u], low, T());
#pragma unroll
      for (int i = 0; i < Vec<T>::kE / 2; ++i) {
        const uint64_t p = Vec<T>::pair(w[u], i);
        acc[i & 1] = f2_add(acc[i & 1], WHOLE ? exp_pair_whole(p, kw) : exp_pair(p, k));
      }
    }
    float lo, hi;
    f2_unpack(f2_add(acc[0], acc[1]), lo, hi);
    sum += WHOLE ? lo + hi : (lo + hi) * k.fix;
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

// How many rows count: in all, and (per_sequence) of each sequence.
struct Counts {
  int64_t total;
  const int32_t* seq;
};
// Those that count_kernel left.
__device__ __forceinline__ Counts listed_counts(const RowArgs& a) {
  return Counts{a.head->total, a.seq_count};
}
// 1 / (the number of tokens a token's term is divided by).
__device__ __forceinline__ double token_weight(const RowArgs& a, const Counts& n, int64_t r) {
  return 1.0 / static_cast<double>(a.per_sequence ? a.n0 * n.seq[a.in.seq(r)] : n.total);
}

// What the clipped policy loss knows of a token besides its log-probability.
struct Token {
  float adv, old, ref;
};
__device__ __forceinline__ Token load_token(const RowArgs& a, int64_t r) {
  const int64_t b = a.in.seq(r), t = r - b * a.in.n1;
  return Token{a.adv[b * a.adv_s0 + t * a.adv_s1], a.old_logps ? a.old_logps[r] : 0.f,
               a.ref_logps ? a.ref_logps[r] : 0.f};
}

// log(s) of a row's sum, to 1e-12: a row's threads wait for it (policy over 3 x 611 rows of
// 100277 bf16 takes 158.5 us, with log() 161.9; over 8 x 1024 of 8000 60.8 and 61.6). s = 2^e f,
// f in [sqrt(1/2), sqrt(2)), and with t = (f - 1) / (f + 1), |t| < 0.172,
//   log f = 2 artanh t = 2 t + 2 t^3 (1/3 + t^2 / 5 + ... + t^10 / 13),
// whose remainder is 5e-13. t is a quotient in fp32, corrected once by its residual in fp64. A sum
// holds its maximum's 1, or it is NaN, and so is its logarithm. Every rounding is written
// out, so that all who call it with one s get the same bits.
__device__ __forceinline__ double log_sum(float s) {
  const uint32_t bits = __float_as_uint(s);
  const int e = static_cast<int>(bits - 0x3f3504f3u) >> 23;  // sqrt(1/2)
  const float f = __uint_as_float(bits - (static_cast<uint32_t>(e) << 23));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(f, 1.f)));
  const double fd = f, rd = r, num = __dsub_rn(fd, 1.0), den = __dadd_rn(fd, 1.0);
  const double q = __fmul_rn(__fsub_rn(f, 1.f), r);
  const double t = __fma_rn(__fma_rn(-q, den, num), rd, q);
  const double t2 = __dmul_rn(t, t), t4 = __dmul_rn(t2, t2), two_t = __dadd_rn(t, t);
  const double p0 = __fma_rn(t2, 1.0 / 5, 1.0 / 3), p1 = __fma_rn(t2, 1.0 / 9, 1.0 / 7),
               p2 = __fma_rn(t2, 1.0 / 13, 1.0 / 11);
  const double p = __fma_rn(t4, __fma_rn(t4, p2, p1), p0);
  const double y = __fma_rn(__dmul_rn(two_t, t2), p, __fma_rn(e, 0.6931471805599453, two_t));
  return bits - 0x00800000u < 0x7f000000u ? y : NAN;
}
// A token's log-probability from what its row left.
__device__ __forceinline__ double token_lp(const RowArgs& a, float x, float m, float s) {
  return __fma_rn(__dsub_rn(x, m), a.inv_tau, -log_sum(s));
}

// e^d - 1 to 8e-6 of itself: beside a bf16 step of 2^-9 nothing, but e^d - 1 as it stands would
// keep 2e-7 of 1 and so nothing of a small d.
__device__ __forceinline__ float expm1_fast(float d) {
  return fabsf(d) < 0.03125f ? d * fmaf(d, fmaf(d, 1.f / 6, 0.5f), 1.f) : __expf(d) - 1.f;
}

// dL/dlp of one token of the clipped policy loss over its weight, and (LOSS) its loss and KL.
// F = double for what is returned, float for the gradient's coefficient (FAST: of a bf16 row). Both
// take differences of log-probabilities, and the side of a clip end, from the same fp64 numbers:
// a gradient row is clipped exactly where the returned loss is, and a KL term keeps the digits of
// a small d.
template <typename F, bool LOSS, bool FAST = false>
__device__ __forceinline__ F policy_token(const RowArgs& a, const Token& tk, double lp, F* loss,
                                          F* kl) {
  const F A = tk.adv;
  // on-policy the ratio is 1, and NaN for a log-probability that is not finite
  const double up = __dsub_rn(lp, a.old_logps ? static_cast<double>(tk.old) : lp);
  const F ratio = FAST ? static_cast<F>(__expf(static_cast<float>(up))) : exp(static_cast<F>(up));
  // min(r A, clip(r) A) is the clipped one; not for a NaN ratio
  const bool clipped = A > F(0) ? up > a.log_hi : A < F(0) && up < a.log_lo;
  F coef = clipped ? F(0) : -ratio * A;
  F d_kl = F(0);
  if (a.ref_logps) {
    const double d = __dsub_rn(tk.ref, lp);
    const F e = FAST ? static_cast<F>(expm1_fast(static_cast<float>(d))) : expm1(static_cast<F>(d));
    d_kl = e == static_cast<F>(INFINITY) ? e : e - static_cast<F>(d);
    // with a coefficient of 0 the KL is returned alone: it may be infinite
    if (a.kl_coef != 0.0) coef -= static_cast<F>(a.kl_coef) * e;
  }
  if (LOSS) {
    *kl = d_kl;
    *loss = (a.kl_coef != 0.0 ? static_cast<F>(a.kl_coef) * d_kl : F(0)) -
            (clipped ? static_cast<F>(A > F(0) ? 1.0 + a.clip_hi : 1.0 - a.clip_lo) : ratio) * A;
  }
  return coef;
}

// ---- kernels ---------------------------------------------------------------------

// Lists the rows that enter the loss in their order (list[0 .. total)), then the others from the
// end backwards, counts them for each sequence, and clears the ticket. The CTAs of one cluster
// count `chunk` rows each, add up the counts in front of their own and list theirs. The list's
// order, and with it the order of every sum, is always the same. Two passes over the targets,
// bound by their latency: 7.7 us at 16384 rows and 9.1 us at 65536 (CTAs that recount the rows
// in front of theirs: 9.0 us and 19.7 us).
constexpr int kCountThreads = 1024;
constexpr int kCountRows = 8;
constexpr int kCountBlock = kCountThreads * kCountRows;
constexpr int kCountCluster = 8;
__global__ void __launch_bounds__(kCountThreads) count_kernel(RowArgs a, int32_t chunk) {
  constexpr int kCells = kCountRows * kCountThreads / 32;  // a warp's rows at one offset
  __shared__ int32_t s_cell[kCells];
  __shared__ int32_t s_sum, s_end, s_cta[kCountCluster];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x, ctas = gridDim.x;  // one cluster
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // a CTA's shared memory may be written only once it runs: waited for behind the counting
  if (ctas > 1) ptx::cluster_arrive();
  const int64_t r0 = static_cast<int64_t>(rank) * chunk, r1 = min(a.T, r0 + chunk);
  bool in[kCountRows];
  const auto load = [&](int64_t at) {
#pragma unroll
    for (int j = 0; j < kCountRows; ++j) {
      const int64_t r = at + j * kCountThreads + tid;
      int64_t target;
      in[j] = r < r1 && row_counts(a, r, target);
    }
  };
  if (tid == 0) {
    s_sum = 0;
    if (rank == 0) a.head->ticket = 0;
  }
  if (a.per_sequence)
    for (int64_t b = rank * kCountThreads + tid; b < a.n0; b += ctas * kCountThreads)
      a.seq_count[b] = 0;
  int before = 0;
  if (ctas > 1) {
    int n = 0;
    for (int64_t at = r0; at < r1; at += kCountBlock) {
      load(at);
#pragma unroll
      for (int j = 0; j < kCountRows; ++j) n += in[j];
    }
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if (lane == 0) atomicAdd(&s_sum, n);
    __syncthreads();
    ptx::cluster_wait();
    if (tid < ctas)
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(
                       ptx::mapa_shared(ptx::smem_u32(&s_cta[rank]), tid)),
                   "r"(s_sum)
                   : "memory");
    ptx::cluster_sync();
    for (int j = 0; j < rank; ++j) before += s_cta[j];
  } else {
    load(r0);
    __syncthreads();
  }
  for (int64_t at = r0; at < r1; at += kCountBlock) {
    if (chunk > kCountBlock) load(at);
    uint32_t ballot[kCountRows];
#pragma unroll
    for (int j = 0; j < kCountRows; ++j) {
      ballot[j] = __ballot_sync(0xffffffffu, in[j]);
      if (lane == 0) s_cell[j * 32 + warp] = __popc(ballot[j]);
      if (a.per_sequence) {
        const int64_t b = a.in.seq(min(at + j * kCountThreads + tid, a.T - 1));
        // a warp inside one sequence adds once
        const bool one = __all_sync(0xffffffffu, __shfl_sync(0xffffffffu, b, 0) == b);
        if (one ? lane == 0 && ballot[j] != 0 : in[j])
          atomicAdd(&a.seq_count[b], one ? __popc(ballot[j]) : 1);
      }
    }
    __syncthreads();
    if (warp == 0) {
      int n[kCells / 32], sum = 0;
#pragma unroll
      for (int j = 0; j < kCells / 32; ++j) {
        n[j] = s_cell[lane * (kCells / 32) + j];
        sum += n[j];
      }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      int rank_of = before + incl - sum;
#pragma unroll
      for (int j = 0; j < kCells / 32; ++j) {
        s_cell[lane * (kCells / 32) + j] = rank_of;
        rank_of += n[j];
      }
      if (lane == 31) s_end = rank_of;
    }
    __syncthreads();
    before = s_end;
#pragma unroll
    for (int j = 0; j < kCountRows; ++j) {
      const int64_t r = at + j * kCountThreads + tid;
      // counted rows in front of r
      const int64_t rank_of = s_cell[j * 32 + warp] + __popc(ballot[j] & ((1u << lane) - 1u));
      if (in[j])
        a.list[rank_of] = static_cast<int32_t>(r);
      else if (r < r1)
        a.list[a.T - 1 - (r - rank_of)] = static_cast<int32_t>(r);
    }
    __syncthreads();
  }
  // the last of them have no rows when there are few
  if (rank == ctas - 1 && tid == 0) a.head->total = before;
}

// Few rows are counted by each CTA that needs the numbers, which saves the launch of
// count_kernel (and its latency, which the first rows would wait for).
constexpr int64_t kSelfRows = 1024;  // by the CTAs of direct_kernel and token_kernel

// Rows from `from` on, n of them, that count: the share of thread t of G.
template <int G>
__device__ __forceinline__ int count_rows(const RowArgs& a, int64_t from, int64_t n, int t) {
  int sum = 0;
#pragma unroll 8
  for (int64_t i = t; i < n; i += G) {
    int64_t target;
    sum += row_counts(a, from + i, target);
  }
  return sum;
}

// What a row that does not count leaves in the policy loss's outputs.
__device__ __forceinline__ void zero_outputs(const RowArgs& a, int64_t r) {
  if (a.logps) a.logps[r] = 0.f;
  if (a.coef) a.coef[r] = 0.f;
  if (a.stats) a.stats[r] = make_float2(0.f, 0.f);
}

// One token's terms in fp64, from what its row left: its share of the loss and of the KL, its
// log-probability, and what the backward needs.
template <int OBJ>
__device__ __forceinline__ double2 token_terms(const RowArgs& a, const Counts& n, int64_t r) {
  const RowStat st = a.row[r];
  if (OBJ == kDistill) {
    // sum_k p_k (log p_k - log q_k), p_k = p'_k / t
    const double t = st.x, log_s = log(static_cast<double>(st.s));
    if (t == 0.0) return make_double2(0.0, 0.0);
    return make_double2((st.a / t * a.inv_tau - log(t) + log_s) /
                            (static_cast<double>(n.total) * a.inv_tau * a.inv_tau),
                        0.0);
  }
  const double w = token_weight(a, n, r), lp = token_lp(a, st.x, st.m, st.s);
  double loss, kl;
  const double coef = policy_token<double, true>(a, load_token(a, r), lp, &loss, &kl);
  a.logps[r] = static_cast<float>(lp);
  if (a.coef) a.coef[r] = static_cast<float>(w * coef);
  if (a.stats) a.stats[r] = make_float2(st.m, isnan(st.x) ? NAN : 1.f / st.s);
  return make_double2(w * loss, w * kl);
}

// A gradient row of zeros, which L2 gives up first.
template <typename T, int G>
__device__ __forceinline__ void zero_row(const RowArgs& a, int64_t r, int tid) {
  if (a.dx == nullptr) return;
  T* dx = static_cast<T*>(a.dx) + a.out.at(r);
  const Span<T> so(dx, a.V);
  uint4* dv = reinterpret_cast<uint4*>(dx + so.head);
  for (int v = tid; v < so.nvec; v += G) __stcs(dv + v, make_uint4(0u, 0u, 0u, 0u));
  if (tid < kEdges && so.edge(tid) >= 0) put(dx + so.edge(tid), 0.f);
}

// token_logprobs: a group of G threads a row, U vectors of a thread in flight. Long rows are bound
// by DRAM's reads (4096 x 32000 bf16, three quarters of them counted: 36 us, 5.5 TB/s), short
// ones by the latency of a row's chain of loads and reductions (65536 x 512: 26 us, 1.9 TB/s).
// Several rows for each group, their targets loaded and logarithms taken together, gave nothing.
constexpr int stat_threads(int G) { return G > 128 ? G : 128; }
template <typename T, int G, bool WHOLE, int U>
__global__ void __launch_bounds__(stat_threads(G)) logprobs_kernel(RowArgs a) {
  __shared__ float redf[G / 32];
  __shared__ double redd[G / 32];
  const int tid = threadIdx.x % G;
  const int64_t r = blockIdx.x * int64_t{stat_threads(G) / G} + threadIdx.x / G;
  if (r >= a.T) return;
  if (r == 0 && tid == 0 && a.head) a.head->ticket = 0;  // pair_kernel's
  int64_t target;
  if (!row_counts(a, r, target)) {
    if (tid == 0) {
      a.logps[r] = 0.f;
      if (a.stats) a.stats[r] = make_float2(0.f, 0.f);
    }
    zero_row<T, G>(a, r, tid);  // the gradient's kernel has the rest to write
    return;
  }
  const T* x = static_cast<const T*>(a.x) + a.in.at(r);
  const bool ok = target >= 0 && target < a.V;
  const float xt = ok ? to_f(x[target]) : 0.f;
  const Span<T> sp(x, a.V);
  float m;
  double s;
  thread_stats<T, G, U, WHOLE>(x, sp, tid, a.c, a.c_lo, m, s);
  group_combine<G, WHOLE>(m, s, a, redf, redd);
  if (tid == 0) {
    const double up = WHOLE ? about_max(m, a) : 0.0, log_s = log(s) + up;
    const double lp =
        ok ? (static_cast<double>(xt) - m) * a.inv_tau + (WHOLE ? ex2_error(xt, a) : 0.0) - log_s
           : NAN;
    if (!ok) atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
    a.logps[r] = static_cast<float>(lp);
    if (a.lp64) a.lp64[r] = lp;
    if (a.stats)
      a.stats[r] =
          make_float2(m, ok ? static_cast<float>(1.0 / s) * expf(static_cast<float>(-up)) : NAN);
  }
}

// ---- a teacher's entries of one row -----------------------------------------------

// Unnormalised weights p' = exp((t - t_max) / tau), checked indices (-1: no weight) and the
// student's logits there, of the row's K entries, by one warp. `d_sum`: sum of
// p' ((t - t_max) - x); `p_sum`: sum of p'; `t_sum`: the same in fp32, 0 for a row without an
// entry; `bad`: an entry with a weight has its index outside the vocabulary.
struct TeacherSums {
  double d_sum, p_sum;
  float t_sum;
  bool bad;
  // sum of p' ((t - t_max) - (x - m)), RowStat::a
  __device__ __forceinline__ double about(float m) const {
    return bad ? NAN : d_sum + p_sum * static_cast<double>(m);
  }
};
template <typename T>
__device__ __forceinline__ TeacherSums teacher_weights(const RowArgs& a, int64_t r, const T* x,
                                                       int lane, float* s_p, float* s_x,
                                                       int32_t* s_id) {
  constexpr int kU = 4;
  const int64_t at = r * a.K;
  float tm = -INFINITY;
  for (int k0 = lane; k0 < a.K; k0 += 32 * kU) {
    float t[kU], xv[kU];
    int64_t id[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = k0 + 32 * u;
      t[u] = k < a.K ? teacher_logit(a, at + k) : -INFINITY;
      id[u] = k < a.K ? teacher_id(a, at + k) : -1;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const bool use = t[u] != -INFINITY && id[u] >= 0 && id[u] < a.V;
      xv[u] = use ? to_f(x[id[u]]) : 0.f;
      if (!use) id[u] = -1;
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int k = k0 + 32 * u;
      tm = fmaxf(tm, t[u]);
      if (k < a.K) {
        s_p[k] = t[u];
        s_x[k] = xv[u];
        s_id[k] = static_cast<int32_t>(id[u]);
      }
    }
  }
  for (int k = a.K + lane; k < a.K4; k += 32) {
    s_p[k] = 0.f;
    s_id[k] = -1;
  }
  tm = warp_max(tm);
  double sum = 0.0, d_sum = 0.0;
  bool bad = false;
  for (int k = lane; k < a.K; k += 32) {  // each lane reads back its own entries
    const float t = s_p[k];
    float p = 0.f;
    if (t != -INFINITY) {
      const float d = t - tm;
      p = expf(static_cast<float>(static_cast<double>(d) * a.inv_tau));
      sum += static_cast<double>(p);
      bad |= p != 0.f && s_id[k] < 0;
      if (p != 0.f)
        d_sum += static_cast<double>(p) *
                 (static_cast<double>(t) - static_cast<double>(tm) - static_cast<double>(s_x[k]));
    }
    s_p[k] = p;
    if (p == 0.f) s_id[k] = -1;
  }
  bad = __any_sync(0xffffffffu, bad);
  sum = warp_sum(sum);
  return TeacherSums{warp_sum(d_sum), sum, static_cast<float>(sum), bad};
}

// Indices of a row seen once and seen again, by their low bits: an index that is not seen again is
// held by one entry.
template <int BITS>
struct Seen {
  uint32_t once[BITS / 32], twice[BITS / 32];
  __device__ __forceinline__ void clear(int t, int threads) {
    for (int i = t; i < BITS / 32; i += threads) once[i] = twice[i] = 0;
  }
  __device__ __forceinline__ void add(int32_t id) {
    const uint32_t bit = 1u << (id & 31);
    if (atomicOr(&once[id % BITS / 32], bit) & bit) atomicOr(&twice[id % BITS / 32], bit);
  }
  __device__ __forceinline__ bool again(int32_t id) const {
    return twice[id % BITS / 32] >> (id & 31) & 1u;
  }
};

// The value of a gradient row at entry j's index: k (q - p), p the sum of the entries that hold
// this index (`alone`: no other), always in the same order, so that entries which repeat it write
// the same value. Four entries a read; those behind the last hold no index.
__device__ __forceinline__ float teacher_value(const RowArgs& a, int j, bool alone,
                                               const float* s_p, const int32_t* s_id, float q,
                                               float inv_t, float k) {
  if (alone) return k * (q - s_p[j] * inv_t);
  const int32_t id = s_id[j];
  float p0 = 0.f, p1 = 0.f, p2 = 0.f, p3 = 0.f;
#pragma unroll 4
  for (int i = 0; i < a.K4; i += 4) {
    const int4 d = *reinterpret_cast<const int4*>(s_id + i);
    const float4 p = *reinterpret_cast<const float4*>(s_p + i);
    p0 += d.x == id ? p.x : 0.f;
    p1 += d.y == id ? p.y : 0.f;
    p2 += d.z == id ? p.z : 0.f;
    p3 += d.w == id ? p.w : 0.f;
  }
  return k * (q - ((p0 + p1) + (p2 + p3)) * inv_t);
}

// k of a distilled row: tau over the number of rows, 0 for a row without an entry.
__device__ __forceinline__ float row_share(const RowArgs& a, const Counts& n) {
  return static_cast<float>(1.0 / (static_cast<double>(n.total) * a.inv_tau));
}
__device__ __forceinline__ float teacher_coef(const TeacherSums& t, float share) {
  return t.bad ? NAN : (t.t_sum == 0.f ? 0.f : share);
}

// k of a token of the policy loss, for its gradient row: the log-probability and its differences
// as the loss has them, their exponentials in fp32. A bf16 row is rounded to 2^-9, so approximate
// exponentials (8e-6 at worst) serve it.
template <typename T>
__device__ __forceinline__ float policy_coef(const RowArgs& a, const Token& tk, float xt, float m,
                                             float s, float w) {
  return policy_token<float, false, sizeof(T) == 2>(a, tk, token_lp(a, xt, m, s), nullptr,
                                                    nullptr) * w;
}

__device__ __forceinline__ float grad_factor(const RowArgs& a) {
  return a.grad_scale * (a.upstream ? *a.upstream : 1.f);
}

__device__ __forceinline__ void note_bad_index(const RowArgs& a) {
  atomicMax(a.err, static_cast<int32_t>(kDevErrIndex));
}

// ---- rows that fit the registers of a warp or of 128 threads ------------------------

// k (1[v = target] - q_v), or for distill k (q_v - p_v), and what the row leaves for
// token_kernel. G threads hold a row, kE * NV elements each: it is read once, its exponentials
// stay in registers and are scaled and written once. Loads of many resident groups overlap:
// 16384 policy rows of 4096 bf16, three quarters of them counted (235 MB), take 49 us, 4.8 TB/s;
// 65536 of 512 (117 MB) 36 us, bound by the latency of a row's chain. With 64 teacher entries a
// row whole calls take 85 and 81 us instead of 60 and 48, for the latency of their loads.
// Entries whose index another one may hold are told by a bit of it; comparing each with all took
// 145 us over 12258 rows of 1802 fp32 with 244 entries, this 84. (The CTAs of ring_kernel have
// the threads to compare; marking by its producer took longer: 66 and 74 us over 2000 rows of
// 32000 with 200.)
constexpr int kDirectThreads = 128;
template <typename T, int OBJ, int G, int NV>
__global__ void __launch_bounds__(kDirectThreads) direct_kernel(RowArgs a) {
  constexpr int E = Vec<T>::kE, kGroups = kDirectThreads / G;
  __shared__ float redf[2][kDirectThreads / 32], s_k;
  __shared__ TeacherSums s_t[kGroups];
  extern __shared__ __align__(16) char smem[];
  const int tid = threadIdx.x % G, group = threadIdx.x / G, warp = tid >> 5;
  float* s_p = reinterpret_cast<float*>(smem) + group * 3 * a.K4;
  float* s_x = s_p + a.K4;
  int32_t* s_id = reinterpret_cast<int32_t*>(s_x + a.K4);
  __shared__ int32_t s_count[kDirectThreads / 32], s_seq[kGroups];
  // a bit for each element of a row, or nearly
  __shared__ Seen<OBJ == kDistill ? G * NV * E : 32> seen[kGroups];
  if (OBJ == kDistill) seen[group].clear(tid, G);
  ptx::griddep_wait();
  const int64_t r = blockIdx.x * int64_t{kGroups} + group;
  Counts counts = listed_counts(a);
  if (a.self_count) {
    const uint32_t b = a.in.seq(min(r, a.T - 1));
    int n = a.per_sequence ? count_rows<G>(a, b * a.in.n1, a.in.n1, tid)
                           : count_rows<kDirectThreads>(a, 0, a.T, threadIdx.x);
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) s_count[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
    for (int w = 0; w < kDirectThreads / 32; ++w)
      if (!a.per_sequence || G > 32 || w == group) n += s_count[w];
    if (tid == 0) s_seq[group] = n;
    counts = Counts{n, s_seq + group - static_cast<int64_t>(b)};
    __syncthreads();
  }
  if (r >= a.T) return;
  int64_t target = -1;
  if (!row_counts(a, r, target)) {
    zero_row<T, G>(a, r, tid);
    return;
  }
  const T* x = static_cast<const T*>(a.x) + a.in.at(r);
  const Span<T> sp(x, a.V);
  const uint4* xv = sp.vecs(x);
  uint4 w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    w[i] = tid + i * G < sp.nvec ? ld16(xv + tid + i * G) : neg_inf_vec<T>();
  const int edge = tid < kEdges ? sp.edge(tid) : -1;
  const float xe = edge >= 0 ? to_f(x[edge]) : -INFINITY;
  const bool ok = target >= 0 && target < a.V;
  const float xt = ok ? to_f(x[target]) : NAN;
  Token tk{};
  float weight = 0.f;
  if (OBJ == kPolicy) {
    tk = load_token(a, r);
    weight = static_cast<float>(token_weight(a, counts, r) * a.inv_tau);
  } else if (warp == 0) {
    const TeacherSums t = teacher_weights<T>(a, r, x, tid, s_p, s_x, s_id);
    if (tid == 0) s_t[group] = t;
  }
  float m = xe;
#pragma unroll
  for (int i = 0; i < NV; ++i) m = fmaxf(m, Vec<T>::max(w[i]));
  m = warp_max(m);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) redf[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < G / 32; ++j) m = fmaxf(m, redf[0][j]);
  } else {
    __syncwarp();
  }
  if (OBJ == kDistill)
    for (int j = tid; j < a.K; j += G)
      if (s_id[j] >= 0) seen[group].add(s_id[j]);
  const bool far = far_max(m, a.c);
  if (far) {
#pragma unroll
    for (int i = 0; i < NV; ++i) shift_vec<T>(w[i], m);
  }
  const ExpScale ks(far ? 0.f : m, a.c);
  uint64_t e[NV][E / 2];
  uint64_t acc2 = f2_splat(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    exp_vec<T>(w[i], ks, e[i]);
#pragma unroll
    for (int j = 0; j < E / 2; ++j) acc2 = f2_add(acc2, e[i][j]);
  }
  float s, hi;
  f2_unpack(acc2, s, hi);
  const float ee = xe == -INFINITY ? 0.f : ex2((xe - m) * a.c);
  s = warp_sum((s + hi) * ks.fix + ee);
  if (G > 32) {
    if ((threadIdx.x & 31) == 0) redf[1][warp] = s;
    __syncthreads();
    s = 0.f;
#pragma unroll
    for (int j = 0; j < G / 32; ++j) s += redf[1][j];
  } else {
    __syncwarp();
  }
  if (m == -INFINITY) s = NAN;
  const float inv_s = 1.f / s;
  float k = 0.f;
  if (OBJ == kDistill) {
    const TeacherSums t = s_t[group];
    k = teacher_coef(t, row_share(a, counts));
    if (tid == 0) {
      if (t.bad) note_bad_index(a);
      a.row[r] = RowStat{m, s, t.t_sum, 0.f, t.about(m)};
    }
  } else {
    // by one warp: conversions to and from fp64 share a pipe with 2^x
    if (warp == 0) k = policy_coef<T>(a, tk, xt, m, s, weight);
    if (G > 32) {
      if (tid == 0) s_k = k;
      __syncthreads();
      k = s_k;
    }
    if (tid == 0) {
      if (!ok) note_bad_index(a);
      a.row[r] = RowStat{m, s, xt, 0.f, 0.0};
    }
  }
  if (a.dx == nullptr) return;
  k *= grad_factor(a);
  if (k == 0.f) {
    zero_row<T, G>(a, r, tid);
    return;
  }
  T* dx = static_cast<T*>(a.dx) + a.out.at(r);
  const float kq = (OBJ == kDistill ? k : -k) * inv_s;
  const uint64_t kq2 = f2_splat(kq * ks.fix);
  const bool same = same_phase<T>(x, dx);
  uint4* dv = reinterpret_cast<uint4*>(dx + sp.head);
  const auto scaled = [&](int i) {
#pragma unroll
    for (int j = 0; j < E / 2; ++j) e[i][j] = f2_mul(e[i][j], kq2);
    return Vec<T>::pack(e[i]);
  };
  if (same) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (tid + i * G < sp.nvec) dv[tid + i * G] = scaled(i);
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      store_apart<T>(reinterpret_cast<T*>(dv + tid + i * G), scaled(i), tid + i * G < sp.nvec);
  }
  if (edge >= 0) put(dx + edge, ee * kq);
  if (OBJ == kPolicy) {
    // the target's value, by the thread that has just written what the others hold there
    if (ok && tid == sp.owner(static_cast<int>(target), G))
      put(dx + target, k + ex2((xt - m) * a.c) * kq);
  } else {
    group_sync<G>();
    const float inv_t = 1.f / s_t[group].t_sum;
    for (int j = tid; j < a.K; j += G)
      if (s_id[j] >= 0)
        put(dx + s_id[j], teacher_value(a, j, !seen[group].again(s_id[j]), s_p, s_id,
                                        ex2((s_x[j] - m) * a.c) * inv_s, inv_t, k));
  }
}

// ---- rows held by one CTA, or by the CTAs of a cluster ------------------------------

// The same for longer rows. A persistent CTA, two or three of them an SM, holds a row or its share
// of one in the registers of seven or four warps. Its last warp, the producer, brings the next rows
// in through a ring of shared memory with bulk copies, so that HBM is read and written without a
// pause, and with them what else the rows need: their edges, the token's numbers or the teacher's
// entries. A chunk of the ring is free as soon as it is in registers. Rows are held as they are,
// not as exponentials, which are taken twice (for the sum and for the gradient): half the
// registers, hence CTAs that work while others of the SM wait for their reductions.
//
// A cluster of cs CTAs shares rows too long for one, or few rows of any length; its CTAs exchange
// maxima and sums through each other's shared memory.
//
// One CTA a row: 16 x 512 rows of 32000 bf16, two thirds of them counted (872 MB), take 159 us,
// 5.5 TB/s, near what DRAM gives a mix of reads and writes (6.0 TB/s). Each row costs its CTAs some
// 2 us of latency (two reductions, in a cluster the exchange) besides its bytes, so shares that
// leave registers empty are slower: 3 x 611 rows of 100277 (649 MB, four CTAs, 78 percent full)
// take 164 us, 4.0 TB/s; sweeping them twice takes 235 us. Rows held in shared memory instead, the
// gradient of one behind the sums of the next, took 217 us, one or two CTAs an SM.
constexpr int kRingVecs = 18;  // a thread's vectors, at most
constexpr int kChunkVecs = 3;  // of them in a chunk
constexpr int kMaxStages = 9;
template <int WARPS>
struct Ring {
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kChunk = kChunkVecs * kThreads;  // vectors
  static constexpr int kCap = kRingVecs * kThreads;     // vectors of a share, at most
  static constexpr int kCtas = 16 / (WARPS + 1);        // an SM, of 128 registers a thread
  static constexpr int kSmem = 208 * 1024 / kCtas - 2048 * (kCtas - 2);
};
constexpr int kZeroBytes = 8192;                         // source of the rows of zeros
constexpr int kMaxCluster = 8;

// What the producer puts down for a row, so that the consumers' registers hold the row itself.
struct RowInfo {
  int64_t row;        // -1: no more
  char* dx;           // the gradient row, and where this CTA's share of its vectors goes
  char* dv;
  int32_t nv;         // vectors in this CTA's share
  int32_t head, nvec; // the row's Span
  int32_t same;       // the gradient row has the input row's phase
  int32_t target;     // -1 outside the vocabulary
  int32_t owner;      // the thread that holds the target, -1: another CTA's
  float xt, w;
  Token tk;
  TeacherSums t;
  float edge[kEdges];
  int32_t edge_at[kEdges];  // -1: none (all of them in CTAs other than the first)
};

// What a CTA of a cluster knows of a row: its share's maximum and sum.
struct __align__(8) Share {
  float m, s;
};

// Whether element i of a row lies in the share of nv vectors from `start` on; the first CTA's
// share has the edges.
template <typename T>
__device__ __forceinline__ bool in_share(int head, int nvec, int start, int nv, int rank, int i) {
  const int v = (i - head) / Vec<T>::kE - start;
  return i < head || i >= head + nvec * Vec<T>::kE ? rank == 0 : v >= 0 && v < nv;
}
// The thread that holds element i of its share.
template <typename T, int THREADS>
__device__ __forceinline__ int share_owner(const Span<T>& sp, int start, int i) {
  if (i < sp.head || i >= sp.head + sp.nvec * Vec<T>::kE) return sp.owner(i, 1);
  return ((i - sp.head) / Vec<T>::kE - start) % THREADS;
}

template <int THREADS>
__device__ __forceinline__ void ring_sync() {
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ bool ring_all(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(ok)), "n"(THREADS)
      : "memory");
  return r != 0;
}

// Bulk copy into this CTA's shared memory (both addresses and the size multiples of 16 bytes).
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(ptx::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(ptx::smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(ptx::smem_u32(src)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(
                   ptx::smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
// 8 bytes into a CTA of the cluster, counted on its barrier.
__device__ __forceinline__ void store_remote(uint32_t dst, float a, float b, uint32_t bar) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
          dst),
      "f"(a), "f"(b), "r"(bar)
      : "memory");
}

// The rows of one CTA: every step-th of those that count, every grid-th of the others. Listed
// by the CTA itself while they are few, in the order of count_kernel's list.
constexpr int kOwnRows = 256;
constexpr int kOwnSeqs = 256;
// Below this the CTAs are quicker: at 1833 rows 164 us against 165, at 4096 99 against 97, at 8192
// 175 against 165.
constexpr int64_t kOwnTotal = 2048;
struct OwnRows {
  int32_t row[kOwnRows], rest[kOwnRows], seq[kOwnSeqs];
};
template <int THREADS>
__device__ __forceinline__ int list_own(const RowArgs& a, uint32_t first, uint32_t step,
                                        OwnRows* own) {
  constexpr int kWarps = THREADS / 32, kRows = 64 / kWarps;
  constexpr int kCells = kRows * kWarps;  // two a lane, at most
  __shared__ int32_t s_cell[64];
  __shared__ int32_t s_end;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (a.per_sequence)
    for (int b = tid; b < kOwnSeqs; b += THREADS) own->seq[b] = 0;
  int before = 0;  // counted rows of the blocks in front
  const int T = static_cast<int>(a.T);
  for (int r0 = 0; r0 < T; r0 += kRows * THREADS) {
    bool in[kRows];
    uint32_t ballot[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int r = r0 + j * THREADS + tid;
      int64_t target;
      in[j] = r < T && row_counts(a, r, target);
    }
    __syncthreads();  // the cells of the block in front are read, the sequences are cleared
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      ballot[j] = __ballot_sync(0xffffffffu, in[j]);
      if (lane == 0) s_cell[j * kWarps + warp] = __popc(ballot[j]);
      if (a.per_sequence && in[j])
        atomicAdd(&own->seq[a.in.seq(r0 + j * THREADS + tid)], 1);
    }
    __syncthreads();
    if (warp == 0) {
      const int n0 = 2 * lane < kCells ? s_cell[2 * lane] : 0,
                n1 = 2 * lane + 1 < kCells ? s_cell[2 * lane + 1] : 0;
      int incl = n0 + n1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      s_cell[2 * lane] = before + incl - n0 - n1;
      s_cell[2 * lane + 1] = before + incl - n1;
      if (lane == 31) s_end = before + incl;
    }
    __syncthreads();
    before = s_end;
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int r = r0 + j * THREADS + tid;
      const uint32_t rank = s_cell[j * kWarps + warp] + __popc(ballot[j] & ((1u << lane) - 1u));
      if (in[j]) {
        if (rank % step == first) own->row[rank / step] = r;
      } else if (r < T) {
        const uint32_t z = r - rank;
        if (z % gridDim.x == blockIdx.x) own->rest[z / gridDim.x] = r;
      }
    }
  }
  __syncthreads();
  return before;
}

// SHORT: fewer stages than a row may have chunks, for many teacher entries.
template <typename T, int OBJ, int WARPS, bool SHORT>
__global__ void __launch_bounds__((WARPS + 1) * 32, Ring<WARPS>::kCtas)
    ring_kernel(RowArgs a, int cs, int per, int stages) {
  constexpr int E = Vec<T>::kE, kThreads = Ring<WARPS>::kThreads, kChunk = Ring<WARPS>::kChunk;
  extern __shared__ __align__(16) char smem[];
  uint4* zeros = reinterpret_cast<uint4*>(smem);
  uint4* ring = zeros + kZeroBytes / 16;  // [stages][kChunk]
  float* s_p0 = reinterpret_cast<float*>(ring + stages * kChunk);
  float* s_x0 = s_p0 + (stages + 1) * a.K4;  // each [stages + 1][K4]
  int32_t* s_id0 = reinterpret_cast<int32_t*>(s_x0 + (stages + 1) * a.K4);
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], exchanged[2];
  // A row's numbers come with its first chunk and are used until its end. The producer is at
  // most `stages` rows ahead of a row whose first chunk every warp has read, and a warp reads
  // that after it is done with the row before: one slot more than stages.
  __shared__ RowInfo info[kMaxStages + 1];
  __shared__ Share share[2][kMaxCluster];
  __shared__ float red_m[WARPS], red_s[WARPS];
  __shared__ double2 red_t[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = cs > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const int start = rank * per;  // this CTA's first vector of a row; rank 0 has the edges too
  if (tid == 0) {
    for (int i = 0; i < stages; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], WARPS);
    }
    ptx::mbar_init(&exchanged[0], 1);
    ptx::mbar_init(&exchanged[1], 1);
    ptx::fence_mbar_init();
  }
  for (int i = tid; i < kZeroBytes / 16; i += kThreads + 32) zeros[i] = make_uint4(0, 0, 0, 0);
  ptx::fence_proxy_async_smem();  // bulk copies read them
  __syncthreads();
  if (cs > 1) ptx::cluster_sync();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  ptx::griddep_wait();
  __shared__ OwnRows own;
  const int64_t first = blockIdx.x / cs, step = gridDim.x / cs;
  Counts counts = listed_counts(a);
  if (a.self_count)
    counts = Counts{list_own<kThreads + 32>(a, static_cast<uint32_t>(first),
                                                static_cast<uint32_t>(step), &own),
                    own.seq};
  const int64_t total = counts.total;
  const int n_row = total > first ? static_cast<int>((total - first + step - 1) / step) : 0;
  const auto row_of = [&](int i) {
    return a.self_count ? own.row[i] : a.list[first + i * step];
  };

  if (warp == WARPS) {
    // ---- producer: 32 rows' numbers at a time, then each row's copies
    int i = 0, st = 0, slot = 0;  // chunks so far, the next one's stage, the next row's slot
    uint32_t phase = 0;
    bool ok = true, more = true;
    // The rows of zeros, dealt to every CTA, are written between the others by bulk copies from
    // shared memory, which cost the threads that hold rows nothing.
    const int64_t rest = a.T - total;
    const int n_zero = rest > blockIdx.x
                           ? static_cast<int>((rest - blockIdx.x + gridDim.x - 1) / gridDim.x)
                           : 0;
    int z = 0, done = 0;
    const auto rest_of = [&](int i) {
      return a.self_count
                 ? own.rest[i]
                 // from the end backwards, as count_kernel puts them down
                 : a.list[a.T - 1 - blockIdx.x - i * static_cast<int64_t>(gridDim.x)];
    };
    int32_t z_row = n_zero > 0 ? rest_of(0) : 0;
    const auto zero_rows = [&](int until) {
      for (; z < until; ++z) {
        T* dx = static_cast<T*>(a.dx) + a.out.at(z_row);
        if (OBJ == kPolicy && lane == 0) zero_outputs(a, z_row);
        if (z + 1 < n_zero) z_row = rest_of(z + 1);
        if (a.dx == nullptr) continue;
        const Span<T> so(dx, a.V);
        if (lane < kEdges && so.edge(lane) >= 0) put(dx + so.edge(lane), 0.f);
        char* to = reinterpret_cast<char*>(dx + so.head);
        const int bytes = so.nvec * 16;
        for (int at = lane * kZeroBytes; at < bytes; at += 32 * kZeroBytes)
          bulk_store(to + at, zeros, min(kZeroBytes, bytes - at));
        ptx::bulk_commit_group();
      }
    };
    for (int base = 0; more && ok; base += 32) {
      const bool live = base + lane < n_row;
      int64_t row = -1, x_at = 0, dx_at = 0;
      int32_t target = -1;
      Token tk{};
      float xt = NAN, w = 0.f;
      if (live) {
        row = row_of(base + lane);
        x_at = a.in.at(row);
        dx_at = a.out.at(row);
        if (OBJ == kPolicy) {
          const int64_t t = a.targets[row];
          if (t >= 0 && t < a.V) {
            target = static_cast<int32_t>(t);
            xt = to_f((static_cast<const T*>(a.x) + x_at)[t]);
          }
          tk = load_token(a, row);
          w = static_cast<float>(token_weight(a, counts, row) * a.inv_tau);
        } else {
          w = row_share(a, counts);
        }
      }
      const int n = __popc(__ballot_sync(0xffffffffu, live));
      more = n == 32;
      for (int j = 0; j <= n && ok; ++j) {
        if (j == n && more) break;  // the end goes behind the last row
        const int src = j & 31;
        const T* x = static_cast<const T*>(a.x) + __shfl_sync(0xffffffffu, x_at, src);
        T* dx = static_cast<T*>(a.dx) + __shfl_sync(0xffffffffu, dx_at, src);
        const int64_t r = __shfl_sync(0xffffffffu, row, src);
        const Span<T> sp(x, a.V);
        const int nv = j < n ? max(0, min(per, sp.nvec - start)) : 0;
        const uint4* from = sp.vecs(x) + start;
        RowInfo* inf = &info[slot];
        // The first chunk brings the numbers, and there is one even without vectors. The copies
        // for which there is room go out before the numbers are put together.
        const int chunks = max(1, (nv + kChunk - 1) / kChunk);
        const int st_row = st;
        bool numbers = false;
        for (int c = 0; c < chunks || !numbers; ++c) {
          bool room = c < chunks && i < stages;
          if (!room && c < chunks) {
            room = numbers || c == 0 ? ptx::mbar_wait(&empty[st], phase ^ 1u)
                                     : ptx::mbar_try_wait(&empty[st], phase ^ 1u);
            room = __all_sync(0xffffffffu, room);
            if (!room && (numbers || c == 0)) {
              ok = false;
              break;
            }
          }
          if (!room) {
            // all copies are out, or the next has to wait: the numbers
            if (j < n) {
              if (lane < kEdges) {
                const int e = rank == 0 ? sp.edge(lane) : -1;
                inf->edge_at[lane] = e;
                inf->edge[lane] = e >= 0 ? to_f(x[e]) : -INFINITY;
              }
              if (OBJ == kDistill) {
                const TeacherSums t = teacher_weights<T>(a, r, x, lane, s_p0 + slot * a.K4,
                                                         s_x0 + slot * a.K4,
                                                         s_id0 + slot * a.K4);
                if (lane == 0) inf->t = t;
              }
            }
            if (lane == src) {
              inf->row = j < n ? r : -1;
              inf->dx = reinterpret_cast<char*>(dx);
              inf->dv = reinterpret_cast<char*>(dx + sp.head + static_cast<int64_t>(start) * E);
              inf->nv = nv;
              inf->head = sp.head;
              inf->nvec = sp.nvec;
              inf->same = same_phase<T>(x, dx);
              inf->target = target;
              inf->owner =
                  target >= 0 && in_share<T>(sp.head, sp.nvec, start, nv, rank, target)
                      ? share_owner<T, kThreads>(sp, start, target)
                      : -1;
              inf->xt = xt;
              inf->w = w;
              inf->tk = tk;
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&full[st_row]);
            numbers = true;
            --c;  // this chunk again, with a wait
            continue;
          }
          const int m = min(kChunk, nv - c * kChunk);
          if (lane == 0) {
            if (m > 0) {
              mbar_expect_tx(&full[st], m * 16u);
              bulk_load(ring + st * kChunk, from + c * kChunk, m * 16u, &full[st]);
            }
            if (c > 0) ptx::mbar_arrive(&full[st]);
          }
          ++i;
          if (++st == stages) {
            st = 0;
            phase ^= 1u;
          }
        }
        slot = slot == stages ? 0 : slot + 1;
        ++done;
        if (n_zero > 0 && j < n)
          zero_rows(static_cast<int>(static_cast<int64_t>(n_zero) * done / n_row));
      }
    }
    zero_rows(n_zero);
    ptx::bulk_wait_group_all();
    if (!ok) {
      if (lane == 0) atomicMax(a.err, static_cast<int32_t>(kDevErrLossTimeout));
      // copies in flight end before this CTA does
      for (int j = 0; j < min(i, stages); ++j)
        ptx::mbar_wait(&full[(i - 1 - j) % stages], ((i - 1 - j) / stages) & 1);
    }
    __syncwarp();
  } else {
    const float factor = grad_factor(a);
    bool ok = true;
    int st = 0, slot = 0;
    uint32_t phase = 0;
    for (uint32_t i = 0;; ++i) {
      const RowInfo* inf = &info[slot];
      // the row's share into registers, and its maximum
      uint4 w[kRingVecs];
      const int st_row = st;
      ok = ptx::mbar_wait(&full[st], phase) && ok;
      const int nv = inf->nv;
      const float xe = tid < kEdges ? inf->edge[tid] : -INFINITY;
#pragma unroll
      for (int c = 0; c < kRingVecs / kChunkVecs; ++c) {
        if (c == 0 || c * kChunk < nv) {
          if (SHORT && c >= stages) {
            // this chunk takes the stage of one of the same row, which has to be free first
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&empty[st]);
          }
          if (c > 0) ok = ptx::mbar_wait(&full[st], phase) && ok;
          const uint4* buf = ring + st * kChunk + tid;
#pragma unroll
          for (int j = 0; j < kChunkVecs; ++j) w[c * kChunkVecs + j] = buf[j * kThreads];
          if (nv < (c + 1) * kChunk) {  // what the chunk does not fill is old
#pragma unroll
            for (int j = 0; j < kChunkVecs; ++j)
              if (c * kChunk + j * kThreads + tid >= nv)
                w[c * kChunkVecs + j] = neg_inf_vec<T>();
          }
          if (++st == stages) {
            st = 0;
            phase ^= 1u;
          }
        } else {
#pragma unroll
          for (int j = 0; j < kChunkVecs; ++j) w[c * kChunkVecs + j] = neg_inf_vec<T>();
        }
      }
      float m = xe;
#pragma unroll
      for (int j = 0; j < kRingVecs; ++j) m = fmaxf(m, Vec<T>::max(w[j]));
      // every lane has its part of the chunks: those still in the ring are free
      __syncwarp();
      if (lane == 0)
        for (int c = 0, e = st_row; (!SHORT || c < stages) && (c == 0 || c * kChunk < nv); ++c) {
          ptx::mbar_arrive(&empty[e]);
          if (++e == stages) e = 0;
        }
      m = warp_max(m);
      if (lane == 0) red_m[warp] = m;
      // one barrier for the maximum and for every thread's waits: all leave here, or none
      if (!ring_all<kThreads>(ok)) {
        if (tid == 0) atomicMax(a.err, static_cast<int32_t>(kDevErrLossTimeout));
        break;
      }
      if (inf->row < 0) break;
      m = red_m[0];
#pragma unroll
      for (int j = 1; j < WARPS; ++j) m = fmaxf(m, red_m[j]);
      const bool far = far_max(m, a.c);
      if (far) {
#pragma unroll
        for (int j = 0; j < kRingVecs; ++j) shift_vec<T>(w[j], m);
      }
      const ExpScale ks(far ? 0.f : m, a.c);
      uint64_t acc[E / 2];
#pragma unroll
      for (int l = 0; l < E / 2; ++l) acc[l] = f2_splat(0.f);
#pragma unroll
      for (int c = 0; c < kRingVecs / kChunkVecs; ++c) {
        if (c * kChunk < nv) {
#pragma unroll
          for (int j = 0; j < kChunkVecs; ++j) {
            uint64_t e[E / 2];
            exp_vec<T>(w[c * kChunkVecs + j], ks, e);
#pragma unroll
            for (int l = 0; l < E / 2; ++l) acc[l] = f2_add(acc[l], e[l]);
          }
        }
      }
      uint64_t acc2 = f2_add(acc[0], acc[1]);
      if (E == 8) acc2 = f2_add(acc2, f2_add(acc[E / 2 - 2], acc[E / 2 - 1]));
      const float ee = xe == -INFINITY ? 0.f : ex2((xe - m) * a.c);
      float s, hi;
      f2_unpack(acc2, s, hi);
      s = warp_sum((s + hi) * ks.fix + ee);
      if (lane == 0) red_s[warp] = s;
      ring_sync<kThreads>();
      s = 0.f;
#pragma unroll
      for (int j = 0; j < WARPS; ++j) s += red_s[j];
      float scale = 1.f, m_row = m;
      if (cs > 1) {
        const uint32_t b = i & 1;
        if (tid == 0) ptx::mbar_arrive_expect_tx(&exchanged[b], 8u * cs);
        if (tid < cs)
          store_remote(ptx::mapa_shared(ptx::smem_u32(&share[b][rank]), tid), m, s,
                       ptx::mapa_shared(ptx::smem_u32(&exchanged[b]), tid));
        ok = ptx::mbar_wait(&exchanged[b], (i >> 1) & 1) && ok;
        m_row = share[b][0].m;
        for (int j = 1; j < cs; ++j) m_row = fmaxf(m_row, share[b][j].m);
        s = 0.f;
        for (int j = 0; j < cs; ++j) {
          // a share of -inf alone adds nothing
          const Share o = share[b][j];
          s += o.s * (o.m == -INFINITY ? 0.f : ex2((o.m - m_row) * a.c));
        }
        scale = m == -INFINITY ? 0.f : ex2((m - m_row) * a.c);
      }
      if (m_row == -INFINITY) s = NAN;
      const float inv_s = 1.f / s;
      float k;
      if (OBJ == kDistill) {
        k = teacher_coef(inf->t, inf->w);
        if (tid == 0 && rank == 0) {
          if (inf->t.bad) note_bad_index(a);
          a.row[inf->row] = RowStat{m_row, s, inf->t.t_sum, 0.f, inf->t.about(m_row)};
        }
      } else {
        k = policy_coef<T>(a, inf->tk, inf->xt, m_row, s, inf->w);
        if (tid == 0 && rank == 0) {
          if (inf->target < 0) note_bad_index(a);
          a.row[inf->row] = RowStat{m_row, s, inf->xt, 0.f, 0.0};
        }
      }
      k *= factor;
      if (a.dx != nullptr) {
        const bool zero = k == 0.f, same = inf->same;
        const float kq = zero ? 0.f : (OBJ == kDistill ? k : -k) * inv_s * scale;
        const uint64_t kq2 = f2_splat(kq * ks.fix);
        uint4* dv = reinterpret_cast<uint4*>(inf->dv) + tid;
#pragma unroll
        for (int c = 0; c < kRingVecs / kChunkVecs; ++c) {
          if (c * kChunk < nv) {
            uint4 o[kChunkVecs];
#pragma unroll
            for (int j = 0; j < kChunkVecs; ++j) {
              uint64_t e[E / 2];
              exp_vec<T>(w[c * kChunkVecs + j], ks, e);
#pragma unroll
              for (int l = 0; l < E / 2; ++l) e[l] = f2_mul(e[l], kq2);
              o[j] = Vec<T>::pack(e);
            }
            if (same) {
#pragma unroll
              for (int j = 0; j < kChunkVecs; ++j) {
                const int v = c * kChunk + j * kThreads;
                st16_if(dv + v, o[j], v + tid < nv);
              }
            } else {
#pragma unroll
              for (int j = 0; j < kChunkVecs; ++j) {
                const int v = c * kChunk + j * kThreads;
                store_apart<T>(reinterpret_cast<T*>(dv + v), o[j], v + tid < nv);
              }
            }
          }
        }
        T* dx = reinterpret_cast<T*>(inf->dx);
        if (tid < kEdges && inf->edge_at[tid] >= 0) put(dx + inf->edge_at[tid], ee * kq);
        if (!zero) {
          if (OBJ == kPolicy) {
            // the target's value, by the thread that has just written what the others hold there
            if (tid == inf->owner)
              put(dx + inf->target, k - ex2((inf->xt - m_row) * a.c) * inv_s * k);
          } else {
            ring_sync<kThreads>();
            const float* s_p = s_p0 + slot * a.K4;
            const float* s_x = s_x0 + slot * a.K4;
            const int32_t* s_id = s_id0 + slot * a.K4;
            const float inv_t = 1.f / inf->t.t_sum;
            for (int j = tid; j < a.K; j += kThreads)
              if (s_id[j] >= 0 &&
                  in_share<T>(inf->head, inf->nvec, start, nv, rank, s_id[j]))
                put(dx + s_id[j],
                    teacher_value(a, j, false, s_p, s_id, ex2((s_x[j] - m_row) * a.c) * inv_s,
                                  inv_t, k));
          }
        }
      }
      slot = slot == stages ? 0 : slot + 1;
    }
    // the terms of this CTA's tokens: thread 0 wrote what their rows left
    ring_sync<kThreads>();
    double2 terms = make_double2(0.0, 0.0);
    if (rank == 0 && ok)
      for (int i = tid; i < n_row; i += kThreads) {
        const double2 v = token_terms<OBJ>(a, counts, row_of(i));
        terms.x += v.x;
        terms.y += v.y;
      }
    terms.x = warp_sum(terms.x);
    terms.y = warp_sum(terms.y);
    if (lane == 0) red_t[warp] = terms;
    ring_sync<kThreads>();
    if (tid == 0) {
      for (int j = 1; j < WARPS; ++j) {
        terms.x += red_t[j].x;
        terms.y += red_t[j].y;
      }
      a.part[blockIdx.x] = terms;
    }
  }
  if (cs > 1) ptx::cluster_sync();  // no CTA leaves while another may still write to it
}

// ---- rows too long for a cluster -----------------------------------------------------

// One CTA a row, swept twice; the second sweep goes from the row's end, which is in L2 still,
// back to its start. One CTA an SM: its rows of up to 0.8 MB fit in L2 together, those of two do
// not. Bound by the latency of its reads, four 16-byte loads a thread: 768 rows of 300000 bf16
// that count and 256 of zeros (1.08 GB with the gradient) take 305 us, 3.5 TB/s of what has to
// move; two CTAs an SM of half the threads 316 us, a second sweep forwards with one load a
// thread 407 us.
constexpr int kRowThreads = 1024;
template <typename T, int OBJ>
__global__ void __launch_bounds__(kRowThreads) stream_kernel(RowArgs a) {
  constexpr int E = Vec<T>::kE;
  extern __shared__ __align__(16) char smem[];
  float* s_p = reinterpret_cast<float*>(smem);
  float* s_x = s_p + a.K4;
  int32_t* s_id = reinterpret_cast<int32_t*>(s_x + a.K4);
  __shared__ float redf[kRowThreads / 32];
  __shared__ double redd[kRowThreads / 32];
  __shared__ TeacherSums s_t;
  __shared__ float s_k;
  const int tid = threadIdx.x;
  ptx::griddep_wait();
  const Counts counts = listed_counts(a);
  const float factor = grad_factor(a);
  for (int64_t r = blockIdx.x; r < a.T; r += gridDim.x) {
    int64_t target = -1;
    if (!row_counts(a, r, target)) {
      zero_row<T, kRowThreads>(a, r, tid);
      continue;
    }
    const T* x = static_cast<const T*>(a.x) + a.in.at(r);
    const Span<T> sp(x, a.V);
    const bool ok = target >= 0 && target < a.V;
    const float xt = ok ? to_f(x[target]) : NAN;
    const int edge = tid < kEdges ? sp.edge(tid) : -1;
    const float xe = edge >= 0 ? to_f(x[edge]) : 0.f;
    if (OBJ == kDistill && tid < 32) {
      const TeacherSums t = teacher_weights<T>(a, r, x, tid, s_p, s_x, s_id);
      if (tid == 0) s_t = t;
    }
    float m;
    double sd;
    thread_stats<T, kRowThreads, 4, false>(x, sp, tid, a.c, a.c_lo, m, sd);
    group_combine<kRowThreads, false>(m, sd, a, redf, redd);
    const float s = static_cast<float>(sd), inv_s = 1.f / s;
    float k = 0.f;
    if (OBJ == kDistill) {
      k = teacher_coef(s_t, row_share(a, counts));
      if (tid == 0) {
        if (s_t.bad) note_bad_index(a);
        a.row[r] = RowStat{m, s, s_t.t_sum, 0.f, s_t.about(m)};
      }
    } else {
      if (tid < 32)  // one warp's conversions from and to fp64, not those of 32
        k = policy_coef<T>(a, load_token(a, r), xt, m, s,
                           static_cast<float>(token_weight(a, counts, r) * a.inv_tau));
      if (tid == 0) s_k = k;
      __syncthreads();
      k = s_k;
      if (tid == 0) {
        if (!ok) note_bad_index(a);
        a.row[r] = RowStat{m, s, xt, 0.f, 0.0};
      }
    }
    k *= factor;
    if (a.dx != nullptr && k == 0.f) {
      zero_row<T, kRowThreads>(a, r, tid);
    } else if (a.dx != nullptr) {
      T* dx = static_cast<T*>(a.dx) + a.out.at(r);
      const bool same = same_phase<T>(x, dx);
      const bool far = far_max(m, a.c);
      const ExpScale ks(far ? 0.f : m, a.c);
      const float kq = (OBJ == kDistill ? k : -k) * inv_s;
      const uint64_t kq2 = f2_splat(kq * ks.fix);
      const uint4* xv = sp.vecs(x);
      uint4* dv = reinterpret_cast<uint4*>(dx + sp.head);
      constexpr int U = 4, kStep = U * kRowThreads;
      for (int base = (sp.nvec - 1) / kStep * kStep + tid; base >= 0; base -= kStep) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (base + u * kRowThreads < sp.nvec) w[u] = ld16(xv + base + u * kRowThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = base + u * kRowThreads;
          if (far) shift_vec<T>(w[u], m);
          uint64_t e[E / 2];
          exp_vec<T>(w[u], ks, e);
#pragma unroll
          for (int i = 0; i < E / 2; ++i) e[i] = f2_mul(e[i], kq2);
          if (!same)
            store_apart<T>(dx + sp.head + static_cast<int64_t>(v) * E, Vec<T>::pack(e),
                           v < sp.nvec);
          else if (v < sp.nvec)
            __stcs(dv + v, Vec<T>::pack(e));
        }
      }
      if (edge >= 0) put(dx + edge, ex2((xe - m) * a.c) * kq);
      if (OBJ == kPolicy) {
        if (ok && tid == sp.owner(static_cast<int>(target), kRowThreads))
          put(dx + target, k + ex2((xt - m) * a.c) * kq);
      } else {
        __syncthreads();
        const float inv_t = 1.f / s_t.t_sum;
        for (int j = tid; j < a.K; j += kRowThreads)
          if (s_id[j] >= 0)
            put(dx + s_id[j], teacher_value(a, j, false, s_p, s_id,
                                            ex2((s_x[j] - m) * a.c) * inv_s, inv_t, k));
      }
    }
    __syncthreads();
  }
}

// Both sums over a CTA of 32 N threads, in its thread 0.
template <int N>
__device__ __forceinline__ double2 cta_sum(double2 v, double2* red) {
  v.x = warp_sum(v.x);
  v.y = warp_sum(v.y);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < N; ++w) {
      v.x += red[w].x;
      v.y += red[w].y;
    }
  return v;
}

// Whether this CTA is the last of the grid to have written its partial sum.
__device__ __forceinline__ bool last_to_write(const RowArgs& a, double2 v, bool* s_last) {
  if (threadIdx.x == 0) {
    a.part[blockIdx.x] = v;
    __threadfence();
    *s_last = atomicAdd(&a.head->ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (*s_last) __threadfence();
  return *s_last;
}

// The partial sums added in their order: loss and KL.
template <int N>
__device__ __forceinline__ void sum_parts(const RowArgs& a, int n, double2* red) {
  double2 v = make_double2(0.0, 0.0);
  for (int i = threadIdx.x; i < n; i += 32 * N) {
    const double2 p = __ldcg(&a.part[i]);
    v.x += p.x;
    v.y += p.y;
  }
  v = cta_sum<N>(v, red);
  if (threadIdx.x == 0) {
    *a.loss = static_cast<float>(v.x);
    if (a.kl) *a.kl = static_cast<float>(v.y);
  }
}

// The tokens' terms after direct_kernel or stream_kernel; the CTA that ends last adds up.
template <int OBJ>
__global__ void __launch_bounds__(kTokenThreads) token_kernel(RowArgs a) {
  __shared__ double2 red[kTokenThreads / 32], red2[kTokenThreads / 32];
  __shared__ bool s_last;
  __shared__ int32_t s_seq[kSelfRows], s_total;
  ptx::griddep_wait();
  Counts counts = listed_counts(a);
  if (a.self_count) {  // one CTA
    for (int b = threadIdx.x; b < kSelfRows; b += kTokenThreads) s_seq[b] = 0;
    if (threadIdx.x == 0) s_total = 0;
    __syncthreads();
#pragma unroll 4
    for (int r = threadIdx.x; r < a.T; r += kTokenThreads) {
      int64_t target;
      if (!row_counts(a, r, target)) continue;
      atomicAdd(&s_total, 1);
      if (a.per_sequence) atomicAdd(&s_seq[a.in.seq(r)], 1);
    }
    __syncthreads();
    counts = Counts{s_total, s_seq};
  }
  double2 v = make_double2(0.0, 0.0);
  for (int64_t r = blockIdx.x * static_cast<int64_t>(kTokenThreads) + threadIdx.x; r < a.T;
       r += gridDim.x * static_cast<int64_t>(kTokenThreads)) {
    int64_t target;
    if (row_counts(a, r, target)) {
      const double2 t = token_terms<OBJ>(a, counts, r);
      v.x += t.x;
      v.y += t.y;
    } else if (OBJ == kPolicy) {
      zero_outputs(a, r);
    }
  }
  v = cta_sum<kTokenThreads / 32>(v, red);
  if (a.self_count) {
    if (threadIdx.x == 0) {
      *a.loss = static_cast<float>(v.x);
      if (a.kl) *a.kl = static_cast<float>(v.y);
    }
    return;
  }
  if (last_to_write(a, v, &s_last)) sum_parts<kTokenThreads / 32>(a, gridDim.x, red2);
}

// The sums that the CTAs of ring_kernel left.
__global__ void __launch_bounds__(256) finish_kernel(RowArgs a, int n) {
  __shared__ double2 red[8];
  ptx::griddep_wait();
  sum_parts<8>(a, n, red);
}

// One CTA per pair: the two sequences' summed log ratios, the pair's loss and dL/dlp of its
// tokens; the CTA that ends last adds the losses up.
constexpr int kPairThreads = 512;
__global__ void __launch_bounds__(kPairThreads) pair_kernel(RowArgs a, int64_t P, double beta,
                                                            double smooth, float* rewards) {
  constexpr int kW = kPairThreads / 32;
  __shared__ double2 red[kW], red2[kW];
  __shared__ float s_dh;
  __shared__ bool s_last;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  ptx::griddep_wait();
  const int64_t p = blockIdx.x, S = a.T / (2 * P);
  double2 sum = make_double2(0.0, 0.0);
  for (int64_t i = threadIdx.x; i < 2 * S; i += kPairThreads) {
    const bool side = i >= S;
    const int64_t r = side ? (p + P) * S + i - S : p * S + i;
    if (a.targets[r] == a.ignore) continue;
    const double d = a.lp64[r] - (a.ref_logps ? static_cast<double>(a.ref_logps[r]) : 0.0);
    sum.x += side ? 0.0 : d;
    sum.y += side ? d : 0.0;
  }
  sum = cta_sum<kW>(sum, red);
  double2 loss = make_double2(0.0, 0.0);
  if (threadIdx.x == 0) {
    const double won = beta * sum.x, lost = beta * sum.y, h = won - lost;
    rewards[p] = static_cast<float>(won);
    rewards[p + P] = static_cast<float>(lost);
    // no smoothing: no second term, which is infinite for a rejected token without probability
    loss.x = ((1.0 - smooth) * softplus(-h) + (smooth > 0.0 ? smooth * softplus(h) : 0.0)) /
             static_cast<double>(P);
    // sigma(-h) = 1 / (1 + e^h)
    s_dh = static_cast<float>((smooth / (1.0 + exp(-h)) - (1.0 - smooth) / (1.0 + exp(h))) * beta /
                              static_cast<double>(P));
  }
  __syncthreads();
  const float dh = s_dh;
  for (int64_t i = threadIdx.x; i < 2 * S; i += kPairThreads) {
    const bool side = i >= S;
    const int64_t r = side ? (p + P) * S + i - S : p * S + i;
    a.coef[r] = a.targets[r] == a.ignore ? 0.f : (side ? -dh : dh);
  }
  if (last_to_write(a, loss, &s_last)) sum_parts<kW>(a, gridDim.x, red2);
}

// Gradient rows from saved statistics: k (1[v = target] - q_v). A group of G threads takes
// G * kBwdU vectors of one row; nothing is reduced, so rows of any length keep every SM busy.
// Bound by DRAM (4 x 333 x 50257 bf16, of which two thirds count: 226 MB in 38 us, 6.0 TB/s).
// Behind the statistics it goes backwards and its stores are the first that L2 gives up, as are
// the rows of zeros before it, so that it finds part of the input there: the preference loss over
// 8 x 512 rows of 32000 takes 115 us, with plain stores 119.
constexpr int kBwdThreads = 256;
constexpr int kBwdU = 4;
template <typename T, int G>
__global__ void __launch_bounds__(kBwdThreads) logprobs_bwd_kernel(RowArgs a, int chunks) {
  constexpr int E = Vec<T>::kE;
  const int tid = threadIdx.x % G;
  const int64_t unit = blockIdx.x * int64_t{kBwdThreads / G} + threadIdx.x / G;
  if (unit >= a.T * chunks) return;
  // behind the statistics: from the last row on, which L2 still holds
  const int64_t at_row = unit / chunks, r = a.zeros_done ? a.T - 1 - at_row : at_row;
  const int chunk = static_cast<int>(unit - at_row * chunks);
  const int v0 = chunk * (G * kBwdU) + tid;
  const T* x = static_cast<const T*>(a.x) + a.in.at(r);
  T* dx = static_cast<T*>(a.dx) + a.out.at(r);
  const int64_t target = a.targets[r];
  const bool counts = target != a.ignore;
  if (a.zeros_done && !counts) {
    // With no other rows the grid would end before pair_kernel, which whatever comes behind it on
    // the stream then would not wait for: one CTA does.
    if (blockIdx.x == 0) ptx::griddep_wait();
    return;
  }
  const Span<T> sp(x, a.V);
  const uint4* xv = sp.vecs(x);
  uint4 w[kBwdU];
  if (counts) {
    // the input is nobody's output: it is on its way before pair_kernel has ended
#pragma unroll
    for (int u = 0; u < kBwdU; ++u)
      if (v0 + u * G < sp.nvec) w[u] = ld16(xv + v0 + u * G);
  }
  ptx::griddep_wait();
  const bool ok = target >= 0 && target < a.V;  // a row of NaN otherwise
  const float k =
      counts ? (ok ? a.g[r] * grad_factor(a) * static_cast<float>(a.inv_tau) : NAN) : 0.f;
  if (k == 0.f) {
    // zeros need no input: whole vectors of the output's own phase
    const Span<T> so(dx, a.V);
    uint4* dv = reinterpret_cast<uint4*>(dx + so.head);
#pragma unroll
    for (int u = 0; u < kBwdU; ++u)
      if (v0 + u * G < so.nvec) dv[v0 + u * G] = make_uint4(0u, 0u, 0u, 0u);
    if (chunk == 0 && tid < kEdges && so.edge(tid) >= 0) put(dx + so.edge(tid), 0.f);
    return;
  }
  const float2 st = a.stats[r];
  const bool far = far_max(st.x, a.c);
  const ExpScale ks(far ? 0.f : st.x, a.c);
  const float kq = -k * st.y;
  const uint64_t kq2 = f2_splat(kq * ks.fix);
  const bool same = same_phase<T>(x, dx);
  uint4* dv = reinterpret_cast<uint4*>(dx + sp.head);
  // the target's value, by the thread that has just written what the others hold there
  const int tv = ok ? static_cast<int>(target) - sp.head : -1;  // its place behind the head
  const float xt = ok ? to_f(x[target]) : 0.f;
  const auto scaled = [&](uint4 x16) {
    uint64_t e[E / 2];
    if (far) shift_vec<T>(x16, st.x);
    exp_vec<T>(x16, ks, e);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) e[i] = f2_mul(e[i], kq2);
    return Vec<T>::pack(e);
  };
  const auto put_target = [&](int v) {
    if (tv >= 0 && tv / E == v) put(dx + target, k + ex2((xt - st.x) * a.c) * kq);
  };
  if (same) {
#pragma unroll
    for (int u = 0; u < kBwdU; ++u) {
      const int v = v0 + u * G;
      if (v >= sp.nvec) continue;
      __stcs(dv + v, scaled(w[u]));
      put_target(v);
    }
  } else {
#pragma unroll
    for (int u = 0; u < kBwdU; ++u) {
      const int v = v0 + u * G;
      if (v - tid >= sp.nvec) continue;  // for all of the group
      store_apart<T>(reinterpret_cast<T*>(dv + v), scaled(w[u]), v < sp.nvec);
      if (v < sp.nvec) put_target(v);
    }
  }
  if (chunk == 0 && tid < kEdges && sp.edge(tid) >= 0) {
    const int i = sp.edge(tid);
    put(dx + i, ex2((to_f(x[i]) - st.x) * a.c) * kq + (i == target ? k : 0.f));
  }
}

// ---- host side ----------------------------------------------------------------

int bad(const char* what) { return set_error(LEMA_ERR_INVALID_ARGUMENT, what); }

// Whether p lies on a multiple of n bytes (null does).
bool on(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Every per-token array of 8-byte and of 4-byte values on its own type's boundary.
int check_aligned(std::initializer_list<const void*> p8, std::initializer_list<const void*> p4) {
  bool ok = true;
  for (const void* p : p8) ok &= on(p, 8);
  for (const void* p : p4) ok &= on(p, 4);
  return ok ? LEMA_OK : set_error(LEMA_ERR_MISALIGNED, "a pointer lies off its type's boundary");
}

// Whether n rows `ld` elements apart stay inside 64-bit offsets.
bool span_ok(int64_t n, int64_t ld) {
  return ld >= 0 && ld <= (int64_t{1} << 60) / std::max<int64_t>(n, 1);
}

// Sizes, strides and temperature shared by every entry point; fills the common fields.
int make_rows(RowArgs& a, const void* x, int x_f32, int64_t n0, int64_t n1, int64_t ld0,
              int64_t ld1, int64_t V, double temperature) {
  a = RowArgs{};
  if (n0 < 0 || n1 < 0) return bad("negative row count");
  if (V <= 0 || V > (1 << 30)) return bad("vocabulary size must be in [1, 2^30]");
  if (!(temperature >= 1e-6 && temperature <= 1e6))
    return bad("temperature must be in [1e-6, 1e6]");
  if (n0 > 0 && n1 > INT32_MAX / n0)
    return set_error(LEMA_ERR_UNSUPPORTED, "more than 2^31 - 1 rows");
  if (n0 * n1 > 0 && x == nullptr) return bad("null logits");
  if (!on(x, x_f32 ? 4 : 2))
    return set_error(LEMA_ERR_MISALIGNED, "logits lie off their type's boundary");
  if (!span_ok(n0, ld0) || !span_ok(n1, ld1)) return bad("row stride negative or past 64 bits");
  a.x = x;
  a.in = RowMap{std::max<int64_t>(n1, 1), ld0, ld1};
  a.out = a.in;
  a.n0 = n0;
  a.T = n0 * n1;
  a.V = static_cast<int32_t>(V);
  a.inv_tau = 1.0 / temperature;
  const double c = 1.4426950408889634 / temperature;
  a.c_full = c;
  a.c = static_cast<float>(c);
  a.c_lo = static_cast<float>(c - static_cast<double>(a.c));
  a.grad_scale = 1.f;
  return LEMA_OK;
}

int set_out(RowArgs& a, void* dx, int x_f32, int64_t ldd0, int64_t ldd1) {
  if (dx == nullptr) return LEMA_OK;
  if (!on(dx, x_f32 ? 4 : 2))
    return set_error(LEMA_ERR_MISALIGNED, "gradient rows lie off their type's boundary");
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

constexpr int64_t kMaxRing = 512;  // CTAs of ring_kernel, at most

// Partial sums: one for each CTA of token_kernel or ring_kernel, or for each pair.
int64_t parts(int64_t n0, int64_t T) { return std::max<int64_t>({token_ctas(T), n0, kMaxRing}); }

int64_t ws_bytes_for(int64_t n0, int64_t T) {
  return kWsHead + round256(n0 * 4) + round256(T * 4) + round256(parts(n0, T) * 16) +
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
  a.list = reinterpret_cast<int32_t*>(p);
  p += round256(a.T * 4);
  a.part = reinterpret_cast<double2*>(p);
  p += round256(parts(a.n0, a.T) * 16);
  a.row = reinterpret_cast<RowStat*>(p);
  a.lp64 = reinterpret_cast<double*>(p);
  return LEMA_OK;
}

// Whole vectors that a row holds, at most.
int max_vecs(const RowArgs& a, int x_f32) { return a.V / (x_f32 ? 4 : 8); }

// A launch in clusters of cs CTAs. `after`: it may begin while the kernel of this call before it
// on the stream still runs (every kernel launched so waits for that one before it touches
// what it wrote).
template <typename... P, typename... A>
int launch(bool after, void (*kern)(P...), int64_t grid, int threads, int smem, int cs,
           cudaStream_t s, A... args) {
  if (grid > INT32_MAX) return set_error(LEMA_ERR_UNSUPPORTED, "too many rows");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = after ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(cs);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cs > 1 ? 2 : 1;
  LEMA_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, args...));
  return LEMA_OK;
}

// A warp a row while four vectors a lane hold it: 65536 rows of 512 bf16 take 26 us, with 128
// threads a row 64 us; 16384 of 1000 take 14 and 23 us.
bool warp_rows(int nvec) { return nvec <= 128; }

template <typename T, int G, bool WHOLE, int U>
int launch_logprobs_g(const RowArgs& a, cudaStream_t s) {
  constexpr int64_t kRows = stat_threads(G) / G;
  logprobs_kernel<T, G, WHOLE, U>
      <<<static_cast<unsigned>((a.T + kRows - 1) / kRows), stat_threads(G), 0, s>>>(a);
  LEMA_CUDA_TRY(cudaGetLastError());
  return LEMA_OK;
}

// As many vectors in flight as a thread has, 8 at most: with 8 for all, 65536 rows of 512 bf16
// took 47 us instead of 26 and 16384 of 4096 took 44 instead of 31, most of their exponentials
// those of absent vectors. Few long rows get more threads: 100 rows of 128256 bf16 take 19.6 us
// with 128, 13.4 with 256 and 11.2 with 512 threads, 450 take 30, 27 and 28; 1500 of 32000 take
// 22, 22 and 28, 6250 of them 9 percent more with 256 than with 128.
template <typename T, bool WHOLE>
int launch_logprobs_t(const RowArgs& a, int nvec, cudaStream_t s) {
  if (nvec <= 32 * 2) return launch_logprobs_g<T, 32, WHOLE, 2>(a, s);
  if (warp_rows(nvec)) return launch_logprobs_g<T, 32, WHOLE, 4>(a, s);
  if (nvec <= 128 * 4) return launch_logprobs_g<T, 128, WHOLE, 4>(a, s);
  if (nvec > 2 * 128 * 8) {  // two sweeps of 128 threads
    if (a.T <= device_sm_count()) return launch_logprobs_g<T, 512, WHOLE, 8>(a, s);
    if (a.T <= 4 * device_sm_count()) return launch_logprobs_g<T, 256, WHOLE, 8>(a, s);
  }
  return launch_logprobs_g<T, 128, WHOLE, 8>(a, s);
}

template <bool WHOLE>
int launch_logprobs(const RowArgs& a, int x_f32, cudaStream_t s) {
  const int nvec = max_vecs(a, x_f32);
  return x_f32 ? launch_logprobs_t<float, WHOLE>(a, nvec, s)
               : launch_logprobs_t<__nv_bfloat16, WHOLE>(a, nvec, s);
}

template <typename T>
int launch_logprobs_bwd_t(const RowArgs& a, int nvec, bool after, cudaStream_t s) {
  // A CTA a chunk, or a warp where more than a fifth of the CTAs' threads would have no vector: the
  // preference loss over 15000 rows of 4296 bf16 takes 106 and 104 us, over 10000 of 9000 117 and
  // 112, over 4096 of 32000 (no such waste) 116 and 125.
  const auto chunks_of = [&](int g) { return std::max(1, (nvec + g * kBwdU - 1) / (g * kBwdU)); };
  const bool waste = chunks_of(kBwdThreads) * (kBwdThreads * kBwdU) > nvec + nvec / 4;
  const int g = waste ? 32 : kBwdThreads, chunks = chunks_of(g);
  const int64_t per = kBwdThreads / g, grid = (a.T * chunks + per - 1) / per;
  if (grid > INT32_MAX) return set_error(LEMA_ERR_UNSUPPORTED, "too many rows");
  const auto kern = g == 32 ? logprobs_bwd_kernel<T, 32> : logprobs_bwd_kernel<T, kBwdThreads>;
  return launch(after, kern, grid, kBwdThreads, 0, 1, s, a, chunks);
}

// `after`: directly behind pair_kernel of the same call, which it may overlap.
int launch_logprobs_bwd(const RowArgs& a, int x_f32, bool after, cudaStream_t s) {
  const int nvec = max_vecs(a, x_f32);
  return x_f32 ? launch_logprobs_bwd_t<float>(a, nvec, after, s)
               : launch_logprobs_bwd_t<__nv_bfloat16>(a, nvec, after, s);
}

template <int WARPS>
int ring_smem(int stages, int K4) {
  return kZeroBytes + stages * Ring<WARPS>::kChunk * 16 + (stages + 1) * K4 * 12;
}

template <typename Kern>
int allow_smem(Kern kern, int bytes, std::atomic<uint64_t>& done) {
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return set_error(LEMA_ERR_CUDA, "bad device");
  if (!(done.load() >> dev & 1)) {
    LEMA_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done |= uint64_t{1} << dev;
  }
  return LEMA_OK;
}

// Clusters of cs CTAs that are resident at once.
template <int WARPS, typename Kern>
int resident_clusters(Kern kern, int cs, int smem, int* out) {
  static std::atomic<int> cache[64][kMaxCluster + 1];  // Ring::kCtas an SM whatever the kernel
  const int dev = current_device();
  int n = cache[dev][cs].load();
  if (n == 0) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(cs));
    cfg.blockDim = dim3((WARPS + 1) * 32);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(cs);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    LEMA_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
    if (n < 1) return set_error(LEMA_ERR_CUDA, "no cluster fits this device");
    cache[dev][cs].store(n);
  }
  *out = n;
  return LEMA_OK;
}

int launch_count(const RowArgs& a, cudaStream_t s) {
  // a CTA that holds them all starts sooner, by 1.3 us at 4096 rows
  const int ctas = a.T > kCountBlock ? kCountCluster : 1;
  const int64_t warps = (a.T + 32 * ctas - 1) / (32 * ctas);  // of rows, for each CTA
  return launch(false, count_kernel, ctas, kCountThreads, 0, ctas, s, a,
                static_cast<int32_t>(warps * 32));
}

template <typename T, int OBJ, int WARPS, bool SHORT>
int launch_ring(RowArgs a, int cs, int per, int stages, cudaStream_t s) {
  auto kern = ring_kernel<T, OBJ, WARPS, SHORT>;
  static std::atomic<uint64_t> done{0};
  int rc = allow_smem(kern, Ring<WARPS>::kSmem, done);
  if (rc) return rc;
  const int smem = ring_smem<WARPS>(stages, a.K4);
  int clusters = std::min<int>(Ring<WARPS>::kCtas * device_sm_count(), kMaxRing);
  if (cs > 1 && (rc = resident_clusters<WARPS>(kern, cs, smem, &clusters))) return rc;
  const int64_t n = std::min<int64_t>(a.T, std::min<int64_t>(clusters, kMaxRing / cs)) * cs;
  a.self_count = a.T <= kOwnTotal && a.T <= kOwnRows * (n / cs) &&
                 (!a.per_sequence || a.n0 <= kOwnSeqs);
  if (!a.self_count && (rc = launch_count(a, s))) return rc;
  rc = launch(!a.self_count, kern, n, (WARPS + 1) * 32, smem, cs, s, a, cs, per, stages);
  return rc ? rc : launch(true, finish_kernel, 1, 256, 0, 1, s, a, static_cast<int>(n));
}

// Seven warps: 9 stages without a teacher, 8 with 64 entries, 3 with 1024. Only where those are
// fewer than a row may have chunks are they freed one by one, which costs a few instructions a
// chunk: 8 x 512 rows of 32000 with 64 entries take 96.0 us without and 97.3 us with them.
template <typename T, int OBJ, int WARPS>
int launch_ring(const RowArgs& a, int cs, int nvec, cudaStream_t s) {
  // few rows: spread each while SMs would be idle and every thread still has a vector
  while (cs * 2 <= kMaxCluster && a.T * cs * 2 <= device_sm_count() &&
         nvec >= cs * 2 * Ring<WARPS>::kThreads)
    cs *= 2;
  const int per = (nvec + cs - 1) / cs;
  int stages = kMaxStages;
  while (ring_smem<WARPS>(stages, a.K4) > Ring<WARPS>::kSmem) --stages;
  return OBJ == kDistill && stages < kRingVecs / kChunkVecs
             ? launch_ring<T, OBJ, WARPS, OBJ == kDistill>(a, cs, per, stages, s)
             : launch_ring<T, OBJ, WARPS, false>(a, cs, per, stages, s);
}

template <typename T, int OBJ, int G, int NV>
int launch_direct(const RowArgs& a, int64_t grid, int smem, cudaStream_t s) {
  auto kern = direct_kernel<T, OBJ, G, NV>;
  static std::atomic<uint64_t> done{0};
  if (OBJ == kDistill) {  // four warps with 1024 entries each take more than the default 48 KB
    const int rc = allow_smem(kern, kDirectThreads / G * kMaxTeacher * 12, done);
    if (rc) return rc;
  }
  return launch(!a.self_count, kern, grid, kDirectThreads, smem, 1, s, a);
}

// How a row is held, by the vectors it spans. kNv vectors are the 64 elements that a thread
// keeps as fp32. A warp a row while it holds it: policy over 65536 rows of 512 bf16 takes 47 us,
// with 128 threads a row 124 us; over 16384 of 2000 it takes 38 and 48 us. Sets self_count for
// token_kernel, or *done where it is not needed.
template <typename T, int OBJ>
int launch_rows(RowArgs& a, int nvec, bool* done, cudaStream_t s) {
  constexpr int kNv = 64 / Vec<T>::kE;
  const int teacher = a.K4 * 12;
  if (nvec <= 128 * kNv) {
    a.self_count = a.T <= kSelfRows;
    if (!a.self_count) {
      const int rc = launch_count(a, s);
      if (rc) return rc;
    }
    const bool warps = nvec <= 32 * kNv;
    const int64_t per = warps ? kDirectThreads / 32 : 1, grid = (a.T + per - 1) / per;
    const int smem = static_cast<int>(per) * teacher;
    if (nvec <= 8 * kNv) return launch_direct<T, OBJ, 32, kNv / 4>(a, grid, smem, s);
    if (nvec <= 16 * kNv) return launch_direct<T, OBJ, 32, kNv / 2>(a, grid, smem, s);
    if (warps) return launch_direct<T, OBJ, 32, kNv>(a, grid, smem, s);
    if (nvec <= 64 * kNv) return launch_direct<T, OBJ, 128, kNv / 2>(a, grid, smem, s);
    return launch_direct<T, OBJ, 128, kNv>(a, grid, smem, s);
  }
  // What an SM's CTAs hold at once is what keeps DRAM busy while each waits for its reductions: the
  // fewest CTAs a row, of seven warps (two an SM) or of four (three an SM), whichever hold
  // more. Of bf16 policy rows, a quarter not counted, 16000 elements reach 4.0 TB/s with
  // seven warps and 4.6 with four, 32000 4.9 and 4.6, 32264 (two CTAs) 3.5 and 4.6, 50257 4.4
  // (two CTAs) and 4.0 (four).
  const int cs7 = (nvec + Ring<7>::kCap - 1) / Ring<7>::kCap,
            cs4 = (nvec + Ring<4>::kCap - 1) / Ring<4>::kCap;
  if (cs7 > kMaxCluster) {
    const int rc = launch_count(a, s);
    return rc ? rc
              : launch(true, stream_kernel<T, OBJ>,
                       std::min<int64_t>(a.T, device_sm_count()), kRowThreads, teacher, 1, s,
                       a);
  }
  *done = true;
  return cs4 > kMaxCluster || Ring<7>::kCtas * cs4 >= Ring<4>::kCtas * cs7
             ? launch_ring<T, OBJ, 7>(a, cs7, nvec, s)
             : launch_ring<T, OBJ, 4>(a, cs4, nvec, s);
}

// The list of rows, their statistics and gradients, the tokens' terms.
template <int OBJ>
int launch_loss(RowArgs a, int x_f32, cudaStream_t s) {
  bool done = false;  // the tokens' terms are on their way
  a.self_count = 1;
  if (a.T > 0) {
    const int nvec = max_vecs(a, x_f32);
    a.self_count = 0;
    const int rc = x_f32 ? launch_rows<float, OBJ>(a, nvec, &done, s)
                         : launch_rows<__nv_bfloat16, OBJ>(a, nvec, &done, s);
    if (rc) return rc;
  }
  if (done) return LEMA_OK;
  const int64_t ctas = a.self_count ? 1 : token_ctas(a.T);
  return launch(a.T > 0, token_kernel<OBJ>, ctas, kTokenThreads, 0, 1, s, a);
}

// Statistics are read and written as pairs.
int set_stats(RowArgs& a, const float* stats) {
  if (!on(stats, 8)) return bad("stats: 8-byte alignment");
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  return LEMA_OK;
}

int need_err(RowArgs& a) {
  static std::atomic<int32_t*> word[64];  // one a device
  const int dev = current_device();
  if (dev < 0 || dev >= 64) return set_error(LEMA_ERR_CUDA, "bad device");
  a.err = word[dev].load();
  if (a.err == nullptr) word[dev].store(a.err = gemm_error_word());
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
  int rc = make_rows(a, x, x_f32, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (a.T == 0) return LEMA_OK;
  if (!targets || !logps) return bad("null targets or logps");
  if ((rc = check_aligned({targets}, {logps}))) return rc;
  if ((rc = need_err(a))) return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  a.logps = logps;
  if ((rc = set_stats(a, stats))) return rc;
  return launch_logprobs<false>(a, x_f32, static_cast<cudaStream_t>(stream));
}

extern "C" int lema_token_logprobs_bwd(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                       int64_t ld0, int64_t ld1, int64_t V,
                                       const int64_t* targets, int64_t ignore_index,
                                       double temperature, const float* stats,
                                       const float* dlogps, const float* upstream, void* dx,
                                       int64_t ldd0, int64_t ldd1, void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, x_f32, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (a.T == 0) return LEMA_OK;
  if (!targets || !stats || !dlogps || !dx) return bad("null pointer");
  if ((rc = check_aligned({targets}, {dlogps, upstream}))) return rc;
  if ((rc = set_out(a, dx, x_f32, ldd0, ldd1))) return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  if ((rc = set_stats(a, stats))) return rc;
  a.g = dlogps;
  a.upstream = upstream;
  return launch_logprobs_bwd(a, x_f32, false, static_cast<cudaStream_t>(stream));
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
  int rc = make_rows(a, x, x_f32, n0, n1, ld0, ld1, V, 1.0);
  if (rc) return rc;
  if (n0 == 0 || n0 % 2 != 0) return bad("preference_loss needs chosen and rejected sequences");
  if (!(beta > 0.0) || !std::isfinite(beta)) return bad("beta must be positive");
  if (!(label_smoothing >= 0.0 && label_smoothing < 0.5))
    return bad("label_smoothing must be in [0, 0.5)");
  if (!loss || !rewards || (a.T > 0 && (!targets || !logps || !stats || !coef)))
    return bad("null pointer");
  if ((rc = check_aligned({targets}, {ref_logps, logps, coef, loss, rewards}))) return rc;
  if ((rc = set_ws(a, ws, ws_bytes)) || (rc = set_out(a, dx, x_f32, ldd0, ldd1)) ||
      (rc = need_err(a)))
    return rc;
  a.targets = targets;
  a.ignore = ignore_index;
  a.ref_logps = ref_logps;
  a.logps = logps;
  if ((rc = set_stats(a, stats))) return rc;
  a.coef = coef;
  auto s = static_cast<cudaStream_t>(stream);
  a.loss = loss;
  if (a.T > 0) {
    if ((rc = launch_logprobs<true>(a, x_f32, s))) return rc;
  } else {
    LEMA_CUDA_TRY(cudaMemsetAsync(a.head, 0, sizeof(WsHead), s));
  }
  if ((rc = launch(true, pair_kernel, n0 / 2, kPairThreads, 0, 1, s, a, n0 / 2, beta,
                   label_smoothing, rewards)))
    return rc;
  if (dx == nullptr || a.T == 0) return LEMA_OK;
  a.g = coef;
  a.zeros_done = 1;
  a.grad_scale = static_cast<float>(grad_scale);
  return launch_logprobs_bwd(a, x_f32, true, s);
}

extern "C" int lema_policy_loss(const void* x, int32_t x_f32, int64_t n0, int64_t n1, int64_t ld0,
                                int64_t ld1, int64_t V, const int64_t* targets,
                                int64_t ignore_index, double temperature, const float* old_logps,
                                const float* advantages, int64_t adv_s0, int64_t adv_s1,
                                const float* ref_logps, double clip_lo, double clip_hi,
                                double kl_coef, int32_t per_sequence, double grad_scale, void* ws,
                                int64_t ws_bytes, float* logps, float* stats, float* coef,
                                float* loss, float* kl, void* dx, int64_t ldd0, int64_t ldd1,
                                void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, x_f32, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (!(clip_lo >= 0.0 && clip_lo <= 1.0) || !(clip_hi >= 0.0) || !std::isfinite(clip_hi))
    return bad("clip must be in [0, 1] below and finite, >= 0 above");
  if (!(kl_coef >= 0.0) || !std::isfinite(kl_coef)) return bad("kl_coef must be >= 0");
  if (!loss || !kl || (a.T > 0 && (!targets || !advantages || !logps))) return bad("null pointer");
  if ((rc = check_aligned({targets}, {old_logps, advantages, ref_logps, logps, coef, loss, kl})))
    return rc;
  if ((rc = set_ws(a, ws, ws_bytes)) || (rc = set_out(a, dx, x_f32, ldd0, ldd1)) ||
      (rc = need_err(a)))
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
  a.log_lo = std::log(1.0 - clip_lo);
  a.log_hi = std::log(1.0 + clip_hi);
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

extern "C" int lema_distill_loss(const void* x, int32_t x_f32, int64_t n0, int64_t n1,
                                 int64_t ld0, int64_t ld1, int64_t V, const void* teacher_ids,
                                 int32_t ids_i32, const void* teacher_logits, int32_t tl_f32,
                                 int64_t K, const uint8_t* mask, double temperature,
                                 double grad_scale, const float* upstream, void* ws,
                                 int64_t ws_bytes, float* loss, void* dx, int64_t ldd0,
                                 int64_t ldd1, void* stream) {
  clear_error();
  RowArgs a;
  int rc = make_rows(a, x, x_f32, n0, n1, ld0, ld1, V, temperature);
  if (rc) return rc;
  if (!loss) return bad("null loss");
  if (K < 1 || K > kMaxTeacher)
    return set_error(LEMA_ERR_UNSUPPORTED, "between 1 and 1024 teacher entries a row");
  if (a.T > 0 && (!teacher_ids || !teacher_logits)) return bad("null teacher indices or logits");
  if ((rc = check_aligned({}, {loss, upstream}))) return rc;
  if (!on(teacher_ids, ids_i32 ? 4 : 8) || !on(teacher_logits, tl_f32 ? 4 : 2))
    return set_error(LEMA_ERR_MISALIGNED, "teacher entries lie off their type's boundary");
  if ((rc = set_ws(a, ws, ws_bytes)) || (rc = set_out(a, dx, x_f32, ldd0, ldd1)) ||
      (rc = need_err(a)))
    return rc;
  a.teacher_ids = teacher_ids;
  a.ids_i32 = ids_i32;
  a.teacher_logits = teacher_logits;
  a.tl_f32 = tl_f32;
  a.K = static_cast<int32_t>(K);
  a.K4 = (a.K + 3) / 4 * 4;
  a.mask = mask;
  a.grad_scale = static_cast<float>(grad_scale);
  a.upstream = upstream;
  a.loss = loss;
  return launch_loss<kDistill>(a, x_f32, static_cast<cudaStream_t>(stream));
}
