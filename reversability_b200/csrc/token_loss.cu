// Losses on token log-probabilities: the log-probabilities and entropies
// themselves, the clipped policy loss with a KL term, and the paired preference
// loss, each with the gradient of the logits.
//
// Everything is carried in base 2: with c = inv_temp log2(e) and a reference
// value r of the row (an element within 2^8 of its maximum, so nothing
// overflows), e_j = 2^(x_j c - r c), S = sum e_j, W = sum e_j log2 e_j:
//   ln p_j = ln2 (x_j c - r c) - ln S,  entropy = ln S - ln2 W / S
//   dx_j   = g_lp [j = label] + e_j (A + B (x_j c - r c)),
//            A = (-g_lp - g_h (entropy - ln S)) / S, B = -g_h ln2 / S
// x c - r c is one fused multiply-add with one rounding, whatever the size of
// r; keeping r and S apart (not r + log S) keeps p exact when logits are large.
// r is stored raw: where |r c| would overflow (a row with nothing but masks of
// the type's lowest value) the exponent is formed as (x - r) c instead. Sums
// are fp32: a thread adds up partial sums of 16 (fp32) or 32 terms, 13 of them
// at 50257 columns of 16 bits and 32 at 131072 (18 where a warp has the row),
// and those of threads are joined in a fixed order; the gradient is rounded
// once, when it is stored.
#include <type_traits>
#include "vec.cuh"

namespace rk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kHuge = 1e7f;       // |r c| from here on: the exponent as (x - r) c, as r c itself is rounded by more than 1
constexpr float kFloor = -1e30f;    // the reference of a sum that has seen nothing finite
constexpr float kLazy = 8.f;        // a thread's reference follows its maximum once that is 2^8 above
constexpr float kTiny = -200.f;     // 2^-200 is 0 in fp32: exponents are clamped here where they are also a factor

// The label, -1 of a row without one, -2 if it is out of range.
__device__ __forceinline__ int checked_label(int64_t label, int vocab, int ignore_index) {
  return label == ignore_index ? -1 : label < 0 || label >= vocab ? -2 : (int)label;
}

// ---------------------------------------------------------------- 16-byte vectors
template <typename T>
constexpr int kPer = 16 / (int)sizeof(T);

// Pairs of floats in the packed fp32x2 arithmetic of sm_100 (one issue slot for two elements).
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Exponents that are also a factor (entropy) are kept finite; a NaN stays one.
__device__ __forceinline__ uint64_t clamp_pair(uint64_t t) {
  float t0, t1;
  unpair(t, t0, t1);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(t0) : "f"(kTiny));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(t1) : "f"(kTiny));
  return pair(t0, t1);
}
__device__ __forceinline__ uint64_t exp2_pair(uint64_t t) {
  float t0, t1;
  unpair(t, t0, t1);
  return pair(ex2_approx(t0), ex2_approx(t1));
}

template <typename T>
__device__ __forceinline__ void unpack(const uint4& v, uint64_t (&p)[kPer<T> / 2]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (sizeof(T) == 4) {
    p[0] = pair(__uint_as_float(w[0]), __uint_as_float(w[1]));
    p[1] = pair(__uint_as_float(w[2]), __uint_as_float(w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        p[i] = pair(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        p[i] = pair(f.x, f.y);
      }
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack(const uint64_t (&p)[kPer<T> / 2]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
    float f[4];
    unpair(p[0], f[0], f[1]);
    unpair(p[1], f[2], f[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a, b;
      unpair(p[i], a, b);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(a, b);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Largest element of U vectors (NaNs do not count: they reach the sum through the exponential).
template <typename T, int U>
__device__ __forceinline__ float vec_max(const uint4 (&v)[U]) {
  if constexpr (sizeof(T) == 4) {
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[u].x), __uint_as_float(v[u].y)),
                         fmaxf(__uint_as_float(v[u].z), __uint_as_float(v[u].w))));
    return m;
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2 m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const T2* e = reinterpret_cast<const T2*>(&v[u]);
      const T2 n = __hmax2(__hmax2(e[0], e[1]), __hmax2(e[2], e[3]));
      m = u ? __hmax2(m, n) : n;
    }
    return fmaxf(Dt<T>::to_f(m.x), Dt<T>::to_f(m.y));
  }
}

// A row as head elements, 16-byte vectors and tail elements.
template <typename T>
struct RowSpan {
  int head, nvec, tail;
  __device__ __forceinline__ RowSpan(const T* x, int vocab) {
    const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15);
    head = min(off ? (16 - off) / (int)sizeof(T) : 0, vocab);
    nvec = (vocab - head) / kPer<T>;
    tail = vocab - head - nvec * kPer<T>;
  }
};

// ---------------------------------------------------------------- row sums
struct alignas(16) RowSum {
  float r, m, s, w;  // raw reference, r c, sum 2^(x c - m), sum 2^(..) (x c - m)
};
__device__ __forceinline__ RowSum empty_sum() { return {-INFINITY, kFloor, 0.f, 0.f}; }

// Moves a sum to the reference (r, m), m >= a.m.
template <bool ENT>
__device__ __forceinline__ void rebase(RowSum& a, float r, float m) {
  const float d = a.m - m, f = ex2_approx(d);
  if constexpr (ENT) a.w = f > 0.f ? fmaf(d, a.s, a.w) * f : 0.f;
  a.s *= f;
  a.r = r;
  a.m = m;
}

// Adds U vectors at once: one look at their maximum, then U * kPer independent exponentials.
template <typename T, bool ENT, int U>
__device__ __forceinline__ void add_vectors(RowSum& a, const uint4 (&v)[U], float c) {
  const float top = vec_max<T, U>(v);
  if (top * c > a.m + kLazy) rebase<ENT>(a, top, top * c);
  const uint64_t c2 = pair(c, c), m2 = pair(-a.m, -a.m);
  uint64_t s2[2] = {0, 0}, w2[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint64_t p[kPer<T> / 2];
    unpack<T>(v[u], p);
#pragma unroll
    for (int i = 0; i < kPer<T> / 2; ++i) {
      uint64_t t = fma2(p[i], c2, m2);
      if constexpr (ENT) t = clamp_pair(t);
      const uint64_t e = exp2_pair(t);
      s2[i & 1] = add2(s2[i & 1], e);
      if constexpr (ENT) w2[i & 1] = fma2(e, t, w2[i & 1]);
    }
  }
  float s0, s1;
  unpair(add2(s2[0], s2[1]), s0, s1);
  a.s += s0 + s1;
  if constexpr (ENT) {
    unpair(add2(w2[0], w2[1]), s0, s1);
    a.w += s0 + s1;
  }
}
template <bool ENT>
__device__ __forceinline__ void add_element(RowSum& a, float x, float c) {
  if (x * c > a.m + kLazy) rebase<ENT>(a, x, x * c);
  float t = fmaf(x, c, -a.m);
  if (ENT && t < kTiny) t = kTiny;
  const float e = ex2_approx(t);
  a.s += e;
  if constexpr (ENT) a.w = fmaf(e, t, a.w);
}
// Joins the sums of the first N lanes (a power of two; the others hold empty ones) in a fixed order.
template <bool ENT, int N = 32>
__device__ __forceinline__ RowSum warp_join(RowSum a, float c) {
  // r as an integer of the same order, so that one instruction finds the largest
  const int b = __float_as_int(a.r), top = __reduce_max_sync(0xffffffffu, b ^ ((b >> 31) & 0x7fffffff));
  const float r = __int_as_float(top ^ ((top >> 31) & 0x7fffffff));
  rebase<ENT>(a, r, fmaxf(r * c, kFloor));
#pragma unroll
  for (int o = N / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if constexpr (ENT) a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
  if constexpr (N < 32) {  // every lane returns the same sums: what follows branches on them as a warp
    a.s = __shfl_sync(0xffffffffu, a.s, 0);
    if constexpr (ENT) a.w = __shfl_sync(0xffffffffu, a.w, 0);
  }
  return a;
}

// One warp's sums of a whole row in the (x - r) c form, r its largest element: for rows whose reference overflows. In fp64,
// as a lane has up to V / 32 terms one behind the other (in fp32 1.8e-5 off at 300007 columns).
template <typename T>
__device__ __noinline__ RowSum warp_row_sum_far(const T* x, int vocab, float c) {
  const int lane = threadIdx.x & 31;
  RowSum a = {-INFINITY, 0.f, 0.f, 0.f};
  for (int j = lane; j < vocab; j += 32) a.r = fmaxf(a.r, Dt<T>::to_f(x[j]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a.r = fmaxf(a.r, __shfl_xor_sync(0xffffffffu, a.r, o));
  a.m = a.r * c;
  double s = 0.0, w = 0.0;
  for (int j = lane; j < vocab; j += 32) {
    const float t = (Dt<T>::to_f(x[j]) - a.r) * c;
    const float e = ex2_approx(t);
    s += (double)e;
    w += (double)(e > 0.f ? e * t : e);  // e is 0 or NaN here
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    w += __shfl_xor_sync(0xffffffffu, w, o);
  }
  a.s = (float)s;
  a.w = (float)w;
  return a;
}
// Whether a finished row sum has to be formed again in that way (nothing finite seen, or r c out of range).
__device__ __forceinline__ bool is_far(const RowSum& a) { return a.s == 0.f || !(fabsf(a.m) < kHuge); }
__device__ __forceinline__ float exponent(float x, float c, const RowSum& a, bool far) {
  return far ? (x - a.r) * c : fmaf(x, c, -a.m);
}
// The label's log-probability before it is rounded to fp32 (whose steps are 1e-6 at -10): losses are sums of many, in
// which these roundings would show. With the sum's own c and m, so that their rounding cancels. The exponential unit's
// results are 5e-8 low on average (5.0e-8 over [-16, -1], 2.2e-8 over [-1, 0], at most 1.4e-7), and a sum meets it again
// where sums are joined: 8e-8 in all, but for the reference's own term, which is exact. Mean errors left over rows of 1000
// to 50257 normal logits: -4e-8 to 7e-8 at spreads of 0.01 to 2, where they were 4e-8 to 1.5e-7; wider ones are 1.3e-8 of the
// label's distance from the row's mean under p further off, by the rounding of c. Rows of equal logits, whose exponentials
// are exact, become up to 1e-7 too low.
constexpr double kUnitLow = 8e-8;
__device__ __forceinline__ double label_logprob(float x, float c, const RowSum& a, bool far) {
  const double t = far ? ((double)x - (double)a.r) * (double)c : fma((double)x, (double)c, -(double)a.m);
  return t * 0.6931471805599453 - (log((double)a.s) + kUnitLow * (1.0 - (double)__fdividef(1.f, a.s)));
}

// ---------------------------------------------------------------- row gradients
struct RowGrad {
  float a, b, g;  // dx = e (a + b t), + g at the label; t = x c - m
};
__device__ __forceinline__ RowGrad row_grad(float s, float ln_s, float entropy, float g_lp, float g_h) {
  const float inv = 1.f / s;
  return {(-g_lp - g_h * (entropy - ln_s)) * inv, -g_h * kLn2 * inv, g_lp};
}
template <bool ENT>
__device__ __forceinline__ float grad_element(float t, const RowGrad& k) {
  if constexpr (ENT) {
    t = t < kTiny ? kTiny : t;  // keeps a NaN
    return ex2_approx(t) * fmaf(k.b, t, k.a);
  }
  return ex2_approx(t) * k.a;
}
// A vector's gradients, without the label's own term.
template <typename T, bool ENT>
__device__ __forceinline__ uint4 grad_vector(const uint4& v, float c, const RowSum& a, const RowGrad& k) {
  uint64_t p[kPer<T> / 2];
  unpack<T>(v, p);
  const uint64_t c2 = pair(c, c), m2 = pair(-a.m, -a.m), ka = pair(k.a, k.a), kb = pair(k.b, k.b);
#pragma unroll
  for (int i = 0; i < kPer<T> / 2; ++i) {
    uint64_t t = fma2(p[i], c2, m2);
    if constexpr (ENT) t = clamp_pair(t);
    p[i] = mul2(exp2_pair(t), ENT ? fma2(kb, t, ka) : ka);
  }
  return pack<T>(p);
}
// The same, element by element, for the vectors that hold the label and for rows whose reference overflows; `at` is
// the column of the first element.
template <typename T, bool ENT>
__device__ __noinline__ uint4 grad_vector_any(uint4 v, float c, RowSum a, bool far, RowGrad k, int at, int label) {
  T* e = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int i = 0; i < kPer<T>; ++i)
    e[i] = Dt<T>::from_f(grad_element<ENT>(exponent(Dt<T>::to_f(e[i]), c, a, far), k) + (at + i == label ? k.g : 0.f));
  return v;
}
// Stores a vector at `p`, which has the phase of 16 bytes only if `vec`.
template <typename T>
__device__ __forceinline__ void store_vector(T* p, const uint4& v, bool vec) {
  if (vec) {
    __stcs(reinterpret_cast<uint4*>(p), v);
  } else {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < kPer<T>; ++i) p[i] = e[i];
  }
}

// ---------------------------------------------------------------- what a row gives
struct RowOut {
  const int64_t* labels;
  float* logprob;
  float* entropy;  // NULL without ENT
  float* kl;       // policy only, may be NULL
  float2* stats;   // (r, S), may be NULL
  float2* coef;    // policy only, may be NULL
  float2* parts;   // policy only: (w l, w clipped) of a row, for finish_losses
  float4* fine;    // policy only: (the label's logit, r, S, d(w l) / dlp), for finish_losses
  double2* sums;   // policy only: these over the rows of a taker (a CTA, or a cluster)
  const double* weights;  // policy only: sums of the weights of labelled rows, n_weights of them
  int n_weights;          // 0: few rows, whose weights each CTA sums by itself, which saves a launch
  float* denom;    // policy only: where the denominator goes
  const int2* list;    // many rows: (row, label) of those with a label, the others behind; else NULL
  unsigned int* status;
};

// The outputs of a row without a label (label -1, or -2 if it is out of range).
template <bool POLICY>
__device__ __forceinline__ void unlabelled_row(const RowOut& o, int64_t row, int label) {
  if (label == -2) flag_error(o.status, RK_DEV_CE_LABEL);
  o.logprob[row] = 0.f;
  if (o.entropy) o.entropy[row] = 0.f;
  if (o.stats) o.stats[row] = {0.f, 1.f};
  if constexpr (POLICY) {
    if (o.kl) o.kl[row] = 0.f;
    if (o.coef) o.coef[row] = {0.f, 0.f};
  }
}

// The rows of one of `step` takers, the `first`-th: every step-th of the list (labelled rows first, so each taker has
// as many of them as any other, whatever the mask), or without a list every step-th row. Reads one ahead.
struct RowDeal {
  const RowOut& o;
  int64_t rows, at, step;
  int vocab, ignore_index;
  int64_t row;
  int label;
  int2 next;
  __device__ __forceinline__ RowDeal(const RowOut& out, int64_t rows, int vocab, int ignore_index, int64_t first, int64_t step)
      : o(out), rows(rows), at(first), step(step), vocab(vocab), ignore_index(ignore_index) {
    if (at < rows) next = fetch(at);
    settle();
  }
  __device__ __forceinline__ int2 fetch(int64_t i) const {
    return o.list ? o.list[i] : make_int2((int)i, checked_label(o.labels[i], vocab, ignore_index));
  }
  __device__ __forceinline__ void settle() {
    if (at >= rows) return;
    row = next.x;
    label = next.y;
    if (at + step < rows) next = fetch(at + step);
  }
  __device__ __forceinline__ bool more() const { return at < rows; }
  __device__ __forceinline__ void advance() {
    at += step;
    settle();
  }
};

// Lists the rows, labelled ones in front, the others behind, both in order, and writes the outputs of the others; a CTA
// for each 1024 rows, which counts those before its own by itself (a few loads a thread, where a second launch or a
// chain of CTAs would take longer). With POLICY each CTA also sums the weights of its labelled rows; without a list it
// does that alone, over every gridDim-th 1024 rows.
template <bool POLICY>
__global__ void __launch_bounds__(1024) list_rows_kernel(int64_t rows, int vocab, int ignore_index, RowOut o,
                                                         const float* __restrict__ row_weights, int2* __restrict__ list,
                                                         double* __restrict__ weights) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ int warp_before[32], warp_here[32];
  __shared__ double warp_weight[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t base = (int64_t)blockIdx.x * 1024, row = base + threadIdx.x;
  double weight = 0.0;
  int before = 0, label = -1;
  unsigned mask = 0;
  if (list) {
#pragma unroll 8
    for (int64_t r = threadIdx.x; r < base; r += 1024) before += checked_label(o.labels[r], vocab, ignore_index) >= 0;
    if (row < rows) label = checked_label(o.labels[row], vocab, ignore_index);
    mask = __ballot_sync(0xffffffffu, label >= 0);
    before = __reduce_add_sync(0xffffffffu, before);
    if (POLICY && label >= 0) weight = row_weights ? (double)row_weights[row] : 1.0;
  } else {
    for (int64_t r = row; r < rows; r += (int64_t)gridDim.x * 1024)
      if (checked_label(o.labels[r], vocab, ignore_index) >= 0) weight += row_weights ? (double)row_weights[r] : 1.0;
  }
  if constexpr (POLICY) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) weight += __shfl_xor_sync(0xffffffffu, weight, d);
  }
  if (lane == 0) {
    warp_before[warp] = before;
    warp_here[warp] = __popc(mask);
    warp_weight[warp] = weight;
  }
  __syncthreads();
  if (list) {
    const int all_before = __reduce_add_sync(0xffffffffu, warp_before[lane] + (lane < warp ? warp_here[lane] : 0));
    if (row < rows) {
      const int64_t at = all_before + __popc(mask & ((1u << lane) - 1));  // labelled rows before this one
      list[label >= 0 ? at : rows - 1 - (row - at)] = make_int2((int)row, label);
      if (label < 0) unlabelled_row<POLICY>(o, row, label);
    }
  }
  if (POLICY && warp == 0) {
    weight = warp_weight[lane];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) weight += __shfl_xor_sync(0xffffffffu, weight, d);
    if (lane == 0) weights[blockIdx.x] = weight;
  }
}

// ---------------------------------------------------------------- policy loss
struct PolicyRow {
  float kl, loss, slope, clipped, g_lp, g_h;  // slope = dloss / dlp; g_* without the outer scale and inv_temp
};
struct PolicyIn {
  float old, adv, ref, w;
};
__device__ __forceinline__ PolicyIn policy_in(const rk_policy_terms& k, int64_t row) {
  return {k.old_logprobs[row], k.advantages[k.adv_group == 1 ? row : row / k.adv_group],
          k.ref_logprobs ? k.ref_logprobs[row] : 0.f, k.weights ? k.weights[row] : 1.f};
}
__device__ __forceinline__ PolicyRow policy_row(const rk_policy_terms& k, const PolicyIn& in, float lp, float entropy,
                                                float inv_d) {
  PolicyRow o;
  const float adv = in.adv, w = in.w;
  const float ratio = expf(lp - in.old);
  const float free = ratio * adv, held = fminf(fmaxf(ratio, 1.f - k.clip_low), 1.f + k.clip_high) * adv;
  const bool clipped = held < free;
  float kl = 0.f, dkl = 0.f;
  if (k.ref_logprobs) {
    const float drift = in.ref - lp;
    const float em1 = expm1f(drift);
    kl = em1 - drift;
    dkl = -em1;
  }
  o.kl = kl;
  o.slope = w * ((clipped ? 0.f : -free) + k.kl_coef * dkl);
  o.loss = w * (k.kl_coef * kl - (clipped ? held : free) - k.entropy_coef * entropy);
  o.clipped = clipped ? w : 0.f;
  o.g_lp = o.slope * inv_d;
  o.g_h = -w * inv_d * k.entropy_coef;
  return o;
}

// What the reported log-probability was rounded by, times the loss's slope there; nothing for infinite terms.
__device__ __forceinline__ float loss_rounding(float x, float c, const RowSum& a, bool far, float lp, float slope) {
  const float more = slope * (float)(label_logprob(x, c, a, far) - (double)lp);
  return fabsf(more) < INFINITY ? more : 0.f;
}
// Adds that to the loss terms of the first-th and every step-th row after it, of this warp, and sums these. Behind the
// warp's last row, a row a lane: within the rows, the logarithm in fp64 kept a whole CTA waiting (564 us in place of 544 at
// 14848 x 50257).
__device__ __forceinline__ void finish_losses(const RowOut& o, int64_t first, int64_t step, int64_t rows, float c,
                                              int vocab, int ignore_index) {
  __syncwarp();
  double loss = 0.0, clipped = 0.0;
  for (int64_t i = first + (threadIdx.x & 31) * step; i < rows; i += 32 * step) {
    const int2 at = o.list ? o.list[i] : make_int2((int)i, checked_label(o.labels[i], vocab, ignore_index));
    if (at.y < 0) continue;
    const float4 f = o.fine[at.x];
    const float2 part = o.parts[at.x];
    const RowSum a = {f.y, f.y * c, f.z, 0.f};
    loss += (double)part.x + (double)loss_rounding(f.x, c, a, is_far(a), o.logprob[at.x], f.w);
    clipped += (double)part.y;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    loss += __shfl_xor_sync(0xffffffffu, loss, d);
    clipped += __shfl_xor_sync(0xffffffffu, clipped, d);
  }
  if ((threadIdx.x & 31) == 0) o.sums[first] = {loss, clipped};
}

// The sums of two values over the CTA, in a fixed order.
__device__ double2 block_sum2(double a, double b) {
  __shared__ double2 red[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = {a, b};
  __syncthreads();
  double2 s = {0.0, 0.0};
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
    s.x += red[w].x;
    s.y += red[w].y;
  }
  return s;
}

// The sum of the weights of the rows that count, over one warp, from sums[0 .. n) or, without them, from all rows.
__device__ __noinline__ float warp_weight(const double* sums, int n, const int64_t* labels, const float* weights,
                                          int64_t rows, int vocab, int ignore_index) {
  double s = 0.0;
  if (n) {
    for (int i = threadIdx.x & 31; i < n; i += 32) s += sums[i];
  } else {
    for (int64_t r = threadIdx.x & 31; r < rows; r += 32)
      if (checked_label(labels[r], vocab, ignore_index) >= 0) s += weights ? (double)weights[r] : 1.0;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  return (float)s;
}
__device__ __forceinline__ float warp_denominator(const RowOut& o, const rk_policy_terms& k, int64_t rows, int vocab,
                                                  int ignore_index) {
  return k.denominator ? *k.denominator
                       : warp_weight(o.weights, o.n_weights, o.labels, k.weights, rows, vocab, ignore_index);
}

// ---------------------------------------------------------------- rows through a ring in shared memory
// Persistent CTAs; a cluster of C CTAs takes a row, each a contiguous share of its 16-byte vectors. One warp
// issues bulk copies of chunks (four vectors a thread) into a ring, the other warps sum them as they land;
// the CTA, then the cluster, joins its sums in a fixed order; and with a gradient the chunks, still in the ring, are
// turned into it and stored, each slot refilled with the next row's chunk behind that. So the logits cross HBM once
// each way.
// Bounds: HBM (14848 x 50257 x 16 bits: sums 231 us at the measured copy rate, with the gradient 462), and the exponential
// unit, which takes an exponential for each element of a sum and one more for its gradient (331 us at full rate). Measured:
// sums 240 us (6.2 TB/s), with entropy 276; policy loss with its gradient 544 (5.5 TB/s; 484 with the exponentials left
// out), with entropy 583: the unit is 60 % busy, issue slots 47 %, and what waits waits for dependent results of four warps
// a scheduler, which is what two such rings an SM leave room for. 2047 x 32003 x 32 bits, sums: 43 (6.1 TB/s).
// NT summing threads a CTA: shorter rows take smaller rings and more CTAs, so that one row's joins hide behind the
// others' sums. Of a row longer than its ring the first chunks are let go after the sums and loaded again behind the
// others for the gradient: from L2, which holds the rows that are in work.
constexpr int kUnroll = 4;     // vectors a thread takes of a chunk
constexpr int kMaxSlots = 9;
constexpr int kFreeSlots = 2;  // slots that a row longer than the ring leaves to the chunks that pass through
constexpr int kMaxCluster = 8;
constexpr int kMaxRowThreads = 512;
constexpr int64_t chunk_bytes(int nt) { return (int64_t)nt * kUnroll * 16; }

struct RingShared {
  uint64_t full[kMaxSlots], empty[kMaxSlots], joined;
  RowSum part[2][kMaxRowThreads / 32];
  RowSum peer[2][kMaxCluster];
  RowSum sum;
  RowGrad grad;
  int far;
  int abort;
};
constexpr int ring_bytes(int nt, int slots) { return (int)(slots * chunk_bytes(nt)) + (int)sizeof(RingShared); }

// A warp has read its part of a chunk: its slot may be filled again. The fence orders the reads before the copy that
// follows, which writes through the other proxy; without it loads still queued behind stores read the new chunk.
__device__ __forceinline__ void release_slot(uint64_t* empty) {
  fence_proxy_async_smem();
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(empty));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, int rank) {
  uint32_t out;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(addr), "r"(rank));
  return out;
}
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return (int)r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ bool try_wait_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
// Data waits of a CTA that has given up return at once: its threads go on through their rows, so that every barrier
// still gets its arrivals, and the status word tells the host.
__device__ __noinline__ bool ring_wait_long(uint32_t bar, uint32_t parity, unsigned int* status, volatile int* abort) {
  return !*abort && mbar_wait(bar, parity, status, RK_DEV_ROW_TIMEOUT, abort);
}
__device__ __forceinline__ bool ring_wait(uint64_t* bar, uint32_t parity, unsigned int* status, volatile int* abort) {
  return mbar_try_wait(smem_u32(bar), parity) || ring_wait_long(smem_u32(bar), parity, status, abort);
}
template <int NT>
__device__ __forceinline__ void row_bar() {
  __syncwarp();
  asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory");
}

// Warp 0 of each CTA of the cluster: sends `mine` to every CTA and joins what all of them sent, in rank order.
template <bool ENT>
__device__ __forceinline__ RowSum cluster_join(RingShared& sh, const RowSum& mine, float c, int rank, int n, uint32_t& phase,
                                               unsigned int* status) {
  const int lane = threadIdx.x & 31;
  __syncwarp();  // what any lane has read of the row is read before a peer learns that it may write
  if (lane < n) {
    const uint32_t dst = cluster_addr(smem_u32(&sh.peer[phase & 1][rank]), lane);
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(mine.r), "f"(mine.m), "f"(mine.s),
                 "f"(mine.w)
                 : "memory");
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                     cluster_addr(smem_u32(&sh.joined), lane))
                 : "memory");
  }
  bool there = false;
  for (int i = 0; i < 256 && !there; ++i) there = try_wait_cluster(smem_u32(&sh.joined), phase & 1);
  if (!there) {  // reading the timer costs more than the whole exchange, so only a long wait does
    const uint64_t t0 = globaltimer();
    while (!try_wait_cluster(smem_u32(&sh.joined), phase & 1)) {
      if (*(volatile int*)&sh.abort) break;
      if (globaltimer() - t0 > RK_WAIT_LIMIT_NS) {
        flag_error(status, RK_DEV_ROW_TIMEOUT);
        *(volatile int*)&sh.abort = 1;
        break;
      }
    }
  }
  const RowSum a = lane < n ? sh.peer[phase & 1][lane] : empty_sum();
  ++phase;
  return warp_join<ENT, kMaxCluster>(a, c);
}

// A chunk into a thread's sums; src: the thread's first vector of it.
template <typename T, bool ENT, int NT>
__device__ __forceinline__ void sum_chunk(RowSum& a, const uint4* src, int tid, int ch, int nvec, float c) {
  constexpr int kChunk = NT * kUnroll;
  if ((ch + 1) * kChunk <= nvec) {
    uint4 v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = src[u * NT];
    add_vectors<T, ENT, kUnroll>(a, v, c);
  } else {
    for (int i = ch * kChunk + tid; i < nvec; i += NT, src += NT) {
      const uint4 v[1] = {*src};
      add_vectors<T, ENT, 1>(a, v, c);
    }
  }
}
// What a row's gradient is formed from, besides its elements.
struct GradRow {
  RowSum a;
  RowGrad k;
  bool far, vec;  // the (x - r) c form; whether dx has the phase of 16 bytes where x has it
  int hot, label; // the vector that holds the label, if one does
};
// A chunk's gradients, and its slot released as soon as it is read.
template <typename T, bool ENT, int NT>
__device__ __forceinline__ void grad_chunk(const uint4* src, int tid, int ch, const RowSpan<T>& sp, T* dx, float c,
                                           const GradRow& g, uint64_t* empty) {
  constexpr int kChunk = NT * kUnroll;
  const int i0 = ch * kChunk + tid;
  uint4 v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) v[u] = src[u * NT];  // past the row: what the slot held before, unused
  T* to = dx + sp.head + (int64_t)i0 * kPer<T>;
  if (g.vec && !g.far && (ch + 1) * kChunk <= sp.nvec && (unsigned)(g.hot - ch * kChunk) >= (unsigned)kChunk) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = grad_vector<T, ENT>(v[u], c, g.a, g.k);
    release_slot(empty);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) __stcs(reinterpret_cast<uint4*>(to) + u * NT, v[u]);
  } else {
    release_slot(empty);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * NT;
      if (i >= sp.nvec) break;
      const uint4 d = g.far || i == g.hot
                          ? grad_vector_any<T, ENT>(v[u], c, g.a, g.far, g.k, sp.head + i * kPer<T>, g.label)
                          : grad_vector<T, ENT>(v[u], c, g.a, g.k);
      store_vector(to + u * NT * kPer<T>, d, g.vec);
    }
  }
}
// The column of the element before or behind the vectors that thread `tid` takes, or -1: the head in 0..7, the tail in 8..15.
template <typename T>
__device__ __forceinline__ int edge_column(const RowSpan<T>& sp, int tid, int vocab) {
  if (tid >= 16) return -1;
  const int i = tid & 7;
  if (tid < 8) return i < sp.head ? i : -1;
  return i < sp.tail ? vocab - 1 - i : -1;
}
// A row without a label: zeros over the `rank`-th of n shares of its vectors, and rank 0 the elements around them.
template <typename T, int NT>
__device__ __forceinline__ void zero_row(T* dx, int tid, int vocab, int rank, int n) {
  const RowSpan<T> sz(dx, vocab);
  const int v0 = (int)((int64_t)sz.nvec * rank / n), v1 = (int)((int64_t)sz.nvec * (rank + 1) / n);
  for (int i = v0 + tid; i < v1; i += NT) __stcs(reinterpret_cast<uint4*>(dx + sz.head) + i, make_uint4(0, 0, 0, 0));
  if (rank == 0 && tid < sz.head) dx[tid] = Dt<T>::from_f(0.f);
  if (rank == 0 && tid < sz.tail) dx[vocab - 1 - tid] = Dt<T>::from_f(0.f);
}
// One warp: what a row's sums give, and the factors of its gradient; `write`: this warp is the one that stores the former.
template <bool POLICY, bool ENT>
__device__ __forceinline__ RowGrad row_result(const RowOut& o, const rk_policy_terms& k, const PolicyIn& in, int64_t row,
                                              const RowSum& a, bool far, float xl, float c, float inv_d, float scale,
                                              bool write) {
  const float ln_s = logf(a.s);
  const float lp = fmaf(exponent(xl, c, a, far), kLn2, -ln_s);
  const float h = ENT ? ln_s - kLn2 * a.w / a.s : 0.f;
  float g_lp = 0.f, g_h = 0.f;
  write = write && (threadIdx.x & 31) == 0;
  if constexpr (POLICY) {
    const PolicyRow q = policy_row(k, in, lp, h, inv_d);
    g_lp = q.g_lp;
    g_h = q.g_h;
    if (write) {
      o.parts[row] = {q.loss, q.clipped};
      o.fine[row] = {xl, a.r, a.s, q.slope};
      if (o.kl) o.kl[row] = q.kl;
      if (o.coef) o.coef[row] = {q.g_lp, q.g_h};
    }
  }
  if (write) {
    o.logprob[row] = lp;
    if constexpr (ENT) o.entropy[row] = h;
    if (o.stats) o.stats[row] = {a.r, a.s};
  }
  return row_grad(a.s, ln_s, h, g_lp * scale, g_h * scale);
}

// POLICY: the policy loss of the row, and with GRAD its gradient; else the log-probabilities alone. NT summing
// threads, kSlots chunks in the ring, CTAS of them an SM. FITS: the ring holds a row's share (the loops without chunks
// that pass twice take 17 us less, 14848 x 50257 x 16 bits).
template <typename T, bool POLICY, bool GRAD, bool ENT, int NT, int kSlots, int CTAS, bool FITS>
__global__ void __launch_bounds__(NT + 32, CTAS)
    ring_row_kernel(const T* logits, int64_t ld, int vocab, int64_t rows, float c, int ignore_index, int cluster, RowOut o,
                    rk_policy_terms k, T* dlogits, int64_t ldd) {
  constexpr int kWarps = NT / 32, kChunk = NT * kUnroll;  // warps that sum, vectors of a chunk
  extern __shared__ __align__(128) unsigned char ring[];
  RingShared& sh = *reinterpret_cast<RingShared*>(ring + kSlots * kChunk * 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = cluster > 1 ? cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), kWarps);
    }
    mbar_init(smem_u32(&sh.joined), cluster);
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (cluster > 1) cluster_sync();
  pdl_wait();  // inputs are the previous kernel's outputs
  const int64_t first = blockIdx.x / cluster, step = gridDim.x / cluster;
  volatile int* abort = &sh.abort;

  if (warp == kWarps) {
    if (lane == 0) {
      int slot = 0;
      uint32_t turn = 0;  // how often the ring has gone round
      for (RowDeal deal(o, rows, vocab, ignore_index, first, step); deal.more() && !*abort; deal.advance()) {
        if (deal.label < 0) continue;
        const T* x = logits + deal.row * ld;
        const RowSpan<T> sp(x, vocab);
        const int chunks = (sp.nvec + kChunk - 1) / kChunk;
        const int k0 = chunks * rank / cluster, n = chunks * (rank + 1) / cluster - k0;
        const int again = GRAD && !FITS && n > kSlots ? n - (kSlots - kFreeSlots) : 0;
        for (int j = 0; j < n + again; ++j) {
          const int ch = k0 + (j < n ? j : j - n);
          if (turn && !ring_wait(&sh.empty[slot], (turn - 1) & 1, o.status, abort)) break;
          const uint32_t bytes = 16u * (uint32_t)min(kChunk, sp.nvec - ch * kChunk);
          const uint32_t bar = smem_u32(&sh.full[slot]);
          mbar_arrive_expect_tx(bar, bytes);
          bulk_load(smem_u32(ring) + slot * kChunk * 16, x + sp.head + (int64_t)ch * kChunk * kPer<T>, bytes, bar);
          if (++slot == kSlots) {
            slot = 0;
            ++turn;
          }
        }
      }
      if (*abort) {  // nothing may still be on its way when the CTA ends
        for (int i = 0; i < kSlots; ++i) {
          const uint32_t filled = turn + (i < slot ? 1 : 0);
          if (filled) {
            const uint64_t t0 = globaltimer();
            while (!mbar_try_wait(smem_u32(&sh.full[i]), (filled - 1) & 1) && globaltimer() - t0 < RK_WAIT_LIMIT_NS) {
            }
          }
        }
      }
    }
  } else {
    int slot = 0;
    uint32_t turn = 0, parity = 0, phase = 0;
    float inv_d = 0.f, scale = 0.f;
    if (POLICY && warp == 0) {
      const float d = warp_denominator(o, k, rows, vocab, ignore_index);
      if (blockIdx.x == 0 && lane == 0) *o.denom = d;
      inv_d = d != 0.f ? 1.f / d : 0.f;
      scale = k.inv_temp * k.grad_scale * (k.grad_scale_dev ? *k.grad_scale_dev : 1.f);
    }
    for (RowDeal deal(o, rows, vocab, ignore_index, first, step); deal.more(); deal.advance()) {
      const int64_t row = deal.row;
      const int label = deal.label;
      T* dx = GRAD ? dlogits + row * ldd : nullptr;
      if (label < 0) {
        if (!o.list && threadIdx.x == 0 && rank == 0) unlabelled_row<POLICY>(o, row, label);
        if constexpr (GRAD) zero_row<T, NT>(dx, threadIdx.x, vocab, rank, cluster);
        continue;
      }
      const T* x = logits + row * ld;
      const RowSpan<T> sp(x, vocab);
      const int chunks = (sp.nvec + kChunk - 1) / kChunk;
      const int k0 = chunks * rank / cluster, n = chunks * (rank + 1) / cluster - k0;
      const int again = GRAD && !FITS && n > kSlots ? n - (kSlots - kFreeSlots) : 0;  // chunks that pass through twice
      const int edge = rank == 0 ? edge_column(sp, threadIdx.x, vocab) : -1;
      const float xe = edge >= 0 ? Dt<T>::to_f(x[edge]) : 0.f;
      const float xl = warp == 0 ? Dt<T>::to_f(x[label]) : 0.f;
      PolicyIn in = {};
      if (POLICY && warp == 0) in = policy_in(k, row);
      RowSum a = empty_sum();
      {
        int s = slot;
        uint32_t t = turn;
        for (int j = 0; j < n; ++j) {
          const int ch = k0 + j;
          ring_wait(&sh.full[s], t & 1, o.status, abort);
          sum_chunk<T, ENT, NT>(a, reinterpret_cast<const uint4*>(ring) + s * kChunk + threadIdx.x, threadIdx.x, ch, sp.nvec, c);
          const bool passes = !GRAD || j < again;
          if (passes) release_slot(&sh.empty[s]);
          if (++s == kSlots) {
            s = 0;
            ++t;
          }
          if (passes) {  // what stays in the ring begins behind it
            slot = s;
            turn = t;
          }
        }
      }
      if (edge >= 0) add_element<ENT>(a, xe, c);
      a = warp_join<ENT>(a, c);
      if (lane == 0) sh.part[parity][warp] = a;
      row_bar<NT>();
      if (warp == 0) {
        a = warp_join<ENT, kWarps>(lane < kWarps ? sh.part[parity][lane] : empty_sum(), c);
        if (cluster > 1) a = cluster_join<ENT>(sh, a, c, rank, cluster, phase, o.status);
        const bool far = is_far(a);
        if (far) {
          a = warp_row_sum_far(x, vocab, c);
          // no CTA of the cluster may write over the row before all have read it
          if (cluster > 1) cluster_join<ENT>(sh, a, c, rank, cluster, phase, o.status);
        }
        const RowGrad g = row_result<POLICY, ENT>(o, k, in, row, a, far, xl, c, inv_d, scale, rank == 0);
        if (GRAD && lane == 0) {
          sh.sum = a;
          sh.far = far;
          sh.grad = g;
        }
      }
      parity ^= 1;
      if constexpr (GRAD) {
        row_bar<NT>();
        const GradRow g = {sh.sum, sh.grad, sh.far != 0, ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0,
                           (label - sp.head) / kPer<T>, label};
        for (int j = again; j < n + again; ++j) {
          const int ch = k0 + (j < n ? j : j - n);
          if (j >= n) ring_wait(&sh.full[slot], turn & 1, o.status, abort);
          grad_chunk<T, ENT, NT>(reinterpret_cast<const uint4*>(ring) + slot * kChunk + threadIdx.x, threadIdx.x, ch, sp, dx, c, g,
                                 &sh.empty[slot]);
          if (++slot == kSlots) {
            slot = 0;
            ++turn;
          }
        }
        if (edge >= 0) {
          const float t = exponent(xe, c, g.a, g.far);
          dx[edge] = Dt<T>::from_f(grad_element<ENT>(t, g.k) + (edge == label ? g.k.g : 0.f));
        }
      }
    }
    if (POLICY && warp == 0 && rank == 0) finish_losses(o, first, step, rows, c, vocab, ignore_index);
  }
  __syncwarp();
  if (cluster > 1) cluster_sync();  // no CTA ends while another may still send to it
}

// ---------------------------------------------------------------- long fp32 rows: sums and gradients side by side
// One CTA an SM, whose ring holds about two rows: half of its warps sum the row that has come while the other half turn
// the one before it into its gradient, so that neither the copies nor the exponential unit wait for a row's joins. A row's
// factors go from one half to the other through two places with a barrier each way. No circle of waits: the gradients of a
// row wait for its sums alone, its sums for its chunks, these for the slots of rows before it, as a row fits the ring.
// 2047 x 25000 x 32 bits: 72 us (5.7 TB/s), x 32003 96 (5.5), 2000 x 50257 142 (5.65).
constexpr int kSplitThreads = 256, kSplitSlots = 14;
struct SplitShared {
  uint64_t full[kSplitSlots], empty[kSplitSlots], ready[2], taken[2];
  RowSum part[2][kSplitThreads / 32];
  RowSum sum[2];
  RowGrad grad[2];
  int far[2];
  int abort;
};
constexpr int kSplitBytes = (int)(kSplitSlots * chunk_bytes(kSplitThreads)) + (int)sizeof(SplitShared);
static_assert(kSplitBytes + 1024 <= 228 * 1024, "the ring of an SM's CTA");
static_assert(kSplitSlots == 14, "kLongRow: rows that the ring holds");

template <typename T, bool ENT>
__global__ void __launch_bounds__(2 * kSplitThreads + 32, 1)
    split_row_kernel(const T* logits, int64_t ld, int vocab, int64_t rows, float c, int ignore_index, RowOut o,
                    rk_policy_terms k, T* dlogits, int64_t ldd) {
  constexpr int NT = kSplitThreads, kWarps = NT / 32, kChunk = NT * kUnroll;
  extern __shared__ __align__(128) unsigned char ring[];
  SplitShared& sh = *reinterpret_cast<SplitShared*>(ring + kSplitSlots * kChunk * 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSplitSlots; ++i) {
      mbar_init(smem_u32(&sh.full[i]), 1);
      mbar_init(smem_u32(&sh.empty[i]), kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&sh.ready[i]), 1);
      mbar_init(smem_u32(&sh.taken[i]), kWarps);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  pdl_wait();  // inputs are the previous kernel's outputs
  const int64_t first = blockIdx.x, step = gridDim.x;
  volatile int* abort = &sh.abort;
  int slot = 0;
  uint32_t turn = 0;  // how often the ring has gone round
  const auto next_slot = [&] {
    if (++slot == kSplitSlots) {
      slot = 0;
      ++turn;
    }
  };

  if (warp == 2 * kWarps) {  // copies
    if (lane == 0) {
      for (RowDeal deal(o, rows, vocab, ignore_index, first, step); deal.more() && !*abort; deal.advance()) {
        if (deal.label < 0) continue;
        const T* x = logits + deal.row * ld;
        const RowSpan<T> sp(x, vocab);
        for (int ch = 0; ch * kChunk < sp.nvec; ++ch) {
          if (turn && !ring_wait(&sh.empty[slot], (turn - 1) & 1, o.status, abort)) break;
          const uint32_t bytes = 16u * (uint32_t)min(kChunk, sp.nvec - ch * kChunk);
          const uint32_t bar = smem_u32(&sh.full[slot]);
          mbar_arrive_expect_tx(bar, bytes);
          bulk_load(smem_u32(ring) + slot * kChunk * 16, x + sp.head + (int64_t)ch * kChunk * kPer<T>, bytes, bar);
          next_slot();
        }
      }
      if (*abort) {  // nothing may still be on its way when the CTA ends
        for (int i = 0; i < kSplitSlots; ++i) {
          const uint32_t filled = turn + (i < slot ? 1 : 0);
          if (filled) {
            const uint64_t t0 = globaltimer();
            while (!mbar_try_wait(smem_u32(&sh.full[i]), (filled - 1) & 1) && globaltimer() - t0 < RK_WAIT_LIMIT_NS) {
            }
          }
        }
      }
    }
  } else if (warp < kWarps) {  // sums
    float inv_d = 0.f, scale = 0.f;
    if (warp == 0) {
      const float d = warp_denominator(o, k, rows, vocab, ignore_index);
      if (blockIdx.x == 0 && lane == 0) *o.denom = d;
      inv_d = d != 0.f ? 1.f / d : 0.f;
      scale = k.inv_temp * k.grad_scale * (k.grad_scale_dev ? *k.grad_scale_dev : 1.f);
    }
    uint32_t done = 0;  // rows summed
    for (RowDeal deal(o, rows, vocab, ignore_index, first, step); deal.more(); deal.advance()) {
      const int64_t row = deal.row;
      const int label = deal.label;
      if (label < 0) {
        if (!o.list && threadIdx.x == 0) unlabelled_row<true>(o, row, label);
        continue;
      }
      const T* x = logits + row * ld;
      const RowSpan<T> sp(x, vocab);
      const int edge = edge_column(sp, threadIdx.x, vocab);
      const float xe = edge >= 0 ? Dt<T>::to_f(x[edge]) : 0.f;
      const float xl = warp == 0 ? Dt<T>::to_f(x[label]) : 0.f;
      PolicyIn in = {};
      if (warp == 0) in = policy_in(k, row);
      RowSum a = empty_sum();
      for (int ch = 0; ch * kChunk < sp.nvec; ++ch) {
        ring_wait(&sh.full[slot], turn & 1, o.status, abort);
        sum_chunk<T, ENT, NT>(a, reinterpret_cast<const uint4*>(ring) + slot * kChunk + threadIdx.x, threadIdx.x, ch, sp.nvec, c);
        next_slot();
      }
      if (edge >= 0) add_element<ENT>(a, xe, c);
      a = warp_join<ENT>(a, c);
      const int at = done & 1;
      if (lane == 0) sh.part[at][warp] = a;
      row_bar<NT>();
      if (warp == 0) {
        a = warp_join<ENT, kWarps>(lane < kWarps ? sh.part[at][lane] : empty_sum(), c);
        const bool far = is_far(a);
        if (far) a = warp_row_sum_far(x, vocab, c);
        const RowGrad g = row_result<true, ENT>(o, k, in, row, a, far, xl, c, inv_d, scale, true);
        if (done >= 2) ring_wait(&sh.taken[at], ((done >> 1) - 1) & 1, o.status, abort);  // what the row before the last left
        __syncwarp();
        if (lane == 0) {
          sh.sum[at] = a;
          sh.far[at] = far;
          sh.grad[at] = g;
          mbar_arrive(smem_u32(&sh.ready[at]));
        }
      }
      ++done;
    }
    if (warp == 0) finish_losses(o, first, step, rows, c, vocab, ignore_index);
  } else {  // gradients
    const int tid = threadIdx.x - NT;
    uint32_t done = 0;
    for (RowDeal deal(o, rows, vocab, ignore_index, first, step); deal.more(); deal.advance()) {
      const int64_t row = deal.row;
      const int label = deal.label;
      T* dx = dlogits + row * ldd;
      if (label < 0) {
        zero_row<T, NT>(dx, tid, vocab, 0, 1);
        continue;
      }
      const T* x = logits + row * ld;
      const RowSpan<T> sp(x, vocab);
      const int at = done & 1;
      ring_wait(&sh.ready[at], (done >> 1) & 1, o.status, abort);
      const GradRow g = {sh.sum[at], sh.grad[at], sh.far[at] != 0, ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0,
                         (label - sp.head) / kPer<T>, label};
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.taken[at]));
      ++done;
      const int edge = edge_column(sp, tid, vocab);
      if (edge >= 0) {
        const float t = exponent(Dt<T>::to_f(x[edge]), c, g.a, g.far);
        dx[edge] = Dt<T>::from_f(grad_element<ENT>(t, g.k) + (edge == label ? g.k.g : 0.f));
      }
      for (int ch = 0; ch * kChunk < sp.nvec; ++ch) {
        ring_wait(&sh.full[slot], turn & 1, o.status, abort);  // complete, as the sums are; orders the copy's writes
        grad_chunk<T, ENT, NT>(reinterpret_cast<const uint4*>(ring) + slot * kChunk + tid, tid, ch, sp, dx, c, g, &sh.empty[slot]);
        next_slot();
      }
    }
  }
}

// ---------------------------------------------------------------- short rows: one warp each
// The same sums straight from global memory, four vectors a lane in flight, and for the gradient the row once more, from
// L1 or L2. No join but the warp's own, which is what bounds short rows in a ring: 12001 x 1000 x 32 bits 8.9 us for the
// sums (5.4 TB/s, half of it from L2), 27 with the gradient. That is more than sums and gradients from statistics take as
// two launches (20): the policy's logarithm in fp64 stands in each row (1.4 us of the 27 at 12001 rows, 1.7 of 32 at 16384
// x 1001), twice as many CTAs are launched as fit an SM with 64 registers (25.1 with four, but 32.7 in place of 32.4 at
// 16384 x 1001), and no load of the next row is under way while this one is finished.
template <typename T, bool POLICY, bool GRAD, bool ENT>
__global__ void __launch_bounds__(256)
    warp_row_kernel(const T* logits, int64_t ld, int vocab, int64_t rows, float c, int ignore_index, RowOut o,
                    rk_policy_terms k, T* dlogits, int64_t ldd) {
  pdl_wait();  // inputs are the previous kernel's outputs
  const int lane = threadIdx.x & 31;
  float denom = 0.f;
  double loss = 0.0, clipped = 0.0;  // over this warp's rows
  if constexpr (POLICY) {
    denom = warp_denominator(o, k, rows, vocab, ignore_index);
    if (blockIdx.x == 0 && threadIdx.x == 0) *o.denom = denom;
  }
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += (int64_t)gridDim.x * 8) {
    const int label = checked_label(o.labels[row], vocab, ignore_index);
    T* dx = GRAD ? dlogits + row * ldd : nullptr;
    if (label < 0) {
      if (lane == 0) unlabelled_row<POLICY>(o, row, label);
      if constexpr (GRAD) {
        zero_row<T, 32>(dx, lane, vocab, 0, 1);
      }
      continue;
    }
    const T* x = logits + row * ld;
    const RowSpan<T> sp(x, vocab);
    const uint4* xv = reinterpret_cast<const uint4*>(x + sp.head);
    const int edge = edge_column(sp, lane, vocab);
    const float xe = edge >= 0 ? Dt<T>::to_f(x[edge]) : 0.f;
    const float xl = Dt<T>::to_f(x[label]);
    PolicyIn in = {};
    if (POLICY) in = policy_in(k, row);
    RowSum a = empty_sum();
    int i = lane;
    for (; i + 32 * (kUnroll - 1) < sp.nvec; i += 32 * kUnroll) {
      uint4 v[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) v[u] = xv[i + 32 * u];
      add_vectors<T, ENT, kUnroll>(a, v, c);
    }
    for (; i < sp.nvec; i += 32) {
      const uint4 v[1] = {xv[i]};
      add_vectors<T, ENT, 1>(a, v, c);
    }
    if (edge >= 0) add_element<ENT>(a, xe, c);
    a = warp_join<ENT>(a, c);
    const bool far = is_far(a);
    if (far) a = warp_row_sum_far(x, vocab, c);
    const float ln_s = logf(a.s);
    const float lp = fmaf(exponent(xl, c, a, far), kLn2, -ln_s);
    const float h = ENT ? ln_s - kLn2 * a.w / a.s : 0.f;
    float g_lp = 0.f, g_h = 0.f;
    if constexpr (POLICY) {
      const PolicyRow q = policy_row(k, in, lp, h, denom != 0.f ? 1.f / denom : 0.f);
      g_lp = q.g_lp;
      g_h = q.g_h;
      loss += (double)q.loss + (double)loss_rounding(xl, c, a, far, lp, q.slope);
      clipped += (double)q.clipped;
      if (lane == 0) {
        if (o.kl) o.kl[row] = q.kl;
        if (o.coef) o.coef[row] = {q.g_lp, q.g_h};
      }
    }
    if (lane == 0) {
      o.logprob[row] = lp;
      if constexpr (ENT) o.entropy[row] = h;
      if (o.stats) o.stats[row] = {a.r, a.s};
    }
    if constexpr (GRAD) {
      const float scale = k.inv_temp * k.grad_scale * (k.grad_scale_dev ? *k.grad_scale_dev : 1.f);
      const RowGrad gk = row_grad(a.s, ln_s, h, g_lp * scale, g_h * scale);
      const bool vec = ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0;
      __syncwarp();  // every lane has read the label's element and its own before any is written over
      const int hot = (label - sp.head) / kPer<T>;  // the vector that holds the label, if one does
#pragma unroll 4
      for (int i = lane; i < sp.nvec; i += 32) {
        const int at = sp.head + i * kPer<T>;
        const uint4 v = xv[i];
        store_vector(dx + at, far || i == hot ? grad_vector_any<T, ENT>(v, c, a, far, gk, at, label)
                                              : grad_vector<T, ENT>(v, c, a, gk), vec);
      }
      if (edge >= 0)
        dx[edge] = Dt<T>::from_f(grad_element<ENT>(exponent(xe, c, a, far), gk) + (edge == label ? gk.g : 0.f));
    }
  }
  if constexpr (POLICY) {
    __shared__ double2 sums[8];
    if (lane == 0) sums[threadIdx.x >> 5] = {loss, clipped};
    __syncthreads();
    if (threadIdx.x == 0) {
      double2 all = sums[0];
      for (int w = 1; w < 8; ++w) all = {all.x + sums[w].x, all.y + sums[w].y};
      o.sums[blockIdx.x] = all;
    }
  }
}

// ---------------------------------------------------------------- gradients from saved statistics
// No element depends on another: one CTA per (row, segment of 1024 vectors), four of them a thread in flight, so that many
// small CTAs keep HBM busy by themselves. 14848 x 50257 x 16 bits: 445 to 470 us (6.4 to 6.7 TB/s, the copy rate), 2047 x
// 32003 x 32 bits 78 (6.7). Short rows, many of them: one warp each (16384 x 1001 x 16 bits 10 us in place of 31).
constexpr int kBwdThreads = 256, kBwdVecs = 4;

// NT threads: a warp, with a row, or a CTA, with a segment of kBwdVecs vectors a thread.
template <typename T, bool ENT, int NT>
__device__ __forceinline__ void bwd_row(const T* logits, int64_t ld, int vocab, int64_t row, int seg, int tid,
                                        const int64_t* __restrict__ labels, float inv_temp, int ignore_index,
                                        const float2* __restrict__ stats, const float* __restrict__ entropy,
                                        const float* __restrict__ d_logprob, const float* __restrict__ d_entropy,
                                        int64_t coef_stride, float scale_by, const float* __restrict__ scale_dev,
                                        T* dlogits, int64_t ldd) {
  constexpr int kStep = NT * kBwdVecs;
  const int label = checked_label(labels[row], vocab, ignore_index);
  const T* x = logits + row * ld;
  T* dx = dlogits + row * ldd;
  const RowSpan<T> sp(label >= 0 ? x : dx, vocab);
  const int v0 = seg * kStep, v1 = NT == 32 ? sp.nvec : min(v0 + kStep, sp.nvec);
  const int edge = seg == 0 ? edge_column(sp, tid, vocab) : -1;
  if (label < 0) {
#pragma unroll 4
    for (int i = v0 + tid; i < v1; i += NT) __stcs(reinterpret_cast<uint4*>(dx + sp.head) + i, make_uint4(0, 0, 0, 0));
    if (edge >= 0) dx[edge] = Dt<T>::from_f(0.f);
    return;
  }
  const bool vec = ((reinterpret_cast<uintptr_t>(dx) ^ reinterpret_cast<uintptr_t>(x)) & 15) == 0;
  const int hot = (label - sp.head) / kPer<T>;  // the vector that holds the label, if one does
  uint4 v[kBwdVecs];
  const auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < kBwdVecs; ++j)
      if (base + j * NT < v1) v[j] = reinterpret_cast<const uint4*>(x + sp.head)[base + j * NT];
  };
  load(v0 + tid);
  const float c = inv_temp * kLog2e;
  const float scale = inv_temp * scale_by * (scale_dev ? *scale_dev : 1.f);
  const float2 st = stats[row];
  const RowSum a = {st.x, st.x * c, st.y, 0.f};
  const bool far = is_far(a);
  const RowGrad k = row_grad(a.s, ENT ? logf(a.s) : 0.f, ENT ? entropy[row] : 0.f, d_logprob[row * coef_stride] * scale,
                             ENT ? d_entropy[row * coef_stride] * scale : 0.f);
  const auto store = [&](int base) {
#pragma unroll
    for (int j = 0; j < kBwdVecs; ++j) {
      const int i = base + j * NT;
      if (i < v1) {
        const int at = sp.head + i * kPer<T>;
        store_vector(dx + at, far || i == hot ? grad_vector_any<T, ENT>(v[j], c, a, far, k, at, label)
                                              : grad_vector<T, ENT>(v[j], c, a, k), vec);
      }
    }
  };
  store(v0 + tid);
  if constexpr (NT == 32) {
    for (int base = tid + kStep; base < v1; base += kStep) {
      load(base);
      store(base);
    }
  }
  if (edge >= 0)
    dx[edge] = Dt<T>::from_f(grad_element<ENT>(exponent(Dt<T>::to_f(x[edge]), c, a, far), k) + (edge == label ? k.g : 0.f));
}

// BY_WARP: a warp a row; else a CTA a segment.
template <typename T, bool ENT, bool BY_WARP>
__global__ void __launch_bounds__(kBwdThreads)
    logprob_bwd_kernel(const T* logits, int64_t ld, int vocab, int64_t rows, int segments, const int64_t* __restrict__ labels,
                       float inv_temp, int ignore_index, const float2* __restrict__ stats,
                       const float* __restrict__ entropy, const float* __restrict__ d_logprob,
                       const float* __restrict__ d_entropy, int64_t coef_stride, float scale_by,
                       const float* __restrict__ scale_dev, T* dlogits, int64_t ldd) {
  pdl_wait();  // inputs are the previous kernel's outputs
  if constexpr (BY_WARP) {
    const int64_t row = (int64_t)blockIdx.x * (kBwdThreads / 32) + (threadIdx.x >> 5);
    if (row < rows)
      bwd_row<T, ENT, 32>(logits, ld, vocab, row, 0, threadIdx.x & 31, labels, inv_temp, ignore_index, stats, entropy,
                          d_logprob, d_entropy, coef_stride, scale_by, scale_dev, dlogits, ldd);
  } else {
    bwd_row<T, ENT, kBwdThreads>(logits, ld, vocab, blockIdx.x / segments, blockIdx.x % segments, threadIdx.x, labels,
                                 inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, scale_by,
                                 scale_dev, dlogits, ldd);
  }
}

// The takers' sums over the denominator.
__global__ void __launch_bounds__(256) policy_reduce_kernel(const double2* __restrict__ sums, int n,
                                                            const float* __restrict__ denom,
                                                            float* __restrict__ metrics) {
  pdl_wait();  // inputs are the previous kernel's outputs
  double a = 0.0, b = 0.0;
#pragma unroll 5
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const double2 v = sums[i];
    a += v.x;
    b += v.y;
  }
  const double2 sum = block_sum2(a, b);
  if (threadIdx.x == 0) {
    const float d = denom ? *denom : 0.f;
    const double inv = d != 0.f ? 1.0 / d : 0.0;
    metrics[0] = (float)(sum.x * inv);
    metrics[1] = d;
    metrics[2] = (float)(sum.y * inv);
    metrics[3] = 0.f;
  }
}

// ---------------------------------------------------------------- preference loss
struct PairLoss {
  float loss, slope;  // slope = dloss / d gap_chosen
};
__device__ __forceinline__ PairLoss pair_loss_of(const rk_preference_terms& k, double gap_chosen, double gap_rejected) {
  const float diff = (float)(gap_chosen - gap_rejected), u = k.beta * diff;
  if (k.kind == RK_PREF_SIGMOID) {
    const float tail = log1pf(expf(-fabsf(u)));
    return {(1.f - k.smoothing) * (fmaxf(-u, 0.f) + tail) + k.smoothing * (fmaxf(u, 0.f) + tail),
            k.beta * (k.smoothing / (1.f + expf(-u)) - (1.f - k.smoothing) / (1.f + expf(u)))};
  }
  if (k.kind == RK_PREF_HINGE) return {fmaxf(1.f - u, 0.f), u < 1.f ? -k.beta : 0.f};
  const float off = diff - 0.5f / k.beta;
  return {off * off, 2.f * off};
}

// After the rows' statistics: one CTA per pair forms the two gaps in a fixed order, the pair's loss and its rows' factors.
// A gap is a sum of hundreds of differences, each small against its two log-probabilities: it is formed in fp64 from the
// rows' statistics, not from the log-probabilities rounded to fp32.
template <typename T>
__global__ void __launch_bounds__(1024)
    preference_pair_kernel(const T* __restrict__ logits, int64_t ld, const int64_t* __restrict__ labels, int64_t pairs,
                           int64_t length, int vocab, int ignore_index, rk_preference_terms k,
                           const float2* __restrict__ stats, float* __restrict__ rewards, float* __restrict__ pair_loss,
                           float* __restrict__ loss, float* __restrict__ coef) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ double red[2][32];
  const int64_t pair = blockIdx.x;
  const int half = blockDim.x >> 1, side = threadIdx.x >= half, tid = threadIdx.x - side * half, lane = threadIdx.x & 31;
  const int64_t base = (side * pairs + pair) * length;  // half of the CTA for each sequence
  const float c = k.inv_temp * kLog2e;
  double g = 0.0, n = 0.0;
#pragma unroll 4
  for (int64_t t = tid; t < length; t += half) {
    const int64_t row = base + t;
    const int label = checked_label(labels[row], vocab, ignore_index);
    const float2 st = stats[row];
    const double ref = k.ref_logprobs ? (double)k.ref_logprobs[row] : 0.0;
    if (label >= 0) {
      const RowSum a = {st.x, st.x * c, st.y, 0.f};
      g += label_logprob(Dt<T>::to_f(logits[row * ld + label]), c, a, is_far(a)) - ref;
      n += 1.0;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    g += __shfl_xor_sync(0xffffffffu, g, o);
    n += __shfl_xor_sync(0xffffffffu, n, o);
  }
  if (lane == 0) {
    red[0][threadIdx.x >> 5] = g;
    red[1][threadIdx.x >> 5] = n;
  }
  __syncthreads();
  double gap[2] = {0.0, 0.0}, count[2] = {0.0, 0.0};
  for (int i = 0; i < 2; ++i) {
    for (int w = i * (half >> 5); w < (i + 1) * (half >> 5); ++w) {
      gap[i] += red[0][w];
      count[i] += red[1][w];
    }
    if (k.average) gap[i] /= fmax(count[i], 1.0);
  }
  const PairLoss q = pair_loss_of(k, gap[0], gap[1]);
  if (threadIdx.x == 0) {
    (pairs > 1 ? pair_loss + pair : loss)[0] = q.loss;
    rewards[pair] = k.beta * (float)gap[0];
    rewards[pairs + pair] = k.beta * (float)gap[1];
  }
  const float s = (side ? -q.slope : q.slope) / (float)pairs / (k.average ? (float)fmax(count[side], 1.0) : 1.f);
  for (int64_t t = tid; t < length; t += half)
    coef[base + t] = checked_label(labels[base + t], vocab, ignore_index) >= 0 ? s : 0.f;
}

// loss = mean of the pair losses.
__global__ void __launch_bounds__(256) preference_reduce_kernel(const float* __restrict__ pair_loss, int64_t pairs,
                                                                float* __restrict__ loss) {
  pdl_wait();  // inputs are the previous kernel's outputs
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < pairs; i += blockDim.x) s += pair_loss[i];
  s = block_sum2(s, 0.0).x;
  if (threadIdx.x == 0) *loss = (float)(s / (double)pairs);
}

}  // namespace rk

using namespace rk;

namespace {

bool shape_ok(int64_t ld, int64_t vocab, int64_t rows) {
  return rows >= 0 && rows < (1ll << 31) && vocab > 0 && vocab < (1ll << 31) && ld >= vocab;
}

// Up to so many rows each CTA takes every n-th and sums the weights by itself (32 loads a lane, as long as the launch it
// saves). Beyond it a launch sums the weights and, of rows that CTAs take, lists those with labels, as masks would load
// CTAs unevenly (a quarter of 14848 rows masked cost 15 %); with more rows than kListRows the loads even out by
// themselves. Sums alone are worth that launch's 4 us from about 60 us on.
constexpr int64_t kFewRows = 1024, kListRows = 32768, kListBytes = 400ll << 20;
constexpr int kMaxWeights = 64;  // CTAs that sum weights: enough to load them, few enough for a warp to sum again

// Row lengths in bytes at which the forms change. us, one warp a row / ring of 64 / 128 / 256 threads:
//   sums, 4096 rows: 22 KB bf16 18.5/19.0/20.5/27.3, 32 KB fp32 22.6/25.1/24.0/26.0, 40 KB fp32 28.6/32.3/28.7/29.9,
//     48 KB bf16 38.2/36.9/37.4/43.5; 14848 of 100 KB bf16 -/243/241/263; 2047 of 128 KB fp32 -/76/46/43
//   policy with gradient: 8192 rows of 6 KB bf16 32/39, 4096 of 16 KB 44/35.5/39/50, of 24 KB 72/49/52/65 (a warp's second
//     read of its row comes from L2 once 64 rows an SM exceed L1); warp / 64: 16384 of 10 KB bf16 93/98, of 12 KB 116/107, with
//     entropies (which cost the ring's two warps more) 96/134 and 119/147, of 14 KB 144/158, of 20 KB 203/174; fp32 10 KB 85/79
//   policy, fp32, one ring / sums and gradients side by side: 4096 rows of 54 KB 87/91, 72 KB 115/105; 2047 of 100 KB 84/72;
//     2000 of 200 KB 166/142; 300 of 72 KB 16/18. With 16-bit logits, whose exponentials bound both, 14848 of 100 KB 545/555
//   policy, 4096 rows of 60 KB bf16: 128 threads and nine slots three times an SM 104, 256 and seven twice 114
// So sums of 16-bit logits take rings of 128 threads eight times an SM (exponentials bound them, and 40 warps hide more
// than the 28 to 92 bytes cost that the forms with entropies or a policy's terms spill at 48 registers),
// fp32 ones, which HBM bounds, of 256 three times. With fewer rows than four an SM a warp's row takes too long alone, and
// the larger CTAs are faster (64 rows of 100 KB: 5.5 / 6.6).
// 256 KB rows (1500 x 131072 x 16 bits) with gradient and a ring of 256 threads twice an SM or of 512 once: 178 / 151, as
// the larger ring keeps 5 of 8 chunks where the smaller keeps 5 of 16.
constexpr int64_t kWarpRow = 4 * 1024, kWarpRowSum = 36 * 1024, kWarpRowGrad = 8 * 1024;
template <typename T, bool ENT>
constexpr int64_t kWarpRowMany = sizeof(T) == 4 ? kWarpRowGrad : ENT ? 14 * 1024 : 10 * 1024;  // from 32 rows an SM
constexpr int64_t kSmallRow = 6 * chunk_bytes(64), kMidRow = 6 * chunk_bytes(128), kThirdRow = 9 * chunk_bytes(128), kLongRow = 14 * chunk_bytes(256),
                  kSplitRow = 4 * chunk_bytes(256);
// Gradients from statistics, us, a CTA / a warp a row: 16384 rows of 2 KB bf16 31/10, 6 KB 52/36, 10 KB 64/58, 14 KB 78/79,
// fp32 12 KB 64/66; 1200 of 2 KB 3.9/2.9, of 8 KB 4.9/5.6; 100 of 12 KB 2.4/5.2. A warp loads 2 KB at once, so that with few
// rows more than that takes it longer than a CTA.
constexpr int64_t kBwdWarpRow = 12 * 1024, kBwdWarpOnce = 2 * 1024;
// A pair's gaps by 256 threads / 1024, us for the whole loss without gradient of one pair of 64 tokens 4.8/6.3, of 512 7.8/7.2,
// of 8192 69/29.
constexpr int64_t kShortPair = 256;

int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      v = 148;
    return v;
  }();
  return n;
}

// CTAs that share a row: with few rows, enough to occupy an SM each while every CTA still has a chunk.
int cluster_for(int64_t rows, int64_t bytes, int nt) {
  const int64_t chunks = (bytes + chunk_bytes(nt) - 1) / chunk_bytes(nt);
  int c = 1;
  while (c < kMaxCluster && rows * c * 2 <= sm_count() && chunks >= 2 * c) c *= 2;
  return c;
}

template <typename T, bool POLICY, bool GRAD, bool ENT, int NT, int SLOTS, int CTAS, bool FITS>
int launch_ring(const T* x, int64_t ld, int64_t vocab, int64_t rows, float c, int ignore_index, const RowOut& o,
                const rk_policy_terms& k, T* dx, int64_t ldd, int* takers, cudaStream_t s) {
  static_assert(CTAS * (ring_bytes(NT, SLOTS) + 1024) <= 228 * 1024, "the rings of an SM's CTAs");
  auto kernel = ring_row_kernel<T, POLICY, GRAD, ENT, NT, SLOTS, CTAS, FITS>;
  const int st = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kernel), ring_bytes(NT, SLOTS));
  if (st) return st;
  const int cluster = cluster_for(rows, vocab * (int64_t)sizeof(T), NT);
  int64_t ctas = rows * cluster;
  const int64_t most = (int64_t)CTAS * sm_count() / cluster * cluster;
  if (ctas > most) ctas = most;
  *takers = (int)(ctas / cluster);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(NT + 32);
  cfg.dynamicSmemBytes = ring_bytes(NT, SLOTS);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = rk_host::pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  cudaLaunchKernelEx(&cfg, kernel, x, ld, (int)vocab, rows, c, ignore_index, cluster, o, k, dx, ldd);
  return rk_host::launch_status();
}

template <typename T, bool ENT>
int launch_split(const T* x, int64_t ld, int64_t vocab, int64_t rows, float c, int ignore_index, const RowOut& o,
                const rk_policy_terms& k, T* dx, int64_t ldd, int* takers, cudaStream_t s) {
  auto kernel = split_row_kernel<T, ENT>;
  const int st = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kernel), kSplitBytes);
  if (st) return st;
  *takers = (int)(rows < sm_count() ? rows : sm_count());
  rk_host::launch_k(kernel, (unsigned)*takers, 2 * kSplitThreads + 32, kSplitBytes, s, x, ld, (int)vocab, rows, c,
                    ignore_index, o, k, dx, ldd);
  return rk_host::launch_status();
}

// `list`: room for rows (row, label) pairs; `weights`: for kMaxWeights sums; *takers: how many of o.sums are written.
template <typename T, bool POLICY, bool GRAD, bool ENT>
int launch_rows(const T* x, int64_t ld, int64_t vocab, int64_t rows, float inv_temp, int ignore_index, RowOut o,
                const rk_policy_terms& k, T* dx, int64_t ldd, int2* list, double* weights, int* takers, cudaStream_t s) {
  const float c = inv_temp * kLog2e;
  const int64_t bytes = vocab * (int64_t)sizeof(T);
  const bool by_warp = bytes <= (rows < 4 * sm_count() ? kWarpRow : !GRAD ? kWarpRowSum : rows < 32 * sm_count() ? kWarpRowGrad : kWarpRowMany<T, ENT>);
  const bool worth = POLICY || rows * bytes >= kListBytes;
  o.list = rows > kFewRows && rows <= kListRows && !by_warp && worth ? list : nullptr;
  const bool weigh = POLICY && !k.denominator && rows > kFewRows;
  if (o.list || weigh) {
    const int64_t blocks = (rows + 1023) / 1024;
    const int grid = (int)(o.list || blocks < kMaxWeights ? blocks : kMaxWeights);
    o.weights = weights;
    o.n_weights = weigh ? grid : 0;
    rk_host::launch_k(list_rows_kernel<POLICY>, (unsigned)grid, 1024, 0, s, rows, (int)vocab, ignore_index, o, k.weights,
                      const_cast<int2*>(o.list), weights);
    const int st = rk_host::launch_status();
    if (st) return st;
  }
  if (by_warp) {
    const int64_t blocks = (rows + 7) / 8, most = (int64_t)sm_count() * 8;
    *takers = (int)(blocks < most ? blocks : most);
    rk_host::launch_k(warp_row_kernel<T, POLICY, GRAD, ENT>, (unsigned)*takers, 256, 0, s, x, ld, (int)vocab, rows, c,
                      ignore_index, o, k, dx, ldd);
    return rk_host::launch_status();
  }
  const auto ring = [&](auto launch) { return launch(x, ld, vocab, rows, c, ignore_index, o, k, dx, ldd, takers, s); };
  if (bytes <= kSmallRow) return ring(launch_ring<T, POLICY, GRAD, ENT, 64, 6, 8, true>);
  if constexpr (GRAD) {
    if (bytes <= kMidRow) return ring(launch_ring<T, POLICY, GRAD, ENT, 128, 6, 4, true>);
    if constexpr (sizeof(T) == 4) {
      if (bytes > kSplitRow && bytes <= kLongRow && rows >= 4 * sm_count()) return ring(launch_split<T, ENT>);
    }
    if (bytes <= kThirdRow) return ring(launch_ring<T, POLICY, GRAD, ENT, 128, 9, 3, true>);
    if (bytes <= 7 * chunk_bytes(256)) return ring(launch_ring<T, POLICY, GRAD, ENT, 256, 7, 2, true>);
    if (bytes <= kLongRow) return ring(launch_ring<T, POLICY, GRAD, ENT, 256, 7, 2, false>);
    return ring(launch_ring<T, POLICY, GRAD, ENT, 512, 7, 1, false>);
  } else {
    if constexpr (sizeof(T) == 2) {
      if (rows >= 4 * sm_count()) return ring(launch_ring<T, POLICY, GRAD, ENT, 128, 3, 8, true>);
    }
    return ring(launch_ring<T, POLICY, GRAD, ENT, 256, 4, 3, true>);
  }
}

template <typename T>
int logprob_fwd_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                      float inv_temp, int ignore_index, float* logprob, float* entropy, float* stats, void* workspace,
                      cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  int2* list = static_cast<int2*>(workspace);
  RowOut o = {};
  o.labels = labels;
  o.logprob = logprob;
  o.entropy = entropy;
  o.stats = reinterpret_cast<float2*>(stats);
  o.status = rk_host::device_status_ptr();
  const rk_policy_terms none = {};
  int takers;
  if (entropy) return launch_rows<T, false, false, true>(x, ld, vocab, rows, inv_temp, ignore_index, o, none, nullptr, 0, list, nullptr, &takers, s);
  return launch_rows<T, false, false, false>(x, ld, vocab, rows, inv_temp, ignore_index, o, none, nullptr, 0, list, nullptr, &takers, s);
}

template <typename T>
int logprob_bwd_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                      float inv_temp, int ignore_index, const float* stats, const float* entropy,
                      const float* d_logprob, const float* d_entropy, int64_t coef_stride, float scale_by,
                      const float* scale_dev, void* dlogits, int64_t ldd, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  T* dx = static_cast<T*>(dlogits);
  const float2* st = reinterpret_cast<const float2*>(stats);
  const int64_t per = (int64_t)kBwdThreads * kBwdVecs * kPer<T>;
  const bool by_warp = vocab * (int64_t)sizeof(T) <= (rows >= 32 * sm_count() ? kBwdWarpRow : kBwdWarpOnce);
  const int64_t segments = (vocab + per - 1) / per;
  const int64_t block_rows = by_warp ? 1ll << 31 : ((1ll << 31) - 1) / segments;  // rows of one launch
  for (int64_t r = 0; r < rows; r += block_rows) {
    const int64_t n = rows - r < block_rows ? rows - r : block_rows;
    const auto launch = [&](auto kernel) {
      rk_host::launch_k(kernel, (unsigned)(by_warp ? (n + 7) / 8 : n * segments), kBwdThreads, 0, s, x + r * ld, ld, (int)vocab, n,
                        (int)segments, labels + r, inv_temp, ignore_index, st + r, d_entropy ? entropy + r : nullptr,
                        d_logprob + r * coef_stride, d_entropy ? d_entropy + r * coef_stride : nullptr, coef_stride, scale_by,
                        scale_dev, dx + r * ldd, ldd);
    };
    if (by_warp) d_entropy ? launch(logprob_bwd_kernel<T, true, true>) : launch(logprob_bwd_kernel<T, false, true>);
    else d_entropy ? launch(logprob_bwd_kernel<T, true, false>) : launch(logprob_bwd_kernel<T, false, false>);
    const int e = rk_host::launch_status();
    if (e) return e;
  }
  return RK_OK;
}

template <typename T>
int policy_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* actions, int64_t rows, int ignore_index,
                 const rk_policy_terms& k, float* logprob, float* kl, float* entropy, float* metrics, float* stats,
                 float* coef, void* dlogits, int64_t ldd, void* workspace, cudaStream_t s) {
  float* denom = static_cast<float*>(workspace);
  double* weights = reinterpret_cast<double*>(denom + 4);
  double2* sums = reinterpret_cast<double2*>(weights + kMaxWeights);
  float4* fine = reinterpret_cast<float4*>(sums + rows);
  float2* parts = reinterpret_cast<float2*>(fine + rows);
  int2* list = reinterpret_cast<int2*>(parts + rows);
  int takers = 0;  // at most one a row
  int st = RK_OK;
  if (rows > 0) {
    const T* x = static_cast<const T*>(logits);
    T* dx = static_cast<T*>(dlogits);
    RowOut o = {};
    o.labels = actions;
    o.logprob = logprob;
    o.entropy = entropy;
    o.kl = kl;
    o.stats = reinterpret_cast<float2*>(stats);
    o.coef = reinterpret_cast<float2*>(coef);
    o.parts = parts;
    o.fine = fine;
    o.sums = sums;
    o.denom = denom;
    o.status = rk_host::device_status_ptr();
    const float t = k.inv_temp;
    if (entropy)
      st = dx ? launch_rows<T, true, true, true>(x, ld, vocab, rows, t, ignore_index, o, k, dx, ldd, list, weights, &takers, s)
              : launch_rows<T, true, false, true>(x, ld, vocab, rows, t, ignore_index, o, k, dx, ldd, list, weights, &takers, s);
    else
      st = dx ? launch_rows<T, true, true, false>(x, ld, vocab, rows, t, ignore_index, o, k, dx, ldd, list, weights, &takers, s)
              : launch_rows<T, true, false, false>(x, ld, vocab, rows, t, ignore_index, o, k, dx, ldd, list, weights, &takers, s);
    if (st) return st;
  }
  // without rows the denominator was not formed: the kernel takes it as 0
  rk_host::launch_k(policy_reduce_kernel, 1, 256, 0, s, sums, takers, rows > 0 ? denom : nullptr, metrics);
  return rk_host::launch_status();
}

}  // namespace

extern "C" int64_t rk_token_logprob_workspace(int64_t rows) {
  return rows > kFewRows && rows <= kListRows ? rows * 8 : 0;
}

extern "C" int rk_token_logprob_fwd(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                                    float inv_temp, int ignore_index, int dtype, float* logprob, float* entropy,
                                    float* stats, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!shape_ok(ld, vocab, rows)) return RK_ERR_ARG;
  if (!rk_host::dtype_ok(dtype)) return RK_ERR_DTYPE;
  if (rows == 0) return RK_OK;
  const int64_t need = rk_token_logprob_workspace(rows);
  if (!logits || !labels || !logprob || (need && !workspace)) return RK_ERR_ARG;
  if (workspace_bytes < need) return RK_ERR_WORKSPACE;
  if (!rk_host::aligned(stats, 8) || !rk_host::aligned(workspace, 8)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RK_F32: return logprob_fwd_typed<float>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, logprob, entropy, stats, workspace, s);
    case RK_BF16: return logprob_fwd_typed<__nv_bfloat16>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, logprob, entropy, stats, workspace, s);
    default: return logprob_fwd_typed<__half>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, logprob, entropy, stats, workspace, s);
  }
}

extern "C" int rk_token_logprob_bwd(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                                    float inv_temp, int ignore_index, int dtype, const float* stats,
                                    const float* entropy, const float* d_logprob, const float* d_entropy,
                                    int64_t coef_stride, const float* scale_dev, void* dlogits, int64_t ldd,
                                    void* stream) {
  if (!shape_ok(ld, vocab, rows) || ldd < vocab || coef_stride < 1 || (!entropy) != (!d_entropy)) return RK_ERR_ARG;
  if (!rk_host::dtype_ok(dtype)) return RK_ERR_DTYPE;
  if (rows == 0) return RK_OK;
  if (!logits || !labels || !stats || !d_logprob || !dlogits) return RK_ERR_ARG;
  if (!rk_host::aligned(stats, 8)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RK_F32: return logprob_bwd_typed<float>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, 1.f, scale_dev, dlogits, ldd, s);
    case RK_BF16: return logprob_bwd_typed<__nv_bfloat16>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, 1.f, scale_dev, dlogits, ldd, s);
    default: return logprob_bwd_typed<__half>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, 1.f, scale_dev, dlogits, ldd, s);
  }
}

// Four scalars, the sums of weights and of losses, what the rows' losses are finished from, and room for the rows' list.
extern "C" int64_t rk_policy_workspace(int64_t rows) { return 16 + kMaxWeights * 8 + (rows > 0 ? rows : 0) * 48; }

extern "C" int rk_policy_loss(const void* logits, int64_t ld, int64_t vocab, const int64_t* actions, int64_t rows,
                              int ignore_index, int dtype, const rk_policy_terms* terms, float* logprob, float* kl,
                              float* entropy, float* metrics, float* stats, float* coef, void* dlogits, int64_t ldd,
                              void* workspace, int64_t workspace_bytes, void* stream) {
  if (!shape_ok(ld, vocab, rows) || !terms || !metrics || !workspace || terms->adv_group < 1 ||
      (dlogits && ldd < vocab) || (terms->entropy_coef != 0.f && !entropy && rows > 0))
    return RK_ERR_ARG;
  if (rows > 0 && (!logits || !actions || !logprob || !terms->old_logprobs || !terms->advantages)) return RK_ERR_ARG;
  if (!rk_host::dtype_ok(dtype)) return RK_ERR_DTYPE;
  if (workspace_bytes < rk_policy_workspace(rows)) return RK_ERR_WORKSPACE;
  if (!rk_host::aligned(workspace, 16) || !rk_host::aligned(stats, 8) || !rk_host::aligned(coef, 8)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RK_F32: return policy_typed<float>(logits, ld, vocab, actions, rows, ignore_index, *terms, logprob, kl, entropy, metrics, stats, coef, dlogits, ldd, workspace, s);
    case RK_BF16: return policy_typed<__nv_bfloat16>(logits, ld, vocab, actions, rows, ignore_index, *terms, logprob, kl, entropy, metrics, stats, coef, dlogits, ldd, workspace, s);
    default: return policy_typed<__half>(logits, ld, vocab, actions, rows, ignore_index, *terms, logprob, kl, entropy, metrics, stats, coef, dlogits, ldd, workspace, s);
  }
}

namespace {

template <typename T>
int preference_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t pairs, int64_t length,
                     int ignore_index, int dtype, const rk_preference_terms& k, float* logprob, float* rewards, float* loss,
                     float* stats, float* coef, void* dlogits, int64_t ldd, void* workspace, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  float2* st = reinterpret_cast<float2*>(stats);
  const int64_t rows = 2 * pairs * length;
  float* pair_loss = static_cast<float*>(workspace);
  int e = rows ? logprob_fwd_typed<T>(logits, ld, vocab, labels, rows, k.inv_temp, ignore_index, logprob, nullptr, stats,
                                        pair_loss + ((pairs + 3) & ~(int64_t)3), s)
               : RK_OK;
  if (e) return e;
  rk_host::launch_k(preference_pair_kernel<T>, (unsigned)pairs, length > kShortPair ? 1024 : 256, 0, s, x, ld, labels, pairs, length, (int)vocab,
                    ignore_index, k, st, rewards, pair_loss, loss, coef);
  if ((e = rk_host::launch_status())) return e;
  if (pairs > 1) {  // a single pair's loss is the mean already
    rk_host::launch_k(preference_reduce_kernel, 1, 256, 0, s, pair_loss, pairs, loss);
    if ((e = rk_host::launch_status())) return e;
  }
  if (!dlogits || !rows) return RK_OK;
  return logprob_bwd_typed<T>(logits, ld, vocab, labels, rows, k.inv_temp, ignore_index, stats, nullptr, coef, nullptr, 1,
                              k.grad_scale, k.grad_scale_dev, dlogits, ldd, s);
}

}  // namespace

extern "C" int64_t rk_preference_workspace(int64_t pairs, int64_t length) {
  return pairs > 0 && length >= 0 ? 16 + pairs * 4 + rk_token_logprob_workspace(2 * pairs * length) : 0;
}

extern "C" int rk_preference_loss(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t pairs,
                                  int64_t length, int ignore_index, int dtype, const rk_preference_terms* terms,
                                  float* logprob, float* rewards, float* loss, float* stats, float* coef,
                                  void* dlogits, int64_t ldd, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (pairs < 1 || length < 0 || length >= (1ll << 30) || pairs >= (1ll << 31) || !shape_ok(ld, vocab, 2 * pairs * length) ||
      !terms || !rewards || !loss || !workspace || terms->kind < RK_PREF_SIGMOID || terms->kind > RK_PREF_SQUARED ||
      (dlogits && ldd < vocab))
    return RK_ERR_ARG;
  const int64_t rows = 2 * pairs * length;
  if (rows > 0 && (!logits || !labels || !logprob || !stats || !coef)) return RK_ERR_ARG;
  if (!rk_host::dtype_ok(dtype)) return RK_ERR_DTYPE;
  if (workspace_bytes < rk_preference_workspace(pairs, length)) return RK_ERR_WORKSPACE;
  if (!rk_host::aligned(workspace, 16) || !rk_host::aligned(stats, 8)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RK_F32: return preference_typed<float>(logits, ld, vocab, labels, pairs, length, ignore_index, dtype, *terms, logprob, rewards, loss, stats, coef, dlogits, ldd, workspace, s);
    case RK_BF16: return preference_typed<__nv_bfloat16>(logits, ld, vocab, labels, pairs, length, ignore_index, dtype, *terms, logprob, rewards, loss, stats, coef, dlogits, ldd, workspace, s);
    default: return preference_typed<__half>(logits, ld, vocab, labels, pairs, length, ignore_index, dtype, *terms, logprob, rewards, loss, stats, coef, dlogits, ldd, workspace, s);
  }
}
