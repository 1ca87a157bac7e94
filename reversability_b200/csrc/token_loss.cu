// Losses on token log-probabilities: the log-probabilities and entropies
// themselves, the clipped policy loss with a KL term, and the paired preference
// loss, each with the gradient of the logits.
//
// A row's softmax is carried as (m, s, w): m = max z, s = sum exp(z - m),
// w = sum exp(z - m)(z - m), merged online; then ln p_j = (z_j - m) - ln s and
// the entropy is ln s - w / s. Keeping m and ln s apart (not their sum) keeps
// ln p exact to fp32 when the logits are large. z = x * inv_temp in fp32; the
// gradient is rounded once, when it is stored.
#include "vec.cuh"

namespace rk {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct RowSum {
  float m, s, w;
};

// Online merge of two partial sums; a part whose maximum is -inf is empty.
template <bool ENT>
__device__ __forceinline__ RowSum merge_rows(const RowSum& a, const RowSum& b) {
  RowSum r;
  r.m = fmaxf(a.m, b.m);
  if (a.m != a.m || b.m != b.m) r.m = NAN;  // fmaxf drops a NaN
  if (r.m == -INFINITY) return {-INFINITY, 0.f, 0.f};
  const float da = a.m == -INFINITY ? 0.f : a.m - r.m, db = b.m == -INFINITY ? 0.f : b.m - r.m;
  const float fa = a.m == -INFINITY ? 0.f : ex2_approx(da * kLog2e), fb = b.m == -INFINITY ? 0.f : ex2_approx(db * kLog2e);
  r.s = fmaf(a.s, fa, b.s * fb);
  // a part whose factor is 0 lies too far below to count (and da * s may overflow there)
  r.w = ENT ? (fa > 0.f ? fmaf(da, a.s, a.w) * fa : 0.f) + (fb > 0.f ? fmaf(db, b.s, b.w) * fb : 0.f) : 0.f;
  return r;
}

template <bool ENT>
__device__ __forceinline__ RowSum warp_merge(RowSum v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const RowSum u = {__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o),
                      ENT ? __shfl_xor_sync(0xffffffffu, v.w, o) : 0.f};
    v = merge_rows<ENT>(v, u);
  }
  return v;
}

enum { ROW_LIVE = 0, ROW_IGNORED = 1, ROW_BAD = 2 };
__device__ __forceinline__ int row_kind(int64_t label, int vocab, int ignore_index) {
  if (label == ignore_index) return ROW_IGNORED;
  return label < 0 || label >= vocab ? ROW_BAD : ROW_LIVE;
}

// The row's sums over a whole CTA (every thread returns them).
template <typename T, bool ENT>
__device__ RowSum block_row_sum(const T* __restrict__ x, int vocab, float inv_temp, RowSum* sm) {
  RowSum a = {-INFINITY, 0.f, 0.f};
  for (int c = threadIdx.x; c < vocab; c += blockDim.x)
    a = merge_rows<ENT>(a, {Dt<T>::to_f(x[c]) * inv_temp, 1.f, 0.f});
  a = warp_merge<ENT>(a);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) sm[warp] = a;
  __syncthreads();
  RowSum r = lane < (int)(blockDim.x >> 5) ? sm[lane] : RowSum{-INFINITY, 0.f, 0.f};
  r = warp_merge<ENT>(r);
  __syncthreads();
  return r;
}

// Writes one row of gradients: g_lp ([j = label] - p_j) - g_h p_j (ln p_j + entropy), both factors already
// times inv_temp and the outer scale.
template <typename T, bool ENT>
__device__ void block_row_grad(const T* x, T* dx, int vocab, int label, float inv_temp, float m, float ln_s,
                               float entropy, float g_lp, float g_h) {
  for (int c = threadIdx.x; c < vocab; c += blockDim.x) {
    const float lp = (Dt<T>::to_f(x[c]) * inv_temp - m) - ln_s;
    const float p = ex2_approx(lp * kLog2e);
    float d = (c == label ? g_lp : 0.f) - g_lp * p;
    if (ENT && p > 0.f) d -= g_h * p * (lp + entropy);  // p = 0 has lp = -inf
    dx[c] = Dt<T>::from_f(d);
  }
}
template <typename T>
__device__ void block_row_zero(T* dx, int vocab) {
  for (int c = threadIdx.x; c < vocab; c += blockDim.x) dx[c] = Dt<T>::from_f(0.f);
}

// ---------------------------------------------------------------- token log-probabilities
template <typename T, bool ENT>
__global__ void __launch_bounds__(512) logprob_fwd_kernel(const T* __restrict__ logits, int64_t ld, int vocab,
                                                          const int64_t* __restrict__ labels, float inv_temp,
                                                          int ignore_index, float* __restrict__ logprob,
                                                          float* __restrict__ entropy, float2* __restrict__ stats,
                                                          unsigned int* status) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ RowSum sm[32];
  const int64_t row = blockIdx.x;
  const int64_t label = labels[row];
  const int kind = row_kind(label, vocab, ignore_index);
  if (kind != ROW_LIVE) {
    if (threadIdx.x == 0) {
      if (kind == ROW_BAD) flag_error(status, RK_DEV_CE_LABEL);
      logprob[row] = 0.f;
      if (entropy) entropy[row] = 0.f;
      if (stats) stats[row] = {0.f, 0.f};
    }
    return;
  }
  const T* x = logits + row * ld;
  const RowSum r = block_row_sum<T, ENT>(x, vocab, inv_temp, sm);
  if (threadIdx.x == 0) {
    const float ln_s = logf(r.s);
    logprob[row] = (Dt<T>::to_f(x[label]) * inv_temp - r.m) - ln_s;
    if (ENT) entropy[row] = ln_s - r.w / r.s;
    if (stats) stats[row] = {r.m, ln_s};
  }
}

template <typename T, bool ENT>
__global__ void __launch_bounds__(512)
    logprob_bwd_kernel(const T* logits, int64_t ld, int vocab, const int64_t* __restrict__ labels, float inv_temp,
                       int ignore_index, const float2* __restrict__ stats, const float* __restrict__ entropy,
                       const float* __restrict__ d_logprob, const float* __restrict__ d_entropy, int64_t coef_stride,
                       const float* __restrict__ scale_dev, T* dlogits, int64_t ldd) {
  pdl_wait();  // inputs are the previous kernel's outputs
  const int64_t row = blockIdx.x;
  const int64_t label = labels[row];
  T* dx = dlogits + row * ldd;
  if (row_kind(label, vocab, ignore_index) != ROW_LIVE) {
    block_row_zero(dx, vocab);
    return;
  }
  const float scale = inv_temp * (scale_dev ? *scale_dev : 1.f);
  const float2 st = stats[row];
  block_row_grad<T, ENT>(logits + row * ld, dx, vocab, (int)label, inv_temp, st.x, st.y, ENT ? entropy[row] : 0.f,
                         d_logprob[row * coef_stride] * scale, ENT ? d_entropy[row * coef_stride] * scale : 0.f);
}

// ---------------------------------------------------------------- policy loss
// workspace: [0] the denominator, then per row (w l, w clipped)
struct PolicyRow {
  float lp, kl, loss, clipped, g_lp, g_h;  // g_* without the outer scale and inv_temp
};
__device__ __forceinline__ PolicyRow policy_row(const rk_policy_terms& k, int64_t row, float lp, float entropy,
                                                float inv_d) {
  PolicyRow o;
  const float adv = k.advantages[row / k.adv_group];
  const float w = k.weights ? k.weights[row] : 1.f;
  const float ratio = expf(lp - k.old_logprobs[row]);
  const float free = ratio * adv, held = fminf(fmaxf(ratio, 1.f - k.clip_low), 1.f + k.clip_high) * adv;
  const bool clipped = held < free;
  float kl = 0.f, dkl = 0.f;
  if (k.ref_logprobs) {
    const float drift = k.ref_logprobs[row] - lp;
    const float em1 = expm1f(drift);
    kl = em1 - drift;
    dkl = -em1;
  }
  o.lp = lp;
  o.kl = kl;
  o.loss = w * (k.kl_coef * kl - (clipped ? held : free) - k.entropy_coef * entropy);
  o.clipped = clipped ? w : 0.f;
  o.g_lp = w * inv_d * ((clipped ? 0.f : -free) + k.kl_coef * dkl);
  o.g_h = -w * inv_d * k.entropy_coef;
  return o;
}

__device__ double block_sum(double v) {
  __shared__ double red[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) s += red[w];
  __syncthreads();
  return s;
}

__global__ void __launch_bounds__(1024) policy_prepare_kernel(const int64_t* __restrict__ actions, int64_t rows,
                                                              int vocab, int ignore_index, rk_policy_terms k,
                                                              float* __restrict__ denom) {
  pdl_wait();  // inputs are the previous kernel's outputs
  double s = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x)
    if (row_kind(actions[r], vocab, ignore_index) == ROW_LIVE) s += k.weights ? (double)k.weights[r] : 1.0;
  s = block_sum(s);
  if (threadIdx.x == 0) *denom = k.denominator ? *k.denominator : (float)s;
}

template <typename T, bool ENT>
__global__ void __launch_bounds__(512)
    policy_row_kernel(const T* logits, int64_t ld, int vocab, const int64_t* __restrict__ actions, int ignore_index,
                      rk_policy_terms k, const float* __restrict__ denom, float2* __restrict__ parts,
                      float* __restrict__ logprob, float* __restrict__ kl, float* __restrict__ entropy,
                      float2* __restrict__ stats, float2* __restrict__ coef, T* dlogits, int64_t ldd,
                      unsigned int* status) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ RowSum sm[32];
  const int64_t row = blockIdx.x;
  const int64_t label = actions[row];
  const int kind = row_kind(label, vocab, ignore_index);
  if (kind != ROW_LIVE) {
    if (threadIdx.x == 0) {
      if (kind == ROW_BAD) flag_error(status, RK_DEV_CE_LABEL);
      logprob[row] = 0.f;
      parts[row] = {0.f, 0.f};
      if (kl) kl[row] = 0.f;
      if (entropy) entropy[row] = 0.f;
      if (stats) stats[row] = {0.f, 0.f};
      if (coef) coef[row] = {0.f, 0.f};
    }
    if (dlogits) block_row_zero(dlogits + row * ldd, vocab);
    return;
  }
  const T* x = logits + row * ld;
  const float zl = Dt<T>::to_f(x[label]) * k.inv_temp;
  const RowSum r = block_row_sum<T, ENT>(x, vocab, k.inv_temp, sm);
  const float ln_s = logf(r.s), h = ENT ? ln_s - r.w / r.s : 0.f;
  const float d = *denom;
  const PolicyRow o = policy_row(k, row, (zl - r.m) - ln_s, h, d != 0.f ? 1.f / d : 0.f);
  if (threadIdx.x == 0) {
    logprob[row] = o.lp;
    parts[row] = {o.loss, o.clipped};
    if (kl) kl[row] = o.kl;
    if (ENT) entropy[row] = h;
    if (stats) stats[row] = {r.m, ln_s};
    if (coef) coef[row] = {o.g_lp, o.g_h};
  }
  if (dlogits) {
    const float scale = k.inv_temp * k.grad_scale * (k.grad_scale_dev ? *k.grad_scale_dev : 1.f);
    block_row_grad<T, ENT>(x, dlogits + row * ldd, vocab, (int)label, k.inv_temp, r.m, ln_s, h, o.g_lp * scale,
                           o.g_h * scale);
  }
}

__global__ void __launch_bounds__(1024) policy_reduce_kernel(const float2* __restrict__ parts, int64_t rows,
                                                             const float* __restrict__ denom,
                                                             float* __restrict__ metrics) {
  pdl_wait();  // inputs are the previous kernel's outputs
  double a = 0.0, b = 0.0;
  for (int64_t r = threadIdx.x; r < rows; r += blockDim.x) {
    const float2 v = parts[r];
    a += v.x;
    b += v.y;
  }
  a = block_sum(a);
  b = block_sum(b);
  if (threadIdx.x == 0) {
    const float d = *denom;
    const double inv = d != 0.f ? 1.0 / d : 0.0;
    metrics[0] = (float)(a * inv);
    metrics[1] = d;
    metrics[2] = (float)(b * inv);
    metrics[3] = 0.f;
  }
}

// ---------------------------------------------------------------- preference loss
// One CTA per pair: the two sequences' gaps in a fixed order, the pair's loss and its rows' factors.
__global__ void __launch_bounds__(256)
    preference_pair_kernel(const int64_t* __restrict__ labels, int64_t pairs, int64_t length, int vocab,
                           int ignore_index, rk_preference_terms k, const float* __restrict__ logprob,
                           float* __restrict__ rewards, float* __restrict__ pair_loss, float* __restrict__ coef) {
  pdl_wait();  // inputs are the previous kernel's outputs
  const int64_t pair = blockIdx.x;
  double gap[2], count[2];
  for (int side = 0; side < 2; ++side) {
    const int64_t base = (side * pairs + pair) * length;
    double g = 0.0, n = 0.0;
    for (int64_t t = threadIdx.x; t < length; t += blockDim.x) {
      if (row_kind(labels[base + t], vocab, ignore_index) != ROW_LIVE) continue;
      g += (double)logprob[base + t] - (k.ref_logprobs ? (double)k.ref_logprobs[base + t] : 0.0);
      n += 1.0;
    }
    gap[side] = block_sum(g);
    count[side] = block_sum(n);
    if (k.average) gap[side] /= fmax(count[side], 1.0);
  }
  const float diff = (float)(gap[0] - gap[1]);
  const float u = k.beta * diff;
  float loss, slope;  // slope = dloss/d(gap_chosen)
  if (k.kind == RK_PREF_SIGMOID) {
    const float tail = log1pf(expf(-fabsf(u)));
    loss = (1.f - k.smoothing) * (fmaxf(-u, 0.f) + tail) + k.smoothing * (fmaxf(u, 0.f) + tail);
    slope = k.beta * (k.smoothing / (1.f + expf(-u)) - (1.f - k.smoothing) / (1.f + expf(u)));
  } else if (k.kind == RK_PREF_HINGE) {
    loss = fmaxf(1.f - u, 0.f);
    slope = u < 1.f ? -k.beta : 0.f;
  } else {
    const float off = diff - 0.5f / k.beta;
    loss = off * off;
    slope = 2.f * off;
  }
  slope /= (float)pairs;
  if (threadIdx.x == 0) {
    pair_loss[pair] = loss;
    rewards[pair] = k.beta * (float)gap[0];
    rewards[pairs + pair] = k.beta * (float)gap[1];
  }
  for (int side = 0; side < 2; ++side) {
    const int64_t base = (side * pairs + pair) * length;
    const float s = (side ? -slope : slope) / (k.average ? (float)fmax(count[side], 1.0) : 1.f);
    for (int64_t t = threadIdx.x; t < length; t += blockDim.x)
      coef[base + t] = row_kind(labels[base + t], vocab, ignore_index) == ROW_LIVE ? s : 0.f;
  }
}

// loss = mean of the pair losses; scale_out = grad_scale * (*grad_scale_dev) for the gradient pass.
__global__ void __launch_bounds__(256) preference_reduce_kernel(const float* __restrict__ pair_loss, int64_t pairs,
                                                                rk_preference_terms k, float* __restrict__ loss,
                                                                float* __restrict__ scale_out) {
  pdl_wait();  // inputs are the previous kernel's outputs
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < pairs; i += blockDim.x) s += pair_loss[i];
  s = block_sum(s);
  if (threadIdx.x == 0) {
    *loss = (float)(s / (double)pairs);
    *scale_out = k.grad_scale * (k.grad_scale_dev ? *k.grad_scale_dev : 1.f);
  }
}

}  // namespace rk

using namespace rk;

namespace {

bool shape_ok(int64_t ld, int64_t vocab, int64_t rows) {
  return rows >= 0 && rows < (1ll << 31) && vocab > 0 && vocab < (1ll << 31) && ld >= vocab;
}

template <typename T>
int logprob_fwd_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                      float inv_temp, int ignore_index, float* logprob, float* entropy, float* stats,
                      cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  float2* st = reinterpret_cast<float2*>(stats);
  unsigned int* status = rk_host::device_status_ptr();
  if (entropy)
    rk_host::launch_k(logprob_fwd_kernel<T, true>, (unsigned)rows, 512, 0, s, x, ld, (int)vocab, labels, inv_temp,
                      ignore_index, logprob, entropy, st, status);
  else
    rk_host::launch_k(logprob_fwd_kernel<T, false>, (unsigned)rows, 512, 0, s, x, ld, (int)vocab, labels, inv_temp,
                      ignore_index, logprob, entropy, st, status);
  return rk_host::launch_status();
}

template <typename T>
int logprob_bwd_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                      float inv_temp, int ignore_index, const float* stats, const float* entropy,
                      const float* d_logprob, const float* d_entropy, int64_t coef_stride, const float* scale_dev,
                      void* dlogits, int64_t ldd, cudaStream_t s) {
  const T* x = static_cast<const T*>(logits);
  T* dx = static_cast<T*>(dlogits);
  const float2* st = reinterpret_cast<const float2*>(stats);
  if (d_entropy)
    rk_host::launch_k(logprob_bwd_kernel<T, true>, (unsigned)rows, 512, 0, s, x, ld, (int)vocab, labels, inv_temp,
                      ignore_index, st, entropy, d_logprob, d_entropy, coef_stride, scale_dev, dx, ldd);
  else
    rk_host::launch_k(logprob_bwd_kernel<T, false>, (unsigned)rows, 512, 0, s, x, ld, (int)vocab, labels, inv_temp,
                      ignore_index, st, entropy, d_logprob, d_entropy, coef_stride, scale_dev, dx, ldd);
  return rk_host::launch_status();
}

template <typename T>
int policy_typed(const void* logits, int64_t ld, int64_t vocab, const int64_t* actions, int64_t rows, int ignore_index,
                 const rk_policy_terms& k, float* logprob, float* kl, float* entropy, float* metrics, float* stats,
                 float* coef, void* dlogits, int64_t ldd, void* workspace, cudaStream_t s) {
  float* denom = static_cast<float*>(workspace);
  float2* parts = reinterpret_cast<float2*>(denom + 4);
  rk_host::launch_k(policy_prepare_kernel, 1, 1024, 0, s, actions, rows, (int)vocab, ignore_index, k, denom);
  int st = rk_host::launch_status();
  if (st) return st;
  if (rows > 0) {
    const T* x = static_cast<const T*>(logits);
    T* dx = static_cast<T*>(dlogits);
    float2 *S = reinterpret_cast<float2*>(stats), *C = reinterpret_cast<float2*>(coef);
    unsigned int* status = rk_host::device_status_ptr();
    if (entropy)
      rk_host::launch_k(policy_row_kernel<T, true>, (unsigned)rows, 512, 0, s, x, ld, (int)vocab, actions, ignore_index, k,
                        denom, parts, logprob, kl, entropy, S, C, dx, ldd, status);
    else
      rk_host::launch_k(policy_row_kernel<T, false>, (unsigned)rows, 512, 0, s, x, ld, (int)vocab, actions, ignore_index,
                        k, denom, parts, logprob, kl, entropy, S, C, dx, ldd, status);
    st = rk_host::launch_status();
    if (st) return st;
  }
  rk_host::launch_k(policy_reduce_kernel, 1, 1024, 0, s, parts, rows, denom, metrics);
  return rk_host::launch_status();
}

}  // namespace

extern "C" int rk_token_logprob_fwd(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t rows,
                                    float inv_temp, int ignore_index, int dtype, float* logprob, float* entropy,
                                    float* stats, void* stream) {
  if (!shape_ok(ld, vocab, rows)) return RK_ERR_ARG;
  if (!rk_host::dtype_ok(dtype)) return RK_ERR_DTYPE;
  if (rows == 0) return RK_OK;
  if (!logits || !labels || !logprob) return RK_ERR_ARG;
  if (!rk_host::aligned(stats, 8)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case RK_F32: return logprob_fwd_typed<float>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, logprob, entropy, stats, s);
    case RK_BF16: return logprob_fwd_typed<__nv_bfloat16>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, logprob, entropy, stats, s);
    default: return logprob_fwd_typed<__half>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, logprob, entropy, stats, s);
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
    case RK_F32: return logprob_bwd_typed<float>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, scale_dev, dlogits, ldd, s);
    case RK_BF16: return logprob_bwd_typed<__nv_bfloat16>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, scale_dev, dlogits, ldd, s);
    default: return logprob_bwd_typed<__half>(logits, ld, vocab, labels, rows, inv_temp, ignore_index, stats, entropy, d_logprob, d_entropy, coef_stride, scale_dev, dlogits, ldd, s);
  }
}

extern "C" int64_t rk_policy_workspace(int64_t rows) { return 16 + (rows > 0 ? rows : 0) * 8; }

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

extern "C" int64_t rk_preference_workspace(int64_t pairs, int64_t length) {
  (void)length;
  return 16 + (pairs > 0 ? pairs : 0) * 4;
}

extern "C" int rk_preference_loss(const void* logits, int64_t ld, int64_t vocab, const int64_t* labels, int64_t pairs,
                                  int64_t length, int ignore_index, int dtype, const rk_preference_terms* terms,
                                  float* logprob, float* rewards, float* loss, float* stats, float* coef,
                                  void* dlogits, int64_t ldd, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  if (pairs < 1 || length < 0 || length >= (1ll << 31) || pairs >= (1ll << 31) || !shape_ok(ld, vocab, 2 * pairs * length) ||
      !terms || !rewards || !loss || !workspace || terms->kind < RK_PREF_SIGMOID || terms->kind > RK_PREF_SQUARED ||
      (dlogits && ldd < vocab))
    return RK_ERR_ARG;
  const int64_t rows = 2 * pairs * length;
  if (rows > 0 && (!logits || !labels || !logprob || !stats || !coef)) return RK_ERR_ARG;
  if (!rk_host::dtype_ok(dtype)) return RK_ERR_DTYPE;
  if (workspace_bytes < rk_preference_workspace(pairs, length)) return RK_ERR_WORKSPACE;
  if (!rk_host::aligned(workspace, 16) || !rk_host::aligned(stats, 8) || !rk_host::aligned(coef, 8)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  float* scale = static_cast<float*>(workspace);
  float* pair_loss = scale + 4;
  int st = rk_token_logprob_fwd(logits, ld, vocab, labels, rows, terms->inv_temp, ignore_index, dtype, logprob, nullptr,
                                stats, stream);
  if (st) return st;
  rk_host::launch_k(preference_pair_kernel, (unsigned)pairs, 256, 0, s, labels, pairs, length, (int)vocab, ignore_index, *terms,
                    logprob, rewards, pair_loss, coef);
  if ((st = rk_host::launch_status())) return st;
  rk_host::launch_k(preference_reduce_kernel, 1, 256, 0, s, pair_loss, pairs, *terms, loss, scale);
  if ((st = rk_host::launch_status())) return st;
  if (!dlogits) return RK_OK;
  return rk_token_logprob_bwd(logits, ld, vocab, labels, rows, terms->inv_temp, ignore_index, dtype, stats, nullptr,
                              coef, nullptr, 1, scale, dlogits, ldd, stream);
}
