// AdamW over a list of separate tensors, moments in 32 or 8 bits (the update of
// optim.cu for a module's own parameters and gradients instead of one flat
// buffer; Loshchilov & Hutter's decoupled weight decay).
//
// Per element, with the step's constants from the device scalar block:
//   g' = g c;  p1 = p (1 - lr wd);  m' = m + (1 - b1)(g' - m)
//   v' = b2 v + (1 - b2) g'^2;      p2 = p1 - a m' / (sqrt(v') / s + eps)
// a = lr / (1 - b1^t), s = sqrt(1 - b2^t). All in fp32; p and g are rounded only
// when they are stored in a 16-bit type.
//
// 8-bit moments are block-wise (256 elements, one scale; Dettmers et al., "8-bit
// Optimizers via Block-wise Quantization"), in power codes instead of a table:
// m ~ M c|c| / 127^2 and sqrt(v) ~ R c^2 / 255^2. A power code needs one square
// root to write and one product to read, is exact at the block's largest value,
// and its relative step 2/c narrows towards it. Simulated over 4000 steps
// (gradients whose scale spreads log-normally by 1 within a block), the second
// moment's root stays within 4 % (beta2 0.95) and 9 % (0.999) rms of the 32-bit
// one with mean 1.00, against 8 % and 16 % for a float8 (e4m3) code of the root.
// Code 0 of v would leave eps alone under m, so v > 0 is never stored as 0.
//
// The tensor table travels as a kernel parameter: no host-to-device copy, no
// device allocation, and a captured graph replays it.
#include "vec.cuh"

namespace rk {

constexpr int kMultiCap = 64;       // tensors per launch: 64 x 56 bytes, below the 4 KB of a kernel's parameters
constexpr int kQBlock = 256;        // elements that share a scale
constexpr int kChunk = 2048;        // elements per CTA: 8 warps, one scale block each
constexpr int kMultiNormBlocks = 592;

struct MultiTable {
  rk_adamw_tensor t[kMultiCap];
  int n;
  int64_t chunks;
};

// The tensor that holds chunk `c` of the launch, and the chunk's number within it.
__device__ __forceinline__ int find_tensor(const MultiTable& tab, int64_t& c) {
  int i = 0;
  while (i + 1 < tab.n) {
    const int64_t k = (tab.t[i].numel + kChunk - 1) / kChunk;
    if (c < k) break;
    c -= k;
    ++i;
  }
  return i;
}

__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four consecutive elements at `at`, those past n as zero; `vec` says that the tensor's base is aligned for it.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t at, int64_t n, bool vec, float (&v)[4]) {
  if (vec && at + 3 < n) {
    load_vec<T, 4>(p + at, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = at + e < n ? Dt<T>::to_f(p[at + e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t at, int64_t n, bool vec, const float (&v)[4]) {
  if (vec && at + 3 < n) {
    store_vec<T, 4>(p + at, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (at + e < n) p[at + e] = Dt<T>::from_f(v[e]);
  }
}
__device__ __forceinline__ uint32_t load4_codes(const void* p, int64_t at, int64_t n, bool vec) {
  const uint8_t* q = static_cast<const uint8_t*>(p) + at;
  if (vec && at + 3 < n) return *reinterpret_cast<const uint32_t*>(q);
  uint32_t w = 0;
  for (int e = 0; e < 4; ++e)
    if (at + e < n) w |= (uint32_t)q[e] << (8 * e);
  return w;
}
__device__ __forceinline__ void store4_codes(void* p, int64_t at, int64_t n, bool vec, uint32_t w) {
  uint8_t* q = static_cast<uint8_t*>(p) + at;
  if (vec && at + 3 < n) {
    *reinterpret_cast<uint32_t*>(q) = w;
    return;
  }
  for (int e = 0; e < 4; ++e)
    if (at + e < n) q[e] = (uint8_t)(w >> (8 * e));
}
// Byte e of a code word as a float, by placing it in the mantissa of 2^23 (one PRMT and one add;
// conversion instructions run at a quarter of that rate).
template <int E>
__device__ __forceinline__ float code_u8(uint32_t w) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | E)) - 8388608.f;
}
template <int E>
__device__ __forceinline__ float code_s8(uint32_t w) {  // w with the sign bits already flipped
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | E)) - 8388736.f;
}
__device__ __forceinline__ void codes_to_moments(uint32_t mc, uint32_t vc, float fm, float fv, float (&m)[4],
                                                 float (&v)[4]) {
  const uint32_t ms = mc ^ 0x80808080u;
  const float c0 = code_s8<0>(ms), c1 = code_s8<1>(ms), c2 = code_s8<2>(ms), c3 = code_s8<3>(ms);
  m[0] = c0 * fabsf(c0) * fm;
  m[1] = c1 * fabsf(c1) * fm;
  m[2] = c2 * fabsf(c2) * fm;
  m[3] = c3 * fabsf(c3) * fm;
  const float d0 = code_u8<0>(vc), d1 = code_u8<1>(vc), d2 = code_u8<2>(vc), d3 = code_u8<3>(vc);
  const float r0 = d0 * d0 * fv, r1 = d1 * d1 * fv, r2 = d2 * d2 * fv, r3 = d3 * d3 * fv;
  v[0] = r0 * r0;
  v[1] = r1 * r1;
  v[2] = r2 * r2;
  v[3] = r3 * r3;
}
// The nearest integer of |x| < 2^22 in the low bits of the result (x + 1.5 * 2^23).
__device__ __forceinline__ uint32_t round_bits(float x) { return __float_as_uint(x + 12582912.f); }
// 1/scale for the codes; a scale too small for its reciprocal gives 0, and every code of the block 0 (v: 1).
__device__ __forceinline__ float code_factor(float top, float scale) { return scale > 1e-33f ? top / scale : 0.f; }
// Largest of the warp's non-negative floats, by their bits: a NaN is the largest of all and reaches the scale.
__device__ __forceinline__ float warp_max_abs(float x) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(x) & 0x7fffffffu));
}
__device__ __forceinline__ float max_bits(float a, float b) {
  return __uint_as_float(max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(b) & 0x7fffffffu));
}

struct StepConst {
  float coef, step_size, root, decay, beta1, beta2, eps;
};

// One element: m and v become the new moments, r = sqrt(v), p the new parameter.
__device__ __forceinline__ void adamw_element(const StepConst& k, float g, float& p, float& m, float& v, float& r) {
  const float gi = g * k.coef;
  m = fmaf(1.f - k.beta1, gi - m, m);
  v = fmaf(k.beta2, v, (1.f - k.beta2) * gi * gi);
  r = sqrt_approx(v);
  p = fmaf(p, k.decay, -(k.step_size * __fdividef(m, fmaf(r, k.root, k.eps))));
}

template <typename TP, typename TG, bool Q8>
__global__ void __launch_bounds__(256) adamw_multi_kernel(const __grid_constant__ MultiTable tab,
                                                          const float* __restrict__ scalars, float beta1, float beta2,
                                                          float eps) {
  pdl_wait();  // inputs are the previous kernel's outputs
  const StepConst k = {scalars[3], scalars[4], 1.f / scalars[5], scalars[6], beta1, beta2, eps};
  int64_t c = blockIdx.x;
  const rk_adamw_tensor& t = tab.t[find_tensor(tab, c)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = t.numel;
  const int64_t block = c * (kChunk / kQBlock) + warp;  // scale block of this warp
  const int64_t base = block * kQBlock;
  if (base >= n) return;
  TP* P = static_cast<TP*>(t.p);
  const TG* G = static_cast<const TG*>(t.g);
  const bool pv = (reinterpret_cast<uintptr_t>(P) % (4 * sizeof(TP))) == 0;
  const bool gv = (reinterpret_cast<uintptr_t>(G) % (4 * sizeof(TG))) == 0;
  const uintptr_t state_bits = reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq);
  const bool sv = (state_bits % (Q8 ? 4 : 16)) == 0;
  float p[2][4], g[2][4], m[2][4], v[2][4], r[2][4];
  uint32_t mc[2], vc[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t at = base + h * 128 + lane * 4;
    load4(P, at, n, pv, p[h]);
    load4(G, at, n, gv, g[h]);
    if constexpr (Q8) {
      mc[h] = load4_codes(t.exp_avg, at, n, sv);
      vc[h] = load4_codes(t.exp_avg_sq, at, n, sv);
    } else {
      load4(static_cast<const float*>(t.exp_avg), at, n, sv, m[h]);
      load4(static_cast<const float*>(t.exp_avg_sq), at, n, sv, v[h]);
    }
  }
  if constexpr (Q8) {
    const float fm = t.exp_avg_scale[block] * (1.f / (127.f * 127.f));
    const float fv = t.exp_avg_sq_scale[block] * (1.f / (255.f * 255.f));
#pragma unroll
    for (int h = 0; h < 2; ++h) codes_to_moments(mc[h], vc[h], fm, fv, m[h], v[h]);
  }
  float mm = 0.f, rm = 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      adamw_element(k, g[h][e], p[h][e], m[h][e], v[h][e], r[h][e]);
      if constexpr (Q8) {
        mm = max_bits(mm, m[h][e]);
        rm = max_bits(rm, r[h][e]);
      }
    }
    const int64_t at = base + h * 128 + lane * 4;
    store4(P, at, n, pv, p[h]);
    if constexpr (!Q8) {
      store4(static_cast<float*>(t.exp_avg), at, n, sv, m[h]);
      store4(static_cast<float*>(t.exp_avg_sq), at, n, sv, v[h]);
    }
  }
  if constexpr (Q8) {
    mm = warp_max_abs(mm);
    rm = warp_max_abs(rm);
    const float im = code_factor(127.f * 127.f, mm), ir = code_factor(255.f * 255.f, rm);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t wm = 0, wv = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = fminf(sqrt_approx(fabsf(m[h][e]) * im), 127.f);
        const float b = fmaxf(fminf(sqrt_approx(r[h][e] * ir), 255.f), r[h][e] > 0.f ? 1.f : 0.f);
        wm |= (round_bits(copysignf(a, m[h][e])) & 0xffu) << (8 * e);
        wv |= (round_bits(b) & 0xffu) << (8 * e);
      }
      const int64_t at = base + h * 128 + lane * 4;
      store4_codes(t.exp_avg, at, n, sv, wm);
      store4_codes(t.exp_avg_sq, at, n, sv, wv);
    }
    if (lane == 0) {
      t.exp_avg_scale[block] = mm;
      t.exp_avg_sq_scale[block] = rm;
    }
  }
}

template <typename TG>
__global__ void __launch_bounds__(256) sumsq_multi_kernel(const __grid_constant__ MultiTable tab,
                                                          float* __restrict__ partial) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ float red[8];
  float s = 0.f;
  for (int64_t chunk = blockIdx.x; chunk < tab.chunks; chunk += gridDim.x) {
    int64_t c = chunk;
    const rk_adamw_tensor& t = tab.t[find_tensor(tab, c)];
    const TG* G = static_cast<const TG*>(t.g);
    const bool gv = (reinterpret_cast<uintptr_t>(G) % (4 * sizeof(TG))) == 0;
    float g[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) load4(G, c * kChunk + h * 1024 + threadIdx.x * 4, t.numel, gv, g[h]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = fmaf(g[h][e], g[h][e], s);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int w = 0; w < 8; ++w) sum += red[w];
    partial[blockIdx.x] = sum;
  }
}

// scalars as in optim.cu; without partials (no clipping) the coefficient is 1 and the norm is left at 0.
__global__ void __launch_bounds__(256) prepare_multi_kernel(const float* __restrict__ partial, int64_t parts,
                                                            float max_norm, float beta1, float beta2,
                                                            float weight_decay, float* __restrict__ scalars) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ double red[256];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < parts; i += blockDim.x) s += (double)partial[i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int w = blockDim.x / 2; w > 0; w >>= 1) {
    if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const float norm = (float)sqrt(red[0]);
    const float coef = max_norm / (norm + 1e-6f);
    const float lr = scalars[0];
    const float t = scalars[1] + 1.f;
    scalars[1] = t;
    scalars[2] = norm;
    // a NaN norm makes the coefficient NaN (fminf would turn it into 1), so that the step shows it
    scalars[3] = parts == 0 ? 1.f : (coef < 1.f || coef != coef ? coef : 1.f);
    const double bc1 = 1.0 - pow((double)beta1, (double)t);
    const double bc2 = 1.0 - pow((double)beta2, (double)t);
    scalars[4] = (float)(lr / bc1);
    scalars[5] = (float)sqrt(bc2);
    scalars[6] = 1.f - lr * weight_decay;
  }
}

template <typename TO>
__global__ void __launch_bounds__(256) moments_multi_kernel(const __grid_constant__ MultiTable tab) {
  pdl_wait();  // inputs are the previous kernel's outputs
  int64_t c = blockIdx.x;
  const rk_adamw_tensor& t = tab.t[find_tensor(tab, c)];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n = t.numel;
  const int64_t block = c * (kChunk / kQBlock) + warp;
  const int64_t base = block * kQBlock;
  if (base >= n) return;
  TO* M = static_cast<TO*>(t.p);
  TO* V = static_cast<TO*>(const_cast<void*>(t.g));
  const uintptr_t out_bits = reinterpret_cast<uintptr_t>(M) | reinterpret_cast<uintptr_t>(V);
  const bool ov = (out_bits % (4 * sizeof(TO))) == 0;
  const uintptr_t state_bits = reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq);
  const bool sv = (state_bits % 4) == 0;
  const float fm = t.exp_avg_scale[block] * (1.f / (127.f * 127.f));
  const float fv = t.exp_avg_sq_scale[block] * (1.f / (255.f * 255.f));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t at = base + h * 128 + lane * 4;
    float m[4], v[4];
    codes_to_moments(load4_codes(t.exp_avg, at, n, sv), load4_codes(t.exp_avg_sq, at, n, sv), fm, fv, m, v);
    store4(M, at, n, ov, m);
    store4(V, at, n, ov, v);
  }
}

}  // namespace rk

using namespace rk;

namespace {

// Fills `tab` with up to kMultiCap tensors from `tensors[i..n)`, leaving out empty ones; returns the next index,
// or -1 for a null pointer or a negative size.
enum { NEED_P = 1, NEED_STATE = 2, NEED_SCALES = 4 };
int64_t fill_table(MultiTable& tab, const rk_adamw_tensor* tensors, int64_t i, int64_t n, int needs) {
  tab.n = 0;
  tab.chunks = 0;
  for (; i < n && tab.n < kMultiCap; ++i) {
    const rk_adamw_tensor& t = tensors[i];
    if (t.numel < 0) return -1;
    if (t.numel == 0) continue;
    if (!t.g || ((needs & NEED_P) && !t.p) || ((needs & NEED_STATE) && (!t.exp_avg || !t.exp_avg_sq)) ||
        ((needs & NEED_SCALES) && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return -1;
    tab.t[tab.n++] = t;
    tab.chunks += (t.numel + kChunk - 1) / kChunk;
  }
  return i;
}

template <typename TP, typename TG>
int step_typed(const rk_adamw_tensor* tensors, int64_t n, int bits, const float* scalars, float beta1, float beta2,
               float eps, cudaStream_t s) {
  MultiTable tab;
  for (int64_t i = 0; i < n;) {
    i = fill_table(tab, tensors, i, n, NEED_P | NEED_STATE | (bits == 8 ? NEED_SCALES : 0));
    if (i < 0) return RK_ERR_ARG;
    if (tab.n == 0) continue;
    if (tab.chunks >= (1ll << 31)) return RK_ERR_UNSUPPORTED;
    if (bits == 8)
      rk_host::launch_k(adamw_multi_kernel<TP, TG, true>, (unsigned)tab.chunks, 256, 0, s, tab, scalars, beta1, beta2, eps);
    else
      rk_host::launch_k(adamw_multi_kernel<TP, TG, false>, (unsigned)tab.chunks, 256, 0, s, tab, scalars, beta1, beta2, eps);
    const int st = rk_host::launch_status();
    if (st) return st;
  }
  return RK_OK;
}

template <typename TP>
int step_g(const rk_adamw_tensor* tensors, int64_t n, int g_dtype, int bits, const float* scalars, float beta1,
           float beta2, float eps, cudaStream_t s) {
  switch (g_dtype) {
    case RK_F32: return step_typed<TP, float>(tensors, n, bits, scalars, beta1, beta2, eps, s);
    case RK_BF16: return step_typed<TP, __nv_bfloat16>(tensors, n, bits, scalars, beta1, beta2, eps, s);
    case RK_F16: return step_typed<TP, __half>(tensors, n, bits, scalars, beta1, beta2, eps, s);
    default: return RK_ERR_DTYPE;
  }
}

template <typename TG>
int sumsq_typed(const rk_adamw_tensor* tensors, int64_t n, float* partials, cudaStream_t s) {
  MultiTable tab;
  const int64_t end = rk_adamw_multi_parts(n);
  int64_t at = 0;
  for (int64_t i = 0; at < end;) {
    i = fill_table(tab, tensors, i, n, 0);  // past the last tensor: an empty table, whose partials are 0
    if (i < 0) return RK_ERR_ARG;
    rk_host::launch_k(sumsq_multi_kernel<TG>, kMultiNormBlocks, 256, 0, s, tab, partials + at);
    const int st = rk_host::launch_status();
    if (st) return st;
    at += kMultiNormBlocks;
  }
  return RK_OK;
}

template <typename TO>
int moments_typed(const rk_adamw_tensor* tensors, int64_t n, cudaStream_t s) {
  MultiTable tab;
  for (int64_t i = 0; i < n;) {
    i = fill_table(tab, tensors, i, n, NEED_P | NEED_STATE | NEED_SCALES);
    if (i < 0) return RK_ERR_ARG;
    if (tab.n == 0) continue;
    if (tab.chunks >= (1ll << 31)) return RK_ERR_UNSUPPORTED;
    rk_host::launch_k(moments_multi_kernel<TO>, (unsigned)tab.chunks, 256, 0, s, tab);
    const int st = rk_host::launch_status();
    if (st) return st;
  }
  return RK_OK;
}

}  // namespace

extern "C" int64_t rk_adamw_multi_parts(int64_t n) {
  return n <= 0 ? 0 : (n + kMultiCap - 1) / kMultiCap * kMultiNormBlocks;
}

extern "C" int rk_adamw_multi_sumsq(const rk_adamw_tensor* tensors, int64_t n, int g_dtype, float* partials,
                                    void* stream) {
  if (n < 0 || (n > 0 && (!tensors || !partials))) return RK_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (g_dtype) {
    case RK_F32: return sumsq_typed<float>(tensors, n, partials, s);
    case RK_BF16: return sumsq_typed<__nv_bfloat16>(tensors, n, partials, s);
    case RK_F16: return sumsq_typed<__half>(tensors, n, partials, s);
    default: return RK_ERR_DTYPE;
  }
}

extern "C" int rk_adamw_multi_prepare(const float* partials, int64_t parts, float max_norm, float beta1, float beta2,
                                      float weight_decay, float* scalars, void* stream) {
  if (!scalars || parts < 0 || (parts > 0 && !partials)) return RK_ERR_ARG;
  rk_host::launch_k(prepare_multi_kernel, 1, 256, 0, static_cast<cudaStream_t>(stream), partials, parts, max_norm, beta1,
                    beta2, weight_decay, scalars);
  return rk_host::launch_status();
}

extern "C" int rk_adamw_multi_step(const rk_adamw_tensor* tensors, int64_t n, int p_dtype, int g_dtype, int state_bits,
                                   const float* scalars, float beta1, float beta2, float eps, void* stream) {
  if (n < 0 || !scalars || (n > 0 && !tensors)) return RK_ERR_ARG;
  if (state_bits != 8 && state_bits != 32) return RK_ERR_DTYPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (p_dtype) {
    case RK_F32: return step_g<float>(tensors, n, g_dtype, state_bits, scalars, beta1, beta2, eps, s);
    case RK_BF16: return step_g<__nv_bfloat16>(tensors, n, g_dtype, state_bits, scalars, beta1, beta2, eps, s);
    case RK_F16: return step_g<__half>(tensors, n, g_dtype, state_bits, scalars, beta1, beta2, eps, s);
    default: return RK_ERR_DTYPE;
  }
}

extern "C" int rk_adamw_multi_moments(const rk_adamw_tensor* tensors, int64_t n, int out_dtype, void* stream) {
  if (n < 0 || (n > 0 && !tensors)) return RK_ERR_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (out_dtype) {
    case RK_F32: return moments_typed<float>(tensors, n, s);
    case RK_BF16: return moments_typed<__nv_bfloat16>(tensors, n, s);
    case RK_F16: return moments_typed<__half>(tensors, n, s);
    default: return RK_ERR_DTYPE;
  }
}
