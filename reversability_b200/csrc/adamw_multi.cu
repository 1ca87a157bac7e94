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
//
// Bound: HBM, 28 bytes an element with fp32 parameters and gradients and 32-bit
// moments, 16 and 1/16 with 8-bit ones. 456M parameters: 1872 us (6.8 TB/s) and
// 1086 (6.75), with bf16 parameters and gradients 822 (5.6); their moments decoded
// 431 (6.4). The 20.3M decoder's 45 tensors with the norm for clipping: 104 (5.5
// TB/s, three launches). A two-layer test model's 14: 12 us, the launches' own.
#include <type_traits>
#include "vec.cuh"

namespace rk {

constexpr int kMultiCap = 64;       // tensors per launch: 64 x 60 bytes, below the 4 KB of a kernel's parameters
constexpr int kQBlock = 256;        // elements that share a scale
constexpr int kWarps = 8;
constexpr int kTile = kWarps * kQBlock;  // elements that a CTA takes at once
constexpr int kMultiNormBlocks = 592;
constexpr int kSumTiles = 4;        // tiles of a chunk of the norm: eight loads a thread in flight

struct MultiTable {
  rk_adamw_tensor t[kMultiCap];
  int start[kMultiCap + 1];  // first chunk of each tensor; start[n] = all chunks
  int n;
  int tiles;  // tiles of a chunk, which is what a CTA takes
};

// The tensor that holds chunk `c` of the launch.
__device__ __forceinline__ int find_tensor(const MultiTable& tab, int c) {
  int lo = 0, hi = tab.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (c >= tab.start[mid]) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ float sqrt_approx(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four consecutive elements at p; where not all of them exist or p is not aligned for it (`left` >= 0), one by one,
// the first `left` of them, the others zero.
constexpr int kWhole = -1;
template <typename T>
__device__ __forceinline__ void load4(const T* p, int left, float (&v)[4]) {
  if (left == kWhole) {
    load_vec<T, 4>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? Dt<T>::to_f(p[e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int left, const float (&v)[4]) {
  if (left == kWhole) {
    store_vec<T, 4>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) p[e] = Dt<T>::from_f(v[e]);
  }
}
__device__ __forceinline__ uint32_t load4_codes(const uint8_t* p, int left) {
  if (left == kWhole) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) w |= (uint32_t)p[e] << (8 * e);
  return w;
}
__device__ __forceinline__ void store4_codes(uint8_t* p, int left, uint32_t w) {
  if (left == kWhole) {
    *reinterpret_cast<uint32_t*>(p) = w;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e < left) p[e] = (uint8_t)(w >> (8 * e));
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

// The betas' weights, rounded from 64 bits: 1 - beta taken in fp32 is off by up to 2^-25 / (1 - beta) of itself (1.3e-5 at
// 0.999), and so would be the moments. v moves towards g^2 by 1 - beta2 of the difference, so that what fp32 takes off
// beta2 does not add up over a decay of a thousand steps; below 1/2, where the difference would lose a small g^2 beside a
// large v, as the sum of two products. (The sum with a further product for what fp32 takes off beta2, at all betas: 1891
// us in place of 1872 at 456M elements, 106 in place of 104 at 20.3M.)
struct Weights {
  float new1, old2, new2;  // 1 - beta1, beta2, 1 - beta2
};
struct StepConst {
  float coef, step_size, root, decay, eps;
  Weights w;
};

// One element: m and v become the new moments, r = sqrt(v), p the new parameter. The approximate root and reciprocal are
// within 2^-22 together and leave the update as near to 64 bits as exact ones do the plain fp32 form (0.97 times its rms
// error; exact ones 0.90, at 14 % more time with 8-bit moments). DENORMAL: the root of a denormal v too, which otherwise
// counts as 0, and with a small eps the update as infinite.
template <bool DENORMAL>
__device__ __forceinline__ void adamw_element(const StepConst& k, float g, float& p, float& m, float& v, float& r) {
  const float gi = g * k.coef;
  m = fmaf(k.w.new1, gi - m, m);
  v = k.w.old2 >= 0.5f ? fmaf(k.w.new2, fmaf(gi, gi, -v), v) : fmaf(k.w.old2, v, k.w.new2 * gi * gi);
  if constexpr (DENORMAL) asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  else r = sqrt_approx(v);
  p = fmaf(p, k.decay, -(k.step_size * m * rcp_approx(fmaf(r, k.root, k.eps))));
}

// Four codes from four rounded floats (their low bytes).
__device__ __forceinline__ uint32_t pack_codes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// One scale block of a tensor by one warp: lane l has elements 4 l .. 4 l + 3 of each half. WHOLE: all 256 exist and
// every base is aligned for vectors.
template <typename TP, typename TG, bool Q8>
struct BlockIn {
  float p[2][4], m[2][4], v[2][4];
  float g[2][4];
  uint32_t mc[2], vc[2];
  float ms, vs;
};
__device__ __forceinline__ int left_of(const rk_adamw_tensor& t, int64_t at, bool whole) {
  const int64_t have = t.numel - at;
  return whole ? kWhole : (int)(have < 0 ? 0 : have > 4 ? 4 : have);
}
template <typename TP, typename TG, bool Q8, bool WHOLE>
__device__ __forceinline__ void load_block(const rk_adamw_tensor& t, int64_t block, BlockIn<TP, TG, Q8>& in) {
  const int64_t at = block * kQBlock + (threadIdx.x & 31) * 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int left = left_of(t, at + h * 128, WHOLE);
    load4(static_cast<const TP*>(t.p) + at + h * 128, left, in.p[h]);
    load4(static_cast<const TG*>(t.g) + at + h * 128, left, in.g[h]);
    if constexpr (Q8) {
      in.mc[h] = load4_codes(static_cast<const uint8_t*>(t.exp_avg) + at + h * 128, left);
      in.vc[h] = load4_codes(static_cast<const uint8_t*>(t.exp_avg_sq) + at + h * 128, left);
    } else {
      load4(static_cast<const float*>(t.exp_avg) + at + h * 128, left, in.m[h]);
      load4(static_cast<const float*>(t.exp_avg_sq) + at + h * 128, left, in.v[h]);
    }
  }
}
template <typename TP, typename TG, bool Q8, bool WHOLE, bool DENORMAL>
__device__ __forceinline__ void update_block(const rk_adamw_tensor& t, int64_t block, BlockIn<TP, TG, Q8>& in,
                                             const StepConst& k) {
  const int64_t at = block * kQBlock + (threadIdx.x & 31) * 4;
  if constexpr (Q8) {
    const float fm = in.ms * (1.f / (127.f * 127.f)), fv = in.vs * (1.f / (255.f * 255.f));
#pragma unroll
    for (int h = 0; h < 2; ++h) codes_to_moments(in.mc[h], in.vc[h], fm, fv, in.m[h], in.v[h]);
  }
  float mm = 0.f, rm = 0.f, r[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int left = left_of(t, at + h * 128, WHOLE);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      adamw_element<DENORMAL>(k, in.g[h][e], in.p[h][e], in.m[h][e], in.v[h][e], r[h][e]);
      if constexpr (Q8) {
        mm = max_bits(mm, in.m[h][e]);
        rm = max_bits(rm, r[h][e]);
      }
    }
    store4(static_cast<TP*>(t.p) + at + h * 128, left, in.p[h]);
    if constexpr (!Q8) {
      store4(static_cast<float*>(t.exp_avg) + at + h * 128, left, in.m[h]);
      store4(static_cast<float*>(t.exp_avg_sq) + at + h * 128, left, in.v[h]);
    }
  }
  if constexpr (Q8) {
    mm = warp_max_abs(mm);
    rm = warp_max_abs(rm);
    const float im = code_factor(127.f * 127.f, mm), ir = code_factor(255.f * 255.f, rm);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int left = left_of(t, at + h * 128, WHOLE);
      uint32_t a[4], b[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {  // at most 127 and 255 up to rounding, which the nearest integer takes off
        a[e] = round_bits(copysignf(sqrt_approx(fabsf(in.m[h][e]) * im), in.m[h][e]));
        b[e] = round_bits(fmaxf(sqrt_approx(r[h][e] * ir), r[h][e] > 0.f ? 1.f : 0.f));
      }
      store4_codes(static_cast<uint8_t*>(t.exp_avg) + at + h * 128, left, pack_codes(a[0], a[1], a[2], a[3]));
      store4_codes(static_cast<uint8_t*>(t.exp_avg_sq) + at + h * 128, left, pack_codes(b[0], b[1], b[2], b[3]));
    }
    in.ms = mm;
    in.vs = rm;
  }
}

// With 8-bit moments an element brings 10 bytes and takes 50 instructions: loads into registers in front of each
// update kept too little in flight (4.6 TB/s; one block ahead, 4.9). So each lane copies its own elements of the next
// blocks into its own places of shared memory (cp.async, no barrier needed) and takes them from there.
constexpr int kStages = 4;
template <int BYTES>
__device__ __forceinline__ void copy_async(void* smem, const void* global) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(smem)), "l"(global), "n"(BYTES) : "memory");
}
template <typename TP, typename TG>
struct Stage {  // of one CTA
  TP p[2][256][4];
  TG g[2][256][4];
  uint32_t mc[2][256], vc[2][256];
};
template <typename TP, typename TG>
__device__ __forceinline__ void stage_block(const rk_adamw_tensor& t, int64_t block, Stage<TP, TG>& st) {
  const int64_t at = block * kQBlock + (threadIdx.x & 31) * 4;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    copy_async<4 * sizeof(TP)>(st.p[h][threadIdx.x], static_cast<const TP*>(t.p) + at + h * 128);
    copy_async<4 * sizeof(TG)>(st.g[h][threadIdx.x], static_cast<const TG*>(t.g) + at + h * 128);
    copy_async<4>(&st.mc[h][threadIdx.x], static_cast<const uint8_t*>(t.exp_avg) + at + h * 128);
    copy_async<4>(&st.vc[h][threadIdx.x], static_cast<const uint8_t*>(t.exp_avg_sq) + at + h * 128);
  }
}
template <typename T>
__device__ __forceinline__ void unstage4(const T* p, float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = *reinterpret_cast<const float4*>(p);
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = Dt<T>::to_f(e[i]);
  }
}
template <typename TP, typename TG>
__device__ __forceinline__ void unstage_block(const Stage<TP, TG>& st, BlockIn<TP, TG, true>& in) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unstage4(st.p[h][threadIdx.x], in.p[h]);
    unstage4(st.g[h][threadIdx.x], in.g[h]);
    in.mc[h] = st.mc[h][threadIdx.x];
    in.vc[h] = st.vc[h][threadIdx.x];
  }
}
template <typename TP, typename TG, bool Q8>
constexpr int step_smem() { return Q8 ? kStages * (int)sizeof(Stage<TP, TG>) : 0; }

// Whether p is aligned for four elements of `size` bytes.
__device__ __forceinline__ bool vec_ok(const void* p, int size) {
  return (reinterpret_cast<uintptr_t>(p) & (4 * size - 1)) == 0;
}

template <typename TP, typename TG, bool Q8, bool DENORMAL>
__global__ void __launch_bounds__(256) adamw_multi_kernel(const __grid_constant__ MultiTable tab,
                                                          const float* __restrict__ scalars, Weights weights, float eps) {
  const int which = find_tensor(tab, blockIdx.x);
  const rk_adamw_tensor& t = tab.t[which];
  const bool vec = vec_ok(t.p, sizeof(TP)) && vec_ok(t.g, sizeof(TG)) && vec_ok(t.exp_avg, Q8 ? 1 : 4) &&
                   vec_ok(t.exp_avg_sq, Q8 ? 1 : 4);
  // 8-bit moments: a warp takes tab.tiles consecutive blocks, whose scales travel as one load and one store. 32-bit: the
  // CTA's warps take neighbouring blocks (1872 against 1993 us at 456M elements)
  const int64_t chunk = blockIdx.x - tab.start[which];
  const int warp = threadIdx.x >> 5;
  constexpr int kStep = Q8 ? 1 : kWarps;
  const int64_t block = Q8 ? (chunk * kWarps + warp) * tab.tiles : chunk * tab.tiles * kWarps + warp;
  const int64_t blocks = (t.numel + kQBlock - 1) / kQBlock, whole_blocks = vec ? t.numel / kQBlock : 0;
  const auto before = [&](int64_t end) {  // how many of this warp's blocks lie before `end`
    return (int)max((int64_t)0, min((int64_t)tab.tiles, (end - block + kStep - 1) / kStep));
  };
  const int todo = before(blocks), whole = before(whole_blocks);
  const int lane = threadIdx.x & 31;
  pdl_wait();  // inputs are the previous kernel's outputs
  const StepConst k = {scalars[3], scalars[4], 1.f / scalars[5], scalars[6], eps, weights};
  float ms = 0.f, vs = 0.f;
  if (Q8 && lane < todo) {
    ms = t.exp_avg_scale[block + lane];
    vs = t.exp_avg_sq_scale[block + lane];
  }
  const auto update = [&](int i, BlockIn<TP, TG, Q8>& in, auto is_whole) {
    if constexpr (Q8) {
      in.ms = __shfl_sync(0xffffffffu, ms, i);
      in.vs = __shfl_sync(0xffffffffu, vs, i);
    }
    update_block<TP, TG, Q8, decltype(is_whole)::value, DENORMAL>(t, block + i * kStep, in, k);
    if (Q8 && lane == i) {
      ms = in.ms;
      vs = in.vs;
    }
  };
  int i = 0;
  if constexpr (Q8) {
    extern __shared__ __align__(16) unsigned char smem[];
    Stage<TP, TG>* stages = reinterpret_cast<Stage<TP, TG>*>(smem);
#pragma unroll
    for (int j = 0; j < kStages - 1; ++j) {
      if (j < whole) stage_block(t, block + j, stages[j]);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    int at = 0;
    for (; i < whole; ++i) {
      BlockIn<TP, TG, Q8> now;
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      unstage_block(stages[at], now);
      __syncwarp();  // orders the reads of the stage that is filled again
      if (i + kStages - 1 < whole) stage_block(t, block + i + kStages - 1, stages[at ? at - 1 : kStages - 1]);  // taken last
      asm volatile("cp.async.commit_group;" ::: "memory");
      update(i, now, std::true_type{});
      at = at + 1 < kStages ? at + 1 : 0;
    }
  } else {
    for (; i < whole; ++i) {
      BlockIn<TP, TG, Q8> now;
      load_block<TP, TG, Q8, true>(t, block + i * kStep, now);
      update(i, now, std::true_type{});
    }
  }
  for (; i < todo; ++i) {
    BlockIn<TP, TG, Q8> now;
    load_block<TP, TG, Q8, false>(t, block + i * kStep, now);
    update(i, now, std::false_type{});
  }
  if (Q8 && lane < todo) {
    t.exp_avg_scale[block + lane] = ms;
    t.exp_avg_sq_scale[block + lane] = vs;
  }
}

// Squares of the gradients: fp32 per thread over its chunks, a partial sum a CTA, joined in fp64 below; the same order
// every time. 20.3M gradients: 15 us cold (5.4 TB/s).
template <typename TG>
__global__ void __launch_bounds__(256) sumsq_multi_kernel(const __grid_constant__ MultiTable tab,
                                                          float* __restrict__ partial) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ float red[8];
  float s = 0.f;
  for (int chunk = blockIdx.x; chunk < tab.start[tab.n]; chunk += gridDim.x) {
    const int which = find_tensor(tab, chunk);
    const rk_adamw_tensor& t = tab.t[which];
    const TG* G = static_cast<const TG*>(t.g);
    const int64_t c0 = (int64_t)(chunk - tab.start[which]) * kSumTiles * kTile, at = c0 + threadIdx.x * 4;
    const bool whole = vec_ok(G, sizeof(TG)) && c0 + kSumTiles * kTile <= t.numel;
    float g[2 * kSumTiles][4];
#pragma unroll
    for (int h = 0; h < 2 * kSumTiles; ++h) {
      const int64_t have = t.numel - at - h * 1024;
      load4(G + at + h * 1024, whole ? kWhole : (int)(have < 0 ? 0 : have > 4 ? 4 : have), g[h]);
    }
#pragma unroll
    for (int h = 0; h < 2 * kSumTiles; ++h)
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

// beta^t for a whole t, by squaring (pow in fp64 took most of this kernel's 5 us).
__device__ __forceinline__ double power(double beta, float t) {
  double r = 1.0;
  for (unsigned n = (unsigned)t; n; n >>= 1, beta *= beta)
    if (n & 1) r *= beta;
  return r;
}

// scalars as in optim.cu; without partials (no clipping) the coefficient is 1 and the norm is left at 0.
__global__ void __launch_bounds__(256) prepare_multi_kernel(const float* __restrict__ partial, int64_t parts,
                                                            float max_norm, double beta1, double beta2,
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
    const double bc1 = 1.0 - power(beta1, t);
    const double bc2 = 1.0 - power(beta2, t);
    scalars[4] = (float)(lr / bc1);
    scalars[5] = (float)sqrt(bc2);
    scalars[6] = 1.f - lr * weight_decay;
  }
}

// A warp decodes a scale block, lane l its elements 8 l .. 8 l + 7, so that 16-bit values leave in 16-byte stores.
template <typename TO>
__global__ void __launch_bounds__(256) moments_multi_kernel(const __grid_constant__ MultiTable tab) {
  const int which = find_tensor(tab, blockIdx.x);
  const rk_adamw_tensor& t = tab.t[which];
  const int lane = threadIdx.x & 31;
  TO* M = static_cast<TO*>(t.p);
  TO* V = static_cast<TO*>(const_cast<void*>(t.g));
  const uint8_t* M8 = static_cast<const uint8_t*>(t.exp_avg);
  const uint8_t* V8 = static_cast<const uint8_t*>(t.exp_avg_sq);
  const bool vec = ((reinterpret_cast<uintptr_t>(M) | reinterpret_cast<uintptr_t>(V)) & 15) == 0 &&
                   ((reinterpret_cast<uintptr_t>(M8) | reinterpret_cast<uintptr_t>(V8)) & 7) == 0;
  const int64_t first = (int64_t)(blockIdx.x - tab.start[which]) * tab.tiles * (kTile / kQBlock) + (threadIdx.x >> 5);
  pdl_wait();  // inputs are the previous kernel's outputs
#pragma unroll 4
  for (int tile = 0; tile < tab.tiles; ++tile) {
    const int64_t block = first + tile * (kTile / kQBlock);
    const int64_t at = block * kQBlock + lane * 8;
    if (at >= t.numel) break;
    const float fm = t.exp_avg_scale[block] * (1.f / (127.f * 127.f));
    const float fv = t.exp_avg_sq_scale[block] * (1.f / (255.f * 255.f));
    const int64_t have = t.numel - at;
    if (vec && have >= 8) {
      const uint2 mc = *reinterpret_cast<const uint2*>(M8 + at), vc = *reinterpret_cast<const uint2*>(V8 + at);
      float m[2][4], v[2][4], o[8];
      codes_to_moments(mc.x, vc.x, fm, fv, m[0], v[0]);
      codes_to_moments(mc.y, vc.y, fm, fv, m[1], v[1]);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = m[e >> 2][e & 3];
      store_vec<TO, 8>(M + at, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = v[e >> 2][e & 3];
      store_vec<TO, 8>(V + at, o);
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t rest = have - 4 * h;
        const int left = (int)(rest < 0 ? 0 : rest > 4 ? 4 : rest);
        float m[4], v[4];
        codes_to_moments(load4_codes(M8 + at + 4 * h, left), load4_codes(V8 + at + 4 * h, left), fm, fv, m, v);
        store4(M + at + 4 * h, left, m);
        store4(V + at + 4 * h, left, v);
      }
    }
  }
}

}  // namespace rk

using namespace rk;

namespace {

// Tiles of a chunk, that is consecutive blocks of a warp: 8, so that the warp writes its scales as whole 32-byte
// sectors (written one by one, 4 bytes each, they cost 280 of 1376 us at 456M elements), but at least four CTAs for
// each of about 150 SMs.
// With 32-bit moments and for decoding 4 tiles are enough.
int tiles_for(const rk_adamw_tensor* tensors, int64_t n, int most) {
  int64_t all = 0;
  for (int64_t i = 0; i < n; ++i) all += tensors[i].numel > 0 ? tensors[i].numel : 0;
  int tiles = 1;
  while (tiles < most && all >= (int64_t)600 * kTile * 2 * tiles) tiles *= 2;
  return tiles;
}
enum { NEED_P = 1, NEED_STATE = 2, NEED_SCALES = 4 };
// Fills `tab` with up to kMultiCap tensors from `tensors[i..n)`, leaving out empty ones; returns the next index,
// or -1 for a null pointer or a negative size.
int64_t fill_table(MultiTable& tab, const rk_adamw_tensor* tensors, int64_t i, int64_t n, int needs, int tiles) {
  tab.n = 0;
  tab.start[0] = 0;
  tab.tiles = tiles;
  int64_t chunks = 0;
  for (; i < n && tab.n < kMultiCap; ++i) {
    const rk_adamw_tensor& t = tensors[i];
    if (t.numel < 0) return -1;
    if (t.numel == 0) continue;
    if (!t.g || ((needs & NEED_P) && !t.p) || ((needs & NEED_STATE) && (!t.exp_avg || !t.exp_avg_sq)) ||
        ((needs & NEED_SCALES) && (!t.exp_avg_scale || !t.exp_avg_sq_scale)))
      return -1;
    const int64_t mine = (t.numel + tiles * kTile - 1) / (tiles * kTile);
    if (chunks + mine >= (1ll << 31)) {
      if (tab.n == 0) return -1;  // one tensor of more than 2^44 elements
      break;
    }
    tab.t[tab.n++] = t;
    chunks += mine;
    tab.start[tab.n] = (int)chunks;
  }
  return i;
}

// Below it the kernels take the root of a denormal second moment: it is at most 1e-19, 1e-17 once it is corrected for
// beta2 = 0.9999, so beside a larger eps nothing is lost with it. 456M elements with 8-bit moments, us without and with:
// fp32 1086/1087, bf16 gradients 978/980, bf16 parameters too 822/857. With 32-bit moments 1870 either way, so always.
constexpr float kSmallEps = 1e-10f;

template <typename TP, typename TG>
int step_typed(const rk_adamw_tensor* tensors, int64_t n, int bits, const float* scalars, const Weights& w, float eps,
               cudaStream_t s) {
  MultiTable tab;
  const int tiles = tiles_for(tensors, n, bits == 8 ? 8 : 4);
  for (int64_t i = 0; i < n;) {
    i = fill_table(tab, tensors, i, n, NEED_P | NEED_STATE | (bits == 8 ? NEED_SCALES : 0), tiles);
    if (i < 0) return RK_ERR_ARG;
    if (tab.n == 0) continue;
    if (bits == 8) {
      auto kernel = eps < kSmallEps ? adamw_multi_kernel<TP, TG, true, true> : adamw_multi_kernel<TP, TG, true, false>;
      const int e = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kernel), step_smem<TP, TG, true>());
      if (e) return e;
      rk_host::launch_k(kernel, (unsigned)tab.start[tab.n], 256, step_smem<TP, TG, true>(), s, tab, scalars, w, eps);
    } else
      rk_host::launch_k(adamw_multi_kernel<TP, TG, false, true>, (unsigned)tab.start[tab.n], 256, 0, s, tab, scalars, w, eps);
    const int st = rk_host::launch_status();
    if (st) return st;
  }
  return RK_OK;
}

template <typename TP>
int step_g(const rk_adamw_tensor* tensors, int64_t n, int g_dtype, int bits, const float* scalars, const Weights& w,
           float eps, cudaStream_t s) {
  switch (g_dtype) {
    case RK_F32: return step_typed<TP, float>(tensors, n, bits, scalars, w, eps, s);
    case RK_BF16: return step_typed<TP, __nv_bfloat16>(tensors, n, bits, scalars, w, eps, s);
    case RK_F16: return step_typed<TP, __half>(tensors, n, bits, scalars, w, eps, s);
    default: return RK_ERR_DTYPE;
  }
}

template <typename TG>
int sumsq_typed(const rk_adamw_tensor* tensors, int64_t n, float* partials, cudaStream_t s) {
  MultiTable tab;
  const int tiles = kSumTiles;
  const int64_t end = rk_adamw_multi_parts(n);
  int64_t at = 0;
  for (int64_t i = 0; at < end;) {
    i = fill_table(tab, tensors, i, n, 0, tiles);  // past the last tensor: an empty table, whose partials are 0
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
  const int tiles = tiles_for(tensors, n, 4);
  for (int64_t i = 0; i < n;) {
    i = fill_table(tab, tensors, i, n, NEED_P | NEED_STATE | NEED_SCALES, tiles);
    if (i < 0) return RK_ERR_ARG;
    if (tab.n == 0) continue;
    rk_host::launch_k(moments_multi_kernel<TO>, (unsigned)tab.start[tab.n], 256, 0, s, tab);
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

extern "C" int rk_adamw_multi_prepare(const float* partials, int64_t parts, float max_norm, double beta1, double beta2,
                                      float weight_decay, float* scalars, void* stream) {
  if (!scalars || parts < 0 || (parts > 0 && !partials)) return RK_ERR_ARG;
  rk_host::launch_k(prepare_multi_kernel, 1, 256, 0, static_cast<cudaStream_t>(stream), partials, parts, max_norm, beta1,
                    beta2, weight_decay, scalars);
  return rk_host::launch_status();
}

extern "C" int rk_adamw_multi_step(const rk_adamw_tensor* tensors, int64_t n, int p_dtype, int g_dtype, int state_bits,
                                   const float* scalars, double beta1, double beta2, float eps, void* stream) {
  if (n < 0 || !scalars || (n > 0 && !tensors)) return RK_ERR_ARG;
  if (state_bits != 8 && state_bits != 32) return RK_ERR_DTYPE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Weights w = {(float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2)};
  switch (p_dtype) {
    case RK_F32: return step_g<float>(tensors, n, g_dtype, state_bits, scalars, w, eps, s);
    case RK_BF16: return step_g<__nv_bfloat16>(tensors, n, g_dtype, state_bits, scalars, w, eps, s);
    case RK_F16: return step_g<__half>(tensors, n, g_dtype, state_bits, scalars, w, eps, s);
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
