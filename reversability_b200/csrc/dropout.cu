// Dropout from a counter-based generator: the mask is a function of (seed,
// offset, position) and is never stored; the backward, and a reversible
// block's recompute, generate it anew.
//
//   word i = number i % 4 of the Philox 4x32 block (10 rounds) of counter
//            (i / 4, offset), both 64 bits, under the 64-bit key `seed`
//            (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy
//            as 1, 2, 3", SC 2011);
//   kept  iff word i >= round(p 2^32);  y_i = residual_i + (kept ? x_i / (1 - p) : 0)
//
// Bound by memory for fp32 and with a residual. In 16 bits without one an
// element moves 4 bytes and costs 5 wide multiplies and about 9 other
// instructions, about two thirds of the issue slots at full bandwidth.
#include "vec.cuh"

namespace rk {

__device__ __forceinline__ uint4 philox10(uint64_t block, uint64_t offset, uint64_t key) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

struct DropArgs {
  int64_t n;
  uint64_t seed, offset;
  const int64_t* seed_dev;  // used instead of seed when not null
  uint32_t below;           // words up to this one drop ...
  uint32_t all;             // ... unless all bits are set here: nothing drops
  float scale;
};

// V consecutive elements from i0 on (a multiple of 4): elements at or past n are not touched.
template <typename Tx, typename Tr, typename Ty, int V, bool RES, bool VEC>
__device__ __forceinline__ void drop_chunk(const Tx* __restrict__ x, const Tr* __restrict__ res, Ty* __restrict__ y,
                                           int64_t i0, const DropArgs& a, uint64_t key) {
  float v[V], o[V];
  const bool whole = VEC && i0 + V <= a.n;
  if (whole) {
    load_vec<Tx, V>(x + i0, v);
    if (RES) load_vec<Tr, V>(res + i0, o);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[e] = i0 + e < a.n ? Dt<Tx>::to_f(x[i0 + e]) : 0.f;
      if (RES) o[e] = i0 + e < a.n ? Dt<Tr>::to_f(res[i0 + e]) : 0.f;
    }
  }
#pragma unroll
  for (int q = 0; q < V / 4; ++q) {
    const uint4 w = philox10((uint64_t)(i0 >> 2) + q, a.offset, key);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {  // a dropped value is not used, whatever it is
      const float kept = (word[e] | a.all) > a.below ? v[q * 4 + e] * a.scale : 0.f;
      o[q * 4 + e] = RES ? o[q * 4 + e] + kept : kept;
    }
  }
  if (whole) {
    store_vec<Ty, V>(y + i0, o);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (i0 + e < a.n) y[i0 + e] = Dt<Ty>::from_f(o[e]);
  }
}

constexpr int kDropThreads = 256, kDropUnroll = 2;

template <typename Tx, typename Tr, typename Ty, bool RES, bool VEC>
__global__ void __launch_bounds__(kDropThreads)
    dropout_kernel(const Tx* __restrict__ x, const Tr* __restrict__ res, Ty* __restrict__ y, const DropArgs a) {
  pdl_wait();  // inputs are the previous kernel's outputs
  constexpr int V = VEC ? 16 / (int)sizeof(Tx) : 4;
  const uint64_t key = a.seed_dev ? (uint64_t)__ldg(a.seed_dev) : a.seed;
  const int64_t c0 = (int64_t)blockIdx.x * (kDropThreads * kDropUnroll) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kDropUnroll; ++u) {
    const int64_t i0 = (c0 + u * kDropThreads) * V;
    if (i0 < a.n) drop_chunk<Tx, Tr, Ty, V, RES, VEC>(x, res, y, i0, a, key);
  }
}

}  // namespace rk

using namespace rk;

namespace {

template <typename Tx, typename Tr, typename Ty, bool RES>
int launch(const void* x, const void* res, void* y, const DropArgs& a, cudaStream_t s) {
  // vectors of 16 bytes of x; what they take on the other sides is read and written in whole vectors too
  constexpr int V = 16 / (int)sizeof(Tx);
  auto fits = [](const void* p, size_t bytes) { return rk_host::aligned(p, bytes < 16 ? bytes : 16); };
  const bool vec = fits(x, 16) && fits(y, V * sizeof(Ty)) && (!RES || fits(res, V * sizeof(Tr)));
  const int64_t per = (int64_t)kDropThreads * kDropUnroll * (vec ? V : 4);
  const int64_t grid = (a.n + per - 1) / per;
  if (grid >= (1ll << 31)) return RK_ERR_UNSUPPORTED;
  const Tx* xp = static_cast<const Tx*>(x);
  const Tr* rp = static_cast<const Tr*>(res);
  Ty* yp = static_cast<Ty*>(y);
  if (vec) rk_host::launch_k(dropout_kernel<Tx, Tr, Ty, RES, true>, (unsigned)grid, kDropThreads, 0, s, xp, rp, yp, a);
  else rk_host::launch_k(dropout_kernel<Tx, Tr, Ty, RES, false>, (unsigned)grid, kDropThreads, 0, s, xp, rp, yp, a);
  return rk_host::launch_status();
}

// y in x's type or fp32 (a residual is in y's type); without a residual also fp32 in and 16 bits out (the backward
// of a 16-bit branch added to an fp32 residual).
template <typename T>
int launch16(const void* x, const void* res, void* y, int y_dtype, const DropArgs& a, cudaStream_t s) {
  if (y_dtype == RK_F32)
    return res ? launch<T, float, float, true>(x, res, y, a, s) : launch<T, float, float, false>(x, res, y, a, s);
  return res ? launch<T, T, T, true>(x, res, y, a, s) : launch<T, T, T, false>(x, res, y, a, s);
}

}  // namespace

extern "C" int rk_dropout(const void* x, int x_dtype, const void* residual, void* y, int y_dtype, int64_t n, double p,
                          uint64_t seed, const int64_t* seed_dev, uint64_t offset, void* stream) {
  if (!rk_host::dtype_ok(x_dtype) || !rk_host::dtype_ok(y_dtype) ||
      (x_dtype != y_dtype && y_dtype != RK_F32 && (residual || x_dtype != RK_F32)))
    return RK_ERR_DTYPE;
  if (n < 0 || !(p >= 0.0 && p <= 1.0)) return RK_ERR_ARG;
  if (n == 0) return RK_OK;
  if (!x || !y) return RK_ERR_ARG;
  if (seed_dev && !rk_host::aligned(seed_dev, 8)) return RK_ERR_ALIGN;
  DropArgs a{};
  a.n = n;
  a.seed = seed;
  a.offset = offset;
  a.seed_dev = seed_dev;
  const double border = p * 4294967296.0;  // exact: a power of two
  uint64_t words = (uint64_t)border;       // rounded to the nearest even whole number
  const double rest = border - (double)words;
  if (rest > 0.5 || (rest == 0.5 && (words & 1))) ++words;
  a.all = words ? 0u : 0xffffffffu;
  a.below = words ? (uint32_t)(words - 1) : 0u;
  a.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x_dtype == RK_BF16) return launch16<__nv_bfloat16>(x, residual, y, y_dtype, a, s);
  if (x_dtype == RK_F16) return launch16<__half>(x, residual, y, y_dtype, a, s);
  if (y_dtype == RK_F32)
    return residual ? launch<float, float, float, true>(x, residual, y, a, s)
                    : launch<float, float, float, false>(x, residual, y, a, s);
  if (y_dtype == RK_BF16) return launch<float, float, __nv_bfloat16, false>(x, residual, y, a, s);
  return launch<float, float, __half, false>(x, residual, y, a, s);
}
