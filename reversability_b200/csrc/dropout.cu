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
// Bound by memory for fp32 (134M elements 170 us, 6.3 TB/s) and with a residual;
// in 16 bits without one, where an element moves 4 bytes, by the multipliers: 20
// instructions an element, a quarter of them wide multiplies, which only one of
// the two FMA pipes takes (it is busy 80 % of the time, warps stall on it first,
// 2.4 of 10 to 1.0 on memory), half of the rest on the half-rate logic pipe (57
// %). 134M bf16 elements take 115 us (4.7 TB/s; 163 us with one vector after
// the other and nothing shared): what is the same for all blocks of a thread
// (round keys, the second counter word's first product, the first word's
// second) is formed once, pairs are scaled and rounded by one instruction, and
// the next tile is loaded before this one's words are formed. 4 CTAs an SM and
// two vectors a thread: 5 and 6 CTAs 117 and 119 us, one vector 127, four 118.
#include <type_traits>
#include "vec.cuh"

namespace rk {

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u, kPhiloxW0 = 0x9E3779B9u, kPhiloxW1 = 0xBB67AE85u;

// The generator for blocks that share the upper half of their number.
struct Philox {
  uint32_t k0[10], k1[10];
  uint32_t c3k1, l1k0, h2k1, l2;  // parts of rounds 1 and 2
  __device__ __forceinline__ Philox(uint32_t block_hi, uint64_t offset, uint64_t key) {
#pragma unroll
    for (int r = 0; r < 10; ++r) {
      k0[r] = (uint32_t)key + r * kPhiloxW0;
      k1[r] = (uint32_t)(key >> 32) + r * kPhiloxW1;
    }
    const uint64_t b = (uint64_t)(uint32_t)offset * kPhiloxM1;  // round 1 of words 2 and 3
    const uint64_t a = (uint64_t)((uint32_t)(b >> 32) ^ block_hi ^ k0[0]) * kPhiloxM0;  // round 2 of word 0
    c3k1 = (uint32_t)(offset >> 32) ^ k1[0];
    l1k0 = (uint32_t)b ^ k0[1];
    h2k1 = (uint32_t)(a >> 32) ^ k1[1];
    l2 = (uint32_t)a;
  }
  __device__ __forceinline__ void block(uint32_t block_lo, uint32_t (&w)[4]) const {
    const uint64_t a1 = (uint64_t)block_lo * kPhiloxM0;
    const uint64_t b2 = (uint64_t)((uint32_t)(a1 >> 32) ^ c3k1) * kPhiloxM1;
    uint32_t c0 = (uint32_t)(b2 >> 32) ^ l1k0, c1 = (uint32_t)b2, c2 = (uint32_t)a1 ^ h2k1, c3 = l2;
#pragma unroll
    for (int r = 2; r < 10; ++r) {
      const uint64_t a = (uint64_t)c0 * kPhiloxM0, b = (uint64_t)c2 * kPhiloxM1;
      c0 = (uint32_t)(b >> 32) ^ c1 ^ k0[r];
      c2 = (uint32_t)(a >> 32) ^ c3 ^ k1[r];
      c1 = (uint32_t)b;
      c3 = (uint32_t)a;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
  }
};

struct DropArgs {
  int64_t n;
  uint64_t seed, offset;
  const int64_t* seed_dev;  // used instead of seed when not null
  uint32_t border;          // words from this one on keep their element
  float scale;
};

// Two values rounded to a pair of 16-bit ones.
template <typename T>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  uint32_t d;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
template <typename T, int V>
__device__ __forceinline__ void store_rounded(T* __restrict__ p, const float (&v)[V]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t r[V / 2];
#pragma unroll
    for (int k = 0; k < V / 2; ++k) r[k] = round_pair<T>(v[2 * k], v[2 * k + 1]);
    if constexpr (V == 8) *reinterpret_cast<uint4*>(p) = make_uint4(r[0], r[1], r[2], r[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
  } else {
    store_vec<T, V>(p, v);
  }
}

constexpr int kDropThreads = 256, kDropCtas = 4;
// Vectors a thread takes at a time: two, one where the residual takes twice the registers.
__host__ __device__ constexpr int drop_unroll(int size_x, int size_res) { return size_res > size_x ? 1 : 2; }

// V elements of T as they lie in memory.
template <typename T, int V>
struct Packed {
  uint4 q[(V * sizeof(T) + 15) / 16];  // 8 bytes: half of one
  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (V * sizeof(T) == 8) {
      const uint2 h = __ldg(reinterpret_cast<const uint2*>(p));
      q[0] = make_uint4(h.x, h.y, 0u, 0u);
    } else {
#pragma unroll
      for (int i = 0; i < (int)(V * sizeof(T) / 16); ++i) q[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
  }
  __device__ __forceinline__ float2 pair(int k) const {
    const T* e = reinterpret_cast<const T*>(q);
    return make_float2(Dt<T>::to_f(e[2 * k]), Dt<T>::to_f(e[2 * k + 1]));
  }
};

// CTAs walk over tiles of a few vectors of V elements a thread and load the next tile before they form this
// one's words. A tile is an aligned power of two of elements, so the upper half of the block number is the same for
// all of it. What is left behind the last whole tile, and tensors that do not start on vector boundaries (VEC false),
// go element by element.
template <typename Tx, typename Tr, typename Ty, bool RES, bool VEC>
__global__ void __launch_bounds__(kDropThreads, kDropCtas)
    dropout_kernel(const Tx* __restrict__ x, const Tr* __restrict__ res, Ty* __restrict__ y, const DropArgs a) {
  pdl_wait();  // inputs are the previous kernel's outputs
  constexpr int V = 16 / (int)sizeof(Tx), U = drop_unroll((int)sizeof(Tx), RES ? (int)sizeof(Tr) : 0);
  constexpr int PER = kDropThreads * U * V;
  static_assert((PER & (PER - 1)) == 0, "a power of two");
  const uint64_t key = a.seed_dev ? (uint64_t)__ldg(a.seed_dev) : a.seed;
  const int64_t whole = VEC ? a.n / PER : 0, tiles = (a.n + PER - 1) / PER;
  int64_t tile = blockIdx.x;
  Packed<Tx, V> vx[U], nx[U];
  Packed<Tr, V> vr[U], nr[U];
  auto load = [&](int64_t t, Packed<Tx, V>(&px)[U], Packed<Tr, V>(&pr)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t i0 = t * PER + (u * kDropThreads + threadIdx.x) * V;
      px[u].load(x + i0);
      if (RES) pr[u].load(res + i0);
    }
  };
  if (tile < whole) load(tile, vx, vr);
  while (tile < whole) {
    const uint32_t hi = (uint32_t)((tile * PER) >> 34);
    const Philox gen(hi, a.offset, key);
    do {
      const int64_t next = tile + gridDim.x;
      if (next < whole) load(next, nx, nr);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t i0 = tile * PER + (u * kDropThreads + threadIdx.x) * V;
        float o[V];
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
          uint32_t w[4];
          gen.block((uint32_t)(i0 >> 2) + q, w);
#pragma unroll
          for (int e = 0; e < 4; e += 2) {  // a dropped value is not used, whatever it is
            const int k = q * 4 + e;
            const float2 s = __fmul2_rn(vx[u].pair(k / 2), make_float2(a.scale, a.scale));
            const float2 kept = make_float2(w[e] >= a.border ? s.x : 0.f, w[e + 1] >= a.border ? s.y : 0.f);
            const float2 r = RES ? __fadd2_rn(vr[u].pair(k / 2), kept) : kept;
            o[k] = r.x;
            o[k + 1] = r.y;
          }
        }
        store_rounded<Ty, V>(y + i0, o);
        vx[u] = nx[u];
        vr[u] = nr[u];
      }
      tile = next;
    } while (tile < whole && (uint32_t)((tile * PER) >> 34) == hi);
  }
  for (; tile < tiles; tile += gridDim.x) {
    const Philox gen((uint32_t)((tile * PER) >> 34), a.offset, key);
#pragma unroll
    for (int u = threadIdx.x; u < PER / 4; u += kDropThreads) {
      const int64_t i0 = tile * PER + u * 4;
      uint32_t w[4];
      if (i0 < a.n) gen.block((uint32_t)(i0 >> 2), w);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i0 + e < a.n) {
          const float kept = w[e] >= a.border ? Dt<Tx>::to_f(x[i0 + e]) * a.scale : 0.f;
          y[i0 + e] = Dt<Ty>::from_f(RES ? Dt<Tr>::to_f(res[i0 + e]) + kept : kept);
        }
    }
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
  const int64_t per = (int64_t)kDropThreads * drop_unroll((int)sizeof(Tx), RES ? (int)sizeof(Tr) : 0) * V;
  const int64_t tiles = (a.n + per - 1) / per;
  const int64_t grid = tiles < 148 * kDropCtas ? tiles : 148 * kDropCtas;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (words >> 32) {  // everything drops
    const size_t bytes = (size_t)n * rk_host::dtype_size(y_dtype);
    const cudaError_t e = residual ? cudaMemcpyAsync(y, residual, bytes, cudaMemcpyDeviceToDevice, s)
                                   : cudaMemsetAsync(y, 0, bytes, s);
    return e == cudaSuccess ? RK_OK : RK_ERR_LAUNCH;
  }
  a.border = (uint32_t)words;
  a.scale = (float)(1.0 / (1.0 - p));
  if (x_dtype == RK_BF16) return launch16<__nv_bfloat16>(x, residual, y, y_dtype, a, s);
  if (x_dtype == RK_F16) return launch16<__half>(x, residual, y, y_dtype, a, s);
  if (y_dtype == RK_F32)
    return residual ? launch<float, float, float, true>(x, residual, y, a, s)
                    : launch<float, float, float, false>(x, residual, y, a, s);
  if (y_dtype == RK_BF16) return launch<float, float, __nv_bfloat16, false>(x, residual, y, a, s);
  return launch<float, float, __half, false>(x, residual, y, a, s);
}
