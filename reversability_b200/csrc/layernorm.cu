// Layer norm, forward and backward.
//
//   mu = mean x, s = rsqrt(mean (x - mu)^2 + eps), n = (x - mu) s, y = n w + b
//   dx = s (g w - mean(g w) - n mean(g w n)),  dw = sum_rows g n,  db = sum_rows g
//
// Bound by memory: forward x in and y out, backward x and dy in and dx out; a
// row is read once and stays in registers (packed as it was read) through its
// sums, the mean first and then the squares about it, so a large mean costs
// no digits. Rows of up to 1024 elements belong to a warp, wider ones to a
// CTA with 16 elements a thread. The column sums of the backward stay in
// registers over all rows that a warp (CTA) visits; warps of a CTA add theirs
// in shared memory, CTAs leave one partial row each and a second kernel adds
// those in a fixed order: no atomics, the same bits every run.
#include "vec.cuh"

namespace rk {

// Per-column parameters in fp32 or the activations' type; `p` null: the value `fill` everywhere.
struct NormParam {
  const void* p;
  int dtype;
  int vec;  // the base allows vector loads
};

template <typename T, int V>
struct alignas(sizeof(T) * V) RowPack {
  T e[V];
};

// V elements of a row from column c on, zero behind the row's end; read once, so L1 keeps the parameters instead.
template <typename T, int V>
__device__ __forceinline__ RowPack<T, V> load_pack(const T* __restrict__ row, int c, int width) {
  RowPack<T, V> r;
  if (V > 1 && c + V <= width) {
    static_assert(V == 1 || sizeof(T) * V == 16, "packs of 16 bytes");
    uint32_t* d = reinterpret_cast<uint32_t*>(&r);
    if constexpr (V > 1)
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                   : "l"(row + c));
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) r.e[e] = c + e < width ? row[c + e] : Dt<T>::from_f(0.f);
  }
  return r;
}

template <int V, typename T>
__device__ __forceinline__ void param_vec(const T* p, bool vec, int c, int width, float fill, float (&o)[V]) {
  if (vec && c + V <= width) {
    load_vec<T, V>(p + c, o);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = c + e < width ? Dt<T>::to_f(p[c + e]) : fill;
  }
}
template <int V>
__device__ __forceinline__ void load_param(const NormParam& q, int c, int width, float fill, float (&o)[V]) {
  if (!q.p) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = fill;
  } else if (q.dtype == RK_F32) {
    param_vec<V>(static_cast<const float*>(q.p), q.vec, c, width, fill, o);
  } else if (q.dtype == RK_BF16) {
    param_vec<V>(static_cast<const __nv_bfloat16*>(q.p), q.vec, c, width, fill, o);
  } else {
    param_vec<V>(static_cast<const __half*>(q.p), q.vec, c, width, fill, o);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_part(T* __restrict__ row, int c, int width, const float (&v)[V]) {
  if (c + V <= width) {
    store_vec<T, V>(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (c + e < width) row[c + e] = Dt<T>::from_f(v[e]);
  }
}

__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the row's threads, the same value in all of them. CTA rows: one barrier; `red` is one of several buffers
// used in turn, so a buffer is written again only after a barrier that follows its last read.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = lanes_sum(v);
  if (WARP) return v;
  const int warps = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_sum((int)(threadIdx.x & 31) < warps ? red[threadIdx.x & 31] : 0.f);
}

template <typename Tx, typename Ty, int V, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
    layernorm_fwd_kernel(const Tx* __restrict__ x, int64_t ldx, const NormParam w, const NormParam b,
                         Ty* __restrict__ y, int64_t ldy, float2* __restrict__ stats, int64_t rows, int width,
                         float eps) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ float red[WARP ? 1 : 2][32];
  const int T = WARP ? 32 : blockDim.x;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= rows) return;
  RowPack<Tx, V> v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) v[j] = load_pack<Tx, V>(x + row * ldx, (j * T + t) * V, width);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) sum += Dt<Tx>::to_f(v[j].e[e]);
  const float mean = row_sum<WARP>(sum, red[0]) / (float)width;
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float d = Dt<Tx>::to_f(v[j].e[e]) - mean;
      if ((j * T + t) * V + e < width) sq += d * d;
    }
  const float rstd = rsqrtf(row_sum<WARP>(sq, red[WARP ? 0 : 1]) / (float)width + eps);
  if (stats && t == 0) stats[row] = make_float2(mean, rstd);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * T + t) * V;
    if (c >= width) break;
    float wv[V], bv[V], o[V];
    load_param<V>(w, c, width, 1.f, wv);
    load_param<V>(b, c, width, 0.f, bv);
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = fmaf((Dt<Tx>::to_f(v[j].e[e]) - mean) * rstd, wv[e], bv[e]);
    store_part<Ty, V>(y + row * ldy, c, width, o);
  }
}

// partial: [gridDim.x][2][width] fp32 (dw, then db), or null when neither is wanted; dx may be null.
template <typename Tx, typename Tg, int V, int NV, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
    layernorm_bwd_kernel(const Tx* __restrict__ x, int64_t ldx, const NormParam w, const float2* __restrict__ stats,
                         const Tg* __restrict__ dy, int64_t lddy, Tx* __restrict__ dx, int64_t lddx,
                         float* __restrict__ partial, int64_t rows, int width) {
  pdl_wait();  // inputs are the previous kernel's outputs
  extern __shared__ float shared[];  // WARP: [8][2][width] column sums; else 4 x 32 row sums
  const int T = WARP ? 32 : blockDim.x;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t first = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = WARP ? (int64_t)gridDim.x * 8 : gridDim.x;
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[j][e] = db[j][e] = 0.f;
  int turn = 0;
  for (int64_t row = first; row < rows; row += step, turn ^= 1) {
    RowPack<Tx, V> xv[NV];
    RowPack<Tg, V> gv[NV];
    const float2 st = __ldg(stats + row);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * V;
      xv[j] = load_pack<Tx, V>(x + row * ldx, c, width);
      if constexpr (V == 1 || sizeof(Tg) * V == 16) {
        gv[j] = load_pack<Tg, V>(dy + row * lddy, c, width);
      } else {  // a pack of x spans half of or two 16-byte packs of dy
        float f[V];
        if (c + V <= width) {
          load_vec<Tg, V>(dy + row * lddy + c, f);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) f[e] = c + e < width ? Dt<Tg>::to_f(dy[row * lddy + c + e]) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) gv[j].e[e] = Dt<Tg>::from_f(f[e]);
      }
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (j * T + t) * V;
      float wv[V];
      load_param<V>(w, c, width, 1.f, wv);
#pragma unroll
      for (int e = 0; e < V; ++e) {  // behind the row's end g = 0
        const float g = Dt<Tg>::to_f(gv[j].e[e]), n = (Dt<Tx>::to_f(xv[j].e[e]) - st.x) * st.y;
        const float gw = g * wv[e];
        s1 += gw;
        s2 = fmaf(gw, n, s2);
        dw[j][e] = fmaf(g, n, dw[j][e]);
        db[j][e] += g;
      }
    }
    if (dx) {
      const float m1 = row_sum<WARP>(s1, shared + 64 * turn) / (float)width;
      const float m2 = row_sum<WARP>(s2, shared + 64 * turn + 32) / (float)width;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * T + t) * V;
        if (c >= width) break;
        float wv[V], o[V];
        load_param<V>(w, c, width, 1.f, wv);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float n = (Dt<Tx>::to_f(xv[j].e[e]) - st.x) * st.y;
          o[e] = st.y * (Dt<Tg>::to_f(gv[j].e[e]) * wv[e] - m1 - n * m2);
        }
        store_part<Tx, V>(dx + row * lddx, c, width, o);
      }
    }
  }
  if (!partial) return;
  float* out = partial + (int64_t)blockIdx.x * 2 * width;
  if (!WARP) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = (j * T + t) * V + e;
        if (c < width) {
          out[c] = dw[j][e];
          out[width + c] = db[j][e];
        }
      }
    return;
  }
  float* mine = shared + (threadIdx.x >> 5) * 2 * width;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = (j * T + t) * V + e;
      if (c < width) {
        mine[c] = dw[j][e];
        mine[width + c] = db[j][e];
      }
    }
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * width; c += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += shared[k * 2 * width + c];
    out[c] = s;
  }
}

// dw and db from the partial rows: a CTA owns 32 of the 2 * width columns; its 32 warps take the partial rows in
// turn, and one warp adds their sums in order.
template <typename T>
__global__ void __launch_bounds__(1024) layernorm_columns_kernel(const float* __restrict__ partial, int parts, int width,
                                                                T* __restrict__ dw, T* __restrict__ db) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ float red[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < 2 * width)
    for (int p = warp; p < parts; p += 32) s += partial[(int64_t)p * 2 * width + c];
  red[warp][lane] = s;
  __syncthreads();
  if (warp == 0 && c < 2 * width) {
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) v += red[k][lane];
    T* out = c < width ? dw : db;
    if (out) out[c < width ? c : c - width] = Dt<T>::from_f(v);
  }
}

}  // namespace rk

using namespace rk;

namespace {

constexpr int kMaxWidth = 16384;  // 16 elements a thread, 1024 threads
constexpr int kWarpWidth = 1024;  // 32 elements a lane

NormParam make_param(const void* p, int dtype, bool vec16) {
  // a vector of 4 or 8 parameters is read in 16-byte (fp32) or 8/16-byte pieces
  return NormParam{p, dtype, vec16 && rk_host::aligned(p, 16) ? 1 : 0};
}

// Threads of a row's CTA: 16 elements each (scalar rows the same), whole warps.
int cta_threads(int64_t width) { return (int)((width + 16 * 32 - 1) / (16 * 32) * 32); }

bool rows_vec(const void* p, int64_t ld, size_t size, int64_t rows, size_t bytes) {
  return rk_host::aligned(p, bytes) && (rows <= 1 || (ld * size) % bytes == 0);
}

// CTAs of the backward: as many as fit the SMs at once (rows permitting), so partial rows stay few.
int64_t bwd_ctas(int64_t rows, int64_t width) {
  const bool warp = width <= kWarpWidth;
  const int64_t most = warp ? 148 * (width <= 512 ? 4 : 2) : 148 * (width <= 4096 ? 4 : width <= 8192 ? 2 : 1);
  const int64_t want = warp ? (rows + 7) / 8 : rows;
  return want < most ? want : most;
}

struct NormArgs {
  const void *x, *dy;
  int64_t ldx, lddy;
  NormParam w, b;
  void* out;  // y or dx
  int64_t ldo;
  float2* stats;
  float* partial;
  int64_t rows;
  int width;
  float eps;
  bool backward;
  cudaStream_t s;
};

template <typename Tx, typename To, int V, int NV, bool WARP>
int launch(const NormArgs& a) {
  if (!a.backward) {
    const int64_t grid = WARP ? (a.rows + 7) / 8 : a.rows;
    if (grid >= (1ll << 31)) return RK_ERR_UNSUPPORTED;
    rk_host::launch_k(layernorm_fwd_kernel<Tx, To, V, NV, WARP>, (unsigned)grid, WARP ? 256 : cta_threads(a.width), 0, a.s,
                      static_cast<const Tx*>(a.x), a.ldx, a.w, a.b, static_cast<To*>(a.out), a.ldo, a.stats, a.rows,
                      a.width, a.eps);
    return rk_host::launch_status();
  }
  auto kern = layernorm_bwd_kernel<Tx, To, V, NV, WARP>;
  const size_t smem = WARP ? (a.partial ? (size_t)16 * a.width * 4 : 0) : 512;
  if (smem > 48 * 1024)
    if (const int e = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), (int)smem)) return e;
  rk_host::launch_k(kern, (unsigned)bwd_ctas(a.rows, a.width), WARP ? 256 : cta_threads(a.width), smem, a.s,
                    static_cast<const Tx*>(a.x), a.ldx, a.w, a.stats, static_cast<const To*>(a.dy), a.lddy,
                    static_cast<Tx*>(a.out), a.ldo, a.partial, a.rows, a.width);
  return rk_host::launch_status();
}

// Vectors of 16 bytes of x where every row allows them, single elements otherwise.
template <typename Tx, typename To>
int dispatch(const NormArgs& a, bool vec) {
  constexpr int V = 16 / (int)sizeof(Tx);
  const int w = a.width;
  if (w > kWarpWidth) {
    if (vec) return launch<Tx, To, V, 16 / V, false>(a);
    return launch<Tx, To, 1, 16, false>(a);
  }
  if (!vec) return w <= 256 ? launch<Tx, To, 1, 8, true>(a) : launch<Tx, To, 1, 32, true>(a);
  if (w <= 32 * V) return launch<Tx, To, V, 1, true>(a);
  if (w <= 64 * V) return launch<Tx, To, V, 2, true>(a);
  if constexpr (V == 4)
    if (w > 128 * V) return launch<Tx, To, V, 8, true>(a);
  return launch<Tx, To, V, 4, true>(a);
}

// x in fp32: the other side in any type; x in 16 bits: the same type or fp32.
int dispatch_types(const NormArgs& a, int x_dtype, int o_dtype, bool vec) {
  if (x_dtype == RK_F32) {
    if (o_dtype == RK_F32) return dispatch<float, float>(a, vec);
    if (o_dtype == RK_BF16) return dispatch<float, __nv_bfloat16>(a, vec);
    return dispatch<float, __half>(a, vec);
  }
  if (x_dtype == RK_BF16) {
    if (o_dtype == RK_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(a, vec);
    if (o_dtype == RK_F32) return dispatch<__nv_bfloat16, float>(a, vec);
  } else {
    if (o_dtype == RK_F16) return dispatch<__half, __half>(a, vec);
    if (o_dtype == RK_F32) return dispatch<__half, float>(a, vec);
  }
  return RK_ERR_DTYPE;
}

bool types_ok(int x_dtype, int o_dtype, int p_dtype) {
  return rk_host::dtype_ok(x_dtype) && rk_host::dtype_ok(o_dtype) && rk_host::dtype_ok(p_dtype) &&
         (x_dtype == RK_F32 || o_dtype == RK_F32 || x_dtype == o_dtype);
}

// Bytes that V elements (16 bytes of x) take on the other side: its rows must allow vectors of that size, 16 at most.
size_t other_bytes(int x_dtype, int o_dtype) {
  const size_t b = 16 / rk_host::dtype_size(x_dtype) * rk_host::dtype_size(o_dtype);
  return b < 16 ? b : 16;
}

}  // namespace

extern "C" int rk_layernorm_fwd(const void* x, int x_dtype, int64_t ldx, const void* w, const void* b, int param_dtype,
                                void* y, int y_dtype, int64_t ldy, float* stats, int64_t rows, int64_t width, float eps,
                                void* stream) {
  if (!types_ok(x_dtype, y_dtype, param_dtype)) return RK_ERR_DTYPE;
  if (rows < 0 || width <= 0 || (rows > 1 && (ldx < width || ldy < width))) return RK_ERR_ARG;
  if (width > kMaxWidth) return RK_ERR_UNSUPPORTED;
  if (rows == 0) return RK_OK;
  if (!x || !y) return RK_ERR_ARG;
  if (stats && !rk_host::aligned(stats, 8)) return RK_ERR_ALIGN;
  const bool vec = rows_vec(x, ldx, rk_host::dtype_size(x_dtype), rows, 16) &&
                   rows_vec(y, ldy, rk_host::dtype_size(y_dtype), rows, other_bytes(x_dtype, y_dtype));
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.w = make_param(w, param_dtype, vec);
  a.b = make_param(b, param_dtype, vec);
  a.out = y;
  a.ldo = ldy;
  a.stats = reinterpret_cast<float2*>(stats);
  a.rows = rows;
  a.width = (int)width;
  a.eps = eps;
  a.s = static_cast<cudaStream_t>(stream);
  return dispatch_types(a, x_dtype, y_dtype, vec);
}

extern "C" int64_t rk_layernorm_bwd_workspace(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0) return 0;
  return bwd_ctas(rows, width) * 2 * width * (int64_t)sizeof(float);
}

extern "C" int rk_layernorm_bwd(const void* x, int x_dtype, int64_t ldx, const void* w, int param_dtype,
                                const float* stats, const void* dy, int dy_dtype, int64_t lddy, void* dx, int64_t lddx,
                                void* dw, void* db, float* workspace, int64_t workspace_bytes, int64_t rows,
                                int64_t width, void* stream) {
  if (!types_ok(x_dtype, dy_dtype, param_dtype)) return RK_ERR_DTYPE;
  if (rows < 0 || width <= 0 || (rows > 1 && (ldx < width || lddy < width || (dx && lddx < width)))) return RK_ERR_ARG;
  if (width > kMaxWidth) return RK_ERR_UNSUPPORTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool columns = dw || db;
  if (rows && (!x || !dy || !stats)) return RK_ERR_ARG;
  if (rows && !rk_host::aligned(stats, 8)) return RK_ERR_ALIGN;
  if (columns && rows && (!workspace || workspace_bytes < rk_layernorm_bwd_workspace(rows, width))) return RK_ERR_WORKSPACE;
  if (rows && (dx || columns)) {
    const size_t xs = rk_host::dtype_size(x_dtype);
    const bool vec = rows_vec(x, ldx, xs, rows, 16) && (!dx || rows_vec(dx, lddx, xs, rows, 16)) &&
                     rows_vec(dy, lddy, rk_host::dtype_size(dy_dtype), rows, other_bytes(x_dtype, dy_dtype));
    NormArgs a{};
    a.backward = true;
    a.x = x;
    a.ldx = ldx;
    a.dy = dy;
    a.lddy = lddy;
    a.w = make_param(w, param_dtype, vec);
    a.out = dx;
    a.ldo = lddx;
    a.stats = const_cast<float2*>(reinterpret_cast<const float2*>(stats));
    a.partial = columns ? workspace : nullptr;
    a.rows = rows;
    a.width = (int)width;
    a.s = s;
    const int st = dispatch_types(a, x_dtype, dy_dtype, vec);
    if (st != RK_OK) return st;
  }
  if (!columns) return RK_OK;
  const int parts = rows ? (int)bwd_ctas(rows, width) : 0;  // no rows: zeros
  const unsigned grid = (unsigned)((2 * width + 31) / 32);
  if (param_dtype == RK_F32)
    rk_host::launch_k(layernorm_columns_kernel<float>, grid, 1024, 0, s, workspace, parts, (int)width,
                      static_cast<float*>(dw), static_cast<float*>(db));
  else if (param_dtype == RK_BF16)
    rk_host::launch_k(layernorm_columns_kernel<__nv_bfloat16>, grid, 1024, 0, s, workspace, parts, (int)width,
                      static_cast<__nv_bfloat16*>(dw), static_cast<__nv_bfloat16*>(db));
  else
    rk_host::launch_k(layernorm_columns_kernel<__half>, grid, 1024, 0, s, workspace, parts, (int)width,
                      static_cast<__half*>(dw), static_cast<__half*>(db));
  return rk_host::launch_status();
}
