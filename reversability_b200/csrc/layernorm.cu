// Layer norm, forward and backward.
//
//   mu = mean x, s = rsqrt(mean (x - mu)^2 + eps), n = (x - mu) s, y = n w + b
//   dx = s (g w - mean(g w) - n mean(g w n)),  dw = sum_rows g n,  db = sum_rows g
//
// Bound by memory: forward x in and y out, backward x and dy in and dx out; a
// row is read once. Forward, rows of up to 1024 elements belong to a warp,
// wider ones to a CTA with 16 (from 8192 on 32) elements a thread. Backward, a
// thread has at most 16 elements up to 8192 wide: a warp's row to 512, two
// warps' to 1024, four warps' to 2048, then a CTA's; so the column sums, x and
// dy of a row fit in registers, and a row is not read and formed again after
// its sums (32768 x 1024 bf16 on one warp and read twice 52 us, on two and kept
// 40; 512 wide 36 and 26; 8192 x 2048 on CTAs 36, on four warps, which leave
// half as many partial rows, 27). Forward rows on two or four warps were no
// faster. Warps (CTAs) walk over rows, and each lane copies its own elements of
// the next rows into shared memory asynchronously while the current row is
// summed, the mean first and then the squares about it, so a large mean costs
// no digits. (With rows loaded into registers as they were needed the backward
// of 32768 x 1024 bf16 took 152 us: eight warps an SM, each waiting for its
// row.) Arithmetic is on pairs (fp32x2), or instructions would bound it: 16-bit
// rows leave some 14 of them an element at full bandwidth, forward, and 20
// backward, about what a row formed twice takes.
//
// A lane's elements are vectors of 16 bytes of x at 16-byte boundaries, also
// where rows start between those: then the first and last vector of a row are
// used in part. The rows that a CTA visits all start equally far from a
// boundary (their distance is a multiple of 8 rows), so a lane's columns are
// the same in each, its parameters stay in registers or shared memory, and so
// do the column sums of the backward. At the end warps of a CTA add their
// sums in shared memory, CTAs leave one partial row each and a second kernel
// adds those in a fixed order: no atomics, the same bits every run.
//
// 32768 x 1024 bf16: forward 27 us (5.0 TB/s), backward with its columns 41 us
// (4.9 TB/s); 14848 x 256 fp32 to bf16: 5.9 and 11.9 us in L2; 2047 x 5001
// fp32: 16.7 (4.9 TB/s) and 39 us (3.1 TB/s; by single elements 33 and 85): a CTA
// has seven rows there, and 296 partial rows of 40 KB are written and read
// beside 123 MB of rows. Of twice the rows the backward kernel alone takes 53 us
// (4.6 TB/s) and waits for its loads first (3.5 warps of 11.5; barriers 0.9).
#include "vec.cuh"

namespace rk {

// Per-column parameters in fp32 or 16 bits; `p` null: one value everywhere.
struct NormParam {
  const void* p;
  int dtype;
};
__device__ __forceinline__ float param_at(const NormParam& q, int c, int width, float fill) {
  if (!q.p || (unsigned)c >= (unsigned)width) return fill;
  if (q.dtype == RK_F32) return __ldg(static_cast<const float*>(q.p) + c);
  if (q.dtype == RK_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(q.p)[c]);
  return __half2float(static_cast<const __half*>(q.p)[c]);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) RowPack {
  T e[V];
};

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 32) {
    copy_async<16>(dst, src);
    copy_async<16>(dst + 16, static_cast<const char*>(src) + 16);
  } else if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  } else {
    static_assert(BYTES == 8, "packs of 8, 16 or 32 bytes");
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
  }
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Starts the copy of V elements of a row from column c on into this lane's slot. `whole`: all of them lie in the
// matrix, those of an edge vector outside the row too; else what is outside the row is not touched.
template <typename T, int V>
__device__ __forceinline__ void fetch(RowPack<T, V>* slot, const T* __restrict__ row, int c, int width, bool whole) {
  if (whole) {
    copy_async<V * (int)sizeof(T)>(smem_u32(slot), row + c);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      slot->e[e] = (unsigned)(c + e) < (unsigned)width ? row[c + e] : Dt<T>::from_f(0.f);
  }
}

// Rows whose edge vectors, which reach up to V - 1 elements in front of a row and behind it, lie in the matrix: `around`
// others are on either side. (An argument of the kernel: formed in it, 2047 x 5001 fp32 takes 45 us backward in place of 38.)
struct InnerRows {
  int around;
  int64_t rows;
  __device__ __forceinline__ bool has(int64_t row) const { return row >= around && row + around < rows; }
};

// The pairs of a slot; in an edge vector what is outside the row is zero.
template <typename T, int V>
__device__ __forceinline__ void read_slot(const RowPack<T, V>* slot, bool edge, int c, int width, float2 (&v)[V / 2]) {
  const RowPack<T, V> r = *slot;
#pragma unroll
  for (int k = 0; k < V / 2; ++k) v[k] = make_float2(Dt<T>::to_f(r.e[2 * k]), Dt<T>::to_f(r.e[2 * k + 1]));
  if (edge) {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      if ((unsigned)(c + 2 * k) >= (unsigned)width) v[k].x = 0.f;
      if ((unsigned)(c + 2 * k + 1) >= (unsigned)width) v[k].y = 0.f;
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_part(T* __restrict__ row, bool edge, int c, int width, const float2 (&v)[V / 2]) {
  float o[V];
#pragma unroll
  for (int k = 0; k < V / 2; ++k) {
    o[2 * k] = v[k].x;
    o[2 * k + 1] = v[k].y;
  }
  if (!edge) {
    store_vec<T, V>(row + c, o);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if ((unsigned)(c + e) < (unsigned)width) row[c + e] = Dt<T>::from_f(o[e]);
  }
}

// Sums over the row's threads (W warps; 0: the CTA), the same values in all of them. Several warps: one barrier; `red` is
// one of several buffers used in turn, so a buffer is written again only after a barrier that follows its last read.
template <int W, bool TWO>
__device__ __forceinline__ float2 row_sums(float2 v, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    if (TWO) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (W == 1) return v;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) red[warp] = v;
  if constexpr (W > 1) {  // the row's warps only
    asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / W), "n"(32 * W) : "memory");
    if (W == 2) {
      const float2 o = red[warp ^ 1];
      return make_float2(o.x + v.x, o.y + v.y);
    }
    v = red[warp / W * W];
#pragma unroll
    for (int k = 1; k < W; ++k) {
      const float2 o = red[warp / W * W + k];
      v = make_float2(v.x + o.x, v.y + o.y);
    }
    return v;
  }
  __syncthreads();
  v = threadIdx.x % 32 < blockDim.x / 32 ? red[threadIdx.x & 31] : make_float2(0.f, 0.f);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {  // at most 16 warps
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    if (TWO) v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return make_float2(__shfl_sync(0xffffffffu, v.x, 0), TWO ? __shfl_sync(0xffffffffu, v.y, 0) : 0.f);
}

__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// Rows in flight: the one at work and up to two being copied, in at most 100 KB a CTA (the widest rows, whose
// parameters take up to 128 KB beside them: one).
__host__ __device__ constexpr int norm_depth(int elements, int bytes_per_element, bool warp) {
  const int row = elements * bytes_per_element * (warp ? 256 : 512);
  return !warp && elements > 16 ? 1 : 3 * row <= 100 * 1024 ? 3 : 2;
}
// Forward: parameters in registers (CTA rows of 16 elements a thread) or in shared memory, as they meet the lanes'
// vectors. Backward: the weight in shared memory; what its registers would hold is the row.
__host__ __device__ constexpr bool norm_param_regs(int elements, bool warp) { return !warp && elements <= 16; }

// What a thread does in every row that it visits.
template <typename Tx, int V, int NV, int W>
struct RowWalk {
  int T, t;            // threads of a row, and this one's place
  int ph;              // elements between a row's start and the 16-byte boundary (of x) before it
  int64_t row, step;
  uint32_t edge;       // bit j: vector j lies partly outside the row
  __device__ RowWalk(const Tx* x, int64_t ldx, int width) {
    T = W ? 32 * W : blockDim.x;
    t = W ? threadIdx.x % (32 * W) : threadIdx.x;
    if constexpr (W > 0) {  // a CTA's rows are equal mod 8
      row = (blockIdx.x & 7) + 8 * ((int64_t)(blockIdx.x >> 3) * (8 / W) + threadIdx.x / (32 * W));
      step = (int64_t)gridDim.x * (8 / W);
    } else {
      row = blockIdx.x;
      step = gridDim.x;
    }
    // the CTA's first row speaks for all that it visits
    const int64_t first = W ? blockIdx.x & 7 : blockIdx.x;
    ph = (int)((reinterpret_cast<uintptr_t>(x + first * ldx) / sizeof(Tx)) % V);
    edge = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (col(j) < width && (col(j) < 0 || col(j) + V > width)) edge |= 1u << j;
  }
  __device__ __forceinline__ int col(int j) const { return (j * T + t) * V - ph; }
  // Place of pair k of vector (j, t) among the parameters in shared memory: 16-byte pieces, lane beside lane.
  __device__ __forceinline__ int param(int j, int k) const { return ((j * (V / 4) + k / 2) * T + t) * 2 + k % 2; }
  // Column of the pair at place i.
  __device__ __forceinline__ int param_col(int i) const {
    const int piece = i / (2 * T), j = piece / (V / 4);
    return (j * T + i / 2 % T) * V + (piece - j * (V / 4)) * 4 + i % 2 * 2 - ph;
  }
};

template <typename Tx, typename Ty, int V, int NV, int W, int THREADS>
__global__ void __launch_bounds__(THREADS, W ? (NV * V <= 16 ? 4 : 3) : 1)
    layernorm_fwd_kernel(const Tx* __restrict__ x, int64_t ldx, const NormParam w, const NormParam b,
                         Ty* __restrict__ y, int64_t ldy, float2* __restrict__ stats, int64_t rows, int width,
                         float eps, const InnerRows within) {
  constexpr int D = norm_depth(NV * V, (int)sizeof(Tx), W), H = V / 2;
  constexpr bool REGS = norm_param_regs(NV * V, W);
  extern __shared__ uint4 shared[];  // [D][NV][threads] packs of x, then weight and bias, NV * T * V floats each
  __shared__ float2 red[W == 1 ? 1 : 4][16];
  pdl_wait();  // inputs are the previous kernel's outputs
  RowWalk<Tx, V, NV, W> r(x, ldx, width);
  RowPack<Tx, V>* mine = reinterpret_cast<RowPack<Tx, V>*>(shared) + threadIdx.x;
  float2* params = reinterpret_cast<float2*>(reinterpret_cast<RowPack<Tx, V>*>(shared) + D * NV * blockDim.x);
  auto start = [&](int64_t row, int d) {
    if (row < rows) {
      const Tx* src = x + row * ldx;
      const bool inner = within.has(row);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (r.col(j) < width)
          fetch<Tx, V>(mine + (d * NV + j) * blockDim.x, src, r.col(j), width, inner || !(r.edge >> j & 1));
    }
    copies_commit();
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (r.col(j) >= width) mine[(d * NV + j) * blockDim.x] = RowPack<Tx, V>{};
#pragma unroll
  for (int d = 0; d < D - 1; ++d) start(r.row + d * r.step, d);
  float2 wr[REGS ? NV : 1][H], br[REGS ? NV : 1][H];
  if constexpr (REGS) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const int c = r.col(j) + 2 * k;
        wr[j][k] = make_float2(param_at(w, c, width, 1.f), param_at(w, c + 1, width, 1.f));
        br[j][k] = make_float2(param_at(b, c, width, 0.f), param_at(b, c + 1, width, 0.f));
      }
  } else {
    for (int i = threadIdx.x; i < NV * r.T * H; i += blockDim.x) {
      const int c = r.param_col(i);
      params[i] = make_float2(param_at(w, c, width, 1.f), param_at(w, c + 1, width, 1.f));
      params[NV * r.T * H + i] = make_float2(param_at(b, c, width, 0.f), param_at(b, c + 1, width, 0.f));
    }
    __syncthreads();
  }
  const float inv = 1.f / (float)width;
  int d = 0, turn = 0;
  for (int64_t row = r.row; row < rows; row += r.step, turn ^= 1) {
    start(row + (D - 1) * r.step, d == 0 ? D - 1 : d - 1);
    copies_wait<D - 1>();
    float2 v[NV][H];
    float2 sum = both(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      read_slot<Tx, V>(mine + (d * NV + j) * blockDim.x, r.edge >> j & 1, r.col(j), width, v[j]);
#pragma unroll
      for (int k = 0; k < H; ++k) sum = __fadd2_rn(sum, v[j][k]);
    }
    const float mean = row_sums<W, false>(make_float2(sum.x + sum.y, 0.f), red[W == 1 ? 0 : 2 * turn]).x * inv;
    float2 sq = both(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int k = 0; k < H; ++k) v[j][k] = __fadd2_rn(v[j][k], both(-mean));
      if (r.col(j) >= width || (r.edge >> j & 1)) {
#pragma unroll
        for (int k = 0; k < H; ++k) {
          if ((unsigned)(r.col(j) + 2 * k) >= (unsigned)width) v[j][k].x = 0.f;
          if ((unsigned)(r.col(j) + 2 * k + 1) >= (unsigned)width) v[j][k].y = 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < H; ++k) sq = __ffma2_rn(v[j][k], v[j][k], sq);
    }
    const float rstd =
        rsqrtf(row_sums<W, false>(make_float2(sq.x + sq.y, 0.f), red[W == 1 ? 0 : 2 * turn + 1]).x * inv + eps);
    if (stats && r.t == 0) stats[row] = make_float2(mean, rstd);
    Ty* dst = y + row * ldy;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (r.col(j) >= width) break;
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const int at = r.param(j, k);
        v[j][k] = __ffma2_rn(__fmul2_rn(v[j][k], both(rstd)), REGS ? wr[j][k] : params[at],
                             REGS ? br[j][k] : params[NV * r.T * H + at]);
      }
      store_part<Ty, V>(dst, r.edge >> j & 1, r.col(j), width, v[j]);
    }
    d = d + 1 == D ? 0 : d + 1;
  }
  copies_wait<0>();
}

// partial: [gridDim.x][2][width] fp32 (dw, then db), or null when neither is wanted; dx may be null.
template <typename Tx, typename Tg, int V, int NV, int W, int THREADS>
__global__ void __launch_bounds__(THREADS, W > 1 ? 2 : W ? (NV * V <= 8 ? 3 : 2) : 1)
    layernorm_bwd_kernel(const Tx* __restrict__ x, int64_t ldx, const NormParam w, const float2* __restrict__ stats,
                         const Tg* __restrict__ dy, int64_t lddy, Tx* __restrict__ dx, int64_t lddx,
                         float* __restrict__ partial, int64_t rows, int width, const InnerRows within) {
  constexpr int D = norm_depth(NV * V, (int)(sizeof(Tx) + sizeof(Tg)), W), H = V / 2;
  constexpr bool KEEP = NV * V <= 16;  // n and g w stay in registers over the row's sums
  // [D][NV][threads] packs of x, then of dy, then the weight; at the end (W) [8 / W][2][width] column sums
  extern __shared__ uint4 shared[];
  __shared__ float2 red[W == 1 ? 1 : 2][16];
  pdl_wait();  // inputs are the previous kernel's outputs
  RowWalk<Tx, V, NV, W> r(x, ldx, width);
  RowPack<Tx, V>* ring_x = reinterpret_cast<RowPack<Tx, V>*>(shared);
  RowPack<Tg, V>* ring_g = reinterpret_cast<RowPack<Tg, V>*>(ring_x + D * NV * blockDim.x);
  float2* params = reinterpret_cast<float2*>(ring_g + D * NV * blockDim.x);
  RowPack<Tx, V>* mine_x = ring_x + threadIdx.x;
  RowPack<Tg, V>* mine_g = ring_g + threadIdx.x;
  auto start = [&](int64_t row, int d) {
    if (row < rows) {
      const Tx* src = x + row * ldx;
      const Tg* src_g = dy + row * lddy;
      const bool inner = within.has(row);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (r.col(j) < width) {
          fetch<Tx, V>(mine_x + (d * NV + j) * blockDim.x, src, r.col(j), width, inner || !(r.edge >> j & 1));
          fetch<Tg, V>(mine_g + (d * NV + j) * blockDim.x, src_g, r.col(j), width, inner || !(r.edge >> j & 1));
        }
    }
    copies_commit();
  };
#pragma unroll
  for (int d = 0; d < D; ++d)
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (r.col(j) >= width) {
        mine_x[(d * NV + j) * blockDim.x] = RowPack<Tx, V>{};
        mine_g[(d * NV + j) * blockDim.x] = RowPack<Tg, V>{};
      }
#pragma unroll
  for (int d = 0; d < D - 1; ++d) start(r.row + d * r.step, d);
  for (int i = threadIdx.x; i < NV * r.T * H; i += blockDim.x)
    params[i] = make_float2(param_at(w, r.param_col(i), width, 1.f), param_at(w, r.param_col(i) + 1, width, 1.f));
  __syncthreads();
  float2 dw[NV][H], db[NV][H];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < H; ++k) dw[j][k] = db[j][k] = both(0.f);
  const float inv = 1.f / (float)width;
  float2 next = r.row < rows ? __ldg(stats + r.row) : both(0.f);
  int d = 0, turn = 0;
  for (int64_t row = r.row; row < rows; row += r.step, turn ^= 1) {
    const float2 st = next;
    if (row + r.step < rows) next = __ldg(stats + row + r.step);
    start(row + (D - 1) * r.step, d == 0 ? D - 1 : d - 1);
    copies_wait<D - 1>();
    const float2 rs = both(st.y), mu = both(-st.x);
    float2 s1 = both(0.f), s2 = both(0.f);
    float2 kept_n[KEEP ? NV : 1][H], kept_g[KEEP ? NV : 1][H];
#pragma unroll
    for (int j = 0; j < NV; ++j) {  // outside the row g = 0 (and x, but for edges of rows with a mean that is not finite)
      float2 xv[H], gv[H];
      float2(&nk)[H] = kept_n[KEEP ? j : 0];
      float2(&gk)[H] = kept_g[KEEP ? j : 0];
      const bool edge = r.edge >> j & 1;
      read_slot<Tx, V>(mine_x + (d * NV + j) * blockDim.x, edge, r.col(j), width, xv);
      read_slot<Tg, V>(mine_g + (d * NV + j) * blockDim.x, edge, r.col(j), width, gv);
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const float2 n = __fmul2_rn(__fadd2_rn(xv[k], mu), rs);
        const float2 gw = __fmul2_rn(gv[k], params[r.param(j, k)]);
        if (KEEP) {
          nk[k] = n;
          gk[k] = gw;
        }
        s1 = __fadd2_rn(s1, gw);
        s2 = __ffma2_rn(gw, n, s2);
        dw[j][k] = __ffma2_rn(gv[k], n, dw[j][k]);
        db[j][k] = __fadd2_rn(db[j][k], gv[k]);
      }
    }
    if (dx) {
      const float2 m = row_sums<W, true>(make_float2(s1.x + s1.y, s2.x + s2.y), red[W == 1 ? 0 : turn]);
      if (!KEEP) asm volatile("" ::: "memory");  // the row is read from shared memory again: kept, it would spill
      // dx = s g w - s m1 - s m2 n
      const float2 a = both(-st.y * (m.x * inv)), c2 = both(-st.y * (m.y * inv));
      Tx* dst = dx + row * lddx;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (r.col(j) >= width) break;
        float2 xv[H], gv[H];
        const bool edge = r.edge >> j & 1;
        if (!KEEP) {
          read_slot<Tx, V>(mine_x + (d * NV + j) * blockDim.x, false, 0, width, xv);
          read_slot<Tg, V>(mine_g + (d * NV + j) * blockDim.x, false, 0, width, gv);
        }
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const float2 n = KEEP ? kept_n[KEEP ? j : 0][k] : __fmul2_rn(__fadd2_rn(xv[k], mu), rs);
          const float2 gw = KEEP ? kept_g[KEEP ? j : 0][k] : __fmul2_rn(gv[k], params[r.param(j, k)]);
          xv[k] = __ffma2_rn(gw, rs, __ffma2_rn(n, c2, a));
        }
        store_part<Tx, V>(dst, edge, r.col(j), width, xv);
      }
    }
    d = d + 1 == D ? 0 : d + 1;
  }
  copies_wait<0>();
  if (!partial) return;
  float* out = partial + (int64_t)blockIdx.x * 2 * width;
  float* sums = reinterpret_cast<float*>(shared) + threadIdx.x / (32 * (W ? W : 1)) * 2 * width;
  if (W) __syncthreads();  // ring and weight are not read any more
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int c = r.col(j) + e;
      if ((unsigned)c < (unsigned)width) {
        (W ? sums : out)[c] = e & 1 ? dw[j][e / 2].y : dw[j][e / 2].x;
        (W ? sums : out)[width + c] = e & 1 ? db[j][e / 2].y : db[j][e / 2].x;
      }
    }
  if (!W) return;
  __syncthreads();
  for (int c = threadIdx.x; c < 2 * width; c += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 8 / (W ? W : 1); ++k) s += reinterpret_cast<float*>(shared)[k * 2 * width + c];
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

constexpr int kMaxWidth = 16384;  // 32 elements a thread, 512 threads (from the boundary before a row to the one behind)
constexpr int kCtaWidth = 8192;   // 16 elements a thread, 512 threads

// Threads of a row's CTA: `per` elements each, whole warps.
int cta_threads(int64_t elements, int per) { return (int)((elements + per * 32 - 1) / (per * 32) * 32); }

// CTAs for warps' rows, `at_once` a CTA, at most `most` CTAs: a multiple of 8.
int64_t warp_ctas(int64_t rows, int64_t most, int at_once) {
  const int64_t want = (rows + 8 * at_once - 1) / (8 * at_once) * 8;
  return want < most / 8 * 8 ? want : most / 8 * 8;
}

// Threads that an SM holds at 96 registers, where that is another CTA of rows than at the 128 that CTA rows of 16
// elements a thread would rather have (2047 x 5001 fp32 forward 16.7 us, at 128 registers 22.8; 8192 x 4096 bf16, two CTAs
// either way, 33.0 and 31.3, and backward 65 and 52).
constexpr int kHeld = 640;
bool held_pays(int threads) { return kHeld / threads > 512 / threads; }

// CTAs of the backward for rows of `span` elements from boundary to boundary: as many as the SMs hold at once, so
// partial rows stay few; a multiple of 8 where a CTA visits more than one row.
int64_t bwd_ctas(int64_t rows, int64_t span) {
  if (span <= 512) return warp_ctas(rows, 148 * (span <= 256 ? 3 : 2), 8);
  if (span <= 1024) return warp_ctas(rows, 148 * 2, 4);
  if (span <= 2048) return warp_ctas(rows, 148 * 2, 2);
  const int64_t most = 148 * (span <= kCtaWidth ? kHeld / cta_threads(span, 16) : 1) / 8 * 8;
  return rows < most ? rows : most;
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
  int span;  // elements between the boundaries around a row, at most
  float eps;
  bool backward;
  cudaStream_t s;
};

// One row on either side, unless rows are closer together than V - 1 elements.
InnerRows inner_rows(const NormArgs& a, int64_t v) {
  if (a.rows <= 1) return {1, 0};
  const int64_t ld = a.backward && a.lddy < a.ldx ? a.lddy : a.ldx;
  return {(int)(ld >= v - 1 ? 1 : (v - 2 + ld) / ld), a.rows};
}

template <typename Tx, typename Ty, int V, int NV, int W, int THREADS = W ? 256 : 512>
int launch_fwd(const NormArgs& a) {
  const int threads = W ? THREADS : cta_threads(a.span, NV * V);
  if constexpr (W == 0 && NV * V == 16 && THREADS != kHeld)
    if (held_pays(threads)) return launch_fwd<Tx, Ty, V, NV, 0, kHeld>(a);
  const size_t params = norm_param_regs(NV * V, W) ? 0 : (size_t)NV * V * (W ? 32 * W : threads) * 4;
  auto kern = layernorm_fwd_kernel<Tx, Ty, V, NV, W, THREADS>;
  const int bytes = NV * V * (int)sizeof(Tx);
  const size_t smem = (size_t)norm_depth(NV * V, (int)sizeof(Tx), W) * bytes * threads + 2 * params;
  if (smem > 46 * 1024)  // beside 1 KB of row sums
    if (const int e = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), (int)smem)) return e;
  const int64_t fit = 227 * 1024 / (int64_t)(smem + 2048), held = (W ? NV * V <= 16 ? 1024 : 768 : THREADS) / threads;
  const int64_t most = 148 * (fit < held ? fit : held);
  const int64_t grid = W ? warp_ctas(a.rows, most, 8) : a.rows < most ? a.rows : most / 8 * 8;
  rk_host::launch_k(kern, (unsigned)grid, threads, smem, a.s, static_cast<const Tx*>(a.x), a.ldx, a.w, a.b,
                    static_cast<Ty*>(a.out), a.ldo, a.stats, a.rows, a.width, a.eps, inner_rows(a, V));
  return rk_host::launch_status();
}

template <typename Tx, typename Tg, int V, int NV, int W, int THREADS = W ? 256 : 512>
int launch_bwd(const NormArgs& a) {
  const int threads = W ? THREADS : cta_threads(a.span, NV * V);
  if constexpr (W == 0 && NV * V == 16 && THREADS != kHeld)
    if (held_pays(threads)) return launch_bwd<Tx, Tg, V, NV, 0, kHeld>(a);
  auto kern = layernorm_bwd_kernel<Tx, Tg, V, NV, W, THREADS>;
  const int bytes = NV * V * (int)(sizeof(Tx) + sizeof(Tg));
  size_t smem = (size_t)norm_depth(NV * V, (int)(sizeof(Tx) + sizeof(Tg)), W) * bytes * threads +
                (size_t)NV * V * (W ? 32 * W : threads) * 4;
  const size_t sums = (size_t)(W ? 16 / (W ? W : 1) : 0) * a.width * 4;
  if (smem < sums) smem = sums;
  if (smem > 46 * 1024)
    if (const int e = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), (int)smem)) return e;
  rk_host::launch_k(kern, (unsigned)bwd_ctas(a.rows, a.span), threads, smem, a.s, static_cast<const Tx*>(a.x), a.ldx, a.w,
                    a.stats, static_cast<const Tg*>(a.dy), a.lddy, static_cast<Tx*>(a.out), a.ldo, a.partial, a.rows,
                    a.width, inner_rows(a, V));
  return rk_host::launch_status();
}

template <typename Tx, typename To>
int dispatch(const NormArgs& a) {
  constexpr int V = 16 / (int)sizeof(Tx);
  if (a.backward) {
    if (a.span <= 32 * V) return launch_bwd<Tx, To, V, 1, 1>(a);
    if (a.span <= 64 * V) return launch_bwd<Tx, To, V, 2, 1>(a);
    if constexpr (V == 4)
      if (a.span <= 128 * V) return launch_bwd<Tx, To, V, 4, 1>(a);
    if (a.span <= 1024) return launch_bwd<Tx, To, V, 16 / V, 2>(a);
    if (a.span <= 2048) return launch_bwd<Tx, To, V, 16 / V, 4>(a);
    if (a.span <= kCtaWidth) return launch_bwd<Tx, To, V, 16 / V, 0>(a);
    return launch_bwd<Tx, To, V, 32 / V, 0>(a);
  }
  if (a.span <= 32 * V) return launch_fwd<Tx, To, V, 1, 1>(a);
  if (a.span <= 64 * V) return launch_fwd<Tx, To, V, 2, 1>(a);
  if (a.span <= 128 * V) return launch_fwd<Tx, To, V, 4, 1>(a);
  if constexpr (V == 4)
    if (a.span <= 1024) return launch_fwd<Tx, To, V, 8, 1>(a);
  if (a.span <= kCtaWidth) return launch_fwd<Tx, To, V, 16 / V, 0>(a);
  return launch_fwd<Tx, To, V, 32 / V, 0>(a);
}

// x in fp32: the other side in any type; x in 16 bits: the same type or fp32.
int dispatch_types(const NormArgs& a, int x_dtype, int o_dtype) {
  if (x_dtype == RK_F32) {
    if (o_dtype == RK_F32) return dispatch<float, float>(a);
    if (o_dtype == RK_BF16) return dispatch<float, __nv_bfloat16>(a);
    return dispatch<float, __half>(a);
  }
  if (x_dtype == RK_BF16) {
    if (o_dtype == RK_BF16) return dispatch<__nv_bfloat16, __nv_bfloat16>(a);
    if (o_dtype == RK_F32) return dispatch<__nv_bfloat16, float>(a);
  } else {
    if (o_dtype == RK_F16) return dispatch<__half, __half>(a);
    if (o_dtype == RK_F32) return dispatch<__half, float>(a);
  }
  return RK_ERR_DTYPE;
}

bool types_ok(int x_dtype, int o_dtype, int p_dtype) {
  return rk_host::dtype_ok(x_dtype) && rk_host::dtype_ok(o_dtype) && rk_host::dtype_ok(p_dtype) &&
         (x_dtype == RK_F32 || o_dtype == RK_F32 || x_dtype == o_dtype);
}

// Whether every row of `p` (row stride ld) is as far from a boundary, in elements, as the row of x.
bool same_phase(const void* x, int64_t ldx, int x_dtype, const void* p, int64_t ld, int dtype, int64_t rows) {
  const int64_t size = (int64_t)rk_host::dtype_size(x_dtype), other = (int64_t)rk_host::dtype_size(dtype), v = 16 / size;
  if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(p) % other) return false;
  const int64_t a = (int64_t)(reinterpret_cast<uintptr_t>(x) / size), b = (int64_t)(reinterpret_cast<uintptr_t>(p) / other);
  return a % v == b % v && (rows <= 1 || ldx % v == ld % v);
}

// Elements between the 16-byte boundaries around a row: all rows start equally far from one, or anywhere.
int row_span(const void* x, int64_t ldx, int x_dtype, int64_t rows, int64_t width) {
  const int64_t size = (int64_t)rk_host::dtype_size(x_dtype), v = 16 / size;
  const int64_t ph = rows <= 1 || ldx % v == 0 ? (int64_t)(reinterpret_cast<uintptr_t>(x) / size) % v : v - 1;
  return (int)((width + ph + v - 1) / v * v);
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
  if (!same_phase(x, ldx, x_dtype, y, ldy, y_dtype, rows)) return RK_ERR_ALIGN;
  NormArgs a{};
  a.x = x;
  a.ldx = ldx;
  a.w = NormParam{w, param_dtype};
  a.b = NormParam{b, param_dtype};
  a.out = y;
  a.ldo = ldy;
  a.stats = reinterpret_cast<float2*>(stats);
  a.rows = rows;
  a.width = (int)width;
  a.span = row_span(x, ldx, x_dtype, rows, width);
  if (a.span > kMaxWidth) return RK_ERR_UNSUPPORTED;
  a.eps = eps;
  a.s = static_cast<cudaStream_t>(stream);
  return dispatch_types(a, x_dtype, y_dtype);
}

extern "C" int64_t rk_layernorm_bwd_workspace(int64_t rows, int64_t width) {
  if (rows <= 0 || width <= 0) return 0;
  const int64_t a = bwd_ctas(rows, width), b = bwd_ctas(rows, width + 14);  // the spans there may be
  return (a > b ? a : b) * 2 * width * (int64_t)sizeof(float);
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
  int parts = 0;  // no rows: the columns' sums are zeros
  if (rows && (dx || columns)) {
    if (!same_phase(x, ldx, x_dtype, dy, lddy, dy_dtype, rows) ||
        (dx && !same_phase(x, ldx, x_dtype, dx, lddx, x_dtype, rows)))
      return RK_ERR_ALIGN;
    NormArgs a{};
    a.backward = true;
    a.x = x;
    a.ldx = ldx;
    a.dy = dy;
    a.lddy = lddy;
    a.w = NormParam{w, param_dtype};
    a.out = dx;
    a.ldo = lddx;
    a.stats = const_cast<float2*>(reinterpret_cast<const float2*>(stats));
    a.partial = columns ? workspace : nullptr;
    a.rows = rows;
    a.width = (int)width;
    a.span = row_span(x, ldx, x_dtype, rows, width);
    if (a.span > kMaxWidth) return RK_ERR_UNSUPPORTED;
    a.s = s;
    parts = (int)bwd_ctas(rows, a.span);
    const int st = dispatch_types(a, x_dtype, dy_dtype);
    if (st != RK_OK) return st;
  }
  if (!columns) return RK_OK;
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
