// Cross entropy from hidden states in pieces of the vocabulary: neither the
// logits nor anything of their size outlives a piece.
//
//   z = x W^T,  loss_r = ln sum_j exp z_rj - z_r,label
//   dz = (softmax z - [j = label]) g_r,  dx = dz W,  dW = dz^T x
//
// Rows whose label is ignored are left out before anything is multiplied: the
// others are listed and gathered (a padded or masked row costs nothing, and
// what lies in it cannot spread). Forward: one GEMM over the whole vocabulary
// whose epilogue keeps a row's sum of exponentials in registers, against a
// reference that an earlier logit set (fp32 holds terms of up to 2^64 of it; at
// exponents of that size a term is off by 4e-6, which is what a loss may be off
// by), and writes no logits; a row keeps one number, its log-sum-exp. Backward,
// for each piece of the vocabulary: the logits again, turned in the epilogue
// into dz / scale (16 bits; the scale of the loss, with which fp16 would
// underflow, is applied to the fp32 results) in a workspace of rows x piece;
// then the two gradient GEMMs read it: dx adds up over the pieces in fp32, dW of
// the piece is final and leaves in its type.
//
// dz is held in 16 bits because the tensor cores take it so, and half the bytes
// of fp32 pass between the products. Its terms round independently, so sums of
// many gain little: bf16 gradients of 14848 rows are 0.0018 off their 64-bit
// values where their own rounding leaves 0.0017. dW of a handful of rows has only
// as many terms and is off by up to 0.0025. What needs more takes fp32 inputs.
//
// Bound by the tensor cores: 2 M V K operations forward, 6 M V K backward (one
// third of it the logits again). All four GEMMs are one kernel: CTA pairs
// (cta_group::2) on 256 x 256 tiles, each CTA loading its 128 rows of A and
// half of B by TMA (32 KB a 64-wide k block for 4.2 MFLOP, where a single
// CTA's 128 x 256 tile takes 48 KB and is bound by L2), one thread of the pair
// issuing tcgen05.mma into double-buffered tensor memory, sixteen epilogue
// warps a CTA. The gradient products keep the tensor pipe 86 to 88 % busy; at
// K = 256 the two with exponentials in their epilogue keep it and the
// exponential unit, both with 2048 cycles of work a tile, 65 and 53 % busy
// (290 us forward, 390 us for dz at 14848 x 50257). Not faster there: two groups
// of warps on alternate tiles (300), a part of the exponentials as polynomials
// on the FMA pipes (311 to 328). Sums over sliced reductions are added in a
// fixed order: no atomics, the same bits every run.
//
// Whole passes, forward and backward: 14848 x 50257 x 256 bf16 1.57 ms (1.53
// TFLOP with the logits formed twice: 975 TFLOP/s), 32768 x 50257 x 1024 10.9
// ms (1237 TFLOP/s under the power cap, where plain products reach 1391), 3001 x
// 32003 x 328 fp16 with half of the rows ignored 0.23 ms, one row forward 23 us.
#include <cudaTypedefs.h>
#include <mutex>
#include <type_traits>
#include "vec.cuh"

namespace rk {

constexpr int kTile = 256;  // rows and columns of a pair's output tile
constexpr int kHalf = 128;  // of them a CTA's rows of A and rows of B
constexpr int kKb = 64;     // reduction elements of a stage
constexpr float kLog2e = 1.4426950408889634f;

// STATS: running (reference, sum exp) per row; DLOGITS: dz of a piece, 16 bits; ADD: fp32 tiles stored or added, A K-major
// (dx); OUTER: fp32 with A MN-major (dW: slices of it, or scaled to where it belongs); OUTER_T: A MN-major, scaled and
// stored in 16 bits (dW).
enum { STATS = 0, DLOGITS = 1, ADD = 2, OUTER = 3, OUTER_T = 4 };

constexpr int kEpiWarps = 16;
constexpr int kCeThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kStageBytes = 2 * kHalf * kKb * 2;  // A and B of one CTA
__host__ __device__ constexpr uint32_t ce_out_bytes(int m) {
  return m == STATS ? 0 : (m == ADD || m == OUTER) ? kEpiWarps * 4096 : kEpiWarps * 2048;  // a box of 32 rows of 128 bytes a warp
}
// Row tiles of A that stay in shared memory (STATS, DLOGITS, up to `res` k blocks): only the weight streams, half of the
// bytes from L2 (14848 x 50257 x 256 1.60 -> 1.57 ms a pass; in short runs, at full clocks, no faster).
constexpr int kResKb = 4;
__host__ __device__ constexpr uint32_t ce_stage_bytes(int res) { return res ? kStageBytes / 2 : kStageBytes; }
__host__ __device__ constexpr uint32_t ce_res_bytes(int res) { return res * (kStageBytes / 2); }
// As many stages as fit. (Boxes of both chunks, 128 bytes a row, with five stages: dz of 14848 x 50257 x 256 404 us for 393.)
__host__ __device__ constexpr int ce_stages(int m, int res) {
  return (int)((224 * 1024 - ce_out_bytes(m) - ce_res_bytes(res)) / ce_stage_bytes(res));
}
__host__ __device__ constexpr uint32_t ce_smem(int m, int res) {
  return 1024 + ce_res_bytes(res) + ce_stages(m, res) * ce_stage_bytes(res) + ce_out_bytes(m) +
         (2 * ce_stages(m, res) + 8) * 8 + 16;
}

struct CeArgs {
  const int* count;  // rows that are not ignored (device memory)
  int in_place_rows;  // with this count the hidden states are read where they are (-1: never)
  int vocab, width;  // V, K
  int tiles_n;       // column tiles of the output
  int kb;            // k blocks of the reduction (ADD: of the piece; OUTER: given by count)
  int slices;        // ADD, OUTER: slices of the reduction
  int row_tiles;     // OUTER: vocabulary tiles of the piece
  int v0;            // first vocabulary entry of the piece
  int slice_rows;    // ADD, OUTER: rows between slices in the output
  int add;           // ADD: add to what is there
  float2* part;      // STATS: [unit][4 column groups][256 rows]
  float* xlabel;     // STATS: logit at the label, per listed row
  const int* label;  // labels of the listed rows
  const float2* rowc;  // DLOGITS: per listed row (-lse log2 e, factor of dz)
  const float* scale;  // OUTER_T, OUTER to dW itself
  int to_weight;       // OUTER: the output is dW, not a buffer of its tiles
  unsigned int* status;
  // STATS with loss set (few rows): the last CTA to finish joins the rows and writes lse and loss
  int* head;
  const int *pos, *rows_of;
  float *lse, *loss;
  int rows, reduction;
};
constexpr int kFewRows = 32;

// A row's sum of exponentials relative to 2^m. A sum without a reference (m = -inf) is 0, or not a number.
struct RowSum {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void add(float2 p) {
    if (p.x > m) {
      s *= m == -INFINITY ? 1.f : ex2_approx(m - p.x);
      m = p.x;
    }
    s += p.x == -INFINITY ? p.y : p.y * ex2_approx(p.x - m);
  }
  __device__ __forceinline__ void add_lanes() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
      add(make_float2(__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o)));
  }
  __device__ __forceinline__ double lse() const { return (double)m * 0.6931471805599453 + (double)logf(s); }
};

constexpr int kPairs = 74;  // CTA pairs of a B200's 148 SMs

// Segments that the vocabulary's tiles are cut into when there are tiles_m row tiles, so that waves of pairs are full: at
// most eight waves unless there are more row tiles. Called by a warp: a lane a number of waves.
__device__ __forceinline__ int stats_segments(uint32_t tiles_m, uint32_t tiles_n) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t seg = 1;
  if (lane > 0 && lane <= 8 && tiles_m > 0 && kPairs * lane >= tiles_m) seg = min(kPairs * lane / tiles_m, tiles_n);
  float cost = (float)((tiles_m * seg + kPairs - 1) / kPairs) * (float)((tiles_n + seg - 1) / seg);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float c = __shfl_xor_sync(0xffffffffu, cost, o);
    const uint32_t k = __shfl_xor_sync(0xffffffffu, seg, o);
    if (c < cost || (c == cost && k < seg)) {
      cost = c;
      seg = k;
    }
  }
  return (int)seg;
}

// The tiles that a CTA pair visits, in order. STATS: units of one row tile and a run of column tiles, so that a row's
// running values stay in registers; units of the same segment run side by side and share the weight's tiles in L2.
// DLOGITS: equal shares of the tiles, column tiles fastest (a piece of the weight stays in L2).
template <int MODE>
struct CeWalk {
  int unit, units, step, tiles_m, segments;
  int nt, nt_end;
  int m0, n0, kb0, kb1, slice;
  bool first, last;
  __device__ CeWalk(const CeArgs& g, int pair, int pairs) {
    const int rows = *g.count;
    tiles_m = (MODE == OUTER || MODE == OUTER_T) ? g.row_tiles : (rows + kTile - 1) / kTile;
    segments = 1;
    if (MODE == STATS) {
      segments = g.count[2];
      units = tiles_m * segments;
    } else {
      units = tiles_m * g.tiles_n * g.slices;
    }
    unit = pair;
    step = pairs;
    if (MODE == DLOGITS) {
      const int64_t all = units;
      unit = (int)(all * pair / pairs);
      units = (int)(all * (pair + 1) / pairs);
      step = 1;
    }
    kb_all = (MODE == OUTER || MODE == OUTER_T) ? (rows + kKb - 1) / kKb : g.kb;
    if (unit < units) begin(g);
  }
  int kb_all;
  __device__ bool more() const { return unit < units; }
  __device__ void begin(const CeArgs& g) {
    slice = 0;
    kb0 = 0;
    kb1 = kb_all;
    first = true;
    if (MODE == STATS) {  // segment-major
      const int seg = unit / tiles_m;
      m0 = (unit - seg * tiles_m) * kTile;
      nt = (int)((int64_t)seg * g.tiles_n / segments);
      nt_end = (int)((int64_t)(seg + 1) * g.tiles_n / segments);
    } else if (MODE == DLOGITS) {
      const int mt = unit / g.tiles_n;
      m0 = mt * kTile;
      nt = unit - mt * g.tiles_n;
      nt_end = nt + 1;
    } else {  // column tiles fastest: they share A's tile
      const int per = tiles_m * g.tiles_n;
      slice = unit / per;
      const int t = unit - slice * per;
      const int mt = t / g.tiles_n;
      m0 = mt * kTile;
      nt = t - mt * g.tiles_n;
      nt_end = nt + 1;
      kb0 = (int)((int64_t)slice * kb_all / g.slices);
      kb1 = (int)((int64_t)(slice + 1) * kb_all / g.slices);
    }
    n0 = nt * kTile;
    last = MODE == DLOGITS ? nt + 1 == g.tiles_n || unit + 1 == units : nt + 1 == nt_end;
  }
  __device__ void next(const CeArgs& g) {
    if (MODE == STATS && nt + 1 < nt_end) {
      ++nt;
      n0 += kTile;
      first = false;
      last = nt + 1 == nt_end;
      return;
    }
    const int row = m0;
    unit += step;
    if (unit < units) begin(g);
    if (MODE == DLOGITS) first = m0 != row;
  }
};

// Lets the next kernel's prologue start now: it still waits for this one's end before it reads anything.
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Address of this shared-memory location in the pair's first CTA.
__device__ __forceinline__ uint32_t leader_addr(uint32_t a) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(a));
  return r;
}
// Load into this CTA's shared memory, completion counted on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const void* tmap, uint32_t bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs when all MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"((uint16_t)3)
      : "memory");
}
// What it orders are reads of tensor memory, which tcgen05.fence and the barrier itself do; a release at cluster scope
// would be a full fence (the forward of 14848 x 50257 x 256 took 363 us with it).
__device__ __forceinline__ void mbar_arrive_pair(uint32_t addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void store_2d(const void* tmap, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(tmap), "r"(src),
               "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void reduce_add_2d(const void* tmap, uint32_t src, int x, int y) {
  asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   tmap),
               "r"(src), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ float chunk_max(const float* v) {
  float m = v[0];
#pragma unroll
  for (int k = 1; k < 32; ++k) m = fmaxf(m, v[k]);
  return m;
}
// Sum of exp(v) relative to 2^ref.
__device__ __forceinline__ float chunk_sum(const float* v, float ref) {
  const float2 l2 = make_float2(kLog2e, kLog2e);
  const float r = ref == -INFINITY ? 0.f : -ref;
  const float2 r2 = make_float2(r, r);
  float2 s[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float2 t = __ffma2_rn(make_float2(v[2 * k], v[2 * k + 1]), l2, r2);
    s[k & 1] = __fadd2_rn(s[k & 1], make_float2(ex2_approx(t.x), ex2_approx(t.y)));
  }
  return (s[0].x + s[1].x) + (s[0].y + s[1].y);
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t d;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// The end of a forward over at most kFewRows rows: the last CTA joins each row's partial pairs, a warp a row, and adds the
// losses. (A kernel of its own costs a launch and 4 us more of 25.)
__device__ __noinline__ void join_few_rows(const CeArgs& g) {
  __shared__ float row_loss[kFewRows];
  __shared__ int is_last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    is_last = atomicAdd(g.head + 1, 1) == (int)gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!is_last) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = *g.count, pairs = g.count[2] * 4;
  for (int r = warp; r < kFewRows; r += kCeThreads / 32) {
    float l = 0.f;
    if (r < count) {
      RowSum a;
#pragma unroll 4
      for (int k = lane; k < pairs; k += 32) a.add(__ldcg(g.part + k * kTile + r));
      a.add_lanes();
      const double total = a.lse();
      l = (float)(total - (double)__ldcg(g.xlabel + r));
      if (lane == 0) {
        g.lse[r] = (float)total;
        if (g.reduction == 0) g.loss[g.rows_of[r]] = l;
      }
    }
    if (lane == 0) row_loss[r] = l;
  }
  if (g.reduction == 0) {
    if ((int)threadIdx.x < g.rows && g.pos[threadIdx.x] < 0) g.loss[threadIdx.x] = 0.f;
    return;
  }
  __syncthreads();
  if (warp == 0) {
    double a = (double)row_loss[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if (lane == 0) g.loss[0] = (float)(g.reduction == 2 && count ? a / count : a);
  }
}

template <int MODE, typename T, int RES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kCeThreads, 1)
    ce_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmX, const CeArgs g,
                   const uint32_t idesc) {
  static_assert(RES == 0 || MODE == STATS || MODE == DLOGITS, "runs of tiles with the same rows");
  constexpr int STAGES = ce_stages(MODE, RES);
  constexpr uint32_t STAGE = ce_stage_bytes(RES);
  constexpr bool A_MN = MODE == OUTER || MODE == OUTER_T;
  constexpr bool B_MN = MODE == ADD || A_MN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;  // RES: the resident row tile
  uint8_t* sRing = smem + ce_res_bytes(RES);
  uint8_t* sOut = sRing + STAGES * STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sOut + ce_out_bytes(MODE));
  const uint32_t full0 = smem_u32(bars);           // first CTA: both CTAs' loads of a stage have landed
  const uint32_t empty0 = full0 + 8 * STAGES;      // each CTA: the MMAs reading a stage are done
  const uint32_t tfull0 = empty0 + 8 * STAGES;     // each CTA: accumulator b is complete
  const uint32_t tempty0 = tfull0 + 16;            // first CTA: both CTAs' epilogues have read accumulator b
  const uint32_t drain = tempty0 + 16;
  const uint32_t afull = drain + 8;                // RES, first CTA: both CTAs' resident rows have landed
  const uint32_t aempty = afull + 8;               // RES, each CTA: the MMAs reading them are done
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 8);
  volatile int* s_abort = reinterpret_cast<volatile int*>(s_tmem + 1);
  volatile int* s_consumed = reinterpret_cast<volatile int*>(s_tmem + 2);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull0 + 8 * b, 1);
      mbar_init(tempty0 + 8 * b, 2 * kEpiWarps);
    }
    mbar_init(drain, 1);
    mbar_init(afull, 1);
    mbar_init(aempty, 1);
    fence_mbar_init();
    *s_abort = 0;
    *s_consumed = 0;
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
    if (MODE != STATS) tma_prefetch_desc(&tmC);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(s_tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers are set up before either signals the other's
  tc_fence_after();
  const uint32_t tmem_base = *s_tmem;
  pdl_trigger();  // all CTAs of this grid are resident: the next one's take the SMs as these leave them
  pdl_wait();  // inputs are the previous kernels' outputs

  int issued = 0, issued_a = 0;
  if (warp == 0 && lane == 0) {
    // ------------------------------------------------------------ producer (each CTA its own halves)
    // hidden states: gathered, or themselves where every row is listed
    const bool in_place = *g.count == g.in_place_rows;
    const CUtensorMap* mapA = (MODE == STATS || MODE == DLOGITS) && in_place ? &tmX : &tmA;
    const CUtensorMap* mapB = A_MN && in_place ? &tmX : &tmB;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (CeWalk<MODE> w(g, pair, pairs); w.more() && ok; w.next(g)) {
      if (RES && w.first) {  // new rows, once the products of the last ones are done
        ok = mbar_wait(aempty, (uint32_t)(issued_a & 1) ^ 1, g.status, RK_DEV_GEMM_TIMEOUT, s_abort);
        if (!ok) break;
        if (rank == 0) mbar_arrive_expect_tx(afull, 2 * w.kb1 * kHalf * kKb * 2);
        for (int kb = 0; kb < w.kb1; ++kb)
          tma_load_pair(smem_u32(sA + kb * kHalf * kKb * 2), mapA, leader_addr(afull), kb * kKb, w.m0 + rank * kHalf);
        ++issued_a;
      }
      for (int kb = w.kb0; kb < w.kb1; ++kb) {
        if (!mbar_wait(empty0 + 8 * stage, phase ^ 1, g.status, RK_DEV_GEMM_TIMEOUT, s_abort)) {
          ok = false;
          break;
        }
        const uint32_t fb = leader_addr(full0 + 8 * stage);
        if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * stage, 2 * STAGE);
        const uint32_t a = smem_u32(sRing + stage * STAGE), b = RES ? a : a + kHalf * kKb * 2;
        const int k0 = kb * kKb, ra = w.m0 + rank * kHalf, rb = w.n0 + rank * kHalf;
        if constexpr (A_MN) {
          tma_load_pair(a, mapA, fb, ra, k0);
          tma_load_pair(a + 8192, mapA, fb, ra + 64, k0);
        } else if constexpr (RES == 0) {
          tma_load_pair(a, mapA, fb, k0, ra);
        }
        if constexpr (B_MN) {
          const int ky = MODE == ADD ? g.v0 + k0 : k0;
          tma_load_pair(b, mapB, fb, rb, ky);
          tma_load_pair(b + 8192, mapB, fb, rb + 64, ky);
        } else {
          tma_load_pair(b, mapB, fb, k0, g.v0 + rb);
        }
        ++issued;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    // the last stages' releases arrive before the CTA may end
    for (int i = 0; ok && i < STAGES && i < issued; ++i) {
      const int at = issued - 1 - i;
      ok = mbar_wait(empty0 + 8 * (at % STAGES), (uint32_t)((at / STAGES) & 1), g.status, RK_DEV_GEMM_TIMEOUT, s_abort);
    }
    if (RES && ok && issued_a) mbar_wait(aempty, (uint32_t)(issued_a - 1) & 1, g.status, RK_DEV_GEMM_TIMEOUT, s_abort);
  } else if (warp == 1 && lane == 0 && rank == 0) {
    // ------------------------------------------------------------ MMA issuer (the pair's first CTA)
    int stage = 0, acc = 0, consumed = 0;
    uint32_t phase = 0, acc_phase = 0, a_phase = 0;
    bool ok = true;
    for (CeWalk<MODE> w(g, pair, pairs); w.more() && ok; w.next(g)) {
      if (RES && w.first) {
        ok = mbar_wait(afull, a_phase, g.status, RK_DEV_GEMM_TIMEOUT, s_abort);
        if (!ok) break;
        a_phase ^= 1;
      }
      if (!mbar_wait(tempty0 + 8 * acc, acc_phase ^ 1, g.status, RK_DEV_GEMM_TIMEOUT, s_abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem_base + acc * kTile;
      for (int kb = w.kb0; kb < w.kb1; ++kb) {
        if (!mbar_wait(full0 + 8 * stage, phase, g.status, RK_DEV_GEMM_TIMEOUT, s_abort)) {
          ok = false;
          break;
        }
        ++consumed;
        tc_fence_after();
        const uint32_t ring = smem_u32(sRing + stage * STAGE);
        const uint32_t a = RES ? smem_u32(sA + kb * kHalf * kKb * 2) : ring, b = RES ? ring : ring + kHalf * kKb * 2;
#pragma unroll
        for (int j = 0; j < kKb / 16; ++j) {
          const uint64_t ad = A_MN ? smem_desc_sw128(a + j * 2048, 8192, 1024) : smem_desc_sw128(a + j * 32, 16, 1024);
          const uint64_t bd = B_MN ? smem_desc_sw128(b + j * 2048, 8192, 1024) : smem_desc_sw128(b + j * 32, 16, 1024);
          umma_pair(d, ad, bd, idesc, (kb > w.kb0 || j > 0) ? 1u : 0u);
        }
        umma_commit_pair(empty0 + 8 * stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      umma_commit_pair(tfull0 + 8 * acc);
      if (RES && w.last) umma_commit_pair(aempty);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    *s_consumed = consumed;
    if (!ok && consumed) {  // the MMAs already issued finish before tensor memory is released
      asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drain) : "memory");
      mbar_wait(drain, 0, g.status, RK_DEV_GEMM_TIMEOUT, nullptr);
    }
  } else if (warp >= 2) {
    // ------------------------------------------------------------ epilogue: one row a thread, 64 of the tile's columns
    const int quarter = warp & 3;       // tensor-memory lanes of this warp
    const int ew = warp - 2;
    const int cg = ew >> 2;             // its group of 64 columns
    const int local = rank * kHalf + quarter * 32 + lane;  // row of the tile
    uint8_t* buf = sOut + ew * (ce_out_bytes(MODE) / kEpiWarps);
    int acc = 0;
    uint32_t acc_phase = 0;
    const int rows = MODE == STATS || MODE == DLOGITS ? *g.count : 0;
    float run_m = -INFINITY, run_s = 0.f;  // STATS: reference and sum of exp(z - reference), z in units of log 2
    int label = -1;
    float2 rc = make_float2(0.f, 0.f);
    const bool to_weight = MODE == OUTER_T || (MODE == OUTER && g.to_weight);
    const float scale = to_weight ? *g.scale : 1.f;
    for (CeWalk<MODE> w(g, pair, pairs); w.more(); w.next(g)) {
      if ((MODE == STATS || MODE == DLOGITS) && w.first) {
        const int row = w.m0 + local;
        run_m = -INFINITY;
        run_s = 0.f;
        label = row < rows ? __ldg(g.label + row) : -1;
        if (MODE == DLOGITS) rc = row < rows ? __ldg(g.rowc + row) : make_float2(0.f, 0.f);
      }
      bool ok = mbar_wait(tfull0 + 8 * acc, acc_phase, g.status, RK_DEV_GEMM_TIMEOUT, s_abort);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * kTile + cg * 64;
      uint32_t both[2][32];
      tmem_ld_32cols_nowait(t_row, both[0]);
      tmem_ld_32cols_nowait(t_row + 32, both[1]);
      tmem_ld_wait();
      tc_fence_before();  // read: the MMA thread may reuse this accumulator
      __syncwarp();
      if (lane == 0) mbar_arrive_pair(leader_addr(tempty0 + 8 * acc));
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        uint32_t(&r)[32] = both[ch];
        const int c0 = w.n0 + cg * 64 + ch * 32;  // first column of the chunk
        float* v = reinterpret_cast<float*>(r);
        if ((MODE == ADD || A_MN) && w.kb0 >= w.kb1) {  // an empty slice: nothing was accumulated
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0u;
        }
        if constexpr (MODE == STATS) {
          const int valid = g.vocab - c0;
          if (valid < 32) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k >= valid) v[k] = -INFINITY;
          }
          const int li = label - c0;
          if (li >= 0 && li < 32) {
            float xl = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) xl = li == k ? v[k] : xl;
            g.xlabel[w.m0 + local] = xl;
          }
          // Sums are formed against a reference that some earlier logit of the row set, without looking at these first:
          // fp32 holds terms of up to 2^64, and only a sum beyond that takes a new reference (the largest logit so far).
          if (run_m == -INFINITY) run_m = chunk_max(v) * kLog2e;
          float part = chunk_sum(v, run_m);
          if (part > 0x1p64f) {
            const float m = chunk_max(v) * kLog2e;
            run_s *= ex2_approx(run_m - m);
            run_m = m;
            part = chunk_sum(v, m);
          }
          run_s += part;
        } else if constexpr (MODE == DLOGITS) {
          const float2 l2 = make_float2(kLog2e, kLog2e), ref2 = make_float2(rc.x, rc.x);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const float2 t = __ffma2_rn(make_float2(v[2 * k], v[2 * k + 1]), l2, ref2);
            v[2 * k] = ex2_approx(t.x) * rc.y;
            v[2 * k + 1] = ex2_approx(t.y) * rc.y;
          }
          const int li = label - (g.v0 + c0);
          if (li >= 0 && li < 32) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (li == k) v[k] -= rc.y;
          }
          // rows behind the last are zeros also where an infinite weight makes their products something else
          const int valid = label < 0 ? 0 : g.vocab - (g.v0 + c0);
          if (valid < 32) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (k >= valid) v[k] = 0.f;
          }
        } else if constexpr (A_MN) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] *= scale;
        }
        if constexpr (MODE != STATS) {
          constexpr bool wide = MODE == ADD || MODE == OUTER;
          if (lane == 0) stores_read();  // the warp's box is free
          __syncwarp();
          const int y = w.slice * g.slice_rows + w.m0 + rank * kHalf + quarter * 32;
          if constexpr (wide) {  // 32 rows of 128 bytes, 128-byte swizzle
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(buf + lane * 128 + ((j ^ (lane & 7)) * 16)) =
                  make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          } else {  // 32 rows of 64 bytes, 64-byte swizzle
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16)) =
                  make_uint4(pack_pair<T>(v[8 * j], v[8 * j + 1]), pack_pair<T>(v[8 * j + 2], v[8 * j + 3]),
                             pack_pair<T>(v[8 * j + 4], v[8 * j + 5]), pack_pair<T>(v[8 * j + 6], v[8 * j + 7]));
          }
          fence_proxy_async_smem();
          __syncwarp();
          const int yy = to_weight ? g.v0 + y : y;
          if (lane == 0 && (MODE == DLOGITS || (c0 < g.width && (!to_weight || yy < g.vocab)))) {
            if (MODE == ADD && g.add) reduce_add_2d(&tmC, smem_u32(buf), c0, yy);
            else store_2d(&tmC, smem_u32(buf), c0, yy);
            stores_commit();
          }
        }
      }
      if (MODE == STATS && w.last)
        g.part[((int64_t)w.unit * 4 + cg) * kTile + local] = make_float2(run_m, run_s);
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (MODE != STATS && lane == 0) stores_done();
  }
  if constexpr (MODE == STATS) {
    if (g.loss) join_few_rows(g);
  }

  __syncthreads();
  if (*s_abort && threadIdx.x == 0) {
    // Loads in flight land before shared memory is given up. The first CTA's barriers count both CTAs' loads; loads
    // that its barriers no longer follow land within the time waited here.
    if (RES && rank == 0 && issued_a)
      mbar_wait(afull, (uint32_t)(issued_a - 1) & 1, g.status, RK_DEV_GEMM_TIMEOUT, nullptr);
    if (rank == 0)
      for (int i = *s_consumed; i < issued; ++i)
        mbar_wait(full0 + 8 * (i % STAGES), (uint32_t)((i / STAGES) & 1), g.status, RK_DEV_GEMM_TIMEOUT, nullptr);
    const uint64_t t0 = globaltimer();
    while (globaltimer() - t0 < 1000000ull) {
    }
  }
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still signal or read it
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem_base) : "memory");
  }
}

// ---------------------------------------------------------------- rows
// One row of 16-bit elements to a 16-byte boundary, by a warp. The source may start anywhere: a vector of the result is cut
// out of the two aligned ones that hold it, unless those reach behind the array's end or before its start.
__device__ __forceinline__ void copy_row(const uint16_t* __restrict__ src, uint16_t* __restrict__ dst, int width,
                                         const uint16_t* first, const uint16_t* end) {
  const int shift = (int)(reinterpret_cast<uintptr_t>(src) & 15) / 2;  // elements behind a boundary
  for (int c = (threadIdx.x & 31) * 8; c < width; c += 256) {
    const uint16_t* lo = src + c - shift;
    if (lo >= first && lo + (shift ? 16 : 8) <= end) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(lo));
      uint4 o = a;
      if (shift) {
        const uint4 b = __ldg(reinterpret_cast<const uint4*>(lo) + 1);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t x = 0, y = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q)  // words (shift / 2 + k) and the one behind it
            if (q == shift >> 1) {
              x = w[q + k];
              y = w[q + k + 1];
            }
          r[k] = shift & 1 ? __funnelshift_r(x, y, 16) : x;
        }
        o = make_uint4(r[0], r[1], r[2], r[3]);
      }
      *reinterpret_cast<uint4*>(dst + c) = o;  // the pitch has room for whole vectors
    } else {
      for (int e = 0; e < 8 && c + e < width; ++e) dst[c + e] = src[c + e];
    }
  }
}

// Hidden states that the listing kernel gathers itself (forward, few rows; rows behind the last are left as they are: a
// row's logits depend on no other row).
struct FewRows {
  const uint16_t* x;  // null: not this kernel's business
  int64_t ldx, pitch;
  int width, in_place_rows;
  uint16_t* out;
};

// CTAS CTAs (one, or a cluster) list the rows whose label counts: pos[r] = place in the list or -1, label[i] and
// rows_of[i] of listed row i. Labels outside [0, vocab) that are not ignore_index set an error bit and count as ignored.
// Each warp has its share of the rows and reads it twice, to count and to write; a row's place is the number of those
// that count before it, the other CTAs' part of that read from their shared memory.
template <int CTAS>
__global__ void __launch_bounds__(1024)
    ce_list_kernel(const int64_t* __restrict__ labels, int64_t rows, int64_t vocab, int64_t ignore, int* __restrict__ head,
                   int* __restrict__ pos, int* __restrict__ label, int* __restrict__ rows_of, unsigned int* status,
                   const FewRows few) {
  pdl_trigger();
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ int sums[32];
  __shared__ int total;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int rank = CTAS > 1 ? (int)cluster_rank() : 0;
  const int64_t each = (rows + 1024 * CTAS - 1) / (1024 * CTAS) * 32;  // a warp's rows
  const int64_t from = (rank * 32 + warp) * each, to = from + each < rows ? from + each : rows;
  bool bad = false;
  int n = 0;
#pragma unroll 4
  for (int64_t r = from + lane; r < to; r += 32) {
    const int64_t v = __ldg(labels + r);
    const bool counts = v != ignore && v >= 0 && v < vocab;
    bad |= v != ignore && !counts;
    n += counts;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) sums[warp] = n;
  __syncthreads();
  int before = sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  int all = __shfl_sync(0xffffffffu, before, 31);
  int at = __shfl_sync(0xffffffffu, before, warp) - n;
  if constexpr (CTAS > 1) {
    if (threadIdx.x == 0) total = all;
    cluster_sync();
    all = 0;
#pragma unroll
    for (int c = 0; c < CTAS; ++c) {
      int v;
      asm volatile(
          "{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.u32 %0, [a];\n\t}"
          : "=r"(v)
          : "r"(smem_u32(&total)), "r"(c)
          : "memory");
      all += v;
      if (c < rank) at += v;
    }
  }
#pragma unroll 4
  for (int64_t r = from; r < to; r += 32) {
    const int64_t v = r + lane < to ? __ldg(labels + r + lane) : ignore;
    const bool counts = v != ignore && v >= 0 && v < vocab;
    const uint32_t votes = __ballot_sync(0xffffffffu, counts);
    const int i = at + __popc(votes & ((1u << lane) - 1u));
    if (r + lane < to) pos[r + lane] = counts ? i : -1;
    if (counts) {
      label[i] = (int)v;
      rows_of[i] = (int)(r + lane);
    }
    at += __popc(votes);
  }
  if (bad) flag_error(status, RK_DEV_CE_LABEL);
  if (warp == 0 && rank == 0) {
    const int segments = stats_segments((all + kTile - 1) / kTile, (uint32_t)((vocab + kTile - 1) / kTile));
    if (lane == 0) {
      head[0] = all;
      head[1] = 0;  // CTAs of the finish kernel that are done
      head[2] = segments;
    }
  }
  if constexpr (CTAS > 1) {
    cluster_sync();  // the others may still read this CTA's total
  } else if (few.x && all != few.in_place_rows) {
    __syncthreads();
    const uint16_t* behind = few.x + (rows - 1) * few.ldx + few.width;
    for (int i = warp; i < all; i += 32)
      copy_row(few.x + (int64_t)rows_of[i] * few.ldx, few.out + i * few.pitch, few.width, few.x, behind);
  }
}

// Rows of any pitch and address to rows that TMA can read (the weight's).
__global__ void __launch_bounds__(256) ce_copy_kernel(const uint16_t* __restrict__ w, int64_t ldw, int64_t rows, int width,
                                                      int64_t pitch, uint16_t* __restrict__ out) {
  pdl_trigger();
  pdl_wait();  // inputs are the previous kernel's outputs
  const uint16_t* end = w + (rows - 1) * ldw + width;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows; i += (int64_t)gridDim.x * 8)
    copy_row(w + i * ldw, out + i * pitch, width, w, end);
}

struct FactorArgs {
  const float* lse;    // null: no factors are wanted (forward)
  const float* grad;   // the loss's gradient: one, or one a row (reduction 0)
  int reduction;
  float boost;
  float2* rowc;
  float* scale;        // reduction 0: already there (ce_scale_kernel)
};

// Listed rows side by side, `pitch` apart, and zeros up to the next multiple of 256 rows; not if all rows are listed and
// the GEMMs can read them where they are. For the backward also the rows' factors: rowc[i] = (-lse log2 e, f_i) with
// dz = scale f_i (softmax - onehot). One gradient for all rows: f = boost and scale is that gradient (over the count for
// a mean) / boost. One a row: scale is a power of two near the largest finite one / boost and f_i = g_i / scale, exactly. In
// fp16 `boost` is a power of two above 1, so that probabilities down to 2^-37 are held.
__global__ void __launch_bounds__(256) ce_gather_kernel(const uint16_t* __restrict__ x, int64_t ldx, int64_t rows, int width,
                                                        int64_t pitch, const int* __restrict__ head,
                                                        const int* __restrict__ rows_of, uint16_t* __restrict__ out,
                                                        int in_place_rows, const FactorArgs f) {
  pdl_trigger();
  pdl_wait();  // inputs are the previous kernel's outputs
  const int count = head[0];
  if (f.lse) {
    float each = f.boost;
    if (f.reduction == 0) each = 1.f / *f.scale;
    else if (blockIdx.x == 0 && threadIdx.x == 0)
      *f.scale = count ? (f.reduction == 2 ? f.grad[0] / (float)count : f.grad[0]) / f.boost : 0.f;  // no rows: zeros
    for (int i = blockIdx.x * 256 + threadIdx.x; i < count; i += gridDim.x * 256)
      f.rowc[i] = make_float2(-f.lse[i] * kLog2e, f.reduction == 0 ? f.grad[rows_of[i]] * each : each);
  }
  if (count == in_place_rows) return;
  const int64_t end = ((int64_t)count + kTile - 1) / kTile * kTile;
  const uint16_t* behind = x + (rows - 1) * ldx + width;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < end; i += (int64_t)gridDim.x * 8) {
    uint16_t* dst = out + i * pitch;
    if (i < count) {
      copy_row(x + (int64_t)rows_of[i] * ldx, dst, width, x, behind);
    } else {
      for (int c = (threadIdx.x & 31) * 8; c < width; c += 256) *reinterpret_cast<uint4*>(dst + c) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
}

// Joins the partial (reference, sum) pairs of 32 rows a CTA: log-sum-exp, loss. Lanes are rows (the pairs of
// neighbouring rows lie side by side), warps take every eighth pair. The last CTA to finish adds the CTAs' sums in
// order (64 bits). reduction: 0 a loss per row, 1 their sum, 2 their mean (0 over no rows).
__global__ void __launch_bounds__(256) ce_finish_kernel(const float2* __restrict__ part,
                                                        const float* __restrict__ xlabel, const int* __restrict__ pos,
                                                        const int* __restrict__ rows_of, int* __restrict__ head,
                                                        float* __restrict__ lse, int64_t rows, int reduction,
                                                        double* __restrict__ sums, float* __restrict__ loss) {
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ float2 joined[8][32];
  __shared__ double block_sum[8];
  __shared__ int is_last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = head[0];
  const int tiles_m = (count + kTile - 1) / kTile;
  const int pairs = head[2] * 4;
  const int64_t r = (int64_t)blockIdx.x * 32 + lane;  // listed row; also a row whose loss is cleared if it is not
  if (pairs <= 64) {
    RowSum a;
    if (r < count) {
      const int mt = (int)r / kTile, local = (int)r - mt * kTile;
#pragma unroll 4
      for (int k = warp; k < pairs; k += 8)
        a.add(part[(((int64_t)(k >> 2) * tiles_m + mt) * 4 + (k & 3)) * kTile + local]);
    }
    joined[warp][lane] = make_float2(a.m, a.s);
  } else {  // few rows with many pairs each: a warp takes four rows, lanes are pairs
    for (int e = 0; e < 4; ++e) {
      const int64_t row = (int64_t)blockIdx.x * 32 + warp * 4 + e;
      RowSum a;
      if (row < count) {
        const int mt = (int)row / kTile, local = (int)row - mt * kTile;
#pragma unroll 4
        for (int k = lane; k < pairs; k += 32)
          a.add(part[(((int64_t)(k >> 2) * tiles_m + mt) * 4 + (k & 3)) * kTile + local]);
      }
      a.add_lanes();
      if (lane == 0) joined[0][warp * 4 + e] = make_float2(a.m, a.s);
      if (lane < 7) joined[1 + lane][warp * 4 + e] = make_float2(-INFINITY, 0.f);
    }
  }
  __syncthreads();
  double l = 0.0;
  if (warp == 0) {
    if (r < count) {
      RowSum a;
#pragma unroll
      for (int k = 0; k < 8; ++k) a.add(joined[k][lane]);
      const double total = a.lse();
      const float row_loss = (float)(total - (double)xlabel[r]);
      lse[r] = (float)total;
      if (reduction == 0) loss[rows_of[r]] = row_loss;
      l = (double)row_loss;
    }
    if (reduction == 0 && r < rows && pos[r] < 0) loss[r] = 0.f;
  }
  if (reduction == 0) return;
  if (warp == 0) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    if (lane == 0) {
      sums[blockIdx.x] = l;
      __threadfence();
      is_last = atomicAdd(head + 1, 1) == (int)gridDim.x - 1;
      __threadfence();
    }
  }
  __syncthreads();
  if (!is_last) return;
  double a = 0.0;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 256) a += __ldcg(sums + b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if (lane == 0) block_sum[warp] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    a = 0.0;
    for (int k = 0; k < 8; ++k) a += block_sum[k];
    if (reduction == 2) a = count ? a / count : 0.0;
    loss[0] = (float)a;
  }
}

// The scale of the backward when each row has a gradient: a power of two near the largest finite one, over boost.
__global__ void __launch_bounds__(1024) ce_scale_kernel(const int* __restrict__ head, const int* __restrict__ rows_of,
                                                        const float* __restrict__ grad, float boost,
                                                        float* __restrict__ scale) {
  pdl_trigger();
  pdl_wait();  // inputs are the previous kernel's outputs
  __shared__ float top[32];
  const int count = head[0];
  const int lane = threadIdx.x & 31;
  float m = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += 1024) {
    const float a = fabsf(grad[rows_of[i]]);
    if (a < INFINITY) m = fmaxf(m, a);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) top[threadIdx.x >> 5] = m;
  __syncthreads();
  m = top[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (threadIdx.x == 0) {
    float unit = 1.f;
    if (m > 0.f) {
      int e;
      frexpf(m, &e);
      unit = ldexpf(1.f, e < -100 ? -100 : e > 100 ? 100 : e);  // the scale and its reciprocal are normal numbers
    }
    *scale = unit / boost;
  }
}

// out[r] = scale * sum of the slices of row pos[r] (zeros where that is -1), or of row r without pos, in slice order. A
// warp takes a row; VEC: rows of out allow stores of four elements.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) ce_reduce_kernel(const float* __restrict__ part, int slices, int64_t slice_rows,
                                                        int64_t pitch, const int* __restrict__ pos,
                                                        const float* __restrict__ scale, T* __restrict__ out,
                                                        int64_t ldo, int64_t rows, int width) {
  pdl_wait();  // inputs are the previous kernel's outputs
  const float f = *scale;
  for (int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * 8) {
    const int64_t i = pos ? pos[r] : r;
#pragma unroll 2
    for (int c = (threadIdx.x & 31) * 4; c < width; c += 128) {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      if (i >= 0) {
        for (int k = 0; k < slices; ++k) {
          float v[4];
          load_vec<float, 4>(part + ((int64_t)k * slice_rows + i) * pitch + c, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] *= f;
      }
      if (VEC) {
        store_vec<T, 4>(out + r * ldo + c, s);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < width) out[r * ldo + c + e] = Dt<T>::from_f(s[e]);
      }
    }
  }
}

}  // namespace rk

using namespace rk;

namespace {

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// [rows, inner] with row pitch ld (elements), boxes of box_inner (64 or 128 bytes) x box_rows.
bool tensor_map(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int64_t ld, int dtype, uint32_t box_inner,
                uint32_t box_rows) {
  auto fn = tensor_map_fn();
  if (!fn) return false;
  const int64_t esz = rk_host::dtype_size(dtype);
  cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)(ld * esz)};
  cuuint32_t box[2] = {box_inner, box_rows};
  cuuint32_t estr[2] = {1, 1};
  const CUtensorMapDataType dt = dtype == RK_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : dtype == RK_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            box_inner * esz == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// dz of one piece. Pieces that stay in L2 cost more in kernels' ends than they save in memory: 64, 128, 256, 512 and 1024
// MB took 1.99, 1.80, 1.68, 1.59 and 1.62 ms at 14848 x 50257 x 256, 13.5, 12.0, 11.3, 10.8 and 10.9 at 32768 x 50257 x 1024.
constexpr int64_t kPieceBytes = 512ll << 20;
// fp32 tiles of dW on their way to rows that TMA cannot write (or the other 16-bit type): a step of the piece's rows at a
// time, and with slices of the reduction the piece (within kPieceBytes). With few rows a piece is the whole vocabulary, and
// its tiles at once would be an fp32 copy of the weight (4 GB at 256 x 128256 x 8192).
constexpr int64_t kStagedBytes = 128ll << 20;

// How the work of (M rows, V, K) is cut. Pure arithmetic, the same for the workspace queries and the calls.
struct CePlan {
  int64_t M, V, K, Mp, Kp, Kq;  // Mp: rows in whole tiles; Kp, Kq: pitch of the gathered rows and of fp32 rows
  int tiles_m, tiles_v, tiles_k, kb_k;
  int units;        // row tiles x segments of the forward, at most
  int piece_tiles;  // vocabulary tiles of a piece
  int dx_slices, dw_slices;
  int dw_step;      // vocabulary tiles of dW staged at a time
};

// Model of the work in microseconds, for choosing among cuts: a k block of a 256 x 256 tile takes a pair about 0.35, a
// tile 1.5 more, a kernel 3, and fp32 slices are moved at 5 TB/s.
double waves_us(int64_t tiles, int64_t slices, int64_t kb) {
  return (double)ceil_div(tiles * slices, kPairs) * (0.35 * (double)ceil_div(kb, slices) + 1.5) + 3.0;
}
double moved_us(double bytes) { return bytes / 5e6 + 3.0; }
int64_t staged_bytes(int64_t tiles, int64_t pitch) { return tiles * kTile * pitch * 4; }

CePlan make_plan(int64_t M, int64_t V, int64_t K) {
  static thread_local CePlan p{};  // of the last sizes asked for: the choice takes some microseconds
  if (p.M == M && p.V == V && p.K == K) return p;
  p = CePlan{};
  p.M = M;
  p.V = V;
  p.K = K;
  p.Mp = up(M, kTile);
  p.Kp = up(K, 8);
  p.Kq = up(K, 4);
  p.tiles_m = (int)(p.Mp / kTile);
  p.tiles_v = (int)ceil_div(V, kTile);
  p.tiles_k = (int)ceil_div(K, kTile);
  p.kb_k = (int)ceil_div(K, kKb);
  p.units = p.tiles_m > 8 * kPairs ? p.tiles_m : 8 * kPairs;  // whatever the number of rows that count
  double best;
  // pieces: as few as the workspace allows or a few more, and slices of dW, by the model
  const int64_t fit = kPieceBytes / (p.Mp * 2 * kTile) > 1 ? kPieceBytes / (p.Mp * 2 * kTile) : 1;
  const int fewest = (int)ceil_div(p.tiles_v, fit);
  const int kb_rows = (int)(p.Mp / kKb);
  best = 1e30;
  for (int n = fewest; n <= fewest + 4 && n <= p.tiles_v; ++n) {
    const int tiles = (int)ceil_div(p.tiles_v, n);
    const int whole = (int)ceil_div(p.tiles_v, tiles) - 1, rest = p.tiles_v - whole * tiles;
    for (int s = 1; s <= 16 && (s == 1 || (kb_rows / s >= 16 && s * staged_bytes(tiles, p.Kq) <= kPieceBytes)); ++s) {
      double t = 0;
      for (int last = 0; last < 2; ++last) {
        const int64_t v = last ? rest : tiles;
        t += (last ? 1 : whole) *
             (waves_us((int64_t)p.tiles_m * v, 1, p.kb_k) + waves_us(v * p.tiles_k, s, kb_rows) +
              (s > 1 ? moved_us((double)v * kTile * (double)K * (8.0 * s + 2.0)) : 0.0) +
              waves_us((int64_t)p.tiles_m * p.tiles_k, 1, v * (kTile / kKb)) + (double)p.Mp * (double)K * 4.0 / 5e6);
      }
      if (t < best) {
        best = t;
        p.piece_tiles = tiles;
        p.dw_slices = s;
      }
    }
  }
  p.dw_step = p.piece_tiles;
  if (p.dw_slices == 1) {  // equal steps
    const int64_t most = kStagedBytes / staged_bytes(1, p.Kq), steps = ceil_div(p.piece_tiles, most > 1 ? most : 1);
    p.dw_step = (int)ceil_div(p.piece_tiles, steps);
  }
  best = 1e30;
  const int kb_piece = p.piece_tiles * (kTile / kKb), pieces = (int)ceil_div(p.tiles_v, p.piece_tiles);
  p.dx_slices = 1;
  for (int s = 1; s <= 16 && (s == 1 || kb_piece / s >= 16); ++s) {
    const double t = pieces * (waves_us((int64_t)p.tiles_m * p.tiles_k, s, kb_piece) +
                               s * (double)p.Mp * (double)K * 8.0 / 5e6) + moved_us((double)p.Mp * (double)K * 4.0 * s);
    if (t < best) {
      best = t;
      p.dx_slices = s;
    }
  }
  return p;
}

// Kept from forward to backward (4-byte words): [count, done, segments, -], pos [M], rows_of [M], lse [M], label [M].
struct CeKept {
  int *head, *pos, *rows_of, *label;
  float* lse;
};
CeKept kept_of(int* k, int64_t M) { return {k, k + 4, k + 4 + M, k + 4 + 3 * M, reinterpret_cast<float*>(k + 4 + 2 * M)}; }

struct Arena {
  char* base;
  int64_t at;
  void* take(int64_t bytes) {
    void* p = base ? base + at : nullptr;
    at += up(bytes, 1024);
    return p;
  }
};

bool w_ready(const void* w, int64_t ldw, int64_t V) { return rk_host::aligned(w, 16) && (V == 1 || ldw % 8 == 0); }

struct FwdSpace {
  void *x, *w;
  float2* part;
  float* xlabel;
  double* sums;
};
int64_t fwd_space(const CePlan& p, bool copy_w, char* base, FwdSpace* f) {
  Arena a{base, 0};
  f->w = a.take(copy_w ? p.V * p.Kp * 2 : 0);
  f->x = a.take(p.Mp * p.Kp * 2);
  f->part = static_cast<float2*>(a.take((int64_t)p.units * 4 * kTile * 8));
  f->xlabel = static_cast<float*>(a.take(p.M * 4));
  f->sums = static_cast<double*>(a.take(ceil_div(p.M, 32) * 8));
  return a.at;
}

struct BwdSpace {
  void *x, *w, *dz;
  float2* rowc;
  float *scale, *dx, *dw;
};
// Tiles of dW are stored in fp32 and converted after that unless each can leave at once, in the operands' type or fp32.
bool dw_direct(const CePlan& p, const void* dw, int64_t lddw, int dw_dtype, int dtype) {
  return p.dw_slices == 1 && (dw_dtype == dtype || dw_dtype == RK_F32) && rk_host::aligned(dw, 16) &&
         lddw * (int64_t)rk_host::dtype_size(dw_dtype) % 16 == 0;
}
int64_t bwd_space(const CePlan& p, bool copy_w, bool dx, bool dw, char* base, BwdSpace* b) {
  Arena a{base, 0};
  b->w = a.take(copy_w ? p.V * p.Kp * 2 : 0);
  b->x = a.take(p.Mp * p.Kp * 2);
  b->dz = a.take(p.Mp * p.piece_tiles * kTile * 2);
  b->rowc = static_cast<float2*>(a.take(p.M * 8));
  b->scale = static_cast<float*>(a.take(4));
  b->dx = static_cast<float*>(a.take(dx ? (int64_t)p.dx_slices * p.Mp * p.Kq * 4 : 0));
  b->dw = static_cast<float*>(a.take(dw ? p.dw_slices * staged_bytes(p.dw_step, p.Kq) : 0));
  return a.at;
}

template <int MODE, typename T, int RES = 0>
int launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const CUtensorMap& tx, const CeArgs& g,
           int dtype, int64_t tiles, cudaStream_t s) {
  constexpr bool a_mn = MODE == OUTER || MODE == OUTER_T, b_mn = MODE == ADD || a_mn;
  constexpr uint32_t smem = ce_smem(MODE, RES);
  static_assert(smem <= 232448 - 256, "shared memory over the per-block limit");
  if constexpr (RES == 0 && (MODE == STATS || MODE == DLOGITS))
    if (g.kb <= kResKb) return launch<MODE, T, kResKb>(ta, tb, tc, tx, g, dtype, tiles, s);
  auto kern = ce_gemm_kernel<MODE, T, RES>;
  if (const int e = rk_host::ensure_smem_attr(reinterpret_cast<const void*>(kern), (int)smem)) return e;
  const int pairs = tiles < kPairs ? (int)tiles : kPairs;
  rk_host::launch_k(kern, 2 * pairs, kCeThreads, smem, s, ta, tb, tc, tx, g,
                    idesc_f16(kTile, kTile, dtype == RK_BF16 ? 1 : 0, a_mn ? 1 : 0, b_mn ? 1 : 0));
  return rk_host::launch_status();
}

int gather(const void* x, int64_t ldx, const CePlan& p, const CeKept& k, void* out, bool in_place, const FactorArgs& f,
           cudaStream_t s) {
  const int64_t blocks = ceil_div(p.Mp, 8);
  const unsigned grid = (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8);
  rk_host::launch_k(ce_gather_kernel, grid, 256, 0, s, static_cast<const uint16_t*>(x), ldx, p.M, (int)p.K, p.Kp, k.head,
                    k.rows_of, static_cast<uint16_t*>(out), in_place ? (int)p.M : -1, f);
  return rk_host::launch_status();
}
// The weight as TMA can read it: itself, or a copy in `space` (whose pitch then replaces ldw).
int weight_rows(const void*& w, int64_t& ldw, const CePlan& p, void* space, cudaStream_t s) {
  if (w_ready(w, ldw, p.V)) {
    if (p.V == 1) ldw = p.Kp;  // one row: its pitch says nothing
    return RK_OK;
  }
  const int64_t blocks = ceil_div(p.V, 8);
  rk_host::launch_k(ce_copy_kernel, (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, s,
                    static_cast<const uint16_t*>(w), ldw, p.V, (int)p.K, p.Kp, static_cast<uint16_t*>(space));
  w = space;
  ldw = p.Kp;
  return rk_host::launch_status();
}
// One CTA for up to 4096 rows (its launch is the cheaper one), a cluster of eight for more.
int list_rows(const int64_t* labels, int64_t ignore, const CePlan& p, const CeKept& k, unsigned int* status,
              const FewRows& few, cudaStream_t s) {
  if (p.M <= 4096) {
    rk_host::launch_k(ce_list_kernel<1>, 1, 1024, 0, s, labels, p.M, p.V, ignore, k.head, k.pos, k.label, k.rows_of, status,
                      few);
    return rk_host::launch_status();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = 8;
  cfg.blockDim = 1024;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = rk_host::pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 8;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, ce_list_kernel<8>, labels, p.M, p.V, ignore, k.head, k.pos, k.label, k.rows_of, status, few);
  return rk_host::launch_status();
}
// Whether TMA can read the hidden states themselves.
bool readable(const void* x, int64_t ldx, const CePlan& p) {
  return rk_host::aligned(x, 16) && (p.M == 1 || ldx % 8 == 0);
}

template <typename T>
int reduce_typed(const float* part, int slices, int64_t slice_rows, int64_t pitch, const int* pos, const float* scale,
                 void* out, int64_t ldo, int64_t rows, int64_t width, cudaStream_t s) {
  const bool vec = width % 4 == 0 && ldo % 4 == 0 && rk_host::aligned(out, 4 * sizeof(T));
  const int64_t blocks = ceil_div(rows, 8);
  auto kern = vec ? ce_reduce_kernel<T, true> : ce_reduce_kernel<T, false>;
  rk_host::launch_k(kern, (unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, s, part, slices, slice_rows, pitch, pos,
                    scale, static_cast<T*>(out), ldo, rows, (int)width);
  return rk_host::launch_status();
}
int reduce(const float* part, int slices, int64_t slice_rows, int64_t pitch, const int* pos, const float* scale, void* out,
           int64_t ldo, int64_t rows, int64_t width, int dtype, cudaStream_t s) {
  if (dtype == RK_F32) return reduce_typed<float>(part, slices, slice_rows, pitch, pos, scale, out, ldo, rows, width, s);
  if (dtype == RK_BF16)
    return reduce_typed<__nv_bfloat16>(part, slices, slice_rows, pitch, pos, scale, out, ldo, rows, width, s);
  return reduce_typed<__half>(part, slices, slice_rows, pitch, pos, scale, out, ldo, rows, width, s);
}

bool sizes_ok(int64_t M, int64_t V, int64_t K) {
  return M >= 0 && V > 0 && K > 0 && M < (1ll << 26) && V < (1ll << 30) && K < (1ll << 24);
}

}  // namespace

extern "C" int64_t rk_linear_ce_kept(int64_t M) { return M < 0 ? 0 : (4 + 4 * M) * 4; }

extern "C" int64_t rk_linear_ce_fwd_workspace(int64_t M, int64_t V, int64_t K, int copy_w) {
  if (!sizes_ok(M, V, K) || M == 0) return 0;
  FwdSpace f;
  return fwd_space(make_plan(M, V, K), copy_w != 0, nullptr, &f);
}

extern "C" int64_t rk_linear_ce_bwd_workspace(int64_t M, int64_t V, int64_t K, int flags) {
  if (!sizes_ok(M, V, K) || M == 0) return 0;
  BwdSpace b;
  return bwd_space(make_plan(M, V, K), flags & 1, !(flags & RK_LINEAR_CE_NO_DX), !(flags & RK_LINEAR_CE_NO_DW), nullptr, &b);
}

extern "C" int rk_linear_ce_fwd(const void* hidden, int64_t ldh, const void* w, int64_t ldw, const int64_t* labels,
                                int64_t ignore_index, int64_t M, int64_t V, int64_t K, int dtype, int reduction,
                                float* loss, void* kept, void* workspace, int64_t workspace_bytes, void* stream) {
  if (dtype != RK_BF16 && dtype != RK_F16) return RK_ERR_DTYPE;
  if (!sizes_ok(M, V, K) || (M > 1 && ldh < K) || (V > 1 && ldw < K) || reduction < 0 || reduction > 2 || !kept ||
      (M && (!hidden || !w || !labels)) || (!loss && (M || reduction)))
    return RK_ERR_ARG;
  if (!rk_host::aligned(kept, 16) || !rk_host::aligned(hidden, 2) || !rk_host::aligned(w, 2)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    if (cudaMemsetAsync(kept, 0, 16, s) != cudaSuccess) return RK_ERR_LAUNCH;
    if (reduction && cudaMemsetAsync(loss, 0, 4, s) != cudaSuccess) return RK_ERR_LAUNCH;
    return RK_OK;
  }
  const CePlan p = make_plan(M, V, K);
  FwdSpace f;
  const bool copy_w = !w_ready(w, ldw, V);
  if (!workspace || workspace_bytes < fwd_space(p, copy_w, nullptr, &f)) return RK_ERR_WORKSPACE;
  if (!rk_host::aligned(workspace, 256)) return RK_ERR_ALIGN;
  fwd_space(p, copy_w, static_cast<char*>(workspace), &f);
  const CeKept k = kept_of(static_cast<int*>(kept), M);
  unsigned int* status = rk_host::device_status_ptr();
  const bool in_place = readable(hidden, ldh, p), few = M <= kFewRows;
  FewRows own{};
  if (few)
    own = FewRows{static_cast<const uint16_t*>(hidden), ldh, p.Kp, (int)K, in_place ? (int)M : -1,
                  static_cast<uint16_t*>(f.x)};
  int st = list_rows(labels, ignore_index, p, k, status, own, s);
  if (st != RK_OK) return st;
  if (!few && (st = gather(hidden, ldh, p, k, f.x, in_place, FactorArgs{}, s)) != RK_OK) return st;
  if ((st = weight_rows(w, ldw, p, f.w, s)) != RK_OK) return st;
  CUtensorMap ta, tb, tx;
  if (!tensor_map(&ta, f.x, K, p.Mp, p.Kp, dtype, kKb, kHalf) || !tensor_map(&tb, w, K, V, ldw, dtype, kKb, kHalf))
    return RK_ERR_LAUNCH;
  tx = ta;
  if (in_place && !tensor_map(&tx, hidden, K, M, M == 1 ? p.Kp : ldh, dtype, kKb, kHalf)) return RK_ERR_LAUNCH;
  CeArgs g{};
  g.in_place_rows = in_place ? (int)M : -1;
  g.count = k.head;
  g.vocab = (int)V;
  g.width = (int)K;
  g.tiles_n = p.tiles_v;
  g.kb = p.kb_k;
  g.slices = 1;
  g.part = f.part;
  g.xlabel = f.xlabel;
  g.label = k.label;
  g.status = status;
  if (few) {
    g.head = k.head;
    g.pos = k.pos;
    g.rows_of = k.rows_of;
    g.lse = k.lse;
    g.loss = loss;
    g.rows = (int)M;
    g.reduction = reduction;
  }
  st = launch<STATS, __nv_bfloat16>(ta, tb, ta, tx, g, dtype, kPairs, s);
  if (few || st != RK_OK) return st;
  rk_host::launch_k(ce_finish_kernel, (unsigned)ceil_div(M, 32), 256, 0, s, f.part, f.xlabel, k.pos,
                    k.rows_of, k.head, k.lse, M, reduction, f.sums, loss);
  return rk_host::launch_status();
}

extern "C" int rk_linear_ce_bwd(const void* hidden, int64_t ldh, const void* w, int64_t ldw, const void* kept, int64_t M,
                                int64_t V, int64_t K, int dtype, int reduction, const float* grad, void* dx, int64_t lddx,
                                int dx_dtype, void* dw, int64_t lddw, int dw_dtype, void* workspace,
                                int64_t workspace_bytes, void* stream) {
  if ((dtype != RK_BF16 && dtype != RK_F16) || !rk_host::dtype_ok(dx_dtype) || !rk_host::dtype_ok(dw_dtype))
    return RK_ERR_DTYPE;
  if (!sizes_ok(M, V, K) || (M > 1 && (ldh < K || (dx && lddx < K))) || (V > 1 && (ldw < K || (dw && lddw < K))) ||
      reduction < 0 || reduction > 2 || !kept || (M && (!hidden || !w)) || (!grad && (M || reduction)))
    return RK_ERR_ARG;
  if (!rk_host::aligned(kept, 16) || !rk_host::aligned(hidden, 2) || !rk_host::aligned(w, 2)) return RK_ERR_ALIGN;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (V == 1) lddw = up(K, 8);  // one row: its pitch says nothing
  if (M == 0) {
    if (dw && cudaMemset2DAsync(dw, lddw * rk_host::dtype_size(dw_dtype), 0, K * rk_host::dtype_size(dw_dtype), V, s) !=
                  cudaSuccess)
      return RK_ERR_LAUNCH;
    return RK_OK;
  }
  if (M == 1 && lddx < K) lddx = K;
  if (!dx && !dw) return RK_OK;
  const CePlan p = make_plan(M, V, K);
  BwdSpace b;
  const bool copy_w = !w_ready(w, ldw, V);
  if (!workspace || workspace_bytes < bwd_space(p, copy_w, dx, dw, nullptr, &b)) return RK_ERR_WORKSPACE;
  if (!rk_host::aligned(workspace, 256)) return RK_ERR_ALIGN;
  bwd_space(p, copy_w, dx, dw, static_cast<char*>(workspace), &b);
  const CeKept k = kept_of(const_cast<int*>(static_cast<const int*>(kept)), M);
  float* scale = b.scale;
  const bool in_place = readable(hidden, ldh, p);
  const FactorArgs f{k.lse, grad, reduction, dtype == RK_F16 ? 8192.f : 1.f, b.rowc, scale};
  int st = RK_OK;
  if (reduction == 0) {
    rk_host::launch_k(ce_scale_kernel, 1, 1024, 0, s, k.head, k.rows_of, grad, f.boost, scale);
    if ((st = rk_host::launch_status()) != RK_OK) return st;
  }
  if ((st = gather(hidden, ldh, p, k, b.x, in_place, f, s)) != RK_OK) return st;
  if ((st = weight_rows(w, ldw, p, b.w, s)) != RK_OK) return st;
  const int64_t pitch = (int64_t)p.piece_tiles * kTile;  // of dz
  const bool direct = dw && dw_direct(p, dw, lddw, dw_dtype, dtype);
  CUtensorMap x_k, x_mn, in_k, in_mn, w_k, w_mn, dz_out, dz_k, dz_mn, dx_out{}, dw_out{};
  if (!tensor_map(&x_k, b.x, K, p.Mp, p.Kp, dtype, kKb, kHalf) || !tensor_map(&x_mn, b.x, K, p.Mp, p.Kp, dtype, 64, kKb) ||
      !tensor_map(&w_k, w, K, V, ldw, dtype, kKb, kHalf) || !tensor_map(&w_mn, w, K, V, ldw, dtype, 64, kKb) ||
      !tensor_map(&dz_out, b.dz, pitch, p.Mp, pitch, dtype, 32, 32) ||
      !tensor_map(&dz_k, b.dz, pitch, p.Mp, pitch, dtype, kKb, kHalf) ||
      (dx && !tensor_map(&dx_out, b.dx, K, (int64_t)p.dx_slices * p.Mp, p.Kq, RK_F32, 32, 32)))
    return RK_ERR_LAUNCH;
  in_k = x_k;
  in_mn = x_mn;
  const int64_t ldi = M == 1 ? p.Kp : ldh;
  if (in_place && (!tensor_map(&in_k, hidden, K, M, ldi, dtype, kKb, kHalf) ||
                   !tensor_map(&in_mn, hidden, K, M, ldi, dtype, 64, kKb)))
    return RK_ERR_LAUNCH;
  const int step = direct ? p.piece_tiles : p.dw_step;  // vocabulary tiles of a launch for dW
  if (dw && (direct ? !tensor_map(&dw_out, dw, K, V, lddw, dw_dtype, 32, 32)
                    : !tensor_map(&dw_out, b.dw, K, (int64_t)p.dw_slices * step * kTile, p.Kq, RK_F32, 32, 32)))
    return RK_ERR_LAUNCH;
  CeArgs g{};
  g.in_place_rows = in_place ? (int)M : -1;
  g.count = k.head;
  g.vocab = (int)V;
  g.width = (int)K;
  g.label = k.label;
  g.rowc = b.rowc;
  g.scale = scale;
  g.status = rk_host::device_status_ptr();
  for (int t0 = 0; t0 < p.tiles_v; t0 += p.piece_tiles) {
    const int tiles = p.tiles_v - t0 < p.piece_tiles ? p.tiles_v - t0 : p.piece_tiles;
    const int64_t v0 = (int64_t)t0 * kTile;
    const int64_t live = V - v0 < (int64_t)tiles * kTile ? V - v0 : (int64_t)tiles * kTile;
    g.v0 = (int)v0;
    g.slices = 1;
    g.tiles_n = tiles;
    g.kb = p.kb_k;
    g.row_tiles = p.tiles_m;
    g.slice_rows = 0;
    st = dtype == RK_BF16 ? launch<DLOGITS, __nv_bfloat16>(x_k, w_k, dz_out, in_k, g, dtype, (int64_t)p.tiles_m * tiles, s)
                          : launch<DLOGITS, __half>(x_k, w_k, dz_out, in_k, g, dtype, (int64_t)p.tiles_m * tiles, s);
    if (st != RK_OK) return st;
    if (dx) {
      g.tiles_n = p.tiles_k;
      g.kb = (int)ceil_div(live, kKb);
      g.slices = p.dx_slices;
      g.slice_rows = (int)p.Mp;
      g.add = t0 > 0;
      st = launch<ADD, float>(dz_k, w_mn, dx_out, dz_k, g, dtype, (int64_t)p.tiles_m * p.tiles_k * p.dx_slices, s);
      if (st != RK_OK) return st;
    }
    for (int r0 = 0; dw && r0 < tiles; r0 += step) {
      const int n_tiles = tiles - r0 < step ? tiles - r0 : step;
      const int64_t first = (int64_t)r0 * kTile;  // of the piece's rows of dW, and columns of dz
      if (!tensor_map(&dz_mn, static_cast<uint16_t*>(b.dz) + first, pitch - first, p.Mp, pitch, dtype, 64, kKb))
        return RK_ERR_LAUNCH;
      g.tiles_n = p.tiles_k;
      g.row_tiles = n_tiles;
      g.slices = p.dw_slices;
      g.slice_rows = direct ? 0 : step * kTile;
      const int64_t n = (int64_t)n_tiles * p.tiles_k * p.dw_slices;
      g.to_weight = direct;
      if (!direct || dw_dtype == RK_F32) st = launch<OUTER, float>(dz_mn, x_mn, dw_out, in_mn, g, dtype, n, s);
      else if (dtype == RK_BF16) st = launch<OUTER_T, __nv_bfloat16>(dz_mn, x_mn, dw_out, in_mn, g, dtype, n, s);
      else st = launch<OUTER_T, __half>(dz_mn, x_mn, dw_out, in_mn, g, dtype, n, s);
      if (st != RK_OK) return st;
      if (!direct) {
        char* out = static_cast<char*>(dw) + (v0 + first) * lddw * (int64_t)rk_host::dtype_size(dw_dtype);
        const int64_t left = live - first, rows = left < (int64_t)n_tiles * kTile ? left : (int64_t)n_tiles * kTile;
        if ((st = reduce(b.dw, p.dw_slices, (int64_t)step * kTile, p.Kq, nullptr, scale, out, lddw, rows, K, dw_dtype, s)) !=
            RK_OK)
          return st;
      }
    }
  }
  if (!dx) return RK_OK;
  return reduce(b.dx, p.dx_slices, p.Mp, p.Kq, k.pos, scale, dx, lddx, M, K, dx_dtype, s);
}
