// The whole mixture-of-experts layer for a few tokens (a decode step): router, the chosen experts, their weighted sum.
//
//   v = x, or x w / sqrt(mean x^2 + eps);  l = gate v;  the k largest l, p = softmax over them;
//   out = residual + sum over the k experts e, ascending, of p_e W2_e (act(W1_e v) * (W3_e v))
//
// Bound: HBM, the blocks of the experts that some token chose (each read once for up to M tokens of an expert).
//
// Four launches, each starting while the one before it ends:
//   k_moe_step_route   a cluster a token: norm, logits in 64 bits (a near tie of two experts goes one way), top k, softmax
//   k_moe_step<UP>     a = act(W1 v) * (W3 v) of every (token, expert) pair
//   k_moe_step<DOWN>   W2 a
//   k_moe_step_sum     the weighted sum and the residual
//
// The products run on mma.sync (m16n8k16, fp16 with fp32 sums): sixteen weight rows by eight columns.  An activation is
// 2^s (hi + lo), both fp16 (a power of two for each 256 of them), which keeps 22 bits of the largest: up to 4 tokens have a column for
// each part (M = 4), up to 8 tokens a column each and two products (M = 8).  A single token (M = 1) has the two columns of its
// parts four times, for every fourth group of values: a thread then has the sums of one group in four, and a quarter of the
// scales to apply.  A tile of UP is eight rows of W1 and the same eight of W3, so that one thread holds the gate and the up
// value of a feature.
//
// A block's codes enter as integers in fp16 (signed where the type has no minima) and its scales are applied to the sums of 16
// or 32 products, in fp32; minima are one more product, with the activations' sums over their groups.
//
// A CTA takes a contiguous range of the stages (expert, part of K, group of row tiles).  Two warps have a stage's rows copied
// into a ring in shared memory by tensor copies (one or two instructions a matrix of some 340 clocks each; a bulk copy for each
// row takes 180 to issue, 2900 a stage; each warp's own loads by cp.async 700 to 1300 in the load/store unit; of the 1640 in
// which a stage's 37 KB can come from HBM).  Sixteen warps multiply, each 256 values of K of a tile, for which its activations
// stay in registers while the expert lasts.  Two more add up their results and write.  (Warps that multiply and take turns at
// the copies and sums need no registers for others, but every stage then waits for the one that is late.)
// Nothing waits for another CTA.  The results do not depend on the order in which CTAs run.
//
// Measured, a step from Python with its inputs and weights cold in L2: Q4_K, 4096 -> 14336, 2 of 8 experts, one token 58 us (the
// chosen blocks at 3.4 TB/s), 7 bf16 tokens 170 to 196 us (3.5 to 3.8 TB/s); Q4_K, 8 of 128 experts, one token 30 us (26 in a
// captured graph); Q6_K, 8 of 128 experts, 33 tokens 177 us.  At most 58 % of the copy bandwidth: the products' instructions, which
// take up to three quarters of the issue slots while a stage's bytes are there, are what a faster step would have fewer of.
#include <cooperative_groups.h>
#include <cuda.h>

#include <algorithm>
#include <cstring>
#include <mutex>

#include "xm_gemv_dot.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kMaxTokens = 64, kMaxTop = 16, kMaxStepExperts = 256, kMaxPairs = kMaxTokens * kMaxTop;
constexpr int kWorkers = 16, kCopiers = 2, kFinishers = 2, kStepThreads = (kWorkers + kCopiers + kFinishers) * 32, kMaxRing = 8;
constexpr int kRouteCluster = 8, kRouteThreads = 256;
constexpr int kMaxHidden = 16384;

// How the rows of a stage get into shared memory.
enum Copies {
  kTensor,                     // by tensor maps: rows are whole units of 16 bytes
  kWhole,                      // they are not, but a stage has whole rows: as they lie in the weight
  kRows                        // neither: row by row, from the unit that a row begins in to the one that it ends in
};

struct StepArgs {
  const CUtensorMap *map1, *map3;        // of the E weights (DOWN: map1 of the second products')
  const uint8_t *const *w1, *const *w3;  // their bytes
  const float* src;            // [rows][K]: v of a token (UP), a of a pair (DOWN)
  float* dst;                  // UP: a [P][F];  DOWN: partial results [chunks][P][H]
  float* part;                 // UP with several chunks: partial results [chunks][P][2F]
  int* tickets;                // UP with chunks: of each segment's groups of tiles
  const int* top_e;            // [T][k], ascending
  const float* top_w;
  int T, k, E, act;
  int K, N;                    // N: rows of a result (UP: F, DOWN: H)
  int nsb, chunks, kc, tps;    // 256-blocks of K, parts of K, their 256-blocks, tiles a stage
  int tiles, groups;           // row tiles, and stages that hold them
  int64_t row_bytes;
  // In shared memory a stage is `boxes` times [rows][pitch bytes], each with box_sb 256-blocks of K of its rows (UP: those of
  // W1, then those of W3).
  int boxes, box_sb, pitch, ring, copies;
  const float* residual;       // DOWN
  int64_t residual_stride, out_stride;
  float* out;
};

struct alignas(128) StepShared {
  uint64_t full[kMaxRing], done[kMaxRing], empty[kMaxRing];   // a stage's rows are there, its results are, they are added up
  int n_seg;
  const uint8_t *w1[kMaxStepExperts], *w3[kMaxStepExperts];
  int cnt[kMaxStepExperts], off[kMaxStepExperts];
  unsigned short pair[kMaxPairs], seg_at[kMaxPairs];   // pairs (token * k + slot) by expert, then token; a segment's first
  uint8_t expert[kMaxPairs], rank[kMaxPairs];          // of a pair: its expert, how many of the expert's pairs are before it
  uint8_t seg_e[kMaxPairs], seg_n[kMaxPairs];
};

// ---------------------------------------------------------------------------
// Routing
// ---------------------------------------------------------------------------
struct RouteArgs {
  const void* x;
  int64_t stride;
  const float *norm_w, *gate;
  float eps;
  int T, H, E, k;
  float *v, *top_w;
  int* top_e;
  int *tickets, n_tickets;     // zeroed
};

XM_DEV double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

XM_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
XM_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// A cluster of 8 CTAs a token: each has the whole row and an eighth of the experts, one for each warp, or for several warps
// where there are few (which then take parts of the row).  The logits go to the first CTA's shared memory, the others end.
template <typename XT>
__global__ void __launch_bounds__(kRouteThreads, 3) k_moe_step_route(RouteArgs a) {
  constexpr int WARPS = kRouteThreads / 32;
  extern __shared__ __align__(16) double row[];               // (converted once, not for each expert)
  __shared__ float red[WARPS];
  __shared__ double part[WARPS], all[kMaxStepExperts], val[kMaxTop];
  __shared__ unsigned chosen[WARPS];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), t = (int)(blockIdx.x / kRouteCluster), tid = threadIdx.x, lane = tid & 31,
            warp = tid >> 5;
  cluster_arrive();                        // (the first CTA runs before anything is written to it)
  grid_dep_wait();
  grid_dep_launch();
  for (int i = blockIdx.x * kRouteThreads + tid; i < a.n_tickets; i += gridDim.x * kRouteThreads) a.tickets[i] = 0;
  const int mine = (a.E - rank + kRouteCluster - 1) / kRouteCluster;       // experts rank, rank + 8, ...
  const int most = (a.E + kRouteCluster - 1) / kRouteCluster;
  const int split = most <= 1 ? 8 : most <= 2 ? 4 : most <= 4 ? 2 : 1;     // warps an expert
  const int at_once = WARPS / split, slice = warp % split;
  const int n4 = a.H / 4 / split;                                          // (H is a multiple of 256)
  constexpr int AHEAD = 8;                 // the first loads of the first expert go out before the row is there
  float4 first[AHEAD];
  {
    const int j = warp / split;
    const float4* g = reinterpret_cast<const float4*>(a.gate + (int64_t)(rank + j * kRouteCluster) * a.H) + slice * n4;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      first[i] = j < mine && lane + 32 * i < n4 ? __ldg(g + lane + 32 * i) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const XT* x = (const XT*)a.x + (int64_t)t * a.stride;
  float s = 0.f;
#pragma unroll 8
  for (int i = tid; i < a.H; i += kRouteThreads) {
    const float v = to_f32<XT>(x[i]);
    row[i] = (double)(a.norm_w ? v * a.norm_w[i] : v);
    s = fmaf(v, v, s);
  }
  s = warp_sum(s);
  if (lane == 0) red[warp] = s;
  __syncthreads();
  s = 0.f;
  for (int w = 0; w < WARPS; ++w) s += red[w];
  const float r = a.norm_w ? 1.0f / sqrtf(s / (float)a.H + a.eps) : 1.0f;
  for (int i = rank * kRouteThreads + tid; i < a.H; i += kRouteCluster * kRouteThreads) a.v[(int64_t)t * a.H + i] = (float)row[i] * r;
  cluster_wait();
  double* to = cl.map_shared_rank(all, 0);
  for (int j0 = 0; j0 < mine; j0 += at_once) {
    const int j = j0 + warp / split;
    double d = 0.;
    if (j < mine) {
      const float4* g = reinterpret_cast<const float4*>(a.gate + (int64_t)(rank + j * kRouteCluster) * a.H) + slice * n4;
      const double* v = row + 4 * slice * n4;
      double q[4] = {0., 0., 0., 0.};
      auto add = [&](const float4& w, int i) {
        const double2 u = *reinterpret_cast<const double2*>(v + 4 * i), z = *reinterpret_cast<const double2*>(v + 4 * i + 2);
        q[0] = fma(u.x, (double)w.x, q[0]);
        q[1] = fma(u.y, (double)w.y, q[1]);
        q[2] = fma(z.x, (double)w.z, q[2]);
        q[3] = fma(z.y, (double)w.w, q[3]);
      };
      int i = lane;
      if (j0 == 0) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u, i += 32)
          if (i < n4) add(first[u], i);
      }
#pragma unroll 8
      for (; i < n4; i += 32) add(__ldg(g + i), i);
      d = warp_sum_d((q[0] + q[1]) + (q[2] + q[3]));
    }
    if (split == 1) {
      if (lane == 0 && j < mine) to[rank + j * kRouteCluster] = d * (double)r;
      continue;
    }
    if (lane == 0) part[warp] = d;
    __syncthreads();
    if (tid < at_once && j0 + tid < mine) {
      double z = 0.;
      for (int w = 0; w < split; ++w) z += part[tid * split + w];
      to[rank + (j0 + tid) * kRouteCluster] = z * (double)r;
    }
    __syncthreads();
  }
  cluster_arrive();
  if (rank != 0) return;
  cluster_wait();
  // an expert a thread: how many come before it
  double l = 0., key = 0.;
  if (tid < a.E) {
    l = all[tid];
    key = l == l ? l : -INFINITY;                                       // (NaN: not before any other)
  }
  int before = a.E;
  if (tid < a.E) {
    before = 0;
#pragma unroll 4
    for (int e = 0; e < a.E; ++e) {
      const double o = all[e] == all[e] ? all[e] : -INFINITY;
      before += o > key || (o == key && e < tid);
    }
  }
  const bool in = before < a.k;
  const unsigned b = __ballot_sync(~0u, in);
  if (lane == 0) chosen[warp] = b;
  if (in) val[before] = l;
  __syncthreads();
  if (in) {
    double top = val[0];
    if (!(fabs(top) < INFINITY)) top = 0.;
    float sum = 1e-12f;
    for (int j = 0; j < a.k; ++j) sum += expf((float)(val[j] - top));
    int place = __popc(b & ((1u << lane) - 1));
    for (int w = 0; w < warp; ++w) place += __popc(chosen[w]);
    a.top_e[t * a.k + place] = tid;
    a.top_w[t * a.k + place] = expf((float)(l - top)) / sum;
  }
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------
// a box of a tensor map to shared memory, completing on `bar`
XM_DEV void tensor_g2s(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(smem_u32(dst)), "l"(map), "r"(c0), "r"(c1), "r"(smem_u32(bar)) : "memory");
}
XM_DEV bool mbar_test(uint64_t* bar, uint32_t parity) {        // (half as long as a try_wait, where the phase is complete)
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok != 0;
}

// out[token][row] from the second products' partial results
XM_DEV void step_output(const StepArgs& a, int token, int row) {
  const int P = a.T * a.k;
  float y = 0.f;
  for (int j = 0; j < a.k; ++j) {
    float q = 0.f;
    for (int c = 0; c < a.chunks; ++c) q += __ldcg(a.dst + ((int64_t)c * P + token * a.k + j) * a.N + row);
    y = fmaf(q, __ldcg(a.top_w + token * a.k + j), y);
  }
  if (a.residual) y += a.residual[token * a.residual_stride + row];
  a.out[token * a.out_stride + row] = y;
}

XM_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
XM_DEV void mma_f16_zero(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {       // the first of a sum
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
XM_DEV void mma_f16_k8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
XM_DEV uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// How a thread's 8 values of a group of 32 of K lie (t = lane % 4): 8 t .. 8 t + 7, or, for types whose groups have 16 values
// or whose blocks are not 8-byte aligned, 4 t .. 4 t + 3 of each half.  Either way they enter the products as the pairs (0, 2),
// (1, 3), (4, 6), (5, 7): the order in which words of codes fall apart under masks.
template <int T>
constexpr bool halves() { return T == T_Q6_K || T == T_Q8_0; }

// The 256 values of K that a warp holds, of M tokens: column g (= lane / 4) is token g / 2, hi or lo by g % 2 (M = 4), token g
// in two parts (M = 8), or hi or lo of the one token in the groups g / 2, g / 2 + 4, ... and zero in the others (M = 1).  By
// groups of 32 their pairs, and the sums over groups times 2^-5, of groups 2 t, 2 t + 1 (M = 1: in columns 0 and 1), for the types
// whose weights have offsets.
template <int M>
struct Columns {
  static constexpr int PARTS = M == 8 ? 2 : 1;
  uint32_t b[PARTS][8][4];
  uint32_t sum[PARTS];
  float scale[M == 8 ? 2 : 1];             // 2^s of the tokens that this thread has results of
};
// What a thread has of a tile's results: of its two rows (g, g + 8) the token t (M = 4), the tokens 2 t, 2 t + 1 (M = 8), or a
// quarter of the one token's (M = 1).
template <int M>
struct Result {
  static constexpr int N = M == 8 ? 2 : 1;
  float v[2][N];
  XM_DEV void clear() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[0][i] = v[1][i] = 0.f;
  }
  // v += s0 times the first row's sums, s1 times the second's
  XM_DEV void add(const float (&c)[4], float s0, float s1) {
    if constexpr (M != 8) {
      v[0][0] = fmaf(s0, c[0] + c[1], v[0][0]);
      v[1][0] = fmaf(s1, c[2] + c[3], v[1][0]);
    } else {
      v[0][0] = fmaf(s0, c[0], v[0][0]);
      v[0][1] = fmaf(s0, c[1], v[0][1]);
      v[1][0] = fmaf(s1, c[2], v[1][0]);
      v[1][1] = fmaf(s1, c[3], v[1][1]);
    }
  }
};

// c (+)= the products of 16 values of K (a: of the two rows; i: a pair of pairs of group j); M = 8: of the upper parts
template <int M, bool FIRST>
XM_DEV void mma_group(float (&c)[4], const uint32_t (&a)[4], const Columns<M>& x, int j, int i) {
  if constexpr (FIRST) mma_f16_zero(c, a, x.b[0][j][2 * i], x.b[0][j][2 * i + 1]);
  else mma_f16(c, a, x.b[0][j][2 * i], x.b[0][j][2 * i + 1]);
}
// c = the products of a group of 32.  (M = 8: the lower parts first: added to the sum of the upper ones, each product would lose
// what lies below that sum's 24 bits.)
template <int M>
XM_DEV void mma_32(float (&c)[4], const uint32_t (&a0)[4], const uint32_t (&a1)[4], const Columns<M>& x, int j) {
  if constexpr (M == 8) {
    mma_f16_zero(c, a0, x.b[1][j][0], x.b[1][j][1]);
    mma_f16(c, a1, x.b[1][j][2], x.b[1][j][3]);
    mma_f16(c, a0, x.b[0][j][0], x.b[0][j][1]);
    mma_f16(c, a1, x.b[0][j][2], x.b[0][j][3]);
  } else {
    mma_f16_zero(c, a0, x.b[0][j][0], x.b[0][j][1]);
    mma_f16(c, a1, x.b[0][j][2], x.b[0][j][3]);
  }
}
// The same of a group of 16 (the half i of group j).
template <int M>
XM_DEV void mma_16(float (&c)[4], const uint32_t (&a)[4], const Columns<M>& x, int j, int i) {
  if constexpr (M == 8) {
    mma_f16_zero(c, a, x.b[1][j][2 * i], x.b[1][j][2 * i + 1]);
    mma_f16(c, a, x.b[0][j][2 * i], x.b[0][j][2 * i + 1]);
  } else {
    mma_f16_zero(c, a, x.b[0][j][2 * i], x.b[0][j][2 * i + 1]);
  }
}

// Codes as factors.  A matrix instruction cuts products off some 26 bits below the largest by the exponents of their factors,
// and a subnormal has the exponent of a number up to 2^10 times as large: of codes that enter as the subnormals that their bits
// are, 2^-20 of the largest product was lost, against 2^-26 as numbers, and results were off by 1.4e-6 against 4e-7.  So they
// are made numbers, by one subtraction a pair, or the products are made to end above the cut: with whole numbers below 2^15
// nothing is lost of codes below 2^10 (measured over 250000 sums of 16).  The latter is what one token takes, whose kernel waits
// for its instructions (Q4_K, 8 experts of 14336 x 4096: 59 us a step against 68 with the subtractions, off by 3e-7 to 8e-7
// against 3e-7 to 4e-7); with more tokens both take as long.

// The upper part of an activation, or of a sum of them: what fp16 holds of it, or of its whole number.
template <bool WHOLE>
XM_DEV float upper(float v) { return __half2float(__float2half_rn(WHOLE ? rintf(v) : v)); }

// (1024 + c) - (1024 + bias) of two fp16, exact: numbers from codes below 1024 that lie under fp16 words of 1024.
constexpr uint32_t OVER = 0x64006400u;
XM_DEV uint32_t less(uint32_t u, float bias) {
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __float2half2_rn(1024.f + bias));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Types whose weights enter with the block's own value, not rounded to fp16 as dequantisation rounds it.
template <int T>
constexpr bool own_value() { return T == T_Q4_K || T == T_Q5_K || T == T_Q6_K || T == T_Q8_0; }

// 256 values of K of sixteen rows (r0: the thread's first row, r1: its second).

// Any type, value by value: weights rounded to fp16.
template <int T, int M>
XM_DEV void unit_any(const uint8_t* r0, const uint8_t* r1, int t, const Columns<M>& x, Result<M>& acc) {
  float c[4] = {0.f, 0.f, 0.f, 0.f}, lower[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t w[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* p = r ? r1 : r0;
      float v[8];
      if constexpr (QT<T>::QK == 256) QT<T>::decode8(p, 32 * j + 8 * t, v);
      else QT<T>::decode8(p + j * QT<T>::REC, 8 * t, v);
      w[r][0] = pack2(v[0], v[2]);
      w[r][1] = pack2(v[1], v[3]);
      w[r][2] = pack2(v[4], v[6]);
      w[r][3] = pack2(v[5], v[7]);
    }
    const uint32_t a0[4] = {w[0][0], w[1][0], w[0][1], w[1][1]}, a1[4] = {w[0][2], w[1][2], w[0][3], w[1][3]};
    mma_group<M, false>(c, a0, x, j, 0);
    mma_group<M, false>(c, a1, x, j, 1);
    if constexpr (M == 8) {
      mma_f16(lower, a0, x.b[1][j][0], x.b[1][j][1]);
      mma_f16(lower, a1, x.b[1][j][2], x.b[1][j][3]);
    }
  }
  acc.clear();
  acc.add(c, 1.f, 1.f);
  if constexpr (M == 8) acc.add(lower, 1.f, 1.f);
}

XM_DEV uint4 lds128(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }

XM_DEV uint32_t minus(uint32_t a, uint32_t b) {
  const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// Q4_K, and Q5_K (FIVE): w = d s_j c - dmin m_j.  A word's codes under the masks 0x000f000f and 0x00f000f0: c and 16 c.  The
// scales of a pair of groups come from their bytes as fp16 (1024 + s_2j) - 1024 and, for the upper codes,
// (64 + s_2j+1 / 16) - 64: exact.
template <bool FIVE, int M>
XM_DEV void unit_k(const uint8_t* r0, const uint8_t* r1, int t, const Columns<M>& x, Result<M>& acc) {
  constexpr uint32_t LOW = 0x000f000fu, HIGH = 0x00f000f0u, FIFTH = 0x00100010u;
  constexpr int QS = FIVE ? 48 : 16;
  constexpr bool NUMBERS = M != 1;         // codes as numbers, not as subnormals c 2^-24
  uint32_t sc[2][2], am[2], qh[2][4];
  float d[2], dm[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint4 h = lds128(r ? r1 : r0);
    const float2 dd = __half22float2(*reinterpret_cast<const __half2*>(&h.x));
    d[r] = NUMBERS ? dd.x : dd.x * 0x1p24f;
    dm[r] = dd.y * -0x1p5f;
    sc[r][0] = h.y & 0x3f3f3f3fu;
    sc[r][1] = (h.w & 0x0f0f0f0fu) | ((h.y >> 2) & 0x30303030u);
    const uint32_t m = t < 2 ? h.z & 0x3f3f3f3fu : ((h.w >> 4) & 0x0f0f0f0fu) | ((h.z >> 2) & 0x30303030u);
    am[r] = less(__byte_perm(m, OVER, t & 1 ? 0x7372 : 0x7170), 0.f);      // m_2t, m_2t+1
    if constexpr (FIVE) {
      const uint4 q = lds128((r ? r1 : r0) + 16);             // the fifth bits of groups 2 j, 2 j + 1: word j, bit = value
      qh[r][0] = (q.x >> (8 * t)) & 0xffu;
      qh[r][1] = (q.y >> (8 * t)) & 0xffu;
      qh[r][2] = (q.z >> (8 * t)) & 0xffu;
      qh[r][3] = (q.w >> (8 * t)) & 0xffu;
    }
  }
  float one[2][4];                         // M = 1: the sums of groups t and t + 4
  Result<M> sum;
  sum.clear();
#pragma unroll
  for (int jj = 0; jj < 4; ++jj) {
    uint32_t lo[2][4], hi[2][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint2 q = *reinterpret_cast<const uint2*>((r ? r1 : r0) + QS + 32 * jj + 8 * t);
      // (the fifth bits: one product puts two of them where the codes of a pair have theirs)
      constexpr uint32_t BASE = NUMBERS ? OVER : 0u;
      uint32_t f[4] = {BASE, BASE, BASE, BASE};
      if constexpr (FIVE) {
        const uint32_t b = qh[r][jj];
        f[0] |= (b * ((1u << 4) + (1u << 18))) & FIFTH;
        f[1] |= (b * ((1u << 3) + (1u << 17))) & FIFTH;
        f[2] |= (b * (1u + (1u << 14))) & FIFTH;
        f[3] |= ((b >> 1) * (1u + (1u << 14))) & FIFTH;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? q.x : q.y;
        if constexpr (NUMBERS && !FIVE) {  // 1024 + byte, less 1024 + c: the upper code by the pipe that has more to spare
          const uint32_t u = i & 1 ? __byte_perm(w, OVER, 0x7371) : (w & 0x00ff00ffu) | OVER, v = u & (LOW | OVER);
          lo[r][i] = less(v, 0.f);
          hi[r][i] = minus(u, v);
        } else {
          const uint32_t v = i & 1 ? __byte_perm(w, 0u, 0x4341) : w;      // (bytes 1 and 3)
          lo[r][i] = (v & LOW) | f[i];
          hi[r][i] = (v & HIGH) | (FIVE ? (f[i] ^ BASE) << 4 : 0u) | BASE;
          if constexpr (NUMBERS) {
            lo[r][i] = less(lo[r][i], 0.f);
            hi[r][i] = less(hi[r][i], 0.f);
          }
        }
      }
    }
    float2 s[2];
    if constexpr (M != 1) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t b = __byte_perm(sc[r][jj >> 1], 0x54006400u, jj & 1 ? 0x7352 : 0x7150);
        s[r] = __half22float2(__hadd2(*reinterpret_cast<const __half2*>(&b), __floats2half2_rn(-1024.f, -64.f)));
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int j = 2 * jj + half;
      const uint32_t(&q)[2][4] = half ? hi : lo;
      const uint32_t a0[4] = {q[0][0], q[1][0], q[0][1], q[1][1]}, a1[4] = {q[0][2], q[1][2], q[0][3], q[1][3]};
      if constexpr (M == 1) {
        if (j % 4 == 0) mma_group<M, true>(one[j / 4], a0, x, j, 0);
        else mma_group<M, false>(one[j / 4], a0, x, j, 0);
        mma_group<M, false>(one[j / 4], a1, x, j, 1);
      } else {
        float c[4];
        mma_32(c, a0, a1, x, j);
        sum.add(c, half ? s[0].y : s[0].x, half ? s[1].y : s[1].x);
      }
    }
  }
  if constexpr (M == 1) {
    const float odd = t & 1 ? 0.0625f : 1.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) s[r] = __uint_as_float(__byte_perm(sc[r][i], 0x4B000000u, 0x7650 | t)) - 0x1p23f;
      sum.add(one[i], s[0] * odd, s[1] * odd);
    }
  }
  float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = Columns<M>::PARTS - 1; i >= 0; --i) mma_f16_k8(c, am[0], am[1], x.sum[i]);
  acc.clear();
  acc.add(c, dm[0], dm[1]);
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int i = 0; i < Result<M>::N; ++i) acc.v[r][i] = fmaf(d[r], sum.v[r][i], acc.v[r][i]);
}

// The 32-bit word at a 4-byte (FOUR) or 2-byte aligned address.
template <bool FOUR>
XM_DEV uint32_t lds_word(const uint8_t* p) {
  if constexpr (FOUR) return *reinterpret_cast<const uint32_t*>(p);
  const uint32_t sh = ((uint32_t)(uintptr_t)p & 2) * 8;
  const uint32_t* a = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
  return __funnelshift_r(a[0], a[1], sh);
}

// The bytes 0 and 2, or 1 and 3, of w as numbers less BIAS.
template <int BIAS>
XM_DEV uint32_t signed_pair(uint32_t w, bool odd) { return less(__byte_perm(w, OVER, odd ? 0x7371 : 0x7270), BIAS); }

// Q6_K: w = d s_g (c - 32), groups of 16, records at any even address (every other one at a multiple of four: FOUR).  Codes are
// put together as bytes, four at a time.  (Offsets by the sums of groups, as Q4_K has them, would cost small weights their
// bits: those are differences there.)
template <int M, bool FOUR>
XM_DEV void unit_q6k(const uint8_t* r0, const uint8_t* r1, int t, const Columns<M>& x, Result<M>& acc) {
  uint32_t sc[2][4];                       // s + 128, bytes
  float d[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const uint8_t* p = r ? r1 : r0;
    // words of the scales at 192 and of d behind them
    const uint32_t sh = ((uint32_t)(uintptr_t)p & 2) * 8;
    const uint32_t* a = reinterpret_cast<const uint32_t*>((reinterpret_cast<uintptr_t>(p) + 192) & ~(uintptr_t)3);
    const uint32_t w[5] = {a[0], a[1], a[2], a[3], a[4]};
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[r][i] = __funnelshift_r(w[i], w[i + 1], sh) ^ 0x80808080u;
    const uint32_t dw = w[4] >> sh;
    d[r] = __half2float(__ushort_as_half((unsigned short)dw));
  }
  float one[4][4];                         // M = 1: the sums of groups t, t + 4, ...
  Result<M> sum;
  sum.clear();
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t low[2][2], high[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t* q = r ? r1 : r0;
        low[r][0] = lds_word<FOUR>(q + 64 * h + 16 * p + 4 * t);
        low[r][1] = lds_word<FOUR>(q + 64 * h + 32 + 16 * p + 4 * t);
        high[r] = lds_word<FOUR>(q + 128 + 32 * h + 16 * p + 4 * t);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int g = 8 * h + 2 * i + p;                          // the group of 16
        uint32_t q[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t nib = i < 2 ? low[r][i & 1] : low[r][i & 1] >> 4;
          const uint32_t two = i == 0 ? high[r] << 4 : i == 1 ? high[r] << 2 : i == 2 ? high[r] : high[r] >> 2;
          const uint32_t c4 = (nib & 0x0f0f0f0fu) | (two & 0x30303030u);
          q[r][0] = signed_pair<32>(c4, false);
          q[r][1] = signed_pair<32>(c4, true);
        }
        const uint32_t a[4] = {q[0][0], q[1][0], q[0][1], q[1][1]};
        if constexpr (M == 1) {
          // (groups 4 i + p, then 4 i + 2 + p: the first of a four is p = 0, i even)
          if (p == 0 && !(i & 1)) mma_group<M, true>(one[g >> 2], a, x, g >> 1, g & 1);
          else mma_group<M, false>(one[g >> 2], a, x, g >> 1, g & 1);
        } else {
          float c[4], s[2];
          mma_16(c, a, x, g >> 1, g & 1);
#pragma unroll
          for (int r = 0; r < 2; ++r)
            s[r] = __uint_as_float(__byte_perm(sc[r][g >> 2], 0x4B000000u, 0x7650 | (g & 3))) - (0x1p23f + 128.f);
          sum.add(c, s[0], s[1]);
        }
      }
    }
  if constexpr (M == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float s[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        s[r] = __uint_as_float(__byte_perm(sc[r][i], 0x4B000000u, 0x7650 | t)) - (0x1p23f + 128.f);
      sum.add(one[i], s[0], s[1]);
    }
  }
  acc.clear();
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int i = 0; i < Result<M>::N; ++i) acc.v[r][i] = d[r] * sum.v[r][i];
}

// Q8_0: w = d_j c, eight records of 34 bytes.
template <int M>
XM_DEV void unit_q80(const uint8_t* r0, const uint8_t* r1, int t, const Columns<M>& x, Result<M>& acc) {
  uint32_t dd[2] = {0u, 0u};               // d_2t, d_2t+1
  if constexpr (M != 1) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* p = (r ? r1 : r0) + 68 * t;
      dd[r] = (uint32_t)*reinterpret_cast<const unsigned short*>(p) |
              (uint32_t)*reinterpret_cast<const unsigned short*>(p + 34) << 16;
    }
  }
  acc.clear();
  float one[2][4];                         // M = 1: the sums of groups t and t + 4
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint32_t w[2][2];
    float s[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* p = (r ? r1 : r0) + 34 * j + 2 + 4 * t;
      if (j & 1) {
        w[r][0] = *reinterpret_cast<const uint32_t*>(p);
        w[r][1] = *reinterpret_cast<const uint32_t*>(p + 16);
      } else {
        const uint32_t* a = reinterpret_cast<const uint32_t*>(p - 2);
        w[r][0] = __funnelshift_r(a[0], a[1], 16);
        w[r][1] = __funnelshift_r(a[4], a[5], 16);
      }
      w[r][0] ^= 0x80808080u;
      w[r][1] ^= 0x80808080u;
      if constexpr (M != 1) {
        const uint32_t u = __shfl_sync(~0u, dd[r], (threadIdx.x & 28) | (j >> 1));
        s[r] = __half2float(__ushort_as_half((unsigned short)(j & 1 ? u >> 16 : u & 0xffffu)));
      }
    }
    const uint32_t a0[4] = {signed_pair<128>(w[0][0], false), signed_pair<128>(w[1][0], false),
                            signed_pair<128>(w[0][0], true), signed_pair<128>(w[1][0], true)};
    const uint32_t a1[4] = {signed_pair<128>(w[0][1], false), signed_pair<128>(w[1][1], false),
                            signed_pair<128>(w[0][1], true), signed_pair<128>(w[1][1], true)};
    if constexpr (M == 1) {
      if (j % 4 == 0) mma_group<M, true>(one[j / 4], a0, x, j, 0);
      else mma_group<M, false>(one[j / 4], a0, x, j, 0);
      mma_group<M, false>(one[j / 4], a1, x, j, 1);
    } else {
      float c[4];
      mma_32(c, a0, a1, x, j);
      acc.add(c, s[0], s[1]);
    }
  }
  if constexpr (M == 1) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float s[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)
        s[r] = __half2float(*reinterpret_cast<const __half*>((r ? r1 : r0) + 34 * (t + 4 * i)));
      acc.add(one[i], s[0], s[1]);
    }
  }
}

template <int T, int M>
XM_DEV void unit(const uint8_t* r0, const uint8_t* r1, int t, const Columns<M>& x, Result<M>& acc) {
  static_assert(M != 1 || own_value<T>(), "one scale for a group of values");
  if constexpr (T == T_Q4_K) unit_k<false, M>(r0, r1, t, x, acc);
  else if constexpr (T == T_Q5_K) unit_k<true, M>(r0, r1, t, x, acc);
  else if constexpr (T == T_Q6_K) {
    if (__all_sync(~0u, (((uintptr_t)r0 | (uintptr_t)r1) & 2) == 0)) unit_q6k<M, true>(r0, r1, t, x, acc);
    else unit_q6k<M, false>(r0, r1, t, x, acc);
  }
  else if constexpr (T == T_Q8_0) unit_q80<M>(r0, r1, t, x, acc);
  else unit_any<T, M>(r0, r1, t, x, acc);
}

template <int T>
constexpr int block_bytes() { return QT<T>::QK == 256 ? QT<T>::REC : 8 * QT<T>::REC; }   // of 256 values

template <int T, int M, bool UP>
struct Step {
  static constexpr int RB = block_bytes<T>(), N = Result<M>::N;
  const StepArgs& a;
  StepShared& sm;
  uint8_t* ring;
  float* red;                              // [ring][warp][lane][2 N]
  int lane, warp, g, t, P, per_seg, stage_bytes, s0, s1;

  XM_DEV Step(const StepArgs& a_, StepShared& s, uint8_t* dyn) : a(a_), sm(s) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    g = lane >> 2;
    t = lane & 3;
    P = a.T * a.k;
    ring = dyn;
    stage_bytes = a.boxes * 16 * a.tps * a.pitch;
    red = reinterpret_cast<float*>(dyn + a.ring * stage_bytes);
    per_seg = a.chunks * a.groups;         // stages of a segment: (chunk, group of tiles)
  }
  // A stage's place.
  struct Where {
    int seg, chunk, group;
  };
  XM_DEV Where where(int s) const {
    Where w;
    w.seg = s / per_seg;
    const int in = s - w.seg * per_seg;
    w.chunk = in / a.groups;
    w.group = in - w.chunk * a.groups;
    return w;
  }
  XM_DEV int tiles_of(int group) const { return min(a.tps, a.tiles - group * a.tps); }

  // Which pairs go to which expert, and the segments: an expert and up to M of its pairs.
  XM_DEV void segments() {
    if (a.T == 1) {                        // (in order as they are)
      if ((int)threadIdx.x < P) {
        sm.seg_e[threadIdx.x] = (uint8_t)__ldcg(a.top_e + threadIdx.x);
        sm.seg_at[threadIdx.x] = sm.pair[threadIdx.x] = (unsigned short)threadIdx.x;
        sm.seg_n[threadIdx.x] = 1;
      }
      if (threadIdx.x == 0) sm.n_seg = P;
      __syncthreads();
      share();
      return;
    }
    for (int i = threadIdx.x; i < P; i += kStepThreads) sm.expert[i] = (uint8_t)__ldcg(a.top_e + i);
    for (int e = threadIdx.x; e < a.E; e += kStepThreads) sm.cnt[e] = 0;
    __syncthreads();
    if (warp == 0) {
      for (int i0 = 0; i0 < P; i0 += 32) {
        const int i = i0 + lane, e = i < P ? sm.expert[i] : -1 - lane;
        const unsigned same = __match_any_sync(~0u, e);
        const int before = i < P ? sm.cnt[e] : 0;
        __syncwarp();
        if (i < P) {
          sm.rank[i] = (uint8_t)(before + __popc(same & ((1u << lane) - 1)));
          if (lane == __ffs(same) - 1) sm.cnt[e] = before + __popc(same);
        }
        __syncwarp();
      }
      int at = 0, segs = 0;
      for (int e0 = 0; e0 < a.E; e0 += 32) {
        const int e = e0 + lane, n = e < a.E ? sm.cnt[e] : 0, s = (n + M - 1) / M;
        int sum = n | s << 16;             // (both sums stay below 2^15)
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += u;
        }
        const int first = at + (sum & 0xffff) - n, seg = segs + (sum >> 16) - s;
        if (e < a.E) sm.off[e] = first;
        for (int i = 0; i < s; ++i) {
          sm.seg_e[seg + i] = (uint8_t)e;
          sm.seg_at[seg + i] = (unsigned short)(first + i * M);
          sm.seg_n[seg + i] = (uint8_t)min(M, n - i * M);
        }
        const int all = __shfl_sync(~0u, sum, 31);
        at += all & 0xffff;
        segs += all >> 16;
      }
      if (lane == 0) sm.n_seg = segs;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < P; i += kStepThreads) sm.pair[sm.off[sm.expert[i]] + sm.rank[i]] = (unsigned short)i;
    __syncthreads();
    share();
  }
  // This CTA's stages.
  XM_DEV void share() {
    const int64_t total = (int64_t)sm.n_seg * per_seg;
    s0 = (int)(total * blockIdx.x / gridDim.x);
    s1 = (int)(total * (blockIdx.x + 1) / gridDim.x);
  }

  // One of two threads that have the stage's rows copied to its slot: UP the first those of W1, the second those of W3; DOWN
  // the even and the odd boxes.
  XM_DEV void fill(int s, int slot, int which) {
    const Where w = where(s);
    const int e = sm.seg_e[w.seg];
    uint64_t* bar = &sm.full[slot];
    constexpr int ROWS = UP ? 8 : 16;      // of a tile, of one matrix
    const int block = ROWS * a.tps * a.pitch, first = w.group * a.tps * ROWS;
    uint8_t* to = ring + slot * stage_bytes + (UP ? which * block : 0);
    if (a.copies == kTensor) {
      // (rows past the weight's last and columns past a row's end arrive as zeros; boxes wholly past it are left out)
      const int sbs = min(a.kc, a.nsb - w.chunk * a.kc), n = (sbs + a.box_sb - 1) / a.box_sb;
      const int mine = UP ? n : (n + 1 - which) / 2;
      mbar_arrive_expect_tx(bar, mine * block);
      const CUtensorMap* map = (UP && which ? a.map3 : a.map1) + e;
      for (int b = UP ? 0 : which; b < n; b += UP ? 1 : 2)
        tensor_g2s(to + b * (UP ? 2 : 1) * block, map, (w.chunk * a.kc + b * a.box_sb) * RB / 8, first, bar);
      return;
    }
    const int len = min(a.kc, a.nsb - w.chunk * a.kc) * RB, rows = ROWS * tiles_of(w.group);
    const uint8_t* p = (UP && which ? sm.w3[e] : sm.w1[e]) + first * a.row_bytes + (int64_t)w.chunk * a.kc * RB;
    if (!UP && which) {
      mbar_arrive(bar);
    } else if (a.copies == kWhole) {       // (rows by eights are whole units of 16 bytes)
      mbar_arrive_expect_tx(bar, rows * len);
      bulk_g2s(to, p, rows * len, bar);
    } else {
      auto size = [&](const uint8_t* q) { return (uint32_t)(((uintptr_t)q & 15) + len + 15) & ~15u; };
      uint32_t bytes = 0;
      for (int r = 0; r < rows; ++r) bytes += size(p + r * a.row_bytes);
      mbar_arrive_expect_tx(bar, bytes);
#pragma unroll 1
      for (int r = 0; r < rows; ++r, p += a.row_bytes)
        bulk_g2s(to + r * a.pitch, (const void*)((uintptr_t)p & ~(uintptr_t)15), size(p), bar);
    }
  }

  // This warp's activations of a segment and a chunk.
  static constexpr bool OFFSETS = T == T_Q4_K || T == T_Q5_K;
  XM_DEV void load_columns(Columns<M>& x, int seg, int k0, bool mine) {
    if constexpr (M == 1) load_one(x, seg, k0, mine);
    else load_several(x, seg, k0, mine);
  }
  // The one token's: a lane has the groups g / 2, g / 2 + 4, ... alone.
  XM_DEV void load_one(Columns<M>& x, int seg, int k0, bool mine) {
    constexpr int G = T == T_Q6_K ? 16 : 8, V = 256 / G / 4;     // groups, a lane's values of one
    const int pair = sm.pair[sm.seg_at[seg]], row = UP ? pair / a.k : pair, own = g >> 1;
    const float* p = a.src + (int64_t)row * a.K + k0;
    float v[G / 4][V], m = 0.f;
#pragma unroll
    for (int i = 0; i < G / 4; ++i)
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        // (values 8 t .. 8 t + 7 of a group of 32, or 4 t .. 4 t + 3 of each 16)
        const int at = (own + 4 * i) * (256 / G) + (halves<T>() ? 4 * q + 4 * t : 8 * t + q);
        const float4 u = mine ? __ldcg(reinterpret_cast<const float4*>(p + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[i][q] = u.x;
        v[i][q + 1] = u.y;
        v[i][q + 2] = u.z;
        v[i][q + 3] = u.w;
        m = fmaxf(m, fmaxf(fmaxf(fabsf(u.x), fabsf(u.y)), fmaxf(fabsf(u.z), fabsf(u.w))));
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    const int shift = fp16_row_shift(m);
    const float inv = ldexpf(1.0f, -shift);
    x.scale[0] = ldexpf(1.0f, shift);
    auto part = [&](float f) { return g & 1 ? f - upper<OFFSETS>(f) : upper<OFFSETS>(f); };
    float sum[G / 4];
#pragma unroll
    for (int i = 0; i < G / 4; ++i) {
      float z = 0.f;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        v[i][q] *= inv;
        z += v[i][q];
      }
      z += __shfl_xor_sync(~0u, z, 1);
      z += __shfl_xor_sync(~0u, z, 2);
      sum[i] = z * 0x1p-5f;
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const uint32_t b0 = pack2(part(v[i][q]), part(v[i][q + 2])), b1 = pack2(part(v[i][q + 1]), part(v[i][q + 3]));
#pragma unroll
        for (int c = 0; c < 4; ++c) {      // (zero in the groups that are others')
          const int at = 4 * i + c;        // the group
          const int j = G == 16 ? at / 2 : at, w = G == 16 ? 2 * (at & 1) : q / 2;
          x.b[0][j][w] = c == own ? b0 : 0u;
          x.b[0][j][w + 1] = c == own ? b1 : 0u;
        }
      }
    }
    if constexpr (OFFSETS) {               // groups 2 t, 2 t + 1 in columns 0 and 1: group n is with the lanes of g / 2 = n % 4
      float q[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int n = 2 * t + i;
        const float z0 = __shfl_sync(~0u, sum[0], (n & 3) * 8), z1 = __shfl_sync(~0u, sum[1], (n & 3) * 8);
        q[i] = g < 2 ? part(n < 4 ? z0 : z1) : 0.f;
      }
      x.sum[0] = pack2(q[0], q[1]);
    }
  }
  XM_DEV void load_several(Columns<M>& x, int seg, int k0, bool mine) {
    const int col = M == 4 ? g >> 1 : g;
    const bool there = mine && col < sm.seg_n[seg], rest = M == 4 && (g & 1);      // (this column has the low parts)
    const int pair = there ? sm.pair[sm.seg_at[seg] + col] : 0, row = UP ? pair / a.k : pair;
    const float* p = a.src + (int64_t)row * a.K + k0 + (halves<T>() ? 4 : 8) * t;
    // all of the column's 256 values first: their power of two
    float4 u[8][2];
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        u[j][i] = there ? __ldcg(reinterpret_cast<const float4*>(p + 32 * j + i * (halves<T>() ? 16 : 4)))
                        : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        m = fmaxf(m, fmaxf(fmaxf(fabsf(u[j][i].x), fabsf(u[j][i].y)), fmaxf(fabsf(u[j][i].z), fabsf(u[j][i].w))));
    m = fmaxf(m, __shfl_xor_sync(~0u, m, 1));
    m = fmaxf(m, __shfl_xor_sync(~0u, m, 2));
    const int shift = fp16_row_shift(m);
    const float inv = ldexpf(1.0f, -shift), own = ldexpf(1.0f, shift);
    if constexpr (M == 4) {
      x.scale[0] = __shfl_sync(~0u, own, 8 * t);
    } else {
      x.scale[0] = __shfl_sync(~0u, own, 8 * t);
      x.scale[1] = __shfl_sync(~0u, own, 8 * t + 4);
    }
    float sum[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v[8] = {u[j][0].x * inv, u[j][0].y * inv, u[j][0].z * inv, u[j][0].w * inv,
                    u[j][1].x * inv, u[j][1].y * inv, u[j][1].z * inv, u[j][1].w * inv};
      sum[j] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      float top[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        top[i] = upper<false>(v[i]);
        v[i] -= top[i];
      }
#pragma unroll
      for (int q = 0; q < Columns<M>::PARTS; ++q) {
        const bool lower = q || rest;
        x.b[q][j][0] = pack2(lower ? v[0] : top[0], lower ? v[2] : top[2]);
        x.b[q][j][1] = pack2(lower ? v[1] : top[1], lower ? v[3] : top[3]);
        x.b[q][j][2] = pack2(lower ? v[4] : top[4], lower ? v[6] : top[6]);
        x.b[q][j][3] = pack2(lower ? v[5] : top[5], lower ? v[7] : top[7]);
      }
    }
    if constexpr (OFFSETS) {
      float q[2] = {0.f, 0.f};             // sums of groups 2 t, 2 t + 1
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float z = sum[j];
        z += __shfl_xor_sync(~0u, z, 1);
        z += __shfl_xor_sync(~0u, z, 2);
        if (j >> 1 == t) q[j & 1] = z * 0x1p-5f;
      }
#pragma unroll
      for (int c = 0; c < Columns<M>::PARTS; ++c) {
        const bool lower = c || rest;
        x.sum[c] = pack2(lower ? q[0] - upper<false>(q[0]) : upper<false>(q[0]), lower ? q[1] - upper<false>(q[1]) : upper<false>(q[1]));
      }
    }
  }

  // Whether this warp is the one that writes the last of `all` results under a ticket.
  XM_DEV bool last(int* ticket, int all) {
    __threadfence();
    __syncwarp();
    int old = 0;
    if (lane == 0) old = atomicAdd(ticket, 1);
    old = __shfl_sync(~0u, old, 0);
    if (old != all - 1) return false;
    __threadfence();
    return true;
  }

  // The stage's results are added up and written (one warp).
  XM_DEV void finish(int s, int slot, int lap) {
    const Where w = where(s);
    const int at = sm.seg_at[w.seg], n_pairs = sm.seg_n[w.seg], kc = min(a.kc, a.nsb - w.chunk * a.kc);
    const int tiles = tiles_of(w.group), tile0 = w.group * a.tps;
    int pair[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = M == 8 ? 2 * t + n : t;
      pair[n] = i < n_pairs ? sm.pair[at + i] : -1;
    }
    auto result = [&](int n, int i, float gate, float up) {       // a feature of the first products
      a.dst[(int64_t)pair[n] * a.N + (tile0 + i) * 8 + g] = xm_act(a.act, gate) * up;
    };
    mbar_wait_bounded(&sm.done[slot], lap & 1);
    for (int i = 0; i < tiles; ++i) {
      Result<M> v;
      v.clear();
      const float* r = red + ((slot * kWorkers + i * a.kc) * 32 + lane) * 2 * N;
#pragma unroll 4
      for (int q = 0; q < kc; ++q) {
        if constexpr (N == 1) {
          const float2 u = *reinterpret_cast<const float2*>(r + q * 64);
          v.v[0][0] += u.x;
          v.v[1][0] += u.y;
        } else {
          const float4 u = *reinterpret_cast<const float4*>(r + q * 128);
          v.v[0][0] += u.x;
          v.v[0][1] += u.y;
          v.v[1][0] += u.z;
          v.v[1][1] += u.w;
        }
      }
      if constexpr (M == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          v.v[h][0] += __shfl_xor_sync(~0u, v.v[h][0], 1);
          v.v[h][0] += __shfl_xor_sync(~0u, v.v[h][0], 2);
        }
      }
      if (i + 1 == tiles) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[slot]);
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (pair[n] < 0) continue;
        const float y0 = v.v[0][n], y1 = v.v[1][n];
        if (!UP) {
          float* p = a.dst + ((int64_t)w.chunk * P + pair[n]) * a.N + (tile0 + i) * 16 + g;
          p[0] = y0;
          p[8] = y1;
        } else if (a.chunks == 1) {
          result(n, i, y0, y1);
        } else {
          float* p = a.part + ((int64_t)w.chunk * P + pair[n]) * 2 * a.N + (tile0 + i) * 8 + g;
          p[0] = y0;
          p[a.N] = y1;
        }
      }
    }
    __syncwarp();
    if (UP && a.chunks > 1 && last(a.tickets + w.seg * a.groups + w.group, a.chunks)) {
      for (int i = 0; i < tiles; ++i) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (pair[n] < 0) continue;
          float gate = 0.f, up = 0.f;
          for (int q = 0; q < a.chunks; ++q) {
            const float* p = a.part + ((int64_t)q * P + pair[n]) * 2 * a.N + (tile0 + i) * 8 + g;
            gate += __ldcg(p);
            up += __ldcg(p + a.N);
          }
          result(n, i, gate, up);
        }
      }
      __syncwarp();
    }
  }

  XM_DEV void copy(int which) {            // (one thread)
    int slot = 0, lap = 0;
    for (int s = s0; s < s1; ++s) {
      if (lap > 0) mbar_wait_bounded(&sm.empty[slot], (lap - 1) & 1);
      fill(s, slot, which);
      if (++slot == a.ring) {
        slot = 0;
        ++lap;
      }
    }
  }

  XM_DEV void finishes(int which) {        // (every other stage)
    int slot = 0, lap = 0;
    for (int s = s0; s < s1; ++s) {
      if (((s - s0) & 1) == which) finish(s, slot, lap);
      if (++slot == a.ring) {
        slot = 0;
        ++lap;
      }
    }
  }

  XM_DEV void multiply() {
    const int my_tile = warp / a.kc, my_sb = warp - my_tile * a.kc;
    const int my_box = my_sb / a.box_sb, second = (UP ? 8 * a.tps : 8) * a.pitch;      // (from a row to the one with g + 8)
    const int mine_at = my_box * 16 * a.tps * a.pitch + (my_tile * (UP ? 8 : 16) + g) * a.pitch + (my_sb - my_box * a.box_sb) * RB;
    float* const mine_red = red + (warp * 32 + lane) * 2 * N;
    Columns<M> x;
    int slot = 0, lap = 0, left = 0, tile = 0, chunk = 0;
    bool in_k = false;
    for (int s = s0; s < s1; ++s) {
      if (left == 0) {                     // another segment or part of K
        const Where w = where(s);
        left = a.groups - w.group;
        chunk = w.chunk;
        tile = w.group * a.tps + my_tile;
        in_k = my_tile < a.tps && chunk * a.kc + my_sb < a.nsb;
        load_columns(x, w.seg, (chunk * a.kc + my_sb) * 256, in_k);
      }
      if (!mbar_test(&sm.full[slot], lap & 1)) mbar_wait_bounded(&sm.full[slot], lap & 1);
      if (in_k && tile < a.tiles) {
        const uint8_t* r0 = ring + slot * stage_bytes + mine_at;
        const uint8_t* r1 = r0 + second;
        if (RB % 16 != 0 && a.copies == kRows) {    // (a row's bytes begin where they do in 16 bytes of the weight)
          const int n = tile * (UP ? 8 : 16) + g;
          const int64_t col = (int64_t)chunk * a.kc * RB;
          r0 += (int)(n * a.row_bytes + col) & 15;
          r1 += (int)((UP ? n : n + 8) * a.row_bytes + col) & 15;
        }
        Result<M> acc;
        unit<T, M>(r0, r1, t, x, acc);
        float* r = mine_red + slot * (kWorkers * 32 * 2 * N);
        if constexpr (N == 1)
          *reinterpret_cast<float2*>(r) = make_float2(acc.v[0][0] * x.scale[0], acc.v[1][0] * x.scale[0]);
        else
          *reinterpret_cast<float4*>(r) = make_float4(acc.v[0][0] * x.scale[0], acc.v[0][1] * x.scale[N - 1],
                                                      acc.v[1][0] * x.scale[0], acc.v[1][1] * x.scale[N - 1]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.done[slot]);
      if (++slot == a.ring) {
        slot = 0;
        ++lap;
      }
      --left;
      tile += a.tps;
    }
  }
};

template <int T, int M, bool UP>
__global__ void __launch_bounds__(kStepThreads, 1) k_moe_step(StepArgs a) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ StepShared sm;
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.ring; ++i) {
      mbar_init(&sm.full[i], kCopiers);
      mbar_init(&sm.done[i], kWorkers);
      mbar_init(&sm.empty[i], 1);
    }
    fence_mbar_init();
  }
  if (a.copies != kTensor)
    for (int e = threadIdx.x; e < a.E; e += kStepThreads) {
      sm.w1[e] = a.w1[e];
      if (UP) sm.w3[e] = a.w3[e];
    }
  // DOWN reads the routing, and the weights that it names, before its wait: it is complete before DOWN can start, since UP
  // waits for it and only then lets DOWN start
  if (UP) grid_dep_wait();
  grid_dep_launch();
  Step<T, M, UP> step(a, sm, dyn);
  step.segments();
  if (step.warp < kWorkers) {
    if (!UP) grid_dep_wait();
    step.multiply();
  } else if (step.warp < kWorkers + kCopiers) {
    if (step.lane == 0) step.copy(step.warp - kWorkers);
  } else {
    if (!UP) grid_dep_wait();
    step.finishes(step.warp - kWorkers - kCopiers);
  }
}

// The outputs, a thread each.  (The last writer of some rows could add them up in DOWN, but its fence and its ticket cost more
// than a launch that is there when DOWN ends: one token, 2 of 8 experts, 7 us.)
__global__ void __launch_bounds__(256) k_moe_step_sum(StepArgs a) {
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x * 256 + threadIdx.x;
  step_output(a, blockIdx.y, row);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct Plan {
  int nsb, chunks, kc, tps, tiles, groups, boxes, box_sb, pitch, ring, smem, copies;
};

// K values a row, `tiles` tiles of sixteen rows; rb: bytes of 256 values, read by 4 bytes (half) or 8; M tokens; up: the first
// products, whose parts of K cost more to put together.
Plan plan(int64_t K, int64_t tiles, int rb, bool half, int M, bool up) {
  Plan p;
  p.nsb = (int)(K / 256);
  p.copies = (int64_t)p.nsb * rb % 16 == 0 ? kTensor : p.nsb <= kWorkers ? kWhole : kRows;
  // parts of K: of as many 256-blocks as leave the fewest warps without work; parts and boxes begin at whole units of 16 bytes
  const int step = p.copies == kTensor ? 16 / std::__gcd(rb, 16) : 1;
  double best = 1e9;
  for (int kc = step; kc <= kWorkers; kc += step) {
    const int chunks = (p.nsb + kc - 1) / kc;
    if (p.copies == kWhole && chunks > 1) continue;
    const double cost = (double)chunks / (kWorkers / kc) * (1 + (up ? 0.25 : 0.04) * (chunks - 1));
    if (cost < best - 1e-9 || (cost < best + 1e-9 && chunks < p.chunks)) {
      best = cost;
      p.kc = kc;
      p.chunks = chunks;
    }
  }
  p.kc = std::min(p.kc, p.nsb);
  p.tps = kWorkers / p.kc;
  p.tiles = (int)tiles;
  p.groups = (p.tiles + p.tps - 1) / p.tps;
  // What the four lanes of a row read should fall on other banks than the next rows': 8 bytes each, rows 32 bytes apart modulo
  // 64; 4 bytes each, 16 apart modulo 32.
  const int odd = half ? 32 : 64, rest = half ? 16 : 32;
  auto pitched = [&](int bytes) {
    bytes = (bytes + 15) / 16 * 16;
    return bytes + (odd + rest - bytes % odd) % odd;
  };
  p.boxes = 1;
  p.box_sb = p.kc;
  if (p.copies == kTensor) {
    // a box row is at most 256 elements of 8 bytes; of the numbers of boxes that allow it the one that wastes least
    int least = 1 << 30;
    for (int boxes = 1; boxes <= p.kc; ++boxes) {
      const int sb = ((p.kc + boxes - 1) / boxes + step - 1) / step * step, n = (p.kc + sb - 1) / sb, pitch = pitched(sb * rb);
      if (pitch <= 2048 && n * pitch + 64 * n < least) {       // (64 bytes a row for another instruction)
        least = n * pitch + 64 * n;
        p.boxes = n;
        p.box_sb = sb;
        p.pitch = pitch;
      }
    }
  } else {
    p.pitch = p.copies == kWhole ? p.kc * rb : pitched(p.kc * rb + 15);
  }
  const int stage = p.boxes * 16 * p.tps * p.pitch, red = kWorkers * 32 * 2 * (M == 8 ? 2 : 1) * 4;
  p.ring = std::min(kMaxRing, (227 * 1024 - (int)sizeof(StepShared) - 1024) / (stage + red));
  p.smem = p.ring * (stage + red);
  return p;
}
Plan plan_up(int64_t H, int64_t F, int rb, bool half, int M) { return plan(H, F / 8, rb, half, M, true); }
Plan plan_down(int64_t H, int64_t F, int rb, bool half, int M) { return plan(F, H / 16, rb, half, M, false); }

struct Layout {
  int64_t top_e, top_w, v, a, part, tickets, up_part, bytes;
  int n_tickets;
};
Layout layout(int64_t T, int64_t H, int64_t F, int64_t k, int rb, bool half) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t o = at;
    at += (n * 4 + 255) / 256 * 256;
    return o;
  };
  const int64_t P = T * k;
  const Plan up = plan_up(H, F, rb, half, 4), down = plan_down(H, F, rb, half, 4);    // (parts and groups go by neither M)
  l.top_e = take(P);
  l.top_w = take(P);
  l.v = take(T * H);
  l.a = take(P * F);
  l.part = take((int64_t)down.chunks * P * H);
  l.n_tickets = up.chunks > 1 ? (int)P * up.groups : 0;
  l.tickets = take(l.n_tickets);
  l.up_part = take(up.chunks > 1 ? (int64_t)up.chunks * P * 2 * F : 0);
  l.bytes = at;
  return l;
}

template <auto KERNEL, typename... Args>
cudaError_t step_launch(dim3 grid, int threads, int smem, int cluster, cudaStream_t st, Args... args) {
  static bool done[64] = {};               // (the kernel may have all shared memory, by device)
  int dev = 0;
  cudaError_t e = smem > 0 ? cudaGetDevice(&dev) : cudaSuccess;
  if (e != cudaSuccess) return e;
  if (smem > 0 && (dev >= 64 || !done[dev])) {
    cudaFuncAttributes at;
    e = cudaFuncGetAttributes(&at, KERNEL);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)at.sharedSizeBytes);
    if (e != cudaSuccess) return e;
    if (dev < 64) done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, KERNEL, args...);
}

template <int T, int M>
cudaError_t step_products(StepArgs up, StepArgs down, int64_t H, int64_t F, cudaStream_t st) {
  const int sms = xm_sm_count();
  auto fill = [](StepArgs& a, const Plan& p) {
    a.nsb = p.nsb;
    a.chunks = p.chunks;
    a.kc = p.kc;
    a.tps = p.tps;
    a.tiles = p.tiles;
    a.groups = p.groups;
    a.row_bytes = (int64_t)p.nsb * block_bytes<T>();
    a.boxes = p.boxes;
    a.box_sb = p.box_sb;
    a.pitch = p.pitch;
    a.ring = p.ring;
    a.copies = p.copies;
  };
  const Plan pu = plan_up(H, F, block_bytes<T>(), halves<T>(), M), pd = plan_down(H, F, block_bytes<T>(), halves<T>(), M);
  fill(up, pu);
  fill(down, pd);
  if (pu.ring < 2 || pd.ring < 2) return cudaErrorInvalidConfiguration;    // (no type and size has so few)
  cudaError_t e = step_launch<k_moe_step<T, M, true>>(dim3(sms), kStepThreads, pu.smem, 1, st, up);
  if (e == cudaSuccess) e = step_launch<k_moe_step<T, M, false>>(dim3(sms), kStepThreads, pd.smem, 1, st, down);
  if (e == cudaSuccess) e = step_launch<k_moe_step_sum>(dim3((unsigned)(H / 256), (unsigned)down.T), 256, 0, 1, st, down);
  return e;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static EncodeTiled fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(p);
  });
  return fn;
}

// Sizes that the step takes; qk and record bytes of the type.
int check_sizes(int64_t H, int64_t F, int E, int qtype, int* qk, int* rec) {
  if (!host_qtype_geometry(qtype, qk, rec) || *qk < 32)
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: expert weights of type id %d", qtype);
  if (H < 256 || H % 256 || H > kMaxHidden || F < 256 || F % 256 || F > (1 << 20))
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: experts of %lld -> %lld (multiples of 256; hidden up to %d)",
                        (long long)H, (long long)F, kMaxHidden);
  if (E < 1 || E > kMaxStepExperts)
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: %d experts (up to %d)", E, kMaxStepExperts);
  return XM_OK;
}
bool by_halves(int qtype) { return qtype == T_Q6_K || qtype == T_Q8_0; }
static_assert(halves<T_Q6_K>() && halves<T_Q8_0>() && !halves<T_Q4_K>(), "by_halves() says what halves() does");

// A table: 3 E tensor maps (w1, w3, w2), then 3 E pointers.
struct Table {
  const CUtensorMap* maps;
  const uint8_t* const* weights;
};
Table table_at(const void* d, int E) {
  return {(const CUtensorMap*)d, (const uint8_t* const*)((const uint8_t*)d + (int64_t)3 * E * sizeof(CUtensorMap))};
}

}  // namespace

extern "C" {

int64_t xm_moe_step_workspace_size(int64_t T, int64_t H, int64_t F, int E, int k, int qtype) {
  int qk = 0, rec = 0;
  if (T < 1 || T > kMaxTokens || k < 1 || k > E || k > kMaxTop || check_sizes(H, F, E, qtype, &qk, &rec) != XM_OK) return 0;
  return layout(T, H, F, k, 256 / qk * rec, by_halves(qtype)).bytes;
}

int64_t xm_moe_step_table_size(int E) {
  return E < 1 || E > kMaxStepExperts ? 0 : (int64_t)3 * E * (sizeof(CUtensorMap) + sizeof(void*));
}

int xm_moe_step_table(int qtype, int64_t H, int64_t F, int E, const void* const* h_w1, const void* const* h_w3,
                      const void* const* h_w2, void* h_table) {
  int qk = 0, rec = 0;
  const int st = check_sizes(H, F, E, qtype, &qk, &rec);
  if (st != XM_OK) return st;
  if (!h_w1 || !h_w3 || !h_w2 || !h_table) return xm_set_error(XM_ERR_INVALID, "moe_step_table: null pointer");
  const int rb = 256 / qk * rec;
  const Plan up = plan_up(H, F, rb, by_halves(qtype), 4), down = plan_down(H, F, rb, by_halves(qtype), 4);
  std::memset(h_table, 0, (size_t)xm_moe_step_table_size(E));
  CUtensorMap* maps = (CUtensorMap*)h_table;
  const void** weights = (const void**)(maps + 3 * E);
  for (int i = 0; i < 3 * E; ++i) {
    const void* w = i < E ? h_w1[i] : i < 2 * E ? h_w3[i - E] : h_w2[i - 2 * E];
    if (!w || ((uintptr_t)w & 15))
      return xm_set_error(XM_ERR_INVALID, "moe_step_table: weight %d of expert %d is null or not 16-byte aligned", i / E, i % E);
    weights[i] = w;
    const Plan& p = i < 2 * E ? up : down;
    if (p.copies != kTensor) continue;
    EncodeTiled encode = encode_tiled();
    if (!encode) return xm_set_error(XM_ERR_CUDA, "moe_step_table: cuTensorMapEncodeTiled unavailable");
    CUtensorMap map;                       // (64-byte aligned, which the caller's memory need not be)
    const cuuint64_t dims[2] = {(cuuint64_t)p.nsb * rb / 8, (cuuint64_t)(i < 2 * E ? F : H)};
    const cuuint64_t strides[1] = {(cuuint64_t)p.nsb * rb};
    const cuuint32_t box[2] = {(cuuint32_t)p.pitch / 8, (cuuint32_t)((i < 2 * E ? 8 : 16) * p.tps)}, one[2] = {1, 1};
    const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_INT64, 2, const_cast<void*>(w), dims, strides, box, one,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return xm_set_error(XM_ERR_CUDA, "moe_step_table: tensor map (%d)", (int)r);
    std::memcpy(&maps[i], &map, sizeof(map));
  }
  return XM_OK;
}

int xm_moe_step(const void* d_x, int x_dtype, int64_t T, int64_t H, int64_t x_stride, const float* d_norm_w, float eps,
                const float* d_gate, int E, int k, int64_t F, const void* d_table, int qtype, int activation,
                const float* d_residual, int64_t residual_stride, float* d_out, int64_t out_stride, void* d_workspace,
                int64_t workspace_bytes, void* stream) {
  if (x_dtype != XM_DT_F32 && x_dtype != XM_DT_F16 && x_dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "moe_step: bad element type %d", x_dtype);
  int qk = 0, rec = 0;
  const int ok = check_sizes(H, F, E, qtype, &qk, &rec);
  if (ok != XM_OK) return ok;
  if (T < 0 || T > kMaxTokens) return xm_set_error(XM_ERR_INVALID, "moe_step: %lld tokens (up to %d)", (long long)T, kMaxTokens);
  if (k < 1 || k > E || k > kMaxTop)
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: %d of %d experts (up to %d)", k, E, kMaxTop);
  if (activation < XM_ACT_SILU || activation > XM_ACT_IDENTITY)
    return xm_set_error(XM_ERR_INVALID, "moe_step: unknown activation %d", activation);
  if (x_stride < H || out_stride < H || (d_residual && residual_stride < H))
    return xm_set_error(XM_ERR_INVALID, "moe_step: a row pitch is below %lld values", (long long)H);
  if (T == 0) return XM_OK;
  if (!d_x || !d_gate || !d_table || !d_out || !d_workspace) return xm_set_error(XM_ERR_INVALID, "moe_step: null pointer");
  if (((uintptr_t)d_x & (x_dtype == XM_DT_F32 ? 3 : 1)) || ((uintptr_t)d_gate & 15) || ((uintptr_t)d_workspace & 255) ||
      ((uintptr_t)d_table & 63) || (((uintptr_t)d_norm_w | (uintptr_t)d_residual | (uintptr_t)d_out) & 3))
    return xm_set_error(XM_ERR_INVALID, "moe_step: unaligned pointer");
  const Layout l = layout(T, H, F, k, 256 / qk * rec, by_halves(qtype));
  if (workspace_bytes < l.bytes)
    return xm_set_error(XM_ERR_INVALID, "moe_step: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                        (long long)l.bytes);
  uint8_t* ws = (uint8_t*)d_workspace;
  auto f32 = [&](int64_t o) { return reinterpret_cast<float*>(ws + o); };
  auto i32 = [&](int64_t o) { return reinterpret_cast<int*>(ws + o); };
  cudaStream_t st = (cudaStream_t)stream;
  const RouteArgs r{d_x, x_stride, d_norm_w, d_gate, eps, (int)T, (int)H, E, k, f32(l.v), f32(l.top_w), i32(l.top_e),
                    i32(l.tickets), l.n_tickets};
  const dim3 routes((unsigned)T * kRouteCluster);
  cudaError_t e =
      x_dtype == XM_DT_F32   ? step_launch<k_moe_step_route<float>>(routes, kRouteThreads, (int)H * 8, kRouteCluster, st, r)
      : x_dtype == XM_DT_F16 ? step_launch<k_moe_step_route<__half>>(routes, kRouteThreads, (int)H * 8, kRouteCluster, st, r)
                             : step_launch<k_moe_step_route<__nv_bfloat16>>(routes, kRouteThreads, (int)H * 8, kRouteCluster, st, r);
  if (e == cudaSuccess) {
    const Table t = table_at(d_table, E);
    StepArgs up = {}, down = {};
    up.map1 = t.maps;
    up.map3 = t.maps + E;
    up.w1 = t.weights;
    up.w3 = t.weights + E;
    up.src = f32(l.v);
    up.dst = f32(l.a);
    up.part = f32(l.up_part);
    up.tickets = i32(l.tickets);
    up.top_e = i32(l.top_e);
    up.top_w = f32(l.top_w);
    up.T = (int)T;
    up.k = k;
    up.E = E;
    up.act = activation;
    up.K = (int)H;
    up.N = (int)F;
    down = up;
    down.map1 = t.maps + 2 * E;
    down.w1 = t.weights + 2 * E;
    down.src = f32(l.a);
    down.dst = f32(l.part);
    down.K = (int)F;
    down.N = (int)H;
    down.residual = d_residual;
    down.residual_stride = residual_stride;
    down.out = d_out;
    down.out_stride = out_stride;
    dispatch_quant(qtype, [&]<int Q>() {
      // Four tokens a pass while an expert has some 2.5 of them on average (five and more are then one in twenty): the registers
      // for eight do not fit, and a pass for four takes two thirds of the time.
      if (own_value<Q>() && T == 1) e = step_products<Q, own_value<Q>() ? 1 : 4>(up, down, H, F, st);
      else if (T <= 4 || 2 * T * k <= 5 * E) e = step_products<Q, 4>(up, down, H, F, st);
      else e = step_products<Q, 8>(up, down, H, F, st);
    });
  }
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "moe_step launch: %s", cudaGetErrorString(e));
  return xm_check_launch("moe_step");
}

}  // extern "C"
