// The whole mixture-of-experts layer for a few tokens (a decode step): router, the chosen experts, their weighted sum.
//
//   v = x, or x w / sqrt(mean x^2 + eps);  l = gate v;  the k largest l, p = softmax over them;
//   out = residual + sum over the k experts e, ascending, of p_e W2_e (act(W1_e v) * (W3_e v))
//
// Bound: HBM, the blocks of the experts that some token chose (each read once for up to 4 NT tokens of an expert).
//
// Three launches, each starting while the one before it ends:
//   k_moe_step_route   a cluster a token: norm, logits in 64 bits (a near tie of two experts goes one way), top k, softmax
//   k_moe_step<UP>     a = act(W1 v) * (W3 v) of every (token, expert) pair
//   k_moe_step<DOWN>   W2 a; whoever writes the last partial result of some output rows adds them up
//
// The products run on mma.sync (m16n8k16, fp16 with fp32 sums): sixteen weight rows by eight columns, a column pair per
// token: x = 2^s (hi + 2^-11 lo), both fp16, so that an activation keeps some 22 bits.  A tile of UP is eight rows of W1 and
// the same eight of W3, so that one thread holds the gate and the up value of a feature.
//
// A CTA takes a contiguous range of the stages (expert, part of K, group of row tiles).  One warp copies the rows of a stage
// into a ring in shared memory (bulk copies) and, once the 16 other warps have multiplied them, adds up their results; each
// of those holds 256 values of K of a tile, for which its activations stay in registers while the expert lasts.  Nothing
// waits for another CTA.  The results do not depend on the order in which CTAs run.
#include <cooperative_groups.h>

#include <algorithm>

#include "xm_gemv_dot.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kMaxTokens = 64, kMaxTop = 16, kMaxStepExperts = 256, kMaxPairs = kMaxTokens * kMaxTop;
constexpr int kWorkers = 16, kStepThreads = (kWorkers + 1) * 32, kMaxRing = 8;
constexpr int kRouteCluster = 8, kRouteThreads = 256;
constexpr int kMaxHidden = 16384;

struct StepArgs {
  const void* const* w1;       // (device arrays of E pointers; DOWN: w1 = the second products' weights)
  const void* const* w3;
  const float* src;            // [rows][K]: v of a token (UP), a of a pair (DOWN)
  const float* src_max;        // its largest magnitudes
  float* dst;                  // UP: a [P][F];  DOWN: partial results [chunks][P][H]
  unsigned* dst_max;           // UP: the largest magnitude of a, as bits
  float* part;                 // UP with several chunks: partial results [chunks][P][2F]
  int* tickets;                // of each group of tiles (DOWN), of each (pair group, group of tiles) (UP with chunks)
  const int* top_e;            // [T][k], ascending
  const float* top_w;
  int T, k, E, act;
  int K, N;                    // N: rows of a result (UP: F, DOWN: H)
  int nsb, chunks, kc, tps;    // 256-blocks of K, parts of K, their 256-blocks, tiles a stage
  int tiles, groups;           // row tiles, and stages that hold them
  int64_t row_bytes;
  int pitch, ring;
  const float* residual;       // DOWN
  int64_t residual_stride, out_stride;
  float* out;
};

struct alignas(128) StepShared {
  uint64_t full[kMaxRing], done[kMaxRing];
  int n_seg, last;
  int cnt[kMaxStepExperts], off[kMaxStepExperts];
  unsigned short pair[kMaxPairs];                      // pairs (token * k + slot) by expert, then token
  unsigned short seg_e[kMaxPairs], seg_at[kMaxPairs], seg_n[kMaxPairs];
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
  float *v, *v_max, *top_w;
  int* top_e;
  unsigned* a_max;             // [T * k], zeroed
  int *tickets, n_tickets;     // zeroed
};

XM_DEV double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// A cluster of 8 CTAs a token: each has the whole row and an eighth of the experts.
template <typename XT>
__global__ void __launch_bounds__(kRouteThreads) k_moe_step_route(RouteArgs a) {
  extern __shared__ __align__(16) float row[];
  __shared__ float red[32];
  __shared__ double part[kMaxStepExperts / kRouteCluster][kRouteThreads / 32], logit[kMaxStepExperts / kRouteCluster];
  __shared__ int chosen[kMaxTop];
  __shared__ float weight[kMaxTop];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = (int)cl.block_rank(), t = (int)(blockIdx.x / kRouteCluster), tid = threadIdx.x, lane = tid & 31,
            warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  for (int i = blockIdx.x * kRouteThreads + tid; i < a.n_tickets; i += gridDim.x * kRouteThreads) a.tickets[i] = 0;
  if (rank == 0 && tid < a.k) a.a_max[t * a.k + tid] = 0u;
  const XT* x = (const XT*)a.x + (int64_t)t * a.stride;
  float s = 0.f;
  for (int i = tid; i < a.H; i += kRouteThreads) {
    const float v = to_f32<XT>(x[i]);
    row[i] = v;
    s = fmaf(v, v, s);
  }
  if (a.norm_w) {
    s = block_sum<kRouteThreads>(s, red);
    const float r = 1.0f / sqrtf(s / (float)a.H + a.eps);
    for (int i = tid; i < a.H; i += kRouteThreads) row[i] = row[i] * r * a.norm_w[i];
  }
  float m = 0.f;
  for (int i = tid; i < a.H; i += kRouteThreads) m = fmaxf(m, fabsf(row[i]));
  m = block_max<kRouteThreads>(m, red);                        // (all of the row is there)
  for (int i = rank * kRouteThreads + tid; i < a.H; i += kRouteCluster * kRouteThreads) a.v[(int64_t)t * a.H + i] = row[i];
  if (rank == 0 && tid == 0) a.v_max[t] = m;
  const int mine = (a.E - rank + kRouteCluster - 1) / kRouteCluster;       // experts rank, rank + 8, ...
#pragma unroll 2
  for (int j = 0; j < mine; ++j) {
    const float4* g = reinterpret_cast<const float4*>(a.gate + (int64_t)(rank + j * kRouteCluster) * a.H);
    double d = 0.;
#pragma unroll 4
    for (int i = tid; i < a.H / 4; i += kRouteThreads) {
      const float4 w = __ldg(g + i), v = *reinterpret_cast<const float4*>(row + 4 * i);
      d = fma((double)v.x, (double)w.x, d);
      d = fma((double)v.y, (double)w.y, d);
      d = fma((double)v.z, (double)w.z, d);
      d = fma((double)v.w, (double)w.w, d);
    }
    d = warp_sum_d(d);
    if (lane == 0) part[j][warp] = d;
  }
  __syncthreads();
  if (tid < mine) {
    double d = 0.;
    for (int w = 0; w < kRouteThreads / 32; ++w) d += part[tid][w];
    logit[tid] = d;
  }
  cl.sync();
  if (rank == 0 && warp == 0) {
    constexpr int EACH = kMaxStepExperts / 32;
    double l[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int e = lane + 32 * i;
      l[i] = e < a.E ? cl.map_shared_rank(logit, e % kRouteCluster)[e / kRouteCluster] : 0.;
    }
    unsigned left = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) left |= (lane + 32 * i < a.E ? 1u : 0u) << i;
    double top = 0., val = 0.;
    int expert = 0;
    for (int j = 0; j < a.k; ++j) {
      double best = -INFINITY;
      int at = 1 << 30;
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const double q = l[i] == l[i] ? l[i] : -INFINITY;             // (NaN: not before any other)
        if ((left >> i & 1) && (at == 1 << 30 || q > best)) {
          best = q;
          at = lane + 32 * i;
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const double q = __shfl_xor_sync(~0u, best, o);
        const int i = __shfl_xor_sync(~0u, at, o);
        if (i != 1 << 30 && (at == 1 << 30 || q > best || (q == best && i < at))) {
          best = q;
          at = i;
        }
      }
      if ((at & 31) == lane) left &= ~(1u << (at >> 5));
      double q = 0.;
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (i == at >> 5) q = l[i];
      q = __shfl_sync(~0u, q, at & 31);                                // (itself, a NaN too)
      if (j == 0) top = best;
      if (lane == j) {
        expert = at;
        val = q;
      }
    }
    if (!(fabs(top) < INFINITY)) top = 0.;
    const float w = lane < a.k ? expf((float)(val - top)) : 0.f;
    const float sum = warp_sum(w) + 1e-12f;
    if (lane < a.k) chosen[lane] = expert;
    __syncwarp();
    if (lane < a.k) {
      int place = 0;
      for (int j = 0; j < a.k; ++j) place += chosen[j] < expert;
      a.top_e[t * a.k + place] = expert;
      a.top_w[t * a.k + place] = w / sum;
    }
  }
  cl.sync();                                                  // rank 0 has read the others' logits
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------
XM_DEV void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
XM_DEV uint32_t pack2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The 256 values of K that a warp holds, of its columns: for each group of 32 the thread's 8 (8 t .. 8 t + 7 of the group,
// t = lane % 4) as pairs (0, 2), (1, 3), (4, 6), (5, 7): the order in which words of 4-bit codes fall apart under masks.
template <int NT>
struct Columns {
  uint32_t b[NT][8][4];
};

// Types whose weights enter with the block's own value, not rounded to fp16 as dequantisation rounds it.
template <int T>
constexpr bool own_value() { return T == T_Q4_K || T == T_Q5_K || T == T_Q6_K || T == T_Q8_0; }

// 256 values of K of sixteen rows, value by value: fp16 weights, or two fp16 each (hi + 2^-11 lo).
template <int T, int NT>
XM_DEV void unit_any(const uint8_t* lo_row, const uint8_t* hi_row, int t, const Columns<NT>& x, float (&acc)[NT][2]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = 0.f;
#pragma unroll 1
  for (int part = 0; part < (own_value<T>() ? 2 : 1); ++part) {
    float c[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t w[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint8_t* p = r ? hi_row : lo_row;
        float v[8];
        if constexpr (QT<T>::QK == 256) QT<T>::decode8(p, 32 * j + 8 * t, v);
        else QT<T>::decode8(p + j * QT<T>::REC, 8 * t, v);
        if (part) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = (v[i] - __half2float(__float2half_rn(v[i]))) * 2048.f;
        }
        w[r][0] = pack2(v[0], v[2]);
        w[r][1] = pack2(v[1], v[3]);
        w[r][2] = pack2(v[4], v[6]);
        w[r][3] = pack2(v[5], v[7]);
      }
      const uint32_t a0[4] = {w[0][0], w[1][0], w[0][1], w[1][1]}, a1[4] = {w[0][2], w[1][2], w[0][3], w[1][3]};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma_f16(c[n], a0, x.b[n][j][0], x.b[n][j][1]);
        mma_f16(c[n], a1, x.b[n][j][2], x.b[n][j][3]);
      }
    }
    const float scale = part ? 0x1p-11f : 1.f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n][0] = fmaf(scale, fmaf(c[n][1], 0x1p-11f, c[n][0]), acc[n][0]);
      acc[n][1] = fmaf(scale, fmaf(c[n][3], 0x1p-11f, c[n][2]), acc[n][1]);
    }
  }
}

template <int T>
constexpr int block_bytes() { return QT<T>::QK == 256 ? QT<T>::REC : 8 * QT<T>::REC; }   // of 256 values

template <int T, int NT, bool UP>
__global__ void __launch_bounds__(kStepThreads, 1) k_moe_step(StepArgs a) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ StepShared sm;
  constexpr int RB = block_bytes<T>(), COLS = 4 * NT;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int stage_bytes = 16 * a.tps * a.pitch;
  uint8_t* ring = dyn;
  float* red = reinterpret_cast<float*>(dyn + a.ring * stage_bytes);       // [ring][worker][lane][2 NT]
  if (UP) grid_dep_wait();
  grid_dep_launch();
  // Which pairs go to which expert, and the segments (an expert and up to COLS of its pairs): from the routing, which is
  // complete before the launch of DOWN can begin (UP waits for it before it lets DOWN start).
  const int P = a.T * a.k;
  if (tid == 0) {
    for (int i = 0; i < a.ring; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.done[i], kWorkers);
    }
    fence_mbar_init();
  }
  for (int e = warp; e < a.E; e += kWorkers + 1) {
    int n = 0;
    for (int i = lane; i < (P + 31) / 32 * 32; i += 32) n += __popc(__ballot_sync(~0u, i < P && __ldcg(a.top_e + i) == e));
    if (lane == 0) sm.cnt[e] = n;
  }
  __syncthreads();
  if (warp == 0) {
    int at = 0, segs = 0;
    for (int e0 = 0; e0 < a.E; e0 += 32) {
      const int e = e0 + lane, n = e < a.E ? sm.cnt[e] : 0, s = (n + COLS - 1) / COLS;
      int pn = n, ps = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(~0u, pn, o), v = __shfl_up_sync(~0u, ps, o);
        if (lane >= o) {
          pn += u;
          ps += v;
        }
      }
      if (e < a.E) sm.off[e] = at + pn - n;
      for (int i = 0; i < s; ++i) {
        const int g = segs + ps - s + i;
        sm.seg_e[g] = (unsigned short)e;
        sm.seg_at[g] = (unsigned short)(at + pn - n + i * COLS);
        sm.seg_n[g] = (unsigned short)min(COLS, n - i * COLS);
      }
      at += __shfl_sync(~0u, pn, 31);
      segs += __shfl_sync(~0u, ps, 31);
    }
    if (lane == 0) sm.n_seg = segs;
  }
  __syncthreads();
  for (int e = warp; e < a.E; e += kWorkers + 1) {
    if (sm.cnt[e] == 0) continue;
    int at = sm.off[e];
    for (int i = lane; i < (P + 31) / 32 * 32; i += 32) {
      const bool is = i < P && __ldcg(a.top_e + i) == e;
      const unsigned b = __ballot_sync(~0u, is);
      if (is) sm.pair[at + __popc(b & ((1u << lane) - 1))] = (unsigned short)i;
      at += __popc(b);
    }
  }
  __syncthreads();
  const int per_seg = a.chunks * a.groups;                     // stages of a segment: (chunk, group of tiles)
  const int64_t total = (int64_t)sm.n_seg * per_seg;
  const int s0 = (int)(total * blockIdx.x / gridDim.x), s1 = (int)(total * (blockIdx.x + 1) / gridDim.x);

  if (warp == kWorkers) {
    // -- copies and results ------------------------------------------------
    const int g = lane >> 2, t = lane & 3;
    auto issue = [&](int s) {
      const int slot = (s - s0) % a.ring, seg = s / per_seg, c = s % per_seg / a.groups, grp = s % a.groups;
      const int e = sm.seg_e[seg], tile0 = grp * a.tps, rows = 16 * min(a.tps, a.tiles - tile0);
      const int len = min(a.kc, a.nsb - c * a.kc) * RB;
      const uint8_t* w1 = (const uint8_t*)a.w1[e];
      const uint8_t* w3 = UP ? (const uint8_t*)a.w3[e] : nullptr;
      uint32_t bytes = 0;
      auto from = [&](int r) {                                 // row r of the stage: its address
        const int tile = tile0 + r / 16, i = r % 16;
        const uint8_t* base = UP && i >= 8 ? w3 : w1;
        const int64_t n = UP ? tile * 8 + i % 8 : tile * 16 + i;
        return base + n * a.row_bytes + (int64_t)c * a.kc * RB;
      };
      auto size = [&](const uint8_t* p) { return (uint32_t)(((uintptr_t)p & 15) + len + 15) & ~15u; };
      for (int r = lane; r < rows; r += 32) bytes += size(from(r));
      bytes = __reduce_add_sync(~0u, bytes);
      if (lane == 0) mbar_arrive_expect_tx(&sm.full[slot], bytes);
      __syncwarp();
      for (int r = lane; r < rows; r += 32) {
        const uint8_t* p = from(r);
        bulk_g2s(ring + slot * stage_bytes + r * a.pitch, (const void*)((uintptr_t)p & ~(uintptr_t)15), size(p), &sm.full[slot]);
      }
    };
    for (int s = s0; s < min(s1, s0 + a.ring); ++s) issue(s);
    if (!UP) grid_dep_wait();
    float most[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) most[n] = 0.f;
    for (int s = s0; s < s1; ++s) {
      const int slot = (s - s0) % a.ring, lap = (s - s0) / a.ring;
      const int seg = s / per_seg, c = s % per_seg / a.groups, grp = s % a.groups;
      const int tile0 = grp * a.tps, tiles = min(a.tps, a.tiles - tile0);
      const int at = sm.seg_at[seg], n_pairs = sm.seg_n[seg], kc = min(a.kc, a.nsb - c * a.kc);
      mbar_wait_bounded(&sm.done[slot], lap & 1);
      for (int i = 0; i < tiles; ++i) {
        float v[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) v[n][0] = v[n][1] = 0.f;
        const float* r = red + ((slot * kWorkers + i * a.kc) * 32 + lane) * 2 * NT;
        for (int w = 0; w < kc; ++w) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float2 q = *reinterpret_cast<const float2*>(r + w * 64 * NT + 2 * n);
            v[n][0] += q.x;
            v[n][1] += q.y;
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (4 * n + t >= n_pairs) continue;
          const int pair = sm.pair[at + 4 * n + t];
          const float scale = ldexpf(1.0f, fp16_row_shift(__ldcg(a.src_max + (UP ? pair / a.k : pair))));
          if (UP) {
            const int f = (tile0 + i) * 8 + g;
            const float gate = v[n][0] * scale, up = v[n][1] * scale;
            if (a.chunks == 1) {
              const float y = xm_act(a.act, gate) * up;
              a.dst[(int64_t)pair * a.N + f] = y;
              most[n] = fmaxf(most[n], fabsf(y));
            } else {
              float* p = a.part + ((int64_t)c * P + pair) * 2 * a.N + f;
              p[0] = gate;
              p[a.N] = up;
            }
          } else {
            float* p = a.dst + ((int64_t)c * P + pair) * a.N + (tile0 + i) * 16 + g;
            p[0] = v[n][0] * scale;
            p[8] = v[n][1] * scale;
          }
        }
      }
      __syncwarp();
      if (s + a.ring < s1) issue(s + a.ring);
      const bool ends = s + 1 == s1 || (s + 1) / per_seg != seg;
      if (UP && a.chunks > 1) {
        // the last chunk's writer of these tiles takes the chunks together
        __threadfence();
        __syncwarp();
        int old = 0;
        if (lane == 0) old = atomicAdd(a.tickets + seg * a.groups + grp, 1);
        old = __shfl_sync(~0u, old, 0);
        if (old == a.chunks - 1) {
          __threadfence();
          for (int i = 0; i < tiles; ++i) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (4 * n + t >= n_pairs) continue;
              const int pair = sm.pair[at + 4 * n + t], f = (tile0 + i) * 8 + g;
              float gate = 0.f, up = 0.f;
              for (int q = 0; q < a.chunks; ++q) {
                const float* p = a.part + ((int64_t)q * P + pair) * 2 * a.N + f;
                gate += __ldcg(p);
                up += __ldcg(p + a.N);
              }
              const float y = xm_act(a.act, gate) * up;
              a.dst[(int64_t)pair * a.N + f] = y;
              most[n] = fmaxf(most[n], fabsf(y));
            }
          }
          __syncwarp();
        }
      }
      if (UP && ends) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float m = most[n];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
          if (g == 0 && 4 * n + t < n_pairs) atomicMax(a.dst_max + sm.pair[at + 4 * n + t], __float_as_uint(m));
          most[n] = 0.f;
        }
      }
      if (!UP) {
        __threadfence();
        __syncwarp();
        int old = 0;
        if (lane == 0) old = atomicAdd(a.tickets + grp, 1);
        old = __shfl_sync(~0u, old, 0);
        if (old == sm.n_seg * a.chunks - 1) {
          __threadfence();
          const int rows = 16 * tiles;
          for (int i = lane; i < rows * a.T; i += 32) {
            const int tok = i / rows, row = tile0 * 16 + i % rows;
            float y = 0.f;
            for (int j = 0; j < a.k; ++j) {
              float q = 0.f;
              for (int ch = 0; ch < a.chunks; ++ch) q += __ldcg(a.dst + ((int64_t)ch * P + tok * a.k + j) * a.N + row);
              y = fmaf(q, __ldcg(a.top_w + tok * a.k + j), y);
            }
            if (a.residual) y += a.residual[tok * a.residual_stride + row];
            a.out[tok * a.out_stride + row] = y;
          }
          __syncwarp();
        }
      }
    }
    return;
  }

  // -- products --------------------------------------------------------------
  if (!UP) grid_dep_wait();
  const int g = lane >> 2, t = lane & 3;
  const int my_tile = warp / a.kc, my_sb = warp % a.kc;
  Columns<NT> x;
  int held = -1;
  for (int s = s0; s < s1; ++s) {
    const int slot = (s - s0) % a.ring, lap = (s - s0) / a.ring;
    const int seg = s / per_seg, c = s % per_seg / a.groups, grp = s % a.groups;
    const bool mine = my_tile < min(a.tps, a.tiles - grp * a.tps) && my_tile < a.tps && c * a.kc + my_sb < a.nsb;
    if (held != s / a.groups) {
      // this segment's activations: column g is token g / 2 of the segment's, hi or lo
      held = s / a.groups;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int col = 4 * n + (g >> 1);
        const bool there = mine && col < sm.seg_n[seg];
        const int pair = there ? sm.pair[sm.seg_at[seg] + col] : 0, row = UP ? pair / a.k : pair;
        const float inv = ldexpf(1.0f, -fp16_row_shift(there ? __ldcg(a.src_max + row) : 0.f));
        const float* p = a.src + (int64_t)row * a.K + (int64_t)(c * a.kc + my_sb) * 256 + 8 * t;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v[8];
          if (there) {
            const float4 u = __ldcg(reinterpret_cast<const float4*>(p + 32 * j)),
                         w = __ldcg(reinterpret_cast<const float4*>(p + 32 * j + 4));
            v[0] = u.x * inv; v[1] = u.y * inv; v[2] = u.z * inv; v[3] = u.w * inv;
            v[4] = w.x * inv; v[5] = w.y * inv; v[6] = w.z * inv; v[7] = w.w * inv;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
          }
          if (g & 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (v[i] - __half2float(__float2half_rn(v[i]))) * 2048.f;
          }
          x.b[n][j][0] = pack2(v[0], v[2]);
          x.b[n][j][1] = pack2(v[1], v[3]);
          x.b[n][j][2] = pack2(v[4], v[6]);
          x.b[n][j][3] = pack2(v[5], v[7]);
        }
      }
    }
    mbar_wait_bounded(&sm.full[slot], lap & 1);
    if (mine) {
      const uint8_t* rows = ring + slot * stage_bytes + my_tile * 16 * a.pitch + my_sb * RB;
      // (a row's bytes begin where they do in 16 bytes of the weight)
      const int tile = grp * a.tps + my_tile;
      auto start = [&](int i) {
        const int64_t n = UP ? tile * 8 + i % 8 : tile * 16 + i;
        return rows + i * a.pitch + (int)((n * a.row_bytes + (int64_t)c * a.kc * RB) & 15);
      };
      float acc[NT][2];
      unit_any<T, NT>(start(g), start(g + 8), t, x, acc);
      float* r = red + ((slot * kWorkers + warp) * 32 + lane) * 2 * NT;
#pragma unroll
      for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(r + 2 * n) = make_float2(acc[n][0], acc[n][1]);
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.done[slot]);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
struct Plan {
  int nsb, chunks, kc, tps, tiles, groups, pitch, ring, smem;
};

// K values a row, `tiles` tiles of sixteen rows, rb bytes of 256 values, NT groups of four columns
Plan plan(int64_t K, int64_t tiles, int rb, int NT) {
  Plan p;
  p.nsb = (int)(K / 256);
  p.chunks = (p.nsb + kWorkers - 1) / kWorkers;
  p.kc = (p.nsb + p.chunks - 1) / p.chunks;
  p.chunks = (p.nsb + p.kc - 1) / p.kc;
  p.tps = kWorkers / p.kc;
  p.tiles = (int)tiles;
  p.groups = (p.tiles + p.tps - 1) / p.tps;
  // rows 32 bytes apart modulo 64: four rows of the words that four lanes read fall on different banks
  p.pitch = (p.kc * rb + 15 + 31) / 32 * 32;
  if (p.pitch % 64 == 0) p.pitch += 32;
  const int stage = 16 * p.tps * p.pitch, red = kWorkers * 32 * 2 * NT * 4;
  p.ring = std::min(kMaxRing, (int)(212 * 1024 / (stage + red)));
  p.smem = p.ring * (stage + red);
  return p;
}

struct Layout {
  int64_t top_e, top_w, v, v_max, a, a_max, part, tickets, up_part, bytes;
  int n_tickets;
};
Layout layout(int64_t T, int64_t H, int64_t F, int64_t k, int rb) {
  Layout l;
  int64_t at = 0;
  auto take = [&](int64_t n) {
    const int64_t o = at;
    at += (n * 4 + 255) / 256 * 256;
    return o;
  };
  const int64_t P = T * k;
  const Plan up = plan(H, F / 8, rb, 1), down = plan(F, H / 16, rb, 1);
  l.top_e = take(P);
  l.top_w = take(P);
  l.v = take(T * H);
  l.v_max = take(T);
  l.a = take(P * F);
  l.a_max = take(P);
  l.part = take((int64_t)down.chunks * P * H);
  l.n_tickets = down.groups + (up.chunks > 1 ? (int)P * up.groups : 0);
  l.tickets = take(l.n_tickets);
  l.up_part = take(up.chunks > 1 ? (int64_t)up.chunks * P * 2 * F : 0);
  l.bytes = at;
  return l;
}

template <typename... KArgs, typename... Args>
cudaError_t step_launch(void (*kernel)(KArgs...), dim3 grid, int threads, int smem, int cluster, cudaStream_t st, Args... args) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
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
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int T, int NT>
cudaError_t step_products(StepArgs up, StepArgs down, int64_t H, int64_t F, cudaStream_t st) {
  const int sms = xm_sm_count();
  auto fill = [](StepArgs& a, const Plan& p) {
    a.nsb = p.nsb;
    a.chunks = p.chunks;
    a.kc = p.kc;
    a.tps = p.tps;
    a.tiles = p.tiles;
    a.groups = p.groups;
    a.pitch = p.pitch;
    a.ring = p.ring;
    a.row_bytes = (int64_t)p.nsb * block_bytes<T>();
  };
  const Plan pu = plan(H, F / 8, block_bytes<T>(), NT), pd = plan(F, H / 16, block_bytes<T>(), NT);
  fill(up, pu);
  fill(down, pd);
  cudaError_t e = step_launch(k_moe_step<T, NT, true>, dim3(sms), kStepThreads, pu.smem, 1, st, up);
  if (e != cudaSuccess) return e;
  return step_launch(k_moe_step<T, NT, false>, dim3(sms), kStepThreads, pd.smem, 1, st, down);
}

}  // namespace

extern "C" {

int64_t xm_moe_step_workspace_size(int64_t T, int64_t H, int64_t F, int E, int k, int qtype) {
  int qk = 0, rec = 0;
  if (T < 1 || T > kMaxTokens || H < 256 || H % 256 || H > kMaxHidden || F < 256 || F % 256 || F > (1 << 20) || E < 1 ||
      E > kMaxStepExperts || k < 1 || k > E || k > kMaxTop || !host_qtype_geometry(qtype, &qk, &rec) || qk < 32)
    return 0;
  return layout(T, H, F, k, 256 / qk * rec).bytes;
}

int xm_moe_step(const void* d_x, int x_dtype, int64_t T, int64_t H, int64_t x_stride, const float* d_norm_w, float eps,
                const float* d_gate, int E, int k, int64_t F, const void* const* d_w1, const void* const* d_w3,
                const void* const* d_w2, int qtype, int activation, const float* d_residual, int64_t residual_stride,
                float* d_out, int64_t out_stride, void* d_workspace, int64_t workspace_bytes, void* stream) {
  if (x_dtype != XM_DT_F32 && x_dtype != XM_DT_F16 && x_dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "moe_step: bad element type %d", x_dtype);
  int qk = 0, rec = 0;
  if (!host_qtype_geometry(qtype, &qk, &rec) || qk < 32)
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: expert weights of type id %d", qtype);
  if (T < 0 || T > kMaxTokens) return xm_set_error(XM_ERR_INVALID, "moe_step: %lld tokens (up to %d)", (long long)T, kMaxTokens);
  if (H < 256 || H % 256 || H > kMaxHidden || F < 256 || F % 256 || F > (1 << 20))
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: experts of %lld -> %lld (multiples of 256; hidden up to %d)",
                        (long long)H, (long long)F, kMaxHidden);
  if (E < 1 || E > kMaxStepExperts || k < 1 || k > E || k > kMaxTop)
    return xm_set_error(XM_ERR_UNSUPPORTED, "moe_step: %d of %d experts (up to %d of up to %d)", k, E, kMaxTop, kMaxStepExperts);
  if (activation < XM_ACT_SILU || activation > XM_ACT_IDENTITY)
    return xm_set_error(XM_ERR_INVALID, "moe_step: unknown activation %d", activation);
  if (x_stride < H || out_stride < H || (d_residual && residual_stride < H))
    return xm_set_error(XM_ERR_INVALID, "moe_step: a row pitch is below %lld values", (long long)H);
  if (T == 0) return XM_OK;
  if (!d_x || !d_gate || !d_w1 || !d_w3 || !d_w2 || !d_out || !d_workspace)
    return xm_set_error(XM_ERR_INVALID, "moe_step: null pointer");
  if (((uintptr_t)d_x & (x_dtype == XM_DT_F32 ? 3 : 1)) || ((uintptr_t)d_gate & 15) || ((uintptr_t)d_workspace & 255) ||
      (((uintptr_t)d_norm_w | (uintptr_t)d_residual | (uintptr_t)d_out) & 3) ||
      (((uintptr_t)d_w1 | (uintptr_t)d_w3 | (uintptr_t)d_w2) & 7))
    return xm_set_error(XM_ERR_INVALID, "moe_step: unaligned pointer");
  const Layout l = layout(T, H, F, k, 256 / qk * rec);
  if (workspace_bytes < l.bytes)
    return xm_set_error(XM_ERR_INVALID, "moe_step: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                        (long long)l.bytes);
  uint8_t* ws = (uint8_t*)d_workspace;
  auto f32 = [&](int64_t o) { return reinterpret_cast<float*>(ws + o); };
  auto i32 = [&](int64_t o) { return reinterpret_cast<int*>(ws + o); };
  cudaStream_t st = (cudaStream_t)stream;
  const RouteArgs r{d_x, x_stride, d_norm_w, d_gate, eps, (int)T, (int)H, E, k, f32(l.v), f32(l.v_max), f32(l.top_w),
                    i32(l.top_e), reinterpret_cast<unsigned*>(ws + l.a_max), i32(l.tickets), l.n_tickets};
  auto route = x_dtype == XM_DT_F32   ? k_moe_step_route<float>
               : x_dtype == XM_DT_F16 ? k_moe_step_route<__half>
                                      : k_moe_step_route<__nv_bfloat16>;
  cudaError_t e = step_launch(route, dim3((unsigned)T * kRouteCluster), kRouteThreads, (int)H * 4, kRouteCluster, st, r);
  if (e == cudaSuccess) {
    StepArgs up = {}, down = {};
    up.w1 = d_w1;
    up.w3 = d_w3;
    up.src = f32(l.v);
    up.src_max = f32(l.v_max);
    up.dst = f32(l.a);
    up.dst_max = reinterpret_cast<unsigned*>(ws + l.a_max);
    up.part = f32(l.up_part);
    const Plan pd = plan(F, H / 16, 256 / qk * rec, 1);
    up.tickets = i32(l.tickets) + pd.groups;
    up.top_e = i32(l.top_e);
    up.top_w = f32(l.top_w);
    up.T = (int)T;
    up.k = k;
    up.E = E;
    up.act = activation;
    up.K = (int)H;
    up.N = (int)F;
    down = up;
    down.w1 = d_w2;
    down.w3 = nullptr;
    down.src = f32(l.a);
    down.src_max = f32(l.a_max);
    down.dst = f32(l.part);
    down.tickets = i32(l.tickets);
    down.K = (int)F;
    down.N = (int)H;
    down.residual = d_residual;
    down.residual_stride = residual_stride;
    down.out = d_out;
    down.out_stride = out_stride;
    dispatch_quant(qtype, [&]<int Q>() {
      e = T <= 4 ? step_products<Q, 1>(up, down, H, F, st) : step_products<Q, 2>(up, down, H, F, st);
    });
  }
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "moe_step launch: %s", cudaGetErrorString(e));
  return xm_check_launch("moe_step");
}

}  // extern "C"
