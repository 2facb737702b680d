// Sampling one token per row of logits from given random numbers.
//
// Row x, temperature T: weights w_i = exp((x_i - max x) / T).  In descending order of x (equal logits:
// ascending index) the kept tokens are a prefix: the first top_k of them; of those, the ones before
// which less than top_p of the top_k's mass lies; of those, the ones with w >= min_p.  The first of
// them is always kept.  The result is the first token i, in index order, at which the kept mass of
// 0 .. i exceeds u times the kept mass.
//
// Masses are whole numbers: w_i is rounded to 2^-F (F = 44, less for more than 2^18 tokens), and sums
// of whole numbers do not depend on their order, so a call gives the same token whatever the launch
// shape.  With 2^17 kept tokens the borders are off by about 1e-11 of the mass.
//
// A cluster of C CTAs per row, each warp a contiguous piece of it; the logits stay in shared memory as fp32, so
// the row is read once (RES; rows that do not fit, of more than 300000 logits, are read again from L2 for
// each pass).  What the CTAs have to tell one another (maxima, totals, histograms) goes through their shared
// memories.
#include <cooperative_groups.h>

#include "xm_gemv_dot.cuh"

namespace cg = cooperative_groups;

namespace {

// order-preserving key of a logit: NaN and -inf below everything else
XM_DEV uint32_t order_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);            // -0 and +0 are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

XM_DEV float from_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct SampleArgs {
  const void* logits;
  int64_t stride;
  int V;
  const float* u;
  float temperature, top_p, min_p;
  int top_k;
  const float *d_temperature, *d_top_p, *d_min_p;
  const int* d_top_k;
  int* ids;
  float* logp;
  int frac_bits;
  bool vec;          // rows allow loads of four logits
  int pieces;        // of 128 logits, of a warp
};

// ---------------------------------------------------------------------------
// A cut through the descending order (top-k: k tokens above it, top-p: a mass) is found by histograms:
// the logits between the largest and the smallest fall into kBins bins by a monotone function, the bin
// in which the count or the mass passes the limit becomes the next interval, until it holds at most
// kList tokens; those are gathered and each one counts what lies before it.  One step is the rule
// (128000 normal logits: some 250 in the fullest of 2048 bins); an interval of one value is cut by index.
//
// Weights: 2^y with y = (x - max) log2(e) / T in 64 bits, by a table of 2^(j / 64) and a polynomial of
// degree 4 on the rest (table-driven exponential after Tang, 1989): 1e-13 of the value, less than the
// rounding to a whole multiple of 2^-F.
//
// Bound: latency for few rows (about seven exchanges across a cluster, some 1 us each); for many the 64-bit
// arithmetic of the weights, ten operations a logit at 64 a clock and SM, about the time that reading the
// logits takes.
// ---------------------------------------------------------------------------
constexpr int kSampleThreads = 512, kBins = 2048, kList = 1024;

struct alignas(16) SampleSmem {
  unsigned long long mass[kBins];
  unsigned cnt[kBins];
  unsigned key[kList], idx[kList];
  unsigned long long w[kList];
  double table[64];
  unsigned long long xch[2][8][4];      // exchange slots: buffer, rank, value
  unsigned long long warp_sum[32];
  unsigned long long red[32][4];
  unsigned list_n;
  int found_bin;
  unsigned long long found_cnt, found_mass;
  unsigned tau;
  int cut;
};

template <typename XT, int NT, bool RES>
struct Sampler {
  cg::cluster_group cl;
  SampleSmem& sm;
  const SampleArgs& a;
  const XT* row;
  float* xs;                                // this thread's logits in shared memory (RES): four at 128 j
  int C, rank, lane, warp, tid, V, first, pieces;   // first: index of this thread's first logit; pieces of 128 a warp
  int turn = 0;
  float mx;
  double c_y, one;
  int frac;
  bool greedy;

  XM_DEV Sampler(const SampleArgs& a_, SampleSmem& s, float* x) : cl(cg::this_cluster()), sm(s), a(a_) {
    C = (int)cl.num_blocks();
    rank = (int)cl.block_rank();
    tid = threadIdx.x;
    lane = tid & 31;
    warp = tid >> 5;
    V = a.V;
    pieces = a.pieces;
    first = (rank * (NT / 32) + warp) * pieces * 128 + lane * 4;
    xs = x + warp * pieces * 128 + lane * 4;
    row = (const XT*)a.logits + (int64_t)(blockIdx.x / C) * a.stride;
  }
  // logits i .. i + 3, NaN and what is past the row as -inf, -0 as 0
  XM_DEV void load(int i, float (&v)[4]) const {
    if (a.vec && i + 3 < V) {
      ld4f<XT>(row + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < V ? to_f32(row[i + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = v[e] > -INFINITY ? v[e] + 0.0f : -INFINITY;
  }
  XM_DEV void get(int j, float (&v)[4]) const {
    if constexpr (RES) {
      const float4 t = *reinterpret_cast<const float4*>(xs + 128 * j);
      v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else {
      load(first + 128 * j, v);
    }
  }
  // f(logit, index) for every logit of this thread that counts
  template <typename F>
  XM_DEV void each(F f) const {
#pragma unroll 1
    for (int j = 0; j < pieces; ++j) {
      float v[4];
      get(j, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (v[e] > -INFINITY) f(v[e], first + 128 * j + e);
    }
  }

  XM_DEV unsigned long long weight(float v) const {
    if (v == mx) return 1ull << frac;
    if (greedy || !(mx < INFINITY)) return 0ull;
    const double y = ((double)v - (double)mx) * c_y;
    if (!(y > -46.0)) return 0ull;
    const double magic = 6755399441055744.0;                      // 1.5 2^52: rounds to a whole number
    const double kd = fma(y, 64.0, magic);
    const int n = __double2loint(kd);
    const double z = fma(kd - magic, -0.015625, y) * 0.6931471805599453;
    const double p = fma(z, fma(z, fma(z, fma(z, 1.0 / 24, 1.0 / 6), 0.5), 1.0), 1.0) * sm.table[n & 63];
    const double t = __hiloint2double(__double2hiint(p) + ((frac + (n >> 6)) << 20), __double2loint(p));
    return (unsigned long long)__double_as_longlong(t + 4503599627370496.0) & 0xfffffffffffffull;   // + 2^52
  }

  // sums (or maxima) of up to 4 values over the cluster, the same in every thread; op 0: sum, 1: max
  template <int N>
  XM_DEV void all(unsigned long long (&v)[N], const int (&op)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long u = __shfl_xor_sync(0xffffffffu, v[i], o);
        v[i] = op[i] ? max(v[i], u) : v[i] + u;
      }
      if (lane == 0) sm.red[warp][i] = v[i];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        unsigned long long u = lane < NT / 32 ? sm.red[lane][i] : 0ull;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long t = __shfl_xor_sync(0xffffffffu, u, o);
          u = op[i] ? max(u, t) : u + t;
        }
        if (lane < C) cl.map_shared_rank(&sm, lane)->xch[turn][rank][i] = u;
      }
    }
    cl.sync();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0ull;
      for (int r = 0; r < C; ++r) {
        const unsigned long long u = sm.xch[turn][r][i];
        v[i] = op[i] ? max(v[i], u) : v[i] + u;
      }
    }
    turn ^= 1;
  }

  // The first index, in order, at which the running sum of f(logit, index) exceeds tgt (share: u times f's total),
  // and that total if wanted; known to every thread, V where none does.
  template <typename F>
  XM_DEV int locate(F f, unsigned long long tgt_or_share, bool share, float u, unsigned long long* total) {
    unsigned long long s = 0;
    each([&](float v, int i) { s += f(v, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sm.warp_sum[warp] = s;
    if (tid == 0) sm.cut = V;
    __syncthreads();
    unsigned long long cta = 0, before = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const unsigned long long t = sm.warp_sum[w];
      if (w < warp) before += t;
      cta += t;
    }
    if (tid < C) cl.map_shared_rank(&sm, tid)->xch[turn][rank][0] = cta;
    cl.sync();
    unsigned long long z = 0;
    for (int r = 0; r < C; ++r) {
      const unsigned long long t = sm.xch[turn][r][0];
      if (r < rank) before += t;
      z += t;
    }
    turn ^= 1;
    unsigned long long tgt = tgt_or_share;
    if (share) {
      tgt = u > 0.f ? (unsigned long long)fmin((double)u * (double)z, 1.8e19) : 0ull;
      tgt = min(tgt, z - 1);
    }
    if (total) *total = z;
    if (before <= tgt && before + s > tgt) {                      // this warp holds it
#pragma unroll 1
      for (int j = 0; j < pieces && before <= tgt; ++j) {
        float v[4];
        get(j, v);
        unsigned long long q[4], c = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          q[e] = v[e] > -INFINITY ? f(v[e], first + 128 * j + e) : 0ull;
          c += q[e];
        }
        unsigned long long up = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned long long t = __shfl_up_sync(0xffffffffu, up, o);
          if (lane >= o) up += t;
        }
        unsigned long long lo = before + up - c;
        if (lo <= tgt && before + up > tgt) {
          int at = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (lo <= tgt) at = e;
            lo += q[e];
          }
          for (int r = 0; r < C; ++r) cl.map_shared_rank(&sm, r)->cut = first + 128 * j + at;
        }
        before += __shfl_sync(0xffffffffu, up, 31);
      }
    }
    cl.sync();
    const int r = sm.cut;
    __syncthreads();
    return r;
  }

  // Cuts the descending order of the logits that `in(logit, index)` names (n of them over the cluster, the largest hi,
  // the smallest lo) where `limit` tokens, or a mass of `limit`, lie before the first token left out: the
  // last kept token's key and index.
  template <bool MASS, typename IN>
  XM_DEV void select(IN in, unsigned long long n, float hi, float lo, unsigned long long limit, uint32_t& tau, int& cut) {
    unsigned long long base = 0;
    for (;;) {
      if (n <= kList) {
        if (tid == 0) sm.list_n = 0;
        cl.sync();
        SampleSmem* to = cl.map_shared_rank(&sm, 0);
        each([&](float v, int i) {
          if (v <= hi && v >= lo && in(v, i)) {
            const unsigned at = atomicAdd(&to->list_n, 1u);
            to->key[at] = order_key(v);
            to->idx[at] = (unsigned)i;
            if (MASS) to->w[at] = weight(v);
          }
        });
        cl.sync();
        if (rank == 0) {
          const unsigned m = sm.list_n;
          for (unsigned i = tid; i < m; i += NT) {
            const unsigned key = sm.key[i], idx = sm.idx[i];
            unsigned long long before = base;
            for (unsigned j = 0; j < m; ++j) {
              const unsigned kj = sm.key[j];
              if (kj > key || (kj == key && sm.idx[j] < idx)) before += MASS ? sm.w[j] : 1ull;
            }
            // the last kept one: it is kept, and what follows it is not (or there is none)
            const unsigned long long mine = MASS ? sm.w[i] : 1ull;
            if (before < limit && (before + mine >= limit)) {
              for (int r = 0; r < C; ++r) {
                SampleSmem* p = cl.map_shared_rank(&sm, r);
                p->tau = key;
                p->cut = (int)idx;
              }
            }
          }
        }
        cl.sync();
        tau = sm.tau;
        cut = sm.cut;
        __syncthreads();
        return;
      }
      if (hi == lo) {                                             // one value: by index
        const unsigned long long w = MASS ? weight(hi) : 1ull, q = w ? (limit - base + w - 1) / w : n;
        tau = order_key(hi);
        cut = locate([&](float v, int i) { return v == hi && in(v, i) ? 1ull : 0ull; }, q - 1, false, 0.f, nullptr);
        return;
      }
      const float half = hi - lo < INFINITY ? 1.f : 0.5f, scale = (kBins - 1) / (hi * half - lo * half);
      auto bin = [&](float v) { return max(0, min(kBins - 1, (int)((hi * half - v * half) * scale))); };
      for (int b = tid; b < kBins; b += NT) {
        sm.cnt[b] = 0u;
        if (MASS) sm.mass[b] = 0ull;
      }
      __syncthreads();
      each([&](float v, int i) {
        if (v <= hi && v >= lo && in(v, i)) {
          const int b = bin(v);
          atomicAdd(&sm.cnt[b], 1u);
          if (MASS) {
            const unsigned long long w = weight(v);
            if (w) atomicAdd(&sm.mass[b], w);
          }
        }
      });
      cl.sync();
      // every CTA sums all bins (the copies lie in the cluster's shared memories) and finds the one
      constexpr int PER = kBins / NT;
      unsigned long long cb[PER], mb[PER], mine = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        cb[j] = mb[j] = 0ull;
        for (int r = 0; r < C; ++r) {
          const SampleSmem* p = cl.map_shared_rank(&sm, r);
          cb[j] += p->cnt[tid * PER + j];
          if (MASS) mb[j] += p->mass[tid * PER + j];
        }
        mine += MASS ? mb[j] : cb[j];
      }
      unsigned long long up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += t;
      }
      if (lane == 31) sm.warp_sum[warp] = up;
      __syncthreads();
      unsigned long long before = base + up - mine;
      for (int w = 0; w < warp; ++w) before += sm.warp_sum[w];
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const unsigned long long v = MASS ? mb[j] : cb[j];
        if (before < limit && before + v >= limit) {
          sm.found_bin = tid * PER + j;
          sm.found_cnt = cb[j];
          sm.found_mass = before;
        }
        before += v;
      }
      __syncthreads();
      const int b = sm.found_bin;
      n = sm.found_cnt;
      base = sm.found_mass;
      // the bin's own extremes are the next interval (a bin holds all of the logits between them)
      float h = -INFINITY, g = INFINITY;
      each([&](float v, int i) {
        if (v <= hi && v >= lo && bin(v) == b && in(v, i)) {
          h = fmaxf(h, v);
          g = fminf(g, v);
        }
      });
      unsigned long long v[2] = {order_key(h), g < INFINITY ? (unsigned long long)(~order_key(g)) : 0ull};
      all(v, {1, 1});                                             // (and the histograms have been read)
      hi = from_key((uint32_t)v[0]);
      lo = from_key(~(uint32_t)v[1]);
    }
  }
};

template <typename XT, int NT, bool RES>
__global__ void __launch_bounds__(NT, 2) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t sample_smem[];
  SampleSmem& sm = *reinterpret_cast<SampleSmem*>(sample_smem);
  grid_dep_wait();
  grid_dep_launch();
  Sampler<XT, NT, RES> s(a, sm, reinterpret_cast<float*>(sample_smem + sizeof(SampleSmem)));
  const int b = (int)(blockIdx.x / s.C), V = a.V;
  float mx = -INFINITY, mn = INFINITY;
  unsigned real = 0;
#pragma unroll 4
  for (int j = 0; j < s.pieces; ++j) {
    float v[4];
    s.load(s.first + 128 * j, v);
    if constexpr (RES) *reinterpret_cast<float4*>(s.xs + 128 * j) = make_float4(v[0], v[1], v[2], v[3]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (v[e] > -INFINITY) {
        mx = fmaxf(mx, v[e]);
        mn = fminf(mn, v[e]);
        ++real;
      }
  }
  if (threadIdx.x < 64) sm.table[threadIdx.x] = exp2((double)threadIdx.x * 0.015625);
  unsigned long long v[3] = {order_key(mx), mn < INFINITY ? (unsigned long long)(~order_key(mn)) : 0ull, real};
  s.all(v, {1, 1, 0});
  if (v[2] == 0) {                                                // nothing to choose from (the whole cluster)
    if (s.rank == 0 && threadIdx.x == 0) {
      a.ids[b] = 0;
      if (a.logp) a.logp[b] = -INFINITY;
    }
    return;
  }
  const unsigned long long n = v[2];
  s.mx = from_key((uint32_t)v[0]);
  const float lowest = from_key(~(uint32_t)v[1]);
  const float T = a.d_temperature ? a.d_temperature[b] : a.temperature;
  const int top_k = a.d_top_k ? a.d_top_k[b] : a.top_k;
  const float top_p = a.d_top_p ? a.d_top_p[b] : a.top_p;
  const float min_p = a.d_min_p ? a.d_min_p[b] : a.min_p;
  s.greedy = !(T > 0.f);
  s.frac = a.frac_bits;
  s.one = (double)(1ull << a.frac_bits);
  s.c_y = s.greedy ? 0.0 : 1.4426950408889634 / (double)T;

  uint32_t tau = 1u;                                              // key 0 is no token
  int cut = V;
  unsigned long long left = n;                                    // tokens that are kept
  auto above = [&](float v, int i) {
    const uint32_t key = order_key(v);
    return key > tau || (key == tau && i <= cut);
  };
  const unsigned long long k = s.greedy ? 1ull : top_k > 0 ? (unsigned long long)top_k : n;
  if (k < n) {
    uint32_t t;
    int c;
    s.template select<false>([](float, int) { return true; }, n, s.mx, lowest, k, t, c);
    tau = t;
    cut = c;
    left = k;
  }
  if (top_p < 1.f && !s.greedy) {
    unsigned long long z[1] = {0ull};
    s.each([&](float v, int i) {
      if (above(v, i)) z[0] += s.weight(v);
    });
    s.all(z, {0});
    const unsigned long long p = max(1ull, (unsigned long long)ceil((double)fmaxf(top_p, 0.f) * (double)z[0]));
    uint32_t t;
    int c;
    s.template select<true>(above, left, s.mx, left < n ? from_key(tau) : lowest, p, t, c);
    tau = t;
    cut = c;
  }
  const unsigned long long wmin = min_p > 0.f ? (unsigned long long)ceil((double)fminf(min_p, 1.f) * s.one) : 0ull;
  auto kept = [&](float v, int i) {
    if (!above(v, i)) return 0ull;
    const unsigned long long w = s.weight(v);
    return w >= wmin ? w : 0ull;
  };
  unsigned long long z = 0;
  const int id = s.locate(kept, 0ull, true, a.u[b], &z);
  if (s.rank == 0 && threadIdx.x == 0) {
    a.ids[b] = id;
    if (a.logp) {
      const float v = to_f32(s.row[id]);
      const double num = v == s.mx ? 0.0 : ((double)v - (double)s.mx) * (s.greedy ? 0.0 : 1.0 / (double)T);
      a.logp[b] = (float)(num - log((double)z / s.one));
    }
  }
}

template <typename XT, bool RES>
cudaError_t sample_launch(SampleArgs a, int64_t B, int C, cudaStream_t st) {
  constexpr int NT = kSampleThreads, kMost = 220 * 1024;
  a.pieces = (a.V + C * (NT / 32) * 128 - 1) / (C * (NT / 32) * 128);
  const int smem = (int)sizeof(SampleSmem) + (RES ? a.pieces * NT * 16 : 0);
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k_sample<XT, NT, RES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, k_sample<XT, NT, RES>, a);
}

template <typename XT>
cudaError_t sample_typed(const SampleArgs& a, int64_t B, cudaStream_t st) {
  // the smallest cluster whose CTAs hold 16384 logits each, larger while the rows leave half of the SMs without work
  int C = 1;
  while (C < 8 && a.V > 16384 * C) C *= 2;
  while (C < 8 && 2 * B * C <= 148 && a.V > 2048 * C) C *= 2;
  return a.V <= 8 * 36864 ? sample_launch<XT, true>(a, B, C, st) : sample_launch<XT, false>(a, B, 8, st);
}

}  // namespace

extern "C" int xm_sample(const void* d_logits, int dtype, int64_t B, int64_t V, int64_t stride, const float* d_u,
                         float temperature, const float* d_temperature, int top_k, const int* d_top_k, float top_p,
                         const float* d_top_p, float min_p, const float* d_min_p, int* d_ids, float* d_logprob,
                         void* stream) {
  if (dtype != XM_DT_F32 && dtype != XM_DT_F16 && dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "sample: bad element type %d", dtype);
  if (B < 0 || B > INT32_MAX / 8 || V < 1 || V > (1 << 30) || stride < V)
    return xm_set_error(XM_ERR_INVALID, "sample: bad sizes");
  if (B == 0) return XM_OK;
  if (!d_logits || !d_u || !d_ids) return xm_set_error(XM_ERR_INVALID, "sample: null pointer");
  if (((uintptr_t)d_logits & (dtype == XM_DT_F32 ? 3 : 1)) || (((uintptr_t)d_u | (uintptr_t)d_temperature |
      (uintptr_t)d_top_k | (uintptr_t)d_top_p | (uintptr_t)d_min_p | (uintptr_t)d_ids | (uintptr_t)d_logprob) & 3))
    return xm_set_error(XM_ERR_INVALID, "sample: unaligned pointer");
  int frac = 62;
  while ((V >> (62 - frac)) > 1 || frac > 44) --frac;      // V 2^frac stays below 2^63
  SampleArgs a{d_logits, stride, (int)V, d_u, temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p,
               d_top_k, d_ids, d_logprob, frac,
               stride % 4 == 0 && ((uintptr_t)d_logits & (dtype == XM_DT_F32 ? 15 : 7)) == 0, 0};
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == XM_DT_F32   ? sample_typed<float>(a, B, st)
                        : dtype == XM_DT_F16 ? sample_typed<__half>(a, B, st)
                                             : sample_typed<__nv_bfloat16>(a, B, st);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
  return xm_check_launch("sample");
}
