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
// A cluster of C CTAs per row, each warp a contiguous piece of it; the logits stay in shared memory, so the row is
// read once (RES; rows that do not fit, of more than 300000 fp32 logits, are read again from L2 for each
// pass).  What the CTAs have to tell one another (maxima, totals, histograms) goes through their shared
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
// A cut through the descending order (top-k: k tokens above it, top-p: a mass) is found by a histogram:
// the logits between the largest and the smallest fall into kBins bins by a monotone function, and the
// cut lies in the bin in which the count or the mass passes the limit.  Where no more than kList tokens lie
// in the bins up to it, or up to the one that min_p ends in (128000 normal logits: some 250 in the fullest of 2048
// bins), they are gathered by one CTA, sorted, cut and drawn from there.  Otherwise the bin becomes the
// next interval until it holds at most kList tokens, which are sorted; an interval of one value is cut
// by index; and the token is drawn by a pass over the row.
//
// Weights: 2^y with y = (x - max) log2(e) / T in 64 bits, by a table of 2^(j / 256) and a polynomial of
// degree 3 on the rest (table-driven exponential after Tang, 1989): 2e-13 of the value, less than the
// rounding to a whole multiple of 2^-F.
//
// Bound: latency for few rows (passes over shared memory and three to eight exchanges across a cluster); for many
// the instructions of the weights, some 25 a logit, ten of them in 64 bits.
// ---------------------------------------------------------------------------
constexpr int kSampleThreads = 512, kBins = 2048, kList = 512, kTable = 256;
static_assert(kList == kSampleThreads, "the list is sorted with one entry a thread");
typedef unsigned long long u64;

struct alignas(16) SampleSmem {
  unsigned cnt[kBins], mass[3][kBins];  // a bin's mass as sums of three 15-bit digits (a CTA has up to 2^17 logits)
  u64 list[kList];
  double table[kTable];
  u64 xch[2][8][4];                     // exchange slots: buffer, rank, value
  u64 warp_sum[32], warp_cnt[32];
  u64 red[32][4];
  unsigned list_n;
  int found_bin;
  u64 found_cnt, found_before, found_upto;
  unsigned tau;
  int cut;
};

template <typename XT, int NT, bool RES>
struct Sampler {
  cg::cluster_group cl;
  SampleSmem& sm;
  const SampleArgs& a;
  const XT* row;
  XT* xs;                                   // this warp's logits in shared memory (RES)
  int C, rank, lane, warp, tid, V, first, pieces;   // first: index of this thread's first logit; pieces of 128 a warp
  int turn = 0;
  float mx;
  double c_y, one;
  float c_f;
  int frac;

  XM_DEV Sampler(const SampleArgs& a_, SampleSmem& s, XT* x) : cl(cg::this_cluster()), sm(s), a(a_) {
    C = (int)cl.num_blocks();
    rank = (int)cl.block_rank();
    tid = threadIdx.x;
    lane = tid & 31;
    warp = tid >> 5;
    V = a.V;
    pieces = a.pieces;
    first = (rank * (NT / 32) + warp) * pieces * 128 + lane * 4;
    xs = x + warp * pieces * 128;
    row = (const XT*)a.logits + (int64_t)(blockIdx.x / C) * a.stride;
  }
  // logits i .. i + 3 as they are, what is past the row as -inf
  XM_DEV void load(int i, XT (&v)[4]) const {
    if (a.vec && i + 3 < V) {
      if constexpr (sizeof(XT) == 4) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(row + i);
      else *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(row + i);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < V ? row[i + e] : (XT)(-INFINITY);
    }
  }
  // the four logits at `at` of a warp's pieces, which start at index `from` in the row and at x in shared memory
  XM_DEV void get(const XT* x, int from, int at, float (&v)[4]) const {
    XT t[4];
    if constexpr (RES) {
      if constexpr (sizeof(XT) == 4) *reinterpret_cast<uint4*>(t) = *reinterpret_cast<const uint4*>(x + at);
      else *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(x + at);
    } else {
      load(from + at, t);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32(t[e]);
  }
  // f(logit, index) for every logit of this thread (NaN and -inf among them)
  template <typename F>
  XM_DEV void each(F f) const {
#pragma unroll 2
    for (int j = 0; j < pieces; ++j) {
      float v[4];
      get(xs, first - lane * 4, 128 * j + lane * 4, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) f(v[e], first + 128 * j + e);
    }
  }

  XM_DEV u64 weight(float v) const {
    const float dx = v - mx;                                      // (only to tell weights below 2^-46 and the maximum)
    if (!(dx * c_f > -47.f)) return v == mx ? 1ull << frac : 0ull;
    const double d = (double)v - (double)mx, magic = 6755399441055744.0;      // 1.5 2^52: rounds to a whole number
    const double kd = fma(d, c_y, magic);                         // c_y: kTable log2(e) / T
    const int n = __double2loint(kd);
    const double r = fma(d, c_y, magic - kd);                     // |r| <= 1/2, in units of 1 / kTable
    constexpr double u = 0.6931471805599453 / kTable;
    const double p = fma(fma(fma(r, u * u * u / 6, u * u / 2), r, u), r, 1.0) * sm.table[n & (kTable - 1)];
    const double t = __hiloint2double(__double2hiint(p) + ((frac + (n >> 8)) << 20), __double2loint(p));
    return (u64)__double_as_longlong(t + 4503599627370496.0) & 0xfffffffffffffull;   // + 2^52
  }

  // sums (op 0) or maxima (op 1) of up to 4 values over the cluster, the same in every thread
  template <int N>
  XM_DEV void all(u64 (&v)[N], const int (&op)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const u64 u = __shfl_xor_sync(0xffffffffu, v[i], o);
        v[i] = op[i] ? max(v[i], u) : v[i] + u;
      }
      if (lane == 0) sm.red[warp][i] = v[i];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        u64 u = lane < NT / 32 ? sm.red[lane][i] : 0ull;
#pragma unroll
        for (int o = NT / 64; o > 0; o >>= 1) {
          const u64 t = __shfl_xor_sync(0xffffffffu, u, o);
          u = op[i] ? max(u, t) : u + t;
        }
        u = __shfl_sync(0xffffffffu, u, 0);
        if (lane < C) cl.map_shared_rank(&sm, lane)->xch[turn][rank][i] = u;
      }
    }
    sync();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0ull;
      for (int r = 0; r < C; ++r) {
        const u64 u = sm.xch[turn][r][i];
        v[i] = op[i] ? max(v[i], u) : v[i] + u;
      }
    }
    turn ^= 1;
  }
  XM_DEV void sync() {
    if (C > 1) cl.sync(); else __syncthreads();
  }

  // inclusive sum of v over the CTA's threads; sum: over all of them
  XM_DEV u64 scan(u64 v, u64* per_warp, u64& sum) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 t = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += t;
    }
    __syncthreads();
    if (lane == 31) per_warp[warp] = v;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const u64 t = per_warp[w];
      if (w < warp) v += t;
      sum += t;
    }
    return v;
  }

  // What u asks for of a mass z: the token at which the running mass exceeds it.
  XM_DEV static u64 target(float u, u64 z) {
    const u64 t = u > 0.f ? (u64)fmin((double)u * (double)z, 1.8e19) : 0ull;
    return min(t, z - 1);
  }

  // The first index, in order, at which the running sum of f(logit, index) exceeds tgt (share: u times f's
  // total), and that total if wanted; known to every thread, V where none does.
  template <typename F>
  XM_DEV int locate(F f, u64 tgt, bool share, float u, u64* total) {
    u64 s = 0;
    each([&](float v, int i) { s += f(v, i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sm.warp_sum[warp] = s;
    if (tid == 0) sm.cut = V;
    __syncthreads();
    u64 cta = 0, before = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) cta += sm.warp_sum[w];
    if (tid < C) cl.map_shared_rank(&sm, tid)->xch[turn][rank][0] = cta;
    sync();
    u64 z = 0;
    for (int r = 0; r < C; ++r) {
      const u64 t = sm.xch[turn][r][0];
      if (r < rank) before += t;
      z += t;
    }
    turn ^= 1;
    if (share) tgt = target(u, z);
    if (total) *total = z;
    // the warp whose pieces hold it: all warps of its CTA go through those, four logits a thread at a time
    u64 lo = 0;
    int holder = -1;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const u64 t = sm.warp_sum[w];
      if (before <= tgt && before + t > tgt) {
        holder = w;
        lo = before;
      }
      before += t;
    }
    if (holder >= 0) {
      const int from = (rank * (NT / 32) + holder) * pieces * 128;
      const XT* xh = xs + (holder - warp) * pieces * 128;
      for (int q0 = 0; q0 < pieces * 32; q0 += NT) {
        const int q = q0 + tid, i = from + 4 * q;
        u64 g[4] = {}, c = 0;
        if (q < pieces * 32) {
          float v[4];
          get(xh, from, 4 * q, v);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            g[e] = f(v[e], i + e);
            c += g[e];
          }
        }
        u64 sum;
        u64 at = lo + scan(c, sm.warp_cnt, sum) - c;
        if (at <= tgt && at + c > tgt) {
          int k = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (at <= tgt) k = e;
            at += g[e];
          }
          for (int r = 0; r < C; ++r) cl.map_shared_rank(&sm, r)->cut = i + k;
        }
        lo += sum;
        if (lo > tgt) break;
      }
    }
    sync();
    const int r = sm.cut;
    __syncthreads();
    return r;
  }

  // The CTA's list in descending order (key, then lowest index), one entry a thread: (key, ~index), 0 behind the
  // last.  Strides of a warp go by shuffles, the others through shared memory.
  XM_DEV u64 sorted(u64 v) {
#pragma unroll 1
    for (int k = 2; k <= NT; k <<= 1) {
#pragma unroll 1
      for (int j = k >> 1; j > 0; j >>= 1) {
        u64 o;
        if (j >= 32) {
          __syncthreads();
          sm.list[tid] = v;
          __syncthreads();
          o = sm.list[tid ^ j];
        } else {
          o = __shfl_xor_sync(0xffffffffu, v, j);
        }
        const bool first_half = (tid & j) == 0, down = (tid & k) == 0;      // down: the larger one to the first half
        v = first_half == down ? max(v, o) : min(v, o);
      }
    }
    return v;
  }
  // rank 0's list from what in(logit, index) names; the caller is behind a sync() that follows list_n = 0
  template <typename IN>
  XM_DEV void gather(IN in) {
    SampleSmem* to = cl.map_shared_rank(&sm, 0);
    each([&](float v, int i) {
      if (in(v, i)) to->list[atomicAdd(&to->list_n, 1u)] = (u64)order_key(v) << 32 | (unsigned)~i;
    });
    sync();
  }
  XM_DEV u64 entry() const { return (unsigned)tid < sm.list_n ? sm.list[tid] : 0ull; }

  // Histogram of the logits that in(logit, index) names between lo and hi, by the function of bin(); then the bin in
  // which the count (or the mass) that starts at `base` reaches `limit`, or limit(total) of it.
  struct Bins {
    float hi, lo, top, half, scale;
    // a monotone function (to the nearest whole number, by adding 2^23); the ends have bins of their own, so a
    // step leaves at least one of them out
    XM_DEV Bins(float h, float l) : hi(h), lo(l) {
      half = hi - lo < INFINITY ? 1.f : 0.5f;
      top = hi * half;
      scale = (kBins - 1) / (top - lo * half);
    }
    XM_DEV int operator()(float v) const {
      const float t = fminf(fmaxf((top - v * half) * scale, 0.f), (float)(kBins - 1)) + 8388608.f;
      return v == hi ? 0 : v == lo ? kBins - 1 : __float_as_int(t) & (kBins - 1);
    }
  };
  template <bool MASS, typename IN, typename LIMIT>
  XM_DEV void histogram(const Bins& bin, IN in, u64 base, LIMIT limit_of, int last_bin) {
    for (int b = tid; b < kBins; b += NT) {
      sm.cnt[b] = 0u;
      if (MASS) sm.mass[0][b] = sm.mass[1][b] = sm.mass[2][b] = 0u;
    }
    if (tid == 0) sm.list_n = 0;
    __syncthreads();
    each([&](float v, int i) {
      if (v <= bin.hi && v >= bin.lo && in(v, i)) {
        const int b = bin(v);
        atomicAdd(&sm.cnt[b], 1u);
        if (MASS) {
          const u64 w = weight(v);
          if (w) {
            atomicAdd(&sm.mass[0][b], (unsigned)w & 0x7fffu);
            atomicAdd(&sm.mass[1][b], (unsigned)(w >> 15) & 0x7fffu);
            atomicAdd(&sm.mass[2][b], (unsigned)(w >> 30));
          }
        }
      }
    });
    sync();
    // every CTA sums all bins over the cluster
    constexpr int PER = kBins / NT;
    static_assert(PER == 4, "a thread's bins are one 16-byte load");
    unsigned cs[PER] = {};
    u64 ds[PER] = {}, mine = 0, count = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < C) {
        const SampleSmem* p = cl.map_shared_rank(&sm, r);
        const uint4 t = reinterpret_cast<const uint4*>(p->cnt)[tid];
        cs[0] += t.x; cs[1] += t.y; cs[2] += t.z; cs[3] += t.w;
        if (MASS) {
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            const uint4 m = reinterpret_cast<const uint4*>(p->mass[k])[tid];
            ds[0] += (u64)m.x << 15 * k; ds[1] += (u64)m.y << 15 * k;
            ds[2] += (u64)m.z << 15 * k; ds[3] += (u64)m.w << 15 * k;
          }
        }
      }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (!MASS) ds[j] = cs[j];
      mine += ds[j];
      count += cs[j];
    }
    u64 total, counted;
    u64 before = scan(mine, sm.warp_sum, total) - mine + base, upto = scan(count, sm.warp_cnt, counted) - count;
    const u64 limit = limit_of(total);
    if (tid == 0) sm.found_upto = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      upto += cs[j];
      if (before < limit && before + ds[j] >= limit) {
        sm.found_bin = tid * PER + j;
        sm.found_cnt = cs[j];
        sm.found_before = before;
        sm.found_upto = upto;
      }
      before += ds[j];
    }
    __syncthreads();
    // tokens in the bins up to last_bin, where that comes first
    if (last_bin < sm.found_bin && last_bin / PER == tid) {
      u64 n = upto;
#pragma unroll
      for (int j = PER - 1; j >= 0; --j)
        if (tid * PER + j > last_bin) n -= cs[j];
      sm.found_upto = n;
    }
    __syncthreads();
  }

  // Cuts the descending order of the logits that in(logit, index) names, between lo and hi, n of them, before which
  // `base` lies: the last kept token's key and index, where `limit` tokens, or a mass of `limit`, lie before the
  // first token left out.
  template <bool MASS, typename IN>
  XM_DEV void select(IN in, u64 n, float hi, float lo, u64 base, u64 limit, uint32_t& tau, int& cut) {
    for (;;) {
      if (n <= kList) {
        if (tid == 0) sm.list_n = 0;
        sync();
        gather([&](float v, int i) { return v <= hi && v >= lo && in(v, i); });
        if (rank == 0) {
          const u64 e = sorted(entry()), w = !e ? 0ull : MASS ? weight(from_key((uint32_t)(e >> 32))) : 1ull;
          u64 sum;
          const u64 upto = base + scan(w, sm.warp_sum, sum);
          if (upto - w < limit && upto >= limit)
            for (int r = 0; r < C; ++r) {
              SampleSmem* p = cl.map_shared_rank(&sm, r);
              p->tau = (uint32_t)(e >> 32);
              p->cut = (int)~(unsigned)e;
            }
        }
        sync();
        tau = sm.tau;
        cut = sm.cut;
        __syncthreads();
        return;
      }
      if (hi == lo) {                                             // one value: by index
        const u64 w = MASS ? weight(hi) : 1ull, q = w ? (limit - base + w - 1) / w : n;
        tau = order_key(hi);
        cut = locate([&](float v, int i) { return v == hi && in(v, i) ? 1ull : 0ull; }, q - 1, false, 0.f, nullptr);
        return;
      }
      const Bins bin(hi, lo);
      histogram<MASS>(bin, in, base, [&](u64) { return limit; }, kBins);
      narrow(bin, in, n, hi, lo, base);
    }
  }
  // The found bin's own extremes are the next interval (the bin holds all of the logits between them).
  template <typename IN>
  XM_DEV void narrow(const Bins& bin, IN in, u64& n, float& hi, float& lo, u64& base) {
    const int b = sm.found_bin;
    n = sm.found_cnt;
    base = sm.found_before;
    float h = -INFINITY, g = INFINITY;
    each([&](float v, int i) {
      if (v <= bin.hi && v >= bin.lo && bin(v) == b && in(v, i)) {
        h = fmaxf(h, v);
        g = fminf(g, v);
      }
    });
    u64 v[2] = {order_key(h), g < INFINITY ? (u64)(~order_key(g)) : 0ull};
    all(v, {1, 1});                                               // (and the histograms have been read)
    hi = from_key((uint32_t)v[0]);
    lo = from_key(~(uint32_t)v[1]);
  }
};

template <typename XT, int NT, bool RES>
__global__ void __launch_bounds__(NT, 2) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t sample_smem[];
  SampleSmem& sm = *reinterpret_cast<SampleSmem*>(sample_smem);
  grid_dep_wait();
  grid_dep_launch();
  Sampler<XT, NT, RES> s(a, sm, reinterpret_cast<XT*>(sample_smem + sizeof(SampleSmem)));
  const int b = (int)(blockIdx.x / s.C), tid = threadIdx.x;
  const float T = a.d_temperature ? a.d_temperature[b] : a.temperature;
  const int top_k = a.d_top_k ? a.d_top_k[b] : a.top_k;
  const float top_p = a.d_top_p ? a.d_top_p[b] : a.top_p;
  const float min_p = a.d_min_p ? a.d_min_p[b] : a.min_p, u = a.u[b];
  const bool greedy = !(T > 0.f), cuts = !greedy && ((top_k > 0 && top_k < a.V) || top_p < 1.f);

  if (tid < kTable) sm.table[tid] = exp2((double)tid / kTable);
  float mx = -INFINITY, mn = INFINITY;
  unsigned real = 0;
#pragma unroll 4
  for (int j = 0; j < s.pieces; ++j) {
    XT v[4];
    s.load(s.first + 128 * j, v);
    if constexpr (RES) {
      XT* to = s.xs + 128 * j + s.lane * 4;
      if constexpr (sizeof(XT) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
      else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(v);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = to_f32(v[e]);
      mx = fmaxf(mx, x);                                          // (a NaN loses)
      if (cuts && x > -INFINITY) {
        mn = fminf(mn, x);
        ++real;
      }
    }
  }
  u64 st[3] = {order_key(mx), mn < INFINITY ? (u64)(~order_key(mn)) : 0ull, real};
  s.all(st, {1, 1, 0});
  if (st[0] == 0) {                                               // nothing to choose from (the whole cluster)
    if (s.rank == 0 && tid == 0) {
      a.ids[b] = 0;
      if (a.logp) a.logp[b] = -INFINITY;
    }
    return;
  }
  const u64 n = st[2];
  s.mx = from_key((uint32_t)st[0]);
  s.frac = a.frac_bits;
  s.one = (double)(1ull << a.frac_bits);
  s.c_y = greedy ? 0.0 : 1.4426950408889634 * kTable / (double)T;
  // (a maximum of +inf, or no temperature: every other weight is 0)
  s.c_f = greedy || !(s.mx < INFINITY) ? INFINITY : (float)(1.4426950408889634 / (double)T);
  auto done = [&](int id, float v, u64 z) {
    a.ids[b] = id;
    if (a.logp) {
      const double num = v == s.mx ? 0.0 : ((double)v - (double)s.mx) / (double)T;
      a.logp[b] = (float)(num - log((double)z / s.one));
    }
  };
  if (greedy) {
    const int id = s.locate([&](float v, int) { return v == s.mx ? 1ull : 0ull; }, 0ull, false, 0.f, nullptr);
    if (s.rank == 0 && tid == 0) done(id, s.mx, 1ull << s.frac);
    return;
  }
  const u64 wmin = min_p > 0.f ? (u64)ceil((double)fminf(min_p, 1.f) * s.one) : 0ull;
  const bool by_count = top_k > 0 && (u64)top_k < n, by_mass = top_p < 1.f;
  auto mass_limit = [&](u64 z) { return max(1ull, (u64)ceil((double)fmaxf(top_p, 0.f) * (double)z)); };

  uint32_t tau = 0;                                               // the last kept token
  int cut = a.V;
  bool cut_any = false;
  auto above = [&](float v, int i) {
    const uint32_t key = order_key(v);
    return key > tau || (key == tau && i <= cut);
  };
  if (by_count || by_mass) {
    float hi = s.mx, lo = from_key(~(uint32_t)st[1]);
    auto every = [](float, int) { return true; };
    const typename Sampler<XT, NT, RES>::Bins bin(hi, lo);
    // the bin that min_p ends in, behind the roundings of its logit and of bin()
    const float below = T * logf(fminf(min_p, 1.f));
    const float v_min = wmin ? s.mx + below - 4e-7f * (fabsf(s.mx) + fabsf(below)) : -INFINITY;
    const int last = hi == lo || !(v_min >= lo) ? kBins : min(kBins - 1, bin(v_min) + 1);
    u64 zt = 0, limit = (u64)top_k, left = n, base = 0;
    bool fits = n <= kList;
    if (fits) {
      if (tid == 0) sm.list_n = 0;
      s.sync();
    } else if (hi < lo || hi > lo) {
      if (by_count) s.template histogram<false>(bin, every, 0ull, [&](u64) { return limit; }, last);
      else s.template histogram<true>(bin, every, 0ull, [&](u64 z) { zt = z; return limit = mass_limit(z); }, last);
      fits = sm.found_upto <= kList;
    }
    if (fits && !(by_count && n > kList && last < sm.found_bin && by_mass)) {
      // everything that can be kept is in one CTA's list
      const int upto = n <= kList ? kBins : min(sm.found_bin, last);
      s.gather([&](float v, int) { return v > -INFINITY && (n <= kList || bin(v) <= upto); });
      if (s.rank != 0) return;
      const u64 e = s.sorted(s.entry());
      const bool in = e && (!by_count || tid < top_k);
      const float v = from_key((uint32_t)(e >> 32));
      const u64 w = in ? s.weight(v) : 0ull;
      u64 sum, z;
      const u64 incl = s.scan(w, sm.warp_sum, sum);
      // (the mass of the top_k, or of all, where the list holds less)
      const u64 p = by_mass ? mass_limit(by_count || n <= kList ? sum : zt) : ~0ull;
      const bool keep = in && incl - w < p && w >= wmin;
      // in index order
      u64 f = s.sorted(keep ? (u64)(unsigned)e << 32 | (uint32_t)(e >> 32) : 0ull);       // (~index, key), descending
      const float vf = from_key((uint32_t)f);
      const u64 wf = f ? s.weight(vf) : 0ull;
      const u64 inf = s.scan(wf, sm.warp_sum, z), tgt = s.target(u, z);
      if (inf - wf <= tgt && inf > tgt) done((int)~(unsigned)(f >> 32), vf, z);
      return;
    }
    if (by_count) {
      if (n > kList && hi > lo) s.narrow(bin, every, left, hi, lo, base);
      s.template select<false>(every, left, hi, lo, base, limit, tau, cut);
      cut_any = true;
      if (by_mass) {
        u64 z[1] = {0ull};
        s.each([&](float v, int i) {
          if (above(v, i)) z[0] += s.weight(v);
        });
        s.all(z, {0});
        uint32_t t;
        int c;
        s.template select<true>(above, limit, s.mx, from_key(tau), 0ull, mass_limit(z[0]), t, c);
        tau = t;
        cut = c;
      }
    } else {
      if (hi > lo) s.narrow(bin, every, left, hi, lo, base);
      else limit = mass_limit(n << s.frac);
      s.template select<true>(every, left, hi, lo, base, limit, tau, cut);
      cut_any = true;
    }
  }
  auto kept = [&](float v, int i) {
    if (cut_any && !above(v, i)) return 0ull;
    const u64 w = s.weight(v);
    return w >= wmin ? w : 0ull;
  };
  u64 z = 0;
  const int id = s.locate(kept, 0ull, true, u, &z);
  if (s.rank == 0 && tid == 0) done(id, to_f32(s.row[id]), z);
}

template <typename XT, bool RES>
cudaError_t sample_launch(SampleArgs a, int64_t B, int C, cudaStream_t st) {
  constexpr int NT = kSampleThreads, kMost = 220 * 1024;
  a.pieces = (a.V + C * (NT / 32) * 128 - 1) / (C * (NT / 32) * 128);
  const int smem = (int)sizeof(SampleSmem) + (RES ? a.pieces * NT * 4 * (int)sizeof(XT) : 0);
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
  // the smallest cluster whose CTAs hold 64 KB of a row each, larger while the rows leave half of the SMs without work

  int C = 1;
  while (C < 8 && a.V * (int64_t)sizeof(XT) > 65536 * C) C *= 2;
  while (C < 8 && 2 * B * C <= 148 && a.V > 2048 * C) C *= 2;
  return a.V * (int64_t)sizeof(XT) <= 8 * 147456 ? sample_launch<XT, true>(a, B, C, st) : sample_launch<XT, false>(a, B, 8, st);
}

}  // namespace

extern "C" int xm_sample(const void* d_logits, int dtype, int64_t B, int64_t V, int64_t stride, const float* d_u,
                         float temperature, const float* d_temperature, int top_k, const int* d_top_k, float top_p,
                         const float* d_top_p, float min_p, const float* d_min_p, int* d_ids, float* d_logprob,
                         void* stream) {
  if (dtype != XM_DT_F32 && dtype != XM_DT_F16 && dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "sample: bad element type %d", dtype);
  if (B < 0 || B > INT32_MAX / 8 || V < 1 || V > (1 << 20) || stride < V)
    return xm_set_error(XM_ERR_INVALID, "sample: bad sizes (1 to 2^20 logits a row)");
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
