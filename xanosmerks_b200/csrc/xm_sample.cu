// Sampling one token per row of logits from given random numbers.
//
// Row x, temperature T: weights w_i = exp((x_i - max x) / T).  In descending order of x (equal logits:
// ascending index) the kept tokens are a prefix: the first top_k of them; of those, the ones before
// which less than top_p of the top_k's mass lies; of those, the ones with w >= min_p.  The first of
// them is always kept.  The result is the first token i, in index order, at which the kept mass of
// 0 .. i exceeds u times the kept mass.
//
// Masses are whole numbers: w_i is rounded to 2^-F (F = 44, less for rows of 2^19 logits and more), and sums
// of whole numbers do not depend on their order, so a call gives the same token whatever the launch
// shape.  With 2^17 kept tokens the borders are off by about 1e-11 of the mass.
//
// A cluster of C CTAs per row, each warp a contiguous piece of it; the logits stay in shared memory, so the row is
// read once (RES; rows that do not fit, of more than 294912 fp32 or 589824 16-bit logits, are read again from L2 for
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
// A cut through the descending order (top-k: k tokens above it, top-p: a mass).  Up to kList tokens that hold
// everything that can be kept are gathered by one CTA, sorted, cut and drawn from there:
// * top_k: every thread has the maxima of four groups of its logits from the pass that loads them.  The top_k-th
//   largest of these has top_k tokens at or above it, so the top_k largest tokens lie in its bin of a histogram of the
//   maxima or above (128000 normal logits, top_k 300: some 305 tokens in 2048 bins).
// * top_p: the cut lies in the bin of a histogram of masses in which the mass passes the limit; min_p bounds the
//   bins that count.
// Where more tokens than that lie above, the bin becomes the next interval of a histogram of all tokens until it
// holds at most kList tokens, which are sorted; an interval of one value is cut by index; and the token is drawn by
// a pass over the row.
//
// Weights: 2^y with y = (x - max) log2(e) / T in 64 bits, by a table of 2^(j / 256) and a polynomial of
// degree 3 on the rest (table-driven exponential after Tang, 1989): 2e-13 of the value, less than the
// rounding to a whole multiple of 2^-F.
//
// Temperature alone, top_k 50, top_p 0.9 alone, in a captured graph with L2 flushed: one row of 32000 fp32 logits 14, 21 and
// 41 us (L2 warm 8, 13, 23); 64 rows of 128000 49, 55 and 121 (a cluster of 8 CTAs a row, two CTAs an SM: 1.7 waves).
// Bound: latency.  For few rows of passes over shared memory and three to eight exchanges across a cluster; for many of the
// weights' chains (some 25 instructions a logit, ten of them in 64 bits, at 64 registers with some 170 bytes of spills: issue
// slots 43 %, DRAM 5 %).  With top_p alone the atomic adds to shared memory come on top (about one lane a clock on an SM:
// that is why a bin's mass is two words, of which the upper one takes carries and weights above 2^-12 only, and why top_k
// counts maxima and not logits).
// ---------------------------------------------------------------------------
constexpr int kSampleThreads = 512, kBins = 2048, kList = 512, kTable = 256;
static_assert(kList == kSampleThreads, "the list is sorted with one entry a thread");
typedef unsigned long long u64;

struct alignas(16) SampleSmem {
  unsigned low[kBins], high[kBins];     // a bin's mass (or count, in low)
  u64 list[kList];
  double table[kTable];
  u64 xch[2][8][2];                     // exchange slots: buffer, rank, value
  u64 warp_sum[32], warp_cnt[32];
  u64 red[16][2];                       // four 32-bit values of each warp
  unsigned list_n;
  int found_bin;
  u64 found_before;
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
#pragma unroll 1
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

  // sums (op 0) or maxima (op 1) of four 32-bit values over the cluster, the same in every thread
  XM_DEV void all(unsigned (&v)[4], const int (&op)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = op[i] ? __reduce_max_sync(0xffffffffu, v[i]) : __reduce_add_sync(0xffffffffu, v[i]);
    if (lane == 0) *reinterpret_cast<uint4*>(sm.red[warp]) = make_uint4(v[0], v[1], v[2], v[3]);
    __syncthreads();
    if (warp == 0) {
      uint4 t = make_uint4(0u, 0u, 0u, 0u);
      if (lane < NT / 32) t = *reinterpret_cast<const uint4*>(sm.red[lane]);
      v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = op[i] ? __reduce_max_sync(0xffffffffu, v[i]) : __reduce_add_sync(0xffffffffu, v[i]);
      if (lane < C)
        *reinterpret_cast<uint4*>(cl.map_shared_rank(&sm, lane)->xch[turn][rank]) = make_uint4(v[0], v[1], v[2], v[3]);
    }
    sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0u;
    for (int r = 0; r < C; ++r) {
      const uint4 t = *reinterpret_cast<const uint4*>(sm.xch[turn][r]);
      v[0] = op[0] ? max(v[0], t.x) : v[0] + t.x;
      v[1] = op[1] ? max(v[1], t.y) : v[1] + t.y;
      v[2] = op[2] ? max(v[2], t.z) : v[2] + t.z;
      v[3] = op[3] ? max(v[3], t.w) : v[3] + t.w;
    }
    turn ^= 1;
  }
  // the sum of v over the cluster's threads
  XM_DEV u64 sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sm.warp_sum[warp] = v;
    __syncthreads();
    u64 cta = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) cta += sm.warp_sum[w];
    return over_ranks(cta, C);
  }
  // the sum of v, the same in every thread of a CTA, over the first n ranks
  XM_DEV u64 over_ranks(u64 v, int n) {
    if (C == 1) return n ? v : 0ull;
    if (tid < C) cl.map_shared_rank(&sm, tid)->xch[turn][rank][0] = v;
    sync();
    v = 0ull;
    for (int r = 0; r < n; ++r) v += sm.xch[turn][r][0];
    turn ^= 1;
    return v;
  }
  XM_DEV void sync() {
    if (C > 1) cl.sync(); else __syncthreads();
  }
  // A CTA's shared memory may be accessed by the others of its cluster once it has started: every CTA says so first,
  // and waits for the others in front of the first exchange (the load of the row lies between).
  XM_DEV void started() const {
    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed;");
  }
  XM_DEV void wait_started() const {
    if (C > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
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

  // n entries, one a thread (0 behind the last, all different), in descending order: each goes to the place that the
  // number of the larger ones gives (of 320 entries a third of the time of a bitonic network).
  XM_DEV u64 sorted(u64 v, int n) {
    __syncthreads();
    sm.list[tid] = v;
    __syncthreads();
    int at = 0;
    if (tid < n) {
#pragma unroll 4
      for (int j = 0; j < n; j += 2) {
        const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(sm.list + j);
        at += (int)(t.x > v) + (int)(t.y > v);
      }
    }
    __syncthreads();
    if (tid < n) sm.list[at] = v;
    __syncthreads();
    return tid < n ? sm.list[tid] : 0ull;
  }
  // List of this CTA: cleared (a __syncthreads() has to follow), filled, and rank 0's view of all of them, one entry
  // a thread, behind a sync() that follows the last push and where they are kList at most.
  XM_DEV void clear_list() {
    if (tid == 0) sm.list_n = 0;
  }
  XM_DEV void push(float v, int i) {
    if (*(volatile unsigned*)&sm.list_n > kList) return;          // more than can be used
    const unsigned at = atomicAdd(&sm.list_n, 1u);
    if (at < kList) sm.list[at] = (u64)order_key(v) << 32 | (unsigned)~i;
  }
  XM_DEV u64 pull() {
    u64 e = 0;
    if (rank == 0) {
      unsigned c[8], at = tid;
#pragma unroll
      for (int r = 0; r < 8; ++r) c[r] = r < C ? cl.map_shared_rank(&sm, r)->list_n : 0u;
      int from = -1;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (from < 0) {
          if (at < c[r]) from = r; else at -= c[r];
        }
      if (from >= 0) e = cl.map_shared_rank(&sm, from)->list[at];
    }
    sync();
    return e;
  }

  struct Bins {
    float hi, lo, top, half, scale;
    // a monotone function (to the nearest whole number, by adding 2^23) that takes what is below lo to the last bin;
    // the ends have bins of their own, so a step leaves at least one of them out
    XM_DEV Bins(float h, float l) : hi(h), lo(l) {
      half = hi - lo < INFINITY ? 1.f : 0.5f;
      top = fminf(hi, 3.402823466e38f) * half;
      scale = (kBins - 1) / (top - lo * half);
    }
    XM_DEV int operator()(float v) const {
      const float t = fminf(fmaxf((top - v * half) * scale, 0.f), (float)(kBins - 1)) + 8388608.f;
      return v == hi ? 0 : v <= lo ? kBins - 1 : __float_as_int(t) & (kBins - 1);
    }
  };
  XM_DEV void clear_bins() {
    for (int b = tid; b < kBins; b += NT) sm.low[b] = sm.high[b] = 0u;
    __syncthreads();
  }
  // (the carries out of the lower words are the same in every order of the additions)
  XM_DEV void add_mass(int b, u64 w) {
    if (!w) return;
    const unsigned l = (unsigned)w, old = atomicAdd(&sm.low[b], l), h = (unsigned)(w >> 32) + (old + l < l);
    if (h) atomicAdd(&sm.high[b], h);
  }
  // The bin of the cluster's histograms, behind a sync(), in which the sum that starts at `base` reaches `limit`, -1
  // where none does, and the sum before it.  Each CTA adds up its share of the bins over the cluster.
  XM_DEV void find(u64 base, u64 limit) {
    static_assert(kBins / 4 <= NT, "a thread's bins are one 16-byte load");
    const int share = kBins / C;
    u64 ds[4] = {}, mine = 0;
    if (4 * tid < share) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < C) {
          const SampleSmem* p = cl.map_shared_rank(&sm, r);
          const uint4 t = reinterpret_cast<const uint4*>(p->low + rank * share)[tid];
          const uint4 h = reinterpret_cast<const uint4*>(p->high + rank * share)[tid];
          ds[0] += (u64)h.x << 32 | t.x; ds[1] += (u64)h.y << 32 | t.y;
          ds[2] += (u64)h.z << 32 | t.z; ds[3] += (u64)h.w << 32 | t.w;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) mine += ds[j];
    if (tid == 0) sm.found_bin = -1;
    u64 total, before = scan(mine, sm.warp_sum, total) - mine + base;        // (holds __syncthreads())
    before += over_ranks(total, rank);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (before < limit && before + ds[j] >= limit)
        for (int r = 0; r < C; ++r) {
          SampleSmem* p = cl.map_shared_rank(&sm, r);
          p->found_bin = rank * share + 4 * tid + j;
          p->found_before = before;
        }
      before += ds[j];
    }
    sync();
  }
  // Puts what lies in the bins up to `upto` on the lists and returns their number; the logits of bin b, which hold
  // every one between their extremes, become the next interval.
  template <typename IN>
  XM_DEV u64 collect(const Bins& bin, IN in, int upto, int b, u64& n, float& hi, float& lo) {
    clear_list();
    __syncthreads();
    float h = -INFINITY, g = INFINITY;
    unsigned v[4] = {};
    each([&](float x, int i) {
      if (!(x <= bin.hi && x > -INFINITY) || !in(x, i)) return;
      const int at = bin(x);
      if (at <= upto) {
        ++v[3];
        push(x, i);
      }
      if (at == b && x >= bin.lo) {
        h = fmaxf(h, x);
        g = fminf(g, x);
        ++v[2];
      }
    });
    v[0] = order_key(h);
    v[1] = v[2] ? ~order_key(g) : 0u;
    all(v, {1, 1, 0, 0});
    hi = from_key(v[0]);
    lo = from_key(~v[1]);
    n = v[2];
    return v[3];
  }

  // Cuts the descending order of the logits that in(logit, index) names, between lo and hi, n of them, before which
  // `base` lies: the last kept token's key and index, where `limit` tokens, or a mass of `limit`, lie before the
  // first token left out.
  template <bool MASS, typename IN>
  XM_DEV void select(IN in, u64 n, float hi, float lo, u64 base, u64 limit, uint32_t& tau, int& cut) {
    for (;;) {
      if (n <= kList) {
        clear_list();
        __syncthreads();
        each([&](float v, int i) {
          if (v <= hi && v >= lo && in(v, i)) push(v, i);
        });
        sync();
        u64 e = pull();
        if (rank == 0) {
          e = sorted(e, (int)n);
          const u64 w = !e ? 0ull : MASS ? weight(from_key((uint32_t)(e >> 32))) : 1ull;
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
      clear_bins();
      each([&](float v, int i) {
        if (v <= hi && v >= lo && in(v, i)) {
          if (MASS) add_mass(bin(v), weight(v)); else atomicAdd(&sm.low[bin(v)], 1u);
        }
      });
      sync();
      find(base, limit);
      base = sm.found_before;
      collect(bin, in, -1, sm.found_bin, n, hi, lo);
    }
  }
};

template <typename XT, int NT, bool RES>
__global__ void __launch_bounds__(NT, 2) k_sample(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t sample_smem[];
  SampleSmem& sm = *reinterpret_cast<SampleSmem*>(sample_smem);
  grid_dep_wait();
  grid_dep_launch();
  Sampler<XT, NT, RES> s(a, sm, reinterpret_cast<XT*>(sample_smem + sizeof(SampleSmem)));
  s.started();
  const int b = (int)(blockIdx.x / s.C), tid = threadIdx.x;
  const float T = a.d_temperature ? a.d_temperature[b] : a.temperature;
  const int top_k = a.d_top_k ? a.d_top_k[b] : a.top_k;
  const float top_p = a.d_top_p ? a.d_top_p[b] : a.top_p;
  const float min_p = a.d_min_p ? a.d_min_p[b] : a.min_p, u = a.u[b];
  const bool greedy = !(T > 0.f), cuts = !greedy && ((top_k > 0 && top_k < a.V) || top_p < 1.f);

  if (tid < kTable) sm.table[tid] = exp2((double)tid / kTable);
  float group[4], mn = INFINITY;                                   // maxima of a quarter of this thread's logits each
#pragma unroll
  for (int e = 0; e < 4; ++e) group[e] = -INFINITY;
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
      group[e] = fmaxf(group[e], x);                              // (a NaN loses)
      if (cuts && x > -INFINITY) {
        mn = fminf(mn, x);
        ++real;
      }
    }
  }
  float least = INFINITY, mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    mx = fmaxf(mx, group[e]);
    if (group[e] > -INFINITY) least = fminf(least, group[e]);
  }
  unsigned st[4] = {order_key(mx), real ? ~order_key(mn) : 0u, real, mx > -INFINITY ? ~order_key(least) : 0u};
  s.wait_started();
  s.all(st, {1, 1, 0, 1});
  if (st[0] == 0) {                                               // nothing to choose from (the whole cluster)
    if (s.rank == 0 && tid == 0) {
      a.ids[b] = 0;
      if (a.logp) a.logp[b] = -INFINITY;
    }
    return;
  }
  const u64 n = st[2];
  s.mx = from_key(st[0]);
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
    typedef typename Sampler<XT, NT, RES>::Bins Bins;
    float hi = s.mx, lo = from_key(~st[1]);
    auto every = [](float v, int) { return v > -INFINITY; };
    // the bin that min_p ends in, behind the roundings of its logit and of bin()
    const float below = T * logf(fminf(min_p, 1.f));
    const float v_min = wmin ? s.mx + below - 4e-7f * (fabsf(s.mx) + fabsf(below)) : -INFINITY;
    u64 zt = 0, limit = (u64)top_k, left = n, base = 0, listed = ~0ull;
    bool whole = n <= kList, uncut = false;                       // uncut: min_p leaves out what top_p would
    if (whole) {
      s.clear_list();
      __syncthreads();
      s.each([&](float v, int i) {
        if (v > -INFINITY) s.push(v, i);
      });
      s.sync();
      listed = n;
    } else if (by_count && top_k <= kList) {
      const Bins bin(hi, from_key(~st[3]));
      if (bin.hi > bin.lo) {
        s.clear_bins();
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (group[e] > -INFINITY) atomicAdd(&sm.low[bin(group[e])], 1u);
        s.sync();
        s.find(0, limit);
        float h, l;
        u64 m;
        listed = s.collect(bin, every, sm.found_bin, -1, m, h, l);
        if (sm.found_bin < 0) listed = ~0ull;
      }
    } else if (by_count && !by_mass && v_min >= lo && hi > lo) {
      const Bins bin(hi, lo);
      float h, l;
      u64 m;
      listed = s.collect(bin, every, min(kBins - 1, bin(v_min) + 1), -1, m, h, l);
    } else if (!by_count && hi > lo) {
      const Bins bin(hi, lo);
      const int last = v_min >= lo ? min(kBins - 1, bin(v_min) + 1) : kBins - 1;
      s.clear_bins();
      s.each([&](float v, int) {
        if (!(v > -INFINITY)) return;
        const u64 w = s.weight(v);
        const int at = bin(v);
        zt += w;
        if (at <= last) s.add_mass(at, w);
      });
      zt = s.sum(zt);
      limit = mass_limit(zt);
      s.find(0, limit);
      const int found = sm.found_bin;
      uncut = found < 0;
      base = sm.found_before;
      listed = s.collect(bin, every, uncut ? last : found, found, left, hi, lo);
    }
    if (listed <= kList) {
      // everything that can be kept is on the lists
      const u64 all = s.pull();
      if (s.rank != 0) return;
      const u64 e = s.sorted(all, (int)listed);
      const bool in = e && (!by_count || tid < top_k);
      const float v = from_key((uint32_t)(e >> 32));
      const u64 w = in ? s.weight(v) : 0ull;
      u64 sum, z;
      const u64 incl = s.scan(w, sm.warp_sum, sum);
      // (the mass of the top_k, or of all, where the list may hold less)
      const u64 p = by_mass ? mass_limit(by_count || whole ? sum : zt) : ~0ull;
      const bool keep = in && incl - w < p && w >= wmin;
      // each kept one adds up those of lower index (the bins hold the indices)
      const unsigned id = keep ? ~(unsigned)e : ~0u;
      const u64 wk = keep ? w : 0ull;
      sm.list[tid] = wk;
      sm.low[tid] = id;
      s.scan(wk, sm.warp_cnt, z);
      const u64 tgt = s.target(u, z);
      const int m = __syncthreads_count(keep);                    // (the first m)
      if (keep) {
        u64 at = 0;
#pragma unroll 2
        for (int j = 0; j < m; j += 4) {
          const uint4 t = *reinterpret_cast<const uint4*>(sm.low + j);
          const ulonglong2 w0 = *reinterpret_cast<const ulonglong2*>(sm.list + j);
          const ulonglong2 w1 = *reinterpret_cast<const ulonglong2*>(sm.list + j + 2);
          if (t.x < id) at += w0.x;
          if (t.y < id) at += w0.y;
          if (t.z < id) at += w1.x;
          if (t.w < id) at += w1.y;
        }
        if (at <= tgt && at + wk > tgt) done((int)id, v, z);
      }
      return;
    }
    if (by_count) {
      s.template select<false>(every, left, hi, lo, base, limit, tau, cut);
      cut_any = true;
      if (by_mass) {
        u64 z = 0;
        s.each([&](float v, int i) {
          if (above(v, i)) z += s.weight(v);
        });
        z = s.sum(z);
        uint32_t t;
        int c;
        s.template select<true>(above, limit, s.mx, from_key(tau), 0ull, mass_limit(z), t, c);
        tau = t;
        cut = c;
      }
    } else if (!uncut) {
      if (hi == lo && left == n) limit = mass_limit(n << s.frac);
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
