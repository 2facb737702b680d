// Log-probability and rank of a given token, entropy, and the largest alternatives of each row of logits, in one pass.
//
// Row x, temperature T, c = log2(e) / T, M its largest logit: w_i = 2^(c (x_i - M)), S and E the sums of w and w c (x - M) over
// all tokens but one of logit M, whose 1 and 0 would take the others' digits with them;
//   logprob_i = ln 2 c (x_i - M) - ln(1 + S),   entropy = ln(1 + S) - ln 2 E / (1 + S):
// no term has another sign, so both are good to some 2^-17 of themselves, next to 0 too.
//   rank = how many tokens have a larger logit, or the same one at a lower index.
//
// M is known at the end only.  Until then weights are relative to r, the largest logit that a CTA sees first (rounds of nothing
// but -inf and NaN are passed over), and vectors with a logit at or above the largest one seen (r, raised whenever twice as much
// has been seen: a few vectors of 16000) stay out of the sums.  Their logits are taken at the end, a thread each, and all but
// one of M join; sums on other references meet by the difference of those, in 64 bits.  Where a weight reaches 2^100, a logit is +inf, or too many
// vectors are left out (equal or rising logits throughout), the CTA takes its part of the row again with its own maximum.  A
// weight's exponent is held above -200, which also gives -inf and NaN logits the weight 0 (and 0 in E).
//
// Alternatives: every warp knows the j-th largest of its lanes' maxima so far; the least of these over the warps, j = ceil(top
// / warps), has at least `top` logits at or above it.  Only vectors with such logits go to a list, and the threshold is raised
// whenever twice as much has been seen (a round's logits are spread over the whole part), so that a few hundred of 128000
// pass.  While some warp has seen fewer than j logits above -inf, all such logits pass.  A list that runs over (equal or rising
// logits throughout, or a mask that leaves thousands of tokens, but none to some warp) sends the CTA to the slow way: one pass a
// place.
//
// C CTAs (a cluster) share a row where rows are few or long.  Bound: HBM and issue for many rows (each logit is read once; some
// eight instructions a logit, sums and exponents two at a time, ranks and maxima of 16-bit logits too), latency for few.
//
// Measured, cold: 2048 rows of 32000 fp32 logits 53 to 57 us (4.6 to 4.9 TB/s); 2000 of 128001 fp16 with 8 alternatives 135 to 142 us
// (3.6 to 3.8 TB/s); 64 of 128000 bf16 with 20, 19.6 us, and one of 32000, 9.2 us, in a captured graph.  (With the largest logit in the sums, and
// entropies below 1e-4 good to three digits or none: 54 to 56, 129, 18.6 and 8.5.)
#include <cooperative_groups.h>

#include "xm_gemv_dot.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kUnroll = 4, kListCap = 2048, kHighMax = 32, kTopMax = 64, kClusterMax = 8;
typedef unsigned long long u64;

struct LogpArgs {
  const void* logits;
  int64_t stride;
  int V, top;
  const void* tokens;
  bool wide_tokens;
  float temperature;
  const float* d_temperature;
  float *logprob, *entropy, *top_logp;
  int *rank, *top_ids;
};

struct Sums {
  float S, E;
  float peak;                              // the largest logit, in neither sum; -inf: none
};

struct alignas(16) LogpSmem {
  u64 list[kListCap];
  int vectors[kListCap];                   // those with a logit for the list
  u64 best[kTopMax];                       // this CTA's largest, in order; 0: none
  u64 merge[kClusterMax * kTopMax];
  float red[kWarps][4];
  u64 red64[kWarps];
  int n, left;
  // vectors left out of the sums, with their places in the row; the order of these
  int n_high;
  uint4 high[kHighMax];
  int high_at[kHighMax], high_order[kHighMax];
  float2 sums[kThreads];                   // each thread's S and E of earlier rounds (few additions in a chain)
  // what the cluster's first CTA reads of each
  Sums part[kWarps];                       // each warp's
  double r;                                // c x reference (log2)
  int above;
  // the row's
  double most, lse;                        // c M, ln(1 + S)
  bool inf;
  int rank;
};

// order-preserving key of a logit: NaN and -inf below everything else
XM_DEV uint32_t logit_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
XM_DEV float key_logit(uint32_t k) {
  return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
XM_DEV u64 entry(float x, int i) { return (u64)logit_key(x) << 32 | (uint32_t)~i; }

XM_DEV float exp2_fast(float t) {
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return e;
}
// two fp32 operations in one instruction
XM_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 z, x, y, z;\n mov.b64 {%0, %1}, z;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
XM_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;\n}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <typename T> XM_DEV T from_f32(float v);
template <> XM_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> XM_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// the next larger number (of +inf: NaN, which compares as nothing does)
XM_DEV float above(float x) {
  if (x == 0.f) return __uint_as_float(1u);
  return __uint_as_float(x > 0.f ? __float_as_uint(x) + 1 : __float_as_uint(x) - 1);
}

template <typename XT>
struct Part {
  static constexpr int VE = 16 / (int)sizeof(XT);   // logits a vector
  const XT* row;                           // logit 0
  const XT* base;                          // the 16-byte boundary at or before it
  int mis, V, v0, nv;                      // logits between them; this CTA's first vector and their number

  XM_DEV bool inner(int v) const { return v * VE >= mis && (v + 1) * VE - mis <= V; }
  XM_DEV int index(int v) const { return v * VE - mis; }
  XM_DEV uint4 raw(int v) const {
    // (read once: L1 keeps nothing)
    return ldg_stream_v4(base + (int64_t)v * VE);
  }
  // the logits of an edge vector; NaN outside of the row
  XM_DEV uint4 edge(int v) const {
    XT t[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      const int at = index(v) + i;
      if (at >= 0 && at < V) t[i] = row[at];
      else if constexpr (sizeof(XT) == 4) reinterpret_cast<uint32_t*>(t)[i] = 0x7fffffffu;
      else reinterpret_cast<uint16_t*>(t)[i] = 0x7fffu;
    }
    uint4 r;
    memcpy(&r, t, 16);
    return r;
  }
  XM_DEV uint4 load(int v) const { return inner(v) ? raw(v) : edge(v); }
  XM_DEV static void values(const uint4& u, float (&x)[VE]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(XT) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else {
        XT two[2];
        memcpy(two, &w[i], 4);
        x[2 * i] = to_f32<XT>(two[0]);
        x[2 * i + 1] = to_f32<XT>(two[1]);
      }
    }
  }
  // f(logit, index) for each logit of this CTA's part
  template <typename F>
  XM_DEV void each(F f) const {
    for (int v = v0 + (int)threadIdx.x; v < v0 + nv; v += kThreads) {
      float x[VE];
      values(load(v), x);
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (index(v) + i >= 0 && index(v) + i < V) f(x[i], index(v) + i);
    }
  }
};

// The j-th largest of the warp's keys (0 if there are fewer).
XM_DEV uint32_t warp_kth(uint32_t key, int j) {
  uint32_t m = 0;
  for (int i = 0; i < j; ++i) {
    m = __reduce_max_sync(~0u, key);
    const unsigned at = __ballot_sync(~0u, key == m);
    if ((int)(threadIdx.x & 31) == __ffs(at) - 1) key = 0;
  }
  return m;
}

// What is seen so far: the block's largest key, and one that at least `top` of its threads have a maximum at or above
// (0: there is none; top = 0: not asked).
struct Seen {
  uint32_t most, kth;
};
// (which: 0 and 1 by turns, or a barrier lies between two calls)
XM_DEV Seen block_seen(uint32_t key, int top, int which, LogpSmem& sm) {
  const uint32_t m = __reduce_max_sync(~0u, key), k = top ? warp_kth(key, (top + kWarps - 1) / kWarps) : 0u;
  if ((threadIdx.x & 31) == 0) {
    sm.red[threadIdx.x >> 5][2 * which] = __uint_as_float(m);
    sm.red[threadIdx.x >> 5][2 * which + 1] = __uint_as_float(k);
  }
  __syncthreads();
  Seen s = {0u, ~0u};
  for (int w = 0; w < kWarps; ++w) {
    s.most = max(s.most, __float_as_uint(sm.red[w][2 * which]));
    s.kth = min(s.kth, __float_as_uint(sm.red[w][2 * which + 1]));
  }
  return s;
}

XM_DEV float block_max_f(float v, LogpSmem& sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) sm.red[threadIdx.x >> 5][0] = v;
  __syncthreads();
  v = sm.red[0][0];
  for (int w = 1; w < kWarps; ++w) v = fmaxf(v, sm.red[w][0]);
  __syncthreads();
  return v;
}
// best = the `top` largest entries of list[0 .. n), n <= kListCap, in order.  False where too many are left (equal logits).
XM_DEV bool best_of_list(LogpSmem& sm, int n, int top) {
  constexpr int EACH = kListCap / kThreads;
  u64 e[EACH], m = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int at = i * kThreads + (int)threadIdx.x;
    e[i] = at < n ? sm.list[at] : 0ull;
    m = e[i] > m ? e[i] : m;
  }
  const uint32_t t = n > kThreads ? block_seen((uint32_t)(m >> 32), top, 0, sm).kth : 0u;
  if (threadIdx.x == 0) sm.left = 0;
  __syncthreads();                                   // (the list is in registers)
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (e[i] && (uint32_t)(e[i] >> 32) >= t) sm.list[atomicAdd(&sm.left, 1)] = e[i];
  __syncthreads();
  const int left = sm.left;
  if (left > 2 * kThreads) return false;
  for (int i = threadIdx.x; i < left; i += kThreads) {
    const u64 mine = sm.list[i];
    int before = 0;
    for (int j = 0; j < left; ++j) before += sm.list[j] > mine;
    if (before < top) sm.best[before] = mine;
  }
  __syncthreads();
  return true;
}

// How many logits of a vector reach a threshold, and their maximum: of 16-bit logits two at a time, in their own type (a
// threshold that is no number of the type is never reached).
template <typename XT>
struct Ranks {
  typedef float Threshold, Most;           // Most: of a vector's maxima
  int n = 0;
  XM_DEV static Threshold threshold(float t) { return t; }
  XM_DEV static Most both(float t) { return t; }
  XM_DEV static Most larger(Most a, Most b) { return fmaxf(a, b); }
  XM_DEV static float value(Most m) { return m; }
  XM_DEV static bool reaches(Most m, Most t) { return m >= t; }
  XM_DEV static Most most_of(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  XM_DEV void add(const uint4& u, Most m, Threshold t) {
    if (m >= t)
      n += (__uint_as_float(u.x) >= t) + (__uint_as_float(u.y) >= t) + (__uint_as_float(u.z) >= t) + (__uint_as_float(u.w) >= t);
  }
  XM_DEV void flush() {}
};
template <typename T2, typename T1>
struct Ranks16 {
  typedef T2 Threshold, Most;
  int n = 0;
  T2 part;                                 // counts of up to 64 vectors: whole numbers of bf16 too (4 a vector and half)
  XM_DEV Ranks16() { memset(&part, 0, 4); }
  XM_DEV static T2 two(uint32_t w) {
    T2 t;
    memcpy(&t, &w, 4);
    return t;
  }
  XM_DEV static T2 both(float t) {         // (a number of the type, an infinity or NaN)
    T2 v;
    v.x = v.y = from_f32<T1>(t);
    return v;
  }
  XM_DEV static T2 larger(T2 a, T2 b) { return __hmax2(a, b); }
  XM_DEV static float value(T2 m) { return fmaxf((float)m.x, (float)m.y); }
  XM_DEV static bool reaches(T2 m, T2 t) { return __hge2_mask(m, t) != 0; }
  XM_DEV static T2 most_of(const uint4& u) { return __hmax2(__hmax2(two(u.x), two(u.y)), __hmax2(two(u.z), two(u.w))); }
  XM_DEV void add(const uint4& u, T2, Threshold t) {
    part = __hadd2(part, __hadd2(__hadd2(__hge2(two(u.x), t), __hge2(two(u.y), t)), __hadd2(__hge2(two(u.z), t), __hge2(two(u.w), t))));
  }
  XM_DEV void flush() {
    n += (int)((float)part.x + (float)part.y);
    memset(&part, 0, 4);
  }
};
template <> struct Ranks<__half> : Ranks16<__half2, __half> {
  XM_DEV static __half2 threshold(float t) { return __half2half2(__float2half_ru(t)); }
};
template <> struct Ranks<__nv_bfloat16> : Ranks16<__nv_bfloat162, __nv_bfloat16> {
  XM_DEV static __nv_bfloat162 threshold(float t) { return __bfloat162bfloat162(__float2bfloat16_ru(t)); }
};

// TOP: whether there are alternatives to find.
template <typename XT, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) k_logprobs(LogpArgs a) {
  constexpr int VE = Part<XT>::VE;
  __shared__ LogpSmem sm;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), cr = (int)cl.block_rank(), b = (int)(blockIdx.x / C);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  Part<XT> p;
  p.row = (const XT*)a.logits + (int64_t)b * a.stride;
  p.base = (const XT*)((uintptr_t)p.row & ~(uintptr_t)15);
  p.mis = (int)(p.row - p.base);
  p.V = a.V;
  const int vectors = (p.mis + a.V + VE - 1) / VE, piece = (vectors + C - 1) / C;
  p.v0 = min(cr * piece, vectors);
  p.nv = min(piece, vectors - p.v0);

  const float T = a.d_temperature ? a.d_temperature[b] : a.temperature;
  const float c = (float)(1.4426950408889634 / (double)T);
  const bool greedy = !(T > 0.f) || !(c < INFINITY);
  const int64_t token = a.wide_tokens ? ((const int64_t*)a.tokens)[b] : ((const int*)a.tokens)[b];
  const bool valid = token >= 0 && token < a.V;
  const float xt = valid ? to_f32<XT>(p.row[token]) : INFINITY;
  const bool seen = xt > -INFINITY;                  // (else every logit above -inf counts, and equal ones below)
  const float thr_hi = seen ? above(xt) : -3.402823466e38f, thr_lo = seen ? xt : thr_hi;
  const int tv = valid ? (p.mis + (int)token) / VE : 0;

  // Rounds of kUnroll vectors a thread; the vectors of a round lie spread over the part.  Vectors at the row's ends, which may
  // hold others' logits too, are the last warp's first.
  const int lo = p.v0 + (p.nv > 0 && !p.inner(p.v0)), end = p.v0 + p.nv - (p.nv > 0 && !p.inner(p.v0 + p.nv - 1) && p.nv > lo - p.v0);
  const int chunks = (end - lo + 31) / 32, rounds = (chunks + kWarps * kUnroll - 1) / (kWarps * kUnroll);
  const int first = lo + rounds * warp * 32 + lane, apart = rounds * kWarps * 32;      // vector u of round r: first + u apart + 32 r
  const uint4* const vectors_at = reinterpret_cast<const uint4*>(p.base);
  const uint4 none = sizeof(XT) == 4 ? make_uint4(0x7fffffffu, 0x7fffffffu, 0x7fffffffu, 0x7fffffffu)
                                     : make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
  uint4 cur[kUnroll], edge = none;
  int edge_v = -1;
  if (warp == kWarps - 1 && lane < 2) {
    edge_v = lane == 0 ? (lo > p.v0 ? p.v0 : -1) : (end < p.v0 + p.nv ? p.v0 + p.nv - 1 : -1);
    if (edge_v >= 0) edge = p.edge(edge_v);
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) cur[u] = first + u * apart < end ? ldg_stream_v4(vectors_at + first + u * apart) : none;
  if (tid == 0) sm.n = sm.n_high = 0;
  // the reference and the list's threshold, from the first round with a logit above -inf
  typedef Ranks<XT> R;
  typename R::Most peak = R::larger(R::most_of(edge), R::both(-INFINITY));      // of what this thread has seen (NaN: nothing)
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) peak = R::larger(peak, R::most_of(cur[u]));
  const bool whole = p.nv * VE <= kListCap;          // a part that the list holds
  const int top = TOP && !whole ? a.top : 0;
  int turn = 0;
  Seen so_far = block_seen(logit_key(R::value(peak)), top, turn, sm);
  int r0 = 0;
  while (so_far.most == 0 && r0 + 1 < rounds) {
    ++r0;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = first + 32 * r0 + u * apart;
      cur[u] = v < end ? ldg_stream_v4(vectors_at + v) : none;
      peak = R::larger(peak, R::most_of(cur[u]));
    }
    so_far = block_seen(logit_key(R::value(peak)), top, turn ^= 1, sm);
  }
  const float ref = so_far.most ? key_logit(so_far.most) : INFINITY;       // (INFINITY: nothing reaches it)
  typename R::Most at_peak = R::both(ref), thr_top = R::both(__uint_as_float(0x7fffffffu));
  // (no threshold yet: every logit above -inf)
  if (top) thr_top = so_far.kth ? R::both(key_logit(so_far.kth)) : R::threshold(-3.402823466e38f);
  typename R::Most gate = TOP && top ? thr_top : at_peak;                  // the smaller of the two
  const float rc = greedy || !(ref < INFINITY) ? 0.f : ref * c;
  const float cc = greedy ? 0.f : c;
  float2 S = make_float2(0.f, 0.f), E = S;
  sm.sums[tid] = make_float2(0.f, 0.f);
  Ranks<XT> ranks;
  typename Ranks<XT>::Threshold at_least_lo = Ranks<XT>::threshold(thr_lo), at_least_hi = Ranks<XT>::threshold(thr_hi);
  // (their conversion is long: not once a vector)
  asm volatile("" : "+r"(reinterpret_cast<uint32_t&>(at_least_lo)), "+r"(reinterpret_cast<uint32_t&>(at_least_hi)));
  auto take = [&](uint4 raw, int v) {
    const typename R::Most most = R::most_of(raw);
    ranks.add(raw, most, v < tv ? at_least_lo : at_least_hi);
    peak = R::larger(peak, most);
    if (R::reaches(most, gate)) {
      if (TOP && R::reaches(most, thr_top)) {        // (which of its logits: later, for all such vectors together)
        const int at = atomicAdd(&sm.n, 1);
        if (at < kListCap) sm.vectors[at] = v;
      }
      if (R::reaches(most, at_peak)) {
        const int at = atomicAdd(&sm.n_high, 1);
        if (at < kHighMax) {
          sm.high[at] = raw;
          sm.high_at[at] = v;
        }
        raw = none;
      }
    }
    float x[VE];
    Part<XT>::values(raw, x);
#pragma unroll
    for (int i = 0; i < VE; i += 2) {
      float2 t = fma2(make_float2(x[i], x[i + 1]), make_float2(cc, cc), make_float2(-rc, -rc));
      t.x = fmaxf(t.x, -200.f);
      t.y = fmaxf(t.y, -200.f);
      const float2 e = make_float2(exp2_fast(t.x), exp2_fast(t.y));
      S = add2(S, e);
      E = fma2(e, t, E);
    }
  };
  if (edge_v >= 0) take(edge, edge_v);
  for (int r = r0; r < rounds; ++r) {
    uint4 next[kUnroll];
    const int v = first + 32 * r;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      next[u] = r + 1 < rounds && v + 32 + u * apart < end ? ldg_stream_v4(vectors_at + v + 32 + u * apart) : none;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) take(cur[u], v + u * apart);
    if ((r & 3) == 3) {
      ranks.flush();
      float2& q = sm.sums[tid];
      q = make_float2(q.x + (S.x + S.y), q.y + (E.x + E.y));
      S = E = make_float2(0.f, 0.f);
    }
    if (r > r0 && (r & (r + 1)) == 0 && r + 1 < rounds) {
      so_far = block_seen(logit_key(R::value(peak)), top, turn ^= 1, sm);
      gate = at_peak = R::both(key_logit(so_far.most));
      if (TOP && so_far.kth) thr_top = R::both(key_logit(so_far.kth));
      if (TOP && top) gate = thr_top;
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) cur[u] = next[u];
  }
  ranks.flush();
  int count = ranks.n;
  float sum_S = sm.sums[tid].x + (S.x + S.y), sum_E = sm.sums[tid].y + (E.x + E.y);
  double r2 = (double)rc;
  float own = -INFINITY;                             // a logit that this thread has beside its sums
  // a logit of exponent t joins them
  auto join = [&](float t) {
    t = fmaxf(t, -200.f);
    const float w = exp2f(t);
    sum_S += w;
    sum_E = fmaf(w, t, sum_E);
  };
  const float seen_most = R::value(peak);
  const bool fine = greedy || (sum_S < 1e38f && fabsf(sum_E) < 1e38f && seen_most < INFINITY && fabsf(rc) < INFINITY &&
                               !(fmaf(seen_most, cc, -rc) >= 100.f));
  const bool again = __syncthreads_or(!fine) || (!greedy && sm.n_high > kHighMax);
  if (again) {
    // another reference: this part's maximum
    float mx = -INFINITY;
    p.each([&](float x, int) { mx = fmaxf(mx, x); });
    mx = block_max_f(mx, sm);
    double s = 0., e = 0.;                           // (one chain of additions through the part)
    p.each([&](float x, int) {
      const float t = x == mx ? 0.f : mx < INFINITY && x > -INFINITY ? fmaxf((x - mx) * c, -200.f) : -200.f, w = exp2_fast(t);
      if (x == mx && own != mx) {
        own = mx;
      } else {
        s += (double)w;
        e += (double)(w * t);
      }
    });
    sum_S = (float)s;
    sum_E = (float)e;
    r2 = (double)mx * (double)c;
  } else {
    // the vectors left out, by their place (the order in which they came must not matter)
    const int n = min(sm.n_high, kHighMax);
    if (tid < n) {
      int before = 0;
      for (int i = 0; i < n; ++i) before += sm.high_at[i] < sm.high_at[tid];
      sm.high_order[before] = tid;
    }
    __syncthreads();
    if (tid / VE < n) own = to_f32<XT>(reinterpret_cast<const XT*>(&sm.high[sm.high_order[tid / VE]])[tid % VE]);
  }
  const uint32_t key = logit_key(own), most_key = __reduce_max_sync(~0u, key);
  const unsigned with_most = __ballot_sync(~0u, key == most_key);
  if (key && lane != __ffs(with_most) - 1) join(again ? 0.f : fmaf(own, cc, -rc));
  sum_S = warp_sum(sum_S);
  sum_E = warp_sum(sum_E);
  if (lane == 0) sm.part[warp] = {sum_S, sum_E, key_logit(most_key)};
  if (!seen) p.each([&](float x, int i) { count += i < token && !(x > -INFINITY); });
  count = __reduce_add_sync(~0u, count);
  if (lane == 0) sm.red64[warp] = (u64)count;
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kWarps; ++w) n += (int)sm.red64[w];
    sm.above = n;
    sm.r = r2;
  }
  if constexpr (TOP) {
    if (tid < kTopMax) sm.best[tid] = 0ull;
    const int listed = sm.n;
    const float floor_top = R::value(thr_top);
    __syncthreads();
    if (tid == 0) sm.n = 0;
    __syncthreads();
    if (whole) {
      p.each([&](float x, int i) { sm.list[atomicAdd(&sm.n, 1)] = entry(x, i); });
    } else if (listed <= kListCap) {
      for (int l = tid; l < listed; l += kThreads) {
        const int v = sm.vectors[l];
        float x[VE];
        Part<XT>::values(p.load(v), x);
#pragma unroll
        for (int i = 0; i < VE; ++i)
          if (x[i] >= floor_top) {
            const int at = atomicAdd(&sm.n, 1);
            if (at < kListCap) sm.list[at] = entry(x[i], p.index(v) + i);
          }
      }
    }
    __syncthreads();
    const int n = listed <= kListCap ? sm.n : listed;
    __syncthreads();
    const bool slow = n > kListCap || !best_of_list(sm, n, a.top);
    if (!slow && !whole && n < a.top) {
      // All logits above -inf are there (a threshold above the lowest one has `top` at or above it): those of -inf follow by their
      // index.  There are enough of them among the part's first 2 kTopMax logits.
      const int i = max(0, p.index(p.v0)) + tid;
      const bool out = tid < 2 * kTopMax && i < min(a.V, p.index(p.v0 + p.nv)) && !(to_f32<XT>(p.row[i]) > -INFINITY);
      const unsigned outs = __ballot_sync(~0u, out);
      if (lane == 0) sm.red64[warp] = (u64)__popc(outs);
      __syncthreads();
      int at = n + __popc(outs & ((1u << lane) - 1));
      for (int w = 0; w < warp; ++w) at += (int)sm.red64[w];
      if (out && at < a.top) sm.best[at] = entry(-INFINITY, i);
    }
    if (slow) {
      u64 last = ~0ull;
      for (int j = 0; j < a.top; ++j) {
        u64 m64 = 0;
        p.each([&](float x, int i) {
          const u64 t = entry(x, i);
          if (t < last && t > m64) m64 = t;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const u64 t = __shfl_xor_sync(~0u, m64, o);
          m64 = t > m64 ? t : m64;
        }
        __syncthreads();
        if (lane == 0) sm.red64[warp] = m64;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) m64 = sm.red64[w] > m64 ? sm.red64[w] : m64;
        if (tid == 0) sm.best[j] = m64;
        last = m64;
      }
    }
  }
  if (C > 1) cl.sync();
  else __syncthreads();
  if (cr == 0) {
    // the warps' sums, on the largest logit (two warps' a lane of the first warp)
    if (warp == 0) {
      const LogpSmem* o[2];
      Sums q[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int at = lane + 32 * h;
        o[h] = C > 1 && at < C * kWarps ? cl.map_shared_rank(&sm, at / kWarps) : &sm;
        q[h] = {0.f, 0.f, -INFINITY};
        if (at < C * kWarps) q[h] = o[h]->part[at % kWarps];
      }
      int rank = lane < C ? (C > 1 ? cl.map_shared_rank(&sm, lane) : &sm)->above : 0;
      rank = __reduce_add_sync(~0u, rank);
      const uint32_t k0 = logit_key(q[0].peak), k1 = logit_key(q[1].peak), largest = __reduce_max_sync(~0u, max(k0, k1));
      const float M = key_logit(largest);
      const bool inf = !(M < INFINITY);
      const double R = (double)M * (double)c;
      const unsigned with0 = __ballot_sync(~0u, k0 == largest), with1 = __ballot_sync(~0u, k1 == largest);
      float s = 0.f, e = 0.f;
      if (largest && !greedy) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t k = h ? k1 : k0;
          const bool own = k == largest && (h ? with0 == 0 && lane == __ffs(with1) - 1 : lane == __ffs(with0) - 1);
          if (inf) {                                 // (parts with such logits count those alone)
            if (k == largest) s += q[h].S + (own ? 0.f : 1.f);
            continue;
          }
          // sums on a reference of d + the largest, up to 2^100 and more: 2^d alone may be below fp32's numbers
          auto add = [&](double d, float S, float E) {
            if (!(d > -250.)) return;
            const float whole = rintf((float)d);
            const double f = (double)exp2f((float)(d - (double)whole)) * __hiloint2double((1023 + (int)whole) << 20, 0);
            s += (float)(f * (double)S);
            e += (float)(f * ((double)E + d * (double)S));
          };
          if (q[h].S > 0.f) add(o[h]->r - R, q[h].S, q[h].E);
          if (k && !own) add((double)q[h].peak * (double)c - R, 1.f, 0.f);
        }
      }
      s = warp_sum(s);
      e = warp_sum(e);
      if (lane == 0) {
        sm.most = R;
        const float lse = log1pf(s);
        sm.lse = lse;
        sm.inf = inf;
        sm.rank = rank;
        a.entropy[b] = fmaxf(0.f, lse - 0.6931471805599453f * (e / (1.f + s)));
      }
    }
    __syncthreads();
    const double most = sm.most, lse = sm.lse;
    const bool inf = sm.inf;
    int rank = sm.rank;
    auto logp = [&](float x, bool first) -> float {
      if (!(x > -INFINITY)) return greedy && first ? 0.f : -INFINITY;
      if (greedy) return first ? 0.f : -INFINITY;
      if (inf) return x < INFINITY ? -INFINITY : (float)-lse;
      return (float)fmin(0.0, 0.6931471805599453 * ((double)x * (double)c - most) - lse);
    };
    if (tid == 0) {
      if (valid) {                                   // equal logits before the token in its own vector
        const int at = max(0, tv * VE - p.mis);
        for (int i = at; seen && i < (int)token; ++i) rank += to_f32<XT>(p.row[i]) == xt;
      }
      a.rank[b] = valid ? rank : -1;
      a.logprob[b] = valid ? logp(xt, rank == 0 && seen) : __uint_as_float(0x7fffffffu);
    }
    if constexpr (TOP) {
      const int all = C * a.top;
      for (int i = tid; i < all; i += kThreads) {
        const LogpSmem* o = C > 1 ? cl.map_shared_rank(&sm, i / a.top) : &sm;
        sm.merge[i] = o->best[i % a.top];
      }
      __syncthreads();
      for (int i = tid; i < all; i += kThreads) {
        const u64 mine = sm.merge[i];
        int before = 0;
        for (int j = 0; j < all; ++j) before += sm.merge[j] > mine;
        if (mine && before < a.top) {
          const float x = key_logit((uint32_t)(mine >> 32));
          a.top_ids[(int64_t)b * a.top + before] = (int)~(uint32_t)mine;
          a.top_logp[(int64_t)b * a.top + before] = logp(x, before == 0 && x > -INFINITY);
        }
      }
    }
  }
  if (C > 1) cl.sync();                              // the others' memory is read until here
}

template <typename XT>
cudaError_t logp_launch(const LogpArgs& a, int64_t B, cudaStream_t st) {
  // one CTA a row; more while the rows leave SMs without work and a CTA would still have a round, or while a part has
  // more than 2^18 logits (the list is made for that)
  int C = 1;
  while (C < kClusterMax && ((B * C < 2 * 148 && a.V > C * kThreads * kUnroll * (16 / (int)sizeof(XT)) / 2) ||
                             a.V > (C << 18)))
    C *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(B * C));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return a.top > 0 ? cudaLaunchKernelEx(&cfg, k_logprobs<XT, true>, a) : cudaLaunchKernelEx(&cfg, k_logprobs<XT, false>, a);
}

}  // namespace

extern "C" int xm_logprobs(const void* d_logits, int dtype, int64_t B, int64_t V, int64_t stride, const void* d_tokens,
                           int token_bytes, float temperature, const float* d_temperature, int top, float* d_logprob,
                           float* d_entropy, int* d_rank, int* d_top_ids, float* d_top_logprobs, void* stream) {
  if (dtype != XM_DT_F32 && dtype != XM_DT_F16 && dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "logprobs: bad element type %d", dtype);
  if (B < 0 || B > INT32_MAX / 8 || V < 1 || V > (1 << 20) || stride < V)
    return xm_set_error(XM_ERR_INVALID, "logprobs: bad sizes (1 to 2^20 logits a row)");
  if (token_bytes != 4 && token_bytes != 8) return xm_set_error(XM_ERR_INVALID, "logprobs: tokens of %d bytes", token_bytes);
  if (top < 0 || top > kTopMax || top > V)
    return xm_set_error(XM_ERR_INVALID, "logprobs: %d alternatives (up to %d, and to the vocabulary)", top, kTopMax);
  if (B == 0) return XM_OK;
  if (!d_logits || !d_tokens || !d_logprob || !d_entropy || !d_rank || (top && (!d_top_ids || !d_top_logprobs)))
    return xm_set_error(XM_ERR_INVALID, "logprobs: null pointer");
  if (((uintptr_t)d_logits & (dtype == XM_DT_F32 ? 3 : 1)) || ((uintptr_t)d_tokens & (token_bytes - 1)) ||
      (((uintptr_t)d_temperature | (uintptr_t)d_logprob | (uintptr_t)d_entropy | (uintptr_t)d_rank |
        (uintptr_t)d_top_ids | (uintptr_t)d_top_logprobs) & 3))
    return xm_set_error(XM_ERR_INVALID, "logprobs: unaligned pointer");
  LogpArgs a{d_logits, stride, (int)V, top, d_tokens, token_bytes == 8, temperature, d_temperature, d_logprob, d_entropy,
             d_top_logprobs, d_rank, d_top_ids};
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = dtype == XM_DT_F32   ? logp_launch<float>(a, B, st)
                        : dtype == XM_DT_F16 ? logp_launch<__half>(a, B, st)
                                             : logp_launch<__nv_bfloat16>(a, B, st);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "logprobs launch: %s", cudaGetErrorString(e));
  return xm_check_launch("logprobs");
}
