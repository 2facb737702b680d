// Log-probability and rank of a given token, entropy, and the largest alternatives of each row of logits, in one pass.
//
// Row x, temperature T, c = log2(e) / T: w_i = 2^(c x_i - r) for a reference r, S = sum w, E = sum w (c x - r);
//   logprob_i = ln 2 (c x_i - r - log2 S),   entropy = ln 2 (log2 S - E / S),
//   rank = how many tokens have a larger logit, or the same one at a lower index.
//
// r is not the row's maximum but that of the logits that a CTA sees first: any r within 2^100 of the maximum gives the same
// sums, so that nothing is rescaled on the way.  Where that does not hold (S below 2^-100, where weights that count would
// vanish, or beyond the numbers) the CTA takes its part of the row again with its own maximum.  A weight's exponent is held above -200, which also gives -inf and NaN logits
// the weight 0 (and 0 in E).
//
// Alternatives: every warp knows the j-th largest of its lanes' maxima so far; the least of these over the warps, j = ceil(top
// / warps), has at least `top` logits at or above it.  Only vectors with such logits go to a list, and the threshold is raised
// whenever twice as much has been seen (a round's logits are spread over the whole part), so that a few hundred of 128000
// pass.  A list that runs over, or a threshold of -inf, sends the CTA to the slow way: one pass a place.
//
// C CTAs (a cluster) share a row where rows are few or long.  Bound: HBM and issue for many rows (each logit is read once; some
// eight instructions a logit, sums and exponents two at a time, ranks and maxima of 16-bit logits too), latency for few.
//
// Measured, cold: 2048 rows of 32000 fp32 logits 55 us (4.7 TB/s); 2000 of 128001 fp16 with 8 alternatives 131 to 137 us (3.8 TB/s,
// three quarters of the issue slots); 64 of 128000 bf16 with 20, 18 us; one of 32000, 8 us in a captured graph.
#include <cooperative_groups.h>

#include "xm_gemv_dot.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kUnroll = 4, kListCap = 2048, kTopMax = 64, kClusterMax = 8;
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

struct alignas(16) LogpSmem {
  u64 list[kListCap];
  int vectors[kListCap];                   // those with a logit for the list
  u64 best[kTopMax];                       // this CTA's largest, in order; 0: none
  u64 merge[kClusterMax * kTopMax];
  float red[kWarps][4];
  u64 red64[kWarps];
  int n, left;
  float ref, thr;
  // what the cluster's first CTA reads of each
  double r;                                // c x reference (log2)
  float S, E, mx;
  int above;
  // the row's
  double lse;
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
XM_DEV float block_sum_f(float v, LogpSmem& sm) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) sm.red[threadIdx.x >> 5][0] = v;
  __syncthreads();
  v = sm.red[0][0];
  for (int w = 1; w < kWarps; ++w) v += sm.red[w][0];
  __syncthreads();
  return v;
}

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

// A logit that at least `top` of the block's threads have a maximum at or above (key 0: there is none).
XM_DEV uint32_t block_threshold(uint32_t key, int top, LogpSmem& sm) {
  const uint32_t m = warp_kth(key, (top + kWarps - 1) / kWarps);
  if ((threadIdx.x & 31) == 0) sm.red[threadIdx.x >> 5][1] = __uint_as_float(m);
  __syncthreads();
  uint32_t t = ~0u;
  for (int w = 0; w < kWarps; ++w) t = min(t, __float_as_uint(sm.red[w][1]));
  __syncthreads();
  return t;
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
  const uint32_t t = n > kThreads ? block_threshold((uint32_t)(m >> 32), top, sm) : 0u;
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
  typedef float Threshold;
  int n = 0;
  XM_DEV static Threshold threshold(float t) { return t; }
  XM_DEV static float max_of(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  XM_DEV void add(const uint4& u, Threshold t) {
    if (max_of(u) >= t)
      n += (__uint_as_float(u.x) >= t) + (__uint_as_float(u.y) >= t) + (__uint_as_float(u.z) >= t) + (__uint_as_float(u.w) >= t);
  }
  XM_DEV void flush() {}
};
template <typename T2, typename T1>
struct Ranks16 {
  typedef T2 Threshold;
  int n = 0;
  T2 part;                                 // counts of up to 64 vectors: whole numbers of bf16 too (4 a vector and half)
  XM_DEV Ranks16() { memset(&part, 0, 4); }
  XM_DEV static T2 two(uint32_t w) {
    T2 t;
    memcpy(&t, &w, 4);
    return t;
  }
  XM_DEV static float max_of(const uint4& u) {
    const T2 m = __hmax2(__hmax2(two(u.x), two(u.y)), __hmax2(two(u.z), two(u.w)));
    return fmaxf((float)m.x, (float)m.y);
  }
  XM_DEV void add(const uint4& u, Threshold t) {
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
  // hold others' logits too, are the last warp's last.
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
  if (tid == 0) sm.n = 0;
  // the reference and the list's threshold
  float m = Ranks<XT>::max_of(edge);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) m = fmaxf(m, Ranks<XT>::max_of(cur[u]));
  m = fmaxf(m, -INFINITY);                           // (NaN: nothing)
  float thr_top = __uint_as_float(0x7fffffffu);
  const bool whole = p.nv * VE <= kListCap;          // a part that the list holds
  bool slow = false;
  if (TOP && !whole) {
    const uint32_t t = block_threshold(logit_key(m), a.top, sm);
    slow = t == 0;
    if (!slow) thr_top = key_logit(t);
  }
  float peak = -INFINITY;                            // of what this thread has seen
  m = block_max_f(m, sm);
  const float ref = m > -INFINITY && m < INFINITY ? m : 0.f;
  const float rc = greedy ? 0.f : ref * c;
  const float cc = greedy ? 0.f : c;
  float2 S = make_float2(0.f, 0.f), E = S;
  Ranks<XT> ranks;
  typename Ranks<XT>::Threshold at_least_lo = Ranks<XT>::threshold(thr_lo), at_least_hi = Ranks<XT>::threshold(thr_hi);
  // (their conversion is long: not once a vector)
  asm volatile("" : "+r"(reinterpret_cast<uint32_t&>(at_least_lo)), "+r"(reinterpret_cast<uint32_t&>(at_least_hi)));
  auto take = [&](const uint4& raw, int v) {
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
    ranks.add(raw, v < tv ? at_least_lo : at_least_hi);
    if constexpr (TOP) {
      const float most = Ranks<XT>::max_of(raw);
      peak = fmaxf(peak, most);
      if (most >= thr_top) {                         // (which of its logits: later, for all such vectors together)
        const int at = atomicAdd(&sm.n, 1);
        if (at < kListCap) sm.vectors[at] = v;
      }
    }
  };
  for (int r = 0; r < rounds; ++r) {
    uint4 next[kUnroll];
    const int v = first + 32 * r;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      next[u] = r + 1 < rounds && v + 32 + u * apart < end ? ldg_stream_v4(vectors_at + v + 32 + u * apart) : none;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) take(cur[u], v + u * apart);
    if ((r & 15) == 15) ranks.flush();
    if constexpr (TOP)
      if (!slow && !whole && r > 0 && (r & (r + 1)) == 0 && r + 1 < rounds) {
        const uint32_t t = block_threshold(logit_key(peak), a.top, sm);
        if (t) thr_top = fmaxf(thr_top, key_logit(t));
      }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) cur[u] = next[u];
  }
  if (edge_v >= 0) take(edge, edge_v);
  ranks.flush();
  int count = ranks.n;
  float s = block_sum_f(S.x + S.y, sm), e = block_sum_f(E.x + E.y, sm);
  double r2 = (double)rc;
  float mx = ref;
  if (greedy) {
    s = 1.f;
    e = 0.f;
  } else if (!(s >= 0x1p-100f && s < 1e38f) || !(fabsf(e) < 1e38f)) {
    // another reference: this part's maximum
    mx = -INFINITY;
    p.each([&](float x, int) { mx = fmaxf(mx, x); });
    mx = block_max_f(mx, sm);
    s = e = 0.f;
    if (mx > -INFINITY) {
      p.each([&](float x, int) {
        const float t = x == mx ? 0.f : fmaxf((x - mx) * c, -200.f), w = exp2_fast(t);
        if (x == mx || mx < INFINITY) {
          s += w;
          e = fmaf(w, t, e);
        }
      });
    }
    s = block_sum_f(s, sm);
    e = block_sum_f(e, sm);
    r2 = (double)mx * (double)c;
  }
  if (!seen) p.each([&](float x, int i) { count += i < token && !(x > -INFINITY); });
  count = __reduce_add_sync(~0u, count);
  if (lane == 0) sm.red64[warp] = (u64)count;
  __syncthreads();
  if (tid == 0) {
    int n = 0;
    for (int w = 0; w < kWarps; ++w) n += (int)sm.red64[w];
    sm.above = n;
    sm.r = r2;
    sm.S = s;
    sm.E = e;
    sm.mx = mx;
  }
  if constexpr (TOP) {
    if (tid < kTopMax) sm.best[tid] = 0ull;
    const int listed = sm.n;
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
          if (x[i] >= thr_top) {
            const int at = atomicAdd(&sm.n, 1);
            if (at < kListCap) sm.list[at] = entry(x[i], p.index(v) + i);
          }
      }
    }
    __syncthreads();
    const int n = listed <= kListCap ? sm.n : listed;
    __syncthreads();
    if (!slow) slow = n > kListCap || !best_of_list(sm, n, a.top);
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
    // the parts' sums, on the largest reference (a part a lane of the first warp)
    if (warp == 0) {
      const LogpSmem* o = C > 1 && lane < C ? cl.map_shared_rank(&sm, lane) : &sm;
      const bool there = lane < C && o->S > 0.f;
      double R = there ? o->r : -INFINITY, part_S = there ? (double)o->S : 0., part_E = there ? (double)o->E : 0.;
      const bool inf_part = there && !(o->mx < INFINITY), inf = __any_sync(~0u, inf_part);
      int rank = lane < C ? o->above : 0;
      const double mine_r = R;
#pragma unroll
      for (int i = kClusterMax / 2; i > 0; i >>= 1) {
        R = fmax(R, __shfl_xor_sync(~0u, R, i));
        rank += __shfl_xor_sync(~0u, rank, i);
      }
      if (inf) {
        part_S = inf_part ? part_S : 0.;
        part_E = 0.;
      } else if (there) {
        const double d = mine_r - R, f = d < 0. ? exp2(d) : 1.;
        part_E = f * (part_E + d * part_S);
        part_S *= f;
      }
#pragma unroll
      for (int i = kClusterMax / 2; i > 0; i >>= 1) {
        part_S += __shfl_xor_sync(~0u, part_S, i);
        part_E += __shfl_xor_sync(~0u, part_E, i);
      }
      if (lane == 0) {
        sm.lse = inf ? log2(part_S) : R + log2(part_S);
        sm.inf = inf;
        sm.rank = rank;
        a.entropy[b] = greedy || !(part_S > 0.) ? 0.f : (float)fmax(0.0, 0.6931471805599453 * (log2(part_S) - part_E / part_S));
      }
    }
    __syncthreads();
    const double lse = sm.lse;
    const bool inf = sm.inf;
    int rank = sm.rank;
    auto logp = [&](float x, bool first) -> float {
      if (!(x > -INFINITY)) return greedy && first ? 0.f : -INFINITY;
      if (greedy) return first ? 0.f : -INFINITY;
      if (inf) return x < INFINITY ? -INFINITY : (float)(-0.6931471805599453 * lse);
      return (float)fmin(0.0, 0.6931471805599453 * ((double)x * (double)c - lse));
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
