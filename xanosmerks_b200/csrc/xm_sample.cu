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
// k_sample: one CTA per row.  The thresholds are found by bisecting the ordered bit pattern of the
// logits, one pass over the row for each bit.
#include "xm_kv.cuh"

namespace {

constexpr int kSampleThreads = 1024;

// order-preserving key of a logit: NaN and -inf below everything else
XM_DEV uint32_t order_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(x + 0.0f);            // -0 and +0 are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

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
};

template <typename XT>
struct Row {
  const XT* x;
  float mx;
  double inv_t;
  double one;        // 2^F
  bool greedy;
  XM_DEV float at(int i) const { return to_f32(x[i]); }
  XM_DEV unsigned long long weight(float v) const {
    if (v == mx) return (unsigned long long)one;
    if (greedy || !(v > -INFINITY) || !(mx < INFINITY)) return 0ull;
    return __double2ull_rn(exp(((double)v - (double)mx) * inv_t) * one);
  }
};

template <typename T>
XM_DEV T block_add(T v, T* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  T r = 0;
  for (int w = 0; w < kSampleThreads / 32; ++w) r += red[w];
  return r;
}

// The first index, in order, at which the running sum of f over the row exceeds tgt; V where none does.
// Each warp owns a contiguous segment.
template <typename F>
XM_DEV int first_above(F f, int V, unsigned long long tgt, unsigned long long* red, int* found) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int W = kSampleThreads / 32;
  const int seg = ((V + W - 1) / W + 31) / 32 * 32, lo = min(V, warp * seg), hi = min(V, lo + seg);
  unsigned long long sum = 0;
  for (int i = lo + lane; i < hi; i += 32) sum += f(i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  if (threadIdx.x == 0) *found = V;
  __syncthreads();
  unsigned long long before = 0;
  for (int w = 0; w < warp; ++w) before += red[w];
  if (before <= tgt && before + sum > tgt) {
    for (int i0 = lo; i0 < hi; i0 += 32) {
      const int i = i0 + lane;
      unsigned long long c = i < hi ? f(i) : 0ull;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long n = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += n;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + c > tgt);
      if (hit) {
        if (lane == 0) *found = i0 + __ffs(hit) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, c, 31);
    }
  }
  __syncthreads();
  return *found;
}

template <typename XT>
__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleArgs a) {
  __shared__ unsigned long long red[32];
  __shared__ float redf[32];
  __shared__ int found;
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x, V = a.V, tid = threadIdx.x;
  Row<XT> r;
  r.x = (const XT*)a.logits + (int64_t)b * a.stride;
  float mx = -INFINITY;
  for (int i = tid; i < V; i += kSampleThreads) mx = fmaxf(mx, r.at(i));
  r.mx = block_max<kSampleThreads>(mx, redf);
  if (!(r.mx > -INFINITY)) {                      // nothing to choose from
    if (tid == 0) {
      a.ids[b] = 0;
      if (a.logp) a.logp[b] = -INFINITY;
    }
    return;
  }
  const float T = a.d_temperature ? a.d_temperature[b] : a.temperature;
  const int top_k = a.d_top_k ? a.d_top_k[b] : a.top_k;
  const float top_p = a.d_top_p ? a.d_top_p[b] : a.top_p;
  const float min_p = a.d_min_p ? a.d_min_p[b] : a.min_p;
  r.greedy = !(T > 0.f);
  r.inv_t = r.greedy ? 0.0 : 1.0 / (double)T;
  r.one = (double)(1ull << a.frac_bits);
  const int k = r.greedy ? 1 : (top_k > 0 && top_k < V ? top_k : V);

  // the largest key that at least k tokens reach
  uint32_t tau = 0;
  unsigned long long quota = V;                   // tokens with key == tau that are kept, lowest index first
  if (k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = tau | (1u << bit);
      unsigned long long n = 0;
      for (int i = tid; i < V; i += kSampleThreads) n += order_key(r.at(i)) >= c;
      if (block_add(n, red) >= (unsigned long long)k) tau = c;
    }
    unsigned long long n = 0;
    for (int i = tid; i < V; i += kSampleThreads) n += order_key(r.at(i)) > tau;
    quota = k - block_add(n, red);
  }
  if (top_p < 1.f && !r.greedy) {
    // mass of the top k; equal logits have equal weights
    unsigned long long z = 0, wt = 0;
    for (int i = tid; i < V; i += kSampleThreads) {
      const float v = r.at(i);
      const uint32_t key = order_key(v);
      if (key > tau) z += r.weight(v);
      if (key == tau) wt = max(wt, r.weight(v));
    }
    z = block_add(z, red);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wt = max(wt, __shfl_xor_sync(0xffffffffu, wt, o));
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = wt;
    __syncthreads();
    for (int w = 0; w < kSampleThreads / 32; ++w) wt = max(wt, red[w]);
    if (k < V) z += quota * wt;                   // (k == V: tau = 0 holds only tokens of weight 0)
    const unsigned long long p = max(1ull, (unsigned long long)ceil((double)fmaxf(top_p, 0.f) * (double)z));
    // the smallest key with less than p above it; mass(key > c) falls as c grows
    uint32_t c = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t t = (c | (1u << bit)) - 1;   // is p or more above t?  then the answer is above t
      unsigned long long g = 0;
      for (int i = tid; i < V; i += kSampleThreads) {
        const float v = r.at(i);
        if (order_key(v) > t) g += r.weight(v);
      }
      if (block_add(g, red) >= p) c |= 1u << bit;
    }
    if (c >= tau) {
      unsigned long long g = 0, wc = 0, n = 0;
      for (int i = tid; i < V; i += kSampleThreads) {
        const float v = r.at(i);
        const uint32_t key = order_key(v);
        if (key > c) g += r.weight(v);
        if (key == c) {
          wc += r.weight(v);
          ++n;
        }
      }
      g = block_add(g, red);
      wc = block_add(wc, red);
      n = block_add(n, red);
      wc = n ? wc / n : 0;
      const unsigned long long q = wc ? (p - g + wc - 1) / wc : n;
      quota = c == tau ? min(quota, q) : q;
      tau = c;
    }
  }
  // ties at tau: those up to index `cut` are kept
  const int cut = first_above([&](int i) { return (unsigned long long)(order_key(r.at(i)) == tau); }, V,
                              quota - 1, red, &found);
  const unsigned long long wmin =
      min_p > 0.f ? (unsigned long long)ceil((double)fminf(min_p, 1.f) * r.one) : 0ull;
  auto kept = [&](int i) {
    const float v = r.at(i);
    const uint32_t key = order_key(v);
    if (key < tau || (key == tau && i > cut)) return 0ull;
    const unsigned long long w = r.weight(v);
    return w >= wmin ? w : 0ull;
  };
  unsigned long long z = 0;
  for (int i = tid; i < V; i += kSampleThreads) z += kept(i);
  z = block_add(z, red);
  const float u = a.u[b];
  unsigned long long tgt = u > 0.f ? (unsigned long long)fmin((double)u * (double)z, 1.8e19) : 0ull;
  tgt = min(tgt, z - 1);
  const int id = first_above(kept, V, tgt, red, &found);
  if (tid == 0) {
    a.ids[b] = id;
    if (a.logp) {
      const float v = r.at(id);
      const double num = v == r.mx ? 0.0 : ((double)v - (double)r.mx) * r.inv_t;
      a.logp[b] = (float)(num - log((double)z / r.one));
    }
  }
}

}  // namespace

extern "C" int xm_sample(const void* d_logits, int dtype, int64_t B, int64_t V, int64_t stride, const float* d_u,
                         float temperature, const float* d_temperature, int top_k, const int* d_top_k, float top_p,
                         const float* d_top_p, float min_p, const float* d_min_p, int* d_ids, float* d_logprob,
                         void* stream) {
  if (dtype != XM_DT_F32 && dtype != XM_DT_F16 && dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "sample: bad element type %d", dtype);
  if (B < 0 || B > INT32_MAX || V < 1 || V > (1 << 30) || stride < V)
    return xm_set_error(XM_ERR_INVALID, "sample: bad sizes");
  if (B == 0) return XM_OK;
  if (!d_logits || !d_u || !d_ids) return xm_set_error(XM_ERR_INVALID, "sample: null pointer");
  if (((uintptr_t)d_logits & (dtype == XM_DT_F32 ? 3 : 1)) || (((uintptr_t)d_u | (uintptr_t)d_temperature |
      (uintptr_t)d_top_k | (uintptr_t)d_top_p | (uintptr_t)d_min_p | (uintptr_t)d_ids | (uintptr_t)d_logprob) & 3))
    return xm_set_error(XM_ERR_INVALID, "sample: unaligned pointer");
  int frac = 62;
  while ((V >> (62 - frac)) > 1 || frac > 44) --frac;      // V 2^frac stays below 2^63
  SampleArgs a{d_logits, stride, (int)V, d_u, temperature, top_p, min_p, top_k, d_temperature, d_top_p, d_min_p,
               d_top_k, d_ids, d_logprob, frac};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)B);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = dtype == XM_DT_F32   ? cudaLaunchKernelEx(&cfg, k_sample<float>, a)
                        : dtype == XM_DT_F16 ? cudaLaunchKernelEx(&cfg, k_sample<__half>, a)
                                             : cudaLaunchKernelEx(&cfg, k_sample<__nv_bfloat16>, a);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "sample launch: %s", cudaGetErrorString(e));
  return xm_check_launch("sample");
}
