// Appending to and reading from the paged key/value cache (layout: xm_kv.cuh).
//
// k_kv_put: one warp per (row, head).  A query or key head x of D values is
// optionally normalised, x' = x w / sqrt(mean(x^2) + eps), and rotated by the
// angles of its position, y[i] = x'[i] cos_i - x'[i + D/2] sin_i and
// y[i + D/2] = x'[i + D/2] cos_i + x'[i] sin_i with (cos, sin) from a table that
// the caller computed in 64 bits.  Queries go to q; keys and values go to their
// slot of the cache as fp16 or as blocks of 32 codes of 4 bits.
//
// A block of 32 values: d = fp16(a / -8) with a the first value of largest
// magnitude, code c = floor(x / d + 8.5) clamped to 0..15.  The codes are exact
// decisions: the sign of the single-rounded fma(-(c - 8.5), |d|, x sign(d)) is
// the sign of x / d - (c - 8.5), so a value next to a border between two codes
// goes to the same side as in the formula.  For the same reason keys that become
// codes are normalised and rotated in 64 bits and rounded once to fp32 (64-bit
// arithmetic runs at half the fp32 rate here and is off the critical path of
// the memory traffic); everything else is fp32.
//
// Bound: memory.  Lane l holds values 2l, 2l + 1 of each half of the head (one
// value per half at D = 64), so the rotation needs no exchange, a half-head is
// one 256-byte load at fp32, and a group of 32 values is 16 lanes.
#include <type_traits>

#include "xm_kv.cuh"

namespace {

// Q4_0 of the groups of 32 values held VPL per lane by 32 / VPL consecutive lanes (VPL = 1 or 2,
// values VPL l, VPL l + 1).  c: the codes; returns the group's d (as fp16).
template <int VPL>
XM_DEV __half q4_group(const float (&x)[VPL], int (&c)[VPL]) {
  constexpr int W = 32 / VPL;                         // lanes of a group
  const int lane = threadIdx.x & 31;
  bool bad = false;
  float mag = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    bad |= !(fabsf(x[i]) < INFINITY);
    mag = fmaxf(mag, fabsf(x[i]));
  }
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) mag = fmaxf(mag, __shfl_xor_sync(0xffffffffu, mag, o));
  const unsigned group = VPL == 1 ? 0xffffffffu : 0xffffu << (lane & 16);
  const bool spoilt = __ballot_sync(0xffffffffu, bad) & group;
  bool mine = false;                                  // this lane holds a value of largest magnitude
  float a = 0.f;
#pragma unroll
  for (int i = VPL - 1; i >= 0; --i)
    if (fabsf(x[i]) == mag) {
      mine = true;
      a = x[i];
    }
  const unsigned who = __ballot_sync(0xffffffffu, mine) & group;
  a = __shfl_sync(0xffffffffu, a, who ? __ffs(who) - 1 : lane);
  // a non-finite value spoils its group: d = NaN, every value of the group reads as NaN
  const __half dh = spoilt ? __ushort_as_half((unsigned short)0x7fff) : __float2half_rn(a * -0.125f);
  const float d = __half2float(dh), ad = fabsf(d);
  const bool blank = !(ad > 0.f && ad < INFINITY);
  const float inv = 1.0f / d;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    int q = 8;
    if (!blank) {
      const float y = d < 0.f ? -x[i] : x[i];
      float e = floorf(fmaf(x[i], inv, 8.5f));
      e = fminf(fmaxf(e, 0.f), 15.f);
      if (e > 0.f && fmaf(8.5f - e, ad, y) < 0.f) e -= 1.f;
      else if (e < 15.f && fmaf(7.5f - e, ad, y) >= 0.f) e += 1.f;
      q = (int)e;
    }
    c[i] = q;
  }
  return dh;
}

// Writes one half of a head (values VPL l + i + half D / 2 on lane l) as codes into row `slot` of a part.
// VALUES: the values' order of the codes instead of the keys'.
template <int D, bool VALUES>
XM_DEV void put_half_q4(const float (&x)[D / 64], int half, uint8_t* part, int page_size, int slot) {
  constexpr int VPL = D / 64, NG = D / 32;
  const int lane = threadIdx.x & 31;
  int c[VPL];
  const __half d = q4_group<VPL>(x, c);
  uint32_t w = 0;                                     // this lane's nibbles
#pragma unroll
  for (int i = 0; i < VPL; ++i) w |= (uint32_t)c[i] << (4 * i);
  const int g = half * (NG / 2) + (VPL * lane) / 32;  // group
  const int e = (VPL * lane) % 32;                    // first value in the group
  constexpr int PER = VALUES ? 4 : 8;                 // values of a word (halfword)
  w <<= 4 * (e % PER);
#pragma unroll
  for (int o = 1; o < PER / VPL; o <<= 1) w |= __shfl_xor_sync(0xffffffffu, w, o);
  uint8_t* row = part + (int64_t)slot * (D / 2);
  if (e % PER == 0) {
    if (VALUES)
      reinterpret_cast<uint16_t*>(row)[NG * (e / 4) + g] = (uint16_t)w;
    else
      reinterpret_cast<uint32_t*>(row)[NG * (e / 8) + g] = w;
  }
  if (e == 0) reinterpret_cast<__half*>(part + (int64_t)page_size * (D / 2))[slot * NG + g] = d;
}

template <typename XT, int VPL>
XM_DEV void load_vals(const XT* p, bool pairs, float (&v)[VPL]) {
  if constexpr (VPL == 2) {
    if (pairs) {
      if constexpr (sizeof(XT) == 4) {
        const float2 f = *reinterpret_cast<const float2*>(p);
        v[0] = f.x; v[1] = f.y;
      } else {
        XT t[2];
        *reinterpret_cast<uint32_t*>(t) = *reinterpret_cast<const uint32_t*>(p);
        v[0] = to_f32(t[0]); v[1] = to_f32(t[1]);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) v[i] = to_f32(p[i]);
}

template <typename QT_, int VPL>
XM_DEV void store_vals(QT_* p, bool pairs, const float (&v)[VPL]) {
  if constexpr (VPL == 2) {
    if (pairs) {
      QT_ t[2];
      if constexpr (sizeof(QT_) == 2 && std::is_same<QT_, __half>::value) {
        t[0] = __float2half_rn(v[0]); t[1] = __float2half_rn(v[1]);
      } else {
        t[0] = __float2bfloat16_rn(v[0]); t[1] = __float2bfloat16_rn(v[1]);
      }
      *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(t);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if constexpr (std::is_same<QT_, __half>::value) p[i] = __float2half_rn(v[i]);
    else p[i] = __float2bfloat16_rn(v[i]);
  }
}

XM_DEV double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One head in arithmetic of type F: normalise and rotate lo (first half) and hi (second half).
template <typename F, int D>
XM_DEV void norm_rotate(float (&lo)[D / 64], float (&hi)[D / 64], const float* __restrict__ w, double eps,
                        const float2* __restrict__ cs) {
  constexpr int VPL = D / 64;
  const int lane = threadIdx.x & 31;
  F a[VPL], b[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    a[i] = (F)lo[i];
    b[i] = (F)hi[i];
  }
  if (w) {
    F ss = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) ss += a[i] * a[i] + b[i] * b[i];
    F r;
    if constexpr (sizeof(F) == 8) r = 1.0 / sqrt(warp_sum_f64(ss) / D + eps);
    else r = 1.0f / sqrtf(warp_sum(ss) * (1.0f / D) + (float)eps);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      a[i] = a[i] * r * (F)__ldg(w + VPL * lane + i);
      b[i] = b[i] * r * (F)__ldg(w + D / 2 + VPL * lane + i);
    }
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if (cs) {
      const float2 t = __ldg(cs + VPL * lane + i);
      lo[i] = (float)(a[i] * (F)t.x - b[i] * (F)t.y);
      hi[i] = (float)(b[i] * (F)t.x + a[i] * (F)t.y);
    } else {
      lo[i] = (float)a[i];
      hi[i] = (float)b[i];
    }
  }
}

struct PutArgs {
  const void* qkv;
  int64_t T, qkv_stride;
  int Hq;
  const float* rope;
  int64_t rope_rows;
  const float *q_norm, *k_norm;
  double eps;
  void* q;
  int64_t q_stride;
  bool in_pairs, out_pairs;     // rows allow loads / stores of two values
  int q_bf16;
};

constexpr int kPutWarps = 8;

template <typename XT, int D, int KV>
__global__ void __launch_bounds__(32 * kPutWarps) k_kv_put(const KvView kv, const PutArgs a) {
  constexpr int VPL = D / 64;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  const int s = kv_sequence(kv, t);
  if (s < 0) return;                                   // behind the last sequence: left as it is
  const int64_t pos = kv_position(kv, s, t);
  bool ok = pos >= 0;
  int64_t page = -1;
  if (ok) {
    if (a.rope && pos >= a.rope_rows) {
      atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
      ok = false;
    } else {
      page = kv_page(kv, s, pos);
      ok = page >= 0;
    }
  }
  const float2* cs = a.rope && ok ? reinterpret_cast<const float2*>(a.rope) + pos * (D / 2) : nullptr;
  const int page_size = 1 << kv.page_shift, slot = (int)(pos & (page_size - 1));
  const int heads = a.Hq + 2 * kv.Hk;
  for (int h = blockIdx.y * kPutWarps + warp; h < heads; h += gridDim.y * kPutWarps) {
    const XT* x = (const XT*)a.qkv + t * a.qkv_stride + (int64_t)h * D;
    float lo[VPL], hi[VPL];
    load_vals<XT, VPL>(x + VPL * lane, a.in_pairs, lo);
    load_vals<XT, VPL>(x + D / 2 + VPL * lane, a.in_pairs, hi);
    if (h < a.Hq) {
      norm_rotate<float, D>(lo, hi, a.q_norm, a.eps, cs);
      if (!ok) {                                       // no position: a query of zeros
#pragma unroll
        for (int i = 0; i < VPL; ++i) lo[i] = hi[i] = 0.f;
      }
      const int64_t o = t * a.q_stride + (int64_t)h * D + VPL * lane;
      if (a.q_bf16) {
        store_vals<__nv_bfloat16, VPL>((__nv_bfloat16*)a.q + o, a.out_pairs, lo);
        store_vals<__nv_bfloat16, VPL>((__nv_bfloat16*)a.q + o + D / 2, a.out_pairs, hi);
      } else {
        store_vals<__half, VPL>((__half*)a.q + o, a.out_pairs, lo);
        store_vals<__half, VPL>((__half*)a.q + o + D / 2, a.out_pairs, hi);
      }
      continue;
    }
    if (!ok) continue;
    const bool is_v = h >= a.Hq + kv.Hk;
    const int hk = h - a.Hq - (is_v ? kv.Hk : 0);
    uint8_t* part = kv.pool + (page * kv.Hk + hk) * kv.head_bytes + (is_v ? kv.head_bytes / 2 : 0);
    if constexpr (KV == XM_KV_F16) {
      if (!is_v) norm_rotate<float, D>(lo, hi, a.k_norm, a.eps, cs);
      __half* row = (__half*)part + (int64_t)slot * D + VPL * lane;
      store_vals<__half, VPL>(row, true, lo);
      store_vals<__half, VPL>(row + D / 2, true, hi);
    } else {
      if (is_v) {
        put_half_q4<D, true>(lo, 0, part, page_size, slot);
        put_half_q4<D, true>(hi, 1, part, page_size, slot);
      } else {
        norm_rotate<double, D>(lo, hi, a.k_norm, a.eps, cs);
        put_half_q4<D, false>(lo, 0, part, page_size, slot);
        put_half_q4<D, false>(hi, 1, part, page_size, slot);
      }
    }
  }
}

// Reads the cached keys and values of the rows back as fp16 values [T][Hk][D]: one warp per (row, KV
// head, part); d (c - 8) is exact in fp32 and rounded once.
template <int D, int KV>
__global__ void __launch_bounds__(32 * kPutWarps) k_kv_get(const KvView kv, __half* __restrict__ k,
                                                           __half* __restrict__ v) {
  constexpr int VPL = D / 64, NG = D / 32;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  const int s = kv_sequence(kv, t);
  if (s < 0) return;
  const int64_t pos = kv_position(kv, s, t);
  const int64_t page = pos >= 0 ? kv_page(kv, s, pos) : -1;
  const int page_size = 1 << kv.page_shift, slot = (int)(pos & (page_size - 1));
  for (int h = blockIdx.y * kPutWarps + warp; h < 2 * kv.Hk; h += gridDim.y * kPutWarps) {
    const bool is_v = h >= kv.Hk;
    const int hk = is_v ? h - kv.Hk : h;
    __half* o = (is_v ? v : k) + (t * kv.Hk + hk) * D + VPL * lane;
    const uint8_t* part = kv.pool + (page * kv.Hk + hk) * kv.head_bytes + (is_v ? kv.head_bytes / 2 : 0);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float x[VPL];
#pragma unroll
      for (int i = 0; i < VPL; ++i) x[i] = 0.f;
      if (page >= 0) {
        if constexpr (KV == XM_KV_F16) {
          load_vals<__half, VPL>((const __half*)part + (int64_t)slot * D + half * (D / 2) + VPL * lane, true, x);
        } else {
          const int g = half * (NG / 2) + (VPL * lane) / 32, e = (VPL * lane) % 32;
          const uint8_t* row = part + (int64_t)slot * (D / 2);
          const uint32_t w = is_v ? (uint32_t)reinterpret_cast<const uint16_t*>(row)[NG * (e / 4) + g] >> (4 * (e % 4))
                                  : reinterpret_cast<const uint32_t*>(row)[NG * (e / 8) + g] >> (4 * (e % 8));
          const float d = __half2float(reinterpret_cast<const __half*>(part + (int64_t)page_size * (D / 2))[slot * NG + g]);
#pragma unroll
          for (int i = 0; i < VPL; ++i) x[i] = d * (float)((int)((w >> (4 * i)) & 15) - 8);
        }
      }
      store_vals<__half, VPL>(o + half * (D / 2), true, x);
    }
  }
}

}  // namespace

// Checks the cache arguments that every entry point takes and fills the view.
int kv_view(const char* who, void* pool, int64_t pages, int kv_type, int Hk, int head_dim, int page_size,
            const int* table, int64_t table_stride, int64_t table_width, const int* cu, const int* lens, int64_t B,
            KvView* out) {
  if (kv_type != XM_KV_F16 && kv_type != XM_KV_Q4_0)
    return xm_set_error(XM_ERR_UNSUPPORTED, "%s: unknown cache type %d", who, kv_type);
  if (head_dim != 64 && head_dim != 128)
    return xm_set_error(XM_ERR_UNSUPPORTED, "%s: head_dim %d (64 or 128)", who, head_dim);
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return xm_set_error(XM_ERR_INVALID, "%s: page size %d (a power of two from 16 to 1024)", who, page_size);
  if (Hk < 1 || Hk > 65535 || pages < 1 || pages > INT32_MAX || B < 1 || B > INT32_MAX || table_width < 1 ||
      table_width > (1 << 30) / page_size || table_stride < 0)
    return xm_set_error(XM_ERR_INVALID, "%s: bad cache sizes", who);
  if (!pool || !table || !lens) return xm_set_error(XM_ERR_INVALID, "%s: null pointer", who);
  if ((uintptr_t)pool & 15) return xm_set_error(XM_ERR_INVALID, "%s: the pool must be 16-byte aligned", who);
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  *out = KvView{(uint8_t*)pool, pages, 2 * kv_part_bytes(kv_type, head_dim, page_size), table, table_stride,
                (int)table_width, cu, lens, (int)B, Hk, shift};
  return XM_OK;
}

namespace {

template <typename... KArgs, typename... Args>
int launch_rows(const char* what, void (*kernel)(KArgs...), int64_t T, int heads, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  // few rows: one head per warp (latency); many: a row per CTA, its warps loop over the heads and reuse the
  // row's place and angles
  const unsigned gy = T >= 1024 ? 1u : (unsigned)((heads + kPutWarps - 1) / kPutWarps);
  cfg.gridDim = dim3((unsigned)T, gy);
  cfg.blockDim = dim3(32 * kPutWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return xm_check_launch(what);
}

template <typename XT>
int put_typed(const KvView& kv, const PutArgs& a, int kv_type, int head_dim, cudaStream_t st) {
  const int heads = a.Hq + 2 * kv.Hk;
  if (head_dim == 128)
    return kv_type == XM_KV_F16 ? launch_rows("kv append", k_kv_put<XT, 128, XM_KV_F16>, a.T, heads, st, kv, a)
                                : launch_rows("kv append", k_kv_put<XT, 128, XM_KV_Q4_0>, a.T, heads, st, kv, a);
  return kv_type == XM_KV_F16 ? launch_rows("kv append", k_kv_put<XT, 64, XM_KV_F16>, a.T, heads, st, kv, a)
                              : launch_rows("kv append", k_kv_put<XT, 64, XM_KV_Q4_0>, a.T, heads, st, kv, a);
}

}  // namespace

extern "C" {

int64_t xm_kv_page_bytes(int kv_type, int Hk, int head_dim, int page_size) {
  if ((kv_type != XM_KV_F16 && kv_type != XM_KV_Q4_0) || (head_dim != 64 && head_dim != 128) || Hk < 1 ||
      page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return 0;
  return 2 * Hk * kv_part_bytes(kv_type, head_dim, page_size);
}

int xm_kv_append(const void* d_qkv, int x_dtype, int64_t T, int64_t qkv_stride, int Hq, int Hk, int head_dim,
                 const float* d_rope, int64_t rope_rows, const float* d_q_norm, const float* d_k_norm, double eps,
                 void* d_pool, int64_t pages, int kv_type, int page_size, const int* d_table, int64_t table_stride,
                 int64_t table_width, const int* d_cu, const int* d_lens, int64_t B, void* d_q, int q_dtype,
                 int64_t q_stride, void* stream) {
  KvView kv;
  if (int rc = kv_view("kv_append", d_pool, pages, kv_type, Hk, head_dim, page_size, d_table, table_stride,
                       table_width, d_cu, d_lens, B, &kv))
    return rc;
  if (T < 0 || T > INT32_MAX || Hq < 1 || Hq > 65535 || Hq % Hk || (!d_cu && T != B))
    return xm_set_error(XM_ERR_INVALID, "kv_append: bad row or head counts (T = B where no row offsets are given)");
  if (x_dtype != XM_DT_F32 && x_dtype != XM_DT_F16 && x_dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "kv_append: bad element type %d", x_dtype);
  if (q_dtype != XM_DT_F16 && q_dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "kv_append: queries are fp16 or bf16, not type %d", q_dtype);
  if (T == 0) return XM_OK;
  if (!d_qkv || !d_q || (d_rope && rope_rows < 1)) return xm_set_error(XM_ERR_INVALID, "kv_append: null pointer");
  const int sz = x_dtype == XM_DT_F32 ? 4 : 2;
  if (qkv_stride < (int64_t)(Hq + 2 * Hk) * head_dim || q_stride < (int64_t)Hq * head_dim ||
      ((uintptr_t)d_qkv & (sz - 1)) || ((uintptr_t)d_q & 1) || ((uintptr_t)d_rope & 7) ||
      (((uintptr_t)d_q_norm | (uintptr_t)d_k_norm) & 3))
    return xm_set_error(XM_ERR_INVALID, "kv_append: bad row pitch or alignment");
  PutArgs a{d_qkv, T, qkv_stride, Hq, d_rope, rope_rows, d_q_norm, d_k_norm, eps, d_q, q_stride,
            qkv_stride % 2 == 0 && ((uintptr_t)d_qkv & (2 * sz - 1)) == 0,
            q_stride % 2 == 0 && ((uintptr_t)d_q & 3) == 0, q_dtype == XM_DT_BF16};
  cudaStream_t st = (cudaStream_t)stream;
  if (x_dtype == XM_DT_F32) return put_typed<float>(kv, a, kv_type, head_dim, st);
  if (x_dtype == XM_DT_F16) return put_typed<__half>(kv, a, kv_type, head_dim, st);
  return put_typed<__nv_bfloat16>(kv, a, kv_type, head_dim, st);
}

int xm_kv_read(const void* d_pool, int64_t pages, int kv_type, int Hk, int head_dim, int page_size,
               const int* d_table, int64_t table_stride, int64_t table_width, const int* d_cu, const int* d_lens,
               int64_t B, int64_t T, void* d_k, void* d_v, void* stream) {
  KvView kv;
  if (int rc = kv_view("kv_read", (void*)d_pool, pages, kv_type, Hk, head_dim, page_size, d_table, table_stride,
                       table_width, d_cu, d_lens, B, &kv))
    return rc;
  if (T < 0 || T > INT32_MAX || (!d_cu && T != B))
    return xm_set_error(XM_ERR_INVALID, "kv_read: bad row count (T = B where no row offsets are given)");
  if (T == 0) return XM_OK;
  if (!d_k || !d_v || (((uintptr_t)d_k | (uintptr_t)d_v) & 3))
    return xm_set_error(XM_ERR_INVALID, "kv_read: null or unaligned output");
  cudaStream_t st = (cudaStream_t)stream;
  if (head_dim == 128)
    return kv_type == XM_KV_F16
               ? launch_rows("kv read", k_kv_get<128, XM_KV_F16>, T, 2 * Hk, st, kv, (__half*)d_k, (__half*)d_v)
               : launch_rows("kv read", k_kv_get<128, XM_KV_Q4_0>, T, 2 * Hk, st, kv, (__half*)d_k, (__half*)d_v);
  return kv_type == XM_KV_F16
             ? launch_rows("kv read", k_kv_get<64, XM_KV_F16>, T, 2 * Hk, st, kv, (__half*)d_k, (__half*)d_v)
             : launch_rows("kv read", k_kv_get<64, XM_KV_Q4_0>, T, 2 * Hk, st, kv, (__half*)d_k, (__half*)d_v);
}

}  // extern "C"
