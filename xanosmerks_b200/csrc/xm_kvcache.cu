// Appending to and reading from the paged key/value cache (layout: xm_kv.cuh).
//
// k_kv_put: a query or key head x of D values is
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
// Bound: memory by the bytes for prompts, but eight prompts of up to 2048 tokens take 89 us (normalised heads, 4 bits; four
// CTAs an SM, 94 with three), nearly twice what the bytes do: issue slots 68 %, 35 % of the warps active, each with one head in
// flight.  Norms and rotations of keys in 64 bits and exact codes are a part of it: 76 without norms, 64 with an fp16 cache, 59
// with neither.  The read takes 19.  Single tokens: latency.  D / 8 lanes take a head, so a warp two heads
// of 128 or four of 64: lane l of them holds the values 4 l .. 4 l + 3 of each half, so the rotation
// needs no exchange, loads and stores are 8 or 16 bytes, and a block of 32 values is 8 lanes.  A
// block's codes are words of 2 lanes (keys) or halfwords of one (values).
#include <type_traits>

#include "xm_kv.cuh"

namespace {

constexpr int kPutWarps = 8;
constexpr unsigned kAll = 0xffffffffu;

// Q4_0 of the block held four values a lane by 8 neighbouring lanes: the lane's four codes as a halfword, d.
XM_DEV uint32_t q4_block(const float (&x)[4], __half& dh) {
  const int lane = threadIdx.x & 31;
  bool bad = false;
  float mag = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bad |= !(fabsf(x[i]) < INFINITY);
    mag = fmaxf(mag, fabsf(x[i]));
  }
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) mag = fmaxf(mag, __shfl_xor_sync(kAll, mag, o));
  const unsigned block = 0xffu << (lane & 24);
  const bool spoilt = __ballot_sync(kAll, bad) & block;
  bool mine = false;                                  // this lane holds a value of largest magnitude: its first
  float a = 0.f;
#pragma unroll
  for (int i = 3; i >= 0; --i)
    if (fabsf(x[i]) == mag) {
      mine = true;
      a = x[i];
    }
  const unsigned who = __ballot_sync(kAll, mine) & block;
  a = __shfl_sync(kAll, a, who ? __ffs(who) - 1 : lane);
  // a non-finite value spoils its block: d = NaN, every value of it reads as NaN
  dh = spoilt ? __ushort_as_half((unsigned short)0x7fff) : __float2half_rn(a * -0.125f);
  const float d = __half2float(dh), ad = fabsf(d);
  if (!(ad > 0.f && ad < INFINITY)) return 0x8888u;
  // x / d + 8 to the nearest whole number, by an approximate reciprocal and the addition of 2^23; within 1e-4 of a
  // border the exact comparisons decide
  const float inv = __fdividef(1.0f, d), magic = 8388608.f;
  float e[4];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float z = fminf(fmaxf(fmaf(x[i], inv, 8.f), 0.f), 15.f), t = z + magic;
    e[i] = t;
    near |= fabsf(z - (t - magic)) > 0.4999f;
  }
  if (__any_sync(__activemask(), near)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = d < 0.f ? -x[i] : x[i], c = e[i] - magic;
      if (c > 0.f && fmaf(8.5f - c, ad, y) < 0.f) e[i] -= 1.f;
      else if (c < 15.f && fmaf(7.5f - c, ad, y) >= 0.f) e[i] += 1.f;
    }
  }
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) codes |= (__float_as_uint(e[i]) & 15u) << (4 * i);
  return codes;
}

// Writes a head (lo, hi: this lane's values of its halves) as codes into row `slot` of a part, where `on`; every
// lane of the warp calls it.  values: the values' order of the codes instead of the keys'.
template <int D>
XM_DEV void put_q4(const float (&lo)[4], const float (&hi)[4], bool values, bool on, uint8_t* part, int page_size,
                   int slot) {
  constexpr int LPH = D / 8, NG = D / 32;
  const int l = threadIdx.x & (LPH - 1), n = l & 7;   // lane of the head; of its block
  __half d[2];
  uint32_t w[2] = {q4_block(lo, d[0]), q4_block(hi, d[1])};
#pragma unroll
  for (int h = 0; h < 2; ++h) {                       // keys: a word is the halfwords of two lanes
    const uint32_t o = __shfl_xor_sync(kAll, w[h], 1);
    if (!values) w[h] = l & 1 ? o | w[h] << 16 : w[h] | o << 16;
  }
  uint32_t s0 = (uint32_t)__half_as_ushort(d[0]) | (uint32_t)__half_as_ushort(d[1]) << 16;
  uint8_t* row = part + (int64_t)slot * (D / 2);
  uint8_t* scales = part + (int64_t)page_size * (D / 2) + slot * (2 * NG);
  if constexpr (NG == 4) {
    // lanes 0-7 hold blocks 0 and 2, lanes 8-15 blocks 1 and 3: the former take both
    const uint32_t o0 = __shfl_xor_sync(kAll, w[0], 8), o1 = __shfl_xor_sync(kAll, w[1], 8);
    const uint32_t o2 = __shfl_xor_sync(kAll, s0, 8);
    if (!on || l >= 8) return;
    if (values)
      *reinterpret_cast<uint2*>(row + 8 * n) = make_uint2(w[0] | o0 << 16, w[1] | o1 << 16);
    else if (!(n & 1))
      *reinterpret_cast<uint4*>(row + 8 * n) = make_uint4(w[0], o0, w[1], o1);
    if (n == 0)
      *reinterpret_cast<uint2*>(scales) = make_uint2((s0 & 0xffffu) | o2 << 16, s0 >> 16 | (o2 & 0xffff0000u));
  } else {
    if (!on) return;
    if (values)
      *reinterpret_cast<uint32_t*>(row + 4 * n) = w[0] | w[1] << 16;
    else if (!(n & 1))
      *reinterpret_cast<uint2*>(row + 4 * n) = make_uint2(w[0], w[1]);
    if (n == 0) *reinterpret_cast<uint32_t*>(scales) = s0;
  }
}

// four neighbouring values; `wide`: the rows allow one load (store)
template <typename XT>
XM_DEV void load4(const XT* p, bool wide, float (&v)[4]) {
  if (wide) {
    ld4f<XT>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = to_f32(p[i]);
  }
}
XM_DEV void store4(void* p, bool bf16, bool wide, const float (&v)[4]) {
  uint2 w;
  if (bf16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  }
  if (wide) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p);
    q[0] = (uint16_t)w.x; q[1] = (uint16_t)(w.x >> 16); q[2] = (uint16_t)w.y; q[3] = (uint16_t)(w.y >> 16);
  }
}

// Heads in arithmetic of type F: normalise (w: this lane's weights of the halves, where `norm`) and rotate (cs:
// (cos, sin) of the lane's four angles, where `turn`).  Every lane of the warp calls it.
template <typename F, int D>
XM_DEV void norm_rotate(float (&lo)[4], float (&hi)[4], bool norm, const float4& wl, const float4& wh, double eps,
                        bool turn, const float2 (&cs)[4]) {
  F a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[i] = (F)lo[i];
    b[i] = (F)hi[i];
  }
  if (__any_sync(kAll, norm)) {
    F ss = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kAll, ss, o);
    if (norm) {
      F r;
      if constexpr (sizeof(F) == 8) r = rsqrt(ss * (1.0 / D) + eps);
      else r = rsqrtf(ss * (1.0f / D) + (float)eps);
      const float l4[4] = {wl.x, wl.y, wl.z, wl.w}, h4[4] = {wh.x, wh.y, wh.z, wh.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = a[i] * r * (F)l4[i];
        b[i] = b[i] * r * (F)h4[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (turn) {
      lo[i] = (float)(a[i] * (F)cs[i].x - b[i] * (F)cs[i].y);
      hi[i] = (float)(b[i] * (F)cs[i].x + a[i] * (F)cs[i].y);
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
  bool in_wide, out_wide, norm_wide;      // rows allow loads / stores of four values
  bool q_bf16;
  int warps;                              // of a row (a power of two): a CTA takes kPutWarps / warps rows
};

template <typename XT, int D, int KV>
__global__ void __launch_bounds__(32 * kPutWarps, 4) k_kv_put(const KvView kv, const PutArgs a) {
  constexpr int LPH = D / 8, HPW = 32 / LPH;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane & (LPH - 1);
  const int64_t t = (int64_t)blockIdx.x * (kPutWarps / a.warps) + warp / a.warps;
  if (t >= a.T) return;
  const int part_of = blockIdx.y * a.warps + (warp & (a.warps - 1));
  const int heads = a.Hq + 2 * kv.Hk, step = gridDim.y * a.warps * HPW;
  int h = part_of * HPW + lane / LPH;
  const XT* x = (const XT*)a.qkv + t * a.qkv_stride + 4 * l;
  // the first head's values start on their way before the row's place is known
  float lo[4] = {}, hi[4] = {};
  if (h < heads) {
    load4<XT>(x + (int64_t)h * D, a.in_wide, lo);
    load4<XT>(x + (int64_t)h * D + D / 2, a.in_wide, hi);
  }
  const KvPlace at = kv_place(kv, t);
  if (at.seq < 0) return;                              // behind the last sequence: left as it is
  const int64_t pos = at.pos;
  bool ok = pos >= 0;
  int64_t page = -1;
  if (ok) {
    if (a.rope && pos >= a.rope_rows) {
      atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
      ok = false;
    } else {
      page = kv_page(kv, at.seq, pos);
      ok = page >= 0;
    }
  }
  float2 cs[4];
  const bool turn = a.rope && ok;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    cs[i] = turn ? __ldg(reinterpret_cast<const float2*>(a.rope) + pos * (D / 2) + 4 * l + i) : make_float2(1.f, 0.f);
  const int page_size = 1 << kv.page_shift, slot = (int)(pos & (page_size - 1));
  for (int first = part_of * HPW; first < heads; first += step) {
    float nlo[4] = {}, nhi[4] = {};                    // the next heads load while these are worked on
    if (h + step < heads) {
      load4<XT>(x + (int64_t)(h + step) * D, a.in_wide, nlo);
      load4<XT>(x + (int64_t)(h + step) * D + D / 2, a.in_wide, nhi);
    }
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + kv.Hk;
    const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    float4 wl = make_float4(0.f, 0.f, 0.f, 0.f), wh = wl;
    if (w) {
      if (a.norm_wide) {
        wl = __ldg(reinterpret_cast<const float4*>(w) + l);
        wh = __ldg(reinterpret_cast<const float4*>(w + D / 2) + l);
      } else {
        wl = make_float4(w[4 * l], w[4 * l + 1], w[4 * l + 2], w[4 * l + 3]);
        wh = make_float4(w[D / 2 + 4 * l], w[D / 2 + 4 * l + 1], w[D / 2 + 4 * l + 2], w[D / 2 + 4 * l + 3]);
      }
    }
    const bool exact = KV == XM_KV_Q4_0 && !is_q && !is_v && h < heads;
    if (!__any_sync(kAll, exact)) {
      norm_rotate<float, D>(lo, hi, w != nullptr, wl, wh, a.eps, turn && !is_v, cs);
    } else {
      float l2[4] = {lo[0], lo[1], lo[2], lo[3]}, h2[4] = {hi[0], hi[1], hi[2], hi[3]};
      norm_rotate<double, D>(l2, h2, exact && w != nullptr, wl, wh, a.eps, turn, cs);
      // (a warp has heads of several kinds only where their counts are odd)
      if (!__all_sync(kAll, exact)) norm_rotate<float, D>(lo, hi, !exact && w != nullptr, wl, wh, a.eps, turn && !is_v, cs);
      if (exact) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = l2[i];
          hi[i] = h2[i];
        }
      }
    }
    if (is_q) {
      if (!ok) {                                       // no position: a query of zeros
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = hi[i] = 0.f;
      }
      uint16_t* o = (uint16_t*)a.q + t * a.q_stride + (int64_t)h * D + 4 * l;
      store4(o, a.q_bf16, a.out_wide, lo);
      store4(o + D / 2, a.q_bf16, a.out_wide, hi);
    }
    const bool store = !is_q && ok && h < heads;
    const int hk = is_v ? h - a.Hq - kv.Hk : h - a.Hq;
    uint8_t* part = kv.pool + (store ? (page * kv.Hk + hk) * kv.head_bytes + (is_v ? kv.head_bytes / 2 : 0) : 0);
    if constexpr (KV == XM_KV_F16) {
      if (store) {
        __half* row = (__half*)part + (int64_t)slot * D + 4 * l;
        store4(row, false, true, lo);
        store4(row + D / 2, false, true, hi);
      }
    } else {
      if (__any_sync(kAll, store)) put_q4<D>(lo, hi, is_v, store, part, page_size, slot);
    }
    h += step;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = nlo[i];
      hi[i] = nhi[i];
    }
  }
}

// Reads the cached keys and values of the rows back as fp16 values [T][Hk][D]: a lane eight neighbouring values of
// a head, one word of codes (keys) or two halfwords (values); d (c - 8) is exact in fp32 and rounded once.
template <int D, int KV>
__global__ void __launch_bounds__(32 * kPutWarps) k_kv_get(const KvView kv, __half* __restrict__ k,
                                                           __half* __restrict__ v, bool wide, int64_t T, int warps) {
  constexpr int LPH = D / 8, HPW = 32 / LPH, NG = D / 32;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane & (LPH - 1);
  const int64_t t = (int64_t)blockIdx.x * (kPutWarps / warps) + warp / warps;
  if (t >= T) return;
  const KvPlace at = kv_place(kv, t);
  if (at.seq < 0) return;
  const int64_t pos = at.pos, page = pos >= 0 ? kv_page(kv, at.seq, pos) : -1;
  const int page_size = 1 << kv.page_shift, slot = (int)(pos & (page_size - 1));
  const int g = c >> 2, e = c & 3;                     // block of the eight values, which eighths of it
  for (int h = (blockIdx.y * warps + (warp & (warps - 1))) * HPW + lane / LPH; h < 2 * kv.Hk; h += gridDim.y * warps * HPW) {
    const bool is_v = h >= kv.Hk;
    const int hk = is_v ? h - kv.Hk : h;
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (page >= 0) {
      const uint8_t* part = kv.pool + (page * kv.Hk + hk) * kv.head_bytes + (is_v ? kv.head_bytes / 2 : 0);
      if constexpr (KV == XM_KV_F16) {
        o = __ldg(reinterpret_cast<const uint4*>(part + (int64_t)slot * (2 * D)) + c);
      } else {
        const uint8_t* row = part + (int64_t)slot * (D / 2);
        uint32_t w;
        if (is_v) {
          const uint16_t* hw = reinterpret_cast<const uint16_t*>(row) + NG * (2 * e) + g;
          w = (uint32_t)__ldg(hw) | (uint32_t)__ldg(hw + NG) << 16;
        } else {
          w = __ldg(reinterpret_cast<const uint32_t*>(row) + NG * e + g);
        }
        const float d = __half2float(reinterpret_cast<const __half*>(part + (int64_t)page_size * (D / 2))[slot * NG + g]);
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = d * i2f_small((int)((w >> (4 * i)) & 15) - 8);
        __half2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        o = *reinterpret_cast<const uint4*>(p);
      }
    }
    __half* to = (is_v ? v : k) + (t * kv.Hk + hk) * D + 8 * c;
    if (wide) {
      *reinterpret_cast<uint4*>(to) = o;
    } else {
      const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(to)[i] = w[i];
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
  if (((uintptr_t)table | (uintptr_t)cu | (uintptr_t)lens) & 3)
    return xm_set_error(XM_ERR_INVALID, "%s: unaligned page table, offsets or lengths", who);
  int shift = 0;
  while ((1 << shift) < page_size) ++shift;
  *out = KvView{(uint8_t*)pool, pages, 2 * kv_part_bytes(kv_type, head_dim, page_size), table, table_stride,
                (int)table_width, cu, lens, (int)B, Hk, shift};
  return XM_OK;
}

namespace {

// Warps of a row: few rows: as many as its heads need, over several CTAs (latency); many: two, so that finding a
// row's place is paid for by half of its heads (8800 rows of 48 heads: see k_kv_put).
struct RowGrid {
  dim3 grid;
  int warps;
};
RowGrid row_grid(int64_t T, int heads, int D) {
  const int per_warp = 256 / D, need = (heads + per_warp - 1) / per_warp;
  if (T >= 1024) return {dim3((unsigned)((T + kPutWarps / 2 - 1) / (kPutWarps / 2))), 2};
  return {dim3((unsigned)T, (unsigned)((need + kPutWarps - 1) / kPutWarps)), kPutWarps};
}

template <typename... KArgs, typename... Args>
int launch_rows(const char* what, void (*kernel)(KArgs...), const RowGrid& g, cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = g.grid;
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
int put_typed(const KvView& kv, PutArgs a, int kv_type, int head_dim, cudaStream_t st) {
  const RowGrid g = row_grid(a.T, a.Hq + 2 * kv.Hk, head_dim);
  a.warps = g.warps;
  if (head_dim == 128)
    return kv_type == XM_KV_F16 ? launch_rows("kv append", k_kv_put<XT, 128, XM_KV_F16>, g, st, kv, a)
                                : launch_rows("kv append", k_kv_put<XT, 128, XM_KV_Q4_0>, g, st, kv, a);
  return kv_type == XM_KV_F16 ? launch_rows("kv append", k_kv_put<XT, 64, XM_KV_F16>, g, st, kv, a)
                              : launch_rows("kv append", k_kv_put<XT, 64, XM_KV_Q4_0>, g, st, kv, a);
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
            qkv_stride % 4 == 0 && ((uintptr_t)d_qkv & (4 * sz - 1)) == 0,
            q_stride % 4 == 0 && ((uintptr_t)d_q & 7) == 0, (((uintptr_t)d_q_norm | (uintptr_t)d_k_norm) & 15) == 0,
            q_dtype == XM_DT_BF16, 0};
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
  const RowGrid g = row_grid(T, 2 * Hk, head_dim);
  const bool wide = (((uintptr_t)d_k | (uintptr_t)d_v) & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (head_dim == 128)
    return kv_type == XM_KV_F16
               ? launch_rows("kv read", k_kv_get<128, XM_KV_F16>, g, st, kv, (__half*)d_k, (__half*)d_v, wide, T, g.warps)
               : launch_rows("kv read", k_kv_get<128, XM_KV_Q4_0>, g, st, kv, (__half*)d_k, (__half*)d_v, wide, T, g.warps);
  return kv_type == XM_KV_F16
             ? launch_rows("kv read", k_kv_get<64, XM_KV_F16>, g, st, kv, (__half*)d_k, (__half*)d_v, wide, T, g.warps)
             : launch_rows("kv read", k_kv_get<64, XM_KV_Q4_0>, g, st, kv, (__half*)d_k, (__half*)d_v, wide, T, g.warps);
}

}  // extern "C"
