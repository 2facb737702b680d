// Attention over the paged key/value cache (layout: xm_kv.cuh).
//
// Row t of sequence s at position p sees the keys 0 .. p of its sequence (with a window w: those above
// p - w, and the first `sinks`); query head h reads KV head h / (Hq / Hk):
//   out = sum_k softmax_k(q . K_k * scale) V_k,  zeros for a row that sees no key.
//
// k_kv_attn: one warp per (row, query head), one pass over the keys with a running maximum and sum;
// lane l holds values 2l, 2l + 1 of each half of the head (one per half at D = 64).
#include <algorithm>
#include <type_traits>

#include "xm_kv.cuh"

int kv_view(const char* who, void* pool, int64_t pages, int kv_type, int Hk, int head_dim, int page_size,
            const int* table, int64_t table_stride, int64_t table_width, const int* cu, const int* lens, int64_t B,
            KvView* out);

namespace {

struct AttnArgs {
  const void* q;
  int64_t T, q_stride;
  int Hq;
  float scale;
  int window, sinks;       // at most 2^30, the largest context
  void* out;
  int64_t out_stride;
  bool q_vec, out_vec;    // rows of q allow loads of 16 bytes, rows of out stores of four values
};

constexpr int kAttnWarps = 8;

// value i of half `half` of lane's values of a cached row
template <int D, int KV>
XM_DEV float kv_value(const uint8_t* part, int page_size, int slot, bool is_v, int half, int i) {
  constexpr int VPL = D / 64, NG = D / 32;
  const int lane = threadIdx.x & 31;
  if constexpr (KV == XM_KV_F16) {
    return __half2float(((const __half*)part)[(int64_t)slot * D + half * (D / 2) + VPL * lane + i]);
  } else {
    const int g = half * (NG / 2) + (VPL * lane + i) / 32, e = (VPL * lane + i) % 32;
    const uint8_t* row = part + (int64_t)slot * (D / 2);
    const uint32_t w = is_v ? (uint32_t)reinterpret_cast<const uint16_t*>(row)[NG * (e / 4) + g] >> (4 * (e % 4))
                            : reinterpret_cast<const uint32_t*>(row)[NG * (e / 8) + g] >> (4 * (e % 8));
    const float d = __half2float(reinterpret_cast<const __half*>(part + (int64_t)page_size * (D / 2))[slot * NG + g]);
    return d * (float)((int)(w & 15) - 8);
  }
}

template <typename QT_, int D, int KV>
__global__ void __launch_bounds__(32 * kAttnWarps) k_kv_attn(const KvView kv, const AttnArgs a) {
  constexpr int VPL = D / 64;
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y * kAttnWarps + (threadIdx.x >> 5);
  const int s = kv_sequence(kv, t);
  if (s < 0 || h >= a.Hq) return;
  const int64_t pos = kv_position(kv, s, t);
  const int hk = h / (a.Hq / kv.Hk);
  const int page_size = 1 << kv.page_shift;
  const QT_* q = (const QT_*)a.q + t * a.q_stride + (int64_t)h * D;
  float qv[2][VPL], o[2][VPL];
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      qv[half][i] = to_f32(q[half * (D / 2) + VPL * lane + i]) * a.scale;
      o[half][i] = 0.f;
    }
  float m = -INFINITY, l = 0.f;
  for (int64_t key = 0; key <= pos; ++key) {
    if (a.window > 0 && key <= pos - a.window && key >= a.sinks) {
      key = pos - a.window;
      continue;
    }
    const int64_t page = kv_page(kv, s, key);
    if (page < 0) continue;
    const uint8_t* part = kv.pool + (page * kv.Hk + hk) * kv.head_bytes;
    const int slot = (int)(key & (page_size - 1));
    float dot = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < VPL; ++i) dot = fmaf(qv[half][i], kv_value<D, KV>(part, page_size, slot, false, half, i), dot);
    dot = warp_sum(dot);
    const float n = fmaxf(m, dot);
    const float f = m == n ? 1.f : expf(m - n), p = dot == n ? 1.f : expf(dot - n);
    m = n;
    l = fmaf(l, f, p);
    const uint8_t* vpart = part + kv.head_bytes / 2;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        o[half][i] = fmaf(o[half][i], f, p * kv_value<D, KV>(vpart, page_size, slot, true, half, i));
  }
  const float inv = l > 0.f ? 1.0f / l : (l == 0.f ? 0.f : l);
  QT_* out = (QT_*)a.out + t * a.out_stride + (int64_t)h * D;
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const float v = o[half][i] * inv;
      if constexpr (std::is_same<QT_, __half>::value) out[half * (D / 2) + VPL * lane + i] = __float2half_rn(v);
      else out[half * (D / 2) + VPL * lane + i] = __float2bfloat16_rn(v);
    }
}

// ---------------------------------------------------------------------------
// Decode: up to 8 NT rows (token, query head) of one KV head of one sequence per CTA; the keys are
// split over the warps of a CTA, and over CTAs in chunks of `chunk` keys whose partial softmaxes
// k_kv_merge joins.
//
// Bound: memory (the cache is read once); the work per byte decides whether that is reached.  A warp
// takes 16 keys at a time on mma.sync m16n8k16 (fp16 operands, fp32 sums) with the keys, or the
// values' dimensions, as the 16 matrix rows and the query rows as the 8 columns:
//   S^T [16 keys x 8 rows] = K q^T,   O^T [D x 8 rows] += V^T P^T.
// Operands come from global memory straight into the fragments: the order of the products' inner
// dimension is free, and the cache's layout was chosen for it.
//
// 4-bit rows are never unpacked to values.  The nibbles 0 and 4 (for keys; 0 of two keys, paired by a
// byte permute, for values) of a word are, after one mask, two fp16 subnormals c 2^-24, the nibbles
// 1 and 5 are c 2^-20: exact, one instruction for two codes.  For values whole bytes (c + 16 c') 2^-24 and
// their high nibbles enter, one instruction less, and the low codes' sums are the difference at the end.  The block scale and the offset of the
// codes stay outside the product:
//   S  = sum over blocks b of d_kb (sum_i q_i c_i - 8 sum_i q_i)       (the offset is the product's
//        initial accumulator),
//   O  = sum_k c_k (p_k d_kb) - 8 sum_k p_k d_kb                       (one more product with constants).
// q is scaled by a power of two per row into fp16's range (exact for fp16 and nearly so for bf16).
// p d is rounded to fp16 once (2^-11); so that it neither overflows nor vanishes whatever the scales
// are, the running reference R of a row is the largest s + log2 of the tile's largest |d|, less 13.
//
// A key behind the mask takes no part whatever its bytes are: its score and its p d are selected
// away, not multiplied by zero.
// ---------------------------------------------------------------------------

constexpr int kDecWarps = 4;
constexpr int kMaxSplits = 128;     // one per thread of the merge

XM_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
XM_DEV uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
XM_DEV void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
XM_DEV void mma_16816_from(float (&d)[4], float c0, float c1, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                           uint32_t b0, uint32_t b1) {   // d = a b + (c0, c1) in both halves of the rows
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
// transposes an 8 x 8 matrix of 16-bit values held two per lane (row lane / 4, columns 2 (lane % 4), + 1)
XM_DEV uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <int W>
XM_DEV void lds_words(uint32_t (&w)[W], uint32_t at) {
  if constexpr (W == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at));
  else if constexpr (W == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(at));
}
// 16 bytes from global to shared memory, asynchronously
XM_DEV void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
XM_DEV float half_of(uint32_t w, int hi) {
  const __half2 h = *reinterpret_cast<const __half2*>(&w);
  return hi ? __high2float(h) : __low2float(h);
}

// Rows [r0, r0 + R) of (token, query head) pairs of one sequence, and the keys that any of them sees:
// units of UK keys, first the ones that hold sinks, then a run up to the last row's position.
struct TileSpan {
  int s, rows;            // sequence; valid rows
  int64_t t0;             // row of the sequence's first new token
  int r0;
  int p_first;            // position of the sequence's first new token
  int pmin, pmax;         // positions of the tile's first and last token
  int ns, a0, n;          // sink units; first unit of the run; units in all
  bool past_table;        // positions past the page table were asked for
  XM_DEV int unit(int v) const { return v < ns ? v : v - ns + a0; }
};

template <int R, int UK>
XM_DEV TileSpan tile_span(const KvView& kv, const AttnArgs& a, int s, int64_t t0, int q_len, int rt, int G) {
  TileSpan x;
  x.s = s;
  x.t0 = t0;
  x.r0 = rt * R;
  x.rows = min(R, q_len * G - x.r0);
  const int len = __ldg(kv.lens + s);
  x.p_first = len - q_len;
  x.pmin = x.p_first + x.r0 / G;
  x.pmax = x.p_first + (x.r0 + x.rows - 1) / G;
  const int64_t cap = (int64_t)kv.table_width << kv.page_shift;
  x.past_table = (int64_t)x.pmax >= cap;
  const int kend = (int)min((int64_t)x.pmax + 1, cap);
  int lo = 0, se = 0;
  if (a.window > 0) {
    lo = max(0, x.pmin - a.window + 1);
    se = min(a.sinks, lo);
  }
  x.a0 = lo / UK;
  x.ns = min((se + UK - 1) / UK, x.a0);
  x.n = kend > 0 ? x.ns + max(0, (kend + UK - 1) / UK - x.a0) : 0;
  return x;
}

XM_DEV bool sees(const AttnArgs& a, int pos, int key) {
  return key <= pos && (a.window == 0 || key > pos - a.window || key < a.sinks);
}

// The rows of sequence s among the call's T, [t0, t0 + q_len) (none of them outside the call, whatever
// the offsets say).
XM_DEV void sequence_rows(const KvView& kv, int64_t T, int s, int64_t& t0, int& q_len) {
  if (!kv.cu) {
    t0 = s;
    q_len = 1;
    return;
  }
  const int first = max(0, min(__ldg(kv.cu + s), (int)T));
  t0 = first;
  q_len = max(0, min(__ldg(kv.cu + s + 1), (int)T) - first);
}

// The tile x of row tiles of R rows over all sequences: its sequence, or -1.  Every thread of the
// warp calls it.
template <int R>
XM_DEV int find_tile(const KvView& kv, int64_t T, int G, int x, int& rt, int64_t& t0, int& q_len) {
  if (!kv.cu) {
    const int per = (G + R - 1) / R;
    const int s = x / per;
    rt = x % per;
    t0 = s;
    q_len = 1;
    return s < kv.B ? s : -1;
  }
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int s0 = 0; s0 < kv.B; s0 += 32) {
    const int s = s0 + lane;
    int64_t first = 0;
    int len = 0;
    if (s < kv.B) sequence_rows(kv, T, s, first, len);
    const int tiles = (int)(((int64_t)len * G + R - 1) / R);
    int c = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int n = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += n;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + c > x);
    if (hit) {
      const int l = __ffs(hit) - 1;
      rt = x - (before + __shfl_sync(0xffffffffu, c - tiles, l));
      t0 = __shfl_sync(0xffffffffu, first, l);
      q_len = __shfl_sync(0xffffffffu, len, l);
      return s0 + l;
    }
    before += __shfl_sync(0xffffffffu, c, 31);
  }
  return -1;
}

// One subtile (16 keys) in a warp's part of shared memory: copied there 16 bytes at a time, and read
// from there as fragments without bank conflicts.  Matrix row i of the keys, and inner index i of the
// values' product, is key key_of(i) of the subtile, so that the four keys that a quarter of the lanes
// reads together are four neighbours, whose pieces a small permutation spreads over the banks.
XM_DEV int key_of(int i) { return (i & 8) | (i & 1) << 2 | (i & 6) >> 1; }

template <int KV, int D>
struct SubTile;
template <int D>
struct SubTile<XM_KV_Q4_0, D> {
  static constexpr int NG = D / 32, ROW = D / 2, P = ROW / 16;     // bytes and 16-byte pieces of a row of codes
  static constexpr int kVAt = 16 * ROW, kKd = 2 * kVAt, kVd = kKd + 32 * NG, kBytes = kVd + 32 * NG;
  uint32_t k[2][NG], v[4][NG / 2], kd[2][NG / 2], kx[2], vd[2][NG / 2];
  // `to`: the subtile in shared memory; `from`: its first key row; `scales`: its first key's scales
  static XM_DEV void copy(uint32_t to, const uint8_t* from, const uint8_t* scales, int64_t v_part, int lane) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      const int c = lane + 32 * i, key = c / P, piece = c % P;
      const int row = (key & 8) | (key & 3) << 1 | (key >> 2 & 1);               // key_of(row) = key
      copy16(to + row * ROW + piece * 16, from + c * 16);
      copy16(to + kVAt + key * ROW + (P == 4 ? piece ^ (key & 2) : piece) * 16, from + v_part + c * 16);
    }
    if (lane < 4 * NG) {
      const int c = lane % (2 * NG), vals = lane / (2 * NG);
      copy16(to + kKd + vals * 32 * NG + c * 16, scales + vals * v_part + c * 16);
    }
  }
  XM_DEV void read_k(uint32_t at, int r, int kq) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lds_words<NG>(k[i], at + r * ROW + kq * (NG * 4) + 8 * i * ROW);
      lds_words<NG / 2>(kd[i], at + kKd + key_of(r) * (2 * NG) + 8 * i * (2 * NG));
      uint32_t x[1] = {0u};                            // the scales of blocks 2 kq, 2 kq + 1
      if (kq < NG / 2) lds_words<1>(x, at + kKd + key_of(r) * (2 * NG) + kq * 4 + 8 * i * (2 * NG));
      kx[i] = x[0];
    }
  }
  XM_DEV void read_v(uint32_t at, int r, int kq) {
#pragma unroll
    for (int i = 0; i < 4; ++i)     // keys kq, kq + 4, kq + 8, kq + 12
      lds_words<NG / 2>(v[i], at + kVAt + kq * ROW + (P == 4 ? (r * 8) ^ (kq & 2) << 4 : r * 4) + 4 * i * ROW);
  }
  XM_DEV void read_vd(uint32_t at, int r) {
#pragma unroll
    for (int i = 0; i < 2; ++i) lds_words<NG / 2>(vd[i], at + kVd + key_of(r) * (2 * NG) + 8 * i * (2 * NG));
  }
};
template <int D>
struct SubTile<XM_KV_F16, D> {
  static constexpr int ROW = 2 * D, P = ROW / 16;                  // 16-byte pieces of a row
  static constexpr int KC = D / 32, VC = D / 64;                   // pieces of a key (per lane) and of a value
  static constexpr int kVAt = 16 * ROW, kBytes = 2 * kVAt;
  uint32_t k[2][KC][4], v[4][VC][4];
  static XM_DEV void copy(uint32_t to, const uint8_t* from, const uint8_t*, int64_t v_part, int lane) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      const int c = lane + 32 * i, key = c / P, piece = c % P;
      copy16(to + key * ROW + (piece ^ (key & 4)) * 16, from + c * 16);
      copy16(to + kVAt + key * ROW + (piece ^ (key & 3) << 1) * 16, from + v_part + c * 16);
    }
  }
  XM_DEV void read_k(uint32_t at, int r, int kq) {
    const int key = key_of(r);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c) lds_words<4>(k[i][c], at + (key + 8 * i) * ROW + ((4 * c + kq) ^ (key & 4)) * 16);
  }
  XM_DEV void read_v(uint32_t at, int r, int kq) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < VC; ++c) lds_words<4>(v[i][c], at + kVAt + (kq + 4 * i) * ROW + (8 * c + (r ^ kq << 1)) * 16);
  }
};

XM_DEV bool non_finite(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }

struct DecArgs {
  int chunk;                // units of a CTA
  int nsplit;
  float* part_o;            // [nsplit][T][Hq][D], where a row has more than one part
  float2* part_ml;
};

template <typename QT_>
XM_DEV void put_out4(QT_* p, bool vec, float4 v) {
  uint2 w;
  if constexpr (std::is_same<QT_, __half>::value) {
    w = make_uint2(half2_bits(v.x, v.y), half2_bits(v.z, v.w));
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    w = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  }
  if (vec) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p);
    q[0] = (uint16_t)w.x; q[1] = (uint16_t)(w.x >> 16); q[2] = (uint16_t)w.y; q[3] = (uint16_t)(w.y >> 16);
  }
}

// Subtiles of a warp at a time, and such steps in a warp's ring (copies for the next ones are in flight
// while one is used).
template <int KV, int D, int NT>
struct DecShape {
  static constexpr int SUB = KV == XM_KV_Q4_0 ? 2 : 1, STAGES = KV == XM_KV_Q4_0 ? 2 : 3;
  static constexpr int kRing = STAGES * SUB * SubTile<KV, D>::kBytes;                       // bytes of a warp
  static constexpr int kJoin = kDecWarps * 8 * NT * ((D + 4) * 4 + 8);                      // reuses the ring
  static constexpr int kQ = NT * (D / 32 * 2 * 256 + 4 * 128);                              // q fragments, q_f, q_off
  static constexpr int kSmem = kQ + (kDecWarps * kRing > kJoin ? kDecWarps * kRing : kJoin);
  static constexpr int kCtas = NT > 1 ? 2 : KV == XM_KV_Q4_0 || D == 64 ? 3 : 2;          // of an SM
};

template <typename QT_, int D, int KV, int NT>
__global__ void __launch_bounds__(32 * kDecWarps, DecShape<KV, D, NT>::kCtas) k_kv_decode(const KvView kv,
                                                                                          const AttnArgs a,
                                                                                          const DecArgs da) {
  using Sub = SubTile<KV, D>;
  using Shape = DecShape<KV, D, NT>;
  constexpr int R = 8 * NT, NG = D / 32, DP = D + 4, SUB = Shape::SUB, STAGES = Shape::STAGES, UK = 16 * SUB;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ __align__(16) uint8_t dec_smem[];
  grid_dep_wait();
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, kq = lane & 3;
  const int G = a.Hq / kv.Hk, hk = blockIdx.x % kv.Hk, split = blockIdx.y;
  int rt, q_len;
  int64_t t0;
  const int s = find_tile<R>(kv, a.T, G, blockIdx.x / kv.Hk, rt, t0, q_len);
  if (s < 0) return;
  const TileSpan ts = tile_span<R, UK>(kv, a, s, t0, q_len, rt, G);
  if (ts.past_table && threadIdx.x == 0) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
  const int parts = (ts.n + da.chunk - 1) / da.chunk;
  if (split > 0 && split >= parts) return;
  const int v_lo = split * da.chunk, v_hi = min(ts.n, v_lo + da.chunk);

  // this lane's columns: rows 2 kq, 2 kq + 1 of every 8
  int pos[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) pos[nt][c] = ts.p_first + min(ts.r0 + 8 * nt + 2 * kq + c, ts.r0 + ts.rows - 1) / G;

  float o[NT][D / 16][4], off[NT][NG][4], R_[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) off[nt][g][0] = off[nt][g][1] = off[nt][g][2] = off[nt][g][3] = 0.f;
    R_[nt][0] = R_[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }

  const int page_mask = (1 << kv.page_shift) - 1;
  const bool one_page = UK == 16 || kv.page_shift >= 5;   // a unit lies in one page (or in two of 16 tokens)
  const int* table = kv.table + (int64_t)s * kv.table_stride;
  const uint8_t* pool = kv.pool + (int64_t)hk * kv.head_bytes;
  const int64_t page_bytes = kv.head_bytes * kv.Hk, v_part = kv.head_bytes / 2;
  const int codes = D / 2 << kv.page_shift;            // 4-bit: bytes of codes in front of the scales
  const int steps = max(0, (v_hi - v_lo - warp + kDecWarps - 1) / kDecWarps);
  const uint32_t ring = smem_u32(dec_smem) + warp * Shape::kRing;

  // q's bytes start on their way before anything else: warp nt takes row 8 nt + r, values 32 g + 8 kq ...
  uint4 q_raw[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) q_raw[g] = make_uint4(0u, 0u, 0u, 0u);
  if (warp < NT && 8 * warp + r < ts.rows) {
    const int gr = ts.r0 + 8 * warp + r;
    const QT_* q = (const QT_*)a.q + (t0 + gr / G) * a.q_stride + (int64_t)(hk * G + gr % G) * D + 8 * kq;
    if (a.q_vec) {
#pragma unroll
      for (int g = 0; g < NG; ++g) q_raw[g] = __ldg(reinterpret_cast<const uint4*>(q + 32 * g));
    } else {
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<QT_*>(&q_raw[g])[i] = q[32 * g + i];
    }
  }

  // the warp's units are v_lo + warp + 4 i; lane l holds the page(s) of i = 32 b + l
  auto page_of = [&](int i, int j) {
    if (i >= steps) return 0;
    const int at = ts.unit(v_lo + warp + i * kDecWarps) * UK + 16 * j >> kv.page_shift;
    return at < kv.table_width ? __ldg(table + at) : -1;
  };
  int pages = page_of(lane, 0), pages_next = steps > 32 ? page_of(32 + lane, 0) : 0;
  unsigned bad_steps = 0;                              // bit i: the step i % 32 has a page outside the pool
  auto fetch = [&](int i) {                            // starts the copies of step i
    if (i < steps) {
      if (i > 0 && (i & 31) == 0) {
        pages = pages_next;
        pages_next = page_of(i + 32 + lane, 0);
      }
      const int key0 = ts.unit(v_lo + warp + i * kDecWarps) * UK;
      bad_steps &= ~(1u << (i & 31));
      const uint8_t* head;
      const uint32_t to = ring + i % STAGES * (SUB * Sub::kBytes);
#pragma unroll
      for (int j = 0; j < SUB; ++j) {
        if (j == 0 || !one_page) {
          int p = __shfl_sync(0xffffffffu, pages, i & 31);
          if (j > 0) p = page_of(i, j);
          const bool in = (unsigned)p < (unsigned)kv.pages;
          if (!in && (j == 0 || key0 + 16 * j <= ts.pmax)) bad_steps |= 1u << (i & 31);
          head = pool + (in ? p : 0) * page_bytes;
        }
        const int slot = key0 + 16 * j & page_mask;
        Sub::copy(to + j * Sub::kBytes, head + slot * Sub::ROW, head + codes + slot * (2 * NG), v_part, lane);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(i);

  // q, by warp nt for all of them: row 8 nt + r, scaled by a power of two into fp16
  const uint32_t q_at = smem_u32(dec_smem) + kDecWarps * Shape::kRing;
  const uint32_t qb_at = q_at + lane * 16, qx_at = q_at + NT * NG * 2 * 256 + lane * 16;
  if (warp < NT) {
    const int nt = warp;
    uint32_t qb[NG][2][2], q_off[2] = {0u, 0u};        // 4-bit: -8 sum of a block's q, as high and low halves
    float q_f[2];                                      // what turns a column's sum into a base-2 score
    float x[NG][8];
    float mx = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) x[g][i] = to_f32(reinterpret_cast<const QT_*>(&q_raw[g])[i]);
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[g][i]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const int sh = fp16_row_shift(mx);
    const float down = a.scale < 0.f ? -ldexpf(1.f, -sh) : ldexpf(1.f, -sh);
    const float f = ldexpf(fabsf(a.scale) * kLog2e, sh + (KV == XM_KV_Q4_0 ? 24 : 0));
    float block[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[g][i] = __half2float(__float2half_rn(x[g][i] * down));
        sum += x[g][i];
      }
      if constexpr (KV == XM_KV_Q4_0) {
        qb[g][0][0] = half2_bits(x[g][0], x[g][4]);
        qb[g][0][1] = half2_bits(x[g][2], x[g][6]);
        qb[g][1][0] = half2_bits(x[g][1] * 0.0625f, x[g][5] * 0.0625f);
        qb[g][1][1] = half2_bits(x[g][3] * 0.0625f, x[g][7] * 0.0625f);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        block[g] = sum * (-8.f * 5.9604644775390625e-8f);
      } else {
        qb[g][0][0] = half2_bits(x[g][0], x[g][1]);
        qb[g][0][1] = half2_bits(x[g][2], x[g][3]);
        qb[g][1][0] = half2_bits(x[g][4], x[g][5]);
        qb[g][1][1] = half2_bits(x[g][6], x[g][7]);
      }
    }
    if constexpr (KV == XM_KV_Q4_0) {                  // inner index 2 kq, 2 kq + 1 is a block; the others are zeros
      float x0 = 0.f, x1 = 0.f;
#pragma unroll
      for (int g = 0; g < NG; g += 2)
        if (kq == g / 2) {
          x0 = block[g];
          x1 = block[g + 1];
        }
      q_off[0] = half2_bits(x0, x1);
      q_off[1] = half2_bits(x0 - half_of(q_off[0], 0), x1 - half_of(q_off[0], 1));
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) q_f[c] = __shfl_sync(0xffffffffu, f, 4 * (2 * kq + c));
  #pragma unroll
    for (int g = 0; g < NG; ++g)
      asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(qb_at + (nt * NG + g) * 512), "r"(qb[g][0][0]),
                   "r"(qb[g][0][1]), "r"(qb[g][1][0]), "r"(qb[g][1][1]) : "memory");
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(qx_at + nt * 512), "r"(__float_as_uint(q_f[0])),
                 "r"(__float_as_uint(q_f[1])), "r"(q_off[0]), "r"(q_off[1]) : "memory");
  }
  __syncthreads();
  float q_f[NT][2];
  uint32_t q_off[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    uint32_t w[4];
    lds_words<4>(w, qx_at + nt * 512);
    q_f[nt][0] = __uint_as_float(w[0]);
    q_f[nt][1] = __uint_as_float(w[1]);
    q_off[nt][0] = w[2];
    q_off[nt][1] = w[3];
  }

  uint32_t eights[4];                                  // codes 8 (kept in registers: the compiler would remake them)
#pragma unroll
  for (int i = 0; i < 4; ++i) asm volatile("mov.u32 %0, 0x00080008;" : "=r"(eights[i]));

  // One step of UK keys from key0 on.  FULL: every row sees every one of them.
  auto step = [&](auto full_, int key0, uint32_t at, bool hidden) {
    constexpr bool FULL = decltype(full_)::value;
    Sub tile[SUB];
    float sc[NT][SUB][4];
#pragma unroll
    for (int j = 0; j < SUB; ++j) {
      tile[j].read_k(at + j * Sub::kBytes, r, kq);
      if constexpr (KV == XM_KV_Q4_0) {
        // the blocks' offsets first: sum of d (-8 sum q)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma_16816_from(sc[nt][j], 0.f, 0.f, tile[j].kx[0], tile[j].kx[1], tile[j].kx[0], tile[j].kx[1], q_off[nt][0],
                         q_off[nt][1]);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint32_t wa = tile[j].k[0][g], wb = tile[j].k[1][g], xa = wa >> 8, xb = wb >> 8;
          const float da_ = half_of(tile[j].kd[0][g / 2], g & 1), db_ = half_of(tile[j].kd[1][g / 2], g & 1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float t[4];
            uint32_t q[4];
            lds_words<4>(q, qb_at + (nt * NG + g) * 512);
            mma_16816_from(t, 0.f, 0.f, wa & 0x000f000fu, wb & 0x000f000fu, xa & 0x000f000fu, xb & 0x000f000fu, q[0],
                           q[1]);
            mma_16816(t, wa & 0x00f000f0u, wb & 0x00f000f0u, xa & 0x00f000f0u, xb & 0x00f000f0u, q[2], q[3]);
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[nt][j][i] = fmaf(i < 2 ? da_ : db_, t[i], sc[nt][j][i]);
          }
        }
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            uint32_t q[4];
            lds_words<4>(q, qb_at + (nt * NG + c) * 512);
            if (c == 0)
              mma_16816_from(sc[nt][j], 0.f, 0.f, tile[j].k[0][0][0], tile[j].k[1][0][0], tile[j].k[0][0][1],
                             tile[j].k[1][0][1], q[0], q[1]);
            else
              mma_16816(sc[nt][j], tile[j].k[0][c][0], tile[j].k[1][c][0], tile[j].k[0][c][1], tile[j].k[1][c][1], q[0],
                        q[1]);
            mma_16816(sc[nt][j], tile[j].k[0][c][2], tile[j].k[1][c][2], tile[j].k[0][c][3], tile[j].k[1][c][3], q[2],
                      q[3]);
          }
      }
    }
    if constexpr (KV == XM_KV_Q4_0) {
#pragma unroll
      for (int j = 0; j < SUB; ++j) tile[j].read_vd(at + j * Sub::kBytes, r);
    }
    // whether any row sees key `at` of subtile j
    auto any_sees = [&](int j, int row) {
      if (FULL) return true;
      const int key = key0 + 16 * j + row;
      return !hidden && key <= ts.pmax && (a.window == 0 || key > ts.pmin - a.window || key < a.sinks);
    };
    int e = 0;                                         // |d| < 2^e for every block scale of the step
    if constexpr (KV == XM_KV_Q4_0) {
      uint32_t m = 0;
#pragma unroll
      for (int j = 0; j < SUB; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool any = any_sees(j, key_of(r) + 8 * i);
#pragma unroll
          for (int w = 0; w < NG / 2; ++w) m = __vmaxu2(m, any ? tile[j].vd[i][w] & 0x7fff7fffu : 0u);
        }
      e = (int)(__reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16)) >> 10) - 14;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (!FULL) {
#pragma unroll
        for (int j = 0; j < SUB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * j + key_of(r) + 8 * (i >> 1);
            if (hidden || !sees(a, pos[nt][i & 1], key)) sc[nt][j][i] = -INFINITY;
          }
      }
      float want[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(sc[nt][0][c], sc[nt][0][c + 2]);
#pragma unroll
        for (int j = 1; j < SUB; ++j) m = fmaxf(m, fmaxf(sc[nt][j][c], sc[nt][j][c + 2]));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
        want[c] = !FULL && m == -INFINITY ? m : fmaf(m, q_f[nt][c], (float)(e - 13));
      }
      // weights stay below 2^15: the reference moves only when they would pass it
      if (__any_sync(0xffffffffu, want[0] > R_[nt][0] + 2.f || want[1] > R_[nt][1] + 2.f)) {
        float al[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float was = R_[nt][c];
          if (want[c] > was + 2.f) R_[nt][c] = want[c];
          al[c] = was == R_[nt][c] ? 1.f : ex2(was - R_[nt][c]);
        }
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          o[nt][i][0] *= al[0]; o[nt][i][1] *= al[1]; o[nt][i][2] *= al[0]; o[nt][i][3] *= al[1];
        }
        if constexpr (KV == XM_KV_Q4_0) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            off[nt][g][0] *= al[0]; off[nt][g][1] *= al[1];
          }
        }
        l[nt][0] *= al[0]; l[nt][1] *= al[1];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float ref = R_[nt][c] == -INFINITY ? 0.f : R_[nt][c];
#pragma unroll
        for (int j = 0; j < SUB; ++j)
#pragma unroll
          for (int h = 0; h < 4; h += 2) {
            const float x = ex2(fmaf(sc[nt][j][c + h], q_f[nt][c], -ref));
            sc[nt][j][c + h] = !FULL && sc[nt][j][c + h] == -INFINITY ? 0.f : x;   // (q_f may be 0)
          }
      }
#pragma unroll
      for (int j = 0; j < SUB; ++j) {
        l[nt][0] += sc[nt][j][0] + sc[nt][j][2];
        l[nt][1] += sc[nt][j][1] + sc[nt][j][3];
      }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int j = 0; j < SUB; ++j) {
      tile[j].read_v(at + j * Sub::kBytes, r, kq);
      if constexpr (KV == XM_KV_Q4_0) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float da_ = half_of(tile[j].vd[0][g / 2], g & 1), db_ = half_of(tile[j].vd[1][g / 2], g & 1);
          const uint32_t sel = g & 1 ? 0x7632u : 0x5410u;
          const uint32_t x = __byte_perm(tile[j].v[0][g / 2], tile[j].v[1][g / 2], sel);
          const uint32_t y = __byte_perm(tile[j].v[2][g / 2], tile[j].v[3][g / 2], sel);
          const uint32_t xs = __byte_perm(x, 0u, 0x4341u), ys = __byte_perm(y, 0u, 0x4341u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float p0 = sc[nt][j][0] * da_, p1 = sc[nt][j][1] * da_, p2 = sc[nt][j][2] * db_, p3 = sc[nt][j][3] * db_;
            if (!FULL) {                               // a masked key's scale may be anything
              p0 = sc[nt][j][0] == 0.f ? 0.f : p0;
              p1 = sc[nt][j][1] == 0.f ? 0.f : p1;
              p2 = sc[nt][j][2] == 0.f ? 0.f : p2;
              p3 = sc[nt][j][3] == 0.f ? 0.f : p3;
            }
            const uint32_t b0 = transpose_8x8(half2_bits(p0, p1)), b1 = transpose_8x8(half2_bits(p2, p3));
            mma_16816(o[nt][2 * g], x & 0x00ff00ffu, xs, y & 0x00ff00ffu, ys, b0, b1);
            mma_16816(o[nt][2 * g + 1], x & 0x00f000f0u, xs & 0x00f000f0u, y & 0x00f000f0u, ys & 0x00f000f0u, b0, b1);
            mma_16816(off[nt][g], eights[0], eights[1], eights[2], eights[3], b0, b1);
          }
        }
      } else {
        if (!FULL) {
          // values behind every row's mask become zeros; a non-finite value that only some rows see is
          // taken out of the product and added to those rows one by one
          unsigned odd = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = kq + 4 * i;
            const bool any = any_sees(j, row);
            bool nf = false;
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                if (!any) tile[j].v[i][c][w] = 0u;
                nf |= non_finite(tile[j].v[i][c][w]);
              }
            if (nf) odd |= 1u << row;
          }
          odd = ts.pmin == ts.pmax ? 0u : __reduce_or_sync(0xffffffffu, odd);
          if (odd) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (odd >> (kq + 4 * i) & 1u)
#pragma unroll
                for (int c = 0; c < D / 64; ++c)
#pragma unroll
                  for (int w = 0; w < 4; ++w) tile[j].v[i][c][w] = 0u;
            for (unsigned left = odd; left; left &= left - 1) {
              const int key = __ffs(left) - 1;
              // this lane's values of the key: 16-byte piece 8 c + r of its row
              uint32_t vw[D / 64][4];
#pragma unroll
              for (int c = 0; c < D / 64; ++c)
                lds_words<4>(vw[c], at + Sub::kVAt + key * Sub::ROW + (8 * c + (r ^ (key & 3) << 1)) * 16);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const int from = ((key & 3) << 1 | (key >> 2 & 1)) * 4 + kq;
                const float a0 = __shfl_sync(0xffffffffu, sc[nt][j][0], from), a1 = __shfl_sync(0xffffffffu, sc[nt][j][1], from);
                const float a2 = __shfl_sync(0xffffffffu, sc[nt][j][2], from), a3 = __shfl_sync(0xffffffffu, sc[nt][j][3], from);
                const float pc[2] = {key < 8 ? a0 : a2, key < 8 ? a1 : a3};
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  if (sees(a, pos[nt][c], key0 + key))
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                      o[nt][i][c] = fmaf(pc[c], half_of(vw[i / 4][i % 4], 0), o[nt][i][c]);
                      o[nt][i][c + 2] = fmaf(pc[c], half_of(vw[i / 4][i % 4], 1), o[nt][i][c + 2]);
                    }
              }
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint32_t b0 = transpose_8x8(half2_bits(sc[nt][j][0], sc[nt][j][1]));
          const uint32_t b1 = transpose_8x8(half2_bits(sc[nt][j][2], sc[nt][j][3]));
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int w = 0; w < 4; ++w)
              mma_16816(o[nt][4 * c + w], __byte_perm(tile[j].v[0][c][w], tile[j].v[1][c][w], 0x5410u),
                        __byte_perm(tile[j].v[0][c][w], tile[j].v[1][c][w], 0x7632u),
                        __byte_perm(tile[j].v[2][c][w], tile[j].v[3][c][w], 0x5410u),
                        __byte_perm(tile[j].v[2][c][w], tile[j].v[3][c][w], 0x7632u), b0, b1);
        }
      }
    }
  };

  // units [fa, fb) of the run, and the first fs, are seen whole by every row
  const int fs = a.window > 0 ? min(ts.ns, a.sinks / UK) : 0;
  const int fa = ts.ns + (a.window > 0 ? max(0, (ts.pmax - a.window + UK) / UK - ts.a0) : 0);
  const int fb = ts.ns + (ts.pmin + 1) / UK - ts.a0;
  for (int i = 0; i < steps; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();                                      // step i has landed, and every lane is done with step i - 1
    const bool hidden = bad_steps >> (i & 31) & 1u;
    fetch(i + STAGES - 1);
    const int v = v_lo + warp + i * kDecWarps, key0 = ts.unit(v) * UK;
    const uint32_t at = ring + i % STAGES * (SUB * Sub::kBytes);
    if (hidden && lane == 0) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
    if (!hidden && ((v >= fa && v < fb) || v < fs)) step(std::true_type{}, key0, at, false);
    else step(std::false_type{}, key0, at, hidden);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                     // the ring's memory is free

  // the warps' parts meet in shared memory
  float(*o_s)[R][DP] = reinterpret_cast<float(*)[R][DP]>(dec_smem);
  float2(*ml_s)[R] = reinterpret_cast<float2(*)[R]>(dec_smem + kDecWarps * R * DP * 4);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x = l[nt][c];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (r == 0) ml_s[warp][8 * nt + 2 * kq + c] = make_float2(R_[nt][c], x);
      float* row = &o_s[warp][8 * nt + 2 * kq + c][0];
      if constexpr (KV == XM_KV_Q4_0) {
        constexpr float k24 = 16777216.f, k20 = 1048576.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float f = off[nt][g][c];
          // o[2g]: whole bytes c + 16 c', o[2g + 1]: 16 c', off: 8, each times 2^-24
          const float lo = o[nt][2 * g + 1][c], hi = o[nt][2 * g + 1][c + 2];
          *reinterpret_cast<float4*>(row + 32 * g + 4 * r) =
              make_float4(k24 * (o[nt][2 * g][c] - lo - f), k20 * (lo - 16.f * f), k24 * (o[nt][2 * g][c + 2] - hi - f),
                          k20 * (hi - 16.f * f));
        }
      } else {
#pragma unroll
        for (int i = 0; i < D / 16; i += 2)
          *reinterpret_cast<float4*>(row + 64 * (i / 4) + 8 * r + 2 * (i % 4)) =
              make_float4(o[nt][i][c], o[nt][i][c + 2], o[nt][i + 1][c], o[nt][i + 1][c + 2]);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < ts.rows * (D / 4); i += 32 * kDecWarps) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) m = fmaxf(m, ml_s[w][row].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float2 ml = ml_s[w][row];
      const float f = ex2(ml.x - ref);
      const float4 x = *reinterpret_cast<const float4*>(&o_s[w][row][d]);
      sum = fmaf(ml.y, f, sum);
      acc.x = fmaf(x.x, f, acc.x);
      acc.y = fmaf(x.y, f, acc.y);
      acc.z = fmaf(x.z, f, acc.z);
      acc.w = fmaf(x.w, f, acc.w);
    }
    const int gr = ts.r0 + row;
    const int64_t t = t0 + gr / G;
    const int h = hk * G + gr % G;
    if (parts <= 1) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      put_out4<QT_>((QT_*)a.out + t * a.out_stride + (int64_t)h * D + d, a.out_vec,
                    make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    } else {
      const int64_t cell = ((int64_t)split * a.T + t) * a.Hq + h;
      *reinterpret_cast<float4*>(da.part_o + cell * D + d) = acc;
      if (d == 0) da.part_ml[cell] = make_float2(m, sum);
    }
  }
}

// Joins the parts of the rows whose keys were split: one CTA per (row, query head), its warps take the
// parts in turn and are summed in a fixed order.
template <typename QT_, int D, int R, int UK>
__global__ void __launch_bounds__(128) k_kv_merge(const KvView kv, const AttnArgs a, const DecArgs da) {
  __shared__ float f_s[kMaxSplits];
  __shared__ float red[4];
  __shared__ __align__(16) float o_s[4][D];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = a.Hq / kv.Hk;
  const int64_t cell = blockIdx.x, cells = a.T * a.Hq, t = cell / a.Hq;
  const int h = (int)(cell % a.Hq);
  const int s = kv_sequence(kv, t);
  if (s < 0) return;
  int64_t t0;
  int q_len;
  sequence_rows(kv, a.T, s, t0, q_len);
  const int gr = (int)(t - t0) * G + h % G;
  const TileSpan ts = tile_span<R, UK>(kv, a, s, t0, q_len, gr / R, G);
  const int parts = (ts.n + da.chunk - 1) / da.chunk;
  if (parts <= 1) return;
  const float2 ml = tid < parts ? __ldcg(&da.part_ml[(int64_t)tid * cells + cell]) : make_float2(-INFINITY, 0.f);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  const int d = lane * 4;
  float m = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float f = ex2(ml.x - (m == -INFINITY ? 0.f : m));
  f_s[tid] = f;
  float sum = warp_sum(ml.y * f);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  if (d < D) {
#pragma unroll 8
    for (int p = warp; p < parts; p += 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(da.part_o + ((int64_t)p * cells + cell) * D + d));
      const float w = f_s[p];
      acc.x = fmaf(x.x, w, acc.x);
      acc.y = fmaf(x.y, w, acc.y);
      acc.z = fmaf(x.z, w, acc.z);
      acc.w = fmaf(x.w, w, acc.w);
    }
    *reinterpret_cast<float4*>(&o_s[warp][d]) = acc;
  }
  __syncthreads();
  if (warp > 0 || d >= D) return;
  sum = (red[0] + red[1]) + (red[2] + red[3]);
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float4 x = *reinterpret_cast<const float4*>(&o_s[w][d]);
    acc.x += x.x;
    acc.y += x.y;
    acc.z += x.z;
    acc.w += x.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  put_out4<QT_>((QT_*)a.out + t * a.out_stride + (int64_t)h * D + d, a.out_vec,
                make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
}

struct DecPlan {
  int nt;               // groups of 8 rows per CTA; 0: the prompt kernel
  int64_t tiles;        // row tiles, at most
  int chunk, nsplit;      // keys of a part; parts, at most
  int64_t ws_bytes;
};

DecPlan dec_plan(int64_t T, int64_t B, int Hq, int Hk, int D, int64_t max_keys, bool ragged) {
  DecPlan p{};
  const int G = Hq / Hk;
  if (T * G > 16 * B && T > B) return p;
  p.nt = T * G <= 8 * B ? 1 : 2;
  const int R = 8 * p.nt;
  p.tiles = ragged ? T * G / R + B : B * ((G + R - 1) / R);
  // few tiles: one wave of three CTAs on each of the 148 SMs; many: chunks of 2048 keys, so that the
  // sequences' different lengths even out.  At least a step for each warp, and no more parts than keep
  // the workspace small
  const int64_t base = p.tiles * Hk, slots = 3 * 148;
  int64_t chunk = 2 * base <= slots ? (max_keys + slots / base - 1) / (slots / base) : 2048;
  chunk = std::max<int64_t>(chunk, 128);
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kMaxSplits, (1 << 17) / std::max<int64_t>(1, T * Hq)));
  chunk = std::max<int64_t>(chunk, (max_keys + most - 1) / most);
  p.chunk = (int)((chunk + 127) / 128 * 128);
  p.nsplit = (int)((max_keys + p.chunk - 1) / p.chunk);
  p.ws_bytes = p.nsplit > 1 ? (int64_t)p.nsplit * T * Hq * (D * 4 + 8) : 0;
  return p;
}

template <typename... KArgs, typename... Args>
int kv_launch(const char* what, void (*kernel)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t st,
              Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
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

template <typename QT_, int D, int KV, int NT>
int decode_kernel(const KvView& kv, const AttnArgs& a, const DecArgs& da, dim3 grid, cudaStream_t st) {
  constexpr int smem = DecShape<KV, D, NT>::kSmem;
  static bool done[64] = {};                           // the attribute is set once per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 && (dev < 0 || dev >= 64 || !done[dev])) {
    const cudaError_t e = cudaFuncSetAttribute(k_kv_decode<QT_, D, KV, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "kv attention: smem attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return kv_launch("kv attention", k_kv_decode<QT_, D, KV, NT>, grid, 32 * kDecWarps, smem, st, kv, a, da);
}

template <typename QT_, int D, int KV>
int decode_launch(const KvView& kv, const AttnArgs& a, const DecPlan& p, void* ws, cudaStream_t st) {
  constexpr int UK = 16 * DecShape<KV, D, 1>::SUB;
  DecArgs da{p.chunk / UK, p.nsplit, (float*)ws, (float2*)((float*)ws + (int64_t)p.nsplit * a.T * a.Hq * D)};
  const dim3 grid((unsigned)(p.tiles * kv.Hk), (unsigned)p.nsplit), mgrid((unsigned)(a.T * a.Hq));
  const int rc = p.nt == 1 ? decode_kernel<QT_, D, KV, 1>(kv, a, da, grid, st)
                           : decode_kernel<QT_, D, KV, 2>(kv, a, da, grid, st);
  if (rc || p.nsplit <= 1) return rc;
  return p.nt == 1 ? kv_launch("kv attention merge", k_kv_merge<QT_, D, 8, UK>, mgrid, 128, 0, st, kv, a, da)
                   : kv_launch("kv attention merge", k_kv_merge<QT_, D, 16, UK>, mgrid, 128, 0, st, kv, a, da);
}

template <typename QT_, int D, int KV>
int attn_launch(const KvView& kv, const AttnArgs& a, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.T, (unsigned)((a.Hq + kAttnWarps - 1) / kAttnWarps));
  cfg.blockDim = dim3(32 * kAttnWarps);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_kv_attn<QT_, D, KV>, kv, a);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "kv attention launch: %s", cudaGetErrorString(e));
  return xm_check_launch("kv attention");
}

template <typename QT_>
int attn_typed(const KvView& kv, const AttnArgs& a, int kv_type, int head_dim, void* ws, cudaStream_t st) {
  const DecPlan p = dec_plan(a.T, kv.B, a.Hq, kv.Hk, head_dim, (int64_t)kv.table_width << kv.page_shift, kv.cu != nullptr);
  if (p.nt) {
    if (head_dim == 128)
      return kv_type == XM_KV_F16 ? decode_launch<QT_, 128, XM_KV_F16>(kv, a, p, ws, st)
                                  : decode_launch<QT_, 128, XM_KV_Q4_0>(kv, a, p, ws, st);
    return kv_type == XM_KV_F16 ? decode_launch<QT_, 64, XM_KV_F16>(kv, a, p, ws, st)
                                : decode_launch<QT_, 64, XM_KV_Q4_0>(kv, a, p, ws, st);
  }
  if (head_dim == 128)
    return kv_type == XM_KV_F16 ? attn_launch<QT_, 128, XM_KV_F16>(kv, a, st) : attn_launch<QT_, 128, XM_KV_Q4_0>(kv, a, st);
  return kv_type == XM_KV_F16 ? attn_launch<QT_, 64, XM_KV_F16>(kv, a, st) : attn_launch<QT_, 64, XM_KV_Q4_0>(kv, a, st);
}

}  // namespace

extern "C" {

int64_t xm_kv_attention_workspace_size(int64_t T, int64_t B, int Hq, int Hk, int head_dim, int64_t max_keys) {
  if (T < 1 || B < 1 || Hq < 1 || Hk < 1 || Hq % Hk || max_keys < 1) return 16;
  return std::max<int64_t>(16, std::max(dec_plan(T, B, Hq, Hk, head_dim, max_keys, true).ws_bytes,
                                        dec_plan(T, B, Hq, Hk, head_dim, max_keys, false).ws_bytes));
}

int xm_kv_attention(const void* d_q, int q_dtype, int64_t T, int64_t q_stride, int Hq, int Hk, int head_dim,
                    float scale, int64_t window, int64_t sinks, const void* d_pool, int64_t pages, int kv_type,
                    int page_size, const int* d_table, int64_t table_stride, int64_t table_width, const int* d_cu,
                    const int* d_lens, int64_t B, void* d_out, int64_t out_stride, void* d_ws, int64_t ws_bytes,
                    void* stream) {
  KvView kv;
  if (int rc = kv_view("kv_attention", (void*)d_pool, pages, kv_type, Hk, head_dim, page_size, d_table, table_stride,
                       table_width, d_cu, d_lens, B, &kv))
    return rc;
  if (T < 0 || T > INT32_MAX || Hq < 1 || Hq > 65535 || Hq % Hk || Hq / Hk > 64 || (!d_cu && T != B))
    return xm_set_error(XM_ERR_INVALID,
                        "kv_attention: bad row or head counts (at most 64 query heads per KV head; T = B where no row "
                        "offsets are given)");
  if (q_dtype != XM_DT_F16 && q_dtype != XM_DT_BF16)
    return xm_set_error(XM_ERR_INVALID, "kv_attention: queries are fp16 or bf16, not type %d", q_dtype);
  if (window < 0 || sinks < 0) return xm_set_error(XM_ERR_INVALID, "kv_attention: negative window or sinks");
  if (T == 0) return XM_OK;
  if (!d_q || !d_out) return xm_set_error(XM_ERR_INVALID, "kv_attention: null pointer");
  if (q_stride < (int64_t)Hq * head_dim || out_stride < (int64_t)Hq * head_dim || (((uintptr_t)d_q | (uintptr_t)d_out) & 1))
    return xm_set_error(XM_ERR_INVALID, "kv_attention: bad row pitch or alignment");
  if (ws_bytes < xm_kv_attention_workspace_size(T, B, Hq, Hk, head_dim, table_width * page_size) || !d_ws ||
      ((uintptr_t)d_ws & 15))
    return xm_set_error(XM_ERR_INVALID, "kv_attention: workspace too small or unaligned");
  const int64_t most = 1 << 30;                      // as good as none
  AttnArgs a{d_q, T, q_stride, Hq, scale, window < most ? (int)window : 0, (int)std::min(sinks, most), d_out, out_stride,
             q_stride % 8 == 0 && ((uintptr_t)d_q & 15) == 0, out_stride % 4 == 0 && ((uintptr_t)d_out & 7) == 0};
  cudaStream_t st = (cudaStream_t)stream;
  return q_dtype == XM_DT_F16 ? attn_typed<__half>(kv, a, kv_type, head_dim, d_ws, st)
                              : attn_typed<__nv_bfloat16>(kv, a, kv_type, head_dim, d_ws, st);
}

}  // extern "C"
