// Attention over the paged key/value cache (layout: xm_kv.cuh).
//
// Row t of sequence s at position p sees the keys 0 .. p of its sequence (with a window w: those above
// p - w, and the first `sinks`); query head h reads KV head h / (Hq / Hk):
//   out = sum_k softmax_k(q . K_k * scale) V_k,  zeros for a row that sees no key.
//
// Few rows per sequence (decode steps): k_kv_decode, bound by reading the cache.  Many (prompts): k_kv_prompt, bound by
// the products and the exponentials.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "xm_kv.cuh"

int kv_view(const char* who, void* pool, int64_t pages, int kv_type, int Hk, int head_dim, int page_size,
            const int* table, int64_t table_stride, int64_t table_width, const int* cu, const int* lens, int64_t B,
            KvView* out);

namespace cg = cooperative_groups;

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

// ---------------------------------------------------------------------------
// Decode: up to 8 NT rows (token, query head) of one KV head of one sequence per CTA; the keys are
// split over the warps of a CTA, and over CTAs in chunks of `chunk` keys whose partial softmaxes
// k_kv_merge joins.
//
// Bound: memory (the cache is read once); the work per byte decides whether that is reached.  8 sequences of up to
// 4096 keys in fp16 (8 KV heads): 24.6 us, 0.59 of the copy bandwidth; 64 sequences of up to 8192 in 4 bits: 118 us, 0.52
// of it.  At three CTAs an SM (168 registers a thread; four spill and are slower) latency is the limit: 17 % of the warps
// active, issue slots 54 %, about 340 instructions per 16 keys and head, DRAM 41 %.  A warp
// takes 16 keys at a time on mma.sync m16n8k16 (fp16 operands, fp32 sums) with the keys, or the
// values' dimensions, as the 16 matrix rows and the query rows as the 8 columns:
//   S^T [16 keys x 8 rows] = K q^T,   O^T [D x 8 rows] += V^T P^T.
// The rows pass through a ring of each warp in shared memory (cp.async) and are read from there as fragments as
// they lie: the order of the products' inner dimension is free, and the cache's layout was chosen for it.
//
// 4-bit rows are never unpacked to values.  The nibbles 0 and 4 (for keys; 0 of two keys, paired by a
// byte permute, for values) of a word are, after one mask, two fp16 subnormals c 2^-24, the nibbles
// 1 and 5 are c 2^-20: exact, one instruction for two codes.  For values whole bytes (c + 16 c') 2^-24 and
// their high nibbles enter, one instruction less, and the low codes' sums are the difference at the end (of sums of up to
// 255 p d in fp32: some 2^-18 of a block's largest value, where p d itself is rounded to 2^-11).
// The block scale and the offset of the codes stay outside the product:
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
constexpr int kMaxJoined = 8;       // CTAs of a cluster

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
  // (the offsets count, not q_len: rows that they name behind the call's last are of the sequence all the same)
  x.p_first = __ldg(kv.lens + s) - (kv.cu ? __ldg(kv.cu + s + 1) - (int)t0 : 1);
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
  int chunk;                // units of a part, at least
  int nsplit;
  float* part_o;            // [nsplit][T][Hq][D], where a row has more than one part; null: joined in a cluster
  float2* part_ml;
  // units of each part of n: at least `chunk`, and as many as leave no more than nsplit parts
  XM_DEV int part_units(int n) const { return max(chunk, (n + nsplit - 1) / nsplit); }
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
  static constexpr int kSmem = kQ + (kDecWarps * kRing > kJoin ? kDecWarps * kRing : kJoin) + 8 * NT * 8;
  static constexpr int kCtas = NT > 1 ? 2 : KV == XM_KV_Q4_0 || D == 64 ? 3 : 2;          // of an SM
};

// ONE_PAGE: a step's unit lies in one page (else in two of 16 tokens, and each is looked up; chosen at run time that costs
// the other page sizes 2 to 4 %: 64 sequences of up to 8192 tokens in 4 bits 121 to 123 us, this way 117).
template <typename QT_, int D, int KV, int NT, bool ONE_PAGE>
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
  if (s < 0) return;                                   // (every CTA of a cluster)
  const TileSpan ts = tile_span<R, UK>(kv, a, s, t0, q_len, rt, G);
  if (ts.past_table && threadIdx.x == 0) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
  // parts of da.chunk units that k_kv_merge joins; or, in a cluster, even shares joined through its shared memories
  const bool joined = da.part_o == nullptr && da.nsplit > 1;
  const int chunk = joined ? (ts.n + da.nsplit - 1) / da.nsplit : da.part_units(ts.n);
  const int parts = joined ? 1 : (ts.n + chunk - 1) / chunk;
  if (!joined && split > 0 && split >= parts) return;
  const int v_lo = min(ts.n, split * chunk), v_hi = min(ts.n, v_lo + chunk);

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
  // Bit i: step i % 32 lies on a page outside the pool (the second of its pages: in bad_second), unless no row sees a key
  // of that page.  (Such a page, behind a window, may be gone: its bytes are masked like those of any hidden key.)
  unsigned bad = 0, bad_second = 0;
  auto needed = [&](int key) {                         // whether any row sees one of 16 keys (a whole unit has one)
    return ONE_PAGE || (key <= ts.pmax && (a.window == 0 || key + 15 > ts.pmin - a.window || key < a.sinks));
  };
  auto fetch = [&](int i) {                            // starts the copies of step i
    if (i < steps) {
      if (i > 0 && (i & 31) == 0) {
        pages = pages_next;
        pages_next = page_of(i + 32 + lane, 0);
      }
      const int key0 = ts.unit(v_lo + warp + i * kDecWarps) * UK;
      bad &= ~(1u << (i & 31));
      if (!ONE_PAGE) bad_second &= ~(1u << (i & 31));
      const uint8_t* head;
      const uint32_t to = ring + i % STAGES * (SUB * Sub::kBytes);
#pragma unroll
      for (int j = 0; j < SUB; ++j) {
        if (j == 0 || !ONE_PAGE) {
          int p = __shfl_sync(0xffffffffu, pages, i & 31);
          if (j > 0) p = page_of(i, j);
          const bool in = (unsigned)p < (unsigned)kv.pages;
          if (!in && needed(key0 + 16 * j)) (j ? bad_second : bad) |= 1u << (i & 31);
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

  // One step of UK keys, its subtiles' from first.x and first.y on (kNoKeys: without a page).  FULL: every row sees every
  // one of them.
  constexpr int kNoKeys = 0x7fffffff - 15;             // behind every position that a table reaches, with the 15 keys after it
  auto step = [&](auto full_, int2 first, uint32_t at) {
    const int keys[2] = {first.x, first.y};
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
      const int key = keys[j] + row;
      return key <= ts.pmax && (a.window == 0 || key > ts.pmin - a.window || key < a.sinks);
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
    unsigned hidden[NT] = {};                          // bit 4 j + i: sc[nt][j][i] is of a key that its row does not see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (!FULL) {
#pragma unroll
        for (int j = 0; j < SUB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = keys[j] + key_of(r) + 8 * (i >> 1);
            if (!sees(a, pos[nt][i & 1], key)) {
              sc[nt][j][i] = -INFINITY;
              hidden[nt] |= 1u << (4 * j + i);
            }
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
            sc[nt][j][c + h] = !FULL && hidden[nt] >> (4 * j + c + h) & 1u ? 0.f : x;
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
            if (!FULL) {                               // a hidden key's scale may be anything (a seen one's counts,
              const unsigned hide = hidden[nt] >> 4 * j;   // however small its weight)
              p0 = hide & 1u ? 0.f : p0;
              p1 = hide & 2u ? 0.f : p1;
              p2 = hide & 4u ? 0.f : p2;
              p3 = hide & 8u ? 0.f : p3;
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
                  if (sees(a, pos[nt][c], keys[j] + key))
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
    const int v = v_lo + warp + i * kDecWarps, key0 = ts.unit(v) * UK;
    const bool hide_x = bad >> (i & 31) & 1u, hide_y = ONE_PAGE ? hide_x : bad_second >> (i & 31) & 1u;
    const bool hidden = hide_x || hide_y;
    const int2 first = make_int2(hide_x ? kNoKeys : key0, hide_y ? kNoKeys : key0 + 16);
    if (hidden && lane == 0) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
    fetch(i + STAGES - 1);
    const uint32_t at = ring + i % STAGES * (SUB * Sub::kBytes);
    if (!hidden && ((v >= fa && v < fb) || v < fs)) step(std::true_type{}, first, at);
    else step(std::false_type{}, first, at);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();                                     // the ring's memory is free

  // the warps' parts meet in shared memory
  float(*o_s)[R][DP] = reinterpret_cast<float(*)[R][DP]>(dec_smem);
  float2(*ml_s)[R] = reinterpret_cast<float2(*)[R]>(dec_smem + kDecWarps * R * DP * 4);
  float2* joint_s = reinterpret_cast<float2*>(dec_smem + Shape::kSmem - R * 8);
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
    if (joined) {                                      // kept where the warps' parts were: only this thread reads those
      *reinterpret_cast<float4*>(&o_s[0][row][d]) = acc;
      if (d == 0) joint_s[row] = make_float2(m, sum);
    } else if (parts <= 1) {
      const float inv = sum == 0.f ? 0.f : 1.0f / sum;
      put_out4<QT_>((QT_*)a.out + t * a.out_stride + (int64_t)h * D + d, a.out_vec,
                    make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    } else {
      const int64_t cell = ((int64_t)split * a.T + t) * a.Hq + h;
      *reinterpret_cast<float4*>(da.part_o + cell * D + d) = acc;
      if (d == 0) da.part_ml[cell] = make_float2(m, sum);
    }
  }
  if (!joined) return;
  // the cluster's parts, in order, each CTA a share of the output
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  for (int i = (int)threadIdx.x + 32 * kDecWarps * split; i < ts.rows * (D / 4); i += 32 * kDecWarps * da.nsplit) {
    const int row = i / (D / 4), d = i % (D / 4) * 4;
    float2 ml[kMaxJoined];
    float4 x[kMaxJoined];
    float m = -INFINITY;
#pragma unroll
    for (int p = 0; p < kMaxJoined; ++p) {
      ml[p] = make_float2(-INFINITY, 0.f);
      x[p] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (p < da.nsplit) {
        ml[p] = *cl.map_shared_rank(&joint_s[row], p);
        x[p] = *reinterpret_cast<const float4*>(cl.map_shared_rank(&o_s[0][row][d], p));
        m = fmaxf(m, ml[p].x);
      }
    }
    const float ref = m == -INFINITY ? 0.f : m;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll
    for (int p = 0; p < kMaxJoined; ++p) {
      const float f = ex2(ml[p].x - ref);
      sum = fmaf(ml[p].y, f, sum);
      acc.x = fmaf(x[p].x, f, acc.x);
      acc.y = fmaf(x[p].y, f, acc.y);
      acc.z = fmaf(x[p].z, f, acc.z);
      acc.w = fmaf(x[p].w, f, acc.w);
    }
    const int gr = ts.r0 + row;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    put_out4<QT_>((QT_*)a.out + (t0 + gr / G) * a.out_stride + (int64_t)(hk * G + gr % G) * D + d, a.out_vec,
                  make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
  cl.sync();                                           // no CTA leaves while its part is read
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
  const int s = kv_place(kv, t).seq;
  if (s < 0) return;
  int64_t t0;
  int q_len;
  sequence_rows(kv, a.T, s, t0, q_len);
  const int gr = (int)(t - t0) * G + h % G;
  const TileSpan ts = tile_span<R, UK>(kv, a, s, t0, q_len, gr / R, G);
  const int chunk = da.part_units(ts.n), parts = (ts.n + chunk - 1) / chunk;
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
  int rows;             // of a CTA of the prompt kernel
  int64_t tiles;        // row tiles, at most
  int chunk, nsplit;      // keys of a part (the prompt kernel: at least); parts, at most
  int64_t ws_bytes;
};

DecPlan dec_plan(int64_t T, int64_t B, int Hq, int Hk, int D, int64_t max_keys, bool ragged) {
  DecPlan p{};
  const int G = Hq / Hk;
  // One kernel for the call, by the mean: a call that mixes steps and prompts is slower than two (63 steps behind up to 8192
  // keys 113 us, a chunk of 450 tokens behind 4096 83, both in one call 438).  Parts come from max_keys, the width of the
  // table: the lengths are on the device (640 keys in a table of 640: 5.4 us, of 131072: 9.4).
  // Up to 32 rows (token, query head) of each KV head a sequence: the decode kernel (32 rows each of 8 sequences of
  // 8192 keys, 8 KV heads: 66 us, with the prompt kernel 148; of one sequence 21 and 27).  Above: the prompt kernel
  // (64 rows each: decode 135, prompt 140; of one sequence 33 and 28, behind 131072 keys 313 and 142).
  if (T * G > 32 * B && T > B) {
    // 256 rows per CTA, unless that leaves SMs without one; and where half of the SMs have none all the same, the
    // keys are split (64 rows of each of 8 KV heads behind 131072 keys, Q4_0: 18 parts take 142 us, one 2289)
    p.rows = (T * G / 256 + B) * Hk >= 148 ? 256 : 128;
    p.tiles = T * G / p.rows + B;
    p.chunk = 512;
    p.nsplit = (int)std::max<int64_t>(1, std::min({148 / (p.tiles * Hk), (max_keys + 511) / 512, (int64_t)kMaxSplits}));
    p.ws_bytes = p.nsplit > 1 ? (int64_t)p.nsplit * T * Hq * (D * 4 + 8) : 0;
    return p;
  }
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
  p.ws_bytes = p.nsplit > kMaxJoined ? (int64_t)p.nsplit * T * Hq * (D * 4 + 8) : 0;
  return p;
}

template <typename... KArgs, typename... Args>
int kv_launch(const char* what, void (*kernel)(KArgs...), dim3 grid, int cluster_y, int threads, int smem, cudaStream_t st,
              Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = attr[1].val.clusterDim.z = 1;
  attr[1].val.clusterDim.y = (unsigned)cluster_y;
  cfg.attrs = attr;
  cfg.numAttrs = cluster_y > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return xm_check_launch(what);
}

template <typename QT_, int D, int KV, int NT, bool ONE_PAGE>
int decode_kernel(const KvView& kv, const AttnArgs& a, const DecArgs& da, dim3 grid, cudaStream_t st) {
  constexpr int smem = DecShape<KV, D, NT>::kSmem;
  static bool done[64] = {};                           // the attribute is set once per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (smem > 48 * 1024 && (dev < 0 || dev >= 64 || !done[dev])) {
    const cudaError_t e = cudaFuncSetAttribute(k_kv_decode<QT_, D, KV, NT, ONE_PAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "kv attention: smem attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return kv_launch("kv attention", k_kv_decode<QT_, D, KV, NT, ONE_PAGE>, grid, da.part_o ? 1 : da.nsplit, 32 * kDecWarps, smem,
                   st, kv, a, da);
}

template <typename QT_, int D, int KV>
int decode_launch(const KvView& kv, const AttnArgs& a, const DecPlan& p, void* ws, cudaStream_t st) {
  constexpr int UK = 16 * DecShape<KV, D, 1>::SUB;
  DecArgs da{p.chunk / UK, p.nsplit, nullptr, nullptr};
  if (p.ws_bytes) {
    da.part_o = (float*)ws;
    da.part_ml = (float2*)(da.part_o + (int64_t)p.nsplit * a.T * a.Hq * D);
  }
  const dim3 grid((unsigned)(p.tiles * kv.Hk), (unsigned)p.nsplit), mgrid((unsigned)(a.T * a.Hq));
  int rc;
  if (UK == 32 && kv.page_shift == 4)
    rc = p.nt == 1 ? decode_kernel<QT_, D, KV, 1, UK == 16>(kv, a, da, grid, st)
                   : decode_kernel<QT_, D, KV, 2, UK == 16>(kv, a, da, grid, st);
  else
    rc = p.nt == 1 ? decode_kernel<QT_, D, KV, 1, true>(kv, a, da, grid, st)
                   : decode_kernel<QT_, D, KV, 2, true>(kv, a, da, grid, st);
  if (rc || !p.ws_bytes) return rc;
  return p.nt == 1 ? kv_launch("kv attention merge", k_kv_merge<QT_, D, 8, UK>, mgrid, 1, 128, 0, st, kv, a, da)
                   : kv_launch("kv attention merge", k_kv_merge<QT_, D, 16, UK>, mgrid, 1, 128, 0, st, kv, a, da);
}

// ---------------------------------------------------------------------------
// Prompts: R = 128 or 256 rows (token, query head) of one KV head of one sequence per CTA, on
// tcgen05.  The cache is walked in units of 128 keys, read once for all of the CTA's rows.
//
//   warps 0-3, 4-7   softmax of row tile 0, 1 (a thread is a row = a lane of tensor memory)
//   warps 8-11       loaders: bring a unit's keys and values into shared memory as fp16
//   warps 12, 13     issue the products of row tile 0, 1 (one thread each); warp 12 allocates tensor memory
//
// S = Q K^T (M = 128 rows, N = 64 keys, a half unit) goes to tensor memory, the softmax warps turn it into P (fp16) in
// place, and O += P V takes P from tensor memory and V as it lies in the cache, dimensions contiguous.  S
// has two buffers per row tile, so the next half's S is computed while this one's softmax runs, and that
// is never held up by the product that reads its P.  Tensor memory: S of tile i, half h at column 128 i + 64 h,
// O of tile i at 256 + D i.
//
// What decides the speed is the chain of one row tile: a row of S is read once, 64 columns into registers (a
// tcgen05.wait::ld waits for every load, and costs some 300 clocks), its maximum taken, P computed.  A prompt of
// 8192 tokens (32 query and 8 KV heads of 128, 4 bits; calls from Python on changing inputs) took 790 us with units of 128
// keys and one S per row tile (PV and S follow one another in the chain: 6100 clocks a unit), 779 with half units and two S,
// 760 with the products issued by an elected lane, 745 with a quarter of the exponentials on the multipliers (ex2_fma), 730
// with one body for masked and whole units, 717 with an eighth of them there: 766 TFLOP/s (in a graph on the same inputs
// 664; fp16 827).  The 4-bit instances spill 16 to 24 bytes at 128 registers, the most that 14 warps leave.  Four chunks of up to
// 1000 tokens behind up to 5000, window 1024, sinks, fp16, 28 query and 4 KV heads of 64: 92 us with two to five
// instructions a column for the mask, 75 with a word of its bits.
//
// 4-bit rows become fp16 here, d (c - 8) rounded once (2^-11): a product per code would need the scales
// inside the tensor core's inner dimension.  The order of the eight values that a word of keys yields is
// kept, and q's is changed to it; the order of a word of values is a permutation of O's columns, undone
// when O is written.  A unit with a scale above 4096 (values past fp16's range) is scaled by 2^-4.
// Norm-wise, over thousands of normal keys, the roundings to fp16 put the outputs off by 1.8e-4 (keys), 1.6e-4 (values)
// and 2.1e-4 (P), 3.3e-4 together; the rounding of an fp16 output alone is 2.0e-4.
//
// The running reference of a row moves only when a score passes it by 8 (P <= 2^8), so O, which stays in
// tensor memory, is rescaled seldom.
//
// Masked keys: their scores are replaced, their values are zeros where no row sees them; a value that is not
// finite and that only some rows see is taken out of the product and added to those rows alone.
//
// Bound: the products (4 R 128 D flops a unit at the tensor peak: 2048 clocks a unit of R = 256, D = 128) and, as much, the
// 128 R exponentials (16 a clock: 2048 clocks a unit); neither is reached, since a row tile's chain (some 5000 clocks a unit:
// waits 800, maximum 1200, exponentials and rounding 2200, loads and stores of tensor memory 700) is only halved by the
// other's.
// ---------------------------------------------------------------------------
constexpr int kUnit = 128;                         // keys of a unit
constexpr int kPromptThreads = 14 * 32;

XM_DEV void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
XM_DEV void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
XM_DEV void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The products of a unit from one asm block each: the issuing thread shares its scheduler with busy warps, so every
// instruction between two products counts.  Descriptors are {low, high} words; only the start (low) moves.
// d = A B^T over 16 K values, K = {4, 8}, blocks of 64 values 16 KB apart
template <int K>
XM_DEV void tc_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc) {
  if constexpr (K == 8)
  asm volatile("{\n .reg .pred p0, p1;\n .reg .b64 da, db;\n .reg .b32 x, y;\n"
               " setp.eq.b32 p0, 0, 0;\n setp.ne.b32 p1, 0, 0;\n"
               " mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p1;\n"
               " add.u32 x, %1, 2;\n add.u32 y, %2, 2;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 4;\n add.u32 y, %2, 4;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 6;\n add.u32 y, %2, 6;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 1024;\n add.u32 y, %2, 1024;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 1026;\n add.u32 y, %2, 1026;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 1028;\n add.u32 y, %2, 1028;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 1030;\n add.u32 y, %2, 1030;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               "}"
               ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc) : "memory");
  else
  asm volatile("{\n .reg .pred p0, p1;\n .reg .b64 da, db;\n .reg .b32 x, y;\n"
               " setp.eq.b32 p0, 0, 0;\n setp.ne.b32 p1, 0, 0;\n"
               " mov.b64 da, {%1, %3};\n mov.b64 db, {%2, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p1;\n"
               " add.u32 x, %1, 2;\n add.u32 y, %2, 2;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 4;\n add.u32 y, %2, 4;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               " add.u32 x, %1, 6;\n add.u32 y, %2, 6;\n mov.b64 da, {x, %3};\n mov.b64 db, {y, %3};\n"
               " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p0;\n"
               "}"
               ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc) : "memory");
}
// d (+)= A B over 64 values, A in tensor memory
XM_DEV void tc_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p0, p1;\n .reg .b64 db;\n .reg .b32 x, y;\n"
               " setp.eq.b32 p0, 0, 0;\n setp.ne.b32 p1, %5, 0;\n"
               " mov.b64 db, {%2, %3};\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p1;\n"
               " add.u32 x, %1, 8;\n add.u32 y, %2, 128;\n mov.b64 db, {y, %3};\n tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, p0;\n"
               " add.u32 x, %1, 16;\n add.u32 y, %2, 256;\n mov.b64 db, {y, %3};\n tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, p0;\n"
               " add.u32 x, %1, 24;\n add.u32 y, %2, 384;\n mov.b64 db, {y, %3};\n tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %4, p0;\n"
               "}"
               ::"r"(d), "r"(a), "r"(b), "r"(high), "r"(idesc), "r"(accumulate) : "memory");
}
XM_DEV void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
XM_DEV void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
XM_DEV void tmem_ld1(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
}
XM_DEV void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
XM_DEV void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
XM_DEV void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
XM_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 128-byte swizzle descriptors: rows of 128 bytes, groups of 8 rows 1024 bytes apart.  Inner dimension
// contiguous (Q, K): the start moves by 32 bytes for 16 values; outer dimension contiguous (V: 64 values a
// row, rows along the inner dimension): blocks of 64 outer values `block` bytes apart, the start moves by
// 2048 bytes for 16 rows.
XM_DEV uint64_t desc_sw128(uint32_t addr, uint32_t block) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | (uint64_t)((block >> 4) & 0x3fffu) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// fp16 x fp16 -> fp32, M = 128, N = n; b_outer: B's outer dimension is contiguous
__host__ __device__ constexpr uint32_t idesc_f16(int n, bool b_outer) {
  return 1u << 4 | (b_outer ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(128 >> 4) << 24;
}

struct PromptInfo {           // of the unit in a stage, written by the loaders
  uint32_t bad[4];            // keys on a page outside the pool
  uint32_t odd[4];            // keys whose values are not finite, taken out of the product
  int k_exp, v_exp;           // the unit's keys / values are scaled by 2^-exp
};

template <int D>
struct PromptShape {
  static constexpr int kTile = 128 * 2 * D;                        // bytes of 128 fp16 rows
  static constexpr int kBlock = 128 * 128;                         // of 64 of their columns
  static constexpr int kSmem = 1024 + 2 * kTile + 4 * kTile + 512;   // Q0 Q1 | K x 2 | V x 2 | barriers
};

struct PromptCtl {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2][2], p_full[2][2], o_done[2][2], drain[2];
  PromptInfo info[2];
  uint32_t tmem;
};

// eight codes of a word of keys as d (c - 8), in the order 0 4 1 5 2 6 3 7; of a word of values, whose halves
// are two blocks (d = their scales), in the order 0 0' 1 1' 2 2' 3 3'
XM_DEV uint4 decode_word(uint32_t w, __half2 d) {
  const uint32_t x = w >> 8, magic = 0x64006400u;       // 1024 + c, 1024 + 16 c
  const uint32_t a = (w & 0x000f000fu) | magic, b = (w & 0x00f000f0u) | magic;
  const uint32_t c = (x & 0x000f000fu) | magic, e = (x & 0x00f000f0u) | magic;
  auto h2 = [](uint32_t v) { return *reinterpret_cast<const __half2*>(&v); };
  auto bits = [](__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); };
  const __half2 off = __float2half2_rn(-1032.f), six = __float2half2_rn(0.0625f), off16 = __float2half2_rn(-72.f);
  return make_uint4(bits(__hmul2(__hadd2(h2(a), off), d)), bits(__hmul2(__hfma2(h2(b), six, off16), d)),
                    bits(__hmul2(__hadd2(h2(c), off), d)), bits(__hmul2(__hfma2(h2(e), six, off16), d)));
}

// A wait that tests once before it suspends (on a phase that is over that is half the time).
XM_DEV bool mbar_wait_soon(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return ok || mbar_wait_bounded(bar, parity);
}

// One lane of the warp, so that the compiler knows that it is one: what only a uniform register can give an instruction
// (the descriptors of a product) is otherwise brought there by a loop over the active lanes.
XM_DEV bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}

// 2^y on the multipliers: y = k + r, |r| <= 1/2, Taylor's polynomial of degree 5 (2.4e-6 of the value; the weights are
// rounded to fp16).  A prompt of 8192 tokens in a captured graph, 4 bits (fp16): with none of the weights this way 684 us
// (797), an eighth 664 (827), a quarter 679 (856), three eighths 675 (895).  NaN stays NaN; below 2^-126 it is 2^-126 (a weight of 0 in fp16, and nothing in
// a sum whose largest term is at least 2^-8).
XM_DEV float2 ex2_fma(float2 y) {
  auto both = [](float v) { return make_float2(v, v); };
  asm("max.NaN.f32 %0, %0, 0fC2FC0000;\n max.NaN.f32 %1, %1, 0fC2FC0000;" : "+f"(y.x), "+f"(y.y));
  const float2 k = __fadd2_rn(y, both(12582912.f));          // 1.5 2^23: rounds to a whole number
  const float2 r = __ffma2_rn(__fadd2_rn(k, both(-12582912.f)), both(-1.f), y);
  float2 p = __ffma2_rn(r, both(1.3333558e-3f), both(9.6181291e-3f));        // ln(2)^i / i!
  p = __ffma2_rn(r, p, both(5.5504109e-2f));
  p = __ffma2_rn(r, p, both(0.24022651f));
  p = __ffma2_rn(r, p, both(0.69314718f));
  p = __ffma2_rn(r, p, both(1.f));
  return __fmul2_rn(p, make_float2(__uint_as_float((__float_as_uint(k.x) << 23) + 0x3f800000u),
                                   __uint_as_float((__float_as_uint(k.y) << 23) + 0x3f800000u)));
}

// the lowest n of 64 bits (any n)
XM_DEV uint64_t below(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

XM_DEV bool loader_any(bool p) {                       // over the 128 loader threads
  uint32_t r;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"((uint32_t)p) : "memory");
  return r != 0;
}

template <typename QT_, int D, int KV, int R>
__global__ void __launch_bounds__(kPromptThreads, 1) k_kv_prompt(const KvView kv, const AttnArgs a, const DecArgs da) {
  using Shape = PromptShape<D>;
  constexpr int NG = D / 32;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ uint8_t prompt_smem[];
  const uint32_t base = (smem_u32(prompt_smem) + 1023u) & ~1023u;
  uint8_t* const base_p = prompt_smem + (base - smem_u32(prompt_smem));
  const uint32_t s_q = base, s_k = s_q + 2 * Shape::kTile, s_v = s_k + 2 * Shape::kTile;
  PromptCtl* ctl = reinterpret_cast<PromptCtl*>(base_p + 6 * Shape::kTile);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dep_wait();
  grid_dep_launch();
  const int G = a.Hq / kv.Hk, hk = blockIdx.x % kv.Hk;
  int rt, q_len;
  int64_t t0;
  // the last tiles of a sequence see the most keys: they start first
  const int s = find_tile<R>(kv, a.T, G, (int)((gridDim.x - 1 - blockIdx.x) / kv.Hk), rt, t0, q_len);
  if (s < 0) return;
  const TileSpan ts = tile_span<R, kUnit>(kv, a, s, t0, q_len, rt, G);
  if (ts.past_table && tid == 0) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
  // this CTA's part of the units (a plan of one part takes them all)
  const int chunk = da.part_units(ts.n), parts = (ts.n + chunk - 1) / chunk, split = blockIdx.y;
  if (split > 0 && split >= parts) return;
  const int v_lo = split * chunk, n = min(ts.n, v_lo + chunk) - v_lo;
  const int tiles = ts.rows > 128 ? 2 : 1;
  const int* table = kv.table + (int64_t)s * kv.table_stride;
  const uint8_t* pool = kv.pool + (int64_t)hk * kv.head_bytes;
  const int64_t page_bytes = kv.head_bytes * kv.Hk, v_part = kv.head_bytes / 2;

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->k_full[i], 128);
      mbar_init(&ctl->v_full[i], 128);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&ctl->s_full[i][h], 1);
        mbar_init(&ctl->p_full[i][h], 128);
        mbar_init(&ctl->o_done[i][h], 1);
      }
      mbar_init(&ctl->k_empty[i], tiles);
      mbar_init(&ctl->v_empty[i], tiles);
    }
    mbar_init(&ctl->drain[0], 1);
    mbar_init(&ctl->drain[1], 1);
    fence_mbar_init();
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // q: a softmax thread brings its row, scaled by a power of two, into the swizzled tile
  float q_f = 0.f;
  const int tile = warp >> 2, row = tid & 127, gr = ts.r0 + 128 * tile + row;
  const bool live = warp < 8 && 128 * tile + row < ts.rows;
  const int64_t my_t = t0 + gr / G;
  const int my_h = hk * G + gr % G, pos = live ? ts.p_first + gr / G : ts.pmax;
  if (warp < 8 && tile < tiles) {
    // 64 values at a time; twice, for the largest magnitude and for the tile (the second time from L1)
    const QT_* q = (const QT_*)a.q + my_t * a.q_stride + (int64_t)my_h * D;
    uint4 raw[8];
    auto read = [&](int c0) {
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        raw[c] = make_uint4(0u, 0u, 0u, 0u);
        if (live) {
          if (a.q_vec) {
            raw[c] = __ldg(reinterpret_cast<const uint4*>(q) + c0 + c);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<QT_*>(&raw[c])[i] = q[8 * (c0 + c) + i];
          }
        }
      }
    };
    float mx = 0.f;
#pragma unroll 1
    for (int c0 = 0; c0 < D / 8; c0 += 8) {
      read(c0);
#pragma unroll
      for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(to_f32(reinterpret_cast<const QT_*>(&raw[c])[i])));
    }
    const int sh = fp16_row_shift(mx);
    const float down = a.scale < 0.f ? -ldexpf(1.f, -sh) : ldexpf(1.f, -sh);
    q_f = fmaxf(ldexpf(fabsf(a.scale) * kLog2e, sh), 1.1754944e-38f);
#pragma unroll 1
    for (int c0 = 0; c0 < D / 8; c0 += 8) {
      if (D > 64) read(c0);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(reinterpret_cast<const QT_*>(&raw[c])[i]) * down;
        uint4 w;
        if constexpr (KV == XM_KV_Q4_0)
          w = make_uint4(half2_bits(x[0], x[4]), half2_bits(x[1], x[5]), half2_bits(x[2], x[6]), half2_bits(x[3], x[7]));
        else
          w = make_uint4(half2_bits(x[0], x[1]), half2_bits(x[2], x[3]), half2_bits(x[4], x[5]), half2_bits(x[6], x[7]));
        *reinterpret_cast<uint4*>(base_p + tile * Shape::kTile + (c0 / 8) * Shape::kBlock + row * 128 +
                                  (c ^ (row & 7)) * 16) = w;
      }
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;

  if (warp >= 12) {
    const int i = warp - 12;                           // the row tile whose products this thread issues
    if (i < tiles && n > 0 && elect_one()) {
      constexpr uint32_t id_s = idesc_f16(64, false), id_o = idesc_f16(D, true), kHalf = 64 * 128 >> 4;
      const uint32_t high = (uint32_t)(desc_sw128(0, 16) >> 32);
      const uint32_t lo_q = (uint32_t)desc_sw128(s_q + i * Shape::kTile, 16), lo_k = (uint32_t)desc_sw128(s_k, 16);
      const uint32_t lo_v = (uint32_t)desc_sw128(s_v, Shape::kBlock);
      const uint32_t t_s = tmem + i * 128, t_o = tmem + 256 + i * D;
      bool ok = true;
      auto issue_s = [&](int u) {                      // S = Q K^T of half unit u
        const int k = u >> 1, h = u & 1;
        if (h == 0) ok = mbar_wait_soon(&ctl->k_full[k & 1], (k >> 1) & 1);
        if (!ok) return;
        tc_fence_after();
        tc_mma_ss<D / 16>(t_s + 64 * h, lo_q, lo_k + (k & 1) * (Shape::kTile >> 4) + h * kHalf, high, id_s);
        tc_commit(&ctl->s_full[i][h]);
        if (h == 1) tc_commit(&ctl->k_empty[k & 1]);
      };
      issue_s(0);
      for (int u = 0; u < 2 * n && ok; ++u) {
        const int k = u >> 1, h = u & 1;
        if (u + 1 < 2 * n) {
          // the other buffer's P has been read when the last product is done
          if (u > 0) ok = mbar_wait_soon(&ctl->o_done[i][h ^ 1], ((u - 1) >> 1) & 1);
          if (ok) issue_s(u + 1);
        }
        if (ok && h == 0) ok = mbar_wait_soon(&ctl->v_full[k & 1], (k >> 1) & 1);
        // (the first half starts O, unless the softmax warps have put taken-out values there)
        const uint32_t* odd = ctl->info[0].odd;
        const bool start = u == 0 && (odd[0] | odd[1]) == 0u;
        if (ok) ok = mbar_wait_soon(&ctl->p_full[i][h], k & 1);
        if (!ok) break;
        tc_fence_after();
        tc_mma_ts(t_o, t_s + 64 * h, lo_v + (k & 1) * (Shape::kTile >> 4) + h * kHalf, high, id_o, !start);
        tc_commit(&ctl->o_done[i][h]);
        if (h == 1) tc_commit(&ctl->v_empty[k & 1]);
      }
      tc_commit(&ctl->drain[i]);                       // nothing of the tensor core's is left in flight
      mbar_wait_bounded(&ctl->drain[i], 0);
    }
    __syncwarp();
  } else if (warp >= 8) {
    const int t = tid - 256;                           // key of a unit (4-bit)
    bool ok = true;
    auto any_sees = [&](int key) {
      return key <= ts.pmax && (a.window == 0 || key > ts.pmin - a.window || key < a.sinks);
    };
    auto all_see = [&](int key) {
      return key <= ts.pmin && (a.window == 0 || key > ts.pmax - a.window || key < a.sinks);
    };
    auto page_of = [&](int key) {
      const int at = key >> kv.page_shift;
      return at < kv.table_width ? __ldg(table + at) : -1;
    };
    auto in_pool = [&](int p) { return (unsigned)p < (unsigned)kv.pages; };
    const int page_mask = (1 << kv.page_shift) - 1;
    if constexpr (KV == XM_KV_Q4_0) {
      // a thread is a key; its page is requested two units ahead, its bytes one (each part when the last is decoded)
      struct Raw {
        uint32_t kw[D / 8], vw[D / 8], kd[NG / 2], vd[NG / 2];
      };
      const int codes = D / 2 << kv.page_shift;
      auto key_of_unit = [&](int k) { return ts.unit(v_lo + min(k, n - 1)) * kUnit + t; };
      auto request = [&](const uint8_t* q, int slot, uint32_t (&w)[D / 8], uint32_t (&d)[NG / 2]) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(q + slot * (D / 2)) + i);
          w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) d[i] = __ldg(reinterpret_cast<const uint32_t*>(q + codes + slot * (2 * NG)) + i);
      };
      int next_page = n > 0 ? page_of(key_of_unit(0)) : -1, slot = 0;
      bool in = false;
      const uint8_t* head = nullptr;
      auto place = [&](int k) {                        // of unit k, whose page has arrived
        in = in_pool(next_page);
        head = pool + (in ? next_page : 0) * page_bytes;
        slot = key_of_unit(k) & page_mask;
        next_page = page_of(key_of_unit(k + 1));
      };
      Raw x;
      if (n > 0) {
        place(0);
        request(head, slot, x.kw, x.kd);
        request(head + v_part, slot, x.vw, x.vd);
      }
      for (int k = 0; k < n; ++k) {                    // (a wait that gives up is not repeated; the barriers go on)
        const int st = k & 1, key = key_of_unit(k);
        const bool seen = in && any_sees(key), bad = !in && any_sees(key);
        bool odd = false;
        uint32_t mk = 0, mv = 0;
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) {
          if (!seen) x.kd[i] = x.vd[i] = 0u;
          mk = __vmaxu2(mk, x.kd[i] & 0x7fff7fffu);
          mv = __vmaxu2(mv, x.vd[i] & 0x7fff7fffu);
        }
        mk = max(mk & 0xffffu, mk >> 16);
        mv = max(mv & 0xffffu, mv >> 16);
        if (mv >= 0x7c00u && !all_see(key)) {
          odd = true;
          mv = 0;
#pragma unroll
          for (int i = 0; i < NG / 2; ++i) x.vd[i] = 0u;
        }
        const bool big_k = loader_any(mk > 0x6c00u), big_v = loader_any(mv > 0x6c00u);     // 4096
        if (k >= 2 && ok) ok = mbar_wait_soon(&ctl->k_empty[st], ((k >> 1) - 1) & 1);
        const __half2 down_k = __float2half2_rn(big_k ? 0.0625f : 1.f), down_v = __float2half2_rn(big_v ? 0.0625f : 1.f);
        uint8_t* to = base_p + (s_k - base) + st * Shape::kTile + t * 128;
#pragma unroll
        for (int p = 0; p < D / 8; ++p) {              // word p: block p % NG, quarter p / NG
          const int g = p % NG, c = 4 * g + p / NG;    // 16-byte chunk of the row: values 8 c ...
          const __half2 dw = *reinterpret_cast<const __half2*>(&x.kd[g / 2]);
          const __half2 d2 = __hmul2(g & 1 ? __high2half2(dw) : __low2half2(dw), down_k);
          *reinterpret_cast<uint4*>(to + (c / 8) * Shape::kBlock + ((c & 7) ^ (t & 7)) * 16) = decode_word(x.kw[p], d2);
        }
        fence_proxy_async_smem();
        mbar_arrive(&ctl->k_full[st]);
        uint32_t vd[NG / 2];
#pragma unroll
        for (int i = 0; i < NG / 2; ++i) vd[i] = x.vd[i];
        if (k + 1 < n) {
          place(k + 1);
          request(head, slot, x.kw, x.kd);
        }
        if (k >= 2 && ok) ok = mbar_wait_soon(&ctl->v_empty[st], ((k >> 1) - 1) & 1);
        to = base_p + (s_v - base) + st * Shape::kTile + t * 128;
#pragma unroll
        for (int p = 0; p < D / 8; ++p) {              // word p is chunk p: columns 8 p ...
          const __half2 dw = *reinterpret_cast<const __half2*>(&vd[p % (NG / 2)]);
          *reinterpret_cast<uint4*>(to + (p / 8) * Shape::kBlock + ((p & 7) ^ (t & 7)) * 16) =
              decode_word(x.vw[p], __hmul2(dw, down_v));
        }
        const unsigned bad_w = __ballot_sync(0xffffffffu, bad), odd_w = __ballot_sync(0xffffffffu, odd);
        if (lane == 0) {
          ctl->info[st].bad[warp - 8] = bad_w;
          ctl->info[st].odd[warp - 8] = odd_w;
          if (bad_w) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
        }
        if (t == 0) {
          ctl->info[st].k_exp = big_k ? 4 : 0;
          ctl->info[st].v_exp = big_v ? 4 : 0;
        }
        fence_proxy_async_smem();
        mbar_arrive(&ctl->v_full[st]);
        if (k + 1 < n) request(head + v_part, slot, x.vw, x.vd);
      }
    } else {
      constexpr int P = D / 8;                         // 16-byte chunks of a row
      constexpr int kRowsAtOnce = 128 / P, kIter = 128 / kRowsAtOnce;
      const int c = t % P, r0 = t / P;
      // lane j of a warp holds the page of the unit's keys 16 j ...
      auto pages_of = [&](int k) { return lane < 8 ? page_of(ts.unit(v_lo + min(k, n - 1)) * kUnit + 16 * lane) : -1; };
      // the copies of one part of a unit: chunk c of rows r0, r0 + kRowsAtOnce, ...
      auto copy = [&](int k, int pages, int64_t part, uint32_t to, uint32_t& bad) {
        const int key0 = ts.unit(v_lo + k) * kUnit;
#pragma unroll
        for (int i = 0; i < kIter; ++i) {
          const int r = r0 + i * kRowsAtOnce, key = key0 + r;
          const int p = __shfl_sync(0xffffffffu, pages, r >> 4);
          const bool in = in_pool(p), seen = any_sees(key);
          if (!in && seen) bad |= 1u << i;
          const uint32_t dst = to + (c / 8) * Shape::kBlock + r * 128 + ((c & 7) ^ (r & 7)) * 16;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                       ::"r"(dst), "l"(pool + (in ? p : 0) * page_bytes + part + (key & page_mask) * (2 * D) + c * 16),
                         "r"(in && seen ? 16u : 0u) : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      // each part of the next unit is requested as soon as its stage is free, K before V
      uint32_t bad_next = 0, bad_now = 0, none = 0;
      int pages = -1;                                  // of the next unit
      if (n > 0) {
        pages = pages_of(0);
        copy(0, pages, 0, s_k, bad_next);
        copy(0, pages, v_part, s_v, none);
        pages = pages_of(1);
      }
      for (int k = 0; k < n; ++k) {                    // (a wait that gives up is not repeated; the barriers go on)
        const int st = k & 1;
        bad_now = bad_next;
        bad_next = 0;
        asm volatile("cp.async.wait_group 1;" ::: "memory");           // K(k)
        fence_proxy_async_smem();
        mbar_arrive(&ctl->k_full[st]);
        if (k + 1 < n) {
          if (k >= 1 && ok) ok = mbar_wait_soon(&ctl->k_empty[st ^ 1], (((k + 1) >> 1) - 1) & 1);
          copy(k + 1, pages, 0, s_k + (st ^ 1) * Shape::kTile, bad_next);
          asm volatile("cp.async.wait_group 1;" ::: "memory");         // V(k)
        } else {
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        // partly seen units: values that are not finite leave the product
        const int key0 = ts.unit(v_lo + k) * kUnit;
        const bool whole = key0 + kUnit - 1 <= ts.pmin &&
                           (a.window == 0 || key0 > ts.pmax - a.window || key0 + kUnit <= a.sinks);
        if (t < 4) ctl->info[st].bad[t] = ctl->info[st].odd[t] = 0u;
        if (t == 0) ctl->info[st].k_exp = ctl->info[st].v_exp = 0;
        if (loader_any(!whole || bad_now)) {           // (also the barrier behind the zeros above)
          for (int i = 0; i < kIter; ++i) {
            const int r = r0 + i * kRowsAtOnce;
            if (bad_now >> i & 1u) atomicOr(&ctl->info[st].bad[r >> 5], 1u << (r & 31));
            if (all_see(key0 + r)) continue;
            uint4* at = reinterpret_cast<uint4*>(base_p + (s_v - base) + st * Shape::kTile + (c / 8) * Shape::kBlock + r * 128 +
                                                 ((c & 7) ^ (r & 7)) * 16);
            const uint4 v = *at;
            if (non_finite(v.x) || non_finite(v.y) || non_finite(v.z) || non_finite(v.w))
              atomicOr(&ctl->info[st].odd[r >> 5], 1u << (r & 31));
          }
          loader_any(false);
          for (int i = 0; i < kIter; ++i) {
            const int r = r0 + i * kRowsAtOnce;
            if (ctl->info[st].odd[r >> 5] >> (r & 31) & 1u)
              *reinterpret_cast<uint4*>(base_p + (s_v - base) + st * Shape::kTile + (c / 8) * Shape::kBlock + r * 128 +
                                        ((c & 7) ^ (r & 7)) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          if (bad_now) atomicOr(&g_xm_device_error, XM_DEVERR_PAGE);
        }
        fence_proxy_async_smem();
        mbar_arrive(&ctl->v_full[st]);
        if (k + 1 < n) {
          if (k >= 1 && ok) ok = mbar_wait_soon(&ctl->v_empty[st ^ 1], (((k + 1) >> 1) - 1) & 1);
          copy(k + 1, pages, v_part, s_v + (st ^ 1) * Shape::kTile, none);
          pages = pages_of(k + 2);
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
  } else if (tile < tiles) {
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;             // this warp's 32 lanes of tensor memory
    const uint32_t t_s = tmem + tile * 128 + lanes, t_o = tmem + 256 + tile * D + lanes;
    // the tile's own rows decide which units need a mask
    const int last = min(ts.rows, 128 * tile + 128) - 1;
    const int pmin = ts.p_first + (ts.r0 + 128 * tile) / G, pmax = ts.p_first + (ts.r0 + last) / G;
    float ref = -INFINITY, l = 0.f;
    bool ok = true;
    for (int u = 0; u < 2 * n; ++u) {
      const int k = u >> 1, h = u & 1, st = k & 1, key0 = ts.unit(v_lo + k) * kUnit + 64 * h;
      ok = (h == 1 || mbar_wait_soon(&ctl->v_full[st], (k >> 1) & 1)) && mbar_wait_soon(&ctl->s_full[tile][h], k & 1);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t v[64];
      {
        uint32_t(&va)[32] = *reinterpret_cast<uint32_t(*)[32]>(&v[0]);
        uint32_t(&vb)[32] = *reinterpret_cast<uint32_t(*)[32]>(&v[32]);
        tmem_ld32(t_s + 64 * h, va);
        tmem_ld32(t_s + 64 * h + 32, vb);
      }
      const PromptInfo& info = ctl->info[st];
      const uint32_t bad0 = info.bad[2 * h], bad1 = info.bad[2 * h + 1], any_odd = info.odd[2 * h] | info.odd[2 * h + 1];
      const bool whole = !(bad0 | bad1) && key0 + 63 <= pmin &&
                         (a.window == 0 || key0 > pmax - a.window || key0 + 64 <= a.sinks);
      const float f = info.k_exp ? q_f * 16.f : q_f;    // never 0: hidden scores stay -inf
      // columns hi .. and, with a window, sk .. lo are hidden from this row
      const int hi = pos - key0, lo = a.window > 0 ? pos - a.window - key0 : -1, sk = a.window > 0 ? a.sinks - key0 : 0;
      tmem_ld_wait();
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      if (!whole) {
        // a bit for each column that this row sees: two instructions a column
        const uint64_t seen = below(hi + 1) & ~(below(lo + 1) & ~below(sk)) & ~((uint64_t)bad1 << 32 | bad0);
        const uint32_t s0 = (uint32_t)seen, s1 = (uint32_t)(seen >> 32);
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (!((c < 32 ? s0 : s1) & 1u << (c & 31))) v[c] = 0xff800000u;
      }
#pragma unroll
      for (int i = 0; i < 64; i += 8)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          m4[j] = fmaxf(m4[j], fmaxf(__uint_as_float(v[i + 2 * j]), __uint_as_float(v[i + 2 * j + 1])));
      const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      const float want = m == -INFINITY ? m : m * f;
      const bool move = want > ref + 8.f;
      const float was = ref;
      if (move) ref = want;
      const float al = was == ref ? 1.f : ex2(was - ref);
      l *= al;
      if (any_odd || (u > 0 && __any_sync(0xffffffffu, move))) {
        if (u > 0) {
          ok = mbar_wait_soon(&ctl->o_done[tile][h ^ 1], ((u - 1) >> 1) & 1);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc_fence_after();
        }
        const float at0 = ref == -INFINITY ? 0.f : ref;
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 8) {
          uint32_t o[8];
          if (u > 0) {
            tmem_ld8(t_o + c0, o);
            tmem_ld_wait();
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = u > 0 ? __float_as_uint(__uint_as_float(o[i]) * al) : 0u;
          if (any_odd) {
            for (int w = 0; w < 2; ++w)
              for (uint32_t left = info.odd[2 * h + w]; left; left &= left - 1) {
                const int c = 32 * w + __ffs(left) - 1;
                uint32_t x;
                tmem_ld1(t_s + 64 * h + c, x);
                tmem_ld_wait();
                // (a row that does not see the key adds nothing, not zero times it)
                const bool see = !(c > hi || (c <= lo && c >= sk));
                const float p = ex2(fmaf(__uint_as_float(x), f, -at0));
                const int key = key0 + c;
                const uint8_t* head = pool + __ldg(table + (key >> kv.page_shift)) * page_bytes + v_part;
                const int slot = key & ((1 << kv.page_shift) - 1);
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                  float val;
                  if constexpr (KV == XM_KV_Q4_0) {    // column 8 q + 2 e + b is value e of block 2 (q % (NG / 2)) + b
                    const int q = (c0 + i) >> 3, e = ((c0 + i) >> 1) & 3, b = i & 1;
                    const int blk = 2 * (q % (NG / 2)) + b;
                    const uint32_t word = __ldg(reinterpret_cast<const uint32_t*>(head + slot * (D / 2)) + q);
                    const int code = (word >> (16 * b + 4 * e)) & 15;
                    const __half d = reinterpret_cast<const __half*>(head + (D / 2 << kv.page_shift))[slot * NG + blk];
                    val = __half2float(d) * (float)(code - 8);
                  } else {
                    val = __half2float(reinterpret_cast<const __half*>(head)[slot * D + c0 + i]);
                  }
#pragma unroll
                  for (int j = 0; j < 8; ++j)
                    if (j == i && see) o[j] = __float_as_uint(fmaf(p, val, __uint_as_float(o[j])));
                }
                __syncwarp();
              }
          }
          tmem_st8(t_o + c0, o);
        }
        tmem_st_wait();
      }
      // P in place of S; scaled up where the values are scaled down
      const float at = ref == -INFINITY ? 0.f : ref, down = info.v_exp ? 4.f - at : -at;
      const float2 ff = make_float2(f, f), sh = make_float2(down, down);
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
      for (int i = 0; i < 64; i += 2) {
        const float2 y = __ffma2_rn(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), ff, sh);
        // one pair of eight without the function unit
        const float2 z = i % 16 == 6 ? ex2_fma(y) : make_float2(ex2(y.x), ex2(y.y));
        if (i & 2) s1 = __fadd2_rn(s1, z); else s0 = __fadd2_rn(s0, z);
        v[i >> 1] = half2_bits(z.x, z.y);
      }
      tmem_st32(t_s + 64 * h, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
      l = fmaf((s0.x + s0.y) + (s1.x + s1.y), info.v_exp ? 0.0625f : 1.f, l);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&ctl->p_full[tile][h]);
    }
    // O / l
    if (n > 0 && ok) ok = mbar_wait_soon(&ctl->o_done[tile][1], (n - 1) & 1);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    const float inv = parts > 1 ? 1.f : ref == -INFINITY ? 0.f : 1.0f / l;
    if (live && parts > 1) da.part_ml[((int64_t)split * a.T + my_t) * a.Hq + my_h] = make_float2(ref, l);
    QT_* out = (QT_*)a.out + my_t * a.out_stride + (int64_t)my_h * D;
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 32) {
      uint32_t v[32];
      if (n > 0 && ok) {
        tmem_ld32(t_o + c0, v);
        tmem_ld_wait();
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0u;
      }
      // eight neighbouring values at a time
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float x[8];
        int dim;
        if constexpr (KV == XM_KV_Q4_0) {              // columns c0 ..: eighths c0 / 8 .. of every block
          // words q = c0 / 8 + 0..3; with n = q / (NG / 2), halves b: block 2 (q % (NG / 2)) + b
          constexpr int PER = NG / 2;                  // words of an eighth
          constexpr int EI = 4 / PER;                  // eighths in 32 columns: values 4 n ... 4 n + 3 of each block
          const int blk = EI == 2 ? b : b % NG, first = EI == 2 ? 0 : 2 * (b / NG);
          dim = 32 * blk + 4 * (c0 / 8 / PER + first);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int word = (first + e / 4) * PER + blk / 2;
            x[e] = __uint_as_float(v[8 * word + 2 * (e & 3) + (blk & 1)]) * inv;
          }
        } else {
          dim = c0 + 8 * b;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(v[8 * b + e]) * inv;
        }
        if (live && parts > 1) {
          float* const part = da.part_o + (((int64_t)split * a.T + my_t) * a.Hq + my_h) * D + dim;
          *reinterpret_cast<float4*>(part) = make_float4(x[0], x[1], x[2], x[3]);
          *reinterpret_cast<float4*>(part + 4) = make_float4(x[4], x[5], x[6], x[7]);
        } else if (live) {
          put_out4<QT_>(out + dim, a.out_vec, make_float4(x[0], x[1], x[2], x[3]));
          put_out4<QT_>(out + dim + 4, a.out_vec, make_float4(x[4], x[5], x[6], x[7]));
        }
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename QT_, int D, int KV, int R>
int prompt_kernel(const KvView& kv, const AttnArgs& a, const DecArgs& da, int64_t tiles, cudaStream_t st) {
  constexpr int smem = PromptShape<D>::kSmem;
  static bool done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(k_kv_prompt<QT_, D, KV, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "kv attention: smem attribute: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) done[dev] = true;
  }
  return kv_launch("kv attention", k_kv_prompt<QT_, D, KV, R>, dim3((unsigned)(tiles * kv.Hk), (unsigned)da.nsplit), 1, kPromptThreads,
                   smem, st, kv, a, da);
}

template <typename QT_, int D, int KV>
int prompt_launch(const KvView& kv, const AttnArgs& a, const DecPlan& p, void* ws, cudaStream_t st) {
  DecArgs da{p.chunk / kUnit, p.nsplit, nullptr, nullptr};
  if (p.rows == 256) return prompt_kernel<QT_, D, KV, 256>(kv, a, da, p.tiles, st);
  if (p.ws_bytes) {
    da.part_o = (float*)ws;
    da.part_ml = (float2*)(da.part_o + (int64_t)p.nsplit * a.T * a.Hq * D);
  }
  const int rc = prompt_kernel<QT_, D, KV, 128>(kv, a, da, p.tiles, st);
  if (rc || p.nsplit == 1) return rc;
  return kv_launch("kv attention merge", k_kv_merge<QT_, D, 128, kUnit>, dim3((unsigned)(a.T * a.Hq)), 1, 128, 0, st, kv, a, da);
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
    return kv_type == XM_KV_F16 ? prompt_launch<QT_, 128, XM_KV_F16>(kv, a, p, ws, st)
                                : prompt_launch<QT_, 128, XM_KV_Q4_0>(kv, a, p, ws, st);
  return kv_type == XM_KV_F16 ? prompt_launch<QT_, 64, XM_KV_F16>(kv, a, p, ws, st)
                              : prompt_launch<QT_, 64, XM_KV_Q4_0>(kv, a, p, ws, st);
}

}  // namespace

extern "C" {

int64_t xm_kv_attention_workspace_size(int64_t T, int64_t B, int Hq, int Hk, int head_dim, int64_t max_keys) {
  if (T < 1 || B < 1 || Hq < 1 || Hk < 1 || Hq % Hk || max_keys < 1) return 0;
  return std::max(dec_plan(T, B, Hq, Hk, head_dim, max_keys, true).ws_bytes,
                  dec_plan(T, B, Hq, Hk, head_dim, max_keys, false).ws_bytes);
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
  if (!std::isfinite(scale)) return xm_set_error(XM_ERR_INVALID, "kv_attention: the scale is not finite");
  if (T == 0) return XM_OK;
  if (!d_q || !d_out) return xm_set_error(XM_ERR_INVALID, "kv_attention: null pointer");
  if (q_stride < (int64_t)Hq * head_dim || out_stride < (int64_t)Hq * head_dim || (((uintptr_t)d_q | (uintptr_t)d_out) & 1))
    return xm_set_error(XM_ERR_INVALID, "kv_attention: bad row pitch or alignment");
  const int64_t need = xm_kv_attention_workspace_size(T, B, Hq, Hk, head_dim, table_width * page_size);
  if (need && (ws_bytes < need || !d_ws || ((uintptr_t)d_ws & 15)))
    return xm_set_error(XM_ERR_INVALID, "kv_attention: workspace too small or unaligned");
  const int64_t most = 1 << 30;                      // as good as none
  AttnArgs a{d_q, T, q_stride, Hq, scale, window < most ? (int)window : 0, (int)std::min(sinks, most), d_out, out_stride,
             q_stride % 8 == 0 && ((uintptr_t)d_q & 15) == 0, out_stride % 4 == 0 && ((uintptr_t)d_out & 7) == 0};
  cudaStream_t st = (cudaStream_t)stream;
  return q_dtype == XM_DT_F16 ? attn_typed<__half>(kv, a, kv_type, head_dim, d_ws, st)
                              : attn_typed<__nv_bfloat16>(kv, a, kv_type, head_dim, d_ws, st);
}

}  // extern "C"
