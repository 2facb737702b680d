// Attention over the paged key/value cache (layout: xm_kv.cuh).
//
// Row t of sequence s at position p sees the keys 0 .. p of its sequence (with a window w: those above
// p - w, and the first `sinks`); query head h reads KV head h / (Hq / Hk):
//   out = sum_k softmax_k(q . K_k * scale) V_k,  zeros for a row that sees no key.
//
// k_kv_attn: one warp per (row, query head), one pass over the keys with a running maximum and sum;
// lane l holds values 2l, 2l + 1 of each half of the head (one per half at D = 64).
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
  int64_t window, sinks;
  void* out;
  int64_t out_stride;
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
int attn_typed(const KvView& kv, const AttnArgs& a, int kv_type, int head_dim, cudaStream_t st) {
  if (head_dim == 128)
    return kv_type == XM_KV_F16 ? attn_launch<QT_, 128, XM_KV_F16>(kv, a, st) : attn_launch<QT_, 128, XM_KV_Q4_0>(kv, a, st);
  return kv_type == XM_KV_F16 ? attn_launch<QT_, 64, XM_KV_F16>(kv, a, st) : attn_launch<QT_, 64, XM_KV_Q4_0>(kv, a, st);
}

}  // namespace

extern "C" {

int64_t xm_kv_attention_workspace_size(int64_t T, int64_t B, int Hq, int Hk, int head_dim, int64_t max_keys) {
  (void)T; (void)B; (void)Hq; (void)Hk; (void)head_dim; (void)max_keys;
  return 16;
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
  if (ws_bytes < xm_kv_attention_workspace_size(T, B, Hq, Hk, head_dim, table_width * page_size) || !d_ws)
    return xm_set_error(XM_ERR_INVALID, "kv_attention: workspace too small");
  AttnArgs a{d_q, T, q_stride, Hq, scale, window, sinks, d_out, out_stride};
  cudaStream_t st = (cudaStream_t)stream;
  return q_dtype == XM_DT_F16 ? attn_typed<__half>(kv, a, kv_type, head_dim, st)
                              : attn_typed<__nv_bfloat16>(kv, a, kv_type, head_dim, st);
}

}  // extern "C"
