// What stands between two blocks: the norm of a block's output, its gate and scale, the residual add, and the norm of the
// residual stream for the next block, in one pass.
//
// Row: v = y, or y w_post / sqrt(mean y^2 + eps);  h' = h + scale gate v;  next = h' w_pre / sqrt(mean h'^2 + eps).
//
// Bound: HBM (h and y read, h' and next written, once each).  A row stays in registers from its loads to its stores, fp32
// throughout: h' is rounded to its type on the way out only, and next comes from the unrounded h'.  Rows of up to 1024 values
// take a warp each (two shuffle reductions, no barrier), longer ones a CTA of up to 1024 threads.  All loads of a row go out
// before the first sum.
//
// Measured, cold: 8192 rows of 4096 values, stream in fp32 and y in bf16, 71 to 74 us (403 MB at 5.4 to 5.6 TB/s, 0.83 to 0.86 of a
// copy); one row of them, or 64, 3.5 us in a captured graph.
#include "xm_gemv_dot.cuh"

namespace {

struct NormArgs {
  const void *h, *y, *gate;
  const float *post, *pre;
  void *out, *next;
  int64_t rows, h_pitch, y_pitch, out_pitch, next_pitch, gate_pitch;
  int64_t rows_per_gate;
  int D, gate_type, next_type;
  bool gate_wide;                 // a gate value for each column (else one for the row)
  float scale, eps;
};

// V consecutive values as fp32; the address is a multiple of min(16, V values) bytes
template <typename T, int V>
XM_DEV void ld_vec(const T* p, float* v) {
  constexpr int B = V * (int)sizeof(T), W = B / 4;
  if constexpr (W == 0) {
    v[0] = to_f32<T>(*p);
  } else {
    uint32_t r[W];
    if constexpr (B >= 16) {
#pragma unroll
      for (int i = 0; i < B / 16; ++i)
        *reinterpret_cast<uint4*>(r + 4 * i) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + 16 * i);
    } else if constexpr (B == 8) {
      *reinterpret_cast<uint2*>(r) = *reinterpret_cast<const uint2*>(p);
    } else {
      r[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        T two[2];
        *reinterpret_cast<uint32_t*>(two) = r[i];
        v[2 * i] = to_f32<T>(two[0]);
        v[2 * i + 1] = to_f32<T>(two[1]);
      }
    }
  }
}

template <typename T> XM_DEV T from_f32(float v);
template <> XM_DEV float from_f32<float>(float v) { return v; }
template <> XM_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> XM_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int V>
XM_DEV void st_vec(T* p, const float* v) {
  constexpr int B = V * (int)sizeof(T), W = B / 4;
  if constexpr (W == 0) {
    *p = from_f32<T>(v[0]);
  } else {
    alignas(16) T t[V];
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = from_f32<T>(v[i]);
    const uint32_t* r = reinterpret_cast<const uint32_t*>(t);
    if constexpr (B >= 16) {
#pragma unroll
      for (int i = 0; i < B / 16; ++i)
        *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(p) + 16 * i) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2],
                                                                                      r[4 * i + 3]);
    } else if constexpr (B == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(r[0], r[1]);
    } else {
      *reinterpret_cast<uint32_t*>(p) = r[0];
    }
  }
}

// The sum over the row's threads: a warp (the block's other warps hold other rows), or the block.
XM_DEV float row_sum(float v, float* red, bool block) {
  v = warp_sum(v);
  if (!block) return v;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += red[w];
  return v;
}

// V: values a load; NP: packs of 8 values a thread.  Vector j of the row's thread t is vector j * (threads of the row) + t.
// MAXT: threads of a block at most; three blocks on an SM where the registers allow it, for the loads that are on their way
// together.
template <typename HT, typename YT, int V, int NP, int MAXT>
__global__ void __launch_bounds__(MAXT, MAXT == 128 || (MAXT == 256 && NP == 2) ? 3 : 1) k_residual_norm(NormArgs a) {
  constexpr int NV = 8 / V * NP;
  __shared__ float red[2][32];
  grid_dep_wait();
  grid_dep_launch();
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= a.rows) return;                              // (whole warps; rows of a block of their own always exist)
  const bool block = blockDim.y == 1 && blockDim.x > 32;
  const int n = a.D / V, step = blockDim.x, t = threadIdx.x;
  const HT* h = (const HT*)a.h + row * a.h_pitch;
  const YT* y = (const YT*)a.y + row * a.y_pitch;
  float hv[NV][V], yv[NV][V];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * step + t;
    if (at < n) {
      ld_vec<YT, V>(y + (int64_t)at * V, yv[j]);
      ld_vec<HT, V>(h + (int64_t)at * V, hv[j]);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) yv[j][i] = hv[j][i] = 0.f;
    }
  }
  if (a.post) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(yv[j][i], yv[j][i], s);
    const float r = 1.0f / sqrtf(row_sum(s, red[0], block) / (float)a.D + a.eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = j * step + t;
      if (at < n) {
        float w[V];
        ld_vec<float, V>(a.post + (int64_t)at * V, w);
#pragma unroll
        for (int i = 0; i < V; ++i) yv[j][i] = yv[j][i] * r * w[i];
      }
    }
  }
  if (a.gate) {
    const int64_t g0 = row / a.rows_per_gate * a.gate_pitch;
    auto apply = [&](auto* g) {
      using GT = std::remove_const_t<std::remove_pointer_t<decltype(g)>>;
      if (a.gate_wide) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int at = j * step + t;
          if (at < n) {
            float w[V];
            ld_vec<GT, V>(g + g0 + (int64_t)at * V, w);
#pragma unroll
            for (int i = 0; i < V; ++i) yv[j][i] *= w[i];
          }
        }
      } else {
        const float w = to_f32<GT>(g[g0]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) yv[j][i] *= w;
      }
    };
    if (a.gate_type == XM_DT_F32) apply((const float*)a.gate);
    else if (a.gate_type == XM_DT_F16) apply((const __half*)a.gate);
    else apply((const __nv_bfloat16*)a.gate);
  }
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      hv[j][i] = fmaf(a.scale, yv[j][i], hv[j][i]);
      if (j * step + t < n) s = fmaf(hv[j][i], hv[j][i], s);
    }
  HT* out = (HT*)a.out + row * a.out_pitch;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * step + t;
    if (at < n) st_vec<HT, V>(out + (int64_t)at * V, hv[j]);
  }
  if (!a.pre) return;
  const float r = 1.0f / sqrtf(row_sum(s, red[1], block) / (float)a.D + a.eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int at = j * step + t;
    if (at < n) {
      float w[V];
      ld_vec<float, V>(a.pre + (int64_t)at * V, w);
#pragma unroll
      for (int i = 0; i < V; ++i) hv[j][i] = hv[j][i] * r * w[i];
      const int64_t o = row * a.next_pitch + (int64_t)at * V;
      if (a.next_type == XM_DT_F32) st_vec<float, V>((float*)a.next + o, hv[j]);
      else if (a.next_type == XM_DT_F16) st_vec<__half, V>((__half*)a.next + o, hv[j]);
      else st_vec<__nv_bfloat16, V>((__nv_bfloat16*)a.next + o, hv[j]);
    }
  }
}

template <typename HT, typename YT, int V, int NP, int MAXT>
cudaError_t norm_launch(const NormArgs& a, cudaStream_t st) {
  const int warps = (a.D + 256 * NP - 1) / (256 * NP);
  const int rows = warps == 1 ? 4 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a.rows + rows - 1) / rows));
  cfg.blockDim = dim3(32 * warps, rows);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_residual_norm<HT, YT, V, NP, MAXT>, a);
}

template <typename HT, typename YT, int V>
cudaError_t norm_np(const NormArgs& a, cudaStream_t st) {
  // a warp a row, then blocks of up to 512 threads; 1024 threads have half of the registers each, and rows of more than
  // 16384 values do not fit into those (some spill)
  if (a.D <= 256) return norm_launch<HT, YT, V, 1, 128>(a, st);
  if (a.D <= 1024) return norm_launch<HT, YT, V, 4, 128>(a, st);
  if (a.D <= 2048) return norm_launch<HT, YT, V, 1, 256>(a, st);
  if (a.D <= 4096) return norm_launch<HT, YT, V, 2, 256>(a, st);
  if (a.D <= 8192) return norm_launch<HT, YT, V, 2, 512>(a, st);
  if (a.D <= 16384) return norm_launch<HT, YT, V, 2, 1024>(a, st);
  return norm_launch<HT, YT, V, 4, 1024>(a, st);
}

template <typename HT, typename YT>
cudaError_t norm_v(const NormArgs& a, int V, cudaStream_t st) {
  return V == 8 ? norm_np<HT, YT, 8>(a, st) : V == 2 ? norm_np<HT, YT, 2>(a, st) : norm_np<HT, YT, 1>(a, st);
}

template <typename HT>
cudaError_t norm_y(const NormArgs& a, int y_type, int V, cudaStream_t st) {
  return y_type == XM_DT_F32   ? norm_v<HT, float>(a, V, st)
         : y_type == XM_DT_F16 ? norm_v<HT, __half>(a, V, st)
                               : norm_v<HT, __nv_bfloat16>(a, V, st);
}

bool is_float_type(int t) { return t == XM_DT_F32 || t == XM_DT_F16 || t == XM_DT_BF16; }
int type_size(int t) { return t == XM_DT_F32 ? 4 : 2; }

}  // namespace

extern "C" int xm_residual_norm(const void* d_h, int h_type, int64_t h_pitch, const void* d_y, int y_type, int64_t y_pitch,
                                int64_t rows, int64_t D, const float* d_post_w, const void* d_gate, int gate_type,
                                int64_t gate_pitch, int gate_wide, int64_t rows_per_gate, float scale,
                                const float* d_pre_w, float eps, void* d_out, int64_t out_pitch, void* d_next,
                                int next_type, int64_t next_pitch, void* stream) {
  if (!is_float_type(h_type) || !is_float_type(y_type) || (d_gate && !is_float_type(gate_type)) ||
      (d_pre_w && !is_float_type(next_type)))
    return xm_set_error(XM_ERR_INVALID, "residual_norm: bad element type");
  if (rows < 0 || rows > INT32_MAX || D < 1 || D > 32768)
    return xm_set_error(XM_ERR_INVALID, "residual_norm: bad sizes (%lld rows of %lld; rows of 1 to 32768 values)",
                        (long long)rows, (long long)D);
  if (h_pitch < D || y_pitch < D || out_pitch < D || (d_pre_w && next_pitch < D))
    return xm_set_error(XM_ERR_INVALID, "residual_norm: a row pitch is below the row's %lld values", (long long)D);
  if (d_gate && (rows_per_gate < 1 || gate_pitch < 0))
    return xm_set_error(XM_ERR_INVALID, "residual_norm: bad gate");
  if (rows == 0) return XM_OK;
  if (!d_h || !d_y || !d_out || (d_pre_w && !d_next)) return xm_set_error(XM_ERR_INVALID, "residual_norm: null pointer");
  // the widest vectors that every row and weight allows: 8, 2 or 1 values
  auto fits = [&](const void* p, int64_t pitch, int size, int V) {
    const int bytes = V * size < 16 ? V * size : 16;
    return !p || (((uintptr_t)p % bytes) == 0 && pitch * size % bytes == 0);
  };
  int V = 8;
  for (; V > 1; V = V == 8 ? 2 : 1)
    if (D % V == 0 && fits(d_h, h_pitch, type_size(h_type), V) && fits(d_y, y_pitch, type_size(y_type), V) &&
        fits(d_out, out_pitch, type_size(h_type), V) && fits(d_pre_w ? d_next : nullptr, next_pitch, type_size(next_type), V) &&
        fits(gate_wide ? d_gate : nullptr, gate_pitch, type_size(gate_type), V) && fits(d_post_w, 0, 4, V) &&
        fits(d_pre_w, 0, 4, V))
      break;
  if (!fits(d_h, h_pitch, type_size(h_type), 1) || !fits(d_y, y_pitch, type_size(y_type), 1) ||
      !fits(d_out, out_pitch, type_size(h_type), 1) || !fits(d_pre_w ? d_next : nullptr, next_pitch, type_size(next_type), 1) ||
      !fits(d_gate, gate_pitch, type_size(gate_type), 1) || !fits(d_post_w, 0, 4, 1) || !fits(d_pre_w, 0, 4, 1))
    return xm_set_error(XM_ERR_INVALID, "residual_norm: unaligned pointer");
  NormArgs a{d_h, d_y, d_gate, d_post_w, d_pre_w, d_out, d_next, rows, h_pitch, y_pitch, out_pitch, next_pitch,
             gate_pitch, rows_per_gate, (int)D, gate_type, next_type, gate_wide != 0, scale, eps};
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = h_type == XM_DT_F32   ? norm_y<float>(a, y_type, V, st)
                        : h_type == XM_DT_F16 ? norm_y<__half>(a, y_type, V, st)
                                              : norm_y<__nv_bfloat16>(a, y_type, V, st);
  if (e != cudaSuccess) return xm_set_error(XM_ERR_CUDA, "residual_norm launch: %s", cudaGetErrorString(e));
  return xm_check_launch("residual_norm");
}
