// Residual addition with its root-mean-square norm, forward and backward.
//
//   forward   t = x + r,  i = (mean(t^2) + eps)^(-1/2),  y = t i w;  outputs y, t and i
//   backward  p = dy w,   dt = ds + i p - t i^3 mean(p t),  dw = sum over rows of dy t i
//             (dt is the gradient of x and of r)
//
// Bound by HBM: forward reads x, r and writes y, t; backward reads dy, ds, t
// and writes dt.  A row belongs to TPR threads which keep it in registers
// between the sum of squares and the scaling, so every element is read once.
// dw: a fixed grid walks the rows with a stride, each thread summing its own
// columns in registers; one partial row per block goes to the workspace and a
// second kernel adds the blocks in order, so the result does not depend on
// the order of execution.
#include <algorithm>

#include "seq_common.cuh"

namespace tmpc {
namespace seq {

constexpr int kNormThreads = 256;
constexpr int kNormMaxD = 16384;

// Sum over the TPR threads of a row (TPR = 32: a warp; else the whole block).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = warp_sum(v);
  if constexpr (TPR > 32) {
    const int w = threadIdx.x >> 5;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += red[i];
  }
  return v;
}

template <typename T, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? kNormThreads : TPR)
    norm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ r, const T* __restrict__ w, T* __restrict__ y,
                    T* __restrict__ t, float* __restrict__ inv, int64_t rows, int d, int64_t xs, int64_t rs,
                    float eps) {
  using P = Pack<T, V>;
  __shared__ float red[32];
  constexpr int RPB = TPR == 32 ? kNormThreads / 32 : 1;
  const int lane = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * RPB + (TPR == 32 ? (threadIdx.x >> 5) : 0);
  if (row >= rows) return;  // whole rows leave together
  const int nv = d / V;
  float s[NV][V];
  P px[NV], pr[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + j * TPR;
    if (c < nv) {
      px[j] = reinterpret_cast<const P*>(x + row * xs)[c];
      if (r) pr[j] = reinterpret_cast<const P*>(r + row * rs)[c];
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + j * TPR;
#pragma unroll
    for (int e = 0; e < V; ++e) s[j][e] = 0.f;
    if (c < nv) {
      P o;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        s[j][e] = to_f(px[j].v[e]) + (r ? to_f(pr[j].v[e]) : 0.f);
        sq = fmaf(s[j][e], s[j][e], sq);
        o.v[e] = from_f<T>(s[j][e]);
      }
      if (t) reinterpret_cast<P*>(t + row * d)[c] = o;
    }
  }
  const float iv = rsqrtf(row_sum<TPR>(sq, red) / (float)d + eps);
  if (inv && lane == 0) inv[row] = iv;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + j * TPR;
    if (c < nv) {
      const P pw = reinterpret_cast<const P*>(w)[c];
      P o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = from_f<T>(s[j][e] * iv * to_f(pw.v[e]));
      reinterpret_cast<P*>(y + row * d)[c] = o;
    }
  }
}

template <typename T, int V, int NV, int TPR>
__global__ void __launch_bounds__(TPR == 32 ? kNormThreads : TPR)
    norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ ds, const T* __restrict__ t,
                    const T* __restrict__ w, const float* __restrict__ inv, T* __restrict__ dt,
                    float* __restrict__ dw_part, int64_t rows, int d) {
  using P = Pack<T, V>;
  __shared__ float red[32];
  constexpr int RPB = TPR == 32 ? kNormThreads / 32 : 1;
  const int lane = TPR == 32 ? (threadIdx.x & 31) : threadIdx.x;
  const int sub = TPR == 32 ? (threadIdx.x >> 5) : 0;
  const int nv = d / V;
  const float invd = 1.f / (float)d;
  float acc[NV][V];
  P pw[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + j * TPR;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[j][e] = 0.f;
    if (c < nv) pw[j] = reinterpret_cast<const P*>(w)[c];
  }
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < rows; row += (int64_t)gridDim.x * RPB) {
    P pt[NV], pd[NV], ps[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * TPR;
      if (c < nv) {
        pt[j] = reinterpret_cast<const P*>(t + row * d)[c];
        pd[j] = reinterpret_cast<const P*>(dy + row * d)[c];
        if (ds) ps[j] = reinterpret_cast<const P*>(ds + row * d)[c];
      }
    }
    const float iv = inv[row];
    float dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + j * TPR < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float a = to_f(pd[j].v[e]), b = to_f(pt[j].v[e]);
          dot = fmaf(a * to_f(pw[j].v[e]), b, dot);
          acc[j][e] = fmaf(a * iv, b, acc[j][e]);
        }
      }
    const float m = row_sum<TPR>(dot, red) * invd * iv * iv * iv;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + j * TPR < nv) {
        P o;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float g = iv * to_f(pd[j].v[e]) * to_f(pw[j].v[e]) - m * to_f(pt[j].v[e]);
          if (ds) g += to_f(ps[j].v[e]);
          o.v[e] = from_f<T>(g);
        }
        reinterpret_cast<P*>(dt + row * d)[lane + j * TPR] = o;
      }
  }
  // The block's rows in order: TPR = 32 adds the warps one after another.
  extern __shared__ float sdw[];
  if constexpr (TPR == 32) {
    for (int s = 0; s < RPB; ++s) {
      if (sub == s) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (lane + j * TPR < nv) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
              float* p = &sdw[(lane + j * TPR) * V + e];
              *p = s == 0 ? acc[j][e] : *p + acc[j][e];
            }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < d; c += kNormThreads) dw_part[(int64_t)blockIdx.x * d + c] = sdw[c];
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (lane + j * TPR < nv) {
#pragma unroll
        for (int e = 0; e < V; ++e) dw_part[(int64_t)blockIdx.x * d + (lane + j * TPR) * V + e] = acc[j][e];
      }
  }
}

// dw[c] = sum over blocks, in a fixed order: 32 columns x 32 row lanes per block.
template <typename T>
__global__ void __launch_bounds__(1024) norm_dw_kernel(const float* __restrict__ part, T* __restrict__ dw, int nblk,
                                                       int d) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float a = 0.f;
  if (c < d)
    for (int b = threadIdx.y; b < nblk; b += 32) a += part[(int64_t)b * d + c];
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  const float v = warp_sum(s[threadIdx.x][threadIdx.y]);
  const int co = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && co < d) dw[co] = from_f<T>(v);
}

// Blocks of the backward pass: eight warps each, four blocks per SM.
inline int norm_bwd_blocks(int64_t rows, int d) {
  const int rpb = d <= 1024 ? kNormThreads / 32 : 1;
  const int64_t need = (rows + rpb - 1) / rpb;
  return (int)std::min<int64_t>(need, 4 * (int64_t)sm_count());
}

// Widest access that divides the row and suits every pointer.
template <typename T>
int vec_elems(int d, int64_t xs, int64_t rs, std::initializer_list<const void*> ptrs) {
  for (int v = 16 / (int)sizeof(T); v > 1; v /= 2) {
    bool ok = d % v == 0 && xs % v == 0 && rs % v == 0;
    for (const void* p : ptrs) ok = ok && aligned(p, v * sizeof(T));
    if (ok) return v;
  }
  return 1;
}

// Calls f<V, NV, TPR>: up to 32 elements per thread, a warp per row to 1024
// columns, a block of 128 to 4096, of 512 to 16384.
template <typename T, int V, typename F>
void norm_shape(int d, F&& f) {
  const int nv = d / V;
  auto pick = [&](auto tpr) {
    constexpr int TPR = decltype(tpr)::value;
    const int per = (nv + TPR - 1) / TPR;
    if (per * V <= 8 && V <= 8) f(std::integral_constant<int, V>{}, std::integral_constant<int, 8 / V>{}, tpr);
    else if (per * V <= 16) f(std::integral_constant<int, V>{}, std::integral_constant<int, 16 / V>{}, tpr);
    else f(std::integral_constant<int, V>{}, std::integral_constant<int, 32 / V>{}, tpr);
  };
  if (d <= 1024) pick(std::integral_constant<int, 32>{});
  else if (d <= 4096) pick(std::integral_constant<int, 128>{});
  else pick(std::integral_constant<int, 512>{});
}

template <typename T, typename F>
void norm_dispatch(int v, int d, F&& f) {
  if constexpr (sizeof(T) == 2)
    if (v == 8) return norm_shape<T, 8>(d, f);
  if (v == 4) return norm_shape<T, 4>(d, f);
  if (v == 2) return norm_shape<T, 2>(d, f);
  return norm_shape<T, 1>(d, f);
}

template <typename T>
int norm_fwd(int64_t rows, int d, const T* x, int64_t xs, const T* r, int64_t rs, const T* w, double eps, T* y, T* t,
             float* inv, cudaStream_t st) {
  if (rows < 0 || rows > INT32_MAX || d < 1 || xs < 0 || rs < 0) return TMPC_ERR_BAD_DIMS;
  if (d > kNormMaxD) return TMPC_ERR_UNSUPPORTED;
  if (rows == 0) return TMPC_OK;
  if (!x || !w || !y || (r && !t)) return TMPC_ERR_NULL_ARG;
  const int v = vec_elems<T>(d, xs, r ? rs : 0, {x, r, w, y, t});
  norm_dispatch<T>(v, d, [&](auto V, auto NV, auto TPR) {
    constexpr int rpb = TPR == 32 ? kNormThreads / 32 : 1;
    norm_fwd_kernel<T, V, NV, TPR><<<(unsigned)((rows + rpb - 1) / rpb), TPR == 32 ? kNormThreads : TPR, 0, st>>>(
        x, r, w, y, t, inv, rows, d, xs, rs, (float)eps);
  });
  return (int)cudaPeekAtLastError();
}

inline size_t norm_ws(int64_t rows, int d) {
  if (rows <= 0 || d < 1) return 0;
  return (size_t)norm_bwd_blocks(rows, d) * d * sizeof(float);
}

template <typename T>
int norm_bwd(int64_t rows, int d, const T* dy, const T* ds, const T* t, const T* w, const float* inv, T* dt, T* dw,
             void* ws, size_t ws_bytes, cudaStream_t st) {
  if (rows < 0 || rows > INT32_MAX || d < 1) return TMPC_ERR_BAD_DIMS;
  if (d > kNormMaxD) return TMPC_ERR_UNSUPPORTED;
  if (!dw) return TMPC_ERR_NULL_ARG;
  if (rows == 0) return (int)cudaMemsetAsync(dw, 0, (size_t)d * sizeof(T), st);
  if (!dy || !t || !w || !inv || !dt) return TMPC_ERR_NULL_ARG;
  if (!ws || ws_bytes < norm_ws(rows, d) || !aligned(ws, 16)) return TMPC_ERR_WORKSPACE;
  const int nblk = norm_bwd_blocks(rows, d);
  const int v = vec_elems<T>(d, 0, 0, {dy, ds, t, w, dt});
  float* part = static_cast<float*>(ws);
  norm_dispatch<T>(v, d, [&](auto V, auto NV, auto TPR) {
    norm_bwd_kernel<T, V, NV, TPR><<<nblk, TPR == 32 ? kNormThreads : TPR, TPR == 32 ? d * sizeof(float) : 0, st>>>(
        dy, ds, t, w, inv, dt, part, rows, d);
  });
  norm_dw_kernel<T><<<(d + 31) / 32, dim3(32, 32), 0, st>>>(part, dw, nblk, d);
  return (int)cudaPeekAtLastError();
}

}  // namespace seq
}  // namespace tmpc

extern "C" {

#define TMPC_NORM_ENTRY(SUF, T)                                                                                      \
  int32_t tmpc_add_rms_norm_##SUF(int64_t rows, int32_t d, const void* x, int64_t x_stride, const void* residual,    \
                                  int64_t residual_stride, const void* weight, double eps, void* y, void* sum,       \
                                  float* inv_rms, tmpc_stream_t stream) {                                            \
    return tmpc::seq::norm_fwd<T>(rows, d, (const T*)x, x_stride, (const T*)residual, residual_stride,               \
                                  (const T*)weight, eps, (T*)y, (T*)sum, inv_rms, (cudaStream_t)stream);             \
  }                                                                                                                  \
  int32_t tmpc_add_rms_norm_backward_##SUF(int64_t rows, int32_t d, const void* dy, const void* dsum,                \
                                           const void* sum, const void* weight, const float* inv_rms, void* dx,      \
                                           void* dweight, void* workspace, size_t workspace_bytes,                   \
                                           tmpc_stream_t stream) {                                                   \
    return tmpc::seq::norm_bwd<T>(rows, d, (const T*)dy, (const T*)dsum, (const T*)sum, (const T*)weight, inv_rms,   \
                                  (T*)dx, (T*)dweight, workspace, workspace_bytes, (cudaStream_t)stream);            \
  }
TMPC_NORM_ENTRY(f32, float)
TMPC_NORM_ENTRY(bf16, __nv_bfloat16)

size_t tmpc_add_rms_norm_workspace_bytes(int64_t rows, int32_t d) { return tmpc::seq::norm_ws(rows, d); }

}  // extern "C"
