// Gated linear layer, forward and backward:
//     h = act(x Wg^T) * (x Wu^T)
//     dg = dh u act'(g), du = dh act(g)
//     dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
// Tiles of 64 x 64 outputs, float products and sums.
#include "seq_common.cuh"

namespace tmpc {
namespace seq {

// act(g) and act'(g).
__device__ __forceinline__ void activation(int act, float g, float& a, float& da) {
  if (act == TMPC_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-g));
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  } else {
    const float c = 0.5f * erfcf(-0.70710678118654752f * g);
    a = g * c;
    da = c + g * 0.39894228040143268f * expf(-0.5f * g * g);
  }
}

// C[m][n] (+)= sum_k A[m sam + k sak] B[n sbn + k sbk], tile 64 x 64.
template <typename T>
struct Tile {
  float a[16][65], b[16][65];
};

template <typename T>
__device__ __forceinline__ void gemm_tile(Tile<T>& s, float (&acc)[4][4], const T* A, int64_t sam, int64_t sak,
                                          const T* B, int64_t sbn, int64_t sbk, int64_t m0, int64_t M, int n0, int N,
                                          int64_t K) {
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  for (int64_t k0 = 0; k0 < K; k0 += 16) {
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += 256) {
      const int am = sak == 1 ? e / 16 : e % 64, ak = sak == 1 ? e % 16 : e / 64;
      const int bn = sbk == 1 ? e / 16 : e % 64, bk = sbk == 1 ? e % 16 : e / 64;
      s.a[ak][am] = (m0 + am < M && k0 + ak < K) ? to_f(A[(m0 + am) * sam + (k0 + ak) * sak]) : 0.f;
      s.b[bk][bn] = (n0 + bn < N && k0 + bk < K) ? to_f(B[(int64_t)(n0 + bn) * sbn + (k0 + bk) * sbk]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(s.a[k][ty * 4 + i], s.b[k][tx * 4 + j], acc[i][j]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) gated_fwd_kernel(const T* x, const T* wg, const T* wu, T* h, T* gate, T* up,
                                                       int64_t N, int d, int f, int act) {
  __shared__ Tile<T> s;
  float g[4][4] = {}, u[4][4] = {};
  const int64_t m0 = (int64_t)blockIdx.x * 64;
  const int n0 = blockIdx.y * 64;
  gemm_tile(s, g, x, d, 1, wg, d, 1, m0, N, n0, f, d);
  gemm_tile(s, u, x, d, 1, wu, d, 1, m0, N, n0, f, d);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + (threadIdx.x / 16) * 4 + i;
      const int n = n0 + (threadIdx.x % 16) * 4 + j;
      if (m < N && n < f) {
        float a, da;
        activation(act, g[i][j], a, da);
        h[m * f + n] = from_f<T>(a * u[i][j]);
        if (gate) {
          gate[m * f + n] = from_f<T>(g[i][j]);
          up[m * f + n] = from_f<T>(u[i][j]);
        }
      }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) gated_dact_kernel(const T* gate, const T* up, const T* dh, T* dg, T* du,
                                                        int64_t n, int act) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float a, da;
    activation(act, to_f(gate[i]), a, da);
    const float y = to_f(dh[i]);
    dg[i] = from_f<T>(y * to_f(up[i]) * da);
    du[i] = from_f<T>(y * a);
  }
}

// out = A1 B1 (+ A2 B2)
template <typename T>
__global__ void __launch_bounds__(256) gemm_kernel(const T* A1, const T* B1, const T* A2, const T* B2, int64_t sam,
                                                  int64_t sak, int64_t sbn, int64_t sbk, T* out, int64_t M, int N,
                                                  int64_t K) {
  __shared__ Tile<T> s;
  float acc[4][4] = {};
  const int64_t m0 = (int64_t)blockIdx.x * 64;
  const int n0 = blockIdx.y * 64;
  gemm_tile(s, acc, A1, sam, sak, B1, sbn, sbk, m0, M, n0, N, K);
  if (A2) gemm_tile(s, acc, A2, sam, sak, B2, sbn, sbk, m0, M, n0, N, K);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + (threadIdx.x / 16) * 4 + i;
      const int n = n0 + (threadIdx.x % 16) * 4 + j;
      if (m < M && n < N) out[m * N + n] = from_f<T>(acc[i][j]);
    }
}

inline int check_gated(int64_t rows, int d, int f, int act) {
  if (rows < 0 || rows > INT32_MAX || d < 1 || f < 1) return TMPC_ERR_BAD_DIMS;
  if ((act != TMPC_ACT_SILU && act != TMPC_ACT_GELU) || d > 65536 || f > 65536) return TMPC_ERR_UNSUPPORTED;
  return TMPC_OK;
}

template <typename T>
int gated_fwd(int64_t rows, int d, int f, const T* x, const T* wg, const T* wu, int act, T* h, T* gate, T* up,
              cudaStream_t st) {
  const int rc = check_gated(rows, d, f, act);
  if (rc) return rc;
  if (rows == 0) return TMPC_OK;
  if (!x || !wg || !wu || !h || (gate == nullptr) != (up == nullptr)) return TMPC_ERR_NULL_ARG;
  gated_fwd_kernel<T><<<dim3((unsigned)((rows + 63) / 64), (f + 63) / 64), 256, 0, st>>>(x, wg, wu, h, gate, up, rows, d,
                                                                                      f, act);
  return (int)cudaPeekAtLastError();
}

inline size_t gated_bwd_ws(int64_t rows, int f, int esize) {
  return rows > 0 && f > 0 ? (size_t)2 * rows * f * esize + 16 : 0;
}

template <typename T>
int gated_bwd(int64_t rows, int d, int f, const T* x, const T* wg, const T* wu, int act, const T* gate, const T* up,
              const T* dh, T* dx, T* dwg, T* dwu, void* ws, size_t ws_bytes, cudaStream_t st) {
  const int rc = check_gated(rows, d, f, act);
  if (rc) return rc;
  if ((dwg == nullptr) != (dwu == nullptr)) return TMPC_ERR_NULL_ARG;
  if (rows == 0) {
    if (!dwg) return TMPC_OK;
    const cudaError_t e = cudaMemsetAsync(dwg, 0, (size_t)f * d * sizeof(T), st);
    return e != cudaSuccess ? (int)e : (int)cudaMemsetAsync(dwu, 0, (size_t)f * d * sizeof(T), st);
  }
  if (!x || !wg || !wu || !gate || !up || !dh) return TMPC_ERR_NULL_ARG;
  if (!ws || ws_bytes < gated_bwd_ws(rows, f, sizeof(T)) || !aligned(ws, 16)) return TMPC_ERR_WORKSPACE;
  T* dg = static_cast<T*>(ws);
  T* du = dg + rows * f;
  gated_dact_kernel<T><<<8 * sm_count(), 256, 0, st>>>(gate, up, dh, dg, du, rows * f, act);
  if (dx)
    gemm_kernel<T><<<dim3((unsigned)((rows + 63) / 64), (d + 63) / 64), 256, 0, st>>>(dg, wg, du, wu, f, 1, 1, d, dx,
                                                                                   rows, d, f);
  if (dwg) {
    const dim3 grid((f + 63) / 64, (d + 63) / 64);
    gemm_kernel<T><<<grid, 256, 0, st>>>(dg, x, nullptr, nullptr, 1, f, 1, d, dwg, f, d, rows);
    gemm_kernel<T><<<grid, 256, 0, st>>>(du, x, nullptr, nullptr, 1, f, 1, d, dwu, f, d, rows);
  }
  return (int)cudaPeekAtLastError();
}

}  // namespace seq
}  // namespace tmpc

extern "C" {

#define TMPC_GATED_ENTRY(SUF, T)                                                                                     \
  int32_t tmpc_gated_linear_##SUF(int64_t rows, int32_t d, int32_t f, const void* x, const void* w_gate,             \
                                  const void* w_up, int32_t act, void* h, void* gate, void* up, void* workspace,     \
                                  size_t workspace_bytes, tmpc_stream_t stream) {                                    \
    (void)workspace;                                                                                                 \
    (void)workspace_bytes;                                                                                           \
    return tmpc::seq::gated_fwd<T>(rows, d, f, (const T*)x, (const T*)w_gate, (const T*)w_up, act, (T*)h, (T*)gate,  \
                                   (T*)up, (cudaStream_t)stream);                                                    \
  }                                                                                                                  \
  int32_t tmpc_gated_linear_backward_##SUF(int64_t rows, int32_t d, int32_t f, const void* x, const void* w_gate,    \
                                           const void* w_up, int32_t act, const void* gate, const void* up,          \
                                           const void* dh, void* dx, void* dw_gate, void* dw_up, void* workspace,    \
                                           size_t workspace_bytes, tmpc_stream_t stream) {                           \
    return tmpc::seq::gated_bwd<T>(rows, d, f, (const T*)x, (const T*)w_gate, (const T*)w_up, act, (const T*)gate,   \
                                   (const T*)up, (const T*)dh, (T*)dx, (T*)dw_gate, (T*)dw_up, workspace,            \
                                   workspace_bytes, (cudaStream_t)stream);                                           \
  }
TMPC_GATED_ENTRY(f32, float)
TMPC_GATED_ENTRY(bf16, __nv_bfloat16)

size_t tmpc_gated_linear_workspace_bytes(int64_t rows, int32_t d, int32_t f, int32_t elem_size) {
  (void)rows, (void)d, (void)f, (void)elem_size;
  return 0;
}
size_t tmpc_gated_linear_backward_workspace_bytes(int64_t rows, int32_t d, int32_t f, int32_t elem_size) {
  (void)d;
  return tmpc::seq::gated_bwd_ws(rows, f, elem_size);
}

}  // extern "C"
