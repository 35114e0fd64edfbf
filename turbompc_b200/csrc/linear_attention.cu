// Linear attention with a decay per head, token by token: forward, backward.
//
//   S_t = d S_{t-1} + k_t v_t^T,   o_t = s S_t^T q_t
//   dS_t = d dS_{t+1} + s q_t do_t^T,   dq_t = s S_t do_t,
//   dk_t = dS_t v_t,   dv_t = dS_t^T k_t
//   dlog d = sum_t <dS_t, d S_{t-1}>
//
// The state lives in registers: a thread owns a column of S (forward, dv) or
// a row (dq, dk).  dlog d needs no product of S and dS inside the sequence:
// with q' = d^(t+1) q and k' = d^-(t+1) k the decay leaves every o_t, and
//   dlog d = sum_t (t+1) (q_t . dq_t - k_t . dk_t) + L <S_L, dS_L>.
#include "seq_attention.cuh"

namespace tmpc {
namespace seq {
namespace rec {

constexpr int kTile = 16;  // tokens staged in shared memory at a time
constexpr int kCols = 128;

// Tokens t0 .. t0 + n - 1 of one head into a [kTile][LD] tile, zero-padded.
template <typename T, int LD>
__device__ __forceinline__ void stage(float (*s)[LD], const TmpcSeqView& w, int b, int t0, int n, int h, int d) {
  for (int e = threadIdx.x; e < kTile * LD; e += blockDim.x) {
    const int t = e / LD, i = e % LD;
    s[t][i] = (t < n && i < d) ? to_f(row_ptr<T>(w, b, t0 + t, h)[i]) : 0.f;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kCols) fwd_kernel(const LinAttnArgs a) {
  __shared__ __align__(16) float sq[kTile][D], sk[kTile][D];
  const int h = blockIdx.y, b = blockIdx.x, g = h / (a.H / a.G), j = threadIdx.x;
  const float dec = exp2f(log2_decay(a.log_decay, h));
  const int len = seq_len(a, b);
  const size_t so = ((size_t)b * a.H + h) * a.dk * a.dv;
  float S[D];
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = (a.state_in && i < a.dk && j < a.dv) ? a.state_in[so + (size_t)i * a.dv + j] : 0.f;
  for (int t0 = 0; t0 < len; t0 += kTile) {
    const int n = min(kTile, len - t0);
    __syncthreads();
    stage<T, D>(sq, a.q, b, t0, n, h, a.dk);
    stage<T, D>(sk, a.k, b, t0, n, g, a.dk);
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      const float v = j < a.dv ? to_f(row_ptr<T>(a.v, b, t0 + t, g)[j]) : 0.f;
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < D; ++i) {
        S[i] = fmaf(dec, S[i], sk[t][i] * v);
        o = fmaf(sq[t][i], S[i], o);
      }
      if (j < a.dv) (row_ptr<T>(a.o, b, t0 + t, h))[j] = from_f<T>(o * a.scale);
    }
  }
  if (j < a.dv)
    for (int t = len; t < a.T; ++t) (row_ptr<T>(a.o, b, t, h))[j] = from_f<T>(0.f);
  if (a.state_out && j < a.dv) {
#pragma unroll
    for (int i = 0; i < D; ++i)
      if (i < a.dk) a.state_out[so + (size_t)i * a.dv + j] = S[i];
  }
}

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) v += red[i];
  return v;
}

// dq: thread i owns row i of S.
template <typename T, int D>
__global__ void __launch_bounds__(kCols) dq_kernel(const LinAttnArgs a) {
  __shared__ __align__(16) float sv[kTile][D], sdo[kTile][D];
  __shared__ double red[4];
  const int h = blockIdx.y, b = blockIdx.x, g = h / (a.H / a.G), i = threadIdx.x;
  const float dec = exp2f(log2_decay(a.log_decay, h));
  const int len = seq_len(a, b);
  const size_t so = ((size_t)b * a.H + h) * a.dk * a.dv;
  float S[D];
#pragma unroll
  for (int j = 0; j < D; ++j) S[j] = (a.state_in && i < a.dk && j < a.dv) ? a.state_in[so + (size_t)i * a.dv + j] : 0.f;
  double dl = 0;
  for (int t0 = 0; t0 < len; t0 += kTile) {
    const int n = min(kTile, len - t0);
    __syncthreads();
    stage<T, D>(sv, a.v, b, t0, n, g, a.dv);
    stage<T, D>(sdo, a.o, b, t0, n, h, a.dv);
    __syncthreads();
    for (int t = 0; t < n; ++t) {
      const float k = i < a.dk ? to_f(row_ptr<T>(a.k, b, t0 + t, g)[i]) : 0.f;
      const float q = i < a.dk ? to_f(row_ptr<T>(a.q, b, t0 + t, h)[i]) : 0.f;
      float dq = 0.f;
#pragma unroll
      for (int j = 0; j < D; ++j) {
        S[j] = fmaf(dec, S[j], sv[t][j] * k);
        dq = fmaf(sdo[t][j], S[j], dq);
      }
      dq *= a.scale;
      dl += (double)(t0 + t + 1) * (double)(q * dq);
      if (i < a.dk) (row_ptr<T>(a.gq, b, t0 + t, h))[i] = from_f<T>(dq);
    }
  }
  if (i < a.dk)
    for (int t = len; t < a.T; ++t) (row_ptr<T>(a.gq, b, t, h))[i] = from_f<T>(0.f);
  if (a.dstate_out && i < a.dk) {
    float e = 0.f;
#pragma unroll
    for (int j = 0; j < D; ++j)
      if (j < a.dv) e = fmaf(S[j], a.dstate_out[so + (size_t)i * a.dv + j], e);
    dl += (double)len * (double)e;
  }
  dl = block_sum(dl, red);
  if (a.dlog && i == 0) reinterpret_cast<double*>(a.dlog)[(size_t)b * a.H + h] = dl;
}

// dk, dv: threads 0 .. 127 own a row of dS, threads 128 .. 255 a column.
template <typename T, int D>
__global__ void __launch_bounds__(2 * kCols) dkv_kernel(const LinAttnArgs a) {
  __shared__ __align__(16) float sq[kTile][D], sk[kTile][D], sv[kTile][D], sdo[kTile][D];
  __shared__ double red[8];
  const int g = blockIdx.y, b = blockIdx.x, rep = a.H / a.G;
  const bool is_row = threadIdx.x < kCols;
  const int i = threadIdx.x % kCols;
  const int mine = is_row ? a.dk : a.dv, other = is_row ? a.dv : a.dk;
  const int len = seq_len(a, b);
  for (int r = 0; r < rep; ++r) {
    const int h = g * rep + r;
    const float dec = exp2f(log2_decay(a.log_decay, h));
    const size_t so = ((size_t)b * a.H + h) * a.dk * a.dv;
    const size_t s_own = is_row ? (size_t)i * a.dv : i, s_step = is_row ? 1 : a.dv;
    float dS[D];
#pragma unroll
    for (int j = 0; j < D; ++j)
      dS[j] = (a.dstate_out && i < mine && j < other) ? a.dstate_out[so + s_own + j * s_step] : 0.f;
    double dl = 0;
    for (int t0 = (len - 1) / kTile * kTile; len > 0 && t0 >= 0; t0 -= kTile) {
      const int n = min(kTile, len - t0);
      __syncthreads();
      stage<T, D>(sq, a.q, b, t0, n, h, a.dk);
      stage<T, D>(sk, a.k, b, t0, n, g, a.dk);
      stage<T, D>(sv, a.v, b, t0, n, g, a.dv);
      stage<T, D>(sdo, a.o, b, t0, n, h, a.dv);
      __syncthreads();
      for (int t = n - 1; t >= 0; --t) {
        const float* outer = is_row ? sdo[t] : sq[t];
        const float* inner = is_row ? sv[t] : sk[t];
        const float x = (i < mine ? (is_row ? sq[t][i] : sdo[t][i]) : 0.f) * a.scale;
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < D; ++j) {
          dS[j] = fmaf(outer[j], x, dS[j]);
          y = fmaf(dS[j], inner[j], y);
          dS[j] *= dec;
        }
        if (is_row && i < mine) dl -= (double)(t0 + t + 1) * (double)(sk[t][i] * y);
        if (i < mine) {
          float* acc = a.acc + (((size_t)b * a.T + t0 + t) * a.G + g) * (a.dk + a.dv) + (is_row ? 0 : a.dk) + i;
          if (r > 0) y += *acc;
          if (r + 1 < rep) *acc = y;
          else (row_ptr<T>(is_row ? a.gk : a.gv, b, t0 + t, g))[i] = from_f<T>(y);
        }
      }
    }
    if (a.dstate_in && is_row && i < a.dk) {
#pragma unroll
      for (int j = 0; j < D; ++j)
        if (j < a.dv) a.dstate_in[so + (size_t)i * a.dv + j] = dS[j];
    }
    dl = block_sum(dl, red);
    if (a.dlog && threadIdx.x == 0) reinterpret_cast<double*>(a.dlog)[((size_t)gridDim.x + b) * a.H + h] = dl;
  }
  if (i < mine)
    for (int t = len; t < a.T; ++t)
      (row_ptr<T>(is_row ? a.gk : a.gv, b, t, g))[i] = from_f<T>(0.f);
}

__global__ void dlog_kernel(const double* part, float* out, int n, int H) {
  __shared__ double red[4];
  const int h = blockIdx.x;
  double s = 0;
  for (int b = threadIdx.x; b < n; b += blockDim.x) s += part[(size_t)b * H + h];
  s = block_sum(s, red);
  if (threadIdx.x == 0) out[h] = (float)s;
}

}  // namespace rec

template <>
size_t LinAttn<float>::forward_ws(const TmpcLinAttnDims*) {
  return 0;
}

template <>
int LinAttn<float>::forward(LinAttnArgs a, const TmpcLinAttnDims* d, char*, cudaStream_t st) {
  by_size(d, [&](auto dd) {
    constexpr int D = decltype(dd)::value;
    rec::fwd_kernel<float, D><<<dim3(a.B, a.H), rec::kCols, 0, st>>>(a);
  });
  return (int)cudaPeekAtLastError();
}

template <>
size_t LinAttn<float>::backward_ws(const TmpcLinAttnDims* d) {
  return (size_t)2 * d->B * d->H * sizeof(double) +
         (d->H > d->G ? (size_t)d->B * d->T * d->G * (d->dk + d->dv) * sizeof(float) : 0);
}

template <>
int LinAttn<float>::backward(LinAttnArgs a, const TmpcLinAttnDims* d, float* dlog_decay, char* ws, cudaStream_t st) {
  a.dlog = reinterpret_cast<float*>(ws);
  a.acc = reinterpret_cast<float*>(ws + (size_t)2 * d->B * d->H * sizeof(double));
  by_size(d, [&](auto dd) {
    constexpr int D = decltype(dd)::value;
    rec::dq_kernel<float, D><<<dim3(a.B, a.H), rec::kCols, 0, st>>>(a);
    rec::dkv_kernel<float, D><<<dim3(a.B, a.G), 2 * rec::kCols, 0, st>>>(a);
  });
  if (dlog_decay)
    rec::dlog_kernel<<<a.H, 128, 0, st>>>(reinterpret_cast<double*>(a.dlog), dlog_decay, 2 * a.B, a.H);
  return (int)cudaPeekAtLastError();
}

// ---------------------------------------------------------------------------
// Entry points
// ---------------------------------------------------------------------------
inline bool null_view(const TmpcSeqView* v, const TmpcLinAttnDims* d) { return !v || (d->T > 0 && !v->ptr); }

inline LinAttnArgs make_args(const TmpcLinAttnDims* d, const TmpcSeqView* q, const TmpcSeqView* k, const TmpcSeqView* v,
                             const TmpcSeqView* o, const float* log_decay, const int32_t* lengths,
                             const float* state_in, double scale) {
  LinAttnArgs a{};
  a.q = *q, a.k = *k, a.v = *v, a.o = *o;
  a.log_decay = log_decay, a.lengths = lengths, a.state_in = state_in;
  a.B = d->B, a.T = d->T, a.H = d->H, a.G = d->G, a.dk = d->dk, a.dv = d->dv;
  a.nseg = 1;
  a.scale = (float)scale;
  return a;
}

template <typename T>
int forward(const TmpcLinAttnDims* d, const TmpcSeqView* q, const TmpcSeqView* k, const TmpcSeqView* v,
            const TmpcSeqView* o, const float* log_decay, const int32_t* lengths, const float* state_in,
            float* state_out, double scale, void* ws, size_t ws_bytes, cudaStream_t st) {
  const int rc = check_dims(d);
  if (rc) return rc;
  if (d->B == 0) return TMPC_OK;
  if (null_view(q, d) || null_view(k, d) || null_view(v, d) || null_view(o, d) || !log_decay) return TMPC_ERR_NULL_ARG;
  const size_t need = LinAttn<T>::forward_ws(d);
  if (need > 0 && (!ws || ws_bytes < need || !aligned(ws, 16))) return TMPC_ERR_WORKSPACE;
  LinAttnArgs a = make_args(d, q, k, v, o, log_decay, lengths, state_in, scale);
  a.state_out = state_out;
  return LinAttn<T>::forward(a, d, static_cast<char*>(ws), st);
}

template <typename T>
int backward(const TmpcLinAttnDims* d, const TmpcSeqView* q, const TmpcSeqView* k, const TmpcSeqView* v,
             const TmpcSeqView* dout, const TmpcSeqView* dq, const TmpcSeqView* dk, const TmpcSeqView* dv,
             const float* log_decay, const int32_t* lengths, const float* state_in, const float* dstate_out,
             float* dlog_decay, float* dstate_in, double scale, void* ws, size_t ws_bytes, cudaStream_t st) {
  const int rc = check_dims(d);
  if (rc) return rc;
  if (d->B == 0) return dlog_decay ? (int)cudaMemsetAsync(dlog_decay, 0, d->H * sizeof(float), st) : TMPC_OK;
  if (null_view(q, d) || null_view(k, d) || null_view(v, d) || null_view(dout, d) || null_view(dq, d) ||
      null_view(dk, d) || null_view(dv, d) || !log_decay)
    return TMPC_ERR_NULL_ARG;
  const size_t need = LinAttn<T>::backward_ws(d);
  if (need > 0 && (!ws || ws_bytes < need || !aligned(ws, 16))) return TMPC_ERR_WORKSPACE;
  LinAttnArgs a = make_args(d, q, k, v, dout, log_decay, lengths, state_in, scale);
  a.gq = *dq, a.gk = *dk, a.gv = *dv;
  a.dstate_out = dstate_out, a.dstate_in = dstate_in;
  return LinAttn<T>::backward(a, d, dlog_decay, static_cast<char*>(ws), st);
}

}  // namespace seq
}  // namespace tmpc

extern "C" {

#define TMPC_LINATTN_ENTRY(SUF, T)                                                                                   \
  int32_t tmpc_linear_attention_##SUF(const TmpcLinAttnDims* dims, const TmpcSeqView* q, const TmpcSeqView* k,       \
                                      const TmpcSeqView* v, const TmpcSeqView* o, const float* log_decay,            \
                                      const int32_t* lengths, const float* state_in, float* state_out, double scale, \
                                      void* workspace, size_t workspace_bytes, tmpc_stream_t stream) {               \
    return tmpc::seq::forward<T>(dims, q, k, v, o, log_decay, lengths, state_in, state_out, scale, workspace,        \
                                 workspace_bytes, (cudaStream_t)stream);                                             \
  }                                                                                                                  \
  int32_t tmpc_linear_attention_backward_##SUF(                                                                      \
      const TmpcLinAttnDims* dims, const TmpcSeqView* q, const TmpcSeqView* k, const TmpcSeqView* v,                 \
      const TmpcSeqView* dout, const TmpcSeqView* dq, const TmpcSeqView* dk, const TmpcSeqView* dv,                  \
      const float* log_decay, const int32_t* lengths, const float* state_in, const float* dstate_out,                \
      float* dlog_decay, float* dstate_in, double scale, void* workspace, size_t workspace_bytes,                    \
      tmpc_stream_t stream) {                                                                                        \
    return tmpc::seq::backward<T>(dims, q, k, v, dout, dq, dk, dv, log_decay, lengths, state_in, dstate_out,         \
                                  dlog_decay, dstate_in, scale, workspace, workspace_bytes, (cudaStream_t)stream);   \
  }
TMPC_LINATTN_ENTRY(f32, float)
TMPC_LINATTN_ENTRY(bf16, __nv_bfloat16)

// The larger of the two types' needs.
size_t tmpc_linear_attention_workspace_bytes(const TmpcLinAttnDims* dims) {
  using namespace tmpc::seq;
  if (check_dims(dims)) return 0;
  return std::max(LinAttn<float>::forward_ws(dims), LinAttn<bf16>::forward_ws(dims));
}
size_t tmpc_linear_attention_backward_workspace_bytes(const TmpcLinAttnDims* dims) {
  using namespace tmpc::seq;
  if (check_dims(dims)) return 0;
  return std::max(LinAttn<float>::backward_ws(dims), LinAttn<bf16>::backward_ws(dims));
}

}  // extern "C"
