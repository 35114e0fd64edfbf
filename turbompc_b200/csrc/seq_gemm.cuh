// Matrix products of the gated linear layer on the tensor cores (tcgen05):
// one persistent kernel, out = sum over terms of A_term B_term with an epilogue
// chosen at compile time.
//
// Operands are bfloat16 arrays [component][outer][inner] read by TMA in 128-byte
// swizzled boxes.  bfloat16 tensors have one component.  A float tensor is held
// as three, x = c0 + c1 + c2 exactly (8 mantissa bits each, by truncation), and
// a float product is the sum of the six component products above 2^-24:
// (0,0) (0,1) (1,0) (1,1) (0,2) (2,0); the accumulator is float in both cases.
//
// A block computes 128 x NT tiles: warp 0 feeds a ring of stages by TMA, warp 1
// issues the products (M 128, N NT, K 16 each) into one of two TMEM
// accumulators, warps 4 .. 11 take a finished accumulator through the epilogue
// while the next one is computed.  Every wait is bounded: a wait that runs out
// sets the block's abort flag, the copies and products in flight are drained
// (bounded again), TMEM is freed, and the outputs not computed are stored as NaN.
#pragma once

#include <cuda.h>

#include "seq_common.cuh"
#include "tma.cuh"

namespace tmpc {
namespace seq {
namespace gemm {

constexpr int BM = 128, BK = 64;
constexpr int kThreads = 384;
constexpr int kEpiWarps = 8;
constexpr int kSmemTotal = 227 * 1024;

enum Mode {
  kAct = 0,   // out = act(A Bg^T) * (A Bu^T); the tile's columns are NT/2 of each
  kDact = 1,  // from the same products and dh: dg | du
  kDx = 2,    // out = A (Bg ; Bu), A = dg | du
  kDw = 3     // partial of A^T B, A = dg | du
};

struct Maps {
  CUtensorMap a, b0, b1;
};

struct Params {
  int64_t M;        // output rows: tokens (kAct, kDact, kDx) or columns of dg | du (kDw)
  int N;            // output columns (kAct, kDact: f)
  int fp;           // columns of dg (and du) in dg | du, a multiple of 64
  int kblocks;      // 64-wide blocks of the reduction axis
  int nterms;       // 1 (bfloat16) or 6 (float)
  int splits;       // kDw: parts of the reduction axis
  int mtiles, ntiles;
  int64_t tiles;
  int act;
  int vec;          // bytes per store of out (and load of dh): 16, 4 or 2
  void* out;        // kAct, kDx: T [M][N]; kDw: float [splits][M][N]
  bf16* dgu;        // kDact: [components][M][2 fp]
  const void* dh;   // kDact: T [M][N]
  uint32_t polls;
};

// act(g) and act'(g).  FAST: the hardware exponential and reciprocal, whose
// errors of a few 2^-22 vanish in bfloat16 results.
template <bool FAST>
__device__ __forceinline__ void activation(int act, float g, float& a, float& da) {
  if (act == TMPC_ACT_SILU) {
    const float e = FAST ? __expf(-g) : expf(-g);  // inf for g < -88: s = 0
    const float s = FAST ? __fdividef(1.f, 1.f + fminf(e, 1e30f)) : 1.f / (1.f + e);
    a = g * s;
    da = s * (1.f + g * (1.f - s));
  } else {
    const float c = 0.5f * erfcf(-0.70710678118654752f * g);
    a = g * c;
    da = c + g * 0.39894228040143268f * (FAST ? __expf(-0.5f * g * g) : expf(-0.5f * g * g));
  }
}

// Component pairs of a float product, largest first.
__device__ __forceinline__ int term_a(int t) { return t == 2 ? 1 : t == 3 ? 1 : t == 5 ? 2 : 0; }
__device__ __forceinline__ int term_b(int t) { return t == 1 ? 1 : t == 3 ? 1 : t == 4 ? 2 : 0; }

__device__ __forceinline__ void split3(float x, bf16 (&c)[3]) {
  // Truncation to the top 16 bits is exact to subtract and cannot overflow; a
  // non-finite value keeps its first component alone.
  const uint32_t top = 0xffff0000u;
  const uint32_t u0 = __float_as_uint(x) & top;
  const bool fin = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
  const float r1 = fin ? x - __uint_as_float(u0) : 0.f;
  const uint32_t u1 = __float_as_uint(r1) & top;
  const float r2 = r1 - __uint_as_float(u1);
  // a NaN whose payload lies in the low bits must not become an infinity
  c[0] = __ushort_as_bfloat16((unsigned short)((x != x ? 0x7fc00000u : u0) >> 16));
  c[1] = __ushort_as_bfloat16((unsigned short)(u1 >> 16));
  c[2] = __ushort_as_bfloat16((unsigned short)(__float_as_uint(r2) >> 16));
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Shared-memory descriptor, 128-byte swizzle.  K-major: rows of 128 bytes (64 K
// elements), groups of 8 rows 1024 bytes apart.  MN-major: each 64-wide box of
// the M / N axis holds one 128-byte row per K; boxes lie 64 rows (8192 bytes)
// apart, groups of 8 K rows 1024 bytes.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, bool mn_major) {
  const uint64_t lbo = mn_major ? 8192 >> 4 : 1, sbo = 1024 >> 4;
  return (uint64_t)((addr & 0x3ffff) >> 4) | lbo << 16 | sbo << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}

__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}

// 16 consecutive accumulator columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Bounded wait that also leaves when another role has given up.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t polls, volatile int* abort_flag) {
  for (uint32_t left = polls; left > 0;) {
    const uint32_t n = left < 4096 ? left : 4096;
    if (mbar_wait_bounded(bar, parity, n)) return true;
    left -= n;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}

// A warp's 32 x CW chunk between its staging rows (one per lane) and global
// memory, coalesced along the rows.
template <typename E, int CW>
struct Chunk {
  static constexpr int kPitch = CW * (int)sizeof(E) + 16;  // 16-byte accesses of 8 rows fall into different banks
  static __device__ __forceinline__ void put(char* stg, int lane, const E (&v)[CW]) {
    constexpr int PER = 16 / sizeof(E);
#pragma unroll
    for (int i = 0; i < CW / PER; ++i) {
      Pack<E, PER> p;
#pragma unroll
      for (int e = 0; e < PER; ++e) p.v[e] = v[i * PER + e];
      *reinterpret_cast<Pack<E, PER>*>(stg + lane * kPitch + i * 16) = p;
    }
  }
  static __device__ __forceinline__ void get(const char* stg, int lane, E (&v)[CW]) {
    constexpr int PER = 16 / sizeof(E);
#pragma unroll
    for (int i = 0; i < CW / PER; ++i) {
      const Pack<E, PER> p = *reinterpret_cast<const Pack<E, PER>*>(stg + lane * kPitch + i * 16);
#pragma unroll
      for (int e = 0; e < PER; ++e) v[i * PER + e] = p.v[e];
    }
  }
  template <typename U, bool STORE>
  static __device__ __forceinline__ void move(char* stg, int lane, E* g, int64_t pitch, int rows, int cols) {
    constexpr int PER = sizeof(U) / sizeof(E), UPR = CW / PER;  // units per row
    static_assert(UPR <= 32 && 32 % UPR == 0, "");
    const int u = lane % UPR;
#pragma unroll 8
    for (int r = lane / UPR; r < 32; r += 32 / UPR) {
      if (r < rows && u * PER < cols) {
        U* gp = reinterpret_cast<U*>(g + r * pitch + u * PER);
        U* sp = reinterpret_cast<U*>(stg + r * kPitch + u * sizeof(U));
        if (STORE) *gp = *sp;
        else *sp = *gp;
      }
    }
  }
  template <bool STORE>
  static __device__ __forceinline__ void move(char* stg, int lane, E* g, int64_t pitch, int rows, int cols, int vec) {
    __syncwarp();
    if (vec == 16) {
      move<uint4, STORE>(stg, lane, g, pitch, rows, cols);
    } else if constexpr (sizeof(E) == 4) {
      move<uint32_t, STORE>(stg, lane, g, pitch, rows, cols);
    } else {
      if (vec == 4) move<uint32_t, STORE>(stg, lane, g, pitch, rows, cols);
      else move<uint16_t, STORE>(stg, lane, g, pitch, rows, cols);
    }
    __syncwarp();
  }
  // E values, one row per lane, to g[row][col].
  static __device__ __forceinline__ void store(char* stg, int lane, const E (&v)[CW], E* g, int64_t pitch, int rows,
                                               int cols, int vec) {
    put(stg, lane, v);
    move<true>(stg, lane, g, pitch, rows, cols, vec);
  }
  static __device__ __forceinline__ void load(char* stg, int lane, E (&v)[CW], const E* g, int64_t pitch, int rows,
                                              int cols, int vec) {
    move<false>(stg, lane, const_cast<E*>(g), pitch, rows, cols, vec);
    get(stg, lane, v);
    __syncwarp();
  }
};

template <int NT>
constexpr int stages() {
  constexpr int per = (BM + NT) * BK * 2;
  constexpr int n = (kSmemTotal - 1024 - 1024 - kEpiWarps * 32 * 80) / per;
  return n > 8 ? 8 : n;
}

struct Barriers {
  uint64_t full[8], empty[8], acc_full[2], acc_empty[2], done;
  uint32_t tmem;
  int abort_flag;
};

template <typename T, int MODE, int NT>
__global__ void __launch_bounds__(kThreads, 1) kernel(const __grid_constant__ Maps maps, const Params p) {
  constexpr int ST = stages<NT>();
  constexpr int kA = BM * BK * 2, kB = NT * BK * 2;
  constexpr bool kAmn = MODE == kDw, kBmn = MODE == kDx || MODE == kDw;
  constexpr bool kDual = MODE == kAct || MODE == kDact;
  constexpr uint32_t kIdesc = 1u << 4 | 1u << 7 | 1u << 10 | (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) |
                              (uint32_t)(NT / 8) << 17 | (uint32_t)(BM / 16) << 24;
  extern __shared__ char raw[];
  char* smem = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  char* sA = smem;
  char* sB = smem + ST * kA;
  char* stage_mem = sB + ST * kB;
  Barriers& bar = *reinterpret_cast<Barriers*>(stage_mem + kEpiWarps * 32 * 80);
  volatile int* abort_flag = &bar.abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&bar.acc_full[i], 1), mbar_init(&bar.acc_empty[i], kEpiWarps);
    mbar_init(&bar.done, 1);
    bar.abort_flag = 0;
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bar.tmem)),
                 "n"(2 * NT)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = bar.tmem;

  auto tile_of = [&](int64_t t, int64_t& m0, int& n0, int& kb0, int& kb1, int& split) {
    split = 0;
    if (MODE == kDw) {  // tiles of one split share their rows of x and dg | du in L2
      const int64_t per = (int64_t)p.mtiles * p.ntiles;
      split = (int)(t / per);
      t %= per;
    }
    m0 = t / p.ntiles * BM;
    n0 = (int)(t % p.ntiles) * (kDual ? NT / 2 : NT);
    kb0 = (int)((int64_t)p.kblocks * split / p.splits);
    kb1 = (int)((int64_t)p.kblocks * (split + 1) / p.splits);
  };

  if (warp == 0 && lane == 0) {  // TMA
    int64_t m0;
    int n0, kb0, kb1, split;
    uint32_t n = 0;  // stages issued
    bool ok = true;
    for (int64_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
      tile_of(t, m0, n0, kb0, kb1, split);
      for (int term = 0; ok && term < p.nterms; ++term) {
        const int ca = term_a(term), cb = term_b(term);
        for (int kb = kb0; kb < kb1; ++kb, ++n) {
          const int s = n % ST;
          if (n >= ST && !(ok = wait(&bar.empty[s], (n / ST - 1) & 1, p.polls, abort_flag))) break;
          uint64_t* full = &bar.full[s];
          mbar_expect_tx(full, kA + kB);
          char *a = sA + s * kA, *b = sB + s * kB;
          if (kAmn) {
            tma_load_3d(a, &maps.a, (int)m0, kb * BK, ca, full);
            tma_load_3d(a + 8192, &maps.a, (int)m0 + 64, kb * BK, ca, full);
          } else {
            tma_load_3d(a, &maps.a, kb * BK, (int)m0, ca, full);
          }
          if (kDual) {
            tma_load_3d(b, &maps.b0, kb * BK, n0, cb, full);
            tma_load_3d(b + kB / 2, &maps.b1, kb * BK, n0, cb, full);
          } else {
            const bool up = MODE == kDx && kb >= p.fp / BK;
            const int k = (up ? kb - p.fp / BK : kb) * BK;
            for (int j = 0; j < NT / 64; ++j)
              tma_load_3d(b + j * 8192, up ? &maps.b1 : &maps.b0, n0 + j * 64, k, cb, full);
          }
        }
      }
    }
    // Nothing may land after the block has left: the last copies of every stage.
    for (uint32_t i = n > ST ? n - ST : 0; i < n; ++i)
      mbar_wait_bounded(&bar.full[i % ST], (i / ST) & 1, kTransferDrainPolls);
  } else if (warp == 1 && lane == 0) {  // products
    int64_t m0;
    int n0, kb0, kb1, split;
    uint32_t n = 0, done_tiles = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x, ++done_tiles) {
      tile_of(t, m0, n0, kb0, kb1, split);
      const uint32_t buf = done_tiles & 1, d = tmem + buf * NT;
      if (done_tiles >= 2 && !(ok = wait(&bar.acc_empty[buf], (done_tiles / 2 - 1) & 1, p.polls, abort_flag))) break;
      fence_after();
      const int iters = (kb1 - kb0) * p.nterms;
      for (int it = 0; it < iters; ++it, ++n) {
        const int s = n % ST;
        if (!(ok = wait(&bar.full[s], (n / ST) & 1, p.polls, abort_flag))) break;
        fence_after();
        const uint64_t da = smem_desc(smem_u32(sA + s * kA), kAmn), db = smem_desc(smem_u32(sB + s * kB), kBmn);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)  // 16 K elements: 32 bytes of a K-major row, 16 rows of an MN-major box
          mma_f16(d, da + k * ((kAmn ? 2048 : 32) >> 4), db + k * ((kBmn ? 2048 : 32) >> 4), kIdesc, it > 0 || k > 0);
        mma_commit(&bar.empty[s]);
      }
      if (ok) mma_commit(&bar.acc_full[buf]);
    }
    if (!ok) {  // TMEM may be freed only after the products in flight
      mma_commit(&bar.done);
      mbar_wait_bounded(&bar.done, 0, kTransferDrainPolls);
    }
  } else if (warp >= 4) {  // epilogue: lanes 32 (warp % 4) .. + 31, half of the columns each
    constexpr int kCols = (kDual ? NT / 2 : NT) / 2;
    constexpr int CW = kCols < 32 || sizeof(T) == 4 || MODE == kDw ? 16 : 32;
    const int quad = warp & 3, half = (warp - 4) >> 2;
    char* stg = stage_mem + (warp - 4) * 32 * 80;
    int64_t m0;
    int n0, kb0, kb1, split;
    uint32_t done_tiles = 0;
    bool ok = true;
    const float nan = __int_as_float(0x7fffffff);
    for (int64_t t = blockIdx.x; t < p.tiles; t += gridDim.x, ++done_tiles) {
      tile_of(t, m0, n0, kb0, kb1, split);
      const uint32_t buf = done_tiles & 1;
      if (ok) ok = wait(&bar.acc_full[buf], (done_tiles / 2) & 1, p.polls, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16) + buf * NT + half * kCols;
      const int64_t row0 = m0 + quad * 32;
      const int rows = (int)(p.M - row0 < 32 ? p.M - row0 : 32);
#pragma unroll 1
      for (int c = 0; c < kCols; c += CW) {
        const int col0 = n0 + half * kCols + c, cols = p.N - col0;
        float v[CW], w[kDual ? CW : 1];
        if (ok) {
#pragma unroll
          for (int i = 0; i < CW; i += 16) {
            tmem_ld16(acc + c + i, *reinterpret_cast<float(*)[16]>(&v[i]));
            if constexpr (kDual) tmem_ld16(acc + NT / 2 + c + i, *reinterpret_cast<float(*)[16]>(&w[i]));
          }
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < CW; ++i) {
            v[i] = nan;
            if constexpr (kDual) w[i] = nan;
          }
        }
        constexpr bool kFast = sizeof(T) == 2;
        if constexpr (MODE == kAct) {
          T h[CW];
#pragma unroll
          for (int i = 0; i < CW; ++i) {
            float a, da;
            activation<kFast>(p.act, v[i], a, da);
            h[i] = from_f<T>(a * w[i]);
          }
          Chunk<T, CW>::store(stg, lane, h, static_cast<T*>(p.out) + row0 * p.N + col0, p.N, rows, cols, p.vec);
        } else if constexpr (MODE == kDact) {
          T y[CW];
          Chunk<T, CW>::load(stg, lane, y, static_cast<const T*>(p.dh) + row0 * p.N + col0, p.N, rows, cols, p.vec);
          constexpr int NC = sizeof(T) == 4 ? 3 : 1;
          bf16 g[NC][CW], u[NC][CW];
#pragma unroll
          for (int i = 0; i < CW; ++i) {
            float a, da;
            activation<kFast>(p.act, v[i], a, da);
            const float dy = to_f(y[i]);
            // columns f .. fp - 1 meet rows of zeros in the next products: they must not be NaN
            const float dg = i < cols ? dy * w[i] * da : 0.f, du = i < cols ? dy * a : 0.f;
            if constexpr (NC == 1) {
              g[0][i] = from_f<bf16>(dg);
              u[0][i] = from_f<bf16>(du);
            } else {
              bf16 s[3];
              split3(dg, s);
              g[0][i] = s[0], g[1][i] = s[1], g[2][i] = s[2];
              split3(du, s);
              u[0][i] = s[0], u[1][i] = s[1], u[2][i] = s[2];
            }
          }
          const int64_t pitch = 2 * (int64_t)p.fp;
          bf16* o = p.dgu + row0 * pitch + col0;
#pragma unroll
          for (int k = 0; k < NC; ++k) {
            Chunk<bf16, CW>::store(stg, lane, g[k], o + k * p.M * pitch, pitch, rows, p.fp - col0, 16);
            Chunk<bf16, CW>::store(stg, lane, u[k], o + k * p.M * pitch + p.fp, pitch, rows, p.fp - col0, 16);
          }
        } else if constexpr (MODE == kDx) {
          T o[CW];
#pragma unroll
          for (int i = 0; i < CW; ++i) o[i] = from_f<T>(v[i]);
          Chunk<T, CW>::store(stg, lane, o, static_cast<T*>(p.out) + row0 * p.N + col0, p.N, rows, cols, p.vec);
        } else {
          Chunk<float, CW>::store(stg, lane, v, static_cast<float*>(p.out) + (split * p.M + row0) * p.N + col0, p.N,
                                  rows, cols, p.vec);
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.acc_empty[buf]);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 2) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(2 * NT) : "memory");
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// A bfloat16 array [components][outer][inner], rows of `pitch` elements (a
// multiple of 8, 16-byte aligned base), read in boxes of 64 x box_outer.
inline int make_map(CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int comps, int64_t pitch,
                    int box_outer) {
  const EncodeFn fn = encode_fn();
  if (!fn) return (int)cudaErrorNotSupported;
  const cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)outer, (cuuint64_t)comps};
  const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)pitch * 2 * (cuuint64_t)outer};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_outer, 1}, es[3] = {1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

template <typename T, int MODE, int NT>
int launch(const Maps& maps, Params p, cudaStream_t st) {
  p.tiles = (int64_t)p.mtiles * p.ntiles * p.splits;
  p.polls = transfer_poll_limit().load();
  const cudaError_t e =
      cudaFuncSetAttribute(kernel<T, MODE, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemTotal);
  if (e != cudaSuccess) return (int)e;
  const int64_t sms = sm_count();
  kernel<T, MODE, NT><<<(unsigned)(p.tiles < sms ? p.tiles : sms), kThreads, kSmemTotal, st>>>(maps, p);
  return (int)cudaPeekAtLastError();
}

}  // namespace gemm
}  // namespace seq
}  // namespace tmpc
