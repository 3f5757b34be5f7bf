// Gated causal scan on CUDA cores: fp32 tensors, and the 16-bit head dims that have no tensor-core kernel.
//
// Math, per (batch, head), with a log decay g_t <= 0 per position:
//     S_t = e^(g_t) S_(t-1) + k_t v_t^T          out_t = S_t^T q_t
// In chunks of 64 positions, G_t = sum of g over the chunk up to and including t, D_ts = e^(G_t - G_s) for s <= t, S the state before
// the chunk, R the gradient of the state after it, A = e^(G_last):
//     out_t = e^(G_t) q_t S            + sum_{s<=t} D_ts (q_t.k_s) v_s          S' = A S + sum_s e^(G_last-G_s) k_s v_s^T
//     dq_t  = e^(G_t) S dO_t           + sum_{s<=t} D_ts (dO_t.v_s) k_s         R before = A R + sum_t e^(G_t) q_t dO_t^T
//     dk_s  = e^(G_last-G_s) R v_s     + sum_{t>=s} D_ts (dO_t.v_s) q_t
//     dv_s  = e^(G_last-G_s) R^T k_s   + sum_{t>=s} D_ts (q_t.k_s) dO_t
//     dg_t  = sum_{u>=t in the chunk} (q_u.dq_u - k_u.dk_u) + <S', R>
// The last line: a pair (t, s) enters dL/dG with + at t and with - at s, and <S', R> is the derivative to a common factor of all
// that crosses the chunk's end.  (One running sum over the whole sequence is the same in exact arithmetic, but it carries the
// roundings of every later position to every earlier one.)  Exponents are differences of sums: G is held in fp64, so that neither
// a state that is dropped (g = -inf, taken as -10000) nor strong decays cost the others digits.  No exponent is taken of a
// difference that causality excludes.
//
// Four kinds of kernel: the chunks' own states, their decayed prefix (suffix), the rows of the chunks (out, or dq, dk and dv as
// three CTAs per chunk), and dg.  A masked position (keep == 0) contributes nothing, lets the state pass unchanged and has zero
// rows; its tensors are not read into any product.  Bound by the fp32 FMA rate and the staging before it.
#pragma once

#include "common.cuh"

namespace cott {

constexpr int kGsChunk = 64;
constexpr int kGsThreads = 256;
constexpr double kGateFloor = -10000.0;  // e^-10000 = 0, and sums of it stay finite

using GatedStrides = cott_strides;  // element strides of (batch, head, position); the innermost dimension is contiguous
struct GatedArgs {
  const void *q, *k, *v, *dout, *gate;
  const unsigned char* keep;
  const float *initial, *dfinal;      // [B*H][value][key]
  float *final_state, *dinitial;
  void *out, *dq, *dk, *dv, *dgate;
  float *prefix, *suffix;             // [B*H][chunks + 1][key][value], [B*H][chunks][key][value]
  float* total;                       // [B*H][chunks]: G_last
  float *qdot, *kdot;                 // [B*H][chunks][64]: q_t.dq_t, k_s.dk_s
  GatedStrides sq, sk, sv, so, sg, sdq, sdk, sdv, sdg;
  int H, N, nchunks, gate_f32, with_initial;
};
__device__ __forceinline__ long long gated_at(const GatedStrides& s, long b, int h, int n) { return b * s.b + h * s.h + n * s.n; }

// one gate as a sum can take it: -inf (and what is below any use) as kGateFloor, NaN as it is; masked: 0
template <typename T>
__device__ __forceinline__ double gated_gate(const GatedArgs& a, long b, int h, int pos) {
  if (a.keep && !a.keep[b * a.N + pos]) return 0.0;
  const long long o = gated_at(a.sg, b, h, pos);
  const float g = a.gate_f32 ? static_cast<const float*>(a.gate)[o] : static_cast<float>(to_acc(static_cast<const T*>(a.gate)[o]));
  return g < static_cast<float>(kGateFloor) ? kGateFloor : static_cast<double>(g);
}
// G of the chunk, by the first warp (two positions a lane); positions past the end have g = 0
template <typename T>
__device__ __forceinline__ void gated_sums(const GatedArgs& a, double* G, long b, int h, int c0) {
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x, p = c0 + 2 * lane;
    const double g0 = p < a.N ? gated_gate<T>(a, b, h, p) : 0.0, g1 = p + 1 < a.N ? gated_gate<T>(a, b, h, p + 1) : 0.0;
    double run = g0 + g1;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += up;
    }
    G[2 * lane] = run - g1;
    G[2 * lane + 1] = run;
  }
}

template <typename T, int N>
__device__ __forceinline__ void gs_load(float (&x)[N], const T* p) {
  struct alignas(sizeof(T) * N) Vec { T e[N]; };
  const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
  for (int e = 0; e < N; ++e) x[e] = to_acc(v.e[e]);
}
template <int N>
__device__ __forceinline__ void gs_lds(float (&x)[N], const float* p) {
  if constexpr (N == 8) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    struct alignas(4 * N) Vec { float e[N]; };
    const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = v.e[e];
  }
}
template <typename T, int N>
__device__ __forceinline__ void gs_store(T* p, const float (&x)[N]) {
  struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec { T e[N]; } v;
#pragma unroll
  for (int e = 0; e < N; ++e) v.e[e] = from_acc<T>(x[e]);
  *reinterpret_cast<Vec*>(p) = v;
}
__device__ __forceinline__ float gs_row_sum(float x) {  // over the 16 threads of a row
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// one [64 x D] tile -> shared memory in fp32 (row stride D + 4); thread (ty, tx) has columns NB tx .. of rows ty + 16 a.  Rows past
// the end and masked rows are zero.
template <typename T, int D>
__device__ __forceinline__ void gs_stage(float* dst, const void* src, const GatedStrides& st, const GatedArgs& g, long b, int h, int c0, int tx, int ty) {
  constexpr int NB = D / 16, LD = D + 4;
#pragma unroll
  for (int a = 0; a < 4; ++a) {
    const int r = ty + 16 * a, pos = c0 + r;
    float x[NB];
#pragma unroll
    for (int e = 0; e < NB; ++e) x[e] = 0.f;
    if (pos < g.N && (!g.keep || g.keep[b * g.N + pos])) gs_load<T, NB>(x, static_cast<const T*>(src) + gated_at(st, b, h, pos) + NB * tx);
#pragma unroll
    for (int e = 0; e < NB; ++e) dst[r * LD + NB * tx + e] = x[e];
  }
}

// A chunk's own state.  REV: sum_t e^(G_t) q_t dO_t^T, else sum_s e^(G_last-G_s) k_s v_s^T.  grid = B*H * chunks.
template <typename T, int D, bool REV>
__global__ void __launch_bounds__(kGsThreads) gated_state_kernel(const GatedArgs g) {
  constexpr int NB = D / 16, LD = D + 4;
  extern __shared__ __align__(16) unsigned char gs_smem[];
  float* sY = reinterpret_cast<float*>(gs_smem);
  float* sZ = sY + kGsChunk * LD;
  __shared__ double G[kGsChunk];
  __shared__ float w[kGsChunk];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const long bh = blockIdx.x / g.nchunks, b = bh / g.H;
  const int chunk = static_cast<int>(blockIdx.x % g.nchunks), c0 = kGsChunk * chunk, h = static_cast<int>(bh % g.H);
  pdl_allow_next();
  pdl_wait_prior();
  gated_sums<T>(g, G, b, h, c0);
  gs_stage<T, D>(sY, REV ? g.q : g.k, REV ? g.sq : g.sk, g, b, h, c0, tx, ty);
  gs_stage<T, D>(sZ, REV ? g.dout : g.v, REV ? g.so : g.sv, g, b, h, c0, tx, ty);
  __syncthreads();
  if (tid < kGsChunk) w[tid] = expf(static_cast<float>(REV ? G[tid] : G[kGsChunk - 1] - G[tid]));
  if (!REV && tid == 0) g.total[blockIdx.x] = static_cast<float>(G[kGsChunk - 1]);
  __syncthreads();
  float acc[NB][NB] = {};
#pragma unroll 4
  for (int s = 0; s < kGsChunk; ++s) {
    float x[NB], y[NB];
    gs_lds<NB>(x, sY + s * LD + NB * ty);
    gs_lds<NB>(y, sZ + s * LD + NB * tx);
#pragma unroll
    for (int i = 0; i < NB; ++i) x[i] *= w[s];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = fmaf(x[i], y[j], acc[i][j]);
  }
  float* dst = (REV ? g.suffix + (bh * g.nchunks + chunk) * static_cast<long>(D * D) : g.prefix + (bh * (g.nchunks + 1) + chunk) * static_cast<long>(D * D));
#pragma unroll
  for (int i = 0; i < NB; ++i) gs_store<float, NB>(dst + (NB * ty + i) * D + NB * tx, acc[i]);
}

// In place: the chunks' own states -> the state before each chunk (REV: the gradient of the state after it).  A thread owns one
// element; eight chunks are loaded at a time so that the chain is arithmetic, not memory round trips.
// grid = (B*H, D*D / 256).
template <int D, bool REV>
__global__ void __launch_bounds__(kGsThreads) gated_prefix_kernel(const GatedArgs g) {
  const long bh = blockIdx.x;
  const int e = blockIdx.y * kGsThreads + threadIdx.x, i = e / D, j = e % D, n = g.nchunks;
  float* p = (REV ? g.suffix + bh * n * static_cast<long>(D * D) : g.prefix + bh * (n + 1) * static_cast<long>(D * D)) + e;
  const float* total = g.total + bh * n;
  const long edge = bh * static_cast<long>(D * D) + static_cast<long>(j) * D + i;  // [value][key]
  pdl_allow_next();
  pdl_wait_prior();
  const float* from = REV ? g.dfinal : g.initial;
  float run = from ? from[edge] : 0.f;
  for (int c = 0; c < n; c += 8) {
    float x[8], a[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int at = REV ? n - 1 - c - u : c + u;
      x[u] = c + u < n ? p[static_cast<long>(at) * (D * D)] : 0.f;
      a[u] = c + u < n ? expf(total[at]) : 1.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (c + u < n) p[static_cast<long>(REV ? n - 1 - c - u : c + u) * (D * D)] = run;
      run = a[u] == 0.f ? x[u] : fmaf(a[u], run, x[u]);  // (a state that is dropped is dropped whatever it holds)
    }
  }
  if (!REV) p[static_cast<long>(n) * (D * D)] = run;
  float* to = REV ? g.dinitial : g.final_state;
  if (to) to[edge] = run;
}

enum { kGsOut = 0, kGsDq = 1, kGsDk = 2, kGsDv = 3 };

// The rows of one chunk: acc = rowfactor (A M) + (mask(A B^T) D) C
//     out: A = q   B = k   C = v   M = S          dq: A = dO  B = v   C = k  M = S^T
//     dk:  A = v   B = dO  C = q   M = R^T        dv: A = k   B = q   C = dO M = R
// The 4 x NB block of a thread: rows ty + 16 a, columns NB tx + e, or tx + 16 e where M enters transposed.
template <typename T, int D, int PASS>
__device__ __forceinline__ void gated_chunk(const GatedArgs& g, float* sA, float* sB, float* sC, float* sP, double* G) {
  constexpr int NB = D / 16, LD = D + 4, LP = kGsChunk + 4;
  constexpr bool LOWER = PASS == kGsOut || PASS == kGsDq, MT = PASS == kGsDq || PASS == kGsDk;
  constexpr int HALF = D > kGsChunk ? kGsChunk : D;  // rows of M that the B tile holds
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const long bh = blockIdx.x / g.nchunks, b = bh / g.H;
  const int chunk = static_cast<int>(blockIdx.x % g.nchunks), c0 = kGsChunk * chunk, h = static_cast<int>(bh % g.H);
  const bool with_state = LOWER ? chunk > 0 || g.with_initial : chunk + 1 < g.nchunks || g.dfinal;
  gated_sums<T>(g, G, b, h, c0);
  if constexpr (PASS == kGsOut) {
    gs_stage<T, D>(sA, g.q, g.sq, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sB, g.k, g.sk, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sC, g.v, g.sv, g, b, h, c0, tx, ty);
  } else if constexpr (PASS == kGsDq) {
    gs_stage<T, D>(sA, g.dout, g.so, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sB, g.v, g.sv, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sC, g.k, g.sk, g, b, h, c0, tx, ty);
  } else if constexpr (PASS == kGsDk) {
    gs_stage<T, D>(sA, g.v, g.sv, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sB, g.dout, g.so, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sC, g.q, g.sq, g, b, h, c0, tx, ty);
  } else {
    gs_stage<T, D>(sA, g.k, g.sk, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sB, g.q, g.sq, g, b, h, c0, tx, ty);
    gs_stage<T, D>(sC, g.dout, g.so, g, b, h, c0, tx, ty);
  }
  __syncthreads();

  {  // P = mask(A B^T) D: rows ty + 16 a, columns tx + 16 b
    float p[4][4] = {};
#pragma unroll 4
    for (int i = 0; i < D; i += 4) {
      float a[4][4], bb[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) gs_lds<4>(a[r], sA + (ty + 16 * r) * LD + i);
#pragma unroll
      for (int r = 0; r < 4; ++r) gs_lds<4>(bb[r], sB + (tx + 16 * r) * LD + i);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < 4; ++c) p[r][c] = fmaf(a[r][e], bb[c][e], p[r][c]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int t = ty + 16 * r, s = tx + 16 * c;
        const bool in = LOWER ? s <= t : s >= t;
        sP[t * LP + s] = in ? p[r][c] * expf(static_cast<float>(LOWER ? G[t] - G[s] : G[s] - G[t])) : 0.f;
      }
  }
  __syncthreads();

  float acc[4][NB] = {};
  if (with_state) {  // acc = A M (or A M^T), 64 rows of M at a time over the B tile, then the row factor
    const float* M = LOWER ? g.prefix + (bh * (g.nchunks + 1) + chunk) * static_cast<long>(D * D) : g.suffix + (bh * g.nchunks + chunk) * static_cast<long>(D * D);
#pragma unroll
    for (int m0 = 0; m0 < D; m0 += HALF) {
      if (m0) __syncthreads();
#pragma unroll
      for (int i = 0; i < HALF / 16; ++i) {
        float x[NB];
        gs_lds<NB>(x, M + (m0 + ty + 16 * i) * D + NB * tx);
#pragma unroll
        for (int e = 0; e < NB; ++e) sB[(ty + 16 * i) * LD + NB * tx + e] = x[e];
      }
      __syncthreads();
      if constexpr (MT) {  // columns tx + 16 j of the result are rows of M
#pragma unroll 2
        for (int i = 0; i < D; i += 4) {
          float a[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r) gs_lds<4>(a[r], sA + (ty + 16 * r) * LD + i);
#pragma unroll
          for (int j = 0; j < HALF / 16; ++j) {
            float bb[4];
            gs_lds<4>(bb, sB + (tx + 16 * j) * LD + i);
#pragma unroll
            for (int jj = 0; jj < NB; ++jj)
              if (jj == j + m0 / 16) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                  for (int r = 0; r < 4; ++r) acc[r][jj] = fmaf(a[r][e], bb[e], acc[r][jj]);
              }
          }
        }
      } else {
#pragma unroll 2
        for (int i = 0; i < HALF; i += 4) {
          float a[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r) gs_lds<4>(a[r], sA + (ty + 16 * r) * LD + m0 + i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float bb[NB];
            gs_lds<NB>(bb, sB + (i + e) * LD + NB * tx);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int j = 0; j < NB; ++j) acc[r][j] = fmaf(a[r][e], bb[j], acc[r][j]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = ty + 16 * r;
      const float f = expf(static_cast<float>(LOWER ? G[t] : G[kGsChunk - 1] - G[t]));
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[r][j] = f == 0.f ? 0.f : acc[r][j] * f;
    }
  }
  // acc += P C by blocks of 16 columns.  A row takes the columns on its side of the diagonal and no other: what a row may not see
  // is left out, not multiplied by zero (an infinity there would make a NaN of it).
#pragma unroll
  for (int blk = 0; blk < 4; ++blk) {
#pragma unroll 2
    for (int s = 16 * blk; s < 16 * blk + 16; s += 4) {
      float p[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (LOWER ? r >= blk : r <= blk) gs_lds<4>(p[r], sP + (ty + 16 * r) * LP + s);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float bb[NB];
        if constexpr (MT) {
#pragma unroll
          for (int j = 0; j < NB; ++j) bb[j] = sC[(s + e) * LD + tx + 16 * j];
        } else {
          gs_lds<NB>(bb, sC + (s + e) * LD + NB * tx);
        }
        const bool own = LOWER ? s + e <= ty + 16 * blk : s + e >= ty + 16 * blk;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if ((LOWER ? r > blk : r < blk) || (r == blk && own)) {
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[r][j] = fmaf(p[r][e], bb[j], acc[r][j]);
          }
      }
    }
  }

  // rows ty + 16 r.  A masked row is zero; dq and dk also leave their products with q and k for dg.
  T* dst = static_cast<T*>(PASS == kGsOut ? g.out : PASS == kGsDq ? g.dq : PASS == kGsDk ? g.dk : g.dv);
  const GatedStrides sd = PASS == kGsOut ? g.so : PASS == kGsDq ? g.sdq : PASS == kGsDk ? g.sdk : g.sdv;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int t = ty + 16 * r, pos = c0 + t;
    const bool in = pos < g.N;
    if (in && g.keep && !g.keep[b * g.N + pos]) {
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[r][j] = 0.f;
    }
    if constexpr (MT) {
      const T* x = static_cast<const T*>(PASS == kGsDq ? g.q : g.k) + gated_at(PASS == kGsDq ? g.sq : g.sk, b, h, pos);
      float dot = 0.f;
      const bool take = in && (!g.keep || g.keep[b * g.N + pos]);
#pragma unroll
      for (int j = 0; j < NB; ++j)
        if (take) dot = fmaf(to_acc(x[tx + 16 * j]), acc[r][j], dot);
      dot = gs_row_sum(dot);
      if (tx == 0) (PASS == kGsDq ? g.qdot : g.kdot)[static_cast<long>(blockIdx.x) * kGsChunk + t] = dot;
      if (in) {
#pragma unroll
        for (int j = 0; j < NB; ++j) dst[gated_at(sd, b, h, pos) + tx + 16 * j] = from_acc<T>(acc[r][j]);
      }
    } else {
      if (in) gs_store<T, NB>(dst + gated_at(sd, b, h, pos) + NB * tx, acc[r]);
    }
  }
}

// FWD: grid = B*H * chunks.  Backward: grid = (B*H * chunks, 3), y = dq, dk, dv.
template <typename T, int D, bool FWD>
__global__ void __launch_bounds__(kGsThreads, D > 64 ? 1 : 3) gated_chunk_kernel(const GatedArgs g) {
  extern __shared__ __align__(16) unsigned char gs_smem[];
  float* sA = reinterpret_cast<float*>(gs_smem);
  float* sB = sA + kGsChunk * (D + 4);
  float* sC = sB + kGsChunk * (D + 4);
  float* sP = sC + kGsChunk * (D + 4);
  __shared__ double G[kGsChunk];
  pdl_allow_next();
  pdl_wait_prior();
  if constexpr (FWD) {
    gated_chunk<T, D, kGsOut>(g, sA, sB, sC, sP, G);
  } else {
    if (blockIdx.y == 0)
      gated_chunk<T, D, kGsDq>(g, sA, sB, sC, sP, G);
    else if (blockIdx.y == 1)
      gated_chunk<T, D, kGsDk>(g, sA, sB, sC, sP, G);
    else
      gated_chunk<T, D, kGsDv>(g, sA, sB, sC, sP, G);
  }
}

// dg of a chunk.  Nothing crosses a gate that drops the state (e^g = 0 in fp32): what lies behind it is left out of the sums before it,
// whatever it holds.  Such a gate has no gradient, nor has the first gate of a sequence that starts from nothing, nor a masked one.
// grid = B*H * chunks.
template <typename T, int D>
__global__ void __launch_bounds__(kGsThreads) gated_dgate_kernel(const GatedArgs g) {
  __shared__ double part[kGsThreads / 32];
  __shared__ double d[kGsChunk];
  const int tid = threadIdx.x, lane = tid & 31;
  const long bh = blockIdx.x / g.nchunks, b = bh / g.H;
  const int chunk = static_cast<int>(blockIdx.x % g.nchunks), c0 = kGsChunk * chunk, h = static_cast<int>(bh % g.H);
  pdl_allow_next();
  pdl_wait_prior();
  double cross = 0.0;
  if (chunk + 1 < g.nchunks || g.dfinal) {
    const float *S = g.prefix + (bh * (g.nchunks + 1) + chunk + 1) * static_cast<long>(D * D), *R = g.suffix + (bh * g.nchunks + chunk) * static_cast<long>(D * D);
#pragma unroll 8
    for (int e = tid; e < D * D; e += kGsThreads) cross = fma(static_cast<double>(S[e]), static_cast<double>(R[e]), cross);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) cross += __shfl_xor_sync(0xffffffffu, cross, off);
  }
  if (lane == 0) part[tid >> 5] = cross;
  if (tid < kGsChunk) {
    const long o = static_cast<long>(blockIdx.x) * kGsChunk + tid;
    d[tid] = static_cast<double>(g.qdot[o]) - static_cast<double>(g.kdot[o]);
  }
  __syncthreads();
  if (tid < 32) {
    cross = 0.0;
#pragma unroll
    for (int w = 0; w < kGsThreads / 32; ++w) cross += part[w];
    // lane l has positions 63 - 2 l and 62 - 2 l.  The sum at a position is its own term and, unless the next gate drops the state,
    // the sum there; the last position's next one is the chunk's end, whose sum is <S', R>.
    const int p1 = c0 + 63 - 2 * lane;
    const double d1 = d[63 - 2 * lane], d0 = d[62 - 2 * lane];
    const bool drop1 = p1 < g.N && expf(static_cast<float>(gated_gate<T>(g, b, h, p1))) == 0.f,
               drop0 = p1 - 1 < g.N && expf(static_cast<float>(gated_gate<T>(g, b, h, p1 - 1))) == 0.f;
    double run = drop0 ? 0.0 : drop1 ? d0 : d0 + d1;  // of what the positions of lanes up to this one hand on, their own part
    int open = !drop0 && !drop1;                      // whether they hand on what comes from behind them
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, run, off);
      const int up_open = __shfl_up_sync(0xffffffffu, open, off);
      if (lane >= off && open) run += up, open = up_open;
    }
    double in = __shfl_up_sync(0xffffffffu, run, 1);
    const int in_open = __shfl_up_sync(0xffffffffu, open, 1);
    in = lane == 0 ? cross : in_open ? in + cross : in;
    const double at1 = d1 + in, at0 = drop1 ? d0 : d0 + at1;
    const double sums[2] = {at1, at0};
    const bool drops[2] = {drop1, drop0};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int pos = c0 + 63 - 2 * lane - u;
      if (pos < g.N) {
        const bool masked = g.keep && !g.keep[b * g.N + pos];
        const bool none = masked || (pos == 0 && !g.with_initial) || drops[u];
        const float x = none ? 0.f : static_cast<float>(sums[u]);
        const long long o = gated_at(g.sdg, b, h, pos);
        if (g.gate_f32)
          static_cast<float*>(g.dgate)[o] = x;
        else
          static_cast<T*>(g.dgate)[o] = from_acc<T>(x);
      }
    }
  }
}

// The tensor-core kernels of the 16-bit types at head dims 64 and 128 (gated_tc_api.cu); `states`, `workspace` as in the C ABI.
bool gated_tc_usable(int D, int dtype);
size_t gated_tc_states_bytes(int B, int H, int N, int D);
size_t gated_tc_workspace_bytes(int B, int H, int N, int D, bool backward);
int gated_tc_fwd(const GatedArgs& g, void* states, void* workspace, int B, int D, int dtype, cudaStream_t stream);
int gated_tc_bwd(const GatedArgs& g, const void* states, void* workspace, int B, int D, int dtype, cudaStream_t stream);

}  // namespace cott
