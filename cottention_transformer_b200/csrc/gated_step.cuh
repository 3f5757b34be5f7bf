// Single-token form of the gated scan (HBM-bound, CUDA cores): per (batch, head) and token
//     state[j][i] = e^g state[j][i] + v[j] k[i]          out[j] = sum_i q[i] state[j][i]
// with the fp32 states [B, H, value, key] in HBM, read and written once per call (T consecutive tokens keep them in registers).
//
// A row of a state is spread over D/4 lanes that own one float4 each; a warp owns 4 KB of a state (16 rows of 64, 8 rows of 128) in
// eight float4 a lane, all of whose loads are in flight together, and needs nothing from any other warp: a row's dot product is a
// shuffle reduction, q and k come straight from the cache as the lane's own piece.  No barrier, no shared memory.
#pragma once

#include "common.cuh"

namespace cott {

constexpr int kStepThreads = 128;
constexpr int kStepRows = 8;  // float4 per lane

struct StepArgs {
  float* state;
  const void *q, *k, *v, *gate;
  void* out;
  cott_strides sq, sk, sv, so, sg;
  long units;  // warps with work
  int H, T, gate_f32;
};

template <typename T> struct alignas(4 * sizeof(T)) Quad { T e[4]; };
template <typename T>
__device__ __forceinline__ float4 ld_quad(const T* p) {
  const Quad<T> v = *reinterpret_cast<const Quad<T>*>(p);
  return make_float4(to_acc(v.e[0]), to_acc(v.e[1]), to_acc(v.e[2]), to_acc(v.e[3]));
}

template <typename T, int D>
__global__ void __launch_bounds__(kStepThreads) gated_step_kernel(const StepArgs a) {
  constexpr int LPR = D / 4, RPI = 32 / LPR, ROWS = RPI * kStepRows, UNITS = D / ROWS;  // lanes per row; rows per load, per warp; warps per state
  static_assert(D % ROWS == 0, "a state is whole warps");
  const int lane = threadIdx.x & 31, piece = lane % LPR;
  const long unit = static_cast<long>(blockIdx.x) * (kStepThreads / 32) + (threadIdx.x >> 5);
  pdl_allow_next();  // (a token loop is a chain of these launches: the next one is placed while this one drains)
  pdl_wait_prior();
  if (unit >= a.units) return;
  const long bh = unit / UNITS, b = bh / a.H, h = bh % a.H;
  const int j0 = static_cast<int>(unit % UNITS) * ROWS + lane / LPR;  // then += RPI
  float* st = a.state + bh * (D * D) + static_cast<long>(j0) * D + 4 * piece;
  float4 s[kStepRows];
#pragma unroll
  for (int r = 0; r < kStepRows; ++r) s[r] = *reinterpret_cast<const float4*>(st + r * RPI * D);
  const T* q = static_cast<const T*>(a.q) + b * a.sq.b + h * a.sq.h + 4 * piece;
  const T* k = static_cast<const T*>(a.k) + b * a.sk.b + h * a.sk.h + 4 * piece;
  const T* v = static_cast<const T*>(a.v) + b * a.sv.b + h * a.sv.h + j0;
  T* out = static_cast<T*>(a.out) + b * a.so.b + h * a.so.h + j0;
  const long long g0 = b * a.sg.b + h * a.sg.h;
#pragma unroll 1
  for (int t = 0; t < a.T; ++t, q += a.sq.n, k += a.sk.n, v += a.sv.n, out += a.so.n) {
    const float4 q4 = ld_quad(q), k4 = ld_quad(k);
    const long long o = g0 + t * a.sg.n;
    const float decay = expf(a.gate_f32 ? static_cast<const float*>(a.gate)[o] : to_acc(static_cast<const T*>(a.gate)[o]));
    float x[kStepRows];
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) x[r] = to_acc(v[r * RPI]);
    if (decay == 0.f) {  // a state that is dropped is dropped whatever it holds
#pragma unroll
      for (int r = 0; r < kStepRows; ++r) s[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
      s[r].x = fmaf(decay, s[r].x, x[r] * k4.x);
      s[r].y = fmaf(decay, s[r].y, x[r] * k4.y);
      s[r].z = fmaf(decay, s[r].z, x[r] * k4.z);
      s[r].w = fmaf(decay, s[r].w, x[r] * k4.w);
      x[r] = fmaf(q4.x, s[r].x, fmaf(q4.y, s[r].y, fmaf(q4.z, s[r].z, q4.w * s[r].w)));
    }
#pragma unroll
    for (int r = 0; r < kStepRows; ++r) {
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1) x[r] += __shfl_xor_sync(0xffffffffu, x[r], off);
      if (piece == 0) out[r * RPI] = from_acc<T>(x[r]);
    }
  }
#pragma unroll
  for (int r = 0; r < kStepRows; ++r) *reinterpret_cast<float4*>(st + r * RPI * D) = s[r];
}

template <typename T, int D>
int launch_gated_step(StepArgs a, long states, cudaStream_t stream) {
  constexpr int UNITS = D / (32 / (D / 4) * kStepRows);
  a.units = states * UNITS;
  COTT_CUDA_TRY(launch_pdl(gated_step_kernel<T, D>, dim3(static_cast<unsigned>((a.units + kStepThreads / 32 - 1) / (kStepThreads / 32))), kStepThreads, 0,
                           stream, a));
  return COTT_OK;
}

}  // namespace cott
