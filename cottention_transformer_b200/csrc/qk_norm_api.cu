// RMS norm of every head of q and k with a learned weight, and the rotary embedding ("rotate every two"), in one pass:
//     n = x rsqrt(mean x^2 + eps)      y = Rot(n w)
// and its backward, with e = Rot^T dy, f = e w:
//     dw = sum over all rows of e n            dx = r (f - n mean(f n)),  r = rsqrt(mean x^2 + eps)
// A row (one head of one position) is spread over D/8 lanes (16 bits) or D/4 lanes (fp32) that own one 16-byte piece each, so every
// access is a whole 16 bytes, pairs of the rotation stay inside a lane and the row sums are shuffles.  fp32 arithmetic, one rounding.
// HBM-bound: every input is read once and every output written once; the backward recomputes r from x.  The gradient of a weight is
// summed in registers over the rows of a thread, over the CTA in shared memory and over the CTAs by a second small kernel, all in a
// fixed order.
#include "common.cuh"

using namespace cott;

namespace {

constexpr int kNormThreads = 256;

template <typename T> struct Piece {
  static constexpr int kElems = 16 / sizeof(T);
  union {
    uint4 u;
    T e[kElems];
  };
  __device__ __forceinline__ Piece() {}
};

// Division of numbers below 2^31 by a number known at launch: m = ceil(2^(31+s) / d) with 2^s >= d has d m - 2^(31+s) < 2^s, which
// is what makes (r m) >> (31+s) exact.  (Two divisions per row are otherwise most of a row's instructions.)
struct Divider {
  unsigned d, m;
  int shift;
};
Divider divider(unsigned d) {
  Divider r = {d, 0, 31};
  int s = 0;
  while ((1ull << s) < d) ++s;
  r.shift = 31 + s;
  r.m = (unsigned)(((1ull << r.shift) + d - 1) / d);
  return r;
}
__device__ __forceinline__ unsigned divide(unsigned r, const Divider& d) {
  return static_cast<unsigned>((static_cast<unsigned long long>(r) * d.m) >> d.shift);
}

struct NormSide {  // q or k
  const void *x, *w, *dy;
  void *y, *dx;
  cott_strides sx, sy, sdy, sdx;
  Divider heads;
  unsigned rows;  // B * N * H
};
struct NormArgs {
  NormSide side[2];
  const float *sin_t, *cos_t;
  float* partial;  // backward: [2][CTAs][D]
  long long table_batch_stride;
  Divider positions;
  int rot, w_f32;
  float eps;
};

// The row numbered `r` of a side: consecutive numbers walk the heads of a position, then the positions, then the batch.
struct RowAt {
  unsigned b, n, h;
};
__device__ __forceinline__ RowAt row_at(unsigned r, const Divider& heads, const Divider& positions) {
  const unsigned p = divide(r, heads), b = divide(p, positions);
  return RowAt{b, p - b * positions.d, r - p * heads.d};
}
__device__ __forceinline__ long long at(const cott_strides& s, const RowAt& r) { return r.b * s.b + r.h * s.h + r.n * s.n; }

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}
// Two products, two multiply-adds in one instruction (the pass is as much bound by its instructions as by memory).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 c;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;\n}"
      : "=f"(c.x), "=f"(c.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return c;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\nfma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// the lane's E weights
template <typename T, int E>
__device__ __forceinline__ void load_weights(float2 (&w)[E / 2], const void* src, int f32, int c) {
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = f32 ? static_cast<const float*>(src)[c + e] : to_acc(static_cast<const T*>(src)[c + e]);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) w[e] = make_float2(x[2 * e], x[2 * e + 1]);
}
// rotates the lane's E/2 pairs; `sign` = -1: the transposed rotation
template <int E>
__device__ __forceinline__ void rotate(float2 (&x)[E / 2], const float* sin_t, const float* cos_t, float sign) {
  float s[E / 2], c[E / 2];
  if constexpr (E == 8) {
    *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sin_t);
    *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cos_t);
  } else {
    *reinterpret_cast<float2*>(s) = *reinterpret_cast<const float2*>(sin_t);
    *reinterpret_cast<float2*>(c) = *reinterpret_cast<const float2*>(cos_t);
  }
#pragma unroll
  for (int i = 0; i < E / 2; ++i) x[i] = fma2(x[i], both(c[i]), mul2(make_float2(x[i].y, x[i].x), make_float2(-sign * s[i], sign * s[i])));
}

// grid = (CTAs, 2): y = q, k.  A CTA takes U groups of rows at a time, all of whose loads are in flight together: with one group
// the pass reached 3.6 TB/s.
template <typename T, int D, int U>
__global__ void __launch_bounds__(kNormThreads) qk_norm_fwd_kernel(const NormArgs a) {
  constexpr int E = Piece<T>::kElems, LPR = D / E, RPC = kNormThreads / LPR;  // elements and lanes of a piece, rows per group
  const NormSide& s = a.side[blockIdx.y];
  const int piece = threadIdx.x % LPR, c = piece * E;
  pdl_allow_next();
  pdl_wait_prior();
  float2 w[E / 2];
  load_weights<T, E>(w, s.w, a.w_f32, c);
  for (unsigned r0 = blockIdx.x * (RPC * U); r0 < s.rows; r0 += gridDim.x * (RPC * U)) {
    RowAt row[U];
    Piece<T> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned r = r0 + u * RPC + threadIdx.x / LPR;
      row[u] = row_at(r < s.rows ? r : s.rows - 1, s.heads, a.positions);
      p[u].u = *reinterpret_cast<const uint4*>(static_cast<const T*>(s.x) + at(s.sx, row[u]) + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 x[E / 2], sum = both(0.f);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        x[e] = make_float2(to_acc(p[u].e[2 * e]), to_acc(p[u].e[2 * e + 1]));
        sum = fma2(x[e], x[e], sum);
      }
      const float rms = rsqrtf(row_sum<LPR>(sum.x + sum.y) * (1.f / D) + a.eps);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) x[e] = mul2(mul2(x[e], both(rms)), w[e]);
      if (c < a.rot) {
        const long long t = row[u].b * a.table_batch_stride + static_cast<long long>(row[u].n) * (a.rot / 2) + c / 2;
        rotate<E>(x, a.sin_t + t, a.cos_t + t, 1.f);
      }
#pragma unroll
      for (int e = 0; e < E / 2; ++e) p[u].e[2 * e] = from_acc<T>(x[e].x), p[u].e[2 * e + 1] = from_acc<T>(x[e].y);
      if (r0 + u * RPC + threadIdx.x / LPR < s.rows) *reinterpret_cast<uint4*>(static_cast<T*>(s.y) + at(s.sy, row[u]) + c) = p[u].u;
    }
  }
}

template <typename T, int D, int U>
__global__ void __launch_bounds__(kNormThreads) qk_norm_bwd_kernel(const NormArgs a) {
  constexpr int E = Piece<T>::kElems, LPR = D / E, RPC = kNormThreads / LPR;
  const NormSide& s = a.side[blockIdx.y];
  const int piece = threadIdx.x % LPR, c = piece * E;
  __shared__ float part[RPC][D];
  pdl_allow_next();
  pdl_wait_prior();
  float2 w[E / 2], dw[E / 2];
  load_weights<T, E>(w, s.w, a.w_f32, c);
#pragma unroll
  for (int e = 0; e < E / 2; ++e) dw[e] = both(0.f);
  for (unsigned r0 = blockIdx.x * (RPC * U); r0 < s.rows; r0 += gridDim.x * (RPC * U)) {
    RowAt row[U];
    Piece<T> p[U], d[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const unsigned r = r0 + u * RPC + threadIdx.x / LPR;
      row[u] = row_at(r < s.rows ? r : s.rows - 1, s.heads, a.positions);
      p[u].u = *reinterpret_cast<const uint4*>(static_cast<const T*>(s.x) + at(s.sx, row[u]) + c);
      d[u].u = *reinterpret_cast<const uint4*>(static_cast<const T*>(s.dy) + at(s.sdy, row[u]) + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = r0 + u * RPC + threadIdx.x / LPR < s.rows;
      float2 x[E / 2], f[E / 2], sum = both(0.f);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        x[e] = make_float2(to_acc(p[u].e[2 * e]), to_acc(p[u].e[2 * e + 1]));
        f[e] = make_float2(to_acc(d[u].e[2 * e]), to_acc(d[u].e[2 * e + 1]));
        sum = fma2(x[e], x[e], sum);
      }
      if (c < a.rot) {
        const long long t = row[u].b * a.table_batch_stride + static_cast<long long>(row[u].n) * (a.rot / 2) + c / 2;
        rotate<E>(f, a.sin_t + t, a.cos_t + t, -1.f);
      }
      const float rms = rsqrtf(row_sum<LPR>(sum.x + sum.y) * (1.f / D) + a.eps);
      float2 dot2 = both(0.f);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        x[e] = mul2(x[e], both(rms));
        if (in) dw[e] = fma2(f[e], x[e], dw[e]);
        f[e] = mul2(f[e], w[e]);
        dot2 = fma2(f[e], x[e], dot2);
      }
      const float dot = row_sum<LPR>(dot2.x + dot2.y) * (1.f / D);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        const float2 g = mul2(fma2(x[e], both(-dot), f[e]), both(rms));
        p[u].e[2 * e] = from_acc<T>(g.x), p[u].e[2 * e + 1] = from_acc<T>(g.y);
      }
      if (in) *reinterpret_cast<uint4*>(static_cast<T*>(s.dx) + at(s.sdx, row[u]) + c) = p[u].u;
    }
  }
#pragma unroll
  for (int e = 0; e < E / 2; ++e) part[threadIdx.x / LPR][c + 2 * e] = dw[e].x, part[threadIdx.x / LPR][c + 2 * e + 1] = dw[e].y;
  __syncthreads();
  for (int e = threadIdx.x; e < D; e += kNormThreads) {
    float sum = 0.f;
#pragma unroll 8
    for (int i = 0; i < RPC; ++i) sum += part[i][e];
    a.partial[(static_cast<long>(blockIdx.y) * gridDim.x + blockIdx.x) * D + e] = sum;
  }
}

// dw of q and of k: the sums of the CTAs, in a fixed order.  grid = (D / 32, 2), block = 1024: 32 columns, 32 threads each.
template <typename T>
__global__ void __launch_bounds__(1024) qk_norm_dw_kernel(const float* __restrict__ partial, void* dqw, void* dkw, int ctas, int D, int w_f32) {
  __shared__ float part[32][33];
  const int col = threadIdx.x & 31, u = threadIdx.x >> 5, e = blockIdx.x * 32 + col;
  pdl_allow_next();
  pdl_wait_prior();
  const float* src = partial + static_cast<long>(blockIdx.y) * ctas * D;
  float sum = 0.f;
#pragma unroll 8
  for (int i = u; i < ctas; i += 32) sum += src[static_cast<long>(i) * D + e];
  part[u][col] = sum;
  __syncthreads();
  if (u == 0) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += part[i][col];
    void* dst = blockIdx.y ? dkw : dqw;
    if (w_f32)
      static_cast<float*>(dst)[e] = sum;
    else
      static_cast<T*>(dst)[e] = from_acc<T>(sum);
  }
}

int check_norm_args(int B, int Hq, int Hk, int N, int D, int dtype, int weight_dtype, const cott_rotary_tables* rotary) {
  if (dtype != COTT_F32 && dtype != COTT_F16 && dtype != COTT_BF16)
    return fail(COTT_ERR_DTYPE, "cott_qk_norm takes float32, float16 or bfloat16 (dtype code %d)", dtype);
  if (weight_dtype != COTT_F32 && weight_dtype != dtype)
    return fail(COTT_ERR_DTYPE, "cott_qk_norm: the weights are float32 or of the tensors' type (dtype code %d)", weight_dtype);
  if (B < 0 || Hq < 0 || Hk < 0 || N < 0) return fail(COTT_ERR_SHAPE, "negative size B=%d Hq=%d Hk=%d N=%d", B, Hq, Hk, N);
  if (D != 32 && D != 64 && D != 128) return fail(COTT_ERR_SHAPE, "cott_qk_norm supports head dims 32, 64 and 128 (got %d)", D);
  if ((double)B * N * (Hq > Hk ? Hq : Hk) > 2147483647.0) return fail(COTT_ERR_SHAPE, "B*H*N too large");
  if (rotary) {
    if (rotary->rot_dim < 8 || rotary->rot_dim % 8 || rotary->rot_dim > D)
      return fail(COTT_ERR_SHAPE, "the rotary dim must be a multiple of 8 and at most the head dim (got %d, %d)", rotary->rot_dim, D);
    if (!rotary->sin_table || !rotary->cos_table) return fail(COTT_ERR_NULL, "null pointer: rotary table");
    if ((reinterpret_cast<uintptr_t>(rotary->sin_table) | reinterpret_cast<uintptr_t>(rotary->cos_table)) & 15 || rotary->table_batch_stride % 4)
      return fail(COTT_ERR_ALIGN, "rotary tables must be 16-byte aligned");
  }
  return COTT_OK;
}
int check_norm_rows(const char* name, const void* p, const cott_strides& s, int dtype) {
  const long long unit = 16 / (long long)dtype_size(dtype);
  if (!p) return fail(COTT_ERR_NULL, "null pointer: %s", name);
  if (reinterpret_cast<uintptr_t>(p) & 15) return fail(COTT_ERR_ALIGN, "%s must be 16-byte aligned", name);
  if (s.b % unit || s.h % unit || s.n % unit) return fail(COTT_ERR_ALIGN, "the strides of %s must be multiples of 16 bytes", name);
  return COTT_OK;
}

int norm_ctas(unsigned rows, int rows_per_cta, int resident) {
  int sm = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sm, cudaDevAttrMultiProcessorCount, dev);
  const long want = ((long)rows + rows_per_cta - 1) / rows_per_cta, most = (long)sm * resident;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}
constexpr int kBwdResident = 4, kFwdGroups = 4, kBwdGroups = 2;

template <typename T, int D>
int launch_norm(const NormArgs& a, bool bwd, void* dqw, void* dkw, cudaStream_t stream) {
  constexpr int RPC = kNormThreads / (D / Piece<T>::kElems);
  const unsigned rows = a.side[0].rows > a.side[1].rows ? a.side[0].rows : a.side[1].rows;
  if (!bwd) {
    // (few rows, as of new tokens: one group per CTA, so that they are spread over the SMs)
    if (rows <= 148u * RPC)
      COTT_CUDA_TRY(launch_pdl(qk_norm_fwd_kernel<T, D, 1>, dim3(norm_ctas(rows, RPC, 64), 2), kNormThreads, 0, stream, a));
    else
      COTT_CUDA_TRY(launch_pdl(qk_norm_fwd_kernel<T, D, kFwdGroups>, dim3(norm_ctas(rows, RPC * kFwdGroups, 64), 2), kNormThreads, 0, stream, a));
    return COTT_OK;
  }
  const int ctas = norm_ctas(rows, RPC * kBwdGroups, kBwdResident);
  COTT_CUDA_TRY(launch_pdl(qk_norm_bwd_kernel<T, D, kBwdGroups>, dim3(ctas, 2), kNormThreads, 0, stream, a));
  COTT_CUDA_TRY(launch_pdl(qk_norm_dw_kernel<T>, dim3(D / 32, 2), 1024, 0, stream, static_cast<const float*>(a.partial), dqw, dkw, ctas, D, a.w_f32));
  return COTT_OK;
}
template <typename T>
int launch_norm_dim(const NormArgs& a, int D, bool bwd, void* dqw, void* dkw, cudaStream_t stream) {
  switch (D) {
    case 32: return launch_norm<T, 32>(a, bwd, dqw, dkw, stream);
    case 64: return launch_norm<T, 64>(a, bwd, dqw, dkw, stream);
    default: return launch_norm<T, 128>(a, bwd, dqw, dkw, stream);
  }
}
int launch_norm_any(const NormArgs& a, int D, int dtype, bool bwd, void* dqw, void* dkw, cudaStream_t stream) {
  switch (dtype) {
    case COTT_F32: return launch_norm_dim<float>(a, D, bwd, dqw, dkw, stream);
    case COTT_F16: return launch_norm_dim<__half>(a, D, bwd, dqw, dkw, stream);
    default: return launch_norm_dim<__nv_bfloat16>(a, D, bwd, dqw, dkw, stream);
  }
}
NormArgs norm_args(const cott_norm_layout* l, const void* q, const void* k, const void* qw, const void* kw, const cott_rotary_tables* rotary, int B,
                   int Hq, int Hk, int N, int D, int weight_dtype, float eps) {
  NormArgs a = {};
  const cott_strides dq = {(long long)Hq * N * D, (long long)N * D, D}, dk = {(long long)Hk * N * D, (long long)N * D, D};
  a.side[0].x = q, a.side[0].w = qw, a.side[0].heads = divider(Hq), a.side[0].rows = (unsigned)((long)B * N * Hq), a.side[0].sx = l ? l->q : dq;
  a.side[1].x = k, a.side[1].w = kw, a.side[1].heads = divider(Hk), a.side[1].rows = (unsigned)((long)B * N * Hk), a.side[1].sx = l ? l->k : dk;
  a.side[0].sy = a.side[0].sdy = l ? l->q_out : dq, a.side[1].sy = a.side[1].sdy = l ? l->k_out : dk;
  a.side[0].sdx = l ? l->dq : dq, a.side[1].sdx = l ? l->dk : dk;
  a.positions = divider(N), a.w_f32 = weight_dtype == COTT_F32, a.eps = eps;
  if (rotary) a.sin_t = rotary->sin_table, a.cos_t = rotary->cos_table, a.rot = rotary->rot_dim, a.table_batch_stride = rotary->table_batch_stride;
  return a;
}

}  // namespace

extern "C" {

int cott_qk_norm_fwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const cott_rotary_tables* rotary, void* q_out, void* k_out,
                     const cott_norm_layout* layout, int B, int Hq, int Hk, int N, int D, float eps, int dtype, int weight_dtype, void* stream) {
  int st = check_norm_args(B, Hq, Hk, N, D, dtype, weight_dtype, rotary);
  if (st) return st;
  if ((long)B * N * (Hq + Hk) == 0) return COTT_OK;
  if (!Hq || !Hk) return fail(COTT_ERR_SHAPE, "q and k need a head each");
  NormArgs a = norm_args(layout, q, k, q_weight, k_weight, rotary, B, Hq, Hk, N, D, weight_dtype, eps);
  a.side[0].y = q_out, a.side[1].y = k_out;
  if ((st = check_norm_rows("q", q, a.side[0].sx, dtype)) || (st = check_norm_rows("q_out", q_out, a.side[0].sy, dtype)) ||
      (st = check_norm_rows("k", k, a.side[1].sx, dtype)) || (st = check_norm_rows("k_out", k_out, a.side[1].sy, dtype)))
    return st;
  if (!q_weight || !k_weight) return fail(COTT_ERR_NULL, "null pointer: weight");
  DeviceScope scope(q);
  COTT_CUDA_TRY(scope.status());
  return launch_norm_any(a, D, dtype, false, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

size_t cott_qk_norm_workspace_bytes(int B, int Hq, int Hk, int N, int D) {
  if (B <= 0 || Hq <= 0 || Hk <= 0 || N <= 0 || D <= 0) return 0;
  return (size_t)2 * norm_ctas(0x7fffffff, 1, kBwdResident) * D * sizeof(float);
}

int cott_qk_norm_bwd(const void* q, const void* k, const void* q_weight, const void* k_weight, const cott_rotary_tables* rotary, const void* dq_out,
                     const void* dk_out, void* workspace, void* dq, void* dk, void* dq_weight, void* dk_weight, const cott_norm_layout* layout, int B,
                     int Hq, int Hk, int N, int D, float eps, int dtype, int weight_dtype, void* stream) {
  int st = check_norm_args(B, Hq, Hk, N, D, dtype, weight_dtype, rotary);
  if (st) return st;
  if (!dq_weight || !dk_weight) return fail(COTT_ERR_NULL, "null pointer: weight gradient");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if ((long)B * N * (Hq + Hk) == 0) {
    DeviceScope scope(dq_weight);
    COTT_CUDA_TRY(scope.status());
    COTT_CUDA_TRY(cudaMemsetAsync(dq_weight, 0, D * dtype_size(weight_dtype), s));
    COTT_CUDA_TRY(cudaMemsetAsync(dk_weight, 0, D * dtype_size(weight_dtype), s));
    return COTT_OK;
  }
  if (!Hq || !Hk) return fail(COTT_ERR_SHAPE, "q and k need a head each");
  NormArgs a = norm_args(layout, q, k, q_weight, k_weight, rotary, B, Hq, Hk, N, D, weight_dtype, eps);
  a.side[0].dy = dq_out, a.side[1].dy = dk_out, a.side[0].dx = dq, a.side[1].dx = dk, a.partial = static_cast<float*>(workspace);
  if ((st = check_norm_rows("q", q, a.side[0].sx, dtype)) || (st = check_norm_rows("k", k, a.side[1].sx, dtype)) ||
      (st = check_norm_rows("dq_out", dq_out, a.side[0].sdy, dtype)) || (st = check_norm_rows("dk_out", dk_out, a.side[1].sdy, dtype)) ||
      (st = check_norm_rows("dq", dq, a.side[0].sdx, dtype)) || (st = check_norm_rows("dk", dk, a.side[1].sdx, dtype)))
    return st;
  if (!q_weight || !k_weight || !workspace) return fail(COTT_ERR_NULL, "null pointer: %s", workspace ? "weight" : "workspace");
  DeviceScope scope(q);
  COTT_CUDA_TRY(scope.status());
  return launch_norm_any(a, D, dtype, true, dq_weight, dk_weight, s);
}

}  // extern "C"
