// RMS norm of every head of q and k with a learned weight, and the rotary embedding ("rotate every two"), in one pass:
//     n = x rsqrt(mean x^2 + eps)      y = Rot(n w)
// and its backward, with e = Rot^T dy, f = e w:
//     dw = sum over all rows of e n            dx = r (f - n mean(f n)),  r = rsqrt(mean x^2 + eps)
// A row (one head of one position) is spread over D/8 lanes (16 bits) or D/4 lanes (fp32) that own one 16-byte piece each, so every
// access is a whole 16 bytes, pairs of the rotation stay inside a lane and the row sums are shuffles.  fp32 arithmetic, one rounding.
// HBM-bound: every input is read once and every output written once; the backward recomputes r from x.  The gradient of a weight is
// summed in registers over the rows of a thread, over the CTA in shared memory and over the CTAs by a second small kernel, all in a
// fixed order.
// (Packed arithmetic, mul2 and fma2: the pass is as much bound by its instructions as by memory.)
#include "common.cuh"

using namespace cott;

namespace {

constexpr int kNormThreads = 256;
constexpr int kSms = 148, kFwdResident = 4, kBwdResident = 3;  // CTAs per SM, by their registers
constexpr int kFwdStages = 3, kBwdStages = 2;

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
// A piece of 16 bytes of this thread's own, from global to its place in shared memory without a register in between.
__device__ __forceinline__ void fetch16(void* smem, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "l"(src) : "memory");
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
#pragma unroll
  for (int off = LPR / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
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
// a position's sines and cosines of the lane's E/2 pairs; apply() rotates, `sign` = -1: by the transposed rotation
template <int E> struct Turn {
  float s[E / 2], c[E / 2];
  __device__ __forceinline__ void load(const float* sin_t, const float* cos_t) {
    if constexpr (E == 8) {
      *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(sin_t);
      *reinterpret_cast<float4*>(c) = *reinterpret_cast<const float4*>(cos_t);
    } else {
      *reinterpret_cast<float2*>(s) = *reinterpret_cast<const float2*>(sin_t);
      *reinterpret_cast<float2*>(c) = *reinterpret_cast<const float2*>(cos_t);
    }
  }
  __device__ __forceinline__ void apply(float2 (&x)[E / 2], float sign) const {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) x[i] = fma2(x[i], both(c[i]), mul2(make_float2(x[i].y, x[i].x), make_float2(-sign * s[i], sign * s[i])));
  }
};

// Both passes.  A thread always has the same piece of a row, and takes every so many-th row: of q and of k both (SIDES = 2: as many
// heads in one as in the other), which share the position's table entries, or of one of them (SIDES = 1: blockIdx.x even q, odd k).
// The pieces of the next STAGES rows are on their way while one is worked on: each thread fetches its own into its own places in
// shared memory, so nobody waits for anybody else.
// B8 H16 N4096, q and k of a packed projection, us forward / backward: one row at a time 74 / 123, four and two rows loaded together
// 60 / 90, fetched ahead 63 / 89 (46 without the rotation: the tables were twice the data), q and k together 46 / 73.
template <typename T, int D, bool BWD, int STAGES, int SIDES>
__global__ void __launch_bounds__(kNormThreads, STAGES == 1 ? 1 : BWD ? kBwdResident : kFwdResident) qk_norm_kernel(const NormArgs a) {
  constexpr int E = Piece<T>::kElems, LPR = D / E, RPC = kNormThreads / LPR;  // elements and lanes of a piece, rows per round
  const int first_side = SIDES == 2 ? 0 : blockIdx.x & 1, cta = SIDES == 2 ? blockIdx.x : blockIdx.x >> 1, ctas = SIDES == 2 ? gridDim.x : gridDim.x >> 1;
  const int c = threadIdx.x % LPR * E;
  const unsigned group = RPC * ctas, rows = a.side[first_side].rows;
  extern __shared__ __align__(16) unsigned char norm_smem[];  // pieces [STAGES][SIDES][x, dy][threads]; at the end [RPC][D] sums
  uint4* buf = reinterpret_cast<uint4*>(norm_smem) + threadIdx.x;
  auto place = [&](int stage, int i, int dy) { return buf + ((stage * SIDES + i) * (BWD ? 2 : 1) + dy) * kNormThreads; };
  pdl_allow_next();
  pdl_wait_prior();
  float2 w[SIDES][E / 2], dw[SIDES][E / 2];
#pragma unroll
  for (int i = 0; i < SIDES; ++i) {
    load_weights<T, E>(w[i], a.side[first_side + i].w, a.w_f32, c);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) dw[i][e] = both(0.f);
  }
  auto fetch = [&](unsigned r, int stage) {
    if (r < rows) {
      const RowAt row = row_at(r, a.side[first_side].heads, a.positions);
#pragma unroll
      for (int i = 0; i < SIDES; ++i) {
        const NormSide& s = a.side[first_side + i];
        fetch16(place(stage, i, 0), static_cast<const T*>(s.x) + at(s.sx, row) + c);
        if constexpr (BWD) fetch16(place(stage, i, 1), static_cast<const T*>(s.dy) + at(s.sdy, row) + c);
      }
    }
    fetch_commit();
  };
  const unsigned first = cta * RPC + threadIdx.x / LPR;
#pragma unroll
  for (int i = 0; i < STAGES; ++i) fetch(first + i * group, i);
  int stage = 0;
  // (as many rounds for every lane of a warp: the rows' sums are exchanged by all)
  for (unsigned r = first; __any_sync(0xffffffffu, r < rows); r += group) {
    fetch_wait<STAGES - 1>();
    Piece<T> p[SIDES], d[SIDES];
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      p[i].u = *place(stage, i, 0);
      if constexpr (BWD) d[i].u = *place(stage, i, 1);
    }
    const bool in = r < rows, turned = c < a.rot;  // (the same for all lanes of a row)
    const RowAt row = row_at(in ? r : rows - 1, a.side[first_side].heads, a.positions);
    Turn<E> turn;
    if (turned) {
      const long long t = row.b * a.table_batch_stride + static_cast<long long>(row.n) * (a.rot / 2) + c / 2;
      turn.load(a.sin_t + t, a.cos_t + t);
    }
    fetch(r + STAGES * group, stage);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      const NormSide& s = a.side[first_side + i];
      float2 x[E / 2], sum = both(0.f);
#pragma unroll
      for (int e = 0; e < E / 2; ++e) {
        x[e] = make_float2(to_acc(p[i].e[2 * e]), to_acc(p[i].e[2 * e + 1]));
        sum = fma2(x[e], x[e], sum);
      }
      const float rms = rsqrtf(row_sum<LPR>(sum.x + sum.y) * (1.f / D) + a.eps);
      if constexpr (!BWD) {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) x[e] = mul2(mul2(x[e], both(rms)), w[i][e]);
        if (turned) turn.apply(x, 1.f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) p[i].e[2 * e] = from_acc<T>(x[e].x), p[i].e[2 * e + 1] = from_acc<T>(x[e].y);
        if (in) *reinterpret_cast<uint4*>(static_cast<T*>(s.y) + at(s.sy, row) + c) = p[i].u;
      } else {
        float2 f[E / 2], dot2 = both(0.f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) f[e] = make_float2(to_acc(d[i].e[2 * e]), to_acc(d[i].e[2 * e + 1]));
        if (turned) turn.apply(f, -1.f);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          x[e] = mul2(x[e], both(rms));
          if (in) dw[i][e] = fma2(f[e], x[e], dw[i][e]);
          f[e] = mul2(f[e], w[i][e]);
          dot2 = fma2(f[e], x[e], dot2);
        }
        const float dot = row_sum<LPR>(dot2.x + dot2.y) * (1.f / D);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
          const float2 g = mul2(fma2(x[e], both(-dot), f[e]), both(rms));
          p[i].e[2 * e] = from_acc<T>(g.x), p[i].e[2 * e + 1] = from_acc<T>(g.y);
        }
        if (in) *reinterpret_cast<uint4*>(static_cast<T*>(s.dx) + at(s.sdx, row) + c) = p[i].u;
      }
    }
  }
  fetch_wait<0>();
  if constexpr (BWD) {
    float(*part)[D] = reinterpret_cast<float(*)[D]>(norm_smem);
#pragma unroll
    for (int i = 0; i < SIDES; ++i) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E / 2; ++e) part[threadIdx.x / LPR][c + 2 * e] = dw[i][e].x, part[threadIdx.x / LPR][c + 2 * e + 1] = dw[i][e].y;
      __syncthreads();
      for (int e = threadIdx.x; e < D; e += kNormThreads) {
        float sum = 0.f;
#pragma unroll 8
        for (int k = 0; k < RPC; ++k) sum += part[k][e];
        a.partial[(static_cast<long>(first_side + i) * ctas + cta) * D + e] = sum;
      }
    }
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

// CTAs of one side (of both, where a CTA takes both): one wave, at most one per round of rows
int norm_ctas(unsigned rows, int rows_per_round, int resident) {
  const long want = ((long)rows + rows_per_round - 1) / rows_per_round, most = kSms * resident;
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

template <typename T, int D, bool BWD, int STAGES, int SIDES>
int launch_norm_as(const NormArgs& a, int ctas, cudaStream_t stream) {
  constexpr int RPC = kNormThreads / (D / Piece<T>::kElems);
  const int pieces = STAGES * SIDES * (BWD ? 2 : 1) * kNormThreads * 16, sums = BWD ? RPC * D * 4 : 0;
  auto kern = qk_norm_kernel<T, D, BWD, STAGES, SIDES>;
  const size_t smem = pieces > sums ? pieces : sums;
  if (smem > 48 * 1024) COTT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  COTT_CUDA_TRY(launch_pdl(kern, dim3(SIDES == 2 ? ctas : 2 * ctas), kNormThreads, smem, stream, a));
  return COTT_OK;
}
template <typename T, int D>
int launch_norm(const NormArgs& a, bool bwd, void* dqw, void* dkw, cudaStream_t stream) {
  constexpr int RPC = kNormThreads / (D / Piece<T>::kElems);
  const bool same = a.side[0].rows == a.side[1].rows;
  const unsigned rows = a.side[0].rows > a.side[1].rows ? a.side[0].rows : a.side[1].rows;
  const int ctas = norm_ctas(rows, RPC, same ? (bwd ? kBwdResident : kFwdResident) : (bwd ? kBwdResident : kFwdResident) / 2);
  if (!bwd) {
    // few rows, as of new tokens: nothing to fetch ahead, and q and k on CTAs of their own
    if ((long)kSms * RPC >= rows) return launch_norm_as<T, D, false, 1, 1>(a, norm_ctas(rows, RPC, 1), stream);
    return same ? launch_norm_as<T, D, false, kFwdStages, 2>(a, ctas, stream) : launch_norm_as<T, D, false, kFwdStages, 1>(a, ctas, stream);
  }
  const int st = same ? launch_norm_as<T, D, true, kBwdStages, 2>(a, ctas, stream) : launch_norm_as<T, D, true, kBwdStages, 1>(a, ctas, stream);
  if (st) return st;
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
