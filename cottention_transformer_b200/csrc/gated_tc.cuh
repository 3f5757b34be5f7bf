// Gated causal scan on the 5th-generation tensor cores: 16-bit tensors, head dims 64 and 128 (mathematics: gated_simt.cuh).
//
// Chunks of 128 positions.  Two kernels share the work of a direction:
//   gated_walk_kernel   walks a sequence (or a segment of it) with the fp32 state in registers, S <- A S + K^T diag(e^(G_last-G_s)) V
//                       (backwards: R <- A R + Q^T diag(e^(G_t)) dO), and leaves the state before (after) every chunk in memory as
//                       the 16-bit operand that the other kernel wants.  The weighted operand is split into a 16-bit head and a
//                       16-bit tail, two MMAs, so that a state is exact to about 2^-17: it lasts for the rest of the sequence.
//   gated_chunk_tc      one CTA per chunk and 64 columns of the result, none of which waits for another:
//                           P   = A B^T           128 x 128 x D      scores, decayed, masked and rounded to 16 bits in registers
//                           acc = A M             128 x 64 x D       the state's part, scaled by the row factor in fp32
//                           acc += P C            128 x 64 x 128     P as the A operand from TMEM
//                       with (A, B, C, M) = (q, k, v, S) for out, (dO, v, k, S^T) for dq, (v, dO, q, R^T) for dk, (k, q, dO, R) for dv.
// HBM-bound: the walk reads two tensors and writes half of one, the chunks read three (four and two states backwards).
//
// The decays of a chunk: D_ts = e^(G_t - G_s) of the 32 x 32 blocks on the diagonal are taken element by element; a block below it
// is the product of a row factor e^(G_t - G_b) and a column factor e^(G_b - G_s) with b the last position before the block's
// rows, both at most 1, so that no factor overflows however strong the decay is.  The scores of dq and dk are rounded alike (up to
// the last bit of a factor), which is what lets q.dq - k.dk cancel in the gradient of the gates.
#pragma once

#include "causal_tc.cuh"
#include "gated_simt.cuh"

namespace cott {

constexpr int kGtChunk = 128;
constexpr int kStateTile = 64 * 128;      // bytes of a [64 x 64] 16-bit tile
constexpr int kWalkThreads = 320;
constexpr int kGtThreads = 256;
constexpr float kGateFloorTc = -200.f;    // e^-200 = 0 in fp32; sums of it keep their digits

enum { kWaitWalkTma = 16, kWaitWalkFree = 17, kWaitWalkPrep = 18, kWaitWalkState = 19, kWaitChunkTma = 20, kWaitChunkMma = 21 };

struct GatedTcArgs {
  const void* gate;
  const unsigned char* keep;
  cott_strides sg;
  const float* edge;        // [B*H][value][key]: the state before the walk's first chunk, or null
  float* last;              // [B*H][value][key]: the state after its last one, or null
  unsigned char* states;    // [B*H][nchunks][D/64][D/64] swizzled tiles; c: before chunk c (REV: after it)
  float* seg_state;         // [B*H][D/64][segments][D][64]: sums of the segments, then the states before them
  float* seg_log;           // [B*H][segments]
  int H, N, nchunks, chunks_per_seg, nseg, gate_f32;
};

template <typename T>
__device__ __forceinline__ float gate_tc(const void* gate, const unsigned char* keep, const cott_strides& sg, int gate_f32, int N, long b, int h, int pos) {
  if (pos >= N || (keep && !keep[b * N + pos])) return 0.f;
  const long long o = b * sg.b + h * sg.h + static_cast<long long>(pos) * sg.n;
  const float g = gate_f32 ? static_cast<const float*>(gate)[o] : to_acc(static_cast<const T*>(gate)[o]);
  return g < kGateFloorTc ? kGateFloorTc : g;
}
// Four consecutive gates a lane -> their inclusive sums over the chunk, from its start or (SUFFIX) the sums of what comes after each of
// them; the whole warp takes part.  Additions only: a difference of two sums that both contain a dropped state would leave the
// short sums beside it few digits.
template <bool SUFFIX>
__device__ __forceinline__ void gate_sums(float (&g)[4], int lane) {
  if constexpr (SUFFIX) {
    const float g3 = g[3], g32 = g[2] + g3, g321 = g[1] + g32;
    float run = g[0] + g321;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const float down = __shfl_down_sync(0xffffffffu, run, off);
      if (lane + off < 32) run += down;
    }
    float after = __shfl_down_sync(0xffffffffu, run, 1);
    if (lane == 31) after = 0.f;
    g[3] = after, g[2] = after + g3, g[1] = after + g32, g[0] = after + g321;
  } else {
    g[1] += g[0], g[2] += g[1], g[3] += g[2];
    float run = g[3];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const float up = __shfl_up_sync(0xffffffffu, run, off);
      if (lane >= off) run += up;
    }
    float before = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) before = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] += before;
  }
}

__device__ __forceinline__ void bulk_store(void* dst, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(ptx::smem_u32(smem_src)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(ptx::smem_u32(smem_dst)), "l"(src), "r"(bytes),
               "r"(ptx::smem_u32(bar))
               : "memory");
}

// One 16-byte piece scaled by w, as a sum of SPLIT 16-bit numbers: each takes what the ones before it have left.
template <typename T, int SPLIT>
__device__ __forceinline__ void scale_split(const uint4& u, uint4 (&out)[SPLIT], float w) {
  const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float2 f = Pack2<T>::unpack(x[e]);
    f.x *= w, f.y *= w;
#pragma unroll
    for (int i = 0; i < SPLIT; ++i) {
      const uint32_t p = Pack2<T>::pack(f.x, f.y);
      reinterpret_cast<uint32_t*>(&out[i])[e] = p;
      const float2 h = Pack2<T>::unpack(p);
      f.x -= h.x, f.y -= h.y;
    }
  }
}

// stages of D/64 tiles of Y and SPLIT of Z, as many as fit
template <int D, int SPLIT> constexpr int walk_stage_bytes() { return (D / 64 + SPLIT) * kTileBytes; }
template <int D, int SPLIT> constexpr int walk_stages() { return 192 * 1024 / walk_stage_bytes<D, SPLIT>() > 4 ? 4 : 192 * 1024 / walk_stage_bytes<D, SPLIT>(); }
template <int D, int SPLIT> constexpr size_t walk_smem() { return 1024 + walk_stages<D, SPLIT>() * walk_stage_bytes<D, SPLIT>() + 2 * (D / 64) * kStateTile; }

// grid = (B*H, segments, D/64): one CTA owns 64 value columns of a segment's state.  Y = K, Z = V, or REV: Y = Q, Z = dO and the
// chunks and segments are numbered from the end of the sequence.  EMIT: starts from the segment's state and leaves the state
// before every chunk; else it sums the segment up, from zero.
//   warps 0-3: state (fp32, in registers: a row of it per thread)    warps 4-7: weighted operand    warp 8: TMA    warp 9: MMA
// SPLIT: into how many 16-bit numbers the weighted operand is split.  Two where the states are wanted as 16-bit operands, three
// where the last one is a result: it is then what fp32 products give.
template <typename T, int D, bool REV, bool EMIT, int SPLIT>
__global__ void __launch_bounds__(kWalkThreads, 1)
gated_walk_kernel(const __grid_constant__ CUtensorMap mapY, const __grid_constant__ CUtensorMap mapZ, const GatedTcArgs a) {
  using namespace ptx;
  constexpr int NT = D / 64, NS = walk_stages<D, SPLIT>(), STAGE = walk_stage_bytes<D, SPLIT>();
  constexpr bool BF = Pack2<T>::kBf16;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* sOut = smem + NS * STAGE;  // 2 x NT state tiles on their way out
  __shared__ uint64_t bar_full[NS], bar_free[NS], bar_prep[NS], bar_u_full[2], bar_u_free[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag_s;
  volatile int* abort_flag = &abort_flag_s;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const long bh = blockIdx.x, b = bh / a.H;
  const int h = static_cast<int>(bh % a.H), seg = blockIdx.y, J = blockIdx.z;
  const int chunk0 = seg * a.chunks_per_seg, nchunks = min(a.chunks_per_seg, a.nchunks - chunk0);
  auto chunk_at = [&](int c) { return REV ? a.nchunks - 1 - (chunk0 + c) : chunk0 + c; };
  const bool last_seg = seg + 1 == a.nseg;
  // the last chunk's own part is wanted only where somebody asks for the state after it
  const int updates = !EMIT || (last_seg && a.last) ? nchunks : nchunks - 1;
  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_free[s], 1);
      mbar_init(&bar_prep[s], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar_u_full[i], 1);
      mbar_init(&bar_u_free[i], 4);
    }
    mbar_fence_init();
    abort_flag_s = 0;
    tma_prefetch_desc(&mapY);
    tma_prefetch_desc(&mapZ);
  }
  if (warp == 9) {
    tmem_alloc(&tmem_slot, 128);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_allow_next();  // (after the allocation: a CTA of the next kernel must not take the columns that one of this still waits for)
  pdl_wait_prior();
  const uint32_t tU = tmem_slot;

  if (warp == 8) {
    if (elect_one()) {
      for (int c = 0; c < updates; ++c) {
        const int s = c % NS, y = chunk_at(c) * kGtChunk;
        if (c >= NS && !wait_bar(&bar_free[s], (c / NS - 1) & 1, abort_flag, kWaitWalkFree, c)) break;
        unsigned char* st = smem + s * STAGE;
        mbar_expect_tx(&bar_full[s], (NT + 1) * kTileBytes);
#pragma unroll
        for (int i = 0; i < NT; ++i) tma_load_tile_x(st + i * kTileBytes, &mapY, &bar_full[s], 64 * i, y, h, static_cast<int>(b));
        tma_load_tile_x(st + NT * kTileBytes, &mapZ, &bar_full[s], 64 * J, y, h, static_cast<int>(b));
      }
    }
  } else if (warp == 9) {
    if (elect_one()) {
      constexpr uint32_t kIdesc = make_idesc(D, 64, BF, true, true);
      for (int c = 0; c < updates; ++c) {
        const int s = c % NS, u = c & 1;
        if (!wait_bar2(&bar_prep[s], (c / NS) & 1, c >= 2 ? &bar_u_free[u] : &bar_prep[s], c >= 2 ? ((c >> 1) - 1) & 1 : (c / NS) & 1, abort_flag,
                       kWaitWalkPrep, c))
          break;
        tc_fence_after_sync();
        const uint32_t st = smem_u32(smem + s * STAGE);
        const uint64_t dY = make_smem_desc(st, kTileBytes, 1024);
#pragma unroll
        for (int i = 0; i < SPLIT; ++i) {
          const uint64_t dZ = mdesc(st + (NT + i) * kTileBytes);
#pragma unroll
          for (int k = 0; k < 8; ++k) mma_ss(tU + 64 * u, dY + 128 * k, dZ + 128 * k, kIdesc, i > 0 || k > 0);
        }
        mma_commit(&bar_free[s]);
        mma_commit(&bar_u_full[u]);
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- weighted operand
    const int wq = warp & 3, row = 32 * wq + lane;
    float g[4];
    bool kp = true;
    auto fetch = [&](int c) {
      const int p0 = chunk_at(c) * kGtChunk;
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = gate_tc<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, p0 + 4 * lane + e);
      kp = !a.keep || (p0 + row < a.N && a.keep[b * a.N + p0 + row]);
    };
    if (updates > 0) fetch(0);
    for (int c = 0; c < updates; ++c) {
      const int s = c % NS;
      gate_sums<!REV>(g, lane);  // G_last - G_s, or G_t
      float G = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __shfl_sync(0xffffffffu, g[e], 8 * wq + (lane >> 2));
        if ((lane & 3) == e) G = x;
      }
      const float w = __expf(G);
      const bool take = kp;
      if (c + 1 < updates) fetch(c + 1);
      if (!wait_bar_warp(&bar_full[s], (c / NS) & 1, abort_flag, kWaitWalkTma, c)) break;
      unsigned char *sY = smem + s * STAGE, *sZ = sY + NT * kTileBytes;
      if (take) {
#pragma unroll 2
        for (int j = 0; j < 8; ++j) {
          uint4 z[SPLIT];
          scale_split<T, SPLIT>(*tile_piece(sZ, row, j), z, w);
#pragma unroll
          for (int i = 0; i < SPLIT; ++i) *tile_piece(sZ + i * kTileBytes, row, j) = z[i];
        }
      } else {  // nothing of a masked position gets into a product
        const uint4 zero = make_uint4(0, 0, 0, 0);
        for (int j = 0; j < 8; ++j) {
          for (int i = 0; i < NT + SPLIT; ++i) *tile_piece(sY + i * kTileBytes, row, j) = zero;
        }
      }
      fence_proxy_async_smem();
      warp_arrive(&bar_prep[s], lane);
    }
  } else {
    // ---------------------------------------------------------------- state
    const int wq = warp, i = D == 64 ? 16 * wq + (lane & 15) : 32 * wq + lane;  // row of the state (a key index)
    const bool mine = D == 128 || lane < 16;                                   // (M = 64: lanes 16-31 hold no row)
    const uint32_t lane_base = static_cast<uint32_t>(32 * wq) << 16;
    float S[64];
    const long edge = bh * static_cast<long>(D * D) + 64l * J * D + i;
    float* seg_row = a.nseg > 1 ? a.seg_state + (((bh * NT + J) * a.nseg + seg) * D + i) * 64 : nullptr;
#pragma unroll
    for (int j = 0; j < 64; ++j) S[j] = 0.f;
    if (EMIT && a.nseg > 1) {
#pragma unroll
      for (int j = 0; j < 64; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(seg_row + j);
        S[j] = f.x, S[j + 1] = f.y, S[j + 2] = f.z, S[j + 3] = f.w;
      }
    } else if (EMIT && a.edge) {
#pragma unroll
      for (int j = 0; j < 64; ++j) S[j] = a.edge[edge + static_cast<long>(j) * D];
    }
    float g[4], log_sum = 0.f;
    auto fetch = [&](int c) {
      const int p0 = chunk_at(c) * kGtChunk;
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = gate_tc<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, p0 + 4 * lane + e);
    };
    auto emit = [&](int slot, int n) {  // n: how many were emitted before
      unsigned char* tile = sOut + ((n & 1) * NT + (D == 128 ? wq >> 1 : 0)) * kStateTile;
      const int r = i & 63;
      if (lane == 0) tma_store_wait_read<1>();  // the copy of two emissions ago has left the buffer
      __syncwarp();
      if (mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4 u;
          u.x = Pack2<T>::pack(S[8 * j], S[8 * j + 1]), u.y = Pack2<T>::pack(S[8 * j + 2], S[8 * j + 3]);
          u.z = Pack2<T>::pack(S[8 * j + 4], S[8 * j + 5]), u.w = Pack2<T>::pack(S[8 * j + 6], S[8 * j + 7]);
          *tile_piece(tile, r, j) = u;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        constexpr int ROWS = D == 64 ? 16 : 32;
        const int r0 = (ROWS * wq) & 63;
        unsigned char* dst = a.states + (((bh * a.nchunks + slot) * NT + (D == 128 ? wq >> 1 : 0)) * NT + J) * static_cast<long>(kStateTile);
        bulk_store(dst + r0 * 128, tile + r0 * 128, ROWS * 128);
        tma_store_commit();
      }
    };
    if (updates > 0) fetch(0);
    bool ok = true;
    for (int c = 0; c < nchunks; ++c) {
      if (EMIT) emit(chunk_at(c), c);
      if (c >= updates) break;
      float total = (g[0] + g[1]) + (g[2] + g[3]);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
      const float A = __expf(total);
      log_sum += total;
      if (c + 1 < updates) fetch(c + 1);
      if (!(ok = wait_bar_warp(&bar_u_full[c & 1], (c >> 1) & 1, abort_flag, kWaitWalkState, c))) break;
      tc_fence_after_sync();
      uint32_t r[32];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        tmem_ld_x32(tU + 64 * (c & 1) + 32 * half + lane_base, r);
        tmem_ld_wait();
        if (A == 0.f) {  // a state that is dropped is dropped whatever it holds
#pragma unroll
          for (int j = 0; j < 32; ++j) S[32 * half + j] = __uint_as_float(r[j]);
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) S[32 * half + j] = fmaf(A, S[32 * half + j], __uint_as_float(r[j]));
        }
      }
      tc_fence_before_sync();
      warp_arrive(&bar_u_free[c & 1], lane);
    }
    if (!EMIT) {
      if (ok && mine) {
#pragma unroll
        for (int j = 0; j < 64; j += 4) *reinterpret_cast<float4*>(seg_row + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
      }
      if (J == 0 && tid == 0) a.seg_log[bh * a.nseg + seg] = log_sum;
    } else if (last_seg && ok && a.last && mine) {
#pragma unroll
      for (int j = 0; j < 64; ++j) a.last[edge + static_cast<long>(j) * D] = S[j];
    }
    if (EMIT && lane == 0) tma_store_wait<0>();
  }

  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag) {  // no load may be in flight when the CTA leaves
    for (int c = updates > NS ? updates - NS : 0; c < updates; ++c) mbar_wait(&bar_full[c % NS], (c / NS) & 1, 64);
  }
  __syncthreads();
  if (warp == 9) tmem_dealloc(tU, 128);
}

// The states before the segments, in place of their sums: run <- e^(log) run + sum.  grid = (B*H * D/64, D * 64 / 256).
template <int D>
__global__ void __launch_bounds__(256) gated_seg_kernel(const GatedTcArgs a) {
  constexpr int NT = D / 64;
  const long t = blockIdx.x, bh = t / NT, J = t % NT;
  const int e = blockIdx.y * 256 + threadIdx.x, i = e / 64, j = e % 64;
  float* p = a.seg_state + t * a.nseg * static_cast<long>(D * 64) + e;
  const float* lg = a.seg_log + bh * a.nseg;
  pdl_allow_next();
  pdl_wait_prior();
  float run = a.edge ? a.edge[bh * static_cast<long>(D * D) + (64 * J + j) * D + i] : 0.f;
  for (int s = 0; s < a.nseg; s += 8) {
    float x[8], d[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      x[u] = s + u < a.nseg ? p[static_cast<long>(s + u) * (D * 64)] : 0.f;
      d[u] = s + u < a.nseg ? __expf(lg[s + u]) : 1.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s + u < a.nseg) p[static_cast<long>(s + u) * (D * 64)] = run;
      run = d[u] == 0.f ? x[u] : fmaf(d[u], run, x[u]);
    }
  }
}

struct GatedChunkArgs {
  const void* gate;
  const unsigned char* keep;
  cott_strides sg;
  const unsigned char *S, *R;          // [B*H][nchunks] state tiles: before, after a chunk
  const void *q, *k;                   // for the products with dq and dk
  cott_strides sq, sk;
  float *qdot, *kdot, *bdot;           // [D/64][B*H][nchunks][128]: q.dq; k.dk within the chunk and across its end
  long units;                          // B*H * nchunks
  int H, N, nchunks, gate_f32, with_first, with_last;  // a state before the first chunk, a gradient after the last one
};
struct GatedMaps {
  CUtensorMap q, k, v, o, dq, dk, dv;  // o: out, or dO
};
template <int D> constexpr int chunk_tc_bytes() { return 2 * (D / 64) * kTileBytes + kTileBytes + (D / 64) * kStateTile; }
template <int D> constexpr size_t chunk_tc_smem() { return 1024 + chunk_tc_bytes<D>(); }

// One pass (kGsOut, kGsDq, kGsDk, kGsDv) over one chunk and one 64-column slice J of its result.
//   warp w: TMEM lanes / rows 32 (w % 4) .., columns 64 (w / 4) .. of the scores and 32 (w / 4) .. of the accumulator
template <typename T, int D, int PASS>
__device__ __forceinline__ void gated_chunk_tc(const CUtensorMap& mapA, const CUtensorMap& mapB, const CUtensorMap& mapC, const CUtensorMap& mapO,
                                               const GatedChunkArgs& a, const long unit, const int J) {
  using namespace ptx;
  constexpr int NT = D / 64;
  constexpr bool BF = Pack2<T>::kBf16, LOWER = PASS == kGsOut || PASS == kGsDq, MT = PASS == kGsDq || PASS == kGsDk;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char *sA = smem, *sB = sA + NT * kTileBytes, *sC = sB + NT * kTileBytes, *sM = sC + kTileBytes;
  __shared__ uint64_t bar_full, bar_mma[3];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag_s;
  __shared__ __align__(16) float sG[kGtChunk], sCol[4][kGtChunk], sDot[2][kGtChunk];  // (read four at a time)
  volatile int* abort_flag = &abort_flag_s;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int wq = warp & 3, hf = warp >> 2, row = 32 * wq + lane;
  const long bh = unit / a.nchunks, b = bh / a.H;
  const int chunk = static_cast<int>(unit % a.nchunks), h = static_cast<int>(bh % a.H), c0 = chunk * kGtChunk;
  const bool with_state = LOWER ? chunk > 0 || a.with_first : chunk + 1 < a.nchunks || a.with_last;
  const uint32_t lane_base = static_cast<uint32_t>(32 * wq) << 16;
  if (tid == 0) {
    mbar_init(&bar_full, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&bar_mma[i], 1);
    mbar_fence_init();
    abort_flag_s = 0;
    tma_prefetch_desc(&mapA);
    tma_prefetch_desc(&mapB);
    tma_prefetch_desc(&mapC);
    tma_prefetch_desc(&mapO);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 128);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_allow_next();
  pdl_wait_prior();
  const uint32_t tP = tmem_slot, tAcc = tP + 64;
  if (warp == 0) {
    if (elect_one()) {
      const int bi = static_cast<int>(b);
      mbar_expect_tx(&bar_full, (2 * NT + 1) * kTileBytes + (with_state ? NT * kStateTile : 0));
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        tma_load_tile_x(sA + i * kTileBytes, &mapA, &bar_full, 64 * i, c0, h, bi);
        tma_load_tile_x(sB + i * kTileBytes, &mapB, &bar_full, 64 * i, c0, h, bi);
      }
      tma_load_tile_x(sC, &mapC, &bar_full, 64 * J, c0, h, bi);
      if (with_state) {
        // out, dv: column J of the tiles of S, R; dq, dk: row J
        const unsigned char* m = LOWER ? a.S + unit * (NT * NT * kStateTile) : a.R + unit * (NT * NT * kStateTile);
#pragma unroll
        for (int i = 0; i < NT; ++i) bulk_load(sM + i * kStateTile, m + (MT ? J * NT + i : i * NT + J) * kStateTile, kStateTile, &bar_full);
      }
    }
    __syncwarp();
  } else if (warp == 4) {
    float g[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) g[e] = gate_tc<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, c0 + 4 * lane + e);
    gate_sums<false>(g, lane);
    *reinterpret_cast<float4*>(&sG[4 * lane]) = make_float4(g[0], g[1], g[2], g[3]);
  }
  const bool kp = !a.keep || (c0 + row < a.N && a.keep[b * a.N + c0 + row]);
  __syncthreads();
  // column factors: of the rows of block w, relative to the boundary between them and the columns
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int w = 2 * i + (tid >> 7), s = tid & 127;
    if (LOWER ? s < 32 * w : s >= 32 * w + 32) sCol[w][s] = __expf(LOWER ? sG[32 * w - 1] - sG[s] : sG[s] - sG[32 * w + 31]);
  }
  if (a.keep) {  // nothing of a masked position gets into a product
    wait_bar_warp(&bar_full, 0, abort_flag, kWaitChunkTma, chunk);
    if (!kp) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (int j = 4 * hf; j < 4 * hf + 4; ++j) {
        for (int i = 0; i < 2 * NT; ++i) *tile_piece(sA + i * kTileBytes, row, j) = zero;
        *tile_piece(sC, row, j) = zero;
      }
    }
    fence_proxy_async_smem();
  }
  __syncthreads();
  constexpr uint32_t kIdescP = make_idesc(128, 128, BF, false, false), kIdescM = make_idesc(128, 64, BF, false, !MT),
                     kIdescC = make_idesc(128, 64, BF, false, true);
  constexpr uint64_t kPanel = kTileBytes >> 4, kPanelM = kStateTile >> 4;
  const uint64_t dA = kdesc(smem_u32(sA));
  if (warp == 0) {
    if (elect_one() && wait_bar1(&bar_full, 0, abort_flag, kWaitChunkTma, chunk)) {
      tc_fence_after_sync();
      const uint64_t dB = kdesc(smem_u32(sB));
#pragma unroll
      for (int k = 0; k < 4 * NT; ++k) mma_ss(tP, dA + (k >> 2) * kPanel + 2 * (k & 3), dB + (k >> 2) * kPanel + 2 * (k & 3), kIdescP, k > 0);
      mma_commit(&bar_mma[0]);
    }
    __syncwarp();
  }
  // ---- the scores: this thread has 64 columns of its row
  wait_bar_warp(&bar_mma[0], 0, abort_flag, kWaitChunkMma, chunk);
  tc_fence_after_sync();
  const float Gr = sG[row];
  const float rowf = __expf(LOWER ? (wq > 0 ? Gr - sG[32 * wq - 1] : 0.f) : sG[32 * wq + 31] - Gr);
  uint32_t pk[32];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int blk = 2 * hf + i;
    if (LOWER ? blk > wq : blk < wq) {
#pragma unroll
      for (int j = 0; j < 16; ++j) pk[16 * i + j] = 0u;
    } else {
      uint32_t r[32];
      tmem_ld_x32(tP + lane_base + 32 * blk, r);
      tmem_ld_wait();
      if (blk == wq) {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 Gs = *reinterpret_cast<const float4*>(&sG[32 * blk + j]);
          const float gs[4] = {Gs.x, Gs.y, Gs.z, Gs.w};
          float x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool in = LOWER ? j + e <= lane : j + e >= lane;
            x[e] = in ? __uint_as_float(r[j + e]) * __expf(LOWER ? Gr - gs[e] : gs[e] - Gr) : 0.f;
          }
          pk[16 * i + j / 2] = Pack2<T>::pack(x[0], x[1]);
          pk[16 * i + j / 2 + 1] = Pack2<T>::pack(x[2], x[3]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          const float4 cf = *reinterpret_cast<const float4*>(&sCol[wq][32 * blk + j]);
          pk[16 * i + j / 2] = Pack2<T>::pack(__uint_as_float(r[j]) * (rowf * cf.x), __uint_as_float(r[j + 1]) * (rowf * cf.y));
          pk[16 * i + j / 2 + 1] = Pack2<T>::pack(__uint_as_float(r[j + 2]) * (rowf * cf.z), __uint_as_float(r[j + 3]) * (rowf * cf.w));
        }
      }
    }
  }
  uint4 x[4];
  const bool dot_row = MT && kp && c0 + row < a.N;
  if (dot_row) {
    const cott_strides& sx = PASS == kGsDq ? a.sq : a.sk;
    const T* p = static_cast<const T*>(PASS == kGsDq ? a.q : a.k) + b * sx.b + h * sx.h + static_cast<long long>(c0 + row) * sx.n + 64 * J + 32 * hf;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = reinterpret_cast<const uint4*>(p)[j];
  }
  auto dot_of = [&](const float (&y)[32]) {
    float d = 0.f;
    if (dot_row) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = Pack2<T>::unpack(u[e]);
          d = fmaf(f.x, y[8 * j + 2 * e], fmaf(f.y, y[8 * j + 2 * e + 1], d));
        }
      }
    }
    return d;
  };
  tc_fence_before_sync();
  __syncthreads();  // all scores have been read: their columns become P (the first 64) and the accumulator
  if (with_state && warp == 0) {
    if (elect_one() && !*abort_flag) {
      tc_fence_after_sync();
      const uint64_t dM = MT ? kdesc(smem_u32(sM)) : mdesc(smem_u32(sM));
#pragma unroll
      for (int k = 0; k < 4 * NT; ++k)
        mma_ss(tAcc, dA + (k >> 2) * kPanel + 2 * (k & 3), MT ? dM + (k >> 2) * kPanelM + 2 * (k & 3) : dM + 128 * k, kIdescM, k > 0);
      mma_commit(&bar_mma[1]);
    }
    __syncwarp();
  }
  tc_fence_after_sync();
#pragma unroll
  for (int i = 0; i < 2; ++i) tmem_st_x16(tP + lane_base + 32 * hf + 16 * i, pk + 16 * i);
  tmem_st_wait();
  float acc[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) acc[j] = 0.f;
  if (with_state) {
    wait_bar_warp(&bar_mma[1], 0, abort_flag, kWaitChunkMma, chunk);
    tc_fence_after_sync();
    const float f = __expf(LOWER ? Gr : sG[kGtChunk - 1] - Gr);
    uint32_t r[32];
    tmem_ld_x32(tAcc + lane_base + 32 * hf, r);
    tmem_ld_wait();
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] = f == 0.f ? 0.f : f * __uint_as_float(r[j]);
  }
  tc_fence_before_sync();
  __syncthreads();  // P is written, the state's part has been read
  if (warp == 0) {
    if (elect_one() && !*abort_flag) {
      tc_fence_after_sync();
      const uint64_t dC = mdesc(smem_u32(sC));
#pragma unroll
      for (int k = 0; k < 8; ++k) mma_ts(tAcc, tP + 8 * k, dC + 128 * k, kIdescC, k > 0);
      mma_commit(&bar_mma[2]);
    }
    __syncwarp();
  }
  wait_bar_warp(&bar_mma[2], 0, abort_flag, kWaitChunkMma, chunk);
  tc_fence_after_sync();
  float dot = 0.f, across = 0.f;
  {
    uint32_t r[32];
    tmem_ld_x32(tAcc + lane_base + 32 * hf, r);
    tmem_ld_wait();
    if constexpr (PASS == kGsDk) across = with_state ? dot_of(acc) : 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] += __uint_as_float(r[j]);
  }
  if constexpr (MT) {
    dot = dot_of(acc) - across;
    if (hf) sDot[0][row] = dot, sDot[1][row] = across;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 u;
    u.x = Pack2<T>::pack(acc[8 * j], acc[8 * j + 1]), u.y = Pack2<T>::pack(acc[8 * j + 2], acc[8 * j + 3]);
    u.z = Pack2<T>::pack(acc[8 * j + 4], acc[8 * j + 5]), u.w = Pack2<T>::pack(acc[8 * j + 6], acc[8 * j + 7]);
    *tile_piece(sC, row, 4 * hf + j) = u;  // (the MMAs that read C have completed)
  }
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    if (elect_one()) {
      if (!*abort_flag) {
        tma_store_tile_x(&mapO, sC, 64 * J, c0, h, static_cast<int>(b));
        tma_store_commit();
        tma_store_wait_read<0>();
      } else {
        mbar_wait(&bar_full, 0, 64);  // no load may be in flight when the CTA leaves
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_dealloc(tP, 128);
  }
  if constexpr (MT) {
    if (!hf) {
      const long o = (J * a.units + unit) * kGtChunk + row;
      (PASS == kGsDq ? a.qdot : a.kdot)[o] = dot + sDot[0][row];
      if (PASS == kGsDk) a.bdot[o] = across + sDot[1][row];
    }
  }
}

// FWD: grid = B*H * chunks * D/64.  Backward: three times as many; the CTAs of a chunk are neighbours, so that its tiles are read
// from memory once and from L2 after that.
template <typename T, int D, bool FWD>
__global__ void __launch_bounds__(kGtThreads, D == 64 ? 3 : 2) gated_chunk_tc_kernel(const __grid_constant__ GatedMaps m, const GatedChunkArgs a) {
  constexpr int NT = D / 64;
  const long t = blockIdx.x;
  if constexpr (FWD) {
    gated_chunk_tc<T, D, kGsOut>(m.q, m.k, m.v, m.o, a, t / NT, static_cast<int>(t % NT));
  } else {
    const long unit = t / (3 * NT);
    const int r = static_cast<int>(t % (3 * NT)), J = r % NT;
    if (r / NT == 0)
      gated_chunk_tc<T, D, kGsDq>(m.o, m.v, m.k, m.dq, a, unit, J);
    else if (r / NT == 1)
      gated_chunk_tc<T, D, kGsDk>(m.v, m.o, m.q, m.dk, a, unit, J);
    else
      gated_chunk_tc<T, D, kGsDv>(m.k, m.q, m.o, m.dv, a, unit, J);
  }
}

// dg of a chunk.  With k.dk split into what the chunk itself contributes and what lies across its end,
//     dg_t = sum_{u>=t} (q_u.dq_u - (k_u.dk_u)_within) + sum_{s<t} (k_s.dk_s)_across + A <S, R>
// counts the pairs that cross t and no others, but for those within the chunk, which are the same rounded products in q.dq and in
// k.dk and cancel.  (gated_simt.cuh has <S', R> for the last two terms; with operands of 16 bits that would leave the roundings of all
// pairs across the chunk's end at every position.)  The two states are the tiles that the products used, whose layouts are alike.
// grid = B*H * chunks, block = 128.
template <typename T, int D>
__global__ void __launch_bounds__(kGtChunk) gated_dgate_tc_kernel(const GatedChunkArgs a, void* dgate, const cott_strides sdg) {
  constexpr int NT = D / 64;
  __shared__ float part[16];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long unit = blockIdx.x, bh = unit / a.nchunks, b = bh / a.H;
  const int chunk = static_cast<int>(unit % a.nchunks), h = static_cast<int>(bh % a.H), pos = chunk * kGtChunk + tid;
  pdl_allow_next();
  pdl_wait_prior();
  const float g = gate_tc<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, pos);
  float cross = 0.f;
  if ((chunk > 0 || a.with_first) && (chunk + 1 < a.nchunks || a.with_last)) {
    const uint4 *S = reinterpret_cast<const uint4*>(a.S + unit * (NT * NT * kStateTile)), *R = reinterpret_cast<const uint4*>(a.R + unit * (NT * NT * kStateTile));
#pragma unroll 4
    for (int e = tid; e < NT * NT * kStateTile / 16; e += kGtChunk) {
      const uint4 x = S[e], y = R[e];
      const uint32_t u[4] = {x.x, x.y, x.z, x.w}, w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Pack2<T>::unpack(u[i]), f2 = Pack2<T>::unpack(w[i]);
        cross = fmaf(f.x, f2.x, fmaf(f.y, f2.y, cross));
      }
    }
  }
  float d = 0.f, across = 0.f;
#pragma unroll
  for (int J = 0; J < NT; ++J) {
    const long o = (J * a.units + unit) * kGtChunk + tid;
    d += a.qdot[o] - a.kdot[o];
    across += a.bdot[o];
  }
  float total = g, run = d, up = across;  // of the warp: the gates' sum, d from the row to the warp's end, across up to the row
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    cross += __shfl_xor_sync(0xffffffffu, cross, off);
    total += __shfl_xor_sync(0xffffffffu, total, off);
  }
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const float x = __shfl_down_sync(0xffffffffu, run, off), y = __shfl_up_sync(0xffffffffu, up, off);
    if (lane + off < 32) run += x;
    if (lane >= off) up += y;
  }
  if (lane == 0) part[warp] = cross, part[4 + warp] = run, part[12 + warp] = total;
  if (lane == 31) part[8 + warp] = up;
  __syncthreads();
  float before = __shfl_up_sync(0xffffffffu, up, 1);
  if (lane == 0) before = 0.f;
  const float A = __expf((part[12] + part[13]) + (part[14] + part[15]));
  float x = run + before + (A == 0.f ? 0.f : A * ((part[0] + part[1]) + (part[2] + part[3])));
  for (int w = 0; w < 4; ++w) x += w > warp ? part[4 + w] : w < warp ? part[8 + w] : 0.f;
  if (pos < a.N) {
    if ((a.keep && !a.keep[b * a.N + pos]) || (pos == 0 && !a.with_first) || g <= kGateFloorTc) x = 0.f;
    const long long o = b * sdg.b + h * sdg.h + static_cast<long long>(pos) * sdg.n;
    if (a.gate_f32)
      static_cast<float*>(dgate)[o] = x;
    else
      static_cast<T*>(dgate)[o] = from_acc<T>(x);
  }
}

}  // namespace cott
