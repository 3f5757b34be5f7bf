// Gated causal scan on the 5th-generation tensor cores: 16-bit tensors, head dims 64 and 128 (mathematics: gated_simt.cuh).
//
// Chunks of 128 positions.  Two kernels share the work of a direction:
//   gated_walk_kernel   walks a sequence (or a segment of it) with the fp32 state in registers, S <- A S + K^T diag(e^(G_last-G_s)) V
//                       (backwards: R <- A R + Q^T diag(e^(G_t)) dO), and leaves the state before (after) every chunk in memory as
//                       the 16-bit operand that the other kernel wants.  The weighted operand is split into a 16-bit head and a
//                       16-bit tail, two MMAs, so that the fp32 state is exact to about 2^-17: it lasts for the rest of the sequence.
//   gated_fwd_tc_kernel, gated_bwd64_kernel, gated_bwd128_kernel   take the chunks, none of which waits for another: scores by MMA,
//                       decayed, masked and rounded to 16 bits in registers, back to TMEM as the A operand of the product with the rows; the state's part in
//                       fp32, scaled by the row factor, beside it.
// Traffic, in tensors (a chunk's state is half a tile at head dim 64, a whole one at 128): the walk reads two and writes the states; the
// chunks read three and the states and write one, backwards four and both states and write three.  Walk and forward run at 0.64 - 0.84 of
// the copy rate; the D 128 backward waits for the loads of its one chunk, the D 64 backward for the round trips of its groups (44 % of
// the DRAM peak, no single part bounds it).
//
// Roundings to 16 bits beside those of the results, half a step each: the decayed scores, as the A operand of the product with the
// rows; the copy of a state that multiplies rows, twice in a walk in segments (as the sum of its segment, and with the state before
// that added).  <S, R> in the gradient of the gates is taken from those copies.  Together with the result's own rounding: 0.6 half steps
// from 64 bits in the 2-norm (0.43 by the result's alone), the gates' gradient up to 0.8.
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
constexpr int kWalkThreads = 448;
constexpr float kLog2e = 1.4426950408889634f;
// In units of log 2: a gate down here drops the state (ex2 is zero below the smallest normal number, 2^-126).  In the walk, whose sums are
// additions towards one end of a chunk only, it counts as this; the chunk kernels keep it out of their sums (DropBits).
constexpr float kGateFloorTc = -128.f;

enum { kWaitWalkTma = 16, kWaitWalkFree = 17, kWaitWalkPrep = 18, kWaitWalkState = 19, kWaitChunkTma = 20, kWaitChunkMma = 21 };

struct GatedTcArgs {
  const void* gate;
  const unsigned char* keep;
  cott_strides sg;
  const float* edge;        // [B*H][value][key]: the state before the walk's first chunk, or null
  float* last;              // [B*H][value][key]: the state after its last one, or null
  unsigned char* states;    // [B*H][nchunks][D/64] swizzled [D x 64] panels (key x value); c: before chunk c (REV: after it)
  float* seg_state;         // [B*H][D/64][segments][D][64]: sums of the segments, then the states before them
  float *seg_log, *chunk_log;  // [B*H][segments], [B*H][nchunks]: log2 of the decay over a segment, from its start to a chunk
  int H, N, nchunks, chunks_per_seg, nseg, gate_f32;
};

// One gate, in units of log 2 (all decays are then one ex2 away).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A gate as it lies in memory: fetched a chunk or two ahead, looked at when it is needed.  (A conversion right behind the load would
// wait for it there: the walk at B8 H16 N4096 took 42 us with that, 33 us without.)
struct RawGate {
  uint32_t bits;
  unsigned char take;
};
template <typename T>
__device__ __forceinline__ RawGate gate_raw(const void* gate, const unsigned char* keep, const cott_strides& sg, int gate_f32, int N, long b, int h, int pos) {
  RawGate r = {0u, 0};
  if (pos < N) {
    const long long o = b * sg.b + h * sg.h + static_cast<long long>(pos) * sg.n;
    r.bits = gate_f32 ? static_cast<const uint32_t*>(gate)[o] : static_cast<const unsigned short*>(gate)[o];
    r.take = keep ? keep[b * N + pos] : 1;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float gate_of(const RawGate& r, int gate_f32) {
  if (!r.take) return 0.f;
  const float g = kLog2e * (gate_f32 ? __uint_as_float(r.bits) : Pack2<T>::unpack(r.bits).x);
  return g < kGateFloorTc ? kGateFloorTc : g;
}
template <typename T>
__device__ __forceinline__ float gate_tc(const void* gate, const unsigned char* keep, const cott_strides& sg, int gate_f32, int N, long b, int h, int pos) {
  return gate_of<T>(gate_raw<T>(gate, keep, sg, gate_f32, N, b, h, pos), gate_f32);
}
// Four consecutive gates a lane -> their inclusive sums over the chunk, from its start or (SUFFIX) the sums of what comes after each of
// them; the whole warp takes part.  Additions only: a difference of two sums that both contain a dropped state would leave the
// short sums beside it few digits.
// Returns the sum of all.
template <bool SUFFIX>
__device__ __forceinline__ float gate_sums(float (&g)[4], int lane) {
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
    return __shfl_sync(0xffffffffu, run, 0);
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
    return __shfl_sync(0xffffffffu, run, 31);
  }
}

// Two barriers at once for a whole warp: one round trip instead of two.
__device__ __forceinline__ bool wait_bar2_warp(uint64_t* bar_a, uint32_t parity_a, uint64_t* bar_b, uint32_t parity_b, volatile int* abort_flag, int code,
                                               int chunk) {
  bool ok = false;
  for (uint32_t i = 0; i < ptx::kMaxPolls && !ok; ++i) {
    const bool a = ptx::mbar_try_wait(bar_a, parity_a), b = ptx::mbar_try_wait(bar_b, parity_b);
    ok = __all_sync(0xffffffffu, a && b);
    if (!ok && *abort_flag) return false;
  }
  if (!ok) {
    *abort_flag = 1;
    atomicCAS(&g_cott_status, 0, (code << 16) | (chunk & 0xffff));
  }
  return ok;
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
// bf16 in two numbers stays in packed 16-bit arithmetic, four instructions a pair instead of ten: with w = wh + wl, t = x wl,
// head = x wh + t, and x wh - head is a number of few bits, which t completes.  (float16 has too little range to hold the factor.)
template <typename T> struct Factor {
  float w;
  typename Vec2<T>::type hi, lo;
  __device__ __forceinline__ explicit Factor(float f) : w(f) {
    const float h = Vec2<T>::head(f);
    hi = Vec2<T>::bcast(h), lo = Vec2<T>::bcast(f - h);
  }
};
template <typename T, int SPLIT>
__device__ __forceinline__ void scale_split(const uint4& u, uint4 (&out)[SPLIT], const Factor<T>& f) {
  if constexpr (SPLIT == 2 && Pack2<T>::kBf16) {
    using V = typename Vec2<T>::type;
    const V* x = reinterpret_cast<const V*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const V t = __hmul2(x[e], f.lo), h = __hfma2(x[e], f.hi, t);
      reinterpret_cast<V*>(&out[0])[e] = h;
      reinterpret_cast<V*>(&out[1])[e] = __hadd2(__hfma2(x[e], f.hi, __hneg2(h)), t);
    }
  } else {
    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 y = Pack2<T>::unpack(x[e]);
      y.x *= f.w, y.y *= f.w;
#pragma unroll
      for (int i = 0; i < SPLIT; ++i) {
        const uint32_t p = Pack2<T>::pack(y.x, y.y);
        reinterpret_cast<uint32_t*>(&out[i])[e] = p;
        const float2 h = Pack2<T>::unpack(p);
        y.x -= h.x, y.y -= h.y;
      }
    }
  }
}

// stages of D/64 tiles of Y and SPLIT of Z, as many as fit
template <int D, int SPLIT> constexpr int walk_stage_bytes() { return (D / 64 + SPLIT) * kTileBytes; }
template <int D, int SPLIT> constexpr int walk_stages() { return 192 * 1024 / walk_stage_bytes<D, SPLIT>() > 4 ? 4 : 192 * 1024 / walk_stage_bytes<D, SPLIT>(); }
template <int D, int SPLIT> constexpr size_t walk_smem() { return 1024 + walk_stages<D, SPLIT>() * walk_stage_bytes<D, SPLIT>() + 2 * (D / 64) * kStateTile; }

// grid = (B*H, segments, D/64): one CTA owns 64 value columns of a segment's state.  Y = K, Z = V, or REV: Y = Q, Z = dO and the
// chunks and segments are numbered from the end of the sequence.  A walk in segments starts each of them from nothing and leaves
// their sums, from which gated_seg_kernel makes the states before them, and gated_patch_kernel adds those, decayed, to the states
// inside.  (Walking a second time from the right states instead reads both tensors again: 62 us of 640 for a direction of B1 H16
// N65536.)
//   warps 0-3: state (fp32, in registers: a row of it per thread)    warp 8: TMA    warp 9: MMA
//   warps 4-7, 10-13: weighted operand of the even / odd chunks
// SPLIT: into how many 16-bit numbers the weighted operand is split.  Two where the states are wanted as 16-bit operands, three
// where the last one is a result: it is then what fp32 products give.
template <typename T, int D, bool REV, int SPLIT>
__global__ void __launch_bounds__(kWalkThreads, 1)
gated_walk_kernel(const __grid_constant__ CUtensorMap mapY, const __grid_constant__ CUtensorMap mapZ, const GatedTcArgs a) {
  using namespace ptx;
  constexpr int NT = D / 64, NS = walk_stages<D, SPLIT>(), STAGE = walk_stage_bytes<D, SPLIT>();
  constexpr bool BF = Pack2<T>::kBf16;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char* sOut = smem + NS * STAGE;  // 2 x NT state tiles on their way out
  // (sums of the gates: the operand warps are at most NS + 2 chunks ahead of the state warps)
  constexpr int NSUM = 8;
  static_assert(NS + 2 < NSUM, "a sum is read before its place is taken again");
  __shared__ uint64_t bar_full[NS], bar_free[NS], bar_prep[NS], bar_u_full[2], bar_u_free[2], bar_sum[NSUM];
  __shared__ float sSum[NSUM];
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
  const int updates = !last_seg || a.last ? nchunks : nchunks - 1;
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
    for (int i = 0; i < NSUM; ++i) mbar_init(&bar_sum[i], 1);
    mbar_fence_init();
    abort_flag_s = 0;
    tma_prefetch_desc(&mapY);
    tma_prefetch_desc(&mapZ);
  }
  constexpr uint32_t kUCols = 64 * SPLIT, kCols = SPLIT == 2 ? 256 : 512;  // the parts of the operand side by side: one MMA, summed when read
  if (warp == 9) {
    tmem_alloc(&tmem_slot, kCols);
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
      constexpr uint32_t kIdesc = make_idesc(D, kUCols, BF, true, true);
      for (int c = 0; c < updates; ++c) {
        const int s = c % NS, u = c & 1;
        if (!wait_bar2(&bar_prep[s], (c / NS) & 1, c >= 2 ? &bar_u_free[u] : &bar_prep[s], c >= 2 ? ((c >> 1) - 1) & 1 : (c / NS) & 1, abort_flag,
                       kWaitWalkPrep, c))
          break;
        tc_fence_after_sync();
        const uint32_t st = smem_u32(smem + s * STAGE);
        const uint64_t dY = make_smem_desc(st, kTileBytes, 1024), dZ = make_smem_desc(st + NT * kTileBytes, kTileBytes, 1024);
#pragma unroll
        for (int k = 0; k < 8; ++k) mma_ss(tU + kUCols * u, dY + 128 * k, dZ + 128 * k, kIdesc, k > 0);
        mma_commit(&bar_free[s]);
        mma_commit(&bar_u_full[u]);
      }
    }
  } else if (warp >= 4) {
    // ---------------------------------------------------------------- weighted operand
    const int wq = warp & 3, row = 32 * wq + lane, mine = warp >= 10 ? 1 : 0;
    RawGate raw[4];
    unsigned char kp = 1;
    const long long g0 = b * a.sg.b + h * a.sg.h + 4 * lane * a.sg.n;
    const unsigned char* keep_b = a.keep ? a.keep + b * a.N : nullptr;
    auto fetch = [&](int c) {
      const int p0 = chunk_at(c) * kGtChunk;
      const long long o = g0 + p0 * a.sg.n;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = p0 + 4 * lane + e < a.N;
        raw[e].bits = !in ? 0u : a.gate_f32 ? static_cast<const uint32_t*>(a.gate)[o + e * a.sg.n] : static_cast<const unsigned short*>(a.gate)[o + e * a.sg.n];
        raw[e].take = !in ? 0 : keep_b ? keep_b[p0 + 4 * lane + e] : 1;
      }
      if (keep_b) kp = p0 + row < a.N ? keep_b[p0 + row] : 0;
    };
    if (updates > mine) fetch(mine);
    for (int c = 0; c < updates; ++c) {
      const int s = c % NS;
      if ((c & 1) != mine) {  // every phase of a barrier has to be seen: a parity cannot tell a phase from the next but one
        if (!wait_bar_warp(&bar_full[s], (c / NS) & 1, abort_flag, kWaitWalkTma, c)) break;
        continue;
      }
      float g[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = gate_of<T>(raw[e], a.gate_f32);
      const float total = gate_sums<!REV>(g, lane);  // G_last - G_s, or G_t
      if (wq == 0 && lane == 0) {
        sSum[c % NSUM] = total;
        mbar_arrive(&bar_sum[c % NSUM]);
      }
      float G = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = __shfl_sync(0xffffffffu, g[e], 8 * wq + (lane >> 2));
        if ((lane & 3) == e) G = x;
      }
      const Factor<T> w(ex2(G));
      const bool take = kp != 0;
      if (c + 2 < updates) fetch(c + 2);
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
    if (a.nseg == 1 && a.edge) {
#pragma unroll
      for (int j = 0; j < 64; ++j) S[j] = a.edge[edge + static_cast<long>(j) * D];
    }
    float log_sum = 0.f;
    auto emit = [&](int slot, int n) {  // n: how many were emitted before
      unsigned char* panel = sOut + (n & 1) * NT * kStateTile;
      if (lane == 0) tma_store_wait_read<1>();  // the copy of two emissions ago has left the buffer
      __syncwarp();
      if (mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint4 u;
          u.x = Pack2<T>::pack(S[8 * j], S[8 * j + 1]), u.y = Pack2<T>::pack(S[8 * j + 2], S[8 * j + 3]);
          u.z = Pack2<T>::pack(S[8 * j + 4], S[8 * j + 5]), u.w = Pack2<T>::pack(S[8 * j + 6], S[8 * j + 7]);
          *tile_piece(panel, i, j) = u;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        constexpr int ROWS = D == 64 ? 16 : 32;
        unsigned char* dst = a.states + ((bh * a.nchunks + slot) * NT + J) * static_cast<long>(NT * kStateTile);
        bulk_store(dst + ROWS * wq * 128, panel + ROWS * wq * 128, ROWS * 128);
        tma_store_commit();
      }
    };
    bool ok = true;
    for (int c = 0; c < nchunks; ++c) {
      emit(chunk_at(c), c);
      if (a.nseg > 1 && J == 0 && tid == 0) a.chunk_log[bh * a.nchunks + chunk_at(c)] = log_sum;
      if (c >= updates) break;
      if (!(ok = wait_bar2_warp(&bar_u_full[c & 1], (c >> 1) & 1, &bar_sum[c % NSUM], (c / NSUM) & 1, abort_flag, kWaitWalkState, c))) break;
      const float total = sSum[c % NSUM], A = ex2(total);
      log_sum += total;
      tc_fence_after_sync();
      if (A == 0.f) {  // a state that is dropped is dropped whatever it holds
#pragma unroll
        for (int j = 0; j < 64; ++j) S[j] = 0.f;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // 16 columns at a time: more of them do not fit beside the state
        uint32_t r[SPLIT][16];
#pragma unroll
        for (int i = 0; i < SPLIT; ++i) tmem_ld_x16(tU + kUCols * (c & 1) + 64 * i + 16 * q + lane_base, r[i]);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float x = __uint_as_float(r[SPLIT - 1][j]);  // the smallest parts first
#pragma unroll
          for (int i = SPLIT - 2; i >= 0; --i) x += __uint_as_float(r[i][j]);
          S[16 * q + j] = fmaf(A, S[16 * q + j], x);
        }
      }
      tc_fence_before_sync();
      warp_arrive(&bar_u_free[c & 1], lane);
    }
    if (ok && updates == nchunks) {
      if (a.nseg > 1) {
        if (mine) {
#pragma unroll
          for (int j = 0; j < 64; j += 4) *reinterpret_cast<float4*>(seg_row + j) = make_float4(S[j], S[j + 1], S[j + 2], S[j + 3]);
        }
        if (J == 0 && tid == 0) a.seg_log[bh * a.nseg + seg] = log_sum;
      } else if (mine) {
#pragma unroll
        for (int j = 0; j < 64; ++j) a.last[edge + static_cast<long>(j) * D] = S[j];
      }
    }
    if (lane == 0) tma_store_wait<0>();
  }

  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag) {  // no load may be in flight when the CTA leaves
    for (int c = updates > NS ? updates - NS : 0; c < updates; ++c) mbar_wait(&bar_full[c % NS], (c / NS) & 1, 64);
  }
  __syncthreads();
  if (warp == 9) tmem_dealloc(tU, kCols);
}

// The states before the segments, in place of their sums, and the state after all of them: run <- e^(log) run + sum.
// grid = (B*H * D/64, D * 64 / 256).  (The last sum is there only where the last state is wanted.)
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
      d[u] = s + u < a.nseg ? ex2(lg[s + u]) : 1.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (s + u < a.nseg) p[static_cast<long>(s + u) * (D * 64)] = run;
      if (s + u < a.nseg) run = d[u] == 0.f ? x[u] : fmaf(d[u], run, x[u]);
    }
  }
  if (a.last) a.last[bh * static_cast<long>(D * D) + (64 * J + j) * D + i] = run;
}

// The states inside a segment += the decayed state before it.  A CTA per chunk and panel; most of those of a head that forgets within
// a segment have nothing to do.  The sum is fp32; what it starts from is the operand that the walk has rounded, so that a state that the
// segment's start reaches carries two roundings.  (One would take the walk's fp32 states through memory, twice the bytes each way.)
// grid = B*H * nchunks * D/64, block = 128.
template <typename T, int D, bool REV>
__global__ void __launch_bounds__(128) gated_patch_kernel(const GatedTcArgs a) {
  constexpr int NT = D / 64;
  const long unit = blockIdx.x / NT, bh = unit / a.nchunks;
  const int J = static_cast<int>(blockIdx.x % NT), chunk = static_cast<int>(unit % a.nchunks), seg = (REV ? a.nchunks - 1 - chunk : chunk) / a.chunks_per_seg;
  pdl_allow_next();
  pdl_wait_prior();
  if (seg == 0 && !a.edge) return;
  const float f = ex2(a.chunk_log[unit]);
  if (f == 0.f) return;
  unsigned char* panel = a.states + (unit * NT + J) * static_cast<long>(NT * kStateTile);
  const float* start = a.seg_state + ((bh * NT + J) * a.nseg + seg) * static_cast<long>(D * 64);
#pragma unroll
  for (int e = threadIdx.x; e < D * 8; e += 128) {  // piece e % 8 of row e / 8
    uint4* p = tile_piece(panel, e >> 3, e & 7);
    const float4 x = *reinterpret_cast<const float4*>(start + 8 * e), y = *reinterpret_cast<const float4*>(start + 8 * e + 4);
    uint4 u = *p;
    const float s[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    uint32_t* w = reinterpret_cast<uint32_t*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 l = Pack2<T>::unpack(w[i]);
      w[i] = Pack2<T>::pack(fmaf(f, s[2 * i], l.x), fmaf(f, s[2 * i + 1], l.y));
    }
    *p = u;
  }
}

// The positions of a chunk whose gates drop the state, a bit each.  The chunk kernels take decays as differences of sums of gates: a
// dropped state in such a sum would cost every later difference its digits, so the sums pass over these gates, and a decay across one
// of them is zero by its bit.  Relative errors of the decays between neighbours of a document, worst and rms over 2000 chunks of gates
// between 0 and -0.5 (these sums emulated on a CPU; float16 rounds by up to 4.9e-4): a quarter of the gates -inf, as a -288 in the
// sums, 1.7e-3 and 1.7e-4, as a bit 6.6e-6 and 8e-7; every second gate -30, which is no drop, 4.2e-4 and 5e-5.
struct __align__(16) DropBits {
  uint32_t w[4];
  // whether one of the positions first .. last does
  __device__ __forceinline__ bool in(int first, int last) const {
    uint32_t found = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = first - 32 * i, b = last - 32 * i;
      const uint32_t from = a <= 0 ? 0xffffffffu : a > 31 ? 0u : 0xffffffffu << a, to = b >= 31 ? 0xffffffffu : b < 0 ? 0u : (2u << b) - 1u;
      found |= w[i] & from & to;
    }
    return found;
  }
};
// Of the 32 columns of a row's own block those that the row sees: LOWER: from the last drop up to the row, or the block's start, to the row;
// else from the row to the position before the next drop, or the block's end.
template <bool LOWER>
__device__ __forceinline__ uint32_t seen_bits(uint32_t drops, int lane) {
  if constexpr (LOWER) {
    const uint32_t upto = (2u << lane) - 1u, d = drops & upto;
    return d ? upto & (0xffffffffu << (31 - __clz(d))) : upto;
  } else {
    const uint32_t after = drops & ~((2u << lane) - 1u);
    return (after ? (after & (0u - after)) - 1u : 0xffffffffu) & (0xffffffffu << lane);
  }
}

struct GatedChunkArgs {
  const void* gate;
  const unsigned char* keep;
  cott_strides sg, sdg;
  const unsigned char *S, *R;  // [B*H][nchunks] states: before, after a chunk
  void* dgate;
  long units;                  // B*H * nchunks
  int H, N, nchunks, gate_f32, with_first, with_last;  // a state before the first chunk, a gradient after the last one
};

// A chunk's gates, four consecutive ones a lane: those that drop the state become 0 and a bit of `drops`, which is set only where there
// are any.  Returns whether there are, for the whole warp.
// (Functions of their own, this and drop_tables: what few chunks need is kept out of the loops.  Inline they cost the backward at head
// dim 64 another 2 us of 172 at B8 H16 N4096.)
__device__ __noinline__ float4 drops_taken(float4 x, DropBits* drops, int lane) {
  float g[4] = {x.x, x.y, x.z, x.w};
  uint32_t bits = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (g[e] <= kGateFloorTc) g[e] = 0.f, bits |= 1u << (4 * (lane & 7) + e);
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, off);
  if ((lane & 7) == 0) drops->w[lane >> 3] = bits;
  return make_float4(g[0], g[1], g[2], g[3]);
}
__device__ __forceinline__ bool take_drops(float (&g)[4], DropBits& drops, int lane) {
  const bool any = __any_sync(0xffffffffu, fminf(fminf(g[0], g[1]), fminf(g[2], g[3])) <= kGateFloorTc);
  if (any) {
    const float4 x = drops_taken(make_float4(g[0], g[1], g[2], g[3]), &drops, lane);
    g[0] = x.x, g[1] = x.y, g[2] = x.z, g[3] = x.w;
  }
  return any;
}
// What the CTAs of both chunk kernels begin with: sums of the gates, and the column factors of the decays of the blocks off the
// diagonal (LOWER: below it).
template <typename T>
__device__ __forceinline__ void chunk_gates(const GatedChunkArgs& a, float* sG, DropBits* drops, int* dropping, long b, int h, int c0, int lane) {
  float g[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) g[e] = gate_tc<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, c0 + 4 * lane + e);
  const bool any = take_drops(g, *drops, lane);
  if (lane == 0) *dropping = any;
  gate_sums<false>(g, lane);
  *reinterpret_cast<float4*>(&sG[4 * lane]) = make_float4(g[0], g[1], g[2], g[3]);
}
template <bool LOWER>
__device__ __forceinline__ void col_factor(float (*sCol)[kGtChunk], const float* sG, const DropBits& drops, bool dropping, int w, int s) {
  if (LOWER ? s >= 32 * w : s < 32 * w + 32) return;
  float f = ex2(LOWER ? sG[32 * w - 1] - sG[s] : sG[s] - sG[32 * w + 31]);
  if (dropping && (LOWER ? drops.in(s + 1, 32 * w - 1) : drops.in(32 * w + 32, s))) f = 0.f;
  sCol[w][s] = f;
}
// What drops change for a row (where there are any; few chunks have them): the columns of its own block that it sees, its factor for the
// blocks off the diagonal.
template <bool LOWER>
__device__ __forceinline__ void row_drops(const DropBits& drops, int wq, int lane, uint32_t& seen, float& block) {
  const uint32_t here = (2u << lane) - 1u, d = drops.w[wq];
  seen = seen_bits<LOWER>(d, lane);
  if (d & (LOWER ? here : ~here)) block = 0.f;
}
__device__ __forceinline__ float2 pair(const uint32_t* r) { return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1])); }
// acc += 16 values times two packed pieces of a row
template <typename T>
__device__ __forceinline__ void dot16_2(float2& acc, const uint32_t* x, const uint4& u, const uint4& w) {
  const uint32_t p[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) acc = fma2(Pack2<T>::unpack(p[j]), pair(x + 2 * j), acc);
}
// 32 columns (block `blk`) of the scores of a row of block wq, decayed, masked (`seen`: in the row's own block) and packed
template <typename T, bool LOWER>
__device__ __forceinline__ void decay_block(uint32_t (&pk)[16], uint32_t taddr_lane, int blk, int wq, uint32_t seen, float Gr, float rowf, const float* sG,
                                            const float* col) {
  if (LOWER ? blk > wq : blk < wq) {
#pragma unroll
    for (int j = 0; j < 16; ++j) pk[j] = 0u;
    return;
  }
  uint32_t r[32];
  ptx::tmem_ld_x32(taddr_lane + 32 * blk, r);
  ptx::tmem_ld_wait();
  if (blk == wq) {
    const float sign = LOWER ? 1.f : -1.f;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 Gs = *reinterpret_cast<const float4*>(&sG[32 * blk + j]);
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        float2 x = fma2(make_float2(-sign, -sign), e ? make_float2(Gs.z, Gs.w) : make_float2(Gs.x, Gs.y), make_float2(sign * Gr, sign * Gr));
        x = mul2(make_float2(ex2(x.x), ex2(x.y)), pair(r + j + e));
        x.x = seen & (1u << (j + e)) ? x.x : 0.f;
        x.y = seen & (2u << (j + e)) ? x.y : 0.f;
        pk[(j + e) / 2] = Pack2<T>::pack(x.x, x.y);
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 cf = *reinterpret_cast<const float4*>(&col[32 * blk + j]);
      const float2 x = mul2(pair(r + j), mul2(make_float2(cf.x, cf.y), make_float2(rowf, rowf)));
      const float2 y = mul2(pair(r + j + 2), mul2(make_float2(cf.z, cf.w), make_float2(rowf, rowf)));
      pk[j / 2] = Pack2<T>::pack(x.x, x.y);
      pk[j / 2 + 1] = Pack2<T>::pack(y.x, y.y);
    }
  }
}
// A state that is dropped is dropped whatever it holds: its products are left out, not multiplied by zero.
template <int N>
__device__ __forceinline__ void drop_if(bool dropped, uint32_t (&x)[N]) {
  if (dropped) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = 0u;
  }
}
// 32 columns of an accumulator, scaled by f (0: whatever they hold)
__device__ __forceinline__ void acc_scaled(float (&acc)[32], uint32_t taddr_lane, float f) {
  uint32_t r[32];
  ptx::tmem_ld_x32(taddr_lane, r);
  ptx::tmem_ld_wait();
  drop_if(f == 0.f, r);
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 x = mul2(pair(r + j), make_float2(f, f));
    acc[j] = x.x, acc[j + 1] = x.y;
  }
}
__device__ __forceinline__ void acc_add(float (&acc)[32], uint32_t taddr_lane) {
  uint32_t r[32];
  ptx::tmem_ld_x32(taddr_lane, r);
  ptx::tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    const float2 x = fma2(pair(r + j), make_float2(1.f, 1.f), make_float2(acc[j], acc[j + 1]));
    acc[j] = x.x, acc[j + 1] = x.y;
  }
}
// 32 columns of a row -> pieces j0 .. j0 + 3 of a tile's row
template <typename T>
__device__ __forceinline__ void stage_row(unsigned char* tile, int row, int j0, const float (&acc)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 u;
    u.x = Pack2<T>::pack(acc[8 * j], acc[8 * j + 1]), u.y = Pack2<T>::pack(acc[8 * j + 2], acc[8 * j + 3]);
    u.z = Pack2<T>::pack(acc[8 * j + 4], acc[8 * j + 5]), u.w = Pack2<T>::pack(acc[8 * j + 6], acc[8 * j + 7]);
    *tile_piece(tile, row, j0 + j) = u;
  }
}
template <typename T>
__device__ __forceinline__ float row_dot32(unsigned char* tile, int row, int j0, const float (&acc)[32]) {
  float2 d = make_float2(0.f, 0.f);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 p = *tile_piece(tile, row, j0 + j);
    const uint32_t u[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) d = fma2(Pack2<T>::unpack(u[e]), make_float2(acc[8 * j + 2 * e], acc[8 * j + 2 * e + 1]), d);
  }
  return d.x + d.y;
}

constexpr int kFwdThreads = 256;
template <int D> constexpr size_t fwd_tc_smem() { return 1024 + 2 * (D / 64) * kTileBytes + kTileBytes + (D / 64) * kStateTile; }

// Forward, one chunk and 64 columns J of the result; grid = B*H * chunks * D/64 (the CTAs of a chunk are neighbours: its q and k are
// read from memory once).  Everything in a CTA is one chain; three CTAs per SM cover each other.
//   warp w: TMEM lanes / rows 32 (w % 4) .., columns 64 (w / 4) .. of the scores and 32 (w / 4) .. of the accumulator
template <typename T, int D>
__global__ void __launch_bounds__(kFwdThreads, D == 64 ? 3 : 2)
gated_fwd_tc_kernel(const __grid_constant__ CUtensorMap mapQ, const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                    const __grid_constant__ CUtensorMap mapO, const GatedChunkArgs a) {
  using namespace ptx;
  constexpr int NT = D / 64;
  constexpr bool BF = Pack2<T>::kBf16;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char *sQ = smem, *sK = sQ + NT * kTileBytes, *sV = sK + NT * kTileBytes, *sS = sV + kTileBytes;
  __shared__ uint64_t bar_full, bar_mma[3];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag_s;
  __shared__ __align__(16) float sG[kGtChunk], sCol[4][kGtChunk];  // (read four at a time)
  __shared__ DropBits drops;  // (where `dropping`)
  __shared__ int dropping;
  volatile int* abort_flag = &abort_flag_s;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int wq = warp & 3, hf = warp >> 2, row = 32 * wq + lane, J = static_cast<int>(blockIdx.x % NT);
  const long unit = blockIdx.x / NT, bh = unit / a.nchunks, b = bh / a.H;
  const int chunk = static_cast<int>(unit % a.nchunks), h = static_cast<int>(bh % a.H), c0 = chunk * kGtChunk;
  const bool with_state = chunk > 0 || a.with_first;
  const uint32_t lane_base = static_cast<uint32_t>(32 * wq) << 16;
  if (tid == 0) {
    mbar_init(&bar_full, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&bar_mma[i], 1);
    mbar_fence_init();
    abort_flag_s = 0;
    tma_prefetch_desc(&mapQ);
    tma_prefetch_desc(&mapK);
    tma_prefetch_desc(&mapV);
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
        tma_load_tile_x(sQ + i * kTileBytes, &mapQ, &bar_full, 64 * i, c0, h, bi);
        tma_load_tile_x(sK + i * kTileBytes, &mapK, &bar_full, 64 * i, c0, h, bi);
      }
      tma_load_tile_x(sV, &mapV, &bar_full, 64 * J, c0, h, bi);
      if (with_state) bulk_load(sS, a.S + (unit * NT + J) * (NT * kStateTile), NT * kStateTile, &bar_full);
    }
    __syncwarp();
  } else if (warp == 4) {
    chunk_gates<T>(a, sG, &drops, &dropping, b, h, c0, lane);
  }
  const bool kp = !a.keep || (c0 + row < a.N && a.keep[b * a.N + c0 + row]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) col_factor<true>(sCol, sG, drops, dropping, 2 * i + (tid >> 7), tid & 127);
  if (a.keep) {  // nothing of a masked position gets into a product
    wait_bar_warp(&bar_full, 0, abort_flag, kWaitChunkTma, chunk);
    if (!kp) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (int j = 4 * hf; j < 4 * hf + 4; ++j)
        for (int i = 0; i < 2 * NT + 1; ++i) *tile_piece(sQ + i * kTileBytes, row, j) = zero;
    }
    fence_proxy_async_smem();
  }
  __syncthreads();
  constexpr uint32_t kIdescP = make_idesc(128, 128, BF, false, false), kIdescAcc = make_idesc(128, 64, BF, false, true);
  constexpr uint64_t kPanel = kTileBytes >> 4;
  const uint64_t dQ = kdesc(smem_u32(sQ));
  if (warp == 0) {
    if (elect_one() && wait_bar1(&bar_full, 0, abort_flag, kWaitChunkTma, chunk)) {
      tc_fence_after_sync();
      const uint64_t dK = kdesc(smem_u32(sK));
#pragma unroll
      for (int k = 0; k < 4 * NT; ++k) mma_ss(tP, dQ + (k >> 2) * kPanel + 2 * (k & 3), dK + (k >> 2) * kPanel + 2 * (k & 3), kIdescP, k > 0);
      mma_commit(&bar_mma[0]);
    }
    __syncwarp();
  }
  wait_bar_warp(&bar_mma[0], 0, abort_flag, kWaitChunkMma, chunk);
  tc_fence_after_sync();
  const float Gr = sG[row];
  float rowf = ex2(wq > 0 ? Gr - sG[32 * wq - 1] : 0.f);
  uint32_t seen = (2u << lane) - 1u;
  bool with_row = kp;  // (a masked row is zero, whatever the state holds)
  if (dropping) {
    row_drops<true>(drops, wq, lane, seen, rowf);
    with_row = kp && !drops.in(0, row);
  }
  uint32_t pk[2][16];
#pragma unroll
  for (int i = 0; i < 2; ++i) decay_block<T, true>(pk[i], tP + lane_base, 2 * hf + i, wq, seen, Gr, rowf, sG, sCol[wq]);
  tc_fence_before_sync();
  __syncthreads();  // all scores have been read: their columns become P (the first 64) and the accumulator
  if (with_state && warp == 0) {
    if (elect_one() && !*abort_flag) {
      tc_fence_after_sync();
      const uint64_t dS = mdesc(smem_u32(sS));
#pragma unroll
      for (int k = 0; k < 4 * NT; ++k) mma_ss(tAcc, dQ + (k >> 2) * kPanel + 2 * (k & 3), dS + 128 * k, kIdescAcc, k > 0);
      mma_commit(&bar_mma[1]);
    }
    __syncwarp();
  }
  tc_fence_after_sync();
#pragma unroll
  for (int i = 0; i < 2; ++i) tmem_st_x16(tP + lane_base + 32 * hf + 16 * i, pk[i]);
  tmem_st_wait();
  float acc[32];
  if (with_state) {
    wait_bar_warp(&bar_mma[1], 0, abort_flag, kWaitChunkMma, chunk);
    tc_fence_after_sync();
    acc_scaled(acc, tAcc + lane_base + 32 * hf, with_row ? ex2(Gr) : 0.f);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] = 0.f;
  }
  tc_fence_before_sync();
  __syncthreads();  // P is written, the state's part has been read
  if (warp == 0) {
    if (elect_one() && !*abort_flag) {
      tc_fence_after_sync();
      const uint64_t dV = mdesc(smem_u32(sV));
#pragma unroll
      for (int k = 0; k < 8; ++k) mma_ts(tAcc, tP + 8 * k, dV + 128 * k, kIdescAcc, k > 0);
      mma_commit(&bar_mma[2]);
    }
    __syncwarp();
  }
  wait_bar_warp(&bar_mma[2], 0, abort_flag, kWaitChunkMma, chunk);
  tc_fence_after_sync();
  acc_add(acc, tAcc + lane_base + 32 * hf);
  stage_row<T>(sV, row, 4 * hf, acc);  // (the MMAs that read V have completed)
  fence_proxy_async_smem();
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    if (elect_one()) {
      if (!*abort_flag) {
        tma_store_tile_x(&mapO, sV, 64 * J, c0, h, static_cast<int>(b));
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
}

struct GatedMaps {
  CUtensorMap q, k, v, o, dq, dk, dv;
};
constexpr int kBwd128Threads = 512;
constexpr int kBwdAhead = 148;  // units: a CTA on each SM
constexpr size_t kBwd128Smem = 1024 + 4 * 2 * kTileBytes + 2 * 4 * kStateTile;

// Backward of one chunk at head dim 128: dq, dk, dv and dg from q, k, v, dO and the two states, each read once; grid = B*H * chunks.
//     E  = dO V^T  (t, s)    dq = e^(G_t) dO S^T        + (E D) K
//     E' = V dO^T  (s, t)    dk = e^(G_last-G_s) V R^T  + (E' D) Q
//     P' = K Q^T   (s, t)    dv = e^(G_last-G_s) K R    + (P' D) dO
// E and its transpose are both computed: an A operand from TMEM cannot be transposed, and two products of 128 x 128 x D cost less
// than a 32 KB tile through shared memory.  Two buffers X and Y in TMEM of 128 columns of scores and 128 of accumulator; every pass is
// scores and state's part (MMA) -> decayed 16-bit scores in place, the state's part read and scaled in fp32 -> scores times rows:
//     E X, E' Y and their states | decay X | decay Y, rows X | rows Y | dq out, P' X and its state | decay X, dk out | rows X | dv out
// Results are staged over the tile that has no reader left: dq over V, dk over Q, dv over K.  The tiles and states fill the SM's
// shared memory, so that a CTA's loads overlap nothing of the CTA before it: the scores begin when dO and V are there, the states and
// the other tiles arrive meanwhile (172 -> 163 us at B1 H16 N16384 bf16, whose traffic alone takes 93), and the CTA after it finds
// its tiles in L2 (3 us).
// With k.dk split into what the chunk itself contributes and what lies across its end,
//     dg_t = sum_{u>=t} (q_u.dq_u - (k_u.dk_u)_within) + sum_{s<t} (k_s.dk_s)_across + A <S, R>
// counts the pairs that cross t and no others, but for those within the chunk, which are the same rounded products in q.dq and in
// k.dk and cancel.  (gated_simt.cuh has <S', R> for the last two terms; with operands of 16 bits that would leave the roundings of all
// pairs across the chunk's end at every position.)
//   warp w: rows 32 (w % 4) .., columns 32 (w / 4) .. of the scores and of the accumulator
template <typename T>
__global__ void __launch_bounds__(kBwd128Threads, 1) gated_bwd128_kernel(const __grid_constant__ GatedMaps m, const GatedChunkArgs a) {
  using namespace ptx;
  constexpr int D = 128, NT = 2, NG = 4;  // 64-column panels, 32-column groups
  constexpr uint32_t kCols = 512, kBuf = 256, kAccAt = 128;
  constexpr bool BF = Pack2<T>::kBf16;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  unsigned char *sQ = smem, *sK = sQ + NT * kTileBytes, *sV = sK + NT * kTileBytes, *sO = sV + NT * kTileBytes, *sS = sO + NT * kTileBytes,
                *sR = sS + NT * NT * kStateTile;
  __shared__ uint64_t bar_full[3], bar_score[3], bar_state[3], bar_rows[3];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag_s;
  __shared__ __align__(16) float sG[kGtChunk], sLow[4][kGtChunk], sUp[4][kGtChunk];
  __shared__ DropBits drops;  // (where `dropping`)
  __shared__ int dropping;
  __shared__ float sQd[NG][kGtChunk], sKd[NG][kGtChunk], sBd[NG][kGtChunk], sCross[4 * NG], sPart[8];
  volatile int* abort_flag = &abort_flag_s;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int wq = warp & 3, cg = warp >> 2, row = 32 * wq + lane;
  const long unit = blockIdx.x, bh = unit / a.nchunks, b = bh / a.H;
  const int chunk = static_cast<int>(unit % a.nchunks), h = static_cast<int>(bh % a.H), c0 = chunk * kGtChunk, bi = static_cast<int>(b);
  const bool with_S = chunk > 0 || a.with_first, with_R = chunk + 1 < a.nchunks || a.with_last;
  const uint32_t lane_base = static_cast<uint32_t>(32 * wq) << 16;
  if (tid == 0) {
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bar_full[i], 1);  // dO and V; the states; K and Q
      mbar_init(&bar_score[i], 1);
      mbar_init(&bar_state[i], 1);
      mbar_init(&bar_rows[i], 1);
    }
    mbar_fence_init();
    abort_flag_s = 0;
    tma_prefetch_desc(&m.q);
    tma_prefetch_desc(&m.k);
    tma_prefetch_desc(&m.v);
    tma_prefetch_desc(&m.o);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_allow_next();
  pdl_wait_prior();
  const uint32_t tX = tmem_slot, tY = tX + kBuf;
  if (warp == 0) {
    if (elect_one()) {
      for (int i = 0; i < 3; i += 2) mbar_expect_tx(&bar_full[i], 2 * NT * kTileBytes);
      mbar_expect_tx(&bar_full[1], ((with_S ? 1 : 0) + (with_R ? 1 : 0)) * NT * NT * kStateTile);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        tma_load_tile_x(sO + i * kTileBytes, &m.o, &bar_full[0], 64 * i, c0, h, bi);
        tma_load_tile_x(sV + i * kTileBytes, &m.v, &bar_full[0], 64 * i, c0, h, bi);
      }
      if (with_S) bulk_load(sS, a.S + unit * (NT * NT * kStateTile), NT * NT * kStateTile, &bar_full[1]);
      if (with_R) bulk_load(sR, a.R + unit * (NT * NT * kStateTile), NT * NT * kStateTile, &bar_full[1]);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        tma_load_tile_x(sK + i * kTileBytes, &m.k, &bar_full[2], 64 * i, c0, h, bi);
        tma_load_tile_x(sQ + i * kTileBytes, &m.q, &bar_full[2], 64 * i, c0, h, bi);
      }
      const long next = unit + kBwdAhead;  // the tiles of the CTA that takes this one's place, into L2
      if (next < a.units) {
        const long nbh = next / a.nchunks;
        const int ny = static_cast<int>(next % a.nchunks) * kGtChunk, nh = static_cast<int>(nbh % a.H), nb = static_cast<int>(nbh / a.H);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          tma_prefetch_tile_x(&m.o, 64 * i, ny, nh, nb);
          tma_prefetch_tile_x(&m.v, 64 * i, ny, nh, nb);
          tma_prefetch_tile_x(&m.k, 64 * i, ny, nh, nb);
          tma_prefetch_tile_x(&m.q, 64 * i, ny, nh, nb);
        }
      }
    }
    __syncwarp();
  } else if (warp == 4) {
    chunk_gates<T>(a, sG, &drops, &dropping, b, h, c0, lane);
  }
  const bool kp = !a.keep || (c0 + row < a.N && a.keep[b * a.N + c0 + row]);
  __syncthreads();
  for (int e = tid; e < 4 * kGtChunk; e += kBwd128Threads) {
    col_factor<true>(sLow, sG, drops, dropping, e >> 7, e & 127);
    col_factor<false>(sUp, sG, drops, dropping, e >> 7, e & 127);
  }
  // (every thread reads rows of the tiles later on, so every thread waits for them; nothing of a masked position gets into a product)
  auto arrived = [&](int which, unsigned char* tiles) {
    wait_bar_warp(&bar_full[which], 0, abort_flag, kWaitChunkTma, chunk);
    if (a.keep) {
      if (!kp) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        for (int j = 0; j < 8; ++j) *tile_piece(tiles + cg * kTileBytes, row, j) = zero;
      }
      fence_proxy_async_smem();
    }
  };
  static_assert(2 * NT == NG);  // (a panel each)
  arrived(0, sV);
  __syncthreads();
  constexpr uint32_t kIdescP = make_idesc(128, 128, BF, false, false), kIdescK = make_idesc(128, D, BF, false, false), kIdescM = make_idesc(128, D, BF, false, true);
  constexpr uint64_t kPanel = kTileBytes >> 4, kStatePanel = (NT * kStateTile) >> 4;
  const uint64_t dQ = kdesc(smem_u32(sQ)), dK = kdesc(smem_u32(sK)), dV = kdesc(smem_u32(sV)), dO = kdesc(smem_u32(sO));
  auto scores = [&](uint32_t t, uint64_t dA, uint64_t dB, uint64_t* bar) {  // t = A B^T
#pragma unroll
    for (int k = 0; k < 4 * NT; ++k) mma_ss(t, dA + (k >> 2) * kPanel + 2 * (k & 3), dB + (k >> 2) * kPanel + 2 * (k & 3), kIdescP, k > 0);
    mma_commit(bar);
  };
  auto times_rows = [&](uint32_t t, unsigned char* tile, uint64_t* bar) {  // acc = (scores in TMEM) rows
    const uint64_t d = make_smem_desc(smem_u32(tile), kTileBytes, 1024);
#pragma unroll
    for (int k = 0; k < 8; ++k) mma_ts(t + kAccAt, t + 8 * k, d + 128 * k, kIdescM, k > 0);
    mma_commit(bar);
  };
  auto times_state_t = [&](uint32_t t, uint64_t dA, unsigned char* state, uint64_t* bar) {  // acc = A M^T
    const uint64_t d = kdesc(smem_u32(state));
#pragma unroll
    for (int k = 0; k < 4 * NT; ++k) mma_ss(t + kAccAt, dA + (k >> 2) * kPanel + 2 * (k & 3), d + (k >> 2) * kStatePanel + 2 * (k & 3), kIdescK, k > 0);
    mma_commit(bar);
  };
  auto times_state = [&](uint32_t t, uint64_t dA, unsigned char* state, uint64_t* bar) {  // acc = A M
    const uint64_t d = make_smem_desc(smem_u32(state), NT * kStateTile, 1024);
#pragma unroll
    for (int k = 0; k < 4 * NT; ++k) mma_ss(t + kAccAt, dA + (k >> 2) * kPanel + 2 * (k & 3), d + 128 * k, kIdescM, k > 0);
    mma_commit(bar);
  };
  // `body` by one thread (chosen by elect.sync where it issues: see elect_one), if nothing has given up; after the barrier that
  // everybody's TMEM accesses came before
  auto issue = [&](bool cond, auto&& body) {
    if (warp == 0) {
      if (elect_one() && cond && !*abort_flag) {
        tc_fence_after_sync();
        body();
      }
      __syncwarp();
    }
  };
  auto sync = [&]() {
    tc_fence_before_sync();
    __syncthreads();
  };
  auto wait = [&](uint64_t* bar) {
    wait_bar_warp(bar, 0, abort_flag, kWaitChunkMma, chunk);
    tc_fence_after_sync();
  };
  const uint32_t my_scores = lane_base, my_acc = lane_base + kAccAt + 32 * cg;
  auto put_scores = [&](uint32_t t, const uint32_t (&pk)[16]) {
    tmem_st_x16(t + lane_base + 16 * cg, pk);
    tmem_st_wait();
  };
  issue(true, [&] {
    scores(tX, dO, dV, &bar_score[0]);
    scores(tY, dV, dO, &bar_score[1]);
  });
  if (warp == 0) wait_bar_warp(&bar_full[1], 0, abort_flag, kWaitChunkTma, chunk);
  issue(true, [&] {
    if (with_S) times_state_t(tX, dO, sS, &bar_state[0]);
    if (with_R) times_state_t(tY, dV, sR, &bar_state[1]);
  });
  const float Gr = sG[row], total = sG[kGtChunk - 1];
  float head = kp ? ex2(Gr) : 0.f, tail = kp ? ex2(total - Gr) : 0.f;  // (a masked row is zero, whatever the states hold)
  float row_low = ex2(wq > 0 ? Gr - sG[32 * wq - 1] : 0.f), row_up = ex2(sG[32 * wq + 31] - Gr);
  uint32_t seen_low = (2u << lane) - 1u, seen_up = 0xffffffffu << lane;
  if (dropping) {
    row_drops<true>(drops, wq, lane, seen_low, row_low);
    row_drops<false>(drops, wq, lane, seen_up, row_up);
    if (drops.in(0, row)) head = 0.f;
    if (drops.in(row + 1, kGtChunk - 1)) tail = 0.f;
  }
  const int panel = cg / 2 * kTileBytes, j0 = 4 * (cg & 1);  // where this thread's 32 columns are in a row of D

  uint32_t pk[16];
  float ax[32], ay[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) ax[j] = 0.f, ay[j] = 0.f;
  // ---- dq: decayed scores X (packed over what the other warps of the rows have read), the state's part
  wait(&bar_score[0]);
  decay_block<T, true>(pk, tX + my_scores, cg, wq, seen_low, Gr, row_low, sG, sLow[wq]);
  sync();
  put_scores(tX, pk);
  if (with_S) {
    wait(&bar_state[0]);
    acc_scaled(ax, tX + my_acc, head);
  }
  // ---- dk: the same in Y
  wait(&bar_score[1]);
  decay_block<T, false>(pk, tY + my_scores, cg, wq, seen_up, Gr, row_up, sG, sUp[wq]);
  arrived(2, sQ);
  sync();
  issue(true, [&] { times_rows(tX, sK, &bar_rows[0]); });
  put_scores(tY, pk);
  if (with_R) {
    wait(&bar_state[1]);
    acc_scaled(ay, tY + my_acc, tail);
  }
  sync();
  issue(true, [&] { times_rows(tY, sQ, &bar_rows[1]); });
  // ---- <S, R>, and what of k.dk lies across the chunk's end
  sBd[cg][row] = with_R ? row_dot32<T>(sK + panel, row, j0, ay) : 0.f;
  float cross = 0.f;
  if (with_S && with_R) {
    wait_bar_warp(&bar_full[1], 0, abort_flag, kWaitChunkTma, chunk);
    const uint4 *s4 = reinterpret_cast<const uint4*>(sS), *r4 = reinterpret_cast<const uint4*>(sR);
#pragma unroll 2
    for (int e = tid; e < NT * NT * kStateTile / 16; e += kBwd128Threads) {
      const uint4 x = s4[e], y = r4[e];
      const uint32_t u[4] = {x.x, x.y, x.z, x.w}, w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = Pack2<T>::unpack(u[i]), f2 = Pack2<T>::unpack(w[i]);
        cross = fmaf(f.x, f2.x, fmaf(f.y, f2.y, cross));
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) cross += __shfl_xor_sync(0xffffffffu, cross, off);
  }
  if (lane == 0) sCross[warp] = cross;
  // ---- dq out, P' into X
  wait(&bar_rows[0]);
  acc_add(ax, tX + my_acc);
  sQd[cg][row] = row_dot32<T>(sQ + panel, row, j0, ax);
  stage_row<T>(sV + panel, row, j0, ax);  // (V's readers: the scores and dk's state part, all complete)
  fence_proxy_async_smem();
  sync();
  issue(true, [&] {
    scores(tX, dK, dQ, &bar_score[2]);
    if (with_R) times_state(tX, dK, sR, &bar_state[2]);
#pragma unroll
    for (int i = 0; i < NT; ++i) tma_store_tile_x(&m.dq, sV + i * kTileBytes, 64 * i, c0, h, bi);
    tma_store_commit();
  });
  // ---- dv: decayed scores X
  wait(&bar_score[2]);
  decay_block<T, false>(pk, tX + my_scores, cg, wq, seen_up, Gr, row_up, sG, sUp[wq]);
  sync();
  put_scores(tX, pk);
  // ---- dk out
  wait(&bar_rows[1]);
  {
    float y[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) y[j] = 0.f;
    acc_add(y, tY + my_acc);
    sKd[cg][row] = row_dot32<T>(sK + panel, row, j0, y);
#pragma unroll
    for (int j = 0; j < 32; ++j) ay[j] += y[j];
  }
  stage_row<T>(sQ + panel, row, j0, ay);  // (Q's readers: dk's rows and P', both complete)
  fence_proxy_async_smem();
  // ---- dv: the state's part, then the rows
#pragma unroll
  for (int j = 0; j < 32; ++j) ax[j] = 0.f;
  if (with_R) {
    wait(&bar_state[2]);
    acc_scaled(ax, tX + my_acc, tail);
  }
  sync();
  issue(true, [&] {
    times_rows(tX, sO, &bar_rows[2]);
#pragma unroll
    for (int i = 0; i < NT; ++i) tma_store_tile_x(&m.dk, sQ + i * kTileBytes, 64 * i, c0, h, bi);
    tma_store_commit();
  });
  // ---- dg (the first four warps: a position each)
  float x = 0.f;
  if (warp < 4) {
    float run = 0.f, up = 0.f;
#pragma unroll
    for (int i = 0; i < NG; ++i) run += sQd[i][row] - sKd[i][row], up += sBd[i][row];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {  // run: from the row to the warp's end; up: to the row
      const float d = __shfl_down_sync(0xffffffffu, run, off), u = __shfl_up_sync(0xffffffffu, up, off);
      if (lane + off < 32) run += d;
      if (lane >= off) up += u;
    }
    if (lane == 0) sPart[warp] = run;
    if (lane == 31) sPart[4 + warp] = up;
    const float before = __shfl_up_sync(0xffffffffu, up, 1);
    x = run + (lane ? before : 0.f);
  }
  // ---- dv out
  wait(&bar_rows[2]);
  acc_add(ax, tX + my_acc);
  stage_row<T>(sK + panel, row, j0, ax);  // (K's readers: dq's rows, P' and dv's state part, all complete)
  fence_proxy_async_smem();
  sync();
  issue(true, [&] {
#pragma unroll
    for (int i = 0; i < NT; ++i) tma_store_tile_x(&m.dv, sK + i * kTileBytes, 64 * i, c0, h, bi);
    tma_store_commit();
  });
  if (tid == 0 && *abort_flag) {  // no load may be in flight when the CTA leaves
    for (int i = 0; i < 3; ++i) mbar_wait(&bar_full[i], 0, 64);
  }
  if (warp == 1) tmem_dealloc(tX, kCols);
  if (warp < 4 && c0 + row < a.N && !*abort_flag) {
    float sr = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * NG; ++i) sr += sCross[i];
    const float A = dropping ? 0.f : ex2(total);
    x += A == 0.f ? 0.f : A * sr;
    for (int w = 0; w < 4; ++w) x += w > wq ? sPart[w] : w < wq ? sPart[4 + w] : 0.f;
    const int pos = c0 + row;
    if (!kp || (pos == 0 && !a.with_first) || gate_tc<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, pos) <= kGateFloorTc) x = 0.f;
    const long long o = b * a.sdg.b + h * a.sdg.h + static_cast<long long>(pos) * a.sdg.n;
    if (a.gate_f32)
      static_cast<float*>(a.dgate)[o] = x;
    else
      static_cast<T*>(a.dgate)[o] = from_acc<T>(x);
  }
  if (warp == 0) tma_store_wait_read<0>();  // (by all lanes: the groups belong to the one that stored)
}

// ---- backward at head dim 64: a persistent kernel ------------------------------------------------------------------------
// The same three passes, a group of eight warps for each, side by side.  A thread owns half a row, and each half is packed in place
// and has its half of the accumulator beside it, so that a warp reads what it alone has written over; everything a group does per
// chunk is a handful of rolled loops that all three run (the one-chunk kernel spent a quarter of its time waiting for instructions
// and another at its barriers):
//     scores, state's part (MMA) -> decay, pack -> rows (MMA) -> rows + scaled state's part -> the group's result tile -> TMA
// dv has no room in TMEM for a second accumulator: its state's part goes where its rows will be added, and is scaled there first.
//   warps 0-7: dq over Q     8-15: dk over K     16-23: dv over V     (rows and TMEM lanes 32 (w % 4) .., half (w / 4) % 2)
//   warps 24-27: gates of the next chunk, masked rows, <S, R>, dg     warp 28: TMA loads
//   warps 29-31, one thread each: the MMAs and the stores of a pass, so that the scores of the next chunk are under way while the
//   last rows of this one are written, and no working warp spends its time on issuing
// Two stages of (dO, V, K, Q, S, R), 80 KB, and a tile per group for its results, so that a stage is free as soon as the last group
// has its products (staged over the tiles instead, a stage was held until the stores had been read: 2000 of a chunk's 8000 cycles).
// B8 H16 N4096 bf16: 144 us, 3.4 TB/s; its traffic, states included, would take 83.  No single part bounds it (of 139 in one run of an
// earlier form: 129 without the decays, 136 without the dot products, 135 without writing dg; what keeps a dropped state and masked rows
// out takes 7 of the 144); the schedulers issue in 64 % of the cycles, and each group waits for its own MMAs.  (One accumulator of 64 columns per group, half as many MMAs, is no faster: 136, and 1 % more for a
// forward and a backward in turn.  L2 prefetches of the chunk after the next cost 8.)
// 128 TMEM columns per group, of which half h has 64: scores, then 32 of packed scores and 32 of the accumulator; 64 each for the
// state's part of dq and dk.
// Barriers that a stage's chunk completes once are kept per stage, so that nobody can be a whole phase ahead of one that waits.
// Every wait is bounded.  After one that gave up every further wait returns at once; the warps that share a named barrier go through
// all of them all the same.
constexpr int kBwd64Threads = 1024;
constexpr int kBwd64Stage = 4 * kTileBytes + 2 * kStateTile;
constexpr size_t kBwd64Smem = 1024 + 2 * kBwd64Stage + 3 * kTileBytes;

struct __align__(16) BwdInfo {  // of a chunk: one more than there are stages, so that a chunk's is made before its tiles arrive
  float G[kGtChunk];
  float low[192], up[192];  // column factors of row blocks 1, 2, 3 (32, 64, 96 columns) and 0, 1, 2 (96, 64, 32 columns)
  DropBits drops;                 // (where `dropping`)
  uint32_t from_s[4], from_r[4];  // unmasked rows that no drop parts from the state before, after the chunk: a bit each
  int has_s, has_r, dropping;
};
__device__ __forceinline__ int low_at(int w) { return 16 * w * (w - 1); }                      // of column 0 of row block w
__device__ __forceinline__ int up_at(int w) { return (w == 0 ? 0 : w == 1 ? 96 : 160) - 32 * (w + 1); }
// What the drops of a chunk change in its tables.  Thread t of four warps, `rows`: the unmasked rows of the warp.
__device__ __noinline__ void drop_tables(BwdInfo* f, int t, uint32_t rows) {
  const DropBits drops = f->drops;
#pragma unroll 1
  for (int w = 0; w < 3; ++w) {
    if (t < 32 * w + 32 && drops.in(t + 1, 32 * w + 31)) f->low[low_at(w + 1) + t] = 0.f;
    if (t >= 32 * w + 32 && drops.in(32 * w + 32, t)) f->up[up_at(w) + t] = 0.f;
  }
  const uint32_t rows_s = rows & __ballot_sync(0xffffffffu, !drops.in(0, t)), rows_r = rows & __ballot_sync(0xffffffffu, !drops.in(t + 1, kGtChunk - 1));
  __syncwarp();
  if ((t & 31) == 0) f->from_s[t >> 5] = rows_s, f->from_r[t >> 5] = rows_r;
}
struct BwdDots {  // a stage's dot products, by halves of the columns
  float qd[2][kGtChunk], kd[2][kGtChunk], bd[2][kGtChunk];
};
__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

template <typename T>
__global__ void __launch_bounds__(kBwd64Threads, 1) gated_bwd64_kernel(const __grid_constant__ GatedMaps m, const GatedChunkArgs a) {
  using namespace ptx;
  constexpr bool BF = Pack2<T>::kBf16;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ BwdInfo info[3];
  __shared__ BwdDots dots[2];
  __shared__ uint64_t bar_full[2], bar_free[2], bar_ready[2], bar_dots[2], bar_state[2], bar_score[3][2], bar_rows[3][2];
  __shared__ uint64_t bar_packed[3], bar_scaled, bar_read[3], bar_staged[3], bar_stored[3];  // a group to its issuing thread, once per chunk each
  __shared__ uint32_t tmem_slot;
  __shared__ float sPart[12];
  __shared__ int abort_flag_s, loads_s;
  volatile int* abort_flag = &abort_flag_s;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int wq = warp & 3, row = 32 * wq + lane;
  const uint32_t lane_base = static_cast<uint32_t>(32 * wq) << 16;
  auto tile_o = [&](int s) { return smem + s * kBwd64Stage; };
  auto tile_v = [&](int s) { return smem + s * kBwd64Stage + kTileBytes; };
  auto tile_k = [&](int s) { return smem + s * kBwd64Stage + 2 * kTileBytes; };
  auto tile_q = [&](int s) { return smem + s * kBwd64Stage + 3 * kTileBytes; };
  auto state_s = [&](int s) { return smem + s * kBwd64Stage + 4 * kTileBytes; };
  auto state_r = [&](int s) { return smem + s * kBwd64Stage + 4 * kTileBytes + kStateTile; };
  auto has_s = [&](int chunk) { return chunk > 0 || a.with_first; };
  auto has_r = [&](int chunk) { return chunk + 1 < a.nchunks || a.with_last; };
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar_full[s], 1);
      mbar_init(&bar_free[s], 28);  // the warps of the passes, four that took <S, R>
      mbar_init(&bar_ready[s], 4);
      mbar_init(&bar_dots[s], 16);
      mbar_init(&bar_state[s], 1);  // of dv
      for (int p = 0; p < 3; ++p) {
        mbar_init(&bar_score[p][s], 1);
        mbar_init(&bar_rows[p][s], 1);
      }
    }
    mbar_init(&bar_scaled, 8);
    for (int p = 0; p < 3; ++p) {
      mbar_init(&bar_packed[p], 8);
      mbar_init(&bar_read[p], 8);
      mbar_init(&bar_staged[p], 8);
      mbar_init(&bar_stored[p], 1);
    }
    mbar_fence_init();
    abort_flag_s = 0;
    loads_s = 0;
    tma_prefetch_desc(&m.q);
    tma_prefetch_desc(&m.k);
    tma_prefetch_desc(&m.v);
    tma_prefetch_desc(&m.o);
  }
  if (warp == 28) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  pdl_allow_next();
  pdl_wait_prior();
  const uint32_t tmem = tmem_slot;

  // E = dO V^T    E' = V dO^T    P' = K Q^T        rows of: K, Q, dO
  auto tile_of = [&](int s, int which) { return smem + s * kBwd64Stage + which * kTileBytes; };  // O 0, V 1, K 2, Q 3
  auto tile_a = [&](int s, int pass) { return tile_of(s, pass); };
  auto tile_b = [&](int s, int pass) { return tile_of(s, pass == 0 ? 1 : pass == 1 ? 0 : 3); };
  auto tile_c = [&](int s, int pass) { return tile_of(s, pass == 0 ? 2 : pass == 1 ? 3 : 0); };
  auto tile_x = [&](int s, int pass) { return tile_of(s, 3 - pass); };  // the rows that dq, dk are multiplied with: Q, K
  auto tile_out = [&](int pass) { return smem + 2 * kBwd64Stage + pass * kTileBytes; };

  if (warp >= 29) {
    // ---------------------------------------------------------------- MMAs and stores of a pass
    const int pass = warp - 29;
    if (elect_one()) {
      constexpr uint32_t kIdescP = make_idesc(128, 128, BF, false, false), kIdescK = make_idesc(128, 64, BF, false, false),
                         kIdescM = make_idesc(128, 32, BF, false, true);
      const uint32_t tP = tmem + 128 * pass;
      const CUtensorMap* out = pass == 0 ? &m.dq : pass == 1 ? &m.dk : &m.dv;
      auto store = [&](long unit, int n) {  // the result of the n-th chunk
        if (!wait_bar1(&bar_staged[pass], n & 1, abort_flag, kWaitAcc, n)) return false;
        const long bh = unit / a.nchunks;
        tma_store_tile(out, tile_out(pass), static_cast<int>(unit % a.nchunks) * kGtChunk, static_cast<int>(bh % a.H), static_cast<int>(bh / a.H));
        tma_store_commit();
        tma_store_wait_read<0>();
        mbar_arrive(&bar_stored[pass]);
        return true;
      };
      int n = 0;
      bool ok = true;
      long unit = blockIdx.x;
      for (; unit < a.units; unit += gridDim.x, ++n) {
        const int s = n & 1, chunk = static_cast<int>(unit % a.nchunks);
        const bool with_state = pass == 0 ? has_s(chunk) : has_r(chunk);
        const uint64_t dA = kdesc(smem_u32(tile_a(s, pass))), dB = kdesc(smem_u32(tile_b(s, pass)));
        if (!(ok = wait_bar2(&bar_ready[s], (n >> 1) & 1, n > 0 ? &bar_read[pass] : &bar_ready[s], n > 0 ? (n - 1) & 1 : 0, abort_flag, kWaitChunkTma, n))) break;
        tc_fence_after_sync();
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_ss(tP, dA + 2 * k, dB + 2 * k, kIdescP, k > 0);
        mma_commit(&bar_score[pass][s]);
        if (pass < 2 && with_state) {  // (complete when the rows are: the same thread commits them)
          const uint64_t d = kdesc(smem_u32(pass == 0 ? state_s(s) : state_r(s)));
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ss(tmem + 384 + 64 * pass, dA + 2 * k, d + 2 * k, kIdescK, k > 0);
        }
        if (n > 0 && !(ok = store(unit - gridDim.x, n - 1))) break;
        if (!(ok = wait_bar1(&bar_packed[pass], n & 1, abort_flag, kWaitScoreReady, n))) break;
        tc_fence_after_sync();
        if (pass == 2) {
          if (with_state) {  // columns 32 hh .. of R: 64 bytes into its rows
            const uint64_t d = mdesc(smem_u32(state_r(s)));
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_ss(tP + 64 * hh + 32, dA + 2 * k, d + 4 * hh + 128 * k, kIdescM, k > 0);
            mma_commit(&bar_state[s]);
          } else {
            mbar_arrive(&bar_state[s]);  // (one phase per chunk, whether there is a state or not; bar_scaled likewise)
          }
          if (!(ok = wait_bar1(&bar_scaled, n & 1, abort_flag, kWaitScoreReady, n))) break;
          tc_fence_after_sync();
        }
        const bool onto = pass == 2 && with_state;  // the rows are added to what is there
        const uint64_t d = mdesc(smem_u32(tile_c(s, pass)));
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(tP + 64 * hh + 32, tP + 8 * (k & 3) + 64 * (k >> 2), d + 4 * hh + 128 * k, kIdescM, k > 0 || onto ? 1u : 0u);
        mma_commit(&bar_rows[pass][s]);
      }
      if (ok && n > 0) store(unit - gridDim.x, n - 1);
    }
  } else if (warp == 28) {
    // ---------------------------------------------------------------- loads
    if (elect_one()) {
      int n = 0;
      for (long unit = blockIdx.x; unit < a.units; unit += gridDim.x, ++n) {
        const int s = n & 1;
        if (n >= 2 && !wait_bar(&bar_free[s], ((n >> 1) - 1) & 1, abort_flag, kWaitWalkFree, n)) break;
        const long bh = unit / a.nchunks;
        const int chunk = static_cast<int>(unit % a.nchunks), h = static_cast<int>(bh % a.H), b = static_cast<int>(bh / a.H), c0 = chunk * kGtChunk;
        mbar_expect_tx(&bar_full[s], 4 * kTileBytes + ((has_s(chunk) ? 1 : 0) + (has_r(chunk) ? 1 : 0)) * kStateTile);
        tma_load_tile(tile_o(s), &m.o, &bar_full[s], c0, h, b);
        tma_load_tile(tile_v(s), &m.v, &bar_full[s], c0, h, b);
        tma_load_tile(tile_k(s), &m.k, &bar_full[s], c0, h, b);
        tma_load_tile(tile_q(s), &m.q, &bar_full[s], c0, h, b);
        if (has_s(chunk)) bulk_load(state_s(s), a.S + unit * kStateTile, kStateTile, &bar_full[s]);
        if (has_r(chunk)) bulk_load(state_r(s), a.R + unit * kStateTile, kStateTile, &bar_full[s]);
        loads_s = n + 1;
      }
    }
  } else if (warp >= 24) {
    // ---------------------------------------------------------------- gates, masked rows, <S, R>, dg
    const int t = tid - 768;  // position
    RawGate raw[4];
    bool own_take = true;  // whether row t counts
    float cross_before = 0.f;
    bool kp_before = true;
    auto fetch = [&](long unit) {
      const long bh = unit / a.nchunks, b = bh / a.H;
      const int c0 = static_cast<int>(unit % a.nchunks) * kGtChunk, h = static_cast<int>(bh % a.H);
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[e] = gate_raw<T>(a.gate, a.keep, a.sg, a.gate_f32, a.N, b, h, c0 + 4 * lane + e);
      if (a.keep) own_take = c0 + t < a.N && a.keep[b * a.N + c0 + t];
    };
    // the sums of a chunk's gates and the column factors, from what was fetched
    auto make_tables = [&](int n, int chunk) {
      BwdInfo& f = info[n % 3];
      named_sync(4, 128);  // (nobody reads what stands there any more)
      float g[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) g[e] = gate_of<T>(raw[e], a.gate_f32);
      const bool dropping = take_drops(g, f.drops, lane);  // (the four warps write the same)
      gate_sums<false>(g, lane);
      if (wq == 0) *reinterpret_cast<float4*>(&f.G[4 * lane]) = make_float4(g[0], g[1], g[2], g[3]);
      if (t == 0) f.has_s = has_s(chunk), f.has_r = has_r(chunk), f.dropping = dropping;
      named_sync(4, 128);
#pragma unroll
      for (int w = 0; w < 3; ++w) {
        if (t < 32 * w + 32) f.low[low_at(w + 1) + t] = ex2(f.G[32 * w + 31] - f.G[t]);
        if (t >= 32 * w + 32) f.up[up_at(w) + t] = ex2(f.G[t] - f.G[32 * w + 31]);
      }
      const uint32_t rows = __ballot_sync(0xffffffffu, own_take);
      if (lane == 0) f.from_s[wq] = rows, f.from_r[wq] = rows;
      if (dropping) drop_tables(&f, t, rows);
    };
    // dg of a chunk that is done (unit u, the n-th of this CTA): its dot products, <S, R> as this warp's part
    auto write_dgate = [&](long u, int n, float cross, bool kept) {
      const BwdInfo& f = info[n % 3];
      wait_bar_warp(&bar_dots[n & 1], (n >> 1) & 1, abort_flag, kWaitAcc, n);
      const long bh = u / a.nchunks, b = bh / a.H;
      const int chunk = static_cast<int>(u % a.nchunks), h = static_cast<int>(bh % a.H), pos = chunk * kGtChunk + t;
      const BwdDots& d = dots[n & 1];
      float run = (d.qd[0][t] + d.qd[1][t]) - (d.kd[0][t] + d.kd[1][t]), up = d.bd[0][t] + d.bd[1][t];
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {  // run: from the row to the warp's end; up: to the row
        const float r = __shfl_down_sync(0xffffffffu, run, off), x = __shfl_up_sync(0xffffffffu, up, off);
        if (lane + off < 32) run += r;
        if (lane >= off) up += x;
      }
      named_sync(4, 128);  // (the sums of the chunk before have been read)
      if (lane == 0) sPart[wq] = run, sPart[8 + wq] = cross;
      if (lane == 31) sPart[4 + wq] = up;
      const float before = __shfl_up_sync(0xffffffffu, up, 1);
      named_sync(4, 128);
      const float A = f.dropping ? 0.f : ex2(f.G[kGtChunk - 1]);
      float x = run + (lane ? before : 0.f) + (A == 0.f ? 0.f : A * ((sPart[8] + sPart[9]) + (sPart[10] + sPart[11])));
      for (int w = 0; w < 4; ++w) x += w > wq ? sPart[w] : w < wq ? sPart[4 + w] : 0.f;
      if (pos < a.N && !*abort_flag) {
        if (!kept || (pos == 0 && !a.with_first) || (f.dropping && f.drops.w[wq] >> lane & 1u)) x = 0.f;
        const long long o = b * a.sdg.b + h * a.sdg.h + static_cast<long long>(pos) * a.sdg.n;
        if (a.gate_f32)
          static_cast<float*>(a.dgate)[o] = x;
        else
          static_cast<T*>(a.dgate)[o] = from_acc<T>(x);
      }
    };
    int n = 0;
    long unit = blockIdx.x;
    bool kept = false;
    if (unit < a.units) {
      fetch(unit);
      make_tables(0, static_cast<int>(unit % a.nchunks));
      kept = own_take;
      if (unit + gridDim.x < a.units) fetch(unit + gridDim.x);
    }
    for (; unit < a.units; unit += gridDim.x, ++n) {
      const int s = n & 1, chunk = static_cast<int>(unit % a.nchunks);
      wait_bar_warp(&bar_full[s], (n >> 1) & 1, abort_flag, kWaitChunkTma, n);
      if (a.keep) {  // nothing of a masked position gets into a product
        if (!kept) {
          const uint4 zero = make_uint4(0, 0, 0, 0);
          for (int j = 0; j < 8; ++j)
            for (int i = 0; i < 4; ++i) *tile_piece(tile_o(s) + i * kTileBytes, t, j) = zero;
        }
        fence_proxy_async_smem();
      }
      warp_arrive(&bar_ready[s], lane);
      float cross = 0.f;
      if (has_s(chunk) && has_r(chunk)) {
        const uint4 *x4 = reinterpret_cast<const uint4*>(state_s(s)), *y4 = reinterpret_cast<const uint4*>(state_r(s));
#pragma unroll
        for (int e = 0; e < kStateTile / 16 / 128; ++e) {
          const uint4 x = x4[t + 128 * e], y = y4[t + 128 * e];
          const uint32_t u[4] = {x.x, x.y, x.z, x.w}, w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 p = Pack2<T>::unpack(u[i]), q = Pack2<T>::unpack(w[i]);
            cross = fmaf(p.x, q.x, fmaf(p.y, q.y, cross));
          }
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) cross += __shfl_xor_sync(0xffffffffu, cross, off);
      }
      warp_arrive(&bar_free[s], lane);
      // the next chunk's tables, where those of two chunks ago were: the tiles that have just arrived are in the stage that it left
      const bool kept_now = kept;
      if (unit + gridDim.x < a.units) {
        make_tables(n + 1, static_cast<int>((unit + gridDim.x) % a.nchunks));
        kept = own_take;
        if (unit + 2 * static_cast<long>(gridDim.x) < a.units) fetch(unit + 2 * static_cast<long>(gridDim.x));
      }
      if (n > 0) write_dgate(unit - gridDim.x, n - 1, cross_before, kp_before);
      cross_before = cross;
      kp_before = kept_now;
    }
    if (n > 0) write_dgate(unit - gridDim.x, n - 1, cross_before, kp_before);
  } else {
    // ---------------------------------------------------------------- the passes
    const int pass = warp >> 3, half = (warp >> 2) & 1;  // 0 dq, 1 dk, 2 dv
    const bool lower = pass == 0;
    const uint32_t tMine = tmem + 128 * pass + 64 * half + lane_base;
    const float sign = lower ? 1.f : -1.f;
    const uint32_t tState = tmem + 384 + 64 * pass + 32 * half + lane_base;
    // several barriers at once: one round trip
    auto wait = [&](int n, auto... bars) {
      const uint32_t parity = (n >> 1) & 1;
      for (uint32_t i = 0; i < kMaxPolls; ++i) {
        bool done = true;
        ((done = mbar_try_wait(bars, parity) && done), ...);
        if (__all_sync(0xffffffffu, done)) return true;
        if (*abort_flag) return false;
      }
      *abort_flag = 1;
      atomicCAS(&g_cott_status, 0, (kWaitChunkMma << 16) | (n & 0xffff));
      return false;
    };
    int n = 0;
    for (long unit = blockIdx.x; unit < a.units; unit += gridDim.x, ++n) {
      const int s = n & 1;
      const BwdInfo& f = info[n % 3];
      unsigned char *sX = tile_x(s, pass), *sOut = tile_out(pass);
      // (tiles are read row by row below: every reader has to see the loads' completion itself)
      if (!wait(n, &bar_full[s], &bar_ready[s], &bar_score[pass][s])) break;
      tc_fence_after_sync();
      const bool with_state = lower ? f.has_s : f.has_r;
      const float Gr = f.G[row], signedG = sign * Gr;
      float rowf = ex2(lower ? (wq > 0 ? Gr - f.G[32 * wq - 1] : 0.f) : f.G[32 * wq + 31] - Gr);
      uint32_t seen = lower ? (2u << lane) - 1u : 0xffffffffu << lane;  // of the diagonal block's columns
      if (f.dropping) {
        if (lower)
          row_drops<true>(f.drops, wq, lane, seen, rowf);
        else
          row_drops<false>(f.drops, wq, lane, seen, rowf);
      }
      const float* col = lower ? f.low + low_at(wq) : f.up + up_at(wq);  // (of a block without factors: not read)
      // decayed, masked, packed in place: the half's first 32 columns into its first 16, then the others into the next 16
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        const int blk = 2 * half + i;
        uint32_t pk[16];
        if (lower ? blk > wq : blk < wq) {
#pragma unroll
          for (int j = 0; j < 16; ++j) pk[j] = 0u;
        } else {
          uint32_t r[32];
          tmem_ld_x32(tMine + 32 * i, r);
          tmem_ld_wait();
          if (blk == wq) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 Gs = *reinterpret_cast<const float4*>(&f.G[32 * blk + j]);
#pragma unroll
              for (int e = 0; e < 4; e += 2) {
                float2 x = fma2(make_float2(-sign, -sign), e ? make_float2(Gs.z, Gs.w) : make_float2(Gs.x, Gs.y), make_float2(signedG, signedG));
                x = mul2(make_float2(ex2(x.x), ex2(x.y)), pair(r + j + e));
                x.x = seen & (1u << (j + e)) ? x.x : 0.f;
                x.y = seen & (2u << (j + e)) ? x.y : 0.f;
                pk[(j + e) / 2] = Pack2<T>::pack(x.x, x.y);
              }
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 cf = *reinterpret_cast<const float4*>(&col[32 * blk + j]);
              const float2 x = mul2(pair(r + j), mul2(make_float2(cf.x, cf.y), make_float2(rowf, rowf)));
              const float2 y = mul2(pair(r + j + 2), mul2(make_float2(cf.z, cf.w), make_float2(rowf, rowf)));
              pk[j / 2] = Pack2<T>::pack(x.x, x.y);
              pk[j / 2 + 1] = Pack2<T>::pack(y.x, y.y);
            }
          }
        }
        tmem_st_x16(tMine + 16 * i, pk);
      }
      tmem_st_wait();
      tc_fence_before_sync();
      warp_arrive(&bar_packed[pass], lane);
      // (a masked row is zero, whatever the state holds)
      const float scale = (lower ? f.from_s[wq] : f.from_r[wq]) >> lane & 1u ? ex2(lower ? Gr : f.G[kGtChunk - 1] - Gr) : 0.f;
      const bool dropped = __any_sync(0xffffffffu, scale == 0.f);
      if (pass == 2) {
        if (with_state) {  // dv: the state's part, scaled where it is
          if (!wait(n, &bar_state[s])) break;
          tc_fence_after_sync();
          uint32_t r[32];
          tmem_ld_x32(tMine + 32, r);
          tmem_ld_wait();
          if (dropped) drop_if(scale == 0.f, r);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 x = mul2(pair(r + j), make_float2(scale, scale));
            r[j] = __float_as_uint(x.x), r[j + 1] = __float_as_uint(x.y);
          }
          tmem_st_x32(tMine + 32, r);
          tmem_st_wait();
          tc_fence_before_sync();
        }
        warp_arrive(&bar_scaled, lane);
      }
      // the rows; and the place of the result: what was there has been stored
      bool ok = false;
      for (uint32_t i = 0; i < kMaxPolls && !ok; ++i) {
        const bool d0 = mbar_try_wait(&bar_rows[pass][s], (n >> 1) & 1), d1 = n == 0 || mbar_try_wait(&bar_stored[pass], (n - 1) & 1);
        ok = __all_sync(0xffffffffu, d0 && d1);
        if (!ok && *abort_flag) break;
      }
      if (!ok) {
        if (!*abort_flag) atomicCAS(&g_cott_status, 0, (kWaitChunkMma << 16) | (n & 0xffff));
        *abort_flag = 1;
        break;
      }
      tc_fence_after_sync();
      // the result's row, and q.dq, k.dk over the half's columns (k.dk by parts)
      float2 dot = make_float2(0.f, 0.f), across = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        uint32_t x[16];
        tmem_ld_x16(tMine + 32 + 16 * i, x);
        uint4 u, w;
        if (pass < 2) {
          u = *tile_piece(sX, row, 4 * half + 2 * i), w = *tile_piece(sX, row, 4 * half + 2 * i + 1);
          uint32_t y[16];
          if (with_state) tmem_ld_x16(tState + 16 * i, y);
          tmem_ld_wait();
          if (pass == 1) dot16_2<T>(dot, x, u, w);
          if (with_state) {
            if (dropped) drop_if(scale == 0.f, y);
            if (pass == 1) dot16_2<T>(across, y, u, w);
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
              const float2 z = fma2(pair(y + j), make_float2(scale, scale), pair(x + j));
              x[j] = __float_as_uint(z.x), x[j + 1] = __float_as_uint(z.y);
            }
          }
          if (pass == 0) dot16_2<T>(dot, x, u, w);
        } else {
          tmem_ld_wait();
        }
        if (i == 1) {
          tc_fence_before_sync();
          warp_arrive(&bar_read[pass], lane);
        }
        u.x = Pack2<T>::pack(__uint_as_float(x[0]), __uint_as_float(x[1])), u.y = Pack2<T>::pack(__uint_as_float(x[2]), __uint_as_float(x[3]));
        u.z = Pack2<T>::pack(__uint_as_float(x[4]), __uint_as_float(x[5])), u.w = Pack2<T>::pack(__uint_as_float(x[6]), __uint_as_float(x[7]));
        w.x = Pack2<T>::pack(__uint_as_float(x[8]), __uint_as_float(x[9])), w.y = Pack2<T>::pack(__uint_as_float(x[10]), __uint_as_float(x[11]));
        w.z = Pack2<T>::pack(__uint_as_float(x[12]), __uint_as_float(x[13])), w.w = Pack2<T>::pack(__uint_as_float(x[14]), __uint_as_float(x[15]));
        *tile_piece(sOut, row, 4 * half + 2 * i) = u;
        *tile_piece(sOut, row, 4 * half + 2 * i + 1) = w;
      }
      fence_proxy_async_smem();
      warp_arrive(&bar_staged[pass], lane);
      if (lane == 0) mbar_arrive(&bar_free[s]);  // (all MMAs of this pass that read the stage have completed, and its rows have been read)
      if (pass < 2) {
        if (pass == 0) {
          dots[s].qd[half][row] = dot.x + dot.y;
        } else {
          dots[s].kd[half][row] = dot.x + dot.y;
          dots[s].bd[half][row] = scale * (across.x + across.y);
        }
        warp_arrive(&bar_dots[s], lane);
      }
    }
  }

  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if (tid == 0 && *abort_flag) {  // no load may be in flight when the CTA leaves
    for (int n = loads_s > 2 ? loads_s - 2 : 0; n < loads_s; ++n) mbar_wait(&bar_full[n & 1], (n >> 1) & 1, 64);
  }
  __syncthreads();
  if (warp == 28) tmem_dealloc(tmem, 512);
}

}  // namespace cott
