// Launchers of the gated scan's tensor-core kernels.
#include "gated_tc.cuh"

using namespace cott;

namespace {

constexpr int kSms = 148;  // (sizes of buffers follow from it: a constant, so that they are the same on every host)

int tc_chunks(int N) { return (N + kGtChunk - 1) / kGtChunk; }

// Into how many segments the walk of a sequence is cut: as many as fit beside each other on the SMs, where that saves more than the two
// short kernels behind it cost (a chunk of a walk takes about 1 us, they take about 10).  (A walk's CTA fills an SM.  From 75 walks on,
// one each, SMs stay idle, and from 149 on a second wave follows: cutting those walks too is not done.)
int walk_segments(long walks, int n) {
  const int room = (int)(kSms / walks);
  if (room < 2) return 1;
  const int per = (n + room - 1) / room;
  return n - per < 10 ? 1 : (n + per - 1) / per;
}
size_t round256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }
size_t seg_bytes(long bh, int N, int D) {
  const int nseg = walk_segments(bh * (D / 64), tc_chunks(N));
  return nseg > 1 ? round256((size_t)bh * nseg * D * D * sizeof(float)) + round256((size_t)bh * nseg * sizeof(float)) +
                        round256((size_t)bh * tc_chunks(N) * sizeof(float))
                  : 0;
}
size_t tile_bytes(int D) { return (size_t)(D / 64) * (D / 64) * kStateTile; }

cott_strides filled(const cott_strides& s, int B, int H, int N, int D) {  // a dimension of one entry may come with any stride
  cott_strides r = s;
  if (N == 1) r.n = D;
  if (H == 1) r.h = D;
  if (B == 1) r.b = D;
  return r;
}
int make_map(CUtensorMap* map, const void* p, const cott_strides& s0, int B, int H, int N, int D, int dtype) {
  const cott_strides s = filled(s0, B, H, N, D);
  const int r = make_tmap_rows64(map, p, dtype == COTT_BF16, B, H, N, TileStrides{s.b, s.h, s.n}, kGtChunk, D);
  return r ? fail(COTT_ERR_CUDA, "TMA descriptor creation failed (%d)", r) : COTT_OK;
}
#define TRY(expr)             \
  do {                        \
    const int _st = (expr);   \
    if (_st) return _st;      \
  } while (0)

template <typename T, int D, bool REV, int SPLIT>
int launch_walk_split(GatedTcArgs a, const CUtensorMap& y, const CUtensorMap& z, long bh, void* seg, cudaStream_t stream) {
  constexpr int NT = D / 64;
  const size_t smem = walk_smem<D, SPLIT>();
  a.nseg = walk_segments(bh * NT, a.nchunks);
  a.chunks_per_seg = (a.nchunks + a.nseg - 1) / a.nseg;
  const dim3 grid((unsigned)bh, a.nseg, NT);
  if (a.nseg > 1) {
    unsigned char* p = static_cast<unsigned char*>(seg);
    a.seg_state = reinterpret_cast<float*>(p);
    p += round256((size_t)bh * a.nseg * D * D * sizeof(float));
    a.seg_log = reinterpret_cast<float*>(p);
    a.chunk_log = reinterpret_cast<float*>(p + round256((size_t)bh * a.nseg * sizeof(float)));
  }
  auto walk = gated_walk_kernel<T, D, REV, SPLIT>;
  COTT_CUDA_TRY(cudaFuncSetAttribute(walk, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  COTT_CUDA_TRY(launch_pdl(walk, grid, kWalkThreads, smem, stream, y, z, a));
  if (a.nseg > 1) {
    COTT_CUDA_TRY(launch_pdl(gated_seg_kernel<D>, dim3((unsigned)(bh * NT), D * 64 / 256), 256, 0, stream, a));
    COTT_CUDA_TRY(launch_pdl(gated_patch_kernel<T, D, REV>, dim3((unsigned)(bh * a.nchunks * NT)), 128, 0, stream, a));
  }
  return COTT_OK;
}
template <typename T, int D, bool REV>
int launch_walk(const GatedTcArgs& a, const CUtensorMap& y, const CUtensorMap& z, long bh, void* seg, cudaStream_t stream) {
  return a.last ? launch_walk_split<T, D, REV, 3>(a, y, z, bh, seg, stream) : launch_walk_split<T, D, REV, 2>(a, y, z, bh, seg, stream);
}

GatedTcArgs walk_args(const GatedArgs& g) {
  GatedTcArgs a = {};
  a.gate = g.gate, a.keep = g.keep, a.sg = g.sg, a.H = g.H, a.N = g.N, a.nchunks = tc_chunks(g.N), a.gate_f32 = g.gate_f32;
  return a;
}
GatedChunkArgs chunk_args(const GatedArgs& g, long bh) {
  GatedChunkArgs c = {};
  c.gate = g.gate, c.keep = g.keep, c.sg = g.sg, c.sdg = g.sdg, c.H = g.H, c.N = g.N, c.nchunks = tc_chunks(g.N), c.gate_f32 = g.gate_f32;
  c.units = bh * c.nchunks, c.with_first = g.with_initial;
  return c;
}

template <typename T, int D>
int run_tc_fwd(const GatedArgs& g, void* states, void* ws, int B, int dtype, cudaStream_t stream) {
  const long bh = (long)B * g.H;
  CUtensorMap q, k, v, o;
  TRY(make_map(&q, g.q, g.sq, B, g.H, g.N, D, dtype));
  TRY(make_map(&k, g.k, g.sk, B, g.H, g.N, D, dtype));
  TRY(make_map(&v, g.v, g.sv, B, g.H, g.N, D, dtype));
  TRY(make_map(&o, g.out, g.so, B, g.H, g.N, D, dtype));
  GatedTcArgs a = walk_args(g);
  a.edge = g.initial, a.last = g.final_state, a.states = static_cast<unsigned char*>(states);
  TRY((launch_walk<T, D, false>(a, k, v, bh, ws, stream)));
  GatedChunkArgs c = chunk_args(g, bh);
  c.S = a.states;
  auto kern = gated_fwd_tc_kernel<T, D>;
  COTT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)fwd_tc_smem<D>()));
  COTT_CUDA_TRY(launch_pdl(kern, dim3((unsigned)(c.units * (D / 64))), kFwdThreads, fwd_tc_smem<D>(), stream, q, k, v, o, c));
  return COTT_OK;
}

template <typename T, int D>
int run_tc_bwd(const GatedArgs& g, const void* states, void* ws, int B, int dtype, cudaStream_t stream) {
  const long bh = (long)B * g.H;
  GatedMaps m;
  TRY(make_map(&m.q, g.q, g.sq, B, g.H, g.N, D, dtype));
  TRY(make_map(&m.k, g.k, g.sk, B, g.H, g.N, D, dtype));
  TRY(make_map(&m.v, g.v, g.sv, B, g.H, g.N, D, dtype));
  TRY(make_map(&m.o, g.dout, g.so, B, g.H, g.N, D, dtype));
  TRY(make_map(&m.dq, g.dq, g.sdq, B, g.H, g.N, D, dtype));
  TRY(make_map(&m.dk, g.dk, g.sdk, B, g.H, g.N, D, dtype));
  TRY(make_map(&m.dv, g.dv, g.sdv, B, g.H, g.N, D, dtype));
  GatedTcArgs a = walk_args(g);
  unsigned char* p = static_cast<unsigned char*>(ws);
  a.edge = g.dfinal, a.last = g.dinitial, a.states = p;
  GatedChunkArgs c = chunk_args(g, bh);
  TRY((launch_walk<T, D, true>(a, m.q, m.o, bh, p + round256(c.units * tile_bytes(D)), stream)));
  c.S = static_cast<const unsigned char*>(states), c.R = a.states, c.dgate = g.dgate, c.with_last = g.dfinal != nullptr;
  if constexpr (D == 64) {
    auto kern = gated_bwd64_kernel<T>;
    COTT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBwd64Smem));
    COTT_CUDA_TRY(launch_pdl(kern, dim3((unsigned)(c.units < kSms ? c.units : kSms)), kBwd64Threads, kBwd64Smem, stream, m, c));
  } else {
    auto kern = gated_bwd128_kernel<T>;
    COTT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kBwd128Smem));
    COTT_CUDA_TRY(launch_pdl(kern, dim3((unsigned)c.units), kBwd128Threads, kBwd128Smem, stream, m, c));
  }
  return COTT_OK;
}

}  // namespace

namespace cott {

bool gated_tc_usable(int D, int dtype) { return (D == 64 || D == 128) && (dtype == COTT_F16 || dtype == COTT_BF16); }

size_t gated_tc_states_bytes(int B, int H, int N, int D) { return (size_t)B * H * tc_chunks(N) * tile_bytes(D); }

size_t gated_tc_workspace_bytes(int B, int H, int N, int D, bool backward) {
  const long bh = (long)B * H;
  if (!backward) return seg_bytes(bh, N, D);
  const size_t units = (size_t)bh * tc_chunks(N);
  return round256(units * tile_bytes(D)) + seg_bytes(bh, N, D);
}

int gated_tc_fwd(const GatedArgs& g, void* states, void* workspace, int B, int D, int dtype, cudaStream_t stream) {
  if (dtype == COTT_BF16)
    return D == 64 ? run_tc_fwd<__nv_bfloat16, 64>(g, states, workspace, B, dtype, stream) : run_tc_fwd<__nv_bfloat16, 128>(g, states, workspace, B, dtype, stream);
  return D == 64 ? run_tc_fwd<__half, 64>(g, states, workspace, B, dtype, stream) : run_tc_fwd<__half, 128>(g, states, workspace, B, dtype, stream);
}
int gated_tc_bwd(const GatedArgs& g, const void* states, void* workspace, int B, int D, int dtype, cudaStream_t stream) {
  if (dtype == COTT_BF16)
    return D == 64 ? run_tc_bwd<__nv_bfloat16, 64>(g, states, workspace, B, dtype, stream) : run_tc_bwd<__nv_bfloat16, 128>(g, states, workspace, B, dtype, stream);
  return D == 64 ? run_tc_bwd<__half, 64>(g, states, workspace, B, dtype, stream) : run_tc_bwd<__half, 128>(g, states, workspace, B, dtype, stream);
}

int gated_tc_status(int* value) {
  COTT_CUDA_TRY(cudaMemcpyFromSymbol(value, g_cott_status, sizeof(int)));
  if (*value) {
    const int zero = 0;
    COTT_CUDA_TRY(cudaMemcpyToSymbol(g_cott_status, &zero, sizeof(int)));
  }
  return COTT_OK;
}

}  // namespace cott
