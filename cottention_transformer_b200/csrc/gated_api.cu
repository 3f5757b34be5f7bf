// C ABI of the gated causal scan and of its single-token form: checks and dispatch.
#include "gated_simt.cuh"
#include "gated_step.cuh"

using namespace cott;

namespace {

int chunks_of(int N) { return (N + kGsChunk - 1) / kGsChunk; }
size_t round16(size_t n) { return (n + 15) & ~static_cast<size_t>(15); }

cott_strides dense(int H, int N, int D) { return cott_strides{(long long)H * N * D, (long long)N * D, D}; }

int check_sizes(const char* what, int B, int H, int N, int D, int dtype, int gate_dtype) {
  if (dtype != COTT_F32 && dtype != COTT_F16 && dtype != COTT_BF16)
    return fail(COTT_ERR_DTYPE, "%s takes float32, float16 or bfloat16 (dtype code %d)", what, dtype);
  if (gate_dtype != COTT_F32 && gate_dtype != dtype)
    return fail(COTT_ERR_DTYPE, "%s: log_decay is float32 or of the tensors' type (dtype code %d)", what, gate_dtype);
  if (B < 0 || H < 0 || N < 0) return fail(COTT_ERR_SHAPE, "negative size B=%d H=%d N=%d", B, H, N);
  if (D != 32 && D != 64 && D != 128) return fail(COTT_ERR_SHAPE, "%s supports head dims 32, 64 and 128 (got %d)", what, D);
  if ((long)B * H * chunks_of(N) > 0x7fffffffL || (long)B * H > 0x1fffffffL) return fail(COTT_ERR_SHAPE, "B*H*N too large");
  return COTT_OK;
}
// rows are read 16 bytes at a time
int check_rows(const char* name, const void* p, const cott_strides& s, int dtype) {
  const long long unit = 16 / (long long)dtype_size(dtype);
  if (!p) return fail(COTT_ERR_NULL, "null pointer: %s", name);
  if (reinterpret_cast<uintptr_t>(p) & 15) return fail(COTT_ERR_ALIGN, "%s must be 16-byte aligned", name);
  if (s.b % unit || s.h % unit || s.n % unit) return fail(COTT_ERR_ALIGN, "the strides of %s must be multiples of 16 bytes", name);
  return COTT_OK;
}
int check_state(const char* name, const void* p) {
  return reinterpret_cast<uintptr_t>(p) & 15 ? fail(COTT_ERR_ALIGN, "%s must be 16-byte aligned", name) : COTT_OK;
}

GatedArgs args_of(const cott_gated_layout* l, int H, int N, int D, int gate_dtype) {
  GatedArgs g = {};
  const cott_strides d = dense(H, N, D), gd = {(long long)H * N, N, 1};
  g.sq = l ? l->q : d, g.sk = l ? l->k : d, g.sv = l ? l->v : d, g.so = l ? l->out : d;
  g.sdq = l ? l->dq : d, g.sdk = l ? l->dk : d, g.sdv = l ? l->dv : d;
  g.sg = l ? l->gate : gd, g.sdg = l ? l->dgate : gd;
  g.H = H, g.N = N, g.nchunks = chunks_of(N), g.gate_f32 = gate_dtype == COTT_F32;
  return g;
}
size_t prefix_floats(int B, int H, int N, int D) { return (size_t)B * H * (chunks_of(N) + 1) * D * D; }
size_t suffix_floats(int B, int H, int N, int D) { return (size_t)B * H * chunks_of(N) * D * D; }

template <typename T, int D, bool REV>
int launch_states(const GatedArgs& g, long states, cudaStream_t stream) {
  const size_t smem = 2 * kGsChunk * (D + 4) * sizeof(float);
  auto kern = gated_state_kernel<T, D, REV>;
  COTT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  COTT_CUDA_TRY(launch_pdl(kern, dim3((unsigned)(states * g.nchunks)), kGsThreads, smem, stream, g));
  COTT_CUDA_TRY(launch_pdl(gated_prefix_kernel<D, REV>, dim3((unsigned)states, D * D / kGsThreads), kGsThreads, 0, stream, g));
  return COTT_OK;
}
template <typename T, int D, bool FWD>
int launch_chunks(const GatedArgs& g, long states, cudaStream_t stream) {
  const size_t smem = (3 * kGsChunk * (D + 4) + kGsChunk * (kGsChunk + 4)) * sizeof(float);
  auto kern = gated_chunk_kernel<T, D, FWD>;
  COTT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  COTT_CUDA_TRY(launch_pdl(kern, dim3((unsigned)(states * g.nchunks), FWD ? 1 : 3), kGsThreads, smem, stream, g));
  return COTT_OK;
}
template <typename T, int D>
int run_fwd(const GatedArgs& g, long states, cudaStream_t stream) {
  int st = launch_states<T, D, false>(g, states, stream);
  return st ? st : launch_chunks<T, D, true>(g, states, stream);
}
template <typename T, int D>
int run_bwd(const GatedArgs& g, long states, cudaStream_t stream) {
  int st = launch_states<T, D, true>(g, states, stream);
  if (st || (st = launch_chunks<T, D, false>(g, states, stream))) return st;
  COTT_CUDA_TRY(launch_pdl(gated_dgate_kernel<T, D>, dim3((unsigned)(states * g.nchunks)), kGsThreads, 0, stream, g));
  return COTT_OK;
}
// float32 at every head dim; the 16-bit types at 32 (64 and 128 are the tensor cores')
template <bool FWD, typename T, int D>
int run_one(const GatedArgs& g, long states, cudaStream_t stream) {
  return FWD ? run_fwd<T, D>(g, states, stream) : run_bwd<T, D>(g, states, stream);
}
template <bool FWD>
int run_any(const GatedArgs& g, int D, int dtype, long states, cudaStream_t stream) {
  if (dtype == COTT_F16) return run_one<FWD, __half, 32>(g, states, stream);
  if (dtype == COTT_BF16) return run_one<FWD, __nv_bfloat16, 32>(g, states, stream);
  switch (D) {
    case 32: return run_one<FWD, float, 32>(g, states, stream);
    case 64: return run_one<FWD, float, 64>(g, states, stream);
    default: return run_one<FWD, float, 128>(g, states, stream);
  }
}

template <typename T>
int run_step(const StepArgs& a, int D, long states, cudaStream_t stream) {
  switch (D) {
    case 32: return launch_gated_step<T, 32>(a, states, stream);
    case 64: return launch_gated_step<T, 64>(a, states, stream);
    default: return launch_gated_step<T, 128>(a, states, stream);
  }
}

}  // namespace

extern "C" {

size_t cott_gated_scan_states_bytes(int B, int H, int N, int D, int dtype) {
  if (B <= 0 || H <= 0 || N <= 0 || check_sizes("cott_gated_scan", B, H, N, D, dtype, COTT_F32)) return 0;
  if (gated_tc_usable(D, dtype)) return gated_tc_states_bytes(B, H, N, D);
  return prefix_floats(B, H, N, D) * sizeof(float) + round16((size_t)B * H * chunks_of(N) * sizeof(float));
}

size_t cott_gated_scan_workspace_bytes(int B, int H, int N, int D, int dtype, int backward) {
  if (B <= 0 || H <= 0 || N <= 0 || check_sizes("cott_gated_scan", B, H, N, D, dtype, COTT_F32)) return 0;
  if (gated_tc_usable(D, dtype)) return gated_tc_workspace_bytes(B, H, N, D, backward != 0);
  if (!backward) return 0;
  return (suffix_floats(B, H, N, D) + 2 * (size_t)B * H * chunks_of(N) * kGsChunk) * sizeof(float);
}

int cott_gated_scan_fwd(const void* q, const void* k, const void* v, const void* log_decay, const unsigned char* keep, const float* initial_state,
                        void* out, float* final_state, void* states, void* workspace, const cott_gated_layout* layout, int B, int H, int N, int D,
                        int dtype, int gate_dtype, void* stream) {
  int st = check_sizes("cott_gated_scan_fwd", B, H, N, D, dtype, gate_dtype);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long n = (long)B * H;
  if ((st = check_state("initial_state", initial_state)) || (st = check_state("final_state", final_state))) return st;
  if (n * N == 0) {
    if (!final_state || n == 0) return COTT_OK;
    DeviceScope scope(final_state);
    COTT_CUDA_TRY(scope.status());
    const size_t bytes = (size_t)n * D * D * sizeof(float);
    if (!initial_state)
      COTT_CUDA_TRY(cudaMemsetAsync(final_state, 0, bytes, s));
    else if (initial_state != final_state)
      COTT_CUDA_TRY(cudaMemcpyAsync(final_state, initial_state, bytes, cudaMemcpyDeviceToDevice, s));
    return COTT_OK;
  }
  GatedArgs g = args_of(layout, H, N, D, gate_dtype);
  if ((st = check_rows("q", q, g.sq, dtype)) || (st = check_rows("k", k, g.sk, dtype)) || (st = check_rows("v", v, g.sv, dtype)) ||
      (st = check_rows("out", out, g.so, dtype)))
    return st;
  if (!log_decay) return fail(COTT_ERR_NULL, "null pointer: log_decay");
  if (!states) return fail(COTT_ERR_NULL, "null pointer: states");
  if ((st = check_state("states", states))) return st;
  DeviceScope scope(q);
  COTT_CUDA_TRY(scope.status());
  g.q = q, g.k = k, g.v = v, g.gate = log_decay, g.keep = keep, g.initial = initial_state, g.out = out, g.final_state = final_state;
  g.with_initial = initial_state != nullptr;
  if (gated_tc_usable(D, dtype)) {
    if (!workspace && gated_tc_workspace_bytes(B, H, N, D, false)) return fail(COTT_ERR_NULL, "null pointer: workspace");
    if ((st = check_state("workspace", workspace))) return st;
    return gated_tc_fwd(g, states, workspace, B, D, dtype, s);
  }
  g.prefix = static_cast<float*>(states), g.total = g.prefix + prefix_floats(B, H, N, D);
  return run_any<true>(g, D, dtype, n, s);
}

int cott_gated_scan_bwd(const void* q, const void* k, const void* v, const void* log_decay, const unsigned char* keep, int with_initial_state,
                        const void* states, const void* dout, const float* dfinal_state, void* workspace, void* dq, void* dk, void* dv,
                        void* dlog_decay, float* dinitial_state, const cott_gated_layout* layout, int B, int H, int N, int D, int dtype,
                        int gate_dtype, void* stream) {
  int st = check_sizes("cott_gated_scan_bwd", B, H, N, D, dtype, gate_dtype);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const long n = (long)B * H;
  if ((st = check_state("dfinal_state", dfinal_state)) || (st = check_state("dinitial_state", dinitial_state))) return st;
  if (n * N == 0) {
    if (!dinitial_state || n == 0) return COTT_OK;
    DeviceScope scope(dinitial_state);
    COTT_CUDA_TRY(scope.status());
    const size_t bytes = (size_t)n * D * D * sizeof(float);
    if (!dfinal_state)
      COTT_CUDA_TRY(cudaMemsetAsync(dinitial_state, 0, bytes, s));
    else if (dfinal_state != dinitial_state)
      COTT_CUDA_TRY(cudaMemcpyAsync(dinitial_state, dfinal_state, bytes, cudaMemcpyDeviceToDevice, s));
    return COTT_OK;
  }
  GatedArgs g = args_of(layout, H, N, D, gate_dtype);
  if ((st = check_rows("q", q, g.sq, dtype)) || (st = check_rows("k", k, g.sk, dtype)) || (st = check_rows("v", v, g.sv, dtype)) ||
      (st = check_rows("dout", dout, g.so, dtype)) || (st = check_rows("dq", dq, g.sdq, dtype)) || (st = check_rows("dk", dk, g.sdk, dtype)) ||
      (st = check_rows("dv", dv, g.sdv, dtype)))
    return st;
  if (!log_decay || !dlog_decay) return fail(COTT_ERR_NULL, "null pointer: %s", log_decay ? "dlog_decay" : "log_decay");
  if (!states || !workspace) return fail(COTT_ERR_NULL, "null pointer: %s", states ? "workspace" : "states");
  if ((st = check_state("states", states)) || (st = check_state("workspace", workspace))) return st;
  DeviceScope scope(q);
  COTT_CUDA_TRY(scope.status());
  g.q = q, g.k = k, g.v = v, g.dout = dout, g.gate = log_decay, g.keep = keep, g.dfinal = dfinal_state, g.dinitial = dinitial_state;
  g.dq = dq, g.dk = dk, g.dv = dv, g.dgate = dlog_decay, g.with_initial = with_initial_state != 0;
  if (gated_tc_usable(D, dtype)) return gated_tc_bwd(g, states, workspace, B, D, dtype, s);
  g.prefix = const_cast<float*>(static_cast<const float*>(states)), g.total = g.prefix + prefix_floats(B, H, N, D);
  g.suffix = static_cast<float*>(workspace), g.qdot = g.suffix + suffix_floats(B, H, N, D), g.kdot = g.qdot + (size_t)n * g.nchunks * kGsChunk;
  return run_any<false>(g, D, dtype, n, s);
}

int cott_gated_step(float* state, const void* q, const void* k, const void* v, const void* log_decay, void* out, const cott_gated_layout* layout,
                    int B, int H, int T, int D, int dtype, int gate_dtype, void* stream) {
  int st = check_sizes("cott_gated_step", B, H, T, D, dtype, gate_dtype);
  if (st) return st;
  if ((long)B * H * T == 0) return COTT_OK;
  const GatedArgs g = args_of(layout, H, T, D, gate_dtype);
  if ((st = check_rows("q", q, g.sq, dtype)) || (st = check_rows("k", k, g.sk, dtype)) || (st = check_rows("v", v, g.sv, dtype)) ||
      (st = check_rows("out", out, g.so, dtype)))
    return st;
  if (!log_decay || !state) return fail(COTT_ERR_NULL, "null pointer: %s", state ? "log_decay" : "state");
  if ((st = check_state("state", state))) return st;
  DeviceScope scope(state);
  COTT_CUDA_TRY(scope.status());
  StepArgs a = {};
  a.state = state, a.q = q, a.k = k, a.v = v, a.gate = log_decay, a.out = out;
  a.sq = g.sq, a.sk = g.sk, a.sv = g.sv, a.so = g.so, a.sg = g.sg, a.H = H, a.T = T, a.gate_f32 = g.gate_f32;
  const long n = (long)B * H;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case COTT_F32: return run_step<float>(a, D, n, s);
    case COTT_F16: return run_step<__half>(a, D, n, s);
    default: return run_step<__nv_bfloat16>(a, D, n, s);
  }
}

}  // extern "C"
