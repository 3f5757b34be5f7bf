"""The gated causal scan: linear attention with a learned decay per head and position.

    S_t = e^(log_decay_t) S_(t-1) + k_t v_t^T          out_t = S_t^T q_t

``gated_scan`` is the form for whole sequences (training, prompts), ``gated_scan_step`` the form for new tokens, which updates
the states in place, and ``GatedScanState`` holds the states of a batch between the two.  With ``log_decay`` = 0 it is the scan
that ``CustomAttention`` computes.  Like that one it takes q and k as they come; ``qk_norm_rotary`` is the pass before it.

float32 is computed in fp32 throughout (``csrc/gated_simt.cuh``); float16 / bfloat16 with head dim 64 or 128 on the tensor cores with
fp32 sums and states (``csrc/gated_tc.cuh``).  There is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _binding, _lib

_DTYPES = (torch.float32, torch.float16, torch.bfloat16)
_DIMS = (32, 64, 128)


def _check(what, q, k, v, log_decay):
    if not (q.is_cuda and k.is_cuda and v.is_cuda and log_decay.is_cuda):
        raise RuntimeError(f"{what} needs CUDA tensors (there is no CPU path)")
    if q.dim() != 4:
        raise ValueError(f"[B, H, N, D] tensors expected, got {q.dim()} dimensions")
    if k.shape != q.shape or v.shape != q.shape:
        raise RuntimeError(f"q, k and v must have the same shape, got {list(q.shape)}, {list(k.shape)} and {list(v.shape)}")
    if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError(f"{what} takes float32, float16 or bfloat16 tensors of one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    if q.shape[-1] not in _DIMS:
        raise RuntimeError(f"{what} supports head dims 32, 64 and 128 (got {q.shape[-1]})")
    if log_decay.shape != q.shape[:3] or log_decay.dtype not in (torch.float32, q.dtype):
        raise RuntimeError(f"log_decay must be [B, H, N] = {list(q.shape[:3])} in float32 or the tensors' type, got {list(log_decay.shape)} in {log_decay.dtype}")
    if not (k.device == q.device and v.device == q.device and log_decay.device == q.device):
        raise RuntimeError("q, k, v and log_decay must be on one device")


def _check_keep(keep, q):
    if keep is not None and (keep.dtype not in (torch.bool, torch.uint8) or tuple(keep.shape) != (q.shape[0], q.shape[2]) or keep.device != q.device):
        raise RuntimeError(f"keep must be a bool [B, N] = {[q.shape[0], q.shape[2]]} tensor on the tensors' device")


def _check_state(name, state, q):
    B, H, _, D = q.shape
    if state is not None and (state.dtype != torch.float32 or tuple(state.shape) != (B, H, D, D) or state.device != q.device):
        raise RuntimeError(f"{name} must be a float32 [B, H, D, D] = {[B, H, D, D]} tensor on the tensors' device")


def rows16(t):
    """``t`` as the kernels read it: rows contiguous, base and strides in multiples of 16 bytes; else a dense copy."""
    unit = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(n == 1 or (s > 0 and s % unit == 0) for n, s in zip(t.shape[:-1], t.stride()[:-1])):
        return t
    c = t.contiguous()
    return c if c.data_ptr() % 16 == 0 else c.clone()


def strides3(t):
    return _lib.CottStrides(*(0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])))


def _state16(t):
    if t is None:
        return None
    c = t.contiguous()
    return c if c.data_ptr() % 16 == 0 else c.clone()


def _layout(q, k, v, out, gate, dq=None, dk=None, dv=None, dgate=None):
    lay = _lib.CottGatedLayout()
    for name, t in zip(("q", "k", "v", "out", "gate", "dq", "dk", "dv", "dgate"), (q, k, v, out, gate, dq, dk, dv, dgate)):
        if t is not None:
            setattr(lay, name, strides3(t))
    return ctypes.byref(lay)


def _bytes(n, device):
    return torch.empty(max(n, 16), dtype=torch.uint8, device=device)


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, keep, initial_state, return_state):
        q, k, v, init = rows16(q), rows16(k), rows16(v), _state16(initial_state)
        kp = None if keep is None else keep.to(torch.uint8, memory_format=torch.contiguous_format, copy=True)
        ctx.save_for_backward(q, k, v, log_decay)
        ctx.kp, ctx.with_initial = kp, init is not None
        ctx.set_materialize_grads(False)
        ops = _binding.visible_ops()
        if ops is not None:
            out, final, ctx.states = ops.gated_fwd(q, k, v, log_decay, kp, init, return_state)
            return (out, final) if return_state else out
        B, H, N, D = q.shape
        code, gcode = _lib.DTYPE_CODE[q.dtype], _lib.DTYPE_CODE[log_decay.dtype]
        L = _lib.lib()
        out = torch.empty_like(v)
        final = torch.empty(B, H, D, D, dtype=torch.float32, device=q.device) if return_state else None
        with torch.cuda.device(q.device):
            states = _bytes(L.cott_gated_scan_states_bytes(B, H, N, D, code), q.device)
            ws = _bytes(L.cott_gated_scan_workspace_bytes(B, H, N, D, code, 0), q.device)
            st = L.cott_gated_scan_fwd(_lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(log_decay), _lib.ptr(kp), _lib.ptr(init), _lib.ptr(out),
                                       _lib.ptr(final), _lib.ptr(states), _lib.ptr(ws), _layout(q, k, v, out, log_decay), B, H, N, D, code, gcode,
                                       _lib.stream_ptr(q.device))
        _lib.check(st, "cott_gated_scan_fwd")
        ctx.states = states
        return (out, final) if return_state else out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dfinal=None):
        q, k, v, log_decay = ctx.saved_tensors
        B, H, N, D = q.shape
        dout = rows16(torch.zeros_like(v) if dout is None else dout.to(q.dtype))
        dfinal = _state16(dfinal)
        code, gcode = _lib.DTYPE_CODE[q.dtype], _lib.DTYPE_CODE[log_decay.dtype]
        L = _lib.lib()
        dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(log_decay)
        dinit = torch.empty(B, H, D, D, dtype=torch.float32, device=q.device) if ctx.needs_input_grad[5] else None
        with torch.cuda.device(q.device):
            ws = _bytes(L.cott_gated_scan_workspace_bytes(B, H, N, D, code, 1), q.device)
            st = L.cott_gated_scan_bwd(_lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(log_decay), _lib.ptr(ctx.kp), int(ctx.with_initial),
                                       _lib.ptr(ctx.states), _lib.ptr(dout), _lib.ptr(dfinal), _lib.ptr(ws), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dv),
                                       _lib.ptr(dg), _lib.ptr(dinit), _layout(q, k, v, dout, log_decay, dq, dk, dv, dg), B, H, N, D, code, gcode,
                                       _lib.stream_ptr(q.device))
        _lib.check(st, "cott_gated_scan_bwd")
        return dq, dk, dv, dg, None, dinit, None


def gated_scan(q, k, v, log_decay, keep=None, initial_state=None, return_state=False):
    """Causal linear attention with a decay: ``S_t = e^(log_decay_t) S_(t-1) + k_t v_t^T``, ``out_t = S_t^T q_t``.

    q, k, v: ``[B, H, N, D]`` CUDA tensors of one type (float32, float16, bfloat16), D = 32, 64 or 128; views (a head split of a
    projection) are read where they lie when their rows are 16-byte aligned.  log_decay: ``[B, H, N]``, float32 or of the same type,
    values <= 0 (``logsigmoid`` of a projection); ``-inf`` drops the state, as at the first position of a packed document.
    keep: optional bool ``[B, N]``, True = un-masked: a masked position contributes nothing, lets the state pass unchanged, and its
    output and gradients are zero; what its rows hold does not matter.
    initial_state: optional float32 ``[B, H, D, D]``, value index first.  Returns ``out``, in the memory order of ``v``, or
    ``(out, state)`` with ``return_state``: the state after the last position, in fp32.

    Differentiable once in q, k, v, log_decay and initial_state (``return_state`` included).  A gate of ``-inf`` (or below about -88,
    where its decay is zero in float32) and the first gate of a sequence without an initial state have no gradient.

    16-bit tensors at head dims 64 and 128: beside its own rounding a result carries those of the decayed scores and of the state's
    copy that multiplies rows (0.6 half steps of the type in the 2-norm, 0.43 by the own rounding alone); the gradient of log_decay up
    to 0.8, also where log_decay is float32.  The states themselves are fp32.  An infinity or NaN in an unmasked row reaches other
    rows of its 128 positions, also those that do not see it.  float16: a state entry, or a score (``q.k``, in the backward
    ``dout.v``) times its decay, beyond 65504 overflows, and what is smaller than the type's smallest step (weights of less than 2^-24
    within 128 positions) is lost."""
    m = _binding.autograd()
    if m is not None:
        r = m.gated_scan(q, k, v, log_decay, keep, initial_state, bool(return_state))
        return tuple(r) if return_state else r[0]
    _check("gated_scan", q, k, v, log_decay)
    _check_keep(keep, q)
    _check_state("initial_state", initial_state, q)
    return _GatedScan.apply(q, k, v, log_decay, keep, initial_state, bool(return_state))


def gated_scan_step(state, q, k, v, log_decay):
    """New tokens of the same recurrence: advances ``state`` (float32 ``[B, H, D, D]``, value index first, contiguous) in place by
    the T >= 1 tokens of q, k, v ``[B, H, T, D]`` and log_decay ``[B, H, T]`` and returns their outputs, in the memory order of
    ``v``.  For generation: not differentiable."""
    m = _binding.autograd()
    if m is not None:
        return m.gated_step(state, q, k, v, log_decay)
    _binding.refuse_transforms("gated_scan_step", state, q, k, v, log_decay)
    ops = _binding.visible_ops()
    if ops is not None:
        return ops.gated_step(state, q, k, v, log_decay)
    _check("gated_scan_step", q, k, v, log_decay)
    _check_state("state", state, q)
    if not state.is_contiguous() or state.data_ptr() % 16:
        raise RuntimeError("the state is updated in place: it must be contiguous and 16-byte aligned")
    if state.is_inference() and not torch.is_inference_mode_enabled():
        raise RuntimeError("Inplace update to inference tensor outside InferenceMode is not allowed: the state was made in inference mode")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (state, q, k, v, log_decay)):
        raise RuntimeError("gated_scan_step is not differentiable: use gated_scan, or call it under torch.no_grad()")
    q, k, v = rows16(q), rows16(k), rows16(v)
    B, H, T, D = q.shape
    out = torch.empty_like(v)
    with torch.cuda.device(q.device):
        st = _lib.lib().cott_gated_step(_lib.ptr(state), _lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(log_decay), _lib.ptr(out),
                                        _layout(q, k, v, out, log_decay), B, H, T, D, _lib.DTYPE_CODE[q.dtype], _lib.DTYPE_CODE[log_decay.dtype],
                                        _lib.stream_ptr(q.device))
    _lib.check(st, "cott_gated_step")
    torch.autograd.graph.increment_version(state)
    return out


class GatedScanState:
    """The recurrent states of a batch: what ``CosAttnDecodeState`` is for the cosine form.  (No position is kept: a gated scan
    has none.)"""

    def __init__(self, batch: int, heads: int, d: int, device="cuda"):
        self.state = torch.zeros(batch, heads, d, d, dtype=torch.float32, device=device)

    def reset(self):
        self.state.zero_()

    def prefill(self, q, k, v, log_decay, keep=None):
        """Absorbs a whole prompt, or a further piece of one, in one call; returns its outputs ``[B, H, T, D]``."""
        with torch.no_grad():
            out, state = gated_scan(q, k, v, log_decay, keep=keep, initial_state=self.state, return_state=True)
            self.state.copy_(state)
        return out

    def step(self, q, k, v, log_decay):
        """Advances the states by T >= 1 tokens per sequence; returns their outputs."""
        with torch.no_grad():
            return gated_scan_step(self.state, q, k, v, log_decay)
