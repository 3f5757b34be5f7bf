"""RMS norm of every head of q and k with a learned weight, and the rotary embedding, in one pass over each."""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _binding, _lib
from .gated import _DIMS, _DTYPES, rows16, strides3


def _check(q, k, q_weight, k_weight):
    if not (q.is_cuda and k.is_cuda and q_weight.is_cuda and k_weight.is_cuda):
        raise RuntimeError("qk_norm_rotary needs CUDA tensors (there is no CPU path)")
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"[B, H, N, D] tensors expected, got {q.dim()} and {k.dim()} dimensions")
    if q.dtype not in _DTYPES or k.dtype != q.dtype:
        raise RuntimeError(f"qk_norm_rotary takes float32, float16 or bfloat16 tensors of one type, got {q.dtype} and {k.dtype}")
    B, _, N, D = q.shape
    if k.shape[0] != B or k.shape[2] != N or k.shape[3] != D:
        raise RuntimeError(f"q and k must agree in all but their heads, got {list(q.shape)} and {list(k.shape)}")
    if D not in _DIMS:
        raise RuntimeError(f"qk_norm_rotary supports head dims 32, 64 and 128 (got {D})")
    for w in (q_weight, k_weight):
        if tuple(w.shape) != (D,) or w.dtype not in (torch.float32, q.dtype) or w.dtype != q_weight.dtype:
            raise RuntimeError(f"the weights must be [D] = [{D}], both in float32 or both of the tensors' type, got {list(w.shape)} in {w.dtype}")
    if not (k.device == q.device and q_weight.device == q.device and k_weight.device == q.device):
        raise RuntimeError("q, k and the weights must be on one device")


def _tables(rotary, q):
    if rotary is None:
        return None, None
    if (rotary[0] is None) != (rotary[1] is None):
        raise RuntimeError("rotary takes the sines and the cosines, one of them is missing")
    if rotary[0] is None:
        return None, None
    sin, cos = (t.to(device=q.device, dtype=torch.float32).contiguous() for t in rotary)
    B, _, N, D = q.shape
    rot = 2 * sin.shape[-1]
    if sin.shape != cos.shape or sin.dim() not in (2, 3) or sin.shape[-2] != N or (sin.dim() == 3 and sin.shape[0] not in (1, B)):
        raise RuntimeError("sin / cos must be [N, rot/2] or [B, N, rot/2]")
    if rot < 8 or rot % 8 or rot > D:
        raise RuntimeError(f"the rotary dim must be a multiple of 8 and at most the head dim (got {rot}, {D})")
    return tuple(t if t.data_ptr() % 16 == 0 else t.clone() for t in (sin, cos))


def _rotary(sin, cos, N):
    if sin is None:
        return None
    per_batch = sin.dim() == 3 and sin.shape[0] > 1
    return ctypes.byref(_lib.CottRotaryTables(_lib.ptr(sin), _lib.ptr(cos), 2 * sin.shape[-1], N * sin.shape[-1] if per_batch else 0))


def _layout(q, k, q_out, k_out, dq=None, dk=None):
    lay = _lib.CottNormLayout()
    for name, t in zip(("q", "k", "q_out", "k_out", "dq", "dk"), (q, k, q_out, k_out, dq, dk)):
        if t is not None:
            setattr(lay, name, strides3(t))
    return ctypes.byref(lay)


class _QKNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, sin, cos, eps):
        q, k, qw, kw = rows16(q), rows16(k), q_weight.contiguous(), k_weight.contiguous()
        ctx.save_for_backward(q, k, qw, kw, sin, cos)
        ctx.eps = eps
        ops = _binding.visible_ops()
        if ops is not None:
            return ops.qk_norm_fwd(q, k, qw, kw, sin, cos, eps)
        B, Hq, N, D = q.shape
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
        with torch.cuda.device(q.device):
            st = _lib.lib().cott_qk_norm_fwd(_lib.ptr(q), _lib.ptr(k), _lib.ptr(qw), _lib.ptr(kw), _rotary(sin, cos, N), _lib.ptr(q_out),
                                             _lib.ptr(k_out), _layout(q, k, q_out, k_out), B, Hq, k.shape[1], N, D, eps, _lib.DTYPE_CODE[q.dtype],
                                             _lib.DTYPE_CODE[qw.dtype], _lib.stream_ptr(q.device))
        _lib.check(st, "cott_qk_norm_fwd")
        return q_out, k_out

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, qw, kw, sin, cos = ctx.saved_tensors
        B, Hq, N, D = q.shape
        dq_out, dk_out = rows16(dq_out.to(q.dtype)), rows16(dk_out.to(q.dtype))
        dq, dk, dqw, dkw = torch.empty_like(q), torch.empty_like(k), torch.empty_like(qw), torch.empty_like(kw)
        L = _lib.lib()
        with torch.cuda.device(q.device):
            ws = torch.empty(max(L.cott_qk_norm_workspace_bytes(B, Hq, k.shape[1], N, D), 16), dtype=torch.uint8, device=q.device)
            st = L.cott_qk_norm_bwd(_lib.ptr(q), _lib.ptr(k), _lib.ptr(qw), _lib.ptr(kw), _rotary(sin, cos, N), _lib.ptr(dq_out), _lib.ptr(dk_out),
                                    _lib.ptr(ws), _lib.ptr(dq), _lib.ptr(dk), _lib.ptr(dqw), _lib.ptr(dkw),
                                    _layout(q, k, dq_out, dk_out, dq, dk), B, Hq, k.shape[1], N, D, ctx.eps, _lib.DTYPE_CODE[q.dtype],
                                    _lib.DTYPE_CODE[qw.dtype], _lib.stream_ptr(q.device))
        _lib.check(st, "cott_qk_norm_bwd")
        return dq, dk, dqw, dkw, None, None, None


def qk_norm_rotary(q, k, q_weight, k_weight, rotary=None, eps=1e-6):
    """``Rot(x / sqrt(mean(x^2) + eps) * weight)`` for every head of q and of k; returns the two results, in the memory order of
    q and k.

    q: ``[B, Hq, N, D]``, k: ``[B, Hk, N, D]`` CUDA tensors of one type (float32, float16, bfloat16), D = 32, 64 or 128; views, such as
    the q and k of a packed ``[B, N, 3, H, D]`` projection, are read where they lie when their rows are 16-byte aligned.
    q_weight, k_weight: ``[D]``, float32 or of the tensors' type.  ``rotary=(sin, cos)``: fp32 ``[N, rot/2]`` or ``[B, N, rot/2]``, as
    ``rotary_packed_`` takes them ("rotate every two" on the first rot elements, a multiple of 8); None: no rotation.
    fp32 arithmetic, one rounding at the end.  Differentiable once in q, k and the weights, whose gradients are fp32 sums in a
    fixed order.  (Weights of ``1 / sqrt(D)`` make it the L2 normalisation of cosine attention.)"""
    m = _binding.autograd()
    if m is not None:
        sin, cos = (None, None) if rotary is None else rotary
        return tuple(m.qk_norm_rotary(q, k, q_weight, k_weight, sin, cos, float(eps)))
    _check(q, k, q_weight, k_weight)
    return _QKNormRotary.apply(q, k, q_weight, k_weight, *_tables(rotary, q), float(eps))
