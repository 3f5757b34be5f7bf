"""The gated scan over sequences that are walked in segments of several chunks, with states that reach from one segment into the next,
against a chunked form in fp64."""
import pytest
import torch

import gated_oracle as O
from test_gated_scan_gpu import NAMES, _inputs, _tol


def _chunked(q, k, v, g, keep=None, init=None, C=64):
    """(out, final state [B, H, value, key]) of the recurrence in fp64, 64 positions at a time."""
    B, H, N, D = q.shape
    g = g.clamp(min=-1000.0)  # (e^-1000 = 0, and differences of sums of it are numbers)
    if keep is not None:
        m = keep[:, None, :, None].to(q.dtype)
        q, k, v, g = q * m, k * m, v * m, g * m[..., 0]
    S = q.new_zeros(B, H, D, D) if init is None else init.mT
    outs = []
    for a in range(0, N, C):
        Q, K, V, G = q[:, :, a:a + C], k[:, :, a:a + C], v[:, :, a:a + C], g[:, :, a:a + C].cumsum(-1)
        W = (G[..., :, None] - G[..., None, :]).tril().exp().tril()
        outs.append(G.exp()[..., None] * (Q @ S) + (Q @ K.mT * W) @ V)
        S = G[..., -1].exp()[..., None, None] * S + ((G[..., -1:] - G).exp()[..., None] * K).mT @ V
    return torch.cat(outs, 2), S.mT


@pytest.mark.parametrize("form", ["plain", "masked", "docs", "init"])
def test_the_chunked_form_is_the_recurrence(form):
    x = _inputs(2, 2, 150, 32, torch.float64, seed=50, masked=form == "masked", docs=form == "docs", init=form == "init")
    q, k, v, g, keep, st = (t if t is None or t.dtype == torch.bool else t.double() for t in x[:6])
    for a, b in zip(_chunked(q, k, v, g, keep, st), O.gated_scan(q, k, v, g, keep, st)):
        assert O.rel(a, b) < 1e-12


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["plain", "masked", "docs", "init", "init_masked"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", [(1, 24, 4100, 64), (1, 12, 4100, 128), (2, 12, 2900, 64), (1, 3, 4100, 64)])
def test_segments_of_several_chunks(shape, dtype, form):
    """16-bit types: 24 walks over 33 chunks are six segments, the last one shorter; (1, 3, ..) is a segment per chunk.  The slowest
    gates lose a factor of e in 2000 positions, several segments.  A copy of a state is rounded twice here (once as the sum of its
    segment, once with the state before that added), within the four half steps that the tolerance has."""
    q, k, v, g, keep, st, do, dst = _inputs(*shape, dtype, seed=51 + sum(shape), masked="masked" in form, init="init" in form)
    H, N = shape[1:3]
    r = torch.Generator().manual_seed(52)
    g = -(torch.logspace(-3.3, -1, H).view(1, H, 1) * (0.5 + torch.rand(shape[:3], generator=r)))
    if form == "docs":
        g[:, :, [700, 701, 2048, 2500]] = float("-inf")
    g = g.to(dtype)
    from cottention_transformer_b200 import gated_scan
    x = [t.cuda() for t in (q, k, v, g)] + ([] if st is None else [st.cuda()])
    kp = None if keep is None else keep.cuda()
    res = []
    for fn, cast in ((lambda *t: gated_scan(*t[:4], keep=kp, initial_state=t[4] if len(t) > 4 else None, return_state=True), lambda t: t),
                     (lambda *t: _chunked(*t[:4], kp, t[4] if len(t) > 4 else None), lambda t: t.double())):
        leaf = [cast(t).detach().requires_grad_() for t in x]
        out, final = fn(*leaf)
        outs, grads = ((out,), (do,)) if form in ("plain", "masked") else ((out, final), (do, dst))
        res.append((out, final, *torch.autograd.grad(outs, leaf, [cast(t.cuda()) for t in grads])))
    for name, a, b in zip(NAMES, *res):
        if name == "dg" and st is None:
            b = b.clone()
            b[:, :, 0] = 0  # (nothing is there that the first gate could decay)
        assert torch.isfinite(a).all() and O.rel(a, b) <= _tol(name, dtype), (name, O.rel(a, b), _tol(name, dtype))
