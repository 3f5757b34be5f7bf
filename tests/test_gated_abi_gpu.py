"""What the C ABI of the gated scan, its step and the q/k norm allows beside what the Python entry points do: results over inputs, dense
tensors without a layout, a backward that runs twice, as many sequences as no grid dimension but the first one holds."""
import ctypes

import pytest
import torch

import gated_oracle as O
from test_gated_scan_gpu import _inputs, _tol, _truth

pytestmark = pytest.mark.gpu


def _lib():
    from cottention_transformer_b200 import _lib as L
    return L


def _buffer(n):
    return torch.full((max(n, 16),), 0xFF, dtype=torch.uint8, device="cuda")  # (as fp32 or 16 bits: NaN)


@pytest.mark.parametrize("dtype,shape", [(torch.float32, (2, 3, 150, 64)), (torch.bfloat16, (2, 3, 150, 32)), (torch.bfloat16, (2, 80, 150, 64)),
                                         (torch.float16, (1, 2, 1700, 64)), (torch.bfloat16, (1, 2, 1500, 128))])
def test_the_state_is_advanced_in_place_and_the_backward_runs_twice(dtype, shape):
    """initial_state is final_state, no layout, buffers full of NaN before the call."""
    m, (B, H, N, D) = _lib(), shape
    L, P, code = m.lib(), m.ptr, m.DTYPE_CODE[dtype]
    q, k, v, g, keep, st, do, dst = (t if t is None else t.cuda() for t in _inputs(*shape, dtype, seed=70, masked=True, init=True))
    from cottention_transformer_b200 import gated_scan
    leaf = [t.requires_grad_() for t in (q, k, v, g)] + [st.clone().requires_grad_()]
    want_out, want_state = gated_scan(*leaf[:4], keep=keep, initial_state=leaf[4], return_state=True)
    want = torch.autograd.grad((want_out, want_state), leaf, (do, dst))
    kp, out, s = keep.to(torch.uint8), torch.empty_like(v), torch.cuda.current_stream().cuda_stream
    states, ws = _buffer(L.cott_gated_scan_states_bytes(B, H, N, D, code)), _buffer(L.cott_gated_scan_workspace_bytes(B, H, N, D, code, 0))
    m.check(L.cott_gated_scan_fwd(P(q), P(k), P(v), P(g), P(kp), P(st), P(out), P(st), P(states), P(ws), None, B, H, N, D, code, code, s), "fwd")
    assert torch.equal(out, want_out) and torch.equal(st, want_state)
    for _ in range(2):
        ws = _buffer(L.cott_gated_scan_workspace_bytes(B, H, N, D, code, 1))
        got = [torch.full_like(t, float("nan")) for t in want]
        dq, dk, dv, dg, dinit = got
        m.check(L.cott_gated_scan_bwd(P(q), P(k), P(v), P(g), P(kp), 1, P(states), P(do), P(dst), P(ws), P(dq), P(dk), P(dv), P(dg), P(dinit), None, B, H, N, D,
                                      code, code, s), "bwd")
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    m.check_device_status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hk,N", [(2, 2, 3), (4, 4, 900), (4, 1, 900), (8, 8, 2500)])
def test_the_norm_over_its_inputs(dtype, Hq, Hk, N):
    """q_out is q, k_out is k; dq is dq_out, dk is dk_out; no layout."""
    m, B, D = _lib(), 2, 64
    L, P, code = m.lib(), m.ptr, m.DTYPE_CODE[dtype]
    from cottention_transformer_b200 import qk_norm_rotary
    r = torch.Generator(device="cuda").manual_seed(71)
    q, dq = (torch.randn(B, Hq, N, D, device="cuda", generator=r).to(dtype) for _ in range(2))
    k, dk = (torch.randn(B, Hk, N, D, device="cuda", generator=r).to(dtype) for _ in range(2))
    w = 1 + 0.1 * torch.randn(2, D, device="cuda", generator=r)
    ang = torch.rand(N, 16, device="cuda", generator=r)
    sin, cos = ang.sin(), ang.cos()
    leaf = [t.clone().requires_grad_() for t in (q, k, w[0], w[1])]
    out = qk_norm_rotary(*leaf, rotary=(sin, cos))
    want = torch.autograd.grad(out, leaf, (dq, dk))
    tab = ctypes.byref(m.CottRotaryTables(P(sin), P(cos), 32, 0))
    s, ws, dw = torch.cuda.current_stream().cuda_stream, _buffer(L.cott_qk_norm_workspace_bytes(B, Hq, Hk, N, D)), torch.empty_like(w)
    m.check(L.cott_qk_norm_bwd(P(q), P(k), P(w[0]), P(w[1]), tab, P(dq), P(dk), P(ws), P(dq), P(dk), P(dw[0]), P(dw[1]), None, B, Hq, Hk, N, D, 1e-6, code, 0, s), "bwd")
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dw[0], dw[1]), want))
    m.check(L.cott_qk_norm_fwd(P(q), P(k), P(w[0]), P(w[1]), tab, P(q), P(k), None, B, Hq, Hk, N, D, 1e-6, code, 0, s), "fwd")
    assert torch.equal(q, out[0]) and torch.equal(k, out[1])


@pytest.mark.parametrize("dtype,D", [(torch.float32, 32), (torch.bfloat16, 64), (torch.float16, 128)])
def test_many_sequences(dtype, D):
    """More (batch, head) pairs than the second and third dimension of a grid take."""
    from cottention_transformer_b200 import gated_scan, gated_scan_step, qk_norm_rotary
    B, H, N = 23000, 3, 2
    few = _inputs(7, H, N, D, dtype, seed=72, init=True)
    at = torch.arange(B) % 7
    q, k, v, g, _, st, do, dst = (t if t is None else t[at].cuda() for t in few)
    leaf = [t.requires_grad_() for t in (q, k, v, g, st)]
    out, state = gated_scan(*leaf[:4], initial_state=st, return_state=True)
    got = (out, state, *torch.autograd.grad((out, state), leaf, (do, dst)))
    want = _truth(*few)
    names = ("out", "state", "dq", "dk", "dv", "dg", "dinit")
    for name, a, b in zip(names, got, want):
        a = a.detach()
        assert all(torch.equal(a[i:i + 7], a[:7]) for i in (7, 7 * 1000, 7 * 3000, B // 7 * 7 - 7))  # the same sequences, the same bits
        assert (a[:B // 7 * 7].view(-1, 7, *a.shape[1:]) == a[None, :7]).all()
        assert O.rel(a[:7], b) <= (_tol(name, dtype) if name != "dg" else 2 * _tol(name, dtype)), name
    del got, leaf, out, state
    with torch.no_grad():
        s = st.detach().clone()
        o = gated_scan_step(s, q, k, v, g)
        assert (s[:B // 7 * 7].view(-1, 7, *s.shape[1:]) == s[None, :7]).all() and O.rel(s[:7], want[1]) <= 1e-6 and O.rel(o[:7], want[0]) <= 1e-6 + torch.finfo(dtype).eps / 2
        w = torch.ones(D, device="cuda")
        a, b = qk_norm_rotary(q, k, w, w)
        assert (a[:B // 7 * 7].view(-1, 7, *a.shape[1:]) == a[None, :7]).all() and O.rel(a[:7], O.qk_norm(few[0].double(), torch.ones(D).double())) <= 4e-6 + torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("compiled", [True, False])
def test_odd_views_of_gates_and_masks(dtype, compiled, monkeypatch):
    """Gates at an odd offset and with gaps, masks as a transposed, an expanded and a byte tensor with any non-zero value."""
    from cottention_transformer_b200 import _binding, gated_scan
    if not compiled:
        monkeypatch.setattr(_binding, "autograd", lambda: None)
    q, k, v, g, keep, _, do, _ = (t if t is None else t.cuda() for t in _inputs(2, 2, 150, 64, dtype, seed=73, masked=True))

    def run(gate, mask):
        leaf = [t.detach().requires_grad_() for t in (q, k, v)]
        gate = gate.requires_grad_()
        out = gated_scan(*leaf, gate, keep=mask)
        return out, *torch.autograd.grad(out, (*leaf, gate), do)

    gaps = torch.full((2, 2, 301), float("nan"), dtype=dtype, device="cuda")
    gaps[:, :, 1::2] = g
    want = run(g.clone(), keep)
    for mask in (keep.t().contiguous().t(), keep.to(torch.uint8) * 254):
        assert all(torch.equal(a, b) for a, b in zip(run(gaps[:, :, 1::2].detach(), mask), want))
    one = keep[1:].expand(2, -1)
    assert all(torch.equal(a, b) for a, b in zip(run(g.clone(), one), run(g.clone(), one.contiguous())))
