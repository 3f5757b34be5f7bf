"""The q/k norm with rotation at the edges of its calls."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("compiled", [True, False])
def test_half_a_pair_of_tables_is_refused(compiled, monkeypatch):
    from cottention_transformer_b200 import _binding, qk_norm_rotary
    if not compiled:
        monkeypatch.setattr(_binding, "autograd", lambda: None)
    q, w, s = torch.randn(2, 3, 10, 64, device="cuda"), torch.ones(64, device="cuda"), torch.zeros(10, 16, device="cuda")
    for grad in (False, True):
        x = q.clone().requires_grad_(grad)
        for pair in ((s, None), (None, s)):
            with pytest.raises(RuntimeError, match="missing"):
                qk_norm_rotary(x, x, w, w, rotary=pair)
        assert torch.equal(qk_norm_rotary(x, x, w, w, rotary=(None, None))[0], qk_norm_rotary(x, x, w, w)[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 16, 16, 701, 64, 32, True), (1, 12, 12, 1801, 128, 64, False), (3, 16, 16, 2001, 32, 8, False),
                                   (2, 16, 4, 1501, 64, 64, False), (2, 4, 12, 1501, 128, 32, True)])
def test_several_rounds_of_rows(shape, dtype, monkeypatch):
    """More rows than the CTAs take at once, in both passes and with as many, fewer and more key than query heads; the last round is not
    full.  The weights' gradients are sums over the rounds, and of q and of k apart."""
    import gated_oracle as O
    from test_qk_norm_gpu import _inputs, _run, _tol, _truth
    B, Hq, Hk, N, D, rot, batched = shape
    for wdtype in {torch.float32, dtype}:
        x = _inputs(B, Hq, Hk, N, D, dtype, wdtype, rot, batched, seed=60 + sum(shape))
        want = _truth(*x)
        for got in O.both_routes(monkeypatch.context(), lambda: _run(*x, view=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))):
            for name, a, b in zip(("q", "k", "dq", "dk", "dqw", "dkw"), got, want):
                assert a.shape == b.shape and O.rel(a, b) <= _tol(name, dtype, wdtype), (name, O.rel(a, b))
