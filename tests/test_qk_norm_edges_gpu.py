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
