"""The decode step under traces, transforms and forward-mode differentiation: refused, not dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_decode_step_is_refused_where_it_would_be_dropped(dtype):
    from cottention_transformer_b200 import CosAttnDecodeState
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(1, 2, 3, 64, device="cuda", generator=g).to(dtype) for _ in range(3))
    nc = torch.full((2,), 0.5, device="cuda")
    st, other = CosAttnDecodeState(1, 2, 64), CosAttnDecodeState(1, 2, 64)
    step = lambda a: st.step(a, k, v, nc)  # noqa: E731
    calls = [lambda: torch.jit.trace(step, (q,), check_trace=False), lambda: torch.func.vmap(step)(q[None]),
             lambda: torch.func.grad(lambda a: step(a).float().sum())(q), lambda: torch.func.jvp(step, (q,), (q,))]
    for call in calls:
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    with fw.dual_level():
        for x in ((fw.make_dual(q, q), k, v, nc), (q, k, fw.make_dual(v, v), nc), (q, k, v, fw.make_dual(nc, nc))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                st.step(*x)
        assert st.cur_s == 1 and (st.state == 0).all()  # nothing has happened
        assert torch.equal(st.step(q, k, v, nc), other.step(q, k, v, nc))
    assert torch.equal(st.state, other.state) and st.cur_s == other.cur_s == 4
