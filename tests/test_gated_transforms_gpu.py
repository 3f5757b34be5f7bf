"""The gated scan, its step and the q/k norm under traces, transforms, forward-mode differentiation, modes, compilation and hooks: run as
they are or refused, never dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fw

pytestmark = pytest.mark.gpu
D = 64


def _x(T, seed=0, dtype=torch.bfloat16):
    r = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(1, 2, T, D, device="cuda", generator=r).to(dtype) for _ in range(3))
    return q, k, v, -torch.rand(1, 2, T, device="cuda", generator=r).to(dtype)


def _state(seed=1):
    return torch.randn(1, 2, D, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _functions():
    """name -> a function of q alone."""
    from cottention_transformer_b200 import GatedScanState, gated_scan, gated_scan_step, qk_norm_rotary
    _, k, v, g = _x(50)
    w, s, st = torch.rand(D, device="cuda"), torch.rand(50, 16, device="cuda"), _state()  # (drawn here: a trace would draw again)
    return {
        "scan": lambda a: gated_scan(a, k, v, g),
        "scan_with_states": lambda a: torch.cat([t.flatten().float() for t in gated_scan(a, k, v, g, initial_state=st, return_state=True)]),
        "norm": lambda a: qk_norm_rotary(a, k, w, w, rotary=(s, 1 - s))[0],
        "prefill": lambda a: GatedScanState(1, 2, D).prefill(a, k, v, g),
        "step": lambda a: gated_scan_step(st.clone(), a, k, v, g),
    }


NAMES = ["scan", "scan_with_states", "norm", "prefill", "step"]


@pytest.mark.parametrize("name", NAMES)
def test_traces_run_the_operators(name):
    f = _functions()[name]
    a, b = _x(50, 2)[0], _x(50, 3)[0]
    traced = torch.jit.trace(f, (a,), check_trace=False)
    assert torch.equal(traced(a), f(a)) and torch.equal(traced(b), f(b))


def test_a_traced_step_advances_its_state():
    from cottention_transformer_b200 import gated_scan_step
    x, y = _x(1, 4), _x(1, 5)
    state, other = torch.zeros(1, 2, D, D, device="cuda"), torch.zeros(1, 2, D, D, device="cuda")
    traced = torch.jit.trace(lambda *t: gated_scan_step(state, *t), x, check_trace=False)
    state.zero_()
    for t in (x, y, x):
        assert torch.equal(traced(*t), gated_scan_step(other, *t)) and torch.equal(state, other)


@pytest.mark.parametrize("binding", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_transforms_are_refused(name, binding, monkeypatch):
    from cottention_transformer_b200 import _binding
    if not binding:
        monkeypatch.setattr(_binding, "module", lambda: None)
    f, a = _functions()[name], _x(50, 2)[0]
    with fw.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        f(fw.make_dual(a, a))
    with fw.dual_level():
        assert fw.unpack_dual(f(a)).tangent is None
    for call in (lambda: torch.func.vmap(f)(a[None]), lambda: torch.func.grad(lambda t: f(t).float().sum())(a), lambda: torch.func.jvp(f, (a,), (a,))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_no_transform_reaches_the_state_of_a_refused_step():
    from cottention_transformer_b200 import gated_scan_step
    x, state = _x(1, 4), _state()
    want = state.clone()
    with fw.dual_level():
        for i in range(4):
            with pytest.raises((RuntimeError, NotImplementedError)):
                gated_scan_step(state, *(fw.make_dual(t, t) if i == j else t for j, t in enumerate(x)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            gated_scan_step(fw.make_dual(state, state), *x)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda q: gated_scan_step(state, q, *x[1:]))(x[0][None])
    assert torch.equal(state, want)


def test_a_step_is_not_traced_without_the_operator(monkeypatch):
    from cottention_transformer_b200 import _binding
    monkeypatch.setattr(_binding, "module", lambda: None)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(_functions()["step"], (_x(50, 2)[0],), check_trace=False)


@pytest.mark.parametrize("name,op", [("scan", "gated_fwd"), ("scan_with_states", "gated_fwd"), ("norm", "qk_norm_fwd"), ("prefill", "gated_fwd"), ("step", "gated_step")])
def test_dispatch_modes_see_the_operators(name, op):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            names.append(str(func))
            return func(*args, **(kwargs or {}))

    names, f, a = [], _functions()[name], _x(50, 2)[0]
    with Seen():
        out = f(a)
    assert f"cottention_b200.{op}.default" in names and torch.equal(out, f(a))
    if name in ("scan", "scan_with_states", "norm"):
        leaf = a.clone().requires_grad_()
        with Seen():
            out = f(leaf)
        do = torch.randn_like(out)
        assert torch.equal(torch.autograd.grad(out, leaf, do)[0], torch.autograd.grad(f(leaf), leaf, do)[0])


def test_saved_tensor_hooks_and_modified_inputs():
    from cottention_transformer_b200 import gated_scan, qk_norm_rotary
    x = _x(50)
    do = torch.randn_like(x[0])
    w = torch.rand(D, device="cuda")
    for call, inputs in ((gated_scan, x), (lambda *t: qk_norm_rotary(*t)[0], (x[0], x[1], w, w.clone()))):
        leaf, packed = [t.clone().requires_grad_() for t in inputs], []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t.shape) or t.clone(), lambda t: t):
            out = call(*leaf)
        assert len(packed) >= 4
        a, b = torch.autograd.grad(out, leaf, do), torch.autograd.grad(call(*leaf), leaf, do)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        q = leaf[0].detach().clone().requires_grad_() * 1
        out = call(q, *leaf[1:])
        q.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.backward(do)


@pytest.mark.parametrize("name", NAMES)
def test_compiled_functions_run_the_operators(name):
    f, a = _functions()[name], _x(50, 2)[0]
    torch._dynamo.reset()
    compiled = torch.compile(lambda t: f(t * 1) * 2, backend="aot_eager")
    assert torch.equal(compiled(a), f(a) * 2)
    if name not in ("prefill", "step"):
        res = []
        for call in (compiled, lambda t: f(t * 1) * 2):
            leaf = a.clone().requires_grad_()
            res.append(torch.autograd.grad(call(leaf).float().square().sum(), leaf)[0])
        assert torch.equal(*res)
