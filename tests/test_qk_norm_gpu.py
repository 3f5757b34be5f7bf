"""RMS norm of the heads of q and k with the rotation, forward and backward, against fp64."""
import pytest
import torch

import gated_oracle as O

pytestmark = pytest.mark.gpu


def _tol(name, dtype, wdtype):
    # one rounding of the result, half a step at most; fp32: a row's sum of D squares and a handful of products.  The gradient of a
    # weight is an fp32 sum over all rows, rounded to the weight's type.
    t = wdtype if name in ("dqw", "dkw") else dtype
    return 4e-6 if t == torch.float32 else torch.finfo(t).eps / 2


def _inputs(B, Hq, Hk, N, D, dtype, wdtype, rot, batched, seed):
    r = torch.Generator().manual_seed(seed)
    q, dq = (torch.randn(B, Hq, N, D, generator=r).mul(2).to(dtype) for _ in range(2))
    k, dk = (torch.randn(B, Hk, N, D, generator=r).to(dtype) for _ in range(2))
    qw, kw = ((1 + 0.3 * torch.randn(D, generator=r)).to(wdtype) for _ in range(2))
    tables = None
    if rot:
        a = torch.randn(*((B, N) if batched else (N,)), rot // 2, generator=r) * 3
        tables = (a.sin(), a.cos())
    return q, k, qw, kw, tables, dq, dk


def _truth(q, k, qw, kw, tables, dq, dk):
    leaf = [t.double().requires_grad_() for t in (q, k, qw, kw)]
    tab = (None, None) if tables is None else (t.double() for t in tables)
    sin, cos = tab
    a, b = O.qk_norm(leaf[0], leaf[2], sin, cos), O.qk_norm(leaf[1], leaf[3], sin, cos)
    return a, b, *torch.autograd.grad((a, b), leaf, (dq.double(), dk.double()))


def _run(q, k, qw, kw, tables, dq, dk, view=lambda t: t):
    from cottention_transformer_b200 import qk_norm_rotary
    leaf = [view(t.cuda()).detach().requires_grad_() for t in (q, k)] + [t.cuda().requires_grad_() for t in (qw, kw)]
    a, b = qk_norm_rotary(*leaf, rotary=None if tables is None else tuple(t.cuda() for t in tables))
    return a, b, *torch.autograd.grad((a, b), leaf, (dq.cuda(), dk.cuda()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 32, 0, False), (1, 2, 2, 5, 64, 64, False), (2, 3, 1, 33, 128, 32, True), (3, 4, 4, 129, 64, 8, True),
                                   (2, 16, 4, 300, 64, 64, False), (1, 5, 3, 1000, 128, 128, False), (70, 4, 2, 1, 64, 32, True)])
def test_matches_fp64(shape, dtype, monkeypatch):
    B, Hq, Hk, N, D, rot, batched = shape
    for wdtype in {torch.float32, dtype}:
        x = _inputs(B, Hq, Hk, N, D, dtype, wdtype, rot, batched, seed=sum(shape))
        want = _truth(*x)
        packed = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
        for view in (lambda t: t, packed):
            first = None
            for got in O.both_routes(monkeypatch.context(), lambda: _run(*x, view=view)):
                for name, a, b in zip(("q", "k", "dq", "dk", "dqw", "dkw"), got, want):
                    assert a.shape == b.shape and O.rel(a, b) <= _tol(name, dtype, wdtype), (name, O.rel(a, b))
                assert first is None or all(torch.equal(s, t) for s, t in zip(first, got))
                first = got


def test_views_of_a_packed_projection():
    from cottention_transformer_b200 import qk_norm_rotary
    B, H, N, D = 2, 4, 77, 64
    q, k, qw, kw, tables, dq, dk = _inputs(B, H, H, N, D, torch.bfloat16, torch.float32, 32, True, seed=3)
    want = _truth(q, k, qw, kw, tables, dq, dk)
    qkv = torch.stack([q, k, torch.zeros_like(k)], 2).permute(0, 3, 2, 1, 4).contiguous().cuda().requires_grad_()
    a, b = qk_norm_rotary(qkv[:, :, 0].transpose(1, 2), qkv[:, :, 1].transpose(1, 2), qw.cuda(), kw.cuda(), rotary=tuple(t.cuda() for t in tables))
    assert a.transpose(1, 2).is_contiguous()
    d, = torch.autograd.grad((a, b), qkv, (dq.cuda(), dk.cuda()))
    for name, s, t in zip(("q", "k", "dq", "dk"), (a, b, d[:, :, 0].transpose(1, 2), d[:, :, 1].transpose(1, 2)), want):
        assert O.rel(s, t) <= _tol(name, torch.bfloat16, torch.float32), name


def test_rows_of_zeros_and_of_large_values():
    """A zero row stays zero and has the finite gradient dy w / sqrt(eps); fp16 rows whose squares pass the type's range."""
    x = list(_inputs(1, 2, 2, 4, 64, torch.float16, torch.float32, 16, False, seed=4))
    x[0][0, 0, 1] = 0
    x[0][0, 1, 2] = 40000.0
    x[5] = x[5] * 1e-2  # (the gradient of a zero row is 1000 times dy)
    got, want = _run(*x), _truth(*x)
    assert (got[0][0, 0, 1] == 0).all()
    for name, a, b in zip(("q", "k", "dq", "dk", "dqw", "dkw"), got, want):
        assert torch.isfinite(a).all() and O.rel(a, b) <= _tol(name, torch.float16, torch.float32), name


def test_offsets_past_32_bits():
    """More than 2^31 elements in a packed projection: the last positions against fp64."""
    from cottention_transformer_b200 import qk_norm_rotary
    H, D, T, dtype = 16, 64, 50, torch.bfloat16
    N = 2 ** 31 // (2 * H * D) + 77
    if torch.cuda.mem_get_info()[0] < 10 * 2 ** 31:
        pytest.skip("not enough device memory")
    r = torch.Generator(device="cuda").manual_seed(8)
    qk = torch.randn(1, N, 2, H, D, dtype=dtype, device="cuda", generator=r).requires_grad_()
    dq, dk = (torch.randn(1, H, N, D, dtype=dtype, device="cuda", generator=r) for _ in range(2))
    _, _, qw, kw, tables, _, _ = _inputs(1, 1, 1, N, D, dtype, torch.float32, 32, False, seed=8)
    a, b = qk_norm_rotary(qk[:, :, 0].transpose(1, 2), qk[:, :, 1].transpose(1, 2), qw.cuda(), kw.cuda(), rotary=tuple(t.cuda() for t in tables))
    d = torch.autograd.grad((a, b), qk, (dq, dk))[0].detach()[:, N - T:].cpu()
    tail = lambda t: t.detach()[:, :, N - T:].cpu()  # noqa: E731
    x = qk.detach()[:, N - T:].cpu()
    want = _truth(x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2), qw, kw, tuple(t[N - T:] for t in tables), tail(dq), tail(dk))
    for name, s, t in zip(("q", "k", "dq", "dk"), (tail(a), tail(b), d[:, :, 0].transpose(1, 2), d[:, :, 1].transpose(1, 2)), want):
        assert O.rel(s, t) <= _tol(name, dtype, torch.float32), name


def test_unit_weights_give_the_l2_normalisation():
    from cottention_transformer_b200 import qk_norm_rotary
    q = torch.randn(2, 3, 50, 64, device="cuda")
    w = torch.full((64,), 64 ** -0.5, device="cuda")
    a, b = qk_norm_rotary(q, q, w, w, eps=0.0)
    assert O.rel(a, torch.nn.functional.normalize(q.double(), dim=-1)) < 1e-6 and torch.equal(a, b)


def test_gradients_against_differences():
    """A central difference of fourth order along a random direction, fp32."""
    from cottention_transformer_b200 import qk_norm_rotary
    q, k, qw, kw, tables, dq, dk = _inputs(1, 2, 2, 40, 64, torch.float32, torch.float32, 32, False, seed=5)
    x = [t.cuda().requires_grad_() for t in (q, k, qw, kw)]
    r = torch.Generator(device="cuda").manual_seed(2)
    step = [torch.randn(t.shape, device="cuda", generator=r) * t.detach().std() for t in x]
    tab = tuple(t.cuda() for t in tables)

    def loss(h):
        a, b = qk_norm_rotary(*(t + h * d for t, d in zip(x, step)), rotary=tab)
        return (a * dq.cuda()).double().sum() + (b * dk.cuda()).double().sum()

    grads = torch.autograd.grad(loss(0.0), x)
    h = 1e-2
    with torch.no_grad():
        num = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
    ana = sum((a.double() * d).sum() for a, d in zip(grads, step))
    assert abs(num - ana) <= 1e-3 * sum((a.double() * d).square().sum() for a, d in zip(grads, step)).sqrt()


def test_layer_of_norm_scan_and_step():
    """The operators as a layer uses them: projection -> norm and rotation -> gated scan in training, the same layer token by token
    in generation; gradients of the whole chain against fp64."""
    from cottention_transformer_b200 import GatedScanState, gated_scan, qk_norm_rotary
    B, H, N, D = 2, 3, 100, 64
    r = torch.Generator().manual_seed(6)
    for dtype in (torch.float32, torch.bfloat16):
        qkv = torch.randn(B, N, 3, H, D, generator=r).to(dtype)
        gate = torch.nn.functional.logsigmoid(2 + torch.randn(B, N, H, generator=r)).to(dtype)
        qw, kw = (torch.full((D,), D ** -0.5) * (1 + 0.1 * torch.randn(D, generator=r)) for _ in range(2))
        ang = torch.arange(N).float()[:, None] * 10000.0 ** (-torch.arange(16).float() / 16)
        tab = (ang.sin(), ang.cos())
        do = torch.randn(B, H, N, D, generator=r).to(dtype)

        leaf = [t.double().requires_grad_() for t in (qkv, gate, qw, kw)]
        q, k, v = (leaf[0][:, :, i].transpose(1, 2) for i in range(3))
        out, _ = O.gated_scan(O.qk_norm(q, leaf[2], *(t.double() for t in tab)), O.qk_norm(k, leaf[3], *(t.double() for t in tab)), v, leaf[1].transpose(1, 2))
        want = (out, *torch.autograd.grad(out, leaf, do.double()))

        leaf = [t.cuda().requires_grad_() for t in (qkv, gate, qw, kw)]
        q, k, v = (leaf[0][:, :, i].transpose(1, 2) for i in range(3))
        qn, kn = qk_norm_rotary(q, k, leaf[2], leaf[3], rotary=tuple(t.cuda() for t in tab))
        out = gated_scan(qn, kn, v, leaf[1].transpose(1, 2))
        got = (out, *torch.autograd.grad(out, leaf, do.cuda()))
        # the roundings of the scan (six half steps at most) and of the two passes around it; the weights' gradients are sums over
        # B H N rows of terms of either sign with those roundings
        tol = 2e-5 if dtype == torch.float32 else 8 * torch.finfo(dtype).eps / 2
        for name, a, b in zip(("out", "dqkv", "dgate", "dqw", "dkw"), got, want):
            assert O.rel(a, b) <= tol, (name, O.rel(a, b))

        s = GatedScanState(B, H, D)
        with torch.no_grad():
            outs = [s.prefill(qn[:, :, :90], kn[:, :, :90], v[:, :, :90], leaf[1].transpose(1, 2)[:, :, :90])]
            for t in range(90, N):
                qt, kt = qk_norm_rotary(q[:, :, t:t + 1], k[:, :, t:t + 1], leaf[2], leaf[3], rotary=tuple(x[t:t + 1].cuda() for x in tab))
                outs.append(s.step(qt, kt, v[:, :, t:t + 1], leaf[1].transpose(1, 2)[:, :, t:t + 1]))
        assert O.rel(torch.cat(outs, 2), want[0]) <= tol


@pytest.mark.parametrize("compiled", [True, False])
def test_refusals(compiled, monkeypatch):
    from cottention_transformer_b200 import _binding, qk_norm_rotary
    if not compiled:
        monkeypatch.setattr(_binding, "autograd", lambda: None)
    q, w = torch.randn(2, 3, 10, 64, device="cuda"), torch.ones(64, device="cuda")
    s = torch.zeros(10, 16, device="cuda")
    for bad, match in [((q.cpu(), q, w, w), "CUDA"), ((q, q.half(), w, w), "one type"), ((q, q[:, :, :9], w, w), "agree"), ((q[..., :48], q[..., :48], w[:48], w[:48]), "head dims"),
                       ((q, q, w[:32], w), "weights"), ((q, q, w.half(), w), "weights"), ((q, q, w.double(), w.double()), "weights")]:
        with pytest.raises(RuntimeError, match=match):
            qk_norm_rotary(*bad)
    with pytest.raises(ValueError, match="dimensions"):
        qk_norm_rotary(q[0], q[0], w, w)
    for tab, match in [((s, s[:9]), "sin / cos"), ((s[:9], s[:9]), "sin / cos"), ((s[:, :3].contiguous(),) * 2, "rotary dim"), ((torch.zeros(10, 36, device="cuda"),) * 2, "rotary dim"),
                       ((s.expand(3, 10, 16),) * 2, "sin / cos")]:
        with pytest.raises(RuntimeError, match=match):
            qk_norm_rotary(q, q, w, w, rotary=tab)
