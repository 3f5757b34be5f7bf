"""The gated causal scan, forward and backward, and its single-token form, against the token-by-token recurrence in fp64."""
import pytest
import torch

import gated_oracle as O

pytestmark = pytest.mark.gpu

NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dinit")


def _u(dtype):
    return torch.finfo(dtype).eps / 2


# 2-norms, relative.  fp32: sums of up to D + 64 products with random signs, a few times 2^-24 sqrt(192) = 8e-7 in every one of two
# products in a row.  16 bits: half a step u each for the decayed scores, for the copy of the state, for the rows that enter a state
# (their weight) and for the result; dg is a difference of sums of two such results, and of a product of two states.
def _tol(name, dtype):
    if dtype == torch.float32:
        return 4e-6 if name != "dg" else 8e-6
    return {"state": 1e-5, "dinit": 2 * _u(dtype)}.get(name, (4 if name != "dg" else 6) * _u(dtype))


def _inputs(B, H, N, D, dtype, seed, gate_dtype=None, masked=False, docs=False, init=False):
    r = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(B, H, N, D, generator=r) for _ in range(4))
    q, k = (torch.nn.functional.normalize(t, dim=-1) for t in (q, k))
    g = torch.nn.functional.logsigmoid(torch.linspace(0.5, 6, max(H, 2))[:H].view(1, H, 1) + torch.randn(B, H, N, generator=r))
    if docs:
        g = g.masked_fill(torch.rand(B, 1, N, generator=r) < 0.03, float("-inf"))
    keep = None
    if masked:
        keep = torch.rand(B, N, generator=r) < 0.7
        keep[0, : N // 3] = False  # positions before the first one that counts
    st = torch.randn(B, H, D, D, generator=r) * D ** -0.5 if init else None
    dst = torch.randn(B, H, D, D, generator=r) * D ** -0.5
    q, k, v, do = (t.to(dtype) for t in (q, k, v, do))
    return q, k, v, g.to(gate_dtype or dtype), keep, st, do, dst


def _truth(q, k, v, g, keep, st, do, dst):
    leaf = [t.double().requires_grad_() for t in (q, k, v, g)] + ([] if st is None else [st.double().requires_grad_()])
    out, final = O.gated_scan(*leaf[:4], keep, leaf[4] if st is not None else None)
    loss = (out * do.double()).sum() + (0 if dst is None else (final * dst.double()).sum())
    return out, final, *torch.autograd.grad(loss, leaf)


def _run(q, k, v, g, keep, st, do, dst, view=lambda t: t):
    from cottention_transformer_b200 import gated_scan
    q, k, v, do = (view(t.cuda()) for t in (q, k, v, do))
    leaf = [t.detach().requires_grad_() for t in (q, k, v, g.cuda())] + ([] if st is None else [st.cuda().requires_grad_()])
    out, final = gated_scan(*leaf[:4], keep=None if keep is None else keep.cuda(), initial_state=leaf[4] if st is not None else None, return_state=True)
    outs, grads = ((out,), (do,)) if dst is None else ((out, final), (do, dst.cuda()))
    return out, final, *torch.autograd.grad(outs, leaf, grads)


def _compare(got, want, dtype):
    for name, a, b in zip(NAMES if len(got) != 6 or got[5].dim() == 3 else NAMES[:5] + NAMES[6:], got, want):
        assert a.shape == b.shape and torch.isfinite(a).all(), name
        if dtype != torch.float32 and name == "dg" and b.norm() < 1e-2:  # short sequences: the differences of next to nothing
            assert (a.detach().double().cpu() - b).norm() < 1e-2 * 6 * _u(dtype) + 1e-6, name
            continue
        assert O.rel(a, b) <= _tol(name, dtype), (name, O.rel(a, b), _tol(name, dtype))


SHAPES = [(1, 1, 1, 64), (1, 2, 2, 128), (2, 3, 63, 32), (1, 2, 64, 64), (2, 2, 65, 64), (1, 2, 127, 128), (1, 2, 128, 64), (1, 3, 129, 128),
          (2, 4, 700, 64), (1, 2, 385, 128),
          (2, 40, 900, 64), (3, 20, 400, 128),  # (more chunks than a CTA per SM takes at once)
          (1, 1, 1700, 64), (1, 2, 1500, 128)]  # (few and long: walked in segments)


@pytest.mark.parametrize("form", ["plain", "masked", "docs", "init"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_matches_the_recurrence(shape, dtype, form):
    x = _inputs(*shape, dtype, seed=sum(shape), masked=form == "masked", docs=form == "docs", init=form == "init")
    x = (*x[:-1], x[-1] if form in ("init", "docs") else None)  # with and without a gradient of the final state
    _compare(_run(*x), _truth(*x), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("level", [-30.0, -8.0, 0.0])
def test_gates_of_one_strength(dtype, level):
    """States that last a fraction of a token, and states that lose nothing at all."""
    q, k, v, g, keep, st, do, dst = _inputs(1, 2, 300, 64, dtype, seed=5, init=True)
    g = torch.full_like(g, level)
    got, want = _run(q, k, v, g, keep, st, do, dst), _truth(q, k, v, g, keep, st, do, dst)
    if level < -1:
        # dg is e^level of the terms that it is summed from: a position's own pair, (q_t.k_t)(dO_t.v_t), stands in q_t.dq_t and in
        # k_t.dk_t and cancels.  Those terms are products |q| |dq| of about 1 x 8, each with a rounding of 2^-24 (16 bits: u, of the
        # same rounded product in both, so that fp32's remains, and the state's), and up to 64 (128) of either kind are summed.
        if dtype == torch.float16 and level == -30.0:
            # the gradient of the initial state is e^-30 of its terms: products below the type's smallest step, 2^-24, which the
            # weighted rows are rounded to in absolute terms (half of it, times the sum of |q| <= 128 over a chunk)
            assert (got[6].double().cpu() - want[6]).abs().max() <= 2 ** -25 * 128
            _compare(got[:5], want[:5], dtype)
        else:
            _compare((*got[:5], *got[6:]), (*want[:5], *want[6:]), dtype)
        rms = (got[5].double().cpu() - want[5]).square().mean().sqrt()
        assert rms <= 8 * 2 ** -24 * 256 ** 0.5 + (0 if dtype == torch.float32 else _u(dtype) * want[5].square().mean().sqrt() * 6 + 1e-4 * _u(dtype) / _u(torch.bfloat16))
    else:
        _compare(got, want, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gates_in_fp32_beside_16_bit_tensors(dtype):
    x = _inputs(2, 2, 200, 64, dtype, seed=6, gate_dtype=torch.float32, init=True)
    got = _run(*x)
    assert got[5].dtype == torch.float32
    _compare(got, _truth(*x), dtype)


def test_without_decay_it_is_the_plain_scan():
    from cottention_transformer_b200 import CustomAttention, gated_scan
    q, k, v, g, *_ = (t.cuda() if t is not None else None for t in _inputs(1, 2, 333, 64, torch.float32, seed=7))
    a, b = gated_scan(q, k, v, torch.zeros_like(g)), CustomAttention.apply(q, k, v)
    assert O.rel(a, b) < 4e-6


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_views_of_a_projection(dtype, D):
    """q, k, v as slices of a packed tensor, gates of a [B, N, H] projection, gradients of any stride."""
    from cottention_transformer_b200 import gated_scan
    B, H, N = 2, 3, 150
    q, k, v, g, keep, st, do, dst = _inputs(B, H, N, D, dtype, seed=8, masked=True)
    want = _truth(q, k, v, g, keep, None, do, None)
    qkv = torch.stack([q, k, v], 2).permute(0, 3, 2, 1, 4).contiguous().cuda().requires_grad_()  # [B, N, 3, H, D]
    gn = g.transpose(1, 2).contiguous().cuda().requires_grad_()
    out = gated_scan(*(qkv[:, :, i].transpose(1, 2) for i in range(3)), gn.transpose(1, 2), keep=keep.cuda())
    assert out.transpose(1, 2).is_contiguous()  # the memory order of v: merging the heads is a view
    dqkv, dg = torch.autograd.grad(out, (qkv, gn), do.cuda().transpose(2, 3).contiguous().transpose(2, 3))
    got = (out, *dqkv.permute(2, 0, 3, 1, 4).unbind(0), dg.transpose(1, 2))
    for name, a, b in zip(("out", "dq", "dk", "dv", "dg"), got, (want[0], *want[2:])):
        assert O.rel(a, b) <= _tol(name, dtype), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_expanded_offset_and_transposed_inputs(dtype):
    from cottention_transformer_b200 import gated_scan
    q, k, v, g, keep, st, do, dst = _inputs(2, 2, 70, 64, dtype, seed=9)
    k1 = k[:, :1].clone()  # one key head for all
    want = _truth(q, k1.expand_as(q), v, g, None, None, do, None)
    off = torch.empty(q.numel() + 1, dtype=dtype, device="cuda")[1:].view_as(q).copy_(q)  # a base off the 16-byte grid
    kk = k1.cuda().requires_grad_()
    vt = v.cuda().transpose(2, 3).contiguous().transpose(2, 3)  # rows that are not contiguous
    out = gated_scan(off, kk.expand(-1, 2, -1, -1), vt, g.cuda())
    assert O.rel(out, want[0]) <= _tol("out", dtype)
    dk, = torch.autograd.grad(out, kk, do.cuda())
    assert O.rel(dk, want[3].sum(1, keepdim=True)) <= 2 * _tol("dk", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_what_masked_rows_hold_does_not_matter(dtype):
    x = _inputs(2, 2, 200, 64, dtype, seed=10, masked=True, init=True)
    q, k, v, g, keep, st, do, dst = x
    want = _run(*x)
    bad = [t.clone() for t in (q, k, v, do)]
    for t, val in zip(bad, (float("nan"), float("inf"), float("-inf"), float("nan"))):
        t[~keep[:, None].expand(t.shape[:3])] = val
    g2 = g.clone()
    g2[~keep[:, None].expand(g.shape)] = float("nan")
    got = _run(*bad[:3], g2, keep, st, bad[3], dst)
    for name, a, b in zip(NAMES, got, want):
        assert torch.equal(a, b), name
        if name in ("out", "dq", "dk", "dv", "dg"):
            assert (a[~keep.cuda()[:, None].expand(a.shape[:3])] == 0).all(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_batch_entry_with_nothing_unmasked(dtype):
    q, k, v, g, keep, st, do, dst = _inputs(2, 2, 130, 64, dtype, seed=11, masked=True, init=True)
    keep[0] = False
    got = _run(q, k, v, g, keep, st, do, dst)
    _compare(got, _truth(q, k, v, g, keep, st, do, dst), dtype)
    assert torch.equal(got[1][0].cpu(), st[0]) and (got[0][0] == 0).all() and torch.equal(got[6][0].cpu(), dst[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_dropped_state_takes_what_it_held_with_it(dtype):
    """A gate of -inf at the first position of a document: nothing of an infinite initial state is left."""
    from cottention_transformer_b200 import gated_scan, gated_scan_step
    q, k, v, g, keep, st, do, dst = (t if t is None else t.cuda() for t in _inputs(1, 2, 90, 64, dtype, seed=12, init=True))
    g[:, :, 0] = float("-inf")
    a, sa = gated_scan(q, k, v, g, initial_state=torch.full_like(st, float("inf")), return_state=True)
    b, sb = gated_scan(q, k, v, g, return_state=True)
    assert torch.equal(a, b) and torch.equal(sa, sb)
    s = torch.full_like(st, float("nan"))
    o = gated_scan_step(s, q[:, :, :1], k[:, :, :1], v[:, :, :1], g[:, :, :1])
    assert torch.isfinite(o).all() and torch.isfinite(s).all()


def test_gradients_against_differences():
    """fp32: a central difference along a random direction of all inputs, h = 1e-2: the third-order term of a function that is
    cubic in q, k, v and smooth in g is below 1e-3 of the slope here, rounding is 2e-7 |L| / h."""
    from cottention_transformer_b200 import gated_scan
    q, k, v, g, keep, st, do, dst = (t if t is None else t.cuda() for t in _inputs(1, 2, 150, 64, torch.float32, seed=13, init=True))
    r = torch.Generator(device="cuda").manual_seed(1)
    x = [t.clone().requires_grad_() for t in (q, k, v, g, st)]
    step = [torch.randn(t.shape, device="cuda", generator=r) * t.detach().std() for t in x]

    def loss(h):
        out, s = gated_scan(*(t + h * d for t, d in zip(x[:4], step)), initial_state=x[4] + h * step[4], return_state=True)
        return (out * do).double().sum() + (s * dst).double().sum()

    grads = torch.autograd.grad(loss(0.0), x)
    h = 1e-2
    with torch.no_grad():
        num = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
    ana = sum((a.double() * d).sum() for a, d in zip(grads, step))
    assert abs(num - ana) <= 2e-3 * sum((a.double() * d).square().sum() for a, d in zip(grads, step)).sqrt() + 1e-3 * abs(ana)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_same_bits_every_time_and_on_both_routes(dtype, monkeypatch):
    x = _inputs(2, 3, 300, 64, dtype, seed=14, masked=True, init=True)
    a = _run(*x)
    for b in O.both_routes(monkeypatch.context(), lambda: _run(*x)):
        assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_pieces_of_a_prompt_then_tokens_are_the_whole():
    from cottention_transformer_b200 import GatedScanState, gated_scan
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        q, k, v, g, *_ = (t if t is None else t.cuda() for t in _inputs(2, 3, 200, 64, dtype, seed=15))
        whole, state = gated_scan(q, k, v, g, return_state=True)
        s = GatedScanState(2, 3, 64)
        at = [0, 70, 71, 190]
        outs = [s.prefill(*(t[:, :, a:b] for t in (q, k, v, g))) for a, b in zip(at, at[1:])]
        outs += [s.step(*(t[:, :, i:i + 1] for t in (q, k, v, g))) for i in range(190, 195)]
        outs.append(s.step(*(t[:, :, 195:] for t in (q, k, v, g))))
        assert O.rel(torch.cat(outs, 2), whole) <= 2 * _tol("out", dtype)
        assert O.rel(s.state, state) <= 2e-5
        s.reset()
        assert (s.state == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 32), (3, 5, 1, 64), (2, 2, 7, 64), (1, 3, 1, 128), (2, 1, 9, 128), (130, 4, 1, 64)])
def test_step_matches_the_recurrence(shape, dtype, monkeypatch):
    from cottention_transformer_b200 import gated_scan_step
    q, k, v, g, keep, st, *_ = _inputs(*shape, dtype, seed=16, init=True, docs=True, gate_dtype=torch.float32 if shape[0] == 3 else None)
    out, final = O.gated_scan(q.double(), k.double(), v.double(), g.double(), None, st.double())
    views = [t.cuda().transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]  # [B, T, H, D], as a projection leaves them

    def run():
        s = st.cuda()
        return gated_scan_step(s, *views, g.cuda()), s

    for o, s in O.both_routes(monkeypatch.context(), run):
        assert o.transpose(1, 2).is_contiguous()
        assert O.rel(o, out) <= (_u(dtype) if dtype != torch.float32 else 1e-6) and O.rel(s, final) <= 1e-6


def test_other_streams_and_graphs():
    """A captured training step replays with new inputs, beside another one; calls on a stream of their own."""
    from cottention_transformer_b200 import gated_scan
    xs = [[t if t is None else t.cuda() for t in _inputs(2, 2, 300, 64, torch.bfloat16, seed=s)] for s in (20, 21)]

    def train(q, k, v, g, do):
        out = gated_scan(q, k, v, g)
        return out, *torch.autograd.grad(out, (q, k, v, g), do)

    want = [[t.clone() for t in train(*(t.requires_grad_() for t in x[:4]), x[6])] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for x in xs:
        leaf = [t.detach().clone().requires_grad_() for t in x[:4]]
        do = x[6].clone()
        with torch.cuda.stream(side):
            got = train(*leaf, do)
            del got
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = train(*leaf, do)
        graphs.append((graph, leaf, do, res))
    for i in (0, 1, 0):  # the two graphs in turn, the inputs exchanged
        for (graph, leaf, do, res), j in zip(graphs, (i, 1 - i)):
            with torch.no_grad():
                for a, b in zip((*leaf, do), (*xs[j][:4], xs[j][6])):
                    a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for (graph, leaf, do, res), j in zip(graphs, (i, 1 - i)):
            assert all(torch.equal(a, b) for a, b in zip(res, want[j]))


def test_a_saved_graph_can_be_walked_twice_and_not_differentiated_again():
    from cottention_transformer_b200 import gated_scan
    q, k, v, g, keep, st, do, dst = (t if t is None else t.cuda().requires_grad_() for t in _inputs(1, 1, 100, 64, torch.float32, seed=22))
    out = gated_scan(q, k, v, g)
    a = torch.autograd.grad(out, (q, k, v, g), do.detach(), retain_graph=True)
    b = torch.autograd.grad(out, (q, k, v, g), do.detach(), retain_graph=True)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    with pytest.raises(RuntimeError):
        c = torch.autograd.grad(out, (q,), do.detach(), create_graph=True)
        torch.autograd.grad(c[0].sum(), q)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 128])
def test_one_decay_per_head(dtype, D):
    """A fixed decay as an expanded view: its gradient is the sum over batch and positions."""
    from cottention_transformer_b200 import gated_scan
    q, k, v, g, keep, st, do, dst = _inputs(2, 3, 200, D, dtype, seed=30)
    d = torch.tensor([-0.5, -0.05, -0.01]).to(dtype)
    want = _truth(q, k, v, d.view(1, 3, 1).expand(2, 3, 200).contiguous(), None, None, do, None)
    leaf = d.cuda().requires_grad_()
    out = gated_scan(q.cuda(), k.cuda(), v.cuda(), leaf.view(1, 3, 1).expand(2, 3, 200))
    assert O.rel(out, want[0]) <= _tol("out", dtype)
    got, = torch.autograd.grad(out, leaf, do.cuda())
    # a sum of 400 terms, each rounded to the type by the operator (u) and with its own error (6 u) in the 2-norm
    err = (got.double().cpu() - want[5].sum((0, 2))).abs()
    assert (err <= 7 * _tol("dg", dtype) * want[5].norm(dim=2).sum(0) + 2 * _u(dtype) * want[5].sum((0, 2)).abs() + 1e-5).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_one_result_alone(dtype):
    """The initial state's gradient where the last state is not asked for, and gradients through the last state alone."""
    from cottention_transformer_b200 import gated_scan
    q, k, v, g, keep, st, do, dst = _inputs(1, 2, 300, 64, dtype, seed=31, init=True)
    want = _truth(q, k, v, g, None, st, do, None)
    leaf = [t.cuda().requires_grad_() for t in (q, k, v, g, st)]
    out = gated_scan(*leaf[:4], initial_state=leaf[4])
    for name, a, b in zip(NAMES[2:], torch.autograd.grad(out, leaf, do.cuda()), want[2:]):
        assert O.rel(a, b) <= _tol(name, dtype), name
    want = _truth(q, k, v, g, None, st, torch.zeros_like(do), dst)
    state = gated_scan(*leaf[:4], initial_state=leaf[4], return_state=True)[1]
    for name, a, b in zip(NAMES[2:], torch.autograd.grad(state, leaf, dst.cuda()), want[2:]):
        assert O.rel(a, b) <= 2 * _tol(name, dtype), name


def test_calls_on_two_streams_at_once():
    from cottention_transformer_b200 import gated_scan
    xs = [[t.cuda() for t in (*_inputs(2, 4, 1000, 64, torch.bfloat16, seed=s)[:4], _inputs(2, 4, 1000, 64, torch.bfloat16, seed=s)[6])] for s in (32, 33)]

    def train(x):
        leaf = [t.detach().requires_grad_() for t in x[:4]]
        out = gated_scan(*leaf)
        return out, *torch.autograd.grad(out, leaf, x[4])

    want = [train(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(5):
        for i, (stream, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(stream):
                got[i].append(train(x))
    torch.cuda.synchronize()
    for w, rs in zip(want, got):
        for r in rs:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_rows_past_the_sequences_are_left_alone():
    """Outputs and states written through a view of a larger buffer: nothing beside it changes."""
    from cottention_transformer_b200 import _lib
    import ctypes
    L = _lib.lib()
    B, H, N, D = 2, 2, 150, 64
    for dtype in (torch.float32, torch.bfloat16):
        q, k, v, g, *_ = (t if t is None else t.cuda() for t in _inputs(B, H, N, D, dtype, seed=34))
        code = _lib.DTYPE_CODE[dtype]
        big = torch.full((B, H, N + 40, D), 7.0, dtype=dtype, device="cuda")
        states = torch.empty(L.cott_gated_scan_states_bytes(B, H, N, D, code), dtype=torch.uint8, device="cuda")
        ws = torch.empty(max(L.cott_gated_scan_workspace_bytes(B, H, N, D, code, 0), 16), dtype=torch.uint8, device="cuda")
        lay = _lib.CottGatedLayout()
        for name, t in (("q", q), ("k", k), ("v", v), ("out", big), ("gate", g)):
            setattr(lay, name, _lib.CottStrides(*t.stride()[:3]))
        _lib.check(L.cott_gated_scan_fwd(_lib.ptr(q), _lib.ptr(k), _lib.ptr(v), _lib.ptr(g), None, None, _lib.ptr(big), None, _lib.ptr(states),
                                         _lib.ptr(ws), ctypes.byref(lay), B, H, N, D, code, code, _lib.stream_ptr(q.device)), "cott_gated_scan_fwd")
        from cottention_transformer_b200 import gated_scan
        assert torch.equal(big[:, :, :N], gated_scan(q, k, v, g)) and (big[:, :, N:] == 7).all()
        _lib.check_device_status()


@pytest.mark.parametrize("D", [64, 32])
def test_offsets_past_32_bits(D):
    """More than 2^31 elements per tensor: the last positions, behind a gate that drops the state, are a sequence of their own."""
    from cottention_transformer_b200 import gated_scan
    dtype, N, T = torch.bfloat16, 2 ** 31 // D + 1234, 700
    if torch.cuda.mem_get_info()[0] < 14 * 2 * N * D:
        pytest.skip("not enough device memory")
    r = torch.Generator(device="cuda").manual_seed(35)
    q, k, v, do = (torch.randn(1, 1, N, D, dtype=dtype, device="cuda", generator=r).mul_(s) for s in (D ** -0.5, D ** -0.5, 1, 1))
    g = torch.nn.functional.logsigmoid(torch.randn(1, 1, N, device="cuda", generator=r) + 2)
    g[:, :, N - T] = float("-inf")
    leaf = [t.requires_grad_() for t in (q, k, v, g)]
    out = gated_scan(*leaf)
    got = [t.detach()[:, :, N - T:].cpu() for t in (out, *torch.autograd.grad(out, leaf, do))]
    x = [t.detach()[:, :, N - T:].cpu() for t in (q, k, v, g)]
    want = _truth(*x, None, None, do[:, :, N - T:].cpu(), None)
    for name, a, b in zip(("out", "dq", "dk", "dv", "dg"), got, (want[0], *want[2:])):
        assert O.rel(a, b) <= _tol(name, dtype), name


def test_empty_sequences():
    from cottention_transformer_b200 import gated_scan, gated_scan_step
    q = torch.empty(2, 3, 0, 64, device="cuda", requires_grad=True)
    g, st = torch.empty(2, 3, 0, device="cuda", requires_grad=True), torch.randn(2, 3, 64, 64, device="cuda", requires_grad=True)
    out, s = gated_scan(q, q, q, g, initial_state=st, return_state=True)
    assert out.shape == q.shape and torch.equal(s, st)
    d = torch.randn_like(s)
    assert torch.equal(torch.autograd.grad(s, st, d)[0], d)
    assert (gated_scan(q, q, q, g, return_state=True)[1] == 0).all()
    with torch.no_grad():
        keepst = st.detach().clone()
        assert gated_scan_step(keepst, q, q, q, g).shape == q.shape and torch.equal(keepst, st)


@pytest.mark.parametrize("compiled", [True, False])
def test_refusals(compiled, monkeypatch):
    from cottention_transformer_b200 import _binding, gated_scan, gated_scan_step
    if not compiled:
        monkeypatch.setattr(_binding, "autograd", lambda: None)
    q = torch.randn(2, 3, 10, 64, device="cuda")
    g = -torch.rand(2, 3, 10, device="cuda")
    st = torch.zeros(2, 3, 64, 64, device="cuda")
    for bad, match in [((q.cpu(), q, q, g), "CUDA"), ((q, q.half(), q, g), "one type"), ((q.double(),) * 3 + (g,), "float32, float16"),
                       ((q, q[:, :2], q, g), "same shape"), ((q[..., :48],) * 3 + (g,), "head dims"), ((q, q, q, g[:, :, :9]), "log_decay"),
                       ((q, q, q, g.half()), "log_decay"), ((q, q, q, g.transpose(1, 2)), "log_decay")]:
        with pytest.raises(RuntimeError, match=match):
            gated_scan(*bad)
        with pytest.raises(RuntimeError, match=match):
            gated_scan_step(st, *bad)
    with pytest.raises(ValueError, match="dimensions"):
        gated_scan(q[0], q[0], q[0], g[0])
    for keep in (torch.ones(2, 9, dtype=torch.bool, device="cuda"), torch.ones(2, 10, device="cuda"), torch.ones(2, 10, dtype=torch.bool)):
        with pytest.raises(RuntimeError, match="keep"):
            gated_scan(q, q, q, g, keep=keep)
    for bad in (st.half(), st[:, :2], st[..., :32], st.cpu()):
        with pytest.raises(RuntimeError, match="initial_state"):
            gated_scan(q, q, q, g, initial_state=bad)
        with pytest.raises(RuntimeError, match="state"):
            gated_scan_step(bad, q, q, q, g)
    with pytest.raises(RuntimeError, match="contiguous"):
        gated_scan_step(st.transpose(2, 3), q, q, q, g)
    with pytest.raises(RuntimeError, match="not differentiable"):
        gated_scan_step(st, q.clone().requires_grad_(), q, q, g)
