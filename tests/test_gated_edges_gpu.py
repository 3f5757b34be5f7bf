"""The gated scan and its neighbours where a state, a mask or a gate is at its limit: against fp64, or against the same call without
what must not matter."""
import pytest
import torch

from test_gated_scan_gpu import _compare, _inputs, _truth

pytestmark = pytest.mark.gpu


def _call(q, k, v, g, keep, st, do, dst):
    """Outputs and all gradients, the gates' and the initial state's among them."""
    from cottention_transformer_b200 import gated_scan
    leaf = [t.cuda().requires_grad_() for t in (q, k, v, g)] + ([] if st is None else [st.cuda().requires_grad_()])
    out, final = gated_scan(*leaf[:4], keep=None if keep is None else keep.cuda(), initial_state=leaf[4] if st is not None else None, return_state=True)
    outs, grads = ((out,), (do.cuda(),)) if dst is None else ((out, final), (do.cuda(), dst.cuda()))
    return out, final, *torch.autograd.grad(outs, leaf, grads)


HELD = [float("inf"), float("nan"), 1e5]  # (1e5: its copy in fp16 is an infinity)
AT = [0, 5, 63, 130]  # the first position of the new document, at a border and inside a chunk


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("at", AT)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_behind_a_dropped_state(dtype, D, at, held):
    """Behind a gate of -inf outputs and gradients are those of a sequence that begins there, whatever the state before it holds."""
    q, k, v, g, _, st, do, dst = _inputs(1, 2, 200, D, dtype, seed=40, init=True)
    g[:, :, at] = float("-inf")
    behind = slice(at, None)
    got = _call(q, k, v, g, None, torch.full_like(st, held), do, dst)
    want = _truth(*(t[:, :, behind] for t in (q, k, v, g)), None, None, do[:, :, behind], dst)
    _compare([t[:, :, behind] if i != 1 else t for i, t in enumerate(got[:6])], want, dtype)


def _before_a_drop(dtype, D, at, held):
    """Before a gate of -inf the gradients are those of a sequence that ends there, whatever the gradient of the last state holds."""
    q, k, v, g, _, st, do, dst = _inputs(1, 2, 200, D, dtype, seed=41, init=True)
    g[:, :, at] = float("-inf")
    before = slice(0, at)
    got = _call(q, k, v, g, None, st, do, torch.full_like(dst, held))
    want = _truth(*(t[:, :, before] for t in (q, k, v, g)), None, st, do[:, :, before], None)
    _compare([got[0][:, :, before], want[1], *(t[:, :, before] for t in got[2:6]), got[6]], want, dtype)


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("at", AT[1:])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_before_a_dropped_state_gradient(dtype, D, at, held):
    _before_a_drop(dtype, D, at, held)


@pytest.mark.parametrize("N", [20, 200])
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_masked_rows_beside_states_that_are_not_finite(dtype, D, N):
    """Padding in front of a document (its gate drops an initial state that holds an infinity) and at the end of a sequence whose
    last state has an infinite gradient: outputs and gradients of masked rows are zero, those of the document what they are alone."""
    q, k, v, g, _, st, do, dst = _inputs(2, 2, N, D, dtype, seed=42, init=True)
    a, b = N // 4, N - N // 4
    keep = torch.zeros(2, N, dtype=torch.bool)
    keep[:, a:b] = True
    g[:, :, a] = float("-inf")
    got = _call(q, k, v, g, keep, torch.full_like(st, float("inf")), do, None)
    doc = slice(a, b)
    want = _truth(*(t[:, :, doc] for t in (q, k, v, g)), None, None, do[:, :, doc], None)
    masked = ~keep[0].cuda()
    for t in (got[0], *got[2:6]):
        assert (t[:, :, masked] == 0).all()
    _compare([t[:, :, doc] if i != 1 else t for i, t in enumerate(got[:6])], want, dtype)
    got = _call(q, k, v, g, keep, st, do, torch.full_like(dst, float("inf")))
    for t in (got[0], *got[2:6]):
        assert (t[:, :, masked] == 0).all()


@pytest.mark.parametrize("gate", [float("-inf"), -1e4, -100.0])
@pytest.mark.parametrize("roles", ["scores", "rows"])
@pytest.mark.parametrize("N", [128, 300])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decays_inside_documents_of_a_few_tokens(dtype, D, N, roles, gate):
    """Packed documents of 2 to 8 tokens.  The inputs are such that every entry of a result is one decay: either all scores are 1 and the
    rows are unit vectors of their position, or the other way round.  A decay is rounded to the type once (u); its exponent is a
    difference of two sums of at most 128 gates below 0.5 / log 2, i.e. numbers below 128 (half an ulp: 2^-18) after at most eight
    additions each: 16 x 2^-18 x log 2 = 4.3e-5, less than 0.1 u of float16.  No document begins within a chunk and ends in the next."""
    r = torch.Generator().manual_seed(43)
    g = -0.5 * torch.rand(1, 1, N, generator=r)
    starts, t = [], 0
    while t < N:
        starts.append(t)
        t = min(t + int(torch.randint(2, 9, (1,), generator=r)), (t // 128 + 1) * 128)
    g[..., starts] = gate
    first = torch.zeros(N, dtype=torch.long)
    first[starts] = 1
    doc = first.cumsum(0)
    sums = torch.where(first.bool(), 0.0, g[0, 0].double()).cumsum(0)
    pos = torch.arange(N)
    W = (sums[:, None] - sums[None]).exp() * ((doc[:, None] == doc[None]) & (pos[:, None] >= pos[None]))  # [t, s]
    unit = torch.eye(D, dtype=dtype)[pos % D].view(1, 1, N, D)
    ones = torch.eye(D, dtype=dtype)[:1].expand(N, D).reshape(1, 1, N, D)
    qk, vo = (ones, unit) if roles == "scores" else (unit, ones)
    out, _, dq, dk, dv, _ = _call(qk, qk, vo, g, None, None, vo, None)
    at = unit[0, 0].double()
    # out_t and dq_t: entry s of row t is the decay from s to t; dv_s and dk_s: entry t of row s
    for got, want in ((out, W @ at), (dv, W.T @ at)) if roles == "scores" else ((dq, W @ at), (dk, W.T @ at)):
        got = got[0, 0].double().cpu()
        assert ((got - want).abs() <= 1.1 * torch.finfo(dtype).eps / 2 * want).all(), ((got - want).abs() / want.clamp(min=1e-9)).max()


@pytest.mark.parametrize("held", HELD)
@pytest.mark.parametrize("at", AT[1:])
@pytest.mark.parametrize("dtype,D", [(torch.float32, 32), (torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 32), (torch.float16, 32)])
def test_gradients_before_a_dropped_state_gradient_on_cuda_cores(dtype, D, at, held):
    _before_a_drop(dtype, D, at, held)


@pytest.mark.parametrize("compiled", [True, False])
def test_a_state_of_inference_mode(compiled, monkeypatch):
    """As torch's own in-place operators: written to inside inference mode, refused outside of it, before anything is written."""
    from cottention_transformer_b200 import GatedScanState, _binding
    if not compiled:
        monkeypatch.setattr(_binding, "autograd", lambda: None)
    x = [t.cuda() for t in _inputs(1, 2, 1, 64, torch.bfloat16, seed=44)[:4]]
    with torch.inference_mode():
        s = GatedScanState(1, 2, 64)
        s.step(*x)
        before = s.state.clone()
    assert before.abs().sum() > 0
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        s.step(*x)
    assert torch.equal(s.state, before)


@pytest.mark.parametrize("code,name", [(1, "TMA"), (6, "accumulator"), (19, "gated walk: state update"), (21, "gated chunk: MMA")])
def test_a_wait_that_gave_up_is_named(code, name):
    """(The self-test's kernel polls a barrier four times, records the code and ends.)"""
    from cottention_transformer_b200 import _lib
    _lib.check(_lib.lib().cott_selftest_device_wait(4, code, 5, _lib.stream_ptr(torch.device("cuda"))), "selftest")
    with pytest.raises(RuntimeError, match=rf"stage {code} \({name}\) at chunk 5"):
        _lib.check_device_status()
    _lib.check_device_status()


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_captured_generation(dtype, D):
    """A prompt with a mask and a token loop (norm with rotation, step) in two graphs that share a memory pool and a state, replayed in
    turn with new inputs."""
    from cottention_transformer_b200 import GatedScanState, qk_norm_rotary
    B, H, N = 2, 3, 200
    runs = [[t if t is None else t.cuda() for t in _inputs(B, H, N + 1, D, dtype, seed=s, masked=True)] for s in (45, 46)]
    w = torch.rand(2, D, device="cuda") + 0.5
    ang = torch.rand(1, 8, device="cuda")

    def prompt(state, q, k, v, g, keep):
        state.reset()
        return state.prefill(*qk_norm_rotary(q, k, w[0], w[1]), v, g, keep=keep)

    def token(state, q, k, v, g):
        return state.step(*qk_norm_rotary(q, k, w[0], w[1], rotary=(ang.sin(), ang.cos())), v, g)

    def split(x):
        q, k, v, g, keep = x[:5]
        return [t[:, :, :N].clone() for t in (q, k, v, g)] + [keep[:, :N].clone()], [t[:, :, N:].clone() for t in (q, k, v, g)]

    want = []
    with torch.no_grad():
        for x in runs:
            state, (a, b) = GatedScanState(B, H, D), split(x)
            want.append([t.clone() for t in (prompt(state, *a), token(state, *b), token(state, *b), state.state)])
        state, (a, b) = GatedScanState(B, H, D), split(runs[0])
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            prompt(state, *a)
            token(state, *b)
        torch.cuda.synchronize()
        first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(first):
            out_a = prompt(state, *a)
        with torch.cuda.graph(second, pool=first.pool()):
            out_b = token(state, *b)
        for i in (1, 0, 1):
            new_a, new_b = split(runs[i])
            for s, t in zip(a + b, new_a + new_b):
                s.copy_(t)
            first.replay()
            got = [out_a.clone()]
            for _ in range(2):
                second.replay()
                got.append(out_b.clone())
            assert all(torch.equal(s, t) for s, t in zip((*got, state.state), want[i]))
