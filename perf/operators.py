"""The operators of a gated linear-attention layer: what is measured of them.

Each case is one dict of plain values.  ``listed()`` holds the named cases, ``draw()`` gives further ones of the same ranges,
``prepare()`` makes what a caller holds before the call, ``run()`` is one pass (in elementary torch operations, or where ``own``
is true through this package's entry points), ``exact()`` the same outputs from the definition in 64 bits and ``work()`` the bytes
and operations that no implementation of the pass can avoid.

Operators (``op`` of a case):
  train    ``gated_scan`` forward and backward: S_t = e^(g_t) S_(t-1) + k_t v_t^T, out_t = S_t^T q_t, and the gradients of q, k, v, g
  prompt   ``gated_scan`` forward with the state that the prompt leaves, from an empty state or one that is there already
  step     ``gated_scan_step``: one token per sequence on the fp32 states, in place
  norm     ``qk_norm_rotary`` forward and backward: RMS norm of every head of q and k with a learned weight, and the rotary
           embedding, on the q and k of a packed projection
  token    ``qk_norm_rotary`` forward for one new token per sequence, each at a position of its own
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64


def listed():
    return [
        # the smallest training call: a short sequence of a small model; launches and host work count here
        dict(name="train_small", op="train", B=1, H=4, N=200, D=64, dtype="bf16", mask=False, docs=False),
        # a batch of 4k-token sequences with 16 heads of 64: the size the plain scan of this package is benchmarked at
        dict(name="train_4k", op="train", B=8, H=16, N=4096, D=64, dtype="bf16", mask=False, docs=False),
        # a padded batch whose length is no multiple of any tile, in fp16, with a head count that does not fill the GPU
        dict(name="train_padded", op="train", B=7, H=12, N=1531, D=64, dtype="fp16", mask=True, docs=False),
        # long-context training of one row of packed documents: the state is dropped where a document begins
        dict(name="train_long", op="train", B=1, H=16, N=65536, D=64, dtype="bf16", mask=False, docs=True),
        # the wide heads
        dict(name="train_d128", op="train", B=1, H=16, N=16384, D=128, dtype="bf16", mask=False, docs=False),
        # fp32, the mode that a model is checked in
        dict(name="train_fp32", op="train", B=2, H=8, N=1024, D=64, dtype="fp32", mask=False, docs=False),
        # serving: a batch of prompts
        dict(name="prompt", op="prompt", B=4, H=16, N=777, D=64, dtype="bf16", start=False),
        # serving: one token per sequence and step, a batch that fills the GPU
        dict(name="step_d64", op="step", B=64, H=16, N=1, D=64, dtype="bf16"),
        dict(name="step_d128", op="step", B=64, H=16, N=1, D=128, dtype="bf16"),
        # q and k of a training batch, weights in fp32 as an optimizer keeps them
        dict(name="norm_4k", op="norm", B=8, H=16, N=4096, D=64, dtype="bf16", weights="fp32", rotary=64, batched=False),
        # wide heads with a partial rotation, positions of each sequence's own, an odd length
        dict(name="norm_d128", op="norm", B=3, H=12, N=1531, D=128, dtype="fp16", weights="fp16", rotary=32, batched=True),
        # the new token of every sequence in a batch that is being generated
        dict(name="token", op="token", B=64, H=16, N=1, D=64, dtype="bf16", weights="bf16", rotary=64, batched=True),
    ]


def _log(rng, lo, hi):
    """An integer between lo and hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case.  A drawn training case has at most the elements of the largest listed one of its kind."""
    op = rng.choice(["train", "train", "long", "wide", "fp32", "prompt", "prompt", "step", "norm", "norm", "token"])
    half = rng.choice(["bf16", "bf16", "fp16"])
    if op == "train":  # batches of short and ordinary sequences
        H, N = rng.choice([1, 4, 6, 8, 12, 16]), _log(rng, 1, 4096)
        return dict(op="train", B=_log(rng, 1, max(1, min(16, 524288 // (H * N)))), H=H, N=N, D=64, dtype=half, mask=rng.random() < 0.5, docs=rng.random() < 0.3)
    if op == "long":  # one sequence
        H = rng.choice([4, 8, 12, 16])
        return dict(op="train", B=1, H=H, N=_log(rng, 4096, 1048576 // H), D=64, dtype=half, mask=False, docs=rng.random() < 0.5)
    if op == "wide":
        H, N = rng.choice([4, 8, 12, 16]), _log(rng, 64, 16384)
        return dict(op="train", B=_log(rng, 1, max(1, min(8, 262144 // (H * N)))), H=H, N=N, D=128, dtype=half, mask=rng.random() < 0.3, docs=False)
    if op == "fp32":
        return dict(op="train", B=rng.choice([1, 2]), H=rng.choice([4, 8]), N=_log(rng, 1, 1024), D=rng.choice([32, 64]), dtype="fp32", mask=rng.random() < 0.5, docs=rng.random() < 0.3)
    if op == "prompt":
        return dict(op="prompt", B=_log(rng, 1, 8), H=rng.choice([8, 12, 16]), N=_log(rng, 2, 4096), D=rng.choice([64, 64, 128]), dtype=half, start=rng.random() < 0.5)
    if op == "step":
        return dict(op="step", B=_log(rng, 1, 64), H=rng.choice([4, 8, 12, 16]), N=1, D=rng.choice([64, 128]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    if op == "norm":
        D, H, N = rng.choice([64, 128]), rng.choice([6, 8, 12, 16]), _log(rng, 16, 4096)
        B = _log(rng, 1, max(1, min(16, 524288 * 64 // (D * H * N))))
        return dict(op="norm", B=B, H=H, N=N, D=D, dtype=rng.choice(["bf16", "fp16", "fp32"]) if B * H * N * D < 8388608 else half, weights="fp32", rotary=rng.choice([0, 16, D]), batched=rng.random() < 0.3)
    return dict(op="token", B=_log(rng, 1, 256), H=rng.choice([4, 8, 12, 16]), N=1, D=rng.choice([64, 128]), dtype=half, weights=rng.choice([half, "fp32"]), rotary=rng.choice([0, 32, 64]), batched=True)


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True)


def prepare(case, seed):
    op, B, H, N, D, dt = case["op"], case["B"], case["H"], case["N"], case["D"], DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=dt):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=gen)

    st = dict(op=op)
    if op in ("norm", "token"):
        qkv = randn(B, N, 3, H, D) * 2  # the projection's output; q and k are views of it, as a model takes them
        st["q"], st["k"] = (qkv[:, :, i].transpose(1, 2).requires_grad_(op == "norm") for i in (0, 1))
        wt = DTYPES[case["weights"]]
        st["qw"], st["kw"] = ((1 + 0.2 * randn(D, dtype=torch.float32)).to(wt).requires_grad_(op == "norm") for _ in range(2))
        st["rotary"] = None
        if case["rotary"]:
            half = case["rotary"] // 2
            pos = torch.arange(N, device="cuda").float()
            if case["batched"]:  # every sequence at a position of its own
                pos = pos + torch.randint(0, 4096, (B, 1), device="cuda", generator=gen)
            angle = pos[..., None] * 10000.0 ** (-torch.arange(half, device="cuda").float() / half)
            st["rotary"] = (torch.sin(angle), torch.cos(angle))
        if op == "norm":
            st["dq"], st["dk"] = randn(B, N, H, D).transpose(1, 2), randn(B, N, H, D).transpose(1, 2)
        return st
    # unit rows, as the plain scan of this package sees them; gates of heads that remember a few tokens and of heads that remember
    # some hundred
    st["q"], st["k"], st["v"] = _unit(randn(B, H, N, D)), _unit(randn(B, H, N, D)), randn(B, H, N, D)
    level = torch.linspace(0.5, 6.0, H, device="cuda") if H > 1 else torch.full((1,), 4.0, device="cuda")
    g = torch.nn.functional.logsigmoid(level[None, :, None] + randn(B, H, N, dtype=torch.float32))
    if case.get("docs"):
        first = torch.rand(B, 1, N, device="cuda", generator=gen) < 1 / 1500
        g = g.masked_fill(first, float("-inf"))
    st["g"] = g.to(dt)
    st["keep"] = st["init"] = None
    if op == "train":
        if case["mask"]:  # right padding, as a batch of sentences of different lengths has it
            lengths = torch.randint(max(1, N // 2), N + 1, (B, 1), device="cuda", generator=gen)
            st["keep"] = torch.arange(N, device="cuda").unsqueeze(0) < lengths
        for name in ("q", "k", "v", "g"):
            st[name].requires_grad_()
        st["dout"] = randn(B, H, N, D)
    elif op == "step" or case["start"]:  # in the middle of a generation
        st["init"] = randn(B, H, D, D, dtype=torch.float32) * D ** -0.5
    return st


def _plain_scan(q, k, v, g, keep, init):
    """Outputs and final state ([B, H, value, key]) in fp32: chunks of 64 positions, the states before them as one weighted sum
    over the chunks; exponents in fp64, since they are differences of long sums."""
    B, H, N, D = q.shape
    q, k, v = q.float(), k.float(), v.float()
    g = g.double().clamp(min=-200.0)  # e^-200 = 0 in fp32
    if keep is not None:
        m = keep[:, None, :, None]
        q, k, v, g = q * m, k * m, v * m, g * m[..., 0]
    pad = -N % CHUNK
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad)).view(B, H, -1, CHUNK, D) for t in (q, k, v))
    g = torch.nn.functional.pad(g, (0, pad)).view(B, H, -1, CHUNK)
    G = g.cumsum(-1)
    total = G[..., -1]
    end = total.cumsum(-1)
    start = end - total
    tril = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    decay = (G[..., :, None] - G[..., None, :]).masked_fill(~tril, float("-inf")).exp().float()
    out = (q @ k.transpose(-1, -2) * decay) @ v
    U = (k * (total[..., None] - G).exp().float()[..., None]).transpose(-1, -2) @ v  # what each chunk adds to the state at its end
    nc = U.shape[2]
    before = torch.ones(nc, nc, dtype=torch.bool, device=q.device).tril(-1)
    mix = (start[..., :, None] - end[..., None, :]).masked_fill(~before, float("-inf")).exp().float()
    S = (mix @ U.flatten(-2)).view_as(U)
    final = (((end[..., -1:] - end).exp().float()[..., None, :]) @ U.flatten(-2)).view(B, H, D, D)
    if init is not None:
        init = init.transpose(-1, -2)
        S = S + start.exp().float()[..., None, None] * init[:, :, None]
        final = final + end[..., -1].exp().float()[..., None, None] * init
    out = out + (q * G.exp().float()[..., None]) @ S
    return out.reshape(B, H, -1, D)[:, :, :N], final.transpose(-1, -2)


def _plain_norm(x, w, rotary, eps=1e-6):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps) * w.float()
    if rotary is not None:
        sin, cos = (t if t.dim() == 2 else t[:, None] for t in rotary)
        rot = 2 * sin.shape[-1]
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), y[..., rot:]], -1)
    return y.to(x.dtype)


def run(st):
    op = st["op"]
    if own:
        from cottention_transformer_b200 import gated_scan, gated_scan_step, qk_norm_rotary
    if op in ("norm", "token"):
        if own:
            q, k = qk_norm_rotary(st["q"], st["k"], st["qw"], st["kw"], rotary=st["rotary"])
        else:
            q, k = _plain_norm(st["q"], st["qw"], st["rotary"]), _plain_norm(st["k"], st["kw"], st["rotary"])
        if op == "token":
            return q, k
        return q, k, *torch.autograd.grad((q, k), (st["q"], st["k"], st["qw"], st["kw"]), (st["dq"], st["dk"]))
    if op == "train":
        if own:
            out = gated_scan(st["q"], st["k"], st["v"], st["g"], keep=st["keep"])
        else:
            out = _plain_scan(st["q"], st["k"], st["v"], st["g"], st["keep"], None)[0].to(st["q"].dtype)
        return out, *torch.autograd.grad(out, (st["q"], st["k"], st["v"], st["g"]), st["dout"])
    if op == "prompt":
        if own:
            return gated_scan(st["q"], st["k"], st["v"], st["g"], initial_state=st["init"], return_state=True)
        out, state = _plain_scan(st["q"], st["k"], st["v"], st["g"], None, st["init"])
        return out.to(st["q"].dtype), state
    state = st["init"]
    if own:
        return gated_scan_step(state, st["q"], st["k"], st["v"], st["g"]), state
    q, k, v = (st[n].float() for n in "qkv")
    state.mul_(st["g"].float().exp()[..., None]).add_(v.transpose(-1, -2) * k)
    return (q @ state.transpose(-1, -2)).to(st["q"].dtype), state


def _exact_scan(q, k, v, g, keep, init, dout):
    """The recurrence in fp64, a chunk of 32 positions at a time, and its gradients from the formulas: dq, dk, dv as weighted sums of
    rows, dg as the derivative to what crosses a position."""
    C, (B, H, N, D) = 32, q.shape
    q, k, v, g = (t.detach().double() for t in (q, k, v, g))
    g = g.clamp(min=-1000.0)
    if keep is not None:
        q, k, v = (t.masked_fill(~keep[:, None, :, None], 0) for t in (q, k, v))
        g = g.masked_fill(~keep[:, None], 0)
    S = q.new_zeros(B, H, D, D) if init is None else init.double().transpose(-1, -2)
    out, states = torch.empty_like(v), []
    spans = [(a, min(a + C, N)) for a in range(0, N, C)]

    def weights(a, b):
        G = g[:, :, a:b].cumsum(-1)
        return G.exp()[..., None], (G[..., -1:] - G).exp()[..., None], (G[..., :, None] - G[..., None, :]).tril().exp().tril(), G[..., -1].exp()[..., None, None]

    for a, b in spans:
        states.append(S)
        head, tail, W, A = weights(a, b)
        Q, K, V = q[:, :, a:b], k[:, :, a:b], v[:, :, a:b]
        out[:, :, a:b] = head * (Q @ S) + (Q @ K.mT * W) @ V
        S = A * S + (tail * K).mT @ V
    final = S
    if dout is None:
        return out, final.mT
    do = dout.double() if keep is None else dout.double().masked_fill(~keep[:, None, :, None], 0)
    dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(g)
    R, after = torch.zeros_like(S), final
    for (a, b), S in zip(reversed(spans), reversed(states)):
        head, tail, W, A = weights(a, b)
        Q, K, V, dO = q[:, :, a:b], k[:, :, a:b], v[:, :, a:b], do[:, :, a:b]
        E, P = dO @ V.mT * W, Q @ K.mT * W
        dq[:, :, a:b] = head * (dO @ S.mT) + E @ K
        dk[:, :, a:b] = tail * (V @ R.mT) + E.mT @ Q
        dv[:, :, a:b] = tail * (K @ R) + P.mT @ dO
        d = (Q * dq[:, :, a:b]).sum(-1) - (K * dk[:, :, a:b]).sum(-1)
        dg[:, :, a:b] = d.flip(-1).cumsum(-1).flip(-1) + (after * R).sum((-1, -2))[..., None]
        R = A * R + (head * Q).mT @ dO
        after = S
    if keep is not None:
        dg = dg.masked_fill(~keep[:, None], 0)
    if init is None:  # nothing is there before the first position that its gate could decay
        dg[:, :, 0] = 0
    return out, dq, dk, dv, dg.masked_fill(g <= -1000.0, 0)


def _exact_norm(x, w, rotary, dy):
    x, w = x.detach().double(), w.detach().double()
    r = (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    n = x * r

    def turn(y, sign):
        if rotary is None:
            return y
        sin, cos = (t.double() if t.dim() == 2 else t.double()[:, None] for t in rotary)
        y, rot = y.clone(), 2 * sin.shape[-1]
        z = torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * torch.complex(cos, sign * sin)
        y[..., :rot] = torch.view_as_real(z).flatten(-2)
        return y

    y = turn(n * w, 1)
    if dy is None:
        return y, None, None
    e = turn(dy.double(), -1)
    f = e * w
    return y, r * (f - n * (f * n).mean(-1, keepdim=True)), (e * n).sum((0, 1, 2))


def exact(case, seed):
    st = prepare(case, seed)
    op = st["op"]
    if op in ("norm", "token"):
        (q, dq, dqw), (k, dk, dkw) = (_exact_norm(st[a], st[a + "w"], st["rotary"], st.get("d" + a)) for a in "qk")
        return (q, k) if op == "token" else (q, k, dq, dk, dqw, dkw)
    return _exact_scan(st["q"], st["k"], st["v"], st["g"], st["keep"], st["init"], st.get("dout"))


def work(case):
    B, H, N, D = case["B"], case["H"], case["N"], case["D"]
    e, rows = DTYPES[case["dtype"]].itemsize, B * H * N
    tensor, state, op = rows * D * e, B * H * D * D * 4, case["op"]
    if op == "train":  # q, k, v, dout in; out, dq, dk, dv out; the gates and their gradient
        return {"bytes": 8 * tensor + 2 * rows * e, "flops": (4 + 8) * rows * D * D}
    if op == "prompt":
        return {"bytes": 4 * tensor + rows * e + state * (2 if case["start"] else 1), "flops": 4 * rows * D * D}
    if op == "step":
        return {"bytes": 2 * state + 4 * tensor + rows * e, "flops": 4 * rows * D * D}
    tables = 4 * case["rotary"] * N * (B if case["batched"] else 1)
    if op == "norm":  # q, k and the gradients of the results in; the results and the gradients of q, k out
        return {"bytes": 8 * tensor + tables, "flops": 30 * rows * D}
    return {"bytes": 4 * tensor + tables, "flops": 12 * rows * D}
