"""Plain fp64 implementations of the gated scan and of the q/k norm with rotation, on the CPU, token by token; their gradients by
autograd.  For the tests only."""
import torch


def gated_scan(q, k, v, g, keep=None, init=None):
    """(out, final state [B, H, value, key]) of S_t = e^(g_t) S_(t-1) + k_t v_t^T, out_t = S_t^T q_t."""
    B, H, N, D = q.shape
    S = q.new_zeros(B, H, D, D) if init is None else init
    outs = []
    for t in range(N):
        S1 = g[:, :, t].exp()[..., None, None] * S + v[:, :, t, :, None] * k[:, :, t, None, :]
        o = (S1 @ q[:, :, t, :, None])[..., 0]
        if keep is not None:
            m = keep[:, t].view(B, 1, 1, 1)
            S1, o = torch.where(m, S1, S), torch.where(m[..., 0], o, torch.zeros_like(o))
        S = S1
        outs.append(o)
    return (torch.stack(outs, 2) if outs else torch.zeros_like(v)), S


def qk_norm(x, w, sin=None, cos=None, eps=1e-6):
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    if sin is None:
        return y
    sin, cos = (t if t.dim() == 2 else t[:, None] for t in (sin, cos))
    rot = 2 * sin.shape[-1]
    a, b = y[..., 0:rot:2], y[..., 1:rot:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), y[..., rot:]], -1)


def rel(a, b):
    """|a - b| / |b| in the 2-norm; 0 where both vanish."""
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp(min=1e-300)).item() if b.norm() > 0 else a.norm().item()


def both_routes(monkeypatch_context, fn):
    """fn() through the compiled binding and through ctypes."""
    from cottention_transformer_b200 import _binding
    yield fn()
    with monkeypatch_context as m:
        m.setattr(_binding, "autograd", lambda: None)
        yield fn()
