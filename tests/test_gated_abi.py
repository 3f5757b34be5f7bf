"""CPU tests of the checks of the gated-scan and q/k-norm entry points: a bad call is an error before any CUDA call."""
import ctypes

import pytest
import torch

F32, F64, F16, BF16 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def L():
    from cottention_transformer_b200 import _lib, build
    build.build()
    return _lib.lib()


def _fwd(L, ptrs=(None,) * 11, B=1, H=1, N=8, D=64, dtype=BF16, gate=BF16):
    return L.cott_gated_scan_fwd(*ptrs, B, H, N, D, dtype, gate, None)


def test_gated_scan_checks(L):
    assert _fwd(L, dtype=F64) == 3 and _fwd(L, dtype=9) == 3 and _fwd(L, gate=F16) == 3
    assert _fwd(L, D=48) == 2 and _fwd(L, N=-1) == 2 and _fwd(L, B=1 << 20, H=1 << 10, N=1 << 20) == 2
    assert _fwd(L) == 1 and b"q" in L.cott_last_error()
    assert _fwd(L, N=0) == 0 and _fwd(L, B=0) == 0  # nothing to do
    p = 0x10000  # never read: the checks come first
    good = [p, p, p, p, None, None, p, None, p, p, None]
    for i, name in ((0, b"q"), (1, b"k"), (2, b"v"), (6, b"out")):
        bad = list(good)
        bad[i] = p + 8
        assert _fwd(L, bad) == 5 and name in L.cott_last_error()
    for i in (3, 8):
        bad = list(good)
        bad[i] = None
        assert _fwd(L, bad) == 1
    for i in (5, 7, 8):
        bad = list(good)
        bad[i] = p + 4
        assert _fwd(L, bad) == 5
    from cottention_transformer_b200 import _lib
    lay = _lib.CottGatedLayout()
    for name in ("q", "k", "v", "out"):
        setattr(lay, name, _lib.CottStrides(64 * 8, 64 * 8, 64))
    lay.v = _lib.CottStrides(64 * 8, 64 * 8, 68)
    good[10] = ctypes.addressof(lay)
    assert _fwd(L, good) == 5 and b"strides of v" in L.cott_last_error()


def test_gated_scan_backward_checks(L):
    p = 0x10000
    good = [p, p, p, p, None, 0, p, p, None, p, p, p, p, p, None, None]

    def bwd(a, **kw):
        s = dict(B=1, H=1, N=8, D=64, dtype=F32, gate=F32) | kw
        return L.cott_gated_scan_bwd(*a, *s.values(), None)

    assert bwd([None] * 5 + [0] + [None] * 10) == 1
    assert bwd(good, D=256) == 2 and bwd(good, dtype=F64) == 3 and bwd(good, N=0) == 0
    for i in (3, 6, 9, 13):
        bad = list(good)
        bad[i] = None
        assert bwd(bad) == 1
    for i in (0, 7, 8, 9, 10, 11, 12, 14):
        bad = list(good)
        bad[i] = p + 4
        assert bwd(bad) == 5


def test_sizes_of_the_buffers(L):
    for dtype in (F32, F16, BF16):
        for D in (32, 64, 128):
            n = L.cott_gated_scan_states_bytes(2, 3, 1000, D, dtype)
            assert n > 0 and L.cott_gated_scan_states_bytes(2, 3, 1001, D, dtype) >= n
            assert L.cott_gated_scan_workspace_bytes(2, 3, 1000, D, dtype, 1) > 0
    assert L.cott_gated_scan_states_bytes(2, 3, 0, 64, F32) == 0 and L.cott_gated_scan_states_bytes(2, 3, 8, 48, F32) == 0
    # in 64 bits
    assert L.cott_gated_scan_states_bytes(1, 64, 1 << 20, 128, F32) > 1 << 32


def test_step_and_norm_checks(L):
    p = 0x10000
    step = lambda a, **kw: L.cott_gated_step(*a, *(dict(B=1, H=1, T=1, D=64, dtype=F16, gate=F16) | kw).values(), None)  # noqa: E731
    good = [p, p, p, p, p, p, None]
    assert step([None] * 7) == 1 and step(good, T=0) == 0 and step(good, D=16) == 2 and step(good, gate=BF16) == 3 and step(good, dtype=F64) == 3
    for i in (0, 1, 2, 3, 5):
        bad = list(good)
        bad[i] = p + 8
        assert step(bad) == 5
    from cottention_transformer_b200 import _lib
    norm = lambda a, **kw: L.cott_qk_norm_fwd(*a, *(dict(B=1, Hq=2, Hk=1, N=3, D=64, eps=1e-6, dtype=BF16, w=F32) | kw).values(), None)  # noqa: E731
    good = [p, p, p, p, None, p, p, None]
    assert norm([None] * 8) == 1 and norm(good, N=0) == 0 and norm(good, D=80) == 2 and norm(good, dtype=F64) == 3 and norm(good, w=F16) == 3
    assert norm(good, Hk=0) == 2 and norm(good, B=1 << 20, N=1 << 20) == 2
    for i in (0, 1, 5, 6):
        bad = list(good)
        bad[i] = p + 8
        assert norm(bad) == 5
    for rot, code in ((4, 2), (12, 2), (72, 2)):
        tab = _lib.CottRotaryTables(p, p, rot, 0)
        bad = list(good)
        bad[4] = ctypes.addressof(tab)
        assert norm(bad) == code
    tab = _lib.CottRotaryTables(p, None, 16, 0)
    assert norm(good[:4] + [ctypes.addressof(tab)] + good[5:]) == 1
    bwd = lambda a, **kw: L.cott_qk_norm_bwd(*a, *(dict(B=1, Hq=2, Hk=1, N=3, D=64, eps=1e-6, dtype=BF16, w=F32) | kw).values(), None)  # noqa: E731
    good = [p, p, p, p, None, p, p, p, p, p, p, p, None]
    for i, code in ((7, 1), (10, 1), (11, 1), (0, 1), (9, 1)):
        bad = list(good)
        bad[i] = None
        assert bwd(bad) == code


def test_cpu_tensors_are_refused():
    from cottention_transformer_b200 import gated_scan, gated_scan_step, qk_norm_rotary
    q, g, w = torch.zeros(1, 1, 4, 64), torch.zeros(1, 1, 4), torch.ones(64)
    for call in (lambda: gated_scan(q, q, q, g), lambda: gated_scan_step(torch.zeros(1, 1, 64, 64), q, q, q, g), lambda: qk_norm_rotary(q, q, w, w)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
