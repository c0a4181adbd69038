"""8-bit 1x1 convolution without a GPU: sizes that its calls ask for and what they refuse (nothing is launched)."""
import ctypes

import pytest

from test_q8_cpu import BUF, lib


def test_sizes_of_the_calls():
    L = lib()
    a, b, c = ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t()
    M, C, N = 20000, 256, 128
    fwd = lambda x=BUF, M=M, C=C, sn=0, sh=None, sw=None, H=M, W=1, N=N, y=BUF, keep=0: (  # noqa: E731
        L.mgn_q8_conv1x1_fwd_bytes(x, M, C, sn or M * C, C if sh is None else sh, 0 if sw is None else sw, H, W, N, y, keep, ctypes.byref(a), ctypes.byref(b)))
    weights = (C * N + N // 128 * C) + (N * C + C // 128 * N)
    packed = M * C + C // 128 * M
    assert L.mgn_q8_conv1x1_bytes(M, C, N, ctypes.byref(a), ctypes.byref(c)) == 0 and a.value == weights + packed
    assert fwd(keep=1) == 0 and a.value == b.value == weights + packed
    assert fwd() == 0 and (a.value, b.value) == (weights, C * N + N // 128 * C)                # packed on the way
    for kw in (dict(x=BUF + 2), dict(y=BUF + 2), dict(sh=C + 8), dict(sn=1, H=M // 2)):        # ... or in a pass of its own
        assert fwd(**kw) == 0 and (a.value, b.value) == (weights + packed, C * N + N // 128 * C), kw
    for kw in (dict(M=-1), dict(C=0), dict(N=0), dict(C=65537), dict(N=65537)):
        assert fwd(**kw) == -22, kw
    bwd = lambda dx, dw, M=M, C=C, N=N: L.mgn_q8_conv1x1_bwd_bytes(M, C, N, dx, dw, ctypes.byref(c))  # noqa: E731
    part = ctypes.c_size_t()
    assert L.mgn_q8_wgrad_workspace_bytes(M, N, C, ctypes.byref(part)) == 0
    assert bwd(1, 1) == 0 and c.value == part.value and bwd(0, 1) == 0 and c.value == part.value and bwd(1, 0) == 0 and c.value == 0
    assert bwd(1, 0, N=19) == 0 and c.value == M * 24 * 2                                      # dy padded, packed on the way
    assert bwd(1, 0, N=640) == 0 and c.value == M * 640 + 5 * M                                # dy packed in a pass of its own
    for kw in (dict(M=-1), dict(C=0), dict(N=65537), dict(M=0x7fffff00, C=8, N=65536)):
        assert bwd(1, 1, **kw) == -22, kw
    assert bwd(1, 0, M=0x7fffff00, C=8, N=65536) == 0                                          # (no rows of dy past 32 bits without dw)
    assert L.mgn_q8_conv1x1_fwd_bytes(BUF, M, C, M * C, C, 0, M, 1, N, BUF, 0, None, ctypes.byref(b)) == -22
    assert L.mgn_q8_conv1x1_bwd_bytes(M, C, N, 1, 1, None) == -22


@pytest.mark.parametrize("sfx", ["", "_f16"])
def test_refusals_of_the_calls(sfx):
    L = lib()
    fwd = lambda x=BUF, M=8, C=16, sn=128, sh=16, sw=16, H=8, W=1, w=BUF, N=16, y=BUF, buf=BUF, nb=1 << 30: (  # noqa: E731
        getattr(L, "mgn_q8_conv1x1_fwd" + sfx)(x, M, C, sn, sh, sw, H, W, w, 0, C, 1, N, None, 0, y, 1, buf, nb, None))
    for kw in (dict(x=None), dict(y=None), dict(w=None), dict(buf=None), dict(buf=BUF + 8), dict(M=-1), dict(C=0), dict(N=0), dict(H=0, sn=0), dict(W=0), dict(H=3), dict(H=1, W=3),
               dict(sn=-1), dict(sh=-16), dict(sw=-1), dict(x=BUF + 1), dict(y=BUF + 1)):
        assert fwd(**kw) == -22, kw
    assert fwd(nb=64) == -28
    bwd = lambda dy=BUF, M=64, C=16, N=16, buf=BUF, dx=BUF, dw=BUF, db=None, ws=BUF, nb=1 << 30: (  # noqa: E731
        getattr(L, "mgn_q8_conv1x1_bwd" + sfx)(dy, M, C, N, buf, dx, dw, db, ws, nb, None))
    for kw in (dict(dy=None), dict(dy=BUF + 2), dict(buf=None), dict(buf=BUF + 2), dict(ws=None), dict(ws=BUF + 4), dict(dx=None, dw=None), dict(dw=None, db=BUF), dict(M=0), dict(C=0),
               dict(N=70000)):
        assert bwd(**kw) == -22, kw
    assert bwd(nb=64) == -28
