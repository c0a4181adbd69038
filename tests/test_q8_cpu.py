"""8-bit operators without a GPU: what the C-ABI and the Python entry points refuse (nothing is launched)."""
import ctypes

import pytest
import torch


def lib():
    from mgnet_amd import _C, build
    build.build()
    return _C.lib()


BUF = 0x100000      # an aligned address that no refused call touches


def test_sizes():
    L = lib()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.mgn_q8_bytes(5, 129, ctypes.byref(a), ctypes.byref(b)) == 0 and (a.value, b.value) == (5 * 144, 2 * 16)
    assert L.mgn_q8_bytes(0, 1, ctypes.byref(a), ctypes.byref(b)) == 0 and (a.value, b.value) == (0, 0)
    for M, C in ((-1, 8), (0x7fffff01, 8), (4, 0), (4, (1 << 20) + 1)):
        assert L.mgn_q8_bytes(M, C, ctypes.byref(a), ctypes.byref(b)) == -22
    assert L.mgn_q8_wgrad_workspace_bytes(1000, 40, 96, ctypes.byref(a)) == 0 and a.value >= 4 * (40 * 96 + 40)
    assert L.mgn_q8_wgrad_workspace_bytes(0, 40, 96, ctypes.byref(a)) == -22
    r = ctypes.c_int()
    assert L.mgn_q8_tail_partial_rows(100, 64, ctypes.byref(r)) == 0 and r.value >= 1
    for M, C in ((0, 64), (10, 12), (10, 0), (10, 8200)):
        assert L.mgn_q8_tail_partial_rows(M, C, ctypes.byref(r)) == -22


@pytest.mark.parametrize("sfx", ["", "_f16"])
def test_c_refusals(sfx):
    L = lib()
    fn = lambda n: getattr(L, n + sfx)  # noqa: E731
    pack = lambda x=BUF, dt=1, M=8, C=16, sn=16, sh=0, sw=0, H=1, W=1, c=BUF, s=BUF: fn("mgn_q8_pack")(x, dt, M, C, sn, sh, sw, H, W, c, s, None)  # noqa: E731
    assert pack(M=0) == 0
    for kw in (dict(x=None), dict(c=None), dict(s=None), dict(dt=2), dict(M=-1), dict(M=0x7fffff01), dict(C=0), dict(sn=-1), dict(H=0), dict(H=3, W=1), dict(c=BUF + 8),
               dict(s=BUF + 4), dict(x=BUF + 1)):
        assert pack(**kw) == -22, kw
    unpack = lambda c=BUF, s=BUF, M=8, C=16, y=BUF, dt=1: fn("mgn_q8_unpack")(c, s, M, C, y, dt, None)  # noqa: E731
    assert unpack(M=0) == 0
    for kw in (dict(c=None), dict(s=None), dict(y=None), dict(dt=-1), dict(C=0), dict(c=BUF + 4), dict(y=BUF + 1)):
        assert unpack(**kw) == -22, kw
    weight = lambda w=BUF, dt=0, N=4, K=4, c=BUF, s=BUF, ct=None, st=None: fn("mgn_q8_pack_weight")(w, dt, K, 1, N, K, c, s, ct, st, None)  # noqa: E731
    for kw in (dict(w=None), dict(N=0), dict(K=0), dict(c=None), dict(s=None), dict(c=None, s=None), dict(ct=BUF), dict(st=BUF), dict(dt=3)):
        assert weight(**kw) == -22, kw
    mm = lambda a=BUF, sa=BUF, M=4, b=BUF, sb=BUF, N=4, K=4, act=0, slope=0.0, out=BUF, f32=0, ldo=4: fn("mgn_q8_matmul")(a, sa, M, b, sb, N, K, None, act, slope, out, f32, ldo, None)  # noqa: E731
    assert mm(M=0) == 0
    for kw in (dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(N=0), dict(K=0), dict(act=3), dict(act=2, slope=1.5), dict(act=2, slope=-0.1), dict(ldo=3), dict(a=BUF + 8), dict(out=BUF + 1), dict(M=-1)):
        assert mm(**kw) == -22, kw
    wg = lambda dy=BUF, ldy=8, M=4, N=8, c=BUF, s=BUF, K=8, dw=BUF, ws=BUF, nb=1 << 30: fn("mgn_q8_wgrad")(dy, ldy, M, N, c, s, K, dw, None, ws, nb, None)  # noqa: E731
    for kw in (dict(dy=None), dict(c=None), dict(dw=None), dict(ws=None), dict(ldy=7), dict(ldy=12), dict(M=0), dict(N=0), dict(K=70000), dict(dy=BUF + 2)):
        assert wg(**kw) == -22, kw
    assert wg(nb=16) == -28
    args = [BUF] * 4
    assert fn("mgn_q8_tail_fwd")(*args, 8, 12, BUF, BUF, BUF, BUF, None) == -22
    assert fn("mgn_q8_tail_fwd")(*args, 8, 16, BUF, BUF, None, BUF, None) == -22
    assert fn("mgn_q8_tail_stats")(BUF + 2, 8, 16, BUF, BUF, None) == -22
    assert fn("mgn_q8_tail_bwd_reduce")(BUF, BUF, BUF, None, BUF, BUF, BUF, 8, 16, BUF, BUF, BUF, BUF, None) == -22
    assert fn("mgn_q8_tail_bwd_apply")(BUF, BUF, BUF, BUF, BUF, BUF, BUF, 0.0, 1e-5, 8, 16, BUF, None) == -22


def test_python_refuses_cpu_tensors_and_wrong_shapes():
    from mgnet_amd.modeling import ops
    from mgnet_amd.modeling.layers import InPlaceABNSync
    x = torch.zeros(1, 16, 4, 4, dtype=torch.bfloat16)
    for f in (lambda: ops.q8_pack(x), lambda: ops.conv1x1_q8(x, torch.zeros(8, 16, 1, 1)), lambda: ops.abn_add_relu_q8(x, InPlaceABNSync(16, activation="identity"), x)):
        with pytest.raises(RuntimeError):
            f()
    for f in (lambda: ops.q8_pack(x[0]), lambda: ops.q8_pack([1.0]), lambda: ops.q8_matmul(x, x)):
        with pytest.raises(ValueError):
            f()


def test_weight_gradient_ranges():
    """row ranges stay within 32-bit offsets, or the sizes are refused before anything is computed"""
    L = lib()
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    for M, N, K in ((66000, 16384, 512), (262144, 4096, 4096), (0x7fffff00, 64, 64), (1 << 27, 19, 320)):
        assert L.mgn_q8_wgrad_workspace_bytes(M, N, K, ctypes.byref(a)) == 0
        per = 4 * ((N * K + N + 3) // 4 * 4)
        assert a.value % per == 0
        rows = -(-(-(-M // (a.value // per))) // 64) * 64
        assert (rows + 256) * max(2 * ((N + 7) // 8 * 8), (K + 15) // 16 * 16) <= 0x7fffffff, (M, N, K)
    assert L.mgn_q8_wgrad_workspace_bytes(0x7fffff00, 65536, 8, ctypes.byref(a)) == -22
    assert L.mgn_q8_conv1x1_bytes(0x7fffff00, 8, 65536, ctypes.byref(a), ctypes.byref(b)) == -22
