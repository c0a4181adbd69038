"""MODEL.Q8 in the training step: every call that the network makes of the 8-bit 1x1 convolution and block tail, forward and backward, with the
step's own activations, weights and gradients, against the definition in 64 bits.  Bounds: as in test_q8_gpu.py (half a step of the result, fp32 sums,
the matrix instruction's cut); the tail's statistics are taken as the step has them and checked for themselves."""
import pytest
import torch

from test_q8_gpu import BF, HF, equal, group_tol, q8_ref, rows
from test_q8_model_gpu import _trainer

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _give_the_memory_back():
    yield
    torch.cuda.empty_cache()


def _recorded(monkeypatch):
    """(convolutions, tails): one dict per forward call, joined by its backward call's"""
    from mgnet_amd import _C
    convs, tails = {}, {}
    fwd, bwd, tail_train, tail_fwd, tail_bwd = (getattr(_C, n) for n in ("q8_conv1x1_fwd", "q8_conv1x1_bwd", "q8_tail_train_fwd", "q8_tail_fwd", "q8_tail_train_bwd"))
    copy = lambda t: None if t is None else t.detach().clone()  # noqa: E731

    def conv_fwd(x, M, C, sn, sh, sw, H, W, w, N, bias, relu, y, keep):
        out = fwd(x, M, C, sn, sh, sw, H, W, w, N, bias, relu, y, keep)
        X = torch.as_strided(x.detach(), (M // (H * W), H, W, C), (sn, sh, sw, 1)).reshape(M, C)
        convs[out[0].data_ptr()] = dict(x=copy(X), w=copy(w), b=copy(bias), relu=relu, y=copy(rows(y)), buf=out[0])      # (buf: its address stays its own)
        return out

    def conv_bwd(dy, M, C, N, buf, dx, dw, db):
        bwd(dy, M, C, N, buf, dx, dw, db)
        convs[buf.data_ptr()].update(dy=copy(rows(dy)), dx=None if dx is None else copy(rows(dx)), dw=copy(dw), db=copy(db))

    def keep_tail(x, shortcut, coef, y, buf):
        tails[buf.data_ptr()] = dict(x=copy(rows(x)), s=copy(rows(shortcut)), coef=copy(coef), y=copy(rows(y)), buf=buf)

    def train_fwd(x, shortcut, M, C, weight, bias, eps, momentum, rm, rv, coef, y, buf):
        tail_train(x, shortcut, M, C, weight, bias, eps, momentum, rm, rv, coef, y, buf)
        keep_tail(x, shortcut, coef, y, buf)

    def plain_fwd(x, shortcut, coef, M, C, y, buf):
        tail_fwd(x, shortcut, coef, M, C, y, buf)
        keep_tail(x, shortcut, coef, y, buf)

    def train_bwd(buf, g, coef, weight, eps, M, C, dz, dx):
        out = tail_bwd(buf, g, coef, weight, eps, M, C, dz, dx)
        tails[buf.data_ptr()].update(g=copy(rows(g)), w=copy(weight), eps=eps, dz=copy(rows(dz)), dx=None if dx is None else copy(rows(dx)), out=copy(out))
        return out
    for name, f in (("q8_conv1x1_fwd", conv_fwd), ("q8_conv1x1_bwd", conv_bwd), ("q8_tail_train_fwd", train_fwd), ("q8_tail_fwd", plain_fwd), ("q8_tail_train_bwd", train_bwd)):
        monkeypatch.setattr(_C, name, f)
    return convs, tails


def _check_conv(c, dtype):
    half, tiny = (2.0 ** -8, 1e-36) if dtype == BF else (2.0 ** -11, 2.0 ** -25)
    x8, w8 = q8_ref(c["x"])[0], q8_ref(c["w"], True)[0]
    N, C = w8.shape
    bias = torch.zeros(N, dtype=torch.float64, device="cuda") if c["b"] is None else c["b"].double()
    ref, S = x8 @ w8.t() + bias, x8.abs() @ w8.abs().t() + bias.abs()
    ref = ref.clamp(min=0) if c["relu"] else ref
    assert bool(((c["y"].double() - ref).abs() <= half * ref.abs() + (1 + half) * ((C + 2) * 2.0 ** -23 * S + group_tol(x8, w8)) + tiny).all())
    g, M = c["dy"], x8.shape[0]
    assert not c["relu"] or not bool(g[~(c["y"] > 0)].any())
    if c["dx"] is not None:
        g8 = q8_ref(g)[0]
        ref, S = g8 @ w8, g8.abs() @ w8.abs()
        assert bool(((c["dx"].double() - ref).abs() <= half * ref.abs() + (1 + half) * ((N + 2) * 2.0 ** -23 * S + group_tol(g8, w8.t())) + tiny).all())
    g = g.double()
    assert bool(((c["dw"].view(N, C).double() - g.t() @ x8).abs() <= (M + 2) * 2.0 ** -23 * (g.abs().t() @ x8.abs()) + 1e-36).all())
    assert c["db"] is None or bool(((c["db"].double() - g.sum(0)).abs() <= (M + 2) * 2.0 ** -23 * g.abs().sum(0) + 1e-36).all())


def _check_tail(t, dtype):
    half, tiny = (2.0 ** -8, 1e-36) if dtype == BF else (2.0 ** -11, 2.0 ** -25)
    u = 2.0 ** -15                                       # (fp32 sums and a handful of fp32 operations: see test_q8_gpu.check_tail)
    x, s, y, w = (t[k].double() for k in ("x", "s", "y", "w"))
    scale, offset, mean, rstd = t["coef"].double()
    # the statistics: of x as the convolution had it before its rounding, where its kernel took them
    assert bool(((mean - x.mean(0)).abs() <= (half + u) * x.abs().mean(0) + tiny).all())
    gain = w.abs() + t["eps"]
    assert bool(((scale - gain * rstd).abs() <= 2.0 ** -21 * gain * rstd).all())
    z = scale * x + offset + s
    size = (scale * x).abs() + offset.abs() + s.abs()
    assert bool(((y - z.clamp(min=0)).abs() <= half * z.abs() + 2.0 ** -22 * size + tiny).all())
    dz = torch.where(t["y"] > 0, t["g"], torch.zeros_like(t["g"]))
    assert equal(t["dz"], dz)
    dz, xh, M = dz.double(), (q8_ref(t["x"])[0] - mean) * rstd, x.shape[0]
    s1, s2, a1, a2 = dz.sum(0), (dz * xh).sum(0), dz.abs().sum(0), (dz.abs() * (xh.abs() + rstd * mean.abs())).sum(0)
    sums1, sums2, dw, db = t["out"].double()
    assert bool(((db - s1).abs() <= u * a1 + 1e-36).all()) and bool(((sums1 - s1).abs() <= u * a1 + 1e-36).all())
    assert bool(((sums2 - s2).abs() <= u * a2 + 1e-36).all()) and bool(((dw - s2 * w.sign()).abs() <= u * a2 + 1e-36).all())
    if t["dx"] is not None:
        ref = gain * rstd * (dz - s1 / M - xh * s2 / M)
        size = gain * rstd * (dz.abs() + a1 / M + (xh.abs() + rstd * mean.abs()) * a2 / M)
        assert bool(((t["dx"].double() - ref).abs() <= half * ref.abs() + (1 + half) * 2 * u * size + tiny).all())


@pytest.mark.parametrize("name", ["bfloat16", "float16"])
def test_every_8_bit_call_of_a_step(name, monkeypatch):
    dtype = BF if name == "bfloat16" else HF
    t, batch = _trainer(("tails", "pointwise"), name)
    if dtype == HF:        # (the first gradients overflow, here as in 16 bits, until the loss scale has come down: three steps from 2^16 to 2^13)
        before = None
        for _ in range(10):
            if before == (before := float(t.optimizer.loss_scale())):
                break
            t.run_step(batch)
    convs, tails = _recorded(monkeypatch)
    for step in range(2):
        losses = t.run_step(batch)
        torch.cuda.synchronize()
        assert all(float(v.detach()) == float(v.detach()) for v in losses.values())
        assert len(tails) == 16 and len(convs) >= 8                # (two encoders of eight blocks; predictors and pose convolutions)
        for k, c in enumerate(convs.values()):
            assert "dy" in c, k
            _check_conv(c, dtype)
        for k, c in enumerate(tails.values()):
            assert "g" in c, k
            _check_tail(c, dtype)
        convs.clear(), tails.clear()
