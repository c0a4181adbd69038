"""8-bit operators at the sizes and in the calls where launches, masks and memory go wrong; tolerances as in test_q8_gpu.py."""
import math

import pytest
import torch

from test_q8_gpu import BF, conv_case, HF, ops, rows, tail_case

pytestmark = pytest.mark.gpu


def test_weight_gradient_of_more_than_2_32_work_items():
    """32768 x 32768 weights: the sums of the partial gradients are 4194432 blocks of 1024 threads, more than one launch dimension holds.  dy and
    x are small whole numbers, so the sums are exact in fp32"""
    M, N = 64, 32768
    g = torch.Generator(device="cuda").manual_seed(3)
    whole = lambda: torch.randint(-7, 8, (1, 1, M, N), generator=g, device="cuda").to(BF).permute(0, 3, 1, 2)  # noqa: E731
    x, dy = whole().requires_grad_(), whole()
    w = torch.zeros((N, N, 1, 1), dtype=BF, device="cuda", requires_grad=True)
    b = torch.zeros(N, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(ops().conv1x1_q8(x, w, b), (w, b), dy)
    G, X = rows(dy).float(), rows(x.detach()).float()
    assert torch.equal(db, G.sum(0))
    for r in (0, 1, 8191, 16384, N - 4096, N - 1):
        k = slice(r, min(r + 64, N))
        assert torch.equal(dw[k, :, 0, 0].float(), (G[:, k].t().double() @ X.double()).float().to(BF).float()), r
    assert torch.equal(dw.view(-1)[-N:].float(), (G[:, -1].double() @ X.double()).float().to(BF).float())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cout", [20, 24, 64])     # (64: the mask's kernel; 20 and 24: no kernel has their width)
def test_relu_mask_takes_what_is_not_finite(cout, dtype):
    """gradients that are infinite or NaN where the output is zero do not reach anything"""
    x, wt, b, dy = conv_case(2, 40, 9, 7, cout, dtype)
    y = ops().conv1x1_q8(x, wt, b, relu=True)
    off = y.detach() == 0
    assert 0.1 < float(off.float().mean()) < 0.9
    want = torch.autograd.grad(y, (x, wt, b), dy.masked_fill(off, 0.0), retain_graph=True)
    for v in (math.inf, -math.inf, math.nan):
        got = torch.autograd.grad(y, (x, wt, b), dy.masked_fill(off, v), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(got, want)), v


def test_block_tail_without_gradients_keeps_nothing(monkeypatch):
    import copy

    from mgnet_amd import _C
    o = ops()
    x, norm, s, _ = tail_case(2, 64, 33, 20, BF, 4)
    other = copy.deepcopy(norm)
    want = o.abn_add_relu_q8(x, norm, s).detach()
    monkeypatch.setattr(_C, "q8_tail_buffer", None)        # (not asked for)
    with torch.no_grad():
        y = o.abn_add_relu_q8(x, other, s)
    assert torch.equal(y, want) and torch.equal(norm.running_mean, other.running_mean) and torch.equal(norm.running_var, other.running_var)


def test_conv1x1_without_gradients_writes_no_codes(monkeypatch):
    from mgnet_amd import _C
    o = ops()
    x, wt, b, _ = conv_case(2, 64, 33, 20, 24, BF)
    keep = []
    fwd = _C.q8_conv1x1_fwd
    monkeypatch.setattr(_C, "q8_conv1x1_fwd", lambda *a: keep.append(int(a[-1])) or fwd(*a))
    want = o.conv1x1_q8(x, wt, b)
    with torch.no_grad():
        assert torch.equal(o.conv1x1_q8(x, wt, b), want)
    assert keep == [1, 0]
