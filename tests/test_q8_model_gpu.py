"""MODEL.Q8: the 8-bit block tails and 1x1 convolutions inside the training step -- they run (and only where they are switched on), the first
step stays near the 16-bit one, a step is reproducible, recorded and replayed bit for bit, and waits with less memory for its backward pass."""
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


def _trainer(q8, dtype="bfloat16", B=2, H=128, W=256, seed=0):
    from mgnet_amd import add_mgnet_config, get_cfg
    from mgnet_amd.data import synthetic_batch
    from mgnet_amd.engine import Trainer
    from mgnet_amd.registry import build_model

    cfg = get_cfg()
    add_mgnet_config(cfg)
    cfg.merge_from_file(os.path.join(ROOT, "configs", "bench-c4-cityscapes-videosequence.yaml"))
    cfg.merge_from_list(["MODEL.DEVICE", "cuda:0", "SOLVER.IMS_PER_BATCH", B, "MODEL.SEM_SEG_HEAD.OHEM_N_MIN", B * H * W // 16, "SOLVER.AMP.DTYPE", dtype,
                         "MODEL.Q8.BLOCK_TAILS", "tails" in q8, "MODEL.Q8.POINTWISE", "pointwise" in q8])
    torch.manual_seed(seed)
    return Trainer(cfg, build_model(cfg)), synthetic_batch(B, H, W, torch.device("cuda:0"), seed=11)


def _count(monkeypatch):
    from mgnet_amd import _C
    calls = {}
    for name in ("q8_tail_fwd", "q8_tail_train_fwd", "q8_conv1x1_fwd", "q8_conv1x1_bwd", "q8_tail_train_bwd"):
        def wrapped(*a, _f=getattr(_C, name), _n=name, **k):
            calls[_n] = calls.get(_n, 0) + 1
            return _f(*a, **k)
        monkeypatch.setattr(_C, name, wrapped)
    return calls


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_step_with_8_bits_is_near_the_16_bit_step(dtype, monkeypatch):
    """forward values differ by the 8-bit rounding of the predictors' and pose convolutions' operands alone (block tails: by one rounding less
    of the normalised map); the losses of the first step agree within it"""
    calls = _count(monkeypatch)
    t, batch = _trainer((), dtype)
    base = {k: float(v) for k, v in t.run_step(batch).items()}
    assert not calls
    t, batch = _trainer(("tails",), dtype)
    tails = {k: float(v) for k, v in t.run_step(batch).items()}
    # ResNet-18 twice (backbone, pose encoder), eight blocks each
    assert calls.get("q8_tail_fwd", 0) + calls.get("q8_tail_train_fwd", 0) == 16 and calls["q8_tail_train_bwd"] == 16 and "q8_conv1x1_fwd" not in calls
    t, batch = _trainer(("tails", "pointwise"), dtype)
    both = {k: float(v) for k, v in t.run_step(batch).items()}
    assert calls["q8_conv1x1_fwd"] == calls["q8_conv1x1_bwd"] >= 8      # six predictors, the pose network's first and last
    for other in (tails, both):
        assert set(other) == set(base)
        for k in base:
            assert other[k] == other[k] and abs(other[k] - base[k]) <= 0.1 * abs(base[k]) + 1e-3, (k, base[k], other[k])


def test_step_with_8_bits_is_reproducible_and_replayed_bit_for_bit():
    ta, ba = _trainer(("tails", "pointwise"))
    tb, bb = _trainer(("tails", "pointwise"))
    la = [{n: float(v) for n, v in ta.run_step(ba).items()} for _ in range(6)]
    lb = [{n: float(v) for n, v in tb.run_step(bb).items()} for _ in range(3)]
    tb.record_plan(bb)
    lb.append({n: float(v) for n, v in tb._plan_losses.items()})
    lb += [{n: float(v) for n, v in tb.replay_plan().items()} for _ in range(2)]
    torch.cuda.synchronize()
    assert la == lb
    for (na, pa), (_, pb) in zip(ta.model.named_parameters(), tb.model.named_parameters()):
        assert torch.equal(pa, pb), na


def test_block_tails_in_8_bits_wait_with_less_memory():
    """what a block tail holds for its backward pass once its input is nobody else's: one byte a value, a scale byte per 64 channels and a
    mask bit -- 1.14 bytes -- against 2 bytes of x (and of y) and the mask"""
    from mgnet_amd.modeling import ops
    from mgnet_amd.modeling.layers import InPlaceABNSync
    norm = InPlaceABNSync(64, activation="identity").cuda()
    n = 4 * 64 * 128 * 64

    def held(fn):
        s = torch.zeros((4, 64, 128, 64), device="cuda", dtype=torch.bfloat16).permute(0, 3, 1, 2)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        # (x as a convolution's output is: not a leaf, which the graph would hold for its gradient)
        leaf = torch.zeros(1, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        out = [fn(torch.randn(4, 64, 128, 64, device="cuda").to(torch.bfloat16).permute(0, 3, 1, 2) + leaf, norm, s).sum() for _ in range(4)]
        return (torch.cuda.memory_allocated() - before) / (4 * n), out
    held(ops.abn_add_relu_q8)          # (workspaces and the allocator's own)
    q, _ = held(ops.abn_add_relu_q8)
    b, _ = held(ops.abn_add_relu)
    assert 1.14 <= q <= 1.2 and b >= 2.1, (q, b)
