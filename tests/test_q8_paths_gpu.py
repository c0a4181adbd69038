"""8-bit operators at the sizes and in the calls where launches, masks and memory go wrong; tolerances as in test_q8_gpu.py."""
import math

import pytest
import torch

from test_q8_gpu import BF, conv_case, F32, group_tol, HF, ops, q8_ref, rand, rand_map, rows, tail_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _give_the_memory_back():
    yield
    torch.cuda.empty_cache()


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


def held(fn):
    """bytes that stay allocated, and the most that were, while fn() runs; its result"""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = fn()
    torch.cuda.synchronize()
    return torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before, out


# (c, cout, map strides): packed on the way, packed in a pass of its own (K > 512; rows that are not contiguous)
FORMS = [(256, 256, False), (640, 64, False), (256, 64, True)]


@pytest.mark.parametrize("c,cout,strided", FORMS)
def test_frozen_weights_leave_only_packed_weights_waiting(c, cout, strided):
    """no weight gradient, so the packed input is not kept for the backward pass: what waits is the transposed weights"""
    o = ops()
    x, wt, b, dy = conv_case(2, c, 64, 128 if not strided else 256, cout, BF)
    if strided:
        x, dy = x.detach()[:, :, :, ::2].requires_grad_(), dy[:, :, :, ::2].contiguous(memory_format=torch.channels_last)
    full = torch.autograd.grad(o.conv1x1_q8(x, wt, b), (x,), dy)[0]
    M = x.shape[0] * x.shape[2] * x.shape[3]
    n, _, y = held(lambda: o.conv1x1_q8(x, wt.detach(), b.detach()))
    assert n - 2 * M * cout < M * c // 2, (n, M * c)
    assert torch.equal(torch.autograd.grad(y, (x,), dy)[0], full)


@pytest.mark.parametrize("c,cout,strided", FORMS)
def test_no_gradient_keeps_and_writes_nothing(c, cout, strided):
    o = ops()
    x, wt, b, _ = conv_case(2, c, 64, 128 if not strided else 256, cout, BF)
    if strided:
        x = x.detach()[:, :, :, ::2].requires_grad_()
    want = o.conv1x1_q8(x, wt, b).detach()
    M = x.shape[0] * x.shape[2] * x.shape[3]

    def call():
        with torch.no_grad():
            return o.conv1x1_q8(x, wt, b)
    n, most, y = held(call)
    assert torch.equal(y, want) and n - 2 * M * cout < 1 << 20
    if c <= 512 and not strided:         # (packed on the way: no room for the codes is taken at all)
        assert most - 2 * M * cout < M * c // 2, (most, M * c)


def test_sizes_of_the_forward_call():
    """what a call needs is what it takes: a byte less is refused, and the rest of a larger buffer stays as it was"""
    import ctypes

    from mgnet_amd import _C
    M, C, N = 700, 64, 40
    x, w = rand((M, C), BF, 1), rand((N, C), F32, 2)
    y = torch.empty((M, N), dtype=BF, device="cuda")
    need, kept = ctypes.c_size_t(), ctypes.c_size_t()
    both = torch.full((1 << 20,), 77, dtype=torch.uint8, device="cuda")

    def call(keep, sw, nbytes):
        return _C.lib().mgn_q8_conv1x1_fwd(x.data_ptr(), M, C, M * sw, sw, 0, M, 1, w.data_ptr(), 0, C, 1, N, None, 0, y.data_ptr(), keep, both.data_ptr(), nbytes,
                                           _C._stream())
    first = {}
    for keep, sw in ((0, C), (1, C), (0, C - 8), (1, C - 8)):       # (rows C - 8 apart overlap: packed in a pass of its own)
        assert _C.lib().mgn_q8_conv1x1_fwd_bytes(x.data_ptr(), M, C, M * sw, sw, 0, M, 1, N, y.data_ptr(), keep, ctypes.byref(need), ctypes.byref(kept)) == 0
        assert kept.value <= need.value and (keep or kept.value < 8192) and (need.value < M * C) == (keep == 0 and sw == C)
        assert call(keep, sw, need.value - 1) == -28
        both.fill_(77)
        assert call(keep, sw, need.value) == 0
        assert bool((both[need.value:] == 77).all())
        assert torch.equal(y, first.setdefault(sw, y.clone()))


def test_backward_takes_no_room_for_what_it_does_not_write():
    """262144 x 256 -> 256: dy is packed on the way, and without a weight gradient there are no partial results"""
    x, wt, b, dy = conv_case(8, 256, 128, 256, 256, BF)
    M, o = 262144, ops()
    y = o.conv1x1_q8(x, wt.detach(), b.detach())        # (autograd.grad for x alone would not tell: needs_input_grad goes by the inputs)
    _, most, _ = held(lambda: torch.autograd.grad(y, (x,), dy))
    assert most < 2 * M * 256 + (8 << 20), most
    y = o.conv1x1_q8(x, wt, b)
    _, most, _ = held(lambda: torch.autograd.grad(y, (x, wt, b), dy))
    assert most < 2 * M * 256 + 512 * (4 * 256 * 257 + 4096), most      # (512 row ranges at most)


@pytest.mark.parametrize("M,C,N", [(700, 64, 40), (700, 64, 19), (300, 640, 96), (300, 96, 640), (500, 24, 8)])
def test_sizes_of_the_backward_call(M, C, N):
    """each combination of gradients runs in the scratch memory that it asks for, not in a byte less, and writes nothing behind it"""
    import ctypes

    from mgnet_amd import _C
    x, w, dy = rand((M, C), BF, 1), rand((N, C), F32, 2), rand((M, N), BF, 3)
    y = torch.empty((M, N), dtype=BF, device="cuda")
    buf, kept = _C.q8_conv1x1_fwd(x, M, C, M * C, C, 0, M, 1, w, N, None, 0, y, 1)
    assert kept == buf.numel()
    most = 0
    ws, need = torch.empty(8 << 20, dtype=torch.uint8, device="cuda"), ctypes.c_size_t()
    for want_dx, want_dw in ((1, 1), (1, 0), (0, 1)):
        assert _C.lib().mgn_q8_conv1x1_bwd_bytes(M, C, N, want_dx, want_dw, ctypes.byref(need)) == 0
        most = max(most, need.value)
        dx, dw, db = torch.empty((M, C), dtype=BF, device="cuda"), torch.empty((N, C), device="cuda"), torch.empty(N, device="cuda")
        p = lambda t, on: t.data_ptr() if on else None  # noqa: E731

        def call(nbytes):
            return _C.lib().mgn_q8_conv1x1_bwd(dy.data_ptr(), M, C, N, buf.data_ptr(), p(dx, want_dx), p(dw, want_dw), p(db, want_dw), ws.data_ptr(), nbytes, _C._stream())
        if need.value:
            assert call(need.value - 1) == -28
        ws.fill_(77)
        assert call(need.value) == 0
        assert bool((ws[need.value:] == 77).all())
        if want_dx and want_dw:
            full = (dx, dw, db)
        assert (not want_dx or torch.equal(dx, full[0])) and (not want_dw or (torch.equal(dw, full[1]) and torch.equal(db, full[2])))
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    assert _C.lib().mgn_q8_conv1x1_bytes(M, C, N, ctypes.byref(a), ctypes.byref(b)) == 0 and b.value >= most     # (enough for every call)


# ---- calls that the documentation allows -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("case", ["both_axes", "rows_expanded", "columns_expanded", "transposed_view", "one_column", "one_row", "offset"])
@pytest.mark.parametrize("dtype", [F32, BF])
def test_weight_tiles_of_any_strides(case, dtype):
    big = rand((300, 420), dtype, 3)
    w = {"both_axes": lambda: big[::2, ::3], "rows_expanded": lambda: big[:1].expand(150, 420), "columns_expanded": lambda: big[:, :1].expand(300, 140),
         "transposed_view": lambda: big.t()[5:, 3:], "one_column": lambda: big[:, 7:8], "one_row": lambda: big.t()[9:10], "offset": lambda: big[1:, 1:]}[case]()
    q, ref = ops().q8_pack(w, tile=True), ops().q8_pack(w.clone(memory_format=torch.contiguous_format), tile=True)
    assert torch.equal(q.codes, ref.codes) and torch.equal(q.scales[:, :w.shape[0]], ref.scales[:, :w.shape[0]])


@pytest.mark.parametrize("wd", [BF, HF])
def test_conv1x1_with_16_bit_parameters(wd):
    """the parameters' values in another type: the same results, gradients in the parameters' type"""
    o = ops()
    x, wt, b, dy = conv_case(2, 72, 11, 13, 40, BF)
    wt, b = (t.detach().to(wd).requires_grad_() for t in (wt, b))
    w32, b32 = (t.detach().float().requires_grad_() for t in (wt, b))
    y, ref = o.conv1x1_q8(x, wt, b), o.conv1x1_q8(x, w32, b32)
    assert torch.equal(y, ref)
    for p, q, t in zip(torch.autograd.grad(y, (x, wt, b), dy), torch.autograd.grad(ref, (x, w32, b32), dy), (x, wt, b)):
        assert p.dtype == t.dtype and torch.equal(p, q.to(t.dtype))


def test_conv1x1_with_a_transposed_weight():
    o = ops()
    x, wt, b, dy = conv_case(1, 64, 9, 10, 48, BF)
    t = wt.detach().transpose(0, 1).contiguous().requires_grad_()
    y, ref = o.conv1x1_q8(x, t.transpose(0, 1), b), o.conv1x1_q8(x, wt, b)
    assert torch.equal(y, ref)
    assert torch.equal(torch.autograd.grad(y, (t,), dy)[0].transpose(0, 1), torch.autograd.grad(ref, (wt,), dy)[0])


def test_backward_twice_and_results_overwritten():
    """a graph that is kept gives the same gradients again, also after inputs and results have been written over (neither is kept, but for the result that
    a ReLU masks by)"""
    o = ops()
    x, wt, b, dy = conv_case(2, 64, 9, 10, 48, BF)
    y = o.conv1x1_q8(x * 1, wt, b)
    first = torch.autograd.grad(y, (x, wt, b), dy, retain_graph=True)
    with torch.no_grad():
        y.zero_(), wt.zero_(), b.zero_()
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, (x, wt, b), dy)))
    y = o.conv1x1_q8(x, wt, b, relu=True)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError):           # (autograd sees it)
        torch.autograd.grad(y, (x,), dy)
    x, norm, s, g = tail_case(2, 40, 7, 9, BF)
    leaves = (x, s, norm.weight, norm.bias)
    y = o.abn_add_relu_q8(x * 1, norm, s * 1)
    first = torch.autograd.grad(y, leaves, g, retain_graph=True)
    with torch.no_grad():
        y.zero_(), x.zero_(), s.zero_()
    assert all(torch.equal(p, q) for p, q in zip(first, torch.autograd.grad(y, leaves, g)))


def test_block_tail_of_one_map_twice():
    """the input as its own shortcut: the gradients of both places add up"""
    o = ops()
    x, norm, _, g = tail_case(2, 72, 9, 8, BF, 6)
    import copy
    other = copy.deepcopy(norm)
    s = x.detach().clone(memory_format=torch.channels_last).requires_grad_()
    y, ref = o.abn_add_relu_q8(x, norm, x), o.abn_add_relu_q8(x, other, s)
    assert torch.equal(y, ref)
    dx, ds = torch.autograd.grad(ref, (x, s), g)
    assert torch.equal(torch.autograd.grad(y, (x,), g)[0], dx + ds)


def test_one_map_into_two_convolutions():
    """two consumers of a map on two streams at once, both backward passes: each call has buffers of its own"""
    o = ops()
    x, w1, b1, d1 = conv_case(4, 128, 40, 60, 64, BF, seed=1)
    _, w2, b2, d2 = conv_case(4, 128, 40, 60, 200, BF, seed=2)
    want = [torch.autograd.grad(o.conv1x1_q8(x, w, b), (x, w, b), d) for w, b, d in ((w1, b1, d1), (w2, b2, d2))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        torch.cuda.synchronize()
        got = []
        for st, w, b, d in zip(streams, (w1, w2), (b1, b2), (d1, d2)):
            with torch.cuda.stream(st):
                got.append(torch.autograd.grad(o.conv1x1_q8(x, w, b), (x, w, b), d))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for a, b in zip(got, want) for p, q in zip(a, b))


@pytest.mark.parametrize("c,cout", [(96, 40), (640, 48)])       # (packed on the way, and in a pass of its own whose codes go)
def test_captured_with_frozen_weights(c, cout):
    o = ops()
    x, wt, b, dy = conv_case(2, c, 14, 10, cout, BF)
    wt, b = wt.detach(), b.detach()
    x = x.detach().requires_grad_()

    def step():
        y = o.conv1x1_q8(x, wt, b, relu=True)
        return y.detach(), torch.autograd.grad(y, (x,), dy)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            out = step()
    torch.cuda.current_stream().wait_stream(side)
    del out
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(4):
        with torch.no_grad():
            x.copy_(rand_map(2, c, 14, 10, BF, 100 + rep))
            wt.copy_(rand((cout, c), F32, 200 + rep, 0.2).view(cout, c, 1, 1) / math.sqrt(c))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(step(), got)), rep


def test_saved_on_the_host_and_recomputed():
    """what waits may wait elsewhere (saved-tensor hooks), or not at all (recomputation)"""
    from torch.utils.checkpoint import checkpoint
    o = ops()
    x, wt, b, dy = conv_case(2, 64, 9, 10, 48, BF)
    want = torch.autograd.grad(o.conv1x1_q8(x, wt, b, True), (x, wt, b), dy)
    with torch.autograd.graph.save_on_cpu():
        y = o.conv1x1_q8(x, wt, b, True)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, wt, b), dy), want))
    y = checkpoint(lambda x: o.conv1x1_q8(x, wt, b, True), x, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, wt, b), dy), want))
    x, norm, s, g = tail_case(2, 40, 7, 9, HF)
    leaves = (x, s, norm.weight, norm.bias)
    want = torch.autograd.grad(o.abn_add_relu_q8(x, norm, s), leaves, g)
    with torch.autograd.graph.save_on_cpu():
        y = o.abn_add_relu_q8(x, norm, s)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, g), want))


def test_product_of_operands_the_other_way_round():
    """row scales and tile scales on either side, a bias that is a view, a result in another type than the source's"""
    o = ops()
    a, b = rand((200, 130), HF, 1), rand((72, 130), F32, 2)
    bias = rand((72, 2), F32, 3, 0.0)[:, 1]
    one = o.q8_matmul(o.q8_pack(a), o.q8_pack(b, tile=True), bias, out_dtype=F32)
    other = o.q8_matmul(o.q8_pack(b, tile=True), o.q8_pack(a), out_dtype=F32).t() + bias
    av, bv = q8_ref(a)[0], q8_ref(b, True)[0]
    tol = (132 + 2) * 2.0 ** -23 * (av.abs() @ bv.abs().t() + bias.abs().double()) + group_tol(av, bv) + 2.0 ** -22 * bias.abs().double()
    for y in (one, other):
        assert bool(((y.double() - av @ bv.t() - bias.double()).abs() <= tol).all())
    assert torch.equal(o.q8_matmul(o.q8_pack(a), o.q8_pack(b, tile=True), bias), one.half())


def test_block_tail_masks_what_is_not_finite():
    o = ops()
    x, norm, s, g = tail_case(2, 72, 9, 8, HF, 9)
    y = o.abn_add_relu_q8(x, norm, s)
    off, leaves = y.detach() == 0, (x, s, norm.weight, norm.bias)
    want = torch.autograd.grad(y, leaves, g.masked_fill(off, 0.0), retain_graph=True)
    for v in (math.inf, math.nan):
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, g.masked_fill(off, v), retain_graph=True), want)), v
