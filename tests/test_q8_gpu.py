"""8-bit operators (csrc/q8.hip through ops): the block format bit for bit, the block-scaled product, the trained 1x1 convolution and the
block tail against the definition in 64 bits.

Tolerances are sums of two parts.  Rounding to the result's type: at most half a step, eps / 2 of the value.  fp32 accumulation of n terms
with absolute sum S: every addition is off by at most one step of the running value, n * 2^-23 * S in all.

The 8-bit product has a third part, which is the matrix instruction's.  It adds the products of 8 neighbouring k before they join the fp32
accumulator, each cut (towards zero) to a multiple of 2^(E - 13), E = the largest sum of two exponents among the 8: 256 * 256 + 2 * 2 gives
65536, 256 * 256 + 2 * 6.5 gives 65544, and the same two products in different groups of 8 lose nothing.  The product with exponent E has 8
significant bits at most and is kept; each of the other 7 loses less than 2^(E - 13) <= 2^-13 * (the group's largest product p): an
output is off by less than 7 * 2^-13 * sum over the groups of p."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def ops():
    from mgnet_amd.modeling import ops
    return ops


# ---- the definition, in 64 bits on the CPU or the GPU --------------------------------------------------------------------------------
def q8_ref(x, tile=False):
    """values [M, C] (float64) and biased exponents [ceil(C/128), M] of the packed form"""
    top = 1.875 * 2.0 ** (15 if x.dtype == HF else 127)
    v = x.double()
    M, C = v.shape
    nb = -(-C // 128)
    out, exps = torch.empty_like(v), torch.empty((nb, M), dtype=torch.int64, device=x.device)
    for k in range(nb):
        b = v[:, 128 * k:128 * (k + 1)]
        fin = torch.isfinite(b)
        c = torch.where(fin, b, 0.0).clamp(-top, top)
        a = c.abs().amax(1) if M else c.new_zeros(0)
        if tile:
            for r in range(0, M, 128):
                a[r:r + 128] = a[r:r + 128].max()
        # smallest e with a <= 448 * 2^e, from below
        f, p = torch.frexp(a)
        e = torch.where(a > 0, (p - 9 + (f > 0.875)).double(), -111.0).clamp(min=-111.0)
        assert bool((a <= 448 * torch.exp2(e)).all()) and bool(((a > 448 * torch.exp2(e - 1)) | (e == -111)).all())
        s = c / torch.exp2(e)[:, None]
        _, p = torch.frexp(s)
        step = torch.exp2((p - 1).clamp(min=-6).double() - 3)
        r = torch.round(s / step) * step * torch.exp2(e)[:, None]
        out[:, 128 * k:128 * (k + 1)] = torch.where(fin, r, math.nan)
        exps[k] = e.long() + 127
    return out, exps


def equal(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def rand(shape, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda")
    return (x * torch.exp(spread * torch.randn(shape[-1], generator=g, device="cuda"))).to(dtype)


def rand_map(n, c, h, w, dtype, seed=0, spread=1.0):
    return rand((n, h, w, c), dtype, seed, spread).permute(0, 3, 1, 2)


def rows(t):
    return t.permute(0, 2, 3, 1).reshape(-1, t.shape[1])


def group_tol(a, b):
    """7 * 2^-13 * sum over the groups of 8 k of the largest |a_k b_k| (see above): [M, N]"""
    a, b = a.abs(), b.abs()
    out = torch.zeros((a.shape[0], b.shape[0]), dtype=torch.float64, device=a.device)
    for k in range(0, a.shape[1], 8):
        p = a[:, None, k] * b[None, :, k]
        for j in range(k + 1, min(k + 8, a.shape[1])):
            p = torch.maximum(p, a[:, None, j] * b[None, :, j])
        out += p
    return 7 * 2.0 ** -13 * out


def check_packed(q, x2, tile=False):
    val, exps = q8_ref(x2, tile)
    M, C = x2.shape
    assert torch.equal(q.scales[:, :M].long(), exps)
    assert equal(q.unpack(F32).double().permute(*((0, 2, 3, 1) if len(q.shape) == 4 else (0, 1))).reshape(M, C), val)
    assert not bool(q.codes[:, C:].any())       # the padding columns are zero


# ---- pack / unpack -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("M,C", [(1, 1), (1, 128), (3, 3), (7, 17), (8, 64), (9, 32), (33, 40), (16, 129), (129, 96), (65, 320), (31, 1000), (1025, 256), (5, 8192)])
def test_pack_matches_the_definition(M, C, dtype):
    x = rand((M, C), dtype, M * 7 + C)
    q = ops().q8_pack(x)
    check_packed(q, x)
    assert equal(q.unpack().double(), q8_ref(x)[0]) and q.unpack().dtype == dtype      # exact in the source's own type
    if dtype != F32:
        assert (q.unpack(F32).double() - x.double()).abs().max() <= (2.0 ** -4) * x.abs().max().double()


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_pack_special_values(dtype):
    fi = torch.finfo(dtype)
    tiny = 2.0 ** -24 if dtype == HF else 2.0 ** -133
    base = rand((16, 256), dtype, 3)
    base[0] = 0
    base[1] = math.nan
    base[2, ::3] = math.inf
    base[3, 5], base[3, 200] = -math.inf, math.nan
    base[4] = fi.min
    base[5, 7] = fi.max
    base[6, :128] = tiny
    base[7] = -0.0
    base[8] = torch.linspace(-1, 1, 256, device="cuda").to(dtype)
    base[9, 0], base[9, 1:128] = 448.0, 2.0 ** -10           # half a step of the smallest code: to even, zero
    base[10, 0], base[10, 1:128] = 448.0, 2.0 ** -10 * 1.5
    base[11, 0], base[11, 1:128] = 448.0 * (1 + 2.0 ** -7), 1.0   # just above: the next exponent
    base[12, :128] = torch.arange(128, device="cuda").to(dtype)
    base[13, :128] = fi.tiny
    q = ops().q8_pack(base)
    check_packed(q, base)
    u = q.unpack()
    assert bool(torch.isnan(u[1]).all()) and bool(torch.isfinite(u[4]).all()) and bool(torch.isfinite(u[5]).all())
    assert torch.equal(torch.isnan(u), ~torch.isfinite(base))


def test_pack_every_bf16_and_fp16():
    """every 16-bit value, alone in its block and next to a larger one"""
    for dtype in (BF, HF):
        v = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
        x = torch.zeros((65536, 128), dtype=dtype, device="cuda")
        x[:, 77] = v
        check_packed(ops().q8_pack(x), x)
        x[:, 3] = torch.where(torch.isfinite(v.float()), (v.float() * 37).clamp(-6e4, 6e4), 0.0).to(dtype)
        check_packed(ops().q8_pack(x), x)


@pytest.mark.parametrize("case", ["nchw", "channel_slice", "row_slice", "stride2", "stride2_odd", "pixel", "column", "expanded", "transposed", "offset1"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_pack_strides(case, dtype):
    m = rand_map(2, 80, 7, 9, dtype, 5)
    x = {"nchw": lambda: m.contiguous(), "channel_slice": lambda: m[:, 16:56], "row_slice": lambda: m[:, :, 2:5], "stride2": lambda: m[:, :, ::2, ::2],
         "stride2_odd": lambda: m[:, 3:, 1::2, ::2], "pixel": lambda: rand((8, 512), dtype, 1).view(8, 512, 1, 1), "column": lambda: m[:, :, :, 4:5],
         "expanded": lambda: rand((1, 80), dtype, 2).view(1, 80, 1, 1).expand(2, 80, 3, 5), "transposed": lambda: rand((40, 24), dtype, 3).t(),
         "offset1": lambda: rand((1, 24 * 40 + 1), dtype, 4)[0, 1:].view(24, 40)}[case]()
    q = ops().q8_pack(x)
    check_packed(q, (rows(x) if x.dim() == 4 else x).contiguous())
    u = q.unpack()
    assert u.shape == x.shape and (x.dim() == 2 or u.is_contiguous(memory_format=torch.channels_last))


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("N,K", [(1, 1), (19, 320), (128, 128), (129, 130), (256, 512), (300, 72)])
def test_pack_weight_and_its_transpose(N, K, dtype):
    from mgnet_amd import _C
    w = rand((N, K), dtype, N + K)
    check_packed(ops().q8_pack(w, tile=True), w, tile=True)
    check_packed(ops().q8_pack(w.t(), tile=True), w.t(), tile=True)
    a, b = torch.empty((N, K), device="cuda"), torch.empty((K, N), device="cuda")
    _C.q8_unpack(_C.q8_pack_weight(w), N, K, a)
    _C.q8_unpack(_C.q8_pack_weight(w, transposed=True), K, N, b)
    assert torch.equal(a, b.t())


def test_empty_and_large():
    o = ops()
    q = o.q8_pack(torch.empty((0, 40), dtype=BF, device="cuda"))
    assert q.unpack().shape == (0, 40)
    w = o.q8_pack(rand((8, 40), F32, 1), tile=True)
    assert o.q8_matmul(q, w).shape == (0, 8)
    assert o.q8_pack(torch.empty((0, 40, 3, 5), dtype=BF, device="cuda")).unpack().shape == (0, 40, 3, 5)
    # offsets past 32 bits: 2.2e9 codes, 4.3 GB of input; the last rows are compared
    M, K = (1 << 21) + 5, 1040
    x = torch.zeros((M, K), dtype=BF, device="cuda")
    x[-300:] = rand((300, K), BF, 9)
    q = o.q8_pack(x)
    ref = q8_ref(x[-300:])[0]
    assert equal(q.unpack()[-300:].double(), ref)
    w = o.q8_pack(rand((24, K), F32, 4), tile=True)
    y = o.q8_matmul(q, w, out_dtype=F32)
    wv = w.unpack().double()
    tol = (K + 2) * 2.0 ** -23 * (ref.abs() @ wv.abs().t()) + group_tol(ref, wv) + 1e-30
    assert bool(((y[-300:].double() - ref @ wv.t()).abs() <= tol).all()) and not bool(y[:1000].any())


# ---- product -------------------------------------------------------------------------------------------------------------------------
def check_product(a, b, bias, act, slope, out_dtype):
    o = ops()
    qa, qb = o.q8_pack(a), o.q8_pack(b, tile=True)
    y = o.q8_matmul(qa, qb, bias, act, slope, out_dtype)
    av, bv = q8_ref(a)[0], q8_ref(b, True)[0]
    K = a.shape[1]
    ref, S = av @ bv.t(), av.abs() @ bv.abs().t()
    if bias is not None:
        ref, S = ref + bias.double(), S + bias.abs().double()
    if act != "none":
        ref = torch.where(ref > 0, ref, ref * (slope if act == "leaky_relu" else 0.0))
    half = {BF: 2.0 ** -8, HF: 2.0 ** -11, F32: 2.0 ** -24}[out_dtype]
    tol = half * ref.abs() + (1 + half) * ((K + 2) * 2.0 ** -23 * S + group_tol(av, bv)) + (2.0 ** -25 if out_dtype == HF else 1e-36)
    assert y.dtype == out_dtype and y.shape == ref.shape
    bad = (y.double() - ref).abs() - tol
    assert bool((bad <= 0).all()), float(bad.max())


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 512, 512), (3, 5, 7), (33, 19, 320), (64, 64, 128), (65, 130, 260), (500, 40, 96), (1000, 257, 640),
                                   (4100, 19, 320), (9000, 32, 64), (8200, 129, 48), (2200, 1025, 384), (33000, 1100, 144), (131073, 257, 32)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_product(M, N, K, dtype):
    a, b = rand((M, K), dtype, M + N), rand((N, K), F32, N + K, 0.3) / math.sqrt(K)
    bias = rand((N,), F32, 2, 0.0)
    check_product(a, b, None, "none", 0.01, dtype)
    check_product(a, b, bias, "leaky_relu" if N % 2 else "relu", 0.01, F32 if M % 2 else dtype)


@pytest.mark.parametrize("M,N,K", [(1, 19, 3000), (33, 1000, 4096), (100, 77, 1400), (1000, 40, 513), (2300, 1030, 1000), (4097, 515, 530), (16380, 1021, 130),
                                   (16380, 1021, 700), (8190, 2045, 64), (60000, 21, 530), (50000, 32, 1100), (16000, 512, 512), (3001, 517, 257)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_product_of_every_tile(M, N, K, dtype):
    """sizes that leave tiles, half steps of k and rows of the result ragged, for each of the product's kernels"""
    a, b = rand((M, K), dtype, M + N), rand((N, K), F32, N + K, 0.3) / math.sqrt(K)
    check_product(a, b, rand((N,), F32, 2, 0.0), "leaky_relu", 0.25, dtype)
    check_product(a, b, None, "none", 0.01, F32)


@pytest.mark.parametrize("M,N,K,ldo,at", [(40, 37, 300, 41, 3), (70, 33, 2000, 33, 1), (2300, 1030, 700, 1035, 5), (16380, 1021, 130, 1021, 7), (60000, 21, 530, 24, 1),
                                          (60000, 21, 200, 23, 9), (50000, 40, 256, 48, 8), (50000, 200, 256, 208, 8), (50000, 200, 256, 201, 1)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_product_leaves_what_lies_around_it(M, N, K, ldo, at, dtype):
    """rows of any pitch from any element on: nothing before, between or behind them is written"""
    from mgnet_amd import _C
    o = ops()
    qa, qb = o.q8_pack(rand((M, K), BF, 1)), o.q8_pack(rand((N, K), F32, 2, 0.0), tile=True)
    whole = torch.full((at + M * ldo + 32,), 7.0, dtype=dtype, device="cuda")
    out = whole[at:at + M * ldo].view(M, ldo)
    pa, pb = qa.buf.data_ptr(), qb.buf.data_ptr()
    _C.check(_C._fn("mgn_q8_matmul", out)(pa, pa + _C.q8_code_bytes(M, K), M, pb, pb + _C.q8_code_bytes(N, K), N, K, None, 0, 0.0, out.data_ptr(),
                                          int(dtype == F32), ldo, _C._stream()), "mgn_q8_matmul")
    ref = o.q8_matmul(qa, qb, out_dtype=dtype)
    close = (out[:, :N].double() - ref.double()).abs() <= 2.0 ** -7 * ref.double().abs() + K * 2.0 ** -12 * float(ref.abs().max())   # (another kernel's order)
    assert bool(close.all())
    out[:, :N] = 7.0
    assert bool((whole == 7.0).all())


def test_product_scales_over_the_whole_range():
    """blocks whose exponents differ by hundreds of binades, and NaN that stay in their rows"""
    o = ops()
    K, M, N = 512, 300, 140
    a = rand((M, K), F32, 1, 0.0) * torch.exp2(torch.randint(-60, 60, (M, 4), device="cuda").float()).repeat_interleave(128, 1)
    b = rand((N, K), F32, 2, 0.0) * torch.exp2(torch.tensor([30.0, -20.0, 0.0, 10.0], device="cuda")).repeat_interleave(128)
    check_product(a, b, None, "none", 0.01, F32)
    a[5, 3], a[255, 300] = math.nan, math.inf
    y = o.q8_matmul(o.q8_pack(a), o.q8_pack(b, tile=True), act="relu")
    bad = torch.isnan(y).any(1).nonzero().flatten().tolist()
    assert bad == [5, 255] and bool(torch.isnan(y[5]).all())


def test_product_of_a_map_and_row_scales():
    """a map gives a map; b may have row scales instead of tile scales"""
    o = ops()
    x, w = rand_map(2, 72, 5, 11, BF, 3), rand((24, 72), BF, 4)
    y = o.q8_matmul(o.q8_pack(x), o.q8_pack(w))
    assert y.shape == (2, 24, 5, 11) and y.is_contiguous(memory_format=torch.channels_last)
    xv, wv = q8_ref(rows(x))[0], q8_ref(w)[0]
    ref = xv @ wv.t()
    assert bool(((rows(y).double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 74 * 2.0 ** -22 * (xv.abs() @ wv.abs().t()) + 1.01 * group_tol(xv, wv)).all())


# ---- 1x1 convolution, trained ----------------------------------------------------------------------------------------------------------
def conv_case(n, c, h, w, cout, dtype, bias=True, relu=False, seed=0):
    x = rand_map(n, c, h, w, dtype, seed).requires_grad_()
    wt = (rand((cout, c), F32, seed + 1, 0.2) / math.sqrt(c)).view(cout, c, 1, 1).requires_grad_()
    b = rand((cout,), F32, seed + 2, 0.0).requires_grad_() if bias else None
    dy = rand_map(n, cout, h, w, dtype, seed + 3, 0.5)
    return x, wt, b, dy


def check_conv(x, wt, b, dy, relu=False):
    o = ops()
    dtype, (cout, c) = x.dtype, wt.shape[:2]
    y = o.conv1x1_q8(x, wt, b, relu)
    leaves = [t for t in (x, wt, b) if t is not None]
    grads = dict(zip(["x", "w", "b"], torch.autograd.grad(y, leaves, dy)))
    half = 2.0 ** -8 if dtype == BF else 2.0 ** -11
    tiny = 2.0 ** -25 if dtype == HF else 1e-36
    x8, w8 = q8_ref(rows(x.detach()))[0], q8_ref(wt.detach().view(cout, c), True)[0]
    bb = b.detach().double() if b is not None else torch.zeros(cout, device="cuda").double()
    ref, S = x8 @ w8.t() + bb, x8.abs() @ w8.abs().t() + bb.abs()
    if relu:
        ref = ref.clamp(min=0)
    tol = half * ref.abs() + (1 + half) * ((c + 2) * 2.0 ** -23 * S + group_tol(x8, w8)) + tiny
    assert y.shape == (x.shape[0], cout, x.shape[2], x.shape[3]) and y.dtype == dtype and y.is_contiguous(memory_format=torch.channels_last)
    assert bool(((rows(y.detach()).double() - ref).abs() <= tol).all())
    g = rows(dy)
    if relu:
        g = g * (rows(y.detach()) > 0)
    g8 = q8_ref(g.contiguous())[0]
    ref, S = g8 @ w8, g8.abs() @ w8.abs()
    tol = half * ref.abs() + (1 + half) * ((cout + 2) * 2.0 ** -23 * S + group_tol(g8, w8.t())) + tiny
    assert grads["x"].shape == x.shape and grads["x"].dtype == dtype
    assert bool(((rows(grads["x"]).double() - ref).abs() <= tol).all())
    M = g.shape[0]
    ref, S = g.double().t() @ x8, g.abs().double().t() @ x8.abs()
    assert grads["w"].dtype == wt.dtype and grads["w"].shape == wt.shape
    assert bool(((grads["w"].view(cout, c).double() - ref).abs() <= (M + 2) * 2.0 ** -23 * S + 1e-36).all())
    if b is not None:
        assert bool(((grads["b"].double() - g.double().sum(0)).abs() <= (M + 2) * 2.0 ** -23 * g.abs().double().sum(0) + 1e-36).all())
    return y, grads


@pytest.mark.parametrize("n,c,h,w,cout", [(1, 1, 1, 1, 1), (2, 96, 23, 41, 40), (1, 8, 3, 5, 19), (3, 130, 9, 7, 21), (2, 256, 17, 31, 256), (8, 512, 1, 1, 128),
                                          (1, 64, 65, 129, 2), (2, 1000, 5, 6, 72), (1, 320, 40, 50, 384)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_conv1x1(n, c, h, w, cout, dtype):
    check_conv(*conv_case(n, c, h, w, cout, dtype))


@pytest.mark.parametrize("relu", [False, True])
def test_conv1x1_without_bias_and_with_relu(relu):
    check_conv(*conv_case(2, 128, 16, 24, 64, BF, bias=False), relu=relu)
    check_conv(*conv_case(2, 128, 16, 24, 48, HF), relu=relu)


def test_conv1x1_strided_operands():
    """an NCHW input, a strided view, NCHW / expanded / offset gradients"""
    x, wt, b, dy = conv_case(2, 64, 14, 22, 24, BF)
    check_conv(x.detach().contiguous().requires_grad_(), wt, b, dy.contiguous())
    check_conv(x.detach()[:, :, ::2, ::2].requires_grad_(), wt, b, dy[:, :, ::2, ::2])
    check_conv(x, wt, b, dy[:, :, :1, :1].expand(2, 24, 14, 22))
    flat = torch.empty(dy.numel() + 1, dtype=BF, device="cuda")
    off = flat[1:].view(2, 14, 22, 24).permute(0, 3, 1, 2)
    off.copy_(dy)
    check_conv(x, wt, b, off)


def test_conv1x1_partial_gradients_and_empty():
    o = ops()
    x, wt, b, dy = conv_case(2, 40, 6, 10, 24, BF)
    _, full = check_conv(x, wt, b, dy)
    for leaves, keys in (((x,), "x"), ((wt,), "w"), ((b,), "b"), ((wt, b), "wb")):
        args = [t if any(t is u for u in leaves) else t.detach() for t in (x, wt, b)]
        got = torch.autograd.grad(o.conv1x1_q8(*args), leaves, dy)
        for k, g in zip(keys, got):
            assert torch.equal(g, full[k])
    e = torch.empty((0, 40, 6, 10), dtype=BF, device="cuda", requires_grad=True)
    y = o.conv1x1_q8(e, wt, b)
    ge, gw, gb = torch.autograd.grad(y, (e, wt, b), torch.empty_like(y))
    assert y.shape == (0, 24, 6, 10) and ge.shape == e.shape and not bool(gw.any()) and not bool(gb.any())


def test_conv1x1_of_rows_past_32_bits():
    """2.16 GB of result and of its gradient: a sample of each output against 64 bits"""
    o = ops()
    M, C, N = 66000, 512, 16384
    x, w = rand((1, 1, M, C), BF, 1, 0.3).permute(0, 3, 1, 2).requires_grad_(), (rand((N, C), F32, 2, 0.2) / math.sqrt(C)).view(N, C, 1, 1).requires_grad_()
    dy = rand((1, 1, M, N), BF, 3, 0.0).permute(0, 3, 1, 2)
    y = o.conv1x1_q8(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    r = torch.tensor([0, 1, 777, 40000, M - 300, M - 2, M - 1], device="cuda")
    n = torch.tensor([0, 5, 127, 128, 9000, N - 1], device="cuda")
    w8, x8 = q8_ref(w.detach().view(N, C), True)[0], q8_ref(rows(x.detach()))[0]
    ref, S = x8[r] @ w8.t(), x8[r].abs() @ w8.abs().t()
    got = rows(y.detach())[r].double()
    assert bool(((got - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * ((C + 2) * 2.0 ** -23 * S + group_tol(x8[r], w8))).all())
    g = rows(dy)
    g8 = q8_ref(g[r])[0]
    ref, S = g8 @ w8, g8.abs() @ w8.abs()
    assert bool(((rows(dx)[r].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * ((N + 2) * 2.0 ** -23 * S + group_tol(g8, w8.t()))).all())
    gn = g[:, n].double()
    assert bool(((dw.view(N, C)[n].double() - gn.t() @ x8).abs() <= (M + 2) * 2.0 ** -23 * (gn.abs().t() @ x8.abs())).all())


def test_maps_past_32_bit_offsets():
    """2.15e9 values: the streaming 1x1 convolution and the block tail, first and last rows against 64 bits"""
    from mgnet_amd.modeling.layers import InPlaceABNSync
    o = ops()
    M, C = (1 << 23) + 133, 256
    r = torch.cat([torch.arange(300), torch.arange(M - 300, M)]).cuda()
    as_map = lambda t: t.view(1, M, 1, -1).permute(0, 3, 1, 2)  # noqa: E731
    x2, g2 = torch.zeros((M, C), dtype=BF, device="cuda"), torch.zeros((M, C), dtype=BF, device="cuda")
    x2[r], g2[r] = rand((600, C), BF, 1, 0.3), rand((600, C), BF, 2, 0.0)
    x, w = as_map(x2).requires_grad_(), (rand((C, C), F32, 3, 0.2) / 16).view(C, C, 1, 1).requires_grad_()
    y = o.conv1x1_q8(x, w, None)
    dx, dw = torch.autograd.grad(y, (x, w), as_map(g2))
    w8, x8, g8, gr = q8_ref(w.detach().view(C, C), True)[0], q8_ref(x2[r])[0], q8_ref(g2[r])[0], g2[r].double()
    for got, a, b in ((rows(y.detach())[r], x8, w8.t()), (rows(dx)[r], g8, w8)):
        ref = a @ b
        assert bool(((got.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 1.01 * ((C + 2) * 2.0 ** -23 * (a.abs() @ b.abs()) + group_tol(a, b.t()))).all())
    assert bool(((dw.view(C, C).double() - gr.t() @ x8).abs() <= 602 * 2.0 ** -23 * (gr.abs().t() @ x8.abs())).all())   # (the other rows add zeros)
    assert not bool(rows(y.detach())[300:M - 300].any()) and not bool(rows(dx)[300:M - 300].any())
    del y, dx
    norm = InPlaceABNSync(C, activation="identity").cuda()
    s = as_map(torch.zeros((M, C), dtype=BF, device="cuda")).requires_grad_()
    y = o.abn_add_relu_q8(x, norm, s)
    dx, ds = torch.autograd.grad(y, (x, s), as_map(g2))
    # Of M rows 600 are not zero: mean and variance from their sums; gain 1 + eps, offset 0.  The statistics are fp32 sums around the mean c of
    # 64 rows of which the first is not zero, c = x[0] / 64: n terms of (x - c)^2 and of x - c in a row (M / (512 * 16) a thread, 16 threads)
    # put the variance off by n 2^-24 (var + (mean - c)^2), the mean by n 2^-24 (|mean| + |c|), twice that with the difference of the two sums
    xr = x2[r].double()
    mean, var = xr.sum(0) / M, (xr * xr).sum(0) / M
    var = var - mean ** 2
    c, n = xr[0] / 64, M / (512 * 16) + 16
    gain = (1 + norm.eps) / torch.sqrt(var + norm.eps)
    lack = n * 2.0 ** -24 * (var + (mean - c) ** 2) / (var + norm.eps)         # of the gain: half the variance's relative share, twice
    assert float(lack.max()) < 0.02
    ref = torch.relu(gain * (xr - mean))
    tol = 2.0 ** -8 * ref + 1.02 * (lack * gain * (xr - mean).abs() + gain * 2 * n * 2.0 ** -24 * (mean.abs() + c.abs())) + 2.0 ** -20 * gain * (xr.abs() + mean.abs())
    assert bool(((rows(y.detach())[r].double() - ref).abs() <= tol).all())
    kept = (rows(y.detach())[r] > 0).double()
    assert equal(rows(ds)[r].double(), gr * kept)
    assert bool(torch.isfinite(rows(dx)[r]).all()) and bool(torch.isfinite(rows(dx)[M // 2:M // 2 + 100]).all())


def test_conv1x1_gradient_against_differences():
    """<dW, V>, <db, v> and <dx, U> against differences of the unquantised convolution in 64 bits: q(.) is off by at most 2^-4 of a value
    (2^-10 * 2^e next to a block's largest, itself under 2^-4 of the term's share here)"""
    x, wt, b, dy = conv_case(1, 128, 9, 8, 128, BF, seed=20)
    y = ops().conv1x1_q8(x, wt, b)
    dx, dw, db = torch.autograd.grad(y, (x, wt, b), dy)
    X, W, B, G = rows(x.detach()).double(), wt.detach().view(128, 128).double(), b.detach().double(), rows(dy).double()
    f = lambda X, W, B: (G * (X @ W.t() + B)).sum()  # noqa: E731
    h = 2.0 ** -10
    for t, grad, kind in ((W, dw.view(128, 128), "W"), (X, rows(dx), "X"), (B, db, "B")):
        V = torch.randn(t.shape, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda").double()
        lo, hi = (f(X + d * (V if kind == "X" else 0), W + d * (V if kind == "W" else 0), B + d * (V if kind == "B" else 0)) for d in (-h, h))
        diff = (hi - lo) / (2 * h)
        got = (grad.double() * V).sum()
        if kind == "B":
            tol = (G.shape[0] + 2) * 2.0 ** -23 * (G.abs() * V.abs()).sum()
        elif kind == "W":
            err = (q8_ref(rows(x.detach()))[0] - X).abs()
            assert bool((err <= 2.0 ** -4 * X.abs() + 2.0 ** -10 * 2.0 ** -7 * X.abs().amax(1, keepdim=True)).all())
            tol = (G.abs().t() @ err * V.abs()).sum() + (G.shape[0] + 2) * 2.0 ** -23 * (G.abs().t() @ X.abs() * V.abs()).sum()
        else:
            G8, W8 = q8_ref(rows(dy).contiguous())[0], q8_ref(wt.detach().view(128, 128), True)[0]
            tol = (((G8 - G).abs() @ W8.abs() + G.abs() @ (W8 - W).abs()) * V.abs()).sum() + (2.0 ** -8 + 130 * 2.0 ** -22 + 7 * 2.0 ** -13) * ((G8.abs() @ W8.abs()) * V.abs()).sum()
        assert abs(float(got - diff)) <= float(tol) + 1e-9 * abs(float(diff)), (kind, float(got), float(diff), float(tol))


# ---- block tail ------------------------------------------------------------------------------------------------------------------------
def tail_case(n, c, h, w, dtype, seed=0):
    from mgnet_amd.modeling.layers import InPlaceABNSync
    norm = InPlaceABNSync(c, momentum=0.01, activation="identity").cuda()
    with torch.no_grad():
        norm.weight.copy_(rand((c,), F32, seed + 5, 0.3))
        norm.bias.copy_(rand((c,), F32, seed + 6, 0.0))
    x = rand_map(n, c, h, w, dtype, seed)
    x = (x + rand_map(1, c, 1, 1, dtype, seed + 1)).requires_grad_()      # channels with a mean
    s = rand_map(n, c, h, w, dtype, seed + 2, 0.2).requires_grad_()
    g = (rand_map(n, c, h, w, dtype, seed + 3, 0.2) + rand_map(1, c, 1, 1, dtype, seed + 4, 0.0)).contiguous(memory_format=torch.channels_last)
    return x, norm, s, g


def check_tail(x, norm, s, g):
    """fp32 sums: at most 16 + 64 rows one after another in a thread and a block (M < 128k), the rest in 64 bits: 96 * 2^-23 < 2^-16 of the
    sum of magnitudes; a handful of further fp32 operations stays below the same bound, so 2^-15 covers every statistic and sum."""
    rm, rv = norm.running_mean.clone().double(), norm.running_var.clone().double()
    dtype, half, u = x.dtype, 2.0 ** -8 if x.dtype == BF else 2.0 ** -11, 2.0 ** -15
    tiny = 2.0 ** -25 if dtype == HF else 1e-36
    y = ops().abn_add_relu_q8(x, norm, s)
    dx, ds, dw, db = torch.autograd.grad(y, (x, s, norm.weight, norm.bias), g)
    X, S, G = rows(x.detach()).double(), rows(s.detach()).double(), rows(g).double()
    M = X.shape[0]
    mean, var = X.mean(0), X.var(0, unbiased=False)
    dev = (X - X[0]).abs().mean(0) + (X - mean).abs().mean(0)
    rstd, w = (var + norm.eps) ** -0.5, norm.weight.detach().double()
    gain = w.abs() + norm.eps
    # the variance comes from sums around the mean of a sample of rows: second moment there, for which the one around the first row stands (at
    # least the variance itself)
    rv_err = u * ((X - X[0]) ** 2).mean(0) / (var + norm.eps)
    xh = (X - mean) * rstd
    ref = (gain * xh + norm.bias.detach().double() + S)
    tol = half * ref.abs() + gain * rstd * (u * dev + u * (X.abs() + mean.abs())) + gain * xh.abs() * (rv_err + u) + u * (norm.bias.detach().double().abs() + S.abs()) + tiny
    Y = rows(y.detach())
    assert bool(((Y.double() - ref.clamp(min=0)).abs() <= tol).all())
    assert bool(((norm.running_mean.double() - (0.99 * rm + 0.01 * mean)).abs() <= u * (rm.abs() + mean.abs() + dev)).all())
    assert bool(((norm.running_var.double() - (0.99 * rv + 0.01 * var * (M / max(M - 1, 1)))).abs() <= u * rv.abs() + 0.02 * (u + rv_err) * (var + norm.eps)).all())
    dz = rows(g) * (Y > 0)
    assert torch.equal(rows(ds), dz)
    dz = dz.double()
    X8 = q8_ref(rows(x.detach()))[0]
    xh8, xe = (X8 - mean) * rstd, rstd * u * dev + ((X8 - mean) * rstd).abs() * (rv_err + u) + u * rstd * (X8.abs() + mean.abs())
    s1, s2 = dz.sum(0), (dz * xh8).sum(0)
    e1 = u * dz.abs().sum(0)
    e2 = u * (dz.abs() * xh8.abs()).sum(0) + (dz.abs() * xe).sum(0)
    assert bool(((db.double() - s1).abs() <= e1 + 1e-36).all())
    assert bool(((dw.double() - s2 * w.sign()).abs() <= e2 + 1e-36).all())
    ref = gain * rstd * (dz - s1 / M - xh8 * s2 / M)
    tol = half * ref.abs() + (1 + half) * gain * rstd * (e1 / M + xh8.abs() * e2 / M + xe * (s2.abs() + e2) / M + (u + rv_err) * (dz.abs() + s1.abs() / M + xh8.abs() * s2.abs() / M)) + tiny
    assert bool(((rows(dx).double() - ref).abs() <= tol).all())
    return y, dx, ds, dw, db


@pytest.mark.parametrize("n,c,h,w", [(1, 8, 1, 2), (2, 512, 9, 13), (8, 64, 1, 1), (2, 24, 11, 5), (1, 320, 7, 7), (2, 128, 33, 65), (3, 72, 64, 96), (1, 1032, 3, 4)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_block_tail(n, c, h, w, dtype):
    check_tail(*tail_case(n, c, h, w, dtype))


def test_block_tail_strided_operands_and_partial_gradients():
    x, norm, s, g = tail_case(2, 64, 12, 20, BF, 3)
    a = check_tail(x.detach().contiguous().requires_grad_(), norm, s.detach().contiguous().requires_grad_(), g.contiguous())
    b = check_tail(x, norm, s, g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    flat = torch.empty(x.numel() + 3, dtype=BF, device="cuda")
    off = flat[3:].view(2, 12, 20, 64).permute(0, 3, 1, 2)
    off.copy_(x.detach())
    check_tail(off.requires_grad_(), norm, s, g)
    y = ops().abn_add_relu_q8(x.detach(), norm, s)
    (ds,) = torch.autograd.grad(y, (s,), g)
    assert torch.equal(ds, b[2])


def test_block_tail_one_row_and_inference():
    o = ops()
    x, norm, s, g = tail_case(1, 16, 1, 1, BF, 5)     # one row: the variance is zero, x_hat too
    check_tail(x, norm, s, g)
    x, norm, s, g = tail_case(2, 40, 5, 6, HF, 6)
    norm.eval()
    with torch.no_grad():
        y = o.abn_add_relu_q8(x, norm, s)
    z = (norm.weight.abs() + norm.eps).view(1, -1, 1, 1) * x.float() / torch.sqrt(norm.running_var + norm.eps).view(1, -1, 1, 1) + norm.bias.view(1, -1, 1, 1)
    ref = torch.relu(z + s.float())
    assert bool(((y.float() - ref).abs() <= 2.0 ** -11 * ref + 2.0 ** -20 * (z.abs() + s.float().abs() + 1)).all())
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(o.abn_add_relu_q8(x, norm, s), (x,), g)


@pytest.mark.parametrize("C", [8, 40, 128, 200])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_block_tail_statistics_of_sparse_channels(C, dtype):
    """channels that are zero almost everywhere, but not in the first row; and channels with a large mean"""
    from mgnet_amd.modeling.layers import InPlaceABNSync
    M = 300000
    x2 = torch.zeros((M, C), dtype=dtype, device="cuda")
    x2[0], x2[M // 3:M // 3 + 5] = 90.0, rand((5, C), dtype, 1, 0.0)
    x2[:, C // 2:] += 100.0
    norm = InPlaceABNSync(C, momentum=1.0, activation="identity").cuda()
    x = x2.view(1, M, 1, C).permute(0, 3, 1, 2)
    y = ops().abn_add_relu_q8(x.requires_grad_(), norm, torch.zeros_like(x))
    xd = x2.double()
    mean, var = xd.mean(0), xd.var(0, unbiased=True)
    # fp32 sums around c, the mean of at least 64 rows, 90 / 64 from the mean at most: n terms a thread and 64 threads at most, n <= M / (512 * 16) + 64
    n, far = M / (512 * 16) + 64, (90 / 64) ** 2
    assert bool(((norm.running_mean.double() - mean).abs() <= 2.0 ** -23 * mean.abs() + 2 * n * 2.0 ** -24 * (90 / 64 + 1)).all())
    assert bool(((norm.running_var.double() - var).abs() <= 2 * n * 2.0 ** -24 * (var + far) + 2.0 ** -22 * var).all())
    assert bool(torch.isfinite(y.float()).all())


def test_block_tail_of_two_ranks(monkeypatch):
    """the exchange of a process group of two, played by one process: each half of the batch sees the whole batch's statistics and sums"""
    from mgnet_amd import _C
    from mgnet_amd.modeling import ops as o, q8
    from mgnet_amd.modeling.layers import InPlaceABNSync
    n, c, h, w = 4, 72, 9, 7
    x, s, dy = (rand_map(n, c, h, w, BF, k, 0.3) for k in (1, 2, 3))

    def norm():
        torch.manual_seed(5)
        m = InPlaceABNSync(c, momentum=0.01, activation="identity").cuda()
        with torch.no_grad():
            m.weight.uniform_(0.5, 1.5)
            m.bias.uniform_(-0.5, 0.5)
        return m

    def run(x, s, dy, m):
        x, s = x.clone(memory_format=torch.channels_last).requires_grad_(), s.clone(memory_format=torch.channels_last).requires_grad_()
        y = o.abn_add_relu_q8(x, m, s)
        return (y.detach(),) + torch.autograd.grad(y, (x, s, m.weight, m.bias), dy)

    whole = norm()
    ref = run(x, s, dy, whole)
    halves = [tuple(t[k:k + 2] for t in (x, s, dy)) for k in (0, 2)]
    M = 2 * h * w
    stats = []
    for xs, _, _ in halves:
        part, shift = _C.q8_tail_stats(rows(xs).contiguous(), M, c)
        stats.append(_C.iabn_from_partials(part, c, M, shift, stats_only=True))
    monkeypatch.setattr(q8, "_dist_active", lambda group: True)
    monkeypatch.setattr(q8.dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(o, "_gather_stats", lambda own, world, group: torch.stack([t.view_as(own) for t in stats]))
    own = []
    monkeypatch.setattr(q8, "_allreduce_sums", lambda t, group: own.append(t.clone()) or t)
    for half in halves:
        run(*half, norm())
    monkeypatch.setattr(q8, "_allreduce_sums", lambda t, group: own[0] + own[1])
    ms = [norm(), norm()]
    got = [run(*half, m) for half, m in zip(halves, ms)]
    # fp32 sums in another order (2^-20 of their terms covers 126 of them), then one rounding on either side
    for k in range(3):
        a, b = torch.cat([g[k] for g in got]).double(), ref[k].double()
        assert bool(((a - b).abs() <= 2.0 ** -7 * b.abs() + 2.0 ** -16 * (1 + b.abs().max())).all()), k
    for k in (3, 4):       # of the whole batch's gradient each rank has its share
        a, b = got[0][k].double() + got[1][k].double(), ref[k].double()
        assert bool(((a - b).abs() <= 2.0 ** -16 * (1 + b.abs().max())).all()), k
    for m in ms:
        for t, r in ((m.running_mean, whole.running_mean), (m.running_var, whole.running_var)):
            assert bool(((t - r).abs() <= 2.0 ** -18 * (1 + r.abs())).all())


def test_nan_and_infinities_reach_the_result():
    """a NaN pixel poisons its own outputs (and, through the statistics, its channel), never another row's"""
    o = ops()
    x, wt, b, dy = conv_case(1, 64, 8, 8, 16, BF)
    x = x.detach().clone(memory_format=torch.channels_last)
    x[0, 5, 2, 3] = math.nan
    y = o.conv1x1_q8(x, wt.detach(), b.detach())
    assert bool(torch.isnan(y[0, :, 2, 3]).all()) and int(torch.isnan(y).sum()) == 16
    x, norm, s, g = tail_case(1, 16, 6, 6, BF, 8)
    x = x.detach().clone(memory_format=torch.channels_last)
    x[0, 3, 1, 1] = math.inf
    y = o.abn_add_relu_q8(x, norm, s.detach())
    assert bool(torch.isnan(y[0, 3]).all()) and not bool(torch.isnan(y[0, :3]).any())


# ---- together --------------------------------------------------------------------------------------------------------------------------
def train_once(o, x, w1, b1, norm, s, w2, g):
    """1x1 convolution -> block tail -> 1x1 convolution, as a bottleneck's end would use them"""
    h = o.conv1x1_q8(x, w1, b1)
    y = o.abn_add_relu_q8(h, norm, s)
    z = o.conv1x1_q8(y, w2)
    return (z,) + torch.autograd.grad(z, (x, w1, b1, norm.weight, norm.bias, s, w2), g)


def chain(seed=0, dtype=BF):
    x, w1, b1, _ = conv_case(2, 96, 10, 14, 64, dtype, seed=seed)
    _, norm, s, _ = tail_case(2, 64, 10, 14, dtype, seed=seed + 30)
    w2 = (rand((40, 64), F32, seed + 50, 0.2) / 8).view(40, 64, 1, 1).requires_grad_()
    return x, w1, b1, norm, s, w2, rand_map(2, 40, 10, 14, dtype, seed + 60)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_chain_is_reproducible_and_near_the_16_bit_chain(dtype):
    o = ops()
    a = chain(1, dtype)
    first = train_once(o, *a)
    again = train_once(o, *a)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    # against the same chain in 64 bits: the 8-bit rounding is uniform noise of at most 2^-4 of a value -- 2^-4 / sqrt(3) of its size -- and
    # enters a result through at most four packed operands one behind the other
    x, w1, b1, norm, s, w2, g = [t.detach().double().requires_grad_() if isinstance(t, torch.Tensor) else t for t in a]
    gam, bet = norm.weight.detach().double().requires_grad_(), norm.bias.detach().double().requires_grad_()
    h = rows(x) @ w1.view(64, 96).t() + b1
    xh = (h - h.mean(0)) / torch.sqrt(h.var(0, unbiased=False) + norm.eps)
    y = torch.relu((gam.abs() + norm.eps) * xh + bet + rows(s))
    z = y @ w2.view(40, 64).t()
    *grads, dh, dy = torch.autograd.grad(z, (x, w1, b1, gam, bet, s, w2, h, y), rows(g))
    share = 4 * 2.0 ** -4 / math.sqrt(3)
    # The noise of h moves some pre-activations across the ReLU's corner.  Such an element's gradient term is not off by a share of itself, it
    # appears or vanishes whole: with F these elements (taken from the two results), a sum over pixels is off by at most the sum of |term| over
    # F, a map by the 2-norm of dy over F.  And the noise of a sum of terms is the share of the terms' 2-norm, which for the norm's weight
    # and bias (sums of both signs) is more than the share of the sum.
    y8 = o.abn_add_relu_q8(o.conv1x1_q8(a[0], a[1], a[2]), a[3], a[4])
    F = (rows(y8.detach()) > 0) != (y > 0)
    dz, xh = torch.where(y > 0, dy, 0.0), xh.detach()
    assert float(F.double().mean()) < 0.05
    flip = float(torch.where(F, dy, 0.0).norm() / dz.norm())
    for k, (p, q) in enumerate(zip(first, [z.detach()] + grads)):
        p = rows(p.detach()) if p.dim() == 4 and p.shape[0] == 2 else p
        q = rows(q) if q.dim() == 4 and q.shape[0] == 2 else q
        if k in (4, 5):
            t = dz * xh if k == 4 else dz
            lost = torch.where(F, (dy * xh if k == 4 else dy).abs(), 0.0).sum(0)
            assert bool(((p.double() - q).abs() <= 4 * share * t.norm(dim=0) + lost).all()), k     # (four deviations)
            continue
        # (b1 stands before a norm over the batch, which takes any constant out again: its gradient is zero, sum dh = 0, and what is left of
        #  it is measured against the terms of that sum)
        rel = float((p.double() - q).norm() / (dh.abs().sum(0) if k == 3 else q).norm())
        assert rel <= share + (flip if k in (1, 2, 3, 6) else 0.0), (k, rel)


@pytest.mark.parametrize("what", ["tile256", "tile128", "tile32", "few", "stream", "conv", "tail", "pack"])
def test_repeats_under_load_are_identical(what):
    """the same call again and again while two other streams keep memory and matrix cores busy: a wait that is too short shows here"""
    o = ops()
    if what in ("conv", "tail"):
        x, wt, b, dy = conv_case(8, 256, 128, 256, 256, BF) if what == "conv" else (None,) * 4
        t = tail_case(8, 64, 256, 512, BF) if what == "tail" else None

        def call():
            if what == "conv":
                y = o.conv1x1_q8(x, wt, b)
                return (y.detach(),) + torch.autograd.grad(y, (x, wt, b), dy)
            xs, norm, sc, g = t
            y = o.abn_add_relu_q8(xs, norm, sc)
            return (y.detach(),) + torch.autograd.grad(y, (xs, sc, norm.weight, norm.bias), g)
    elif what == "pack":
        x = rand((262144, 257), BF, 1)

        def call():
            q = o.q8_pack(x)
            return q.buf, q.unpack()
    else:
        M, N, K = {"tile256": (8192, 8192, 1088), "tile128": (2048, 2048, 2048), "tile32": (60000, 24, 1100), "few": (256, 1024, 4096), "stream": (262144, 256, 256)}[what]
        qa, qb = o.q8_pack(rand((M, K), BF, 1)), o.q8_pack(rand((N, K), F32, 2, 0.3), tile=True)

        def call():
            return (o.q8_matmul(qa, qb),)
    side = [torch.cuda.Stream() for _ in range(2)]
    big, mm = torch.randn(32 << 20, device="cuda"), torch.randn(4096, 4096, device="cuda").to(BF)
    want = call()
    for r in range(10):
        for st in side:
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                big.mul_(1.0001)
                torch.mm(mm, mm)
        assert all(torch.equal(p, q) for p, q in zip(call(), want)), r
    torch.cuda.synchronize()


def test_chain_on_another_stream():
    o = ops()
    a = chain(2)
    want = train_once(o, *a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = train_once(o, *a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))


def test_two_captured_graphs_replayed_against_eager():
    """two graphs of the chain (each with workspaces of its own), replayed in turn with new inputs between the replays"""
    o = ops()
    graphs = []
    for seed in (3, 4):
        a = list(chain(seed))
        a = [t.detach().requires_grad_(t.requires_grad) if isinstance(t, torch.Tensor) else t for t in a]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                out = train_once(o, *a)
        torch.cuda.current_stream().wait_stream(side)
        del out
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = train_once(o, *a)
        graphs.append((graph, a, out))
    for rep in range(4):
        for k, (graph, a, out) in enumerate(graphs):
            with torch.no_grad():
                a[0].copy_(rand_map(2, 96, 10, 14, BF, 100 + 10 * rep + k))
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            want = train_once(o, *a)
            assert all(torch.equal(p, q) for p, q in zip(want, got)), (rep, k)


def test_refusals_on_the_gpu():
    o = ops()
    x = rand_map(1, 16, 4, 4, BF)
    w = torch.zeros((8, 16, 1, 1), device="cuda")
    for bad in (lambda: o.q8_pack(x.double()), lambda: o.q8_pack(x[0]), lambda: o.q8_pack(x, tile=True), lambda: o.conv1x1_q8(x.float(), w),
                lambda: o.conv1x1_q8(x, w[:, :8]), lambda: o.conv1x1_q8(x, torch.zeros((8, 16, 3, 3), device="cuda")), lambda: o.conv1x1_q8(x, w, torch.zeros(7, device="cuda")),
                lambda: o.conv1x1_q8(x, w.cpu()), lambda: o.q8_matmul(o.q8_pack(x), o.q8_pack(torch.zeros((8, 24), device="cuda"), tile=True)),
                lambda: o.q8_matmul(o.q8_pack(x), w), lambda: o.q8_matmul(o.q8_pack(x), o.q8_pack(w.view(8, 16), tile=True), act="gelu"),
                lambda: o.q8_matmul(o.q8_pack(x), o.q8_pack(w.view(8, 16), tile=True), act="leaky_relu", slope=2.0),
                lambda: o.q8_matmul(o.q8_pack(x), o.q8_pack(w.view(8, 16), tile=True), bias=torch.zeros(9, device="cuda")),
                lambda: o.q8_matmul(o.q8_pack(x), o.q8_pack(w.view(8, 16), tile=True), out_dtype=torch.float64), lambda: o.q8_pack(x).unpack(torch.int8)):
        with pytest.raises(ValueError):
            bad()
    from mgnet_amd.modeling.layers import InPlaceABNSync
    norm = InPlaceABNSync(16, activation="identity").cuda()
    leaky = InPlaceABNSync(16).cuda()
    for bad in (lambda: o.abn_add_relu_q8(x, leaky, x), lambda: o.abn_add_relu_q8(x, norm, x.float()), lambda: o.abn_add_relu_q8(x, norm, x[:, :, :2]),
                lambda: o.abn_add_relu_q8(x[:, :12], norm, x[:, :12]), lambda: o.abn_add_relu_q8(x[:, :8], norm, x[:, :8])):
        with pytest.raises(ValueError):
            bad()
