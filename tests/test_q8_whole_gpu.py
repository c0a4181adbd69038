"""8-bit operators on whole numbers: every kernel of the product and of the 1x1 convolution, several tiles a block and ragged ones among them,
against 64 bits and to the bit.

Operands are whole numbers up to 7 times a power of two of their block (of a row and 128 channels, or of a weight tile): codes are exact.  A
product has 6 bits and is a multiple of its blocks' powers of two, and so stands whole in the matrix instruction's sum of 8 neighbouring k, whose
unit is 2^-13 of the largest product's binade.  With every partial sum under 2^24 units the fp32 accumulator is exact in any order, bias and a slope
of 1/4 too; the result is rounded once.  So there is no tolerance: a row, a tile, a scale or a range of rows that is left out, added twice or taken from elsewhere shows.

Which kernel ran is read from the recorder of launches, and compared: a size that another threshold moves to another kernel fails here."""
import ctypes

import pytest
import torch

from test_q8_gpu import BF, F32, HF, check_product, ops, rand, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _give_the_memory_back():
    yield
    torch.cuda.empty_cache()


def launched(fn):
    """fn() and the names of the library's kernels that it launched"""
    from mgnet_amd import _C
    L = _C.lib()
    _C.check(L.mgn_plan_begin(), "mgn_plan_begin")
    try:
        out = fn()
    except BaseException:
        L.mgn_plan_abort()
        raise
    plan, info, names = ctypes.c_void_p(), _C.PlanNodeInfo(), []
    _C.check(L.mgn_plan_end(ctypes.byref(plan)), "mgn_plan_end")
    for i in range(L.mgn_plan_node_count(plan)):
        _C.check(L.mgn_plan_node_info(plan, i, ctypes.byref(info)), "mgn_plan_node_info")
        names.append(info.name.decode())
    L.mgn_plan_free(plan)
    return out, names


def whole(m, k, seed, largest=7, doubled=3, tile=False):
    """[m, k] whole numbers up to `largest` times 1 .. 2^doubled, one power for a row's 128 channels (tile: for 128 rows as well); float32"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(-largest, largest + 1, (m, k), generator=g, device="cuda").float()
    s = torch.exp2(torch.randint(0, doubled + 1, (-(-m // 128) if tile else m, -(-k // 128)), generator=g, device="cuda").float())
    s = s.repeat_interleave(128, 1)[:, :k]
    return x * (s.repeat_interleave(128, 0)[:m] if tile else s)


# ---- product: (M, N, K, result, kernel).  Streaming kernels: more than two tiles a block and a ragged last one, but for the marked cases
LIMIT = 2 ** 24
PRODUCTS = [(270001, 21, 100, BF, "stream_1_any_packed"), (270001, 24, 128, F32, "stream_1_any_packed"), (135001, 1, 200, HF, "stream_2_any_packed"),
            (135001, 32, 256, F32, "stream_2_any_packed"), (67601, 19, 500, BF, "stream_4_any_packed"), (67601, 32, 512, F32, "stream_4_any_packed"),
            (270001, 24, 100, BF, "stream_1_32_packed"), (135001, 32, 136, HF, "stream_2_32_packed"), (67601, 8, 264, BF, "stream_4_32_packed"),
            (270001, 40, 72, BF, "stream_1_128_packed"), (135001, 128, 256, HF, "stream_2_128_packed"), (67601, 120, 384, BF, "stream_4_128_packed"),
            (270001, 256, 72, BF, "stream_1_256_packed"), (135001, 136, 256, HF, "stream_2_256_packed"), (70001, 256, 512, BF, "stream_4_256_packed"),
            (140001, 264, 128, BF, "stream_1_256_packed"), (68001, 520, 200, BF, "stream_2_256_packed"), (25001, 776, 300, HF, "stream_4_256_packed"),
            (30001, 40, 100, BF, "stream_1_128_packed"), (45001, 24, 257, HF, "stream_4_32_packed"),       # (fewer tiles than blocks; three of four blocks of k)
            (1, 1, 1, F32, "mm_small"), (64, 1000, 4000, BF, "mm_small"), (33, 19, 129, HF, "mm_small"), (1300, 1027, 700, F32, "mm_small"),
            (60001, 21, 530, BF, "mm_128x32"), (50003, 32, 1100, F32, "mm_128x32"), (400003, 3, 700, HF, "mm_128x32"),
            (2300, 1030, 700, BF, "mm_128x128"), (16001, 512, 130, F32, "mm_128x128"), (4097, 515, 2050, HF, "mm_128x128"),
            (16380, 1021, 130, BF, "mm_256x256"), (50001, 200, 256, F32, "mm_256x256"), (8190, 2045, 1090, HF, "mm_256x256")]
TILES = ("mm_small", "mm_128x32", "mm_128x128", "mm_256x256")


def test_every_kernel_of_the_product_is_among_the_cases():
    assert {p[4] for p in PRODUCTS} == {f"stream_{k}_{s}_packed" for k in (1, 2, 4) for s in ("any", "32", "128", "256")} | set(TILES)


def _product(M, N, K, dtype):
    o = ops()
    a, b, bias = whole(M, K, M + N), whole(N, K, N + K, tile=True) * 2.0 ** -12, whole(1, N, K)[0] * 2.0 ** -12
    assert K * 49 * 64 + 56 <= LIMIT
    ref = a.double() @ b.double().t()
    return o.q8_pack(a.to(BF)), o.q8_pack(b, tile=True), bias, ref


@pytest.mark.parametrize("M,N,K,dtype,kernel", PRODUCTS)
def test_product_of_whole_numbers(M, N, K, dtype, kernel):
    o = ops()
    qa, qb, bias, ref = _product(M, N, K, dtype)
    y, names = launched(lambda: o.q8_matmul(qa, qb, out_dtype=dtype))
    assert len(names) == 1 and kernel in names[0], names
    assert torch.equal(y, ref.float().to(dtype))
    ref = ref + bias.double()
    assert torch.equal(o.q8_matmul(qa, qb, bias, "leaky_relu", 0.25, dtype), torch.where(ref > 0, ref, ref / 4).float().to(dtype))
    assert torch.equal(o.q8_matmul(qa, qb, bias, "relu", out_dtype=dtype), ref.clamp(min=0).float().to(dtype))


@pytest.mark.parametrize("M,N,K,dtype,kernel", [p for p in PRODUCTS if p[0] < 30000 or "any" in p[4] or p[1] in (3, 21, 200)])
@pytest.mark.parametrize("more,at", [(0, 1), (3, 5), (8, 8)])
def test_product_into_rows_of_any_pitch(M, N, K, dtype, kernel, more, at):
    """rows `more` elements longer than N from element `at` on: the same numbers there, and nothing else"""
    from mgnet_amd import _C
    qa, qb, bias, ref = _product(M, N, K, dtype)
    ldo = N + more
    buf = torch.full((at + M * ldo + 32,), 7.0, dtype=dtype, device="cuda")
    out = buf[at:at + M * ldo].view(M, ldo)
    pa, pb = qa.buf.data_ptr(), qb.buf.data_ptr()
    _C.check(_C._fn("mgn_q8_matmul", out)(pa, pa + _C.q8_code_bytes(M, K), M, pb, pb + _C.q8_code_bytes(N, K), N, K, bias.data_ptr(), 0, 0.0, out.data_ptr(),
                                          int(dtype == F32), ldo, _C._stream()), "mgn_q8_matmul")
    assert torch.equal(out[:, :N], (ref + bias.double()).float().to(dtype))
    out[:, :N] = 7.0
    assert bool((buf == 7.0).all())


# (the largest streams on values of every size, within the bounds of test_q8_gpu.py)
@pytest.mark.parametrize("M,N,K,dtype", [(270001, 24, 96, BF), (140003, 21, 200, F32), (70001, 120, 384, HF), (262147, 256, 72, BF), (135001, 136, 256, BF), (68003, 520, 512, HF)])
def test_streamed_product(M, N, K, dtype):
    a, b = rand((M, K), BF, M + N), rand((N, K), F32, N + K, 0.3) / K ** 0.5
    check_product(a, b, rand((N,), F32, 2, 0.0), "leaky_relu", 0.25, dtype)


# ---- 1x1 convolution: (C, Cout, kernel of the forward call, kernel of the data gradient), 132271 pixels: two rounds or more in every streaming kernel
CONVS = [(96, 19, "1_any_keep", "1_128_h16"), (96, 24, "1_32_keep", "1_128_h16"), (128, 128, "1_128_keep", "1_128_h16"), (64, 256, "1_256_keep", "2_128_h16"),
         (200, 21, "2_any_keep", "1_256_h16"), (136, 32, "2_32_keep", "1_256_h16"), (256, 40, "2_128_keep", "1_256_h16"), (256, 200, "2_256_keep", "2_256_h16"),
         (512, 19, "4_any_keep", "1_256_h16"), (264, 8, "4_32_keep", "1_256_h16"), (384, 120, "4_128_keep", "1_256_h16"), (512, 264, "4_256_keep", "4_256_h16"),
         (24, 100, "mm_", "1_32_h16"), (8, 256, "1_256_keep", "2_32_h16"), (32, 400, "1_256_keep", "4_32_h16"), (40, 512, "1_256_keep", "4_128_h16"),
         (19, 64, "1_128_packed", "1_any_h16"), (21, 200, "mm_", "2_any_h16"), (1, 257, "mm_", "4_any_h16"), (264, 264, "4_256_keep", "4_256_h16"), (640, 48, "mm_", "1_256_h16")]


def test_every_streaming_kernel_is_among_the_convolutions():
    names = {n for c in CONVS for n in c[2:] if n != "mm_" and "packed" not in n}
    assert names == {f"{k}_{s}_{src}" for k in (1, 2, 4) for s in ("any", "32", "128", "256") for src in ("keep", "h16")}


def _conv(M, C, N, dtype, bound=LIMIT):
    assert M * 7 * 2 * 3 * 2 <= bound and C * 7 * 2 * 7 * 4 + 28 <= bound and N * 3 * 2 * 7 * 4 <= bound
    as_map = lambda t: t.to(dtype).view(1, M, 1, -1).permute(0, 3, 1, 2)  # noqa: E731
    x, dy = as_map(whole(M, C, M + C, doubled=1)).requires_grad_(), as_map(whole(M, N, M + N, largest=3, doubled=1))
    w = (whole(N, C, C + N, doubled=2, tile=True) * 2.0 ** -6).view(N, C, 1, 1).requires_grad_()
    b = (whole(1, N, 5, doubled=2)[0] * 2.0 ** -6).requires_grad_()
    return x, w, b, dy


def check_whole(x, w, b, dy, relu=False):
    """-> the kernels of the forward and of the backward call"""
    N, C = w.shape[:2]
    y, fwd = launched(lambda: ops().conv1x1_q8(x, w, b, relu))
    (dx, dw, db), bwd = launched(lambda: torch.autograd.grad(y, (x, w, b), dy))
    X, W, G = rows(x.detach()).double(), w.detach().view(N, C).double(), rows(dy).double()
    ref = X @ W.t() + b.detach().double()
    if relu:
        G = G * (ref > 0)
        ref = ref.clamp(min=0)
    assert torch.equal(rows(y.detach()), ref.float().to(x.dtype))
    assert torch.equal(rows(dx), (G @ W).float().to(x.dtype))
    assert torch.equal(dw.view(N, C), (G.t() @ X).float()) and torch.equal(db, G.sum(0).float())
    return fwd, bwd


@pytest.mark.parametrize("C,N,fwd,dx", CONVS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_conv1x1_of_whole_numbers(C, N, fwd, dx, dtype):
    f, b = check_whole(*_conv(132271, C, N, dtype))
    assert any(fwd in n for n in f) and any(dx in n for n in b), (f, b)


@pytest.mark.parametrize("M", [1, 2, 63, 64, 65, 127, 129, 1000, 4097, 20011])
@pytest.mark.parametrize("C,N", [(8, 8), (1, 130), (257, 3), (520, 136)])
def test_conv1x1_of_few_whole_numbers(M, C, N):
    check_whole(*_conv(M, C, N, BF))
    check_whole(*_conv(M, C, N, HF), relu=True)


@pytest.mark.parametrize("M,C,N", [(66000, 512, 16384), (131200, 8, 8192), (66001, 16384, 16)])
def test_weight_gradient_over_ranges_of_rows(M, C, N):
    """sizes whose rows lie in ranges that 32-bit offsets reach: no row is lost or counted twice where two ranges meet"""
    x, w, b, dy = _conv(M, C, N, BF)
    dw, db = torch.autograd.grad(ops().conv1x1_q8(x, w, b), (w, b), dy)
    X, G = rows(x.detach()).float(), rows(dy)
    assert torch.equal(db, torch.cat([G[:, k:k + 1024].double().sum(0) for k in range(0, N, 1024)]).float())
    for k in range(0, N, 1024):
        assert torch.equal(dw[k:k + 1024, :, 0, 0], (G[:, k:k + 1024].double().t() @ X.double()).float()), k
