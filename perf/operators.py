"""The 8-bit operators as they are measured: cases, inputs, plain forms and the calls a user of mgnet_amd makes.

A block is 128 neighbouring channels of one pixel (one row of the [M, C] matrix that a channels-last map is), or a 128 x 128 tile of a
weight matrix.  It is held as e4m3 codes and one power of two 2^e, with e the smallest exponent for which the block's largest finite
magnitude is at most 448 * 2^e (and e >= -111); a code is the value divided by 2^e, rounded to the nearest e4m3 number, ties to even.
Magnitudes above the largest e4m3 number of the source type (1.875 * 2^127, or 1.875 * 2^15 in fp16) count as that number; NaN and
infinities become NaN.

  checkpoint   x -> codes and exponents -> x^, the way an activation waits for the backward pass
  product      out = act(A B^T + bias) of two packed matrices A [M, K], B [N, K]
  pointwise    a 1x1 convolution trained in 8 bits: y = q(x) q(W)^T + bias; dx = q(dy) q(W); dW = dy^T q(x); db = sum dy
  tail         y = relu(norm(x) + shortcut) with batch statistics, x kept in 8 bits for the backward pass
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128
EPS = 1e-5
MOMENTUM = 0.01


def listed():
    return [
        # the pooled vector of a channel attention: the smallest thing a training step keeps for its backward pass
        {"name": "checkpoint_vector", "kind": "checkpoint", "n": 8, "h": 1, "w": 1, "c": 512, "dtype": "bf16"},
        # a decoder's 256-channel map at 1/8 of a batch of 8 frames of 1024 x 2048
        {"name": "checkpoint_map8", "kind": "checkpoint", "n": 8, "h": 128, "w": 256, "c": 256, "dtype": "bf16"},
        # one vector against a square weight matrix: serving latency
        {"name": "product_row", "kind": "product", "m": 1, "n": 512, "k": 512, "dtype": "bf16", "bias": True, "act": "none"},
        # a 19-class predictor on a padded batch of odd frames
        {"name": "product_classes", "kind": "product", "m": 6930, "n": 19, "k": 320, "dtype": "fp16", "bias": True, "act": "none"},
        # a folded 1x1 convolution + leaky ReLU at inference over the 256-channel maps of 8 frames
        {"name": "product_map8", "kind": "product", "m": 262144, "n": 256, "k": 256, "dtype": "bf16", "bias": True, "act": "leaky_relu"},
        # a large square product: the rate of the matrix cores
        {"name": "product_square", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "bias": False, "act": "none"},
        # training on two small odd crops, few channels, fp16
        {"name": "pointwise_crop", "kind": "pointwise", "n": 2, "h": 23, "w": 41, "c": 96, "cout": 40, "dtype": "fp16"},
        # the pose network's first convolution on the 1/32 maps of 8 frames
        {"name": "pointwise_pose", "kind": "pointwise", "n": 8, "h": 32, "w": 64, "c": 512, "cout": 256, "dtype": "bf16"},
        # the feature fusion's convolution on the 1/8 maps of 8 frames
        {"name": "pointwise_fusion", "kind": "pointwise", "n": 8, "h": 128, "w": 256, "c": 256, "cout": 256, "dtype": "bf16"},
        # the last stage's block tail on two small odd crops
        {"name": "tail_crop", "kind": "tail", "n": 2, "h": 9, "w": 13, "c": 512, "dtype": "fp16"},
        # block tails of the second residual stage, 8 frames
        {"name": "tail_res3", "kind": "tail", "n": 8, "h": 128, "w": 256, "c": 128, "dtype": "bf16"},
        # block tails of the first residual stage, 8 frames: the largest maps of the trunk
        {"name": "tail_res2", "kind": "tail", "n": 8, "h": 256, "w": 512, "c": 64, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """a whole number between low and high, spread over its logarithm"""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["checkpoint", "product", "pointwise", "tail"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "product":
        k, n = _spread(rng, 32, 4096), _spread(rng, 1, 4096)
        m = _spread(rng, 1, min(400000, 2 * 10 ** 11 // (k * n), 2 * 10 ** 8 // max(k, n)))
        return {"kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.5, "act": rng.choice(["none", "relu", "leaky_relu"])}
    n = rng.randint(1, 8)
    case = {"kind": kind, "n": n, "dtype": dtype}
    if kind == "tail":
        c = 8 * _spread(rng, 4, 64)
    else:
        c = _spread(rng, 3, 1024)
    if kind == "checkpoint" and rng.random() < 0.25:
        case["dtype"] = "fp32"
    most = 60 * 10 ** 6 // (n * c)
    if kind == "pointwise":
        c = 8 * max(1, c // 8)
        case["cout"] = _spread(rng, 1, 512)
        most = 60 * 10 ** 6 // (n * max(c, case["cout"]))
    pixels = _spread(rng, 4 if kind == "tail" else 1, max(4, min(most, 32768)))
    h = max(1, int(math.sqrt(pixels / rng.choice([1, 2, 3]))))
    case.update(h=h, w=max(1, pixels // h), c=c)
    return case


def _map(g, case, c, spread=1.0):
    """a channels-last map whose channels have scales of their own, as trained features have"""
    shape = (case["n"], case["h"], case["w"], c)
    x = torch.randn(shape, generator=g, device="cuda")
    x *= torch.exp(spread * torch.randn(c, generator=g, device="cuda"))
    return x.to(DTYPES[case["dtype"]]).permute(0, 3, 1, 2)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}
    if kind == "checkpoint":
        s["x"] = _map(g, case, case["c"])
    elif kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        a = torch.randn(m, k, generator=g, device="cuda")
        a *= torch.exp(torch.randn(k, generator=g, device="cuda"))
        w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        a = a.to(dt)
        if own:
            from mgnet_amd.modeling import ops
            s["a"], s["b"] = ops.q8_pack(a), ops.q8_pack(w, tile=True)
        else:
            s["a"], s["b"] = _pack(a), _pack(w, tile=True)
        s["bias"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
    elif kind == "pointwise":
        s["x"] = _map(g, case, case["c"])
        w = torch.randn(case["cout"], case["c"], 1, 1, generator=g, device="cuda") / math.sqrt(case["c"])
        b = torch.randn(case["cout"], generator=g, device="cuda")
        s["dy"] = _map(g, case, case["cout"], 0.5)
        s["w"], s["b"] = w, b
        if own:
            for k in ("x", "w", "b"):
                s[k].requires_grad_()
    else:
        c = case["c"]
        s["x"] = _map(g, case, c)
        s["shortcut"] = _map(g, case, c, 0.25)
        # a loss's gradient with respect to a channel has a mean of its own
        dy = torch.randn(case["n"], case["h"], case["w"], c, generator=g, device="cuda")
        s["dy"] = (dy + torch.randn(c, generator=g, device="cuda")).to(dt).permute(0, 3, 1, 2)
        s["w"] = 1 + 0.5 * torch.randn(c, generator=g, device="cuda")
        s["b"] = 0.5 * torch.randn(c, generator=g, device="cuda")
        s["mean"], s["var"] = torch.zeros(c, device="cuda"), torch.ones(c, device="cuda")
        if own:
            from mgnet_amd.modeling.layers import InPlaceABNSync
            norm = InPlaceABNSync(c, eps=EPS, momentum=MOMENTUM, activation="identity").cuda()
            with torch.no_grad():
                norm.weight.copy_(s["w"])
                norm.bias.copy_(s["b"])
            s["norm"] = norm
            for k in ("x", "shortcut"):
                s[k].requires_grad_()
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _own(s, kind)
    return {"checkpoint": _plain_checkpoint, "product": _plain_product, "pointwise": _plain_pointwise, "tail": _plain_tail}[kind](s)


def _own(s, kind):
    from mgnet_amd.modeling import ops
    if kind == "checkpoint":
        return ops.q8_pack(s["x"]).unpack()
    if kind == "product":
        return ops.q8_matmul(s["a"], s["b"], bias=s["bias"], act=s["case"]["act"], slope=0.01, out_dtype=DTYPES[s["case"]["dtype"]])
    if kind == "pointwise":
        y = ops.conv1x1_q8(s["x"], s["w"], s["b"])
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    norm = s["norm"]
    y = ops.abn_add_relu_q8(s["x"], norm, s["shortcut"])
    dx, ds, dw, db = torch.autograd.grad(y, (s["x"], s["shortcut"], norm.weight, norm.bias), s["dy"])
    return {"y": y, "dx": dx, "ds": ds, "dw": dw, "db": db}


# ---- plain forms: elementary operations in 32 bits ---------------------------------------------------------------------------------
def _exp2(e):
    """2^(e - 127) of whole numbers 1 <= e <= 254, exactly"""
    return (e.to(torch.int32) << 23).view(torch.float32)


def _pack(x, tile=False):
    """x [M, C] -> codes [M, blocks, 128] (e4m3 numbers, zeros behind the last channel) and biased exponents [M, blocks] (tile: one per
    128 rows, repeated for its rows)"""
    top = 61440.0 if x.dtype == torch.float16 else 1.875 * 2.0 ** 127
    x = x.float()
    m, c = x.shape
    blocks = -(-c // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - c)).view(m, blocks, BLOCK)
    finite = torch.isfinite(x)
    largest = torch.where(finite, x.abs(), 0.0).clamp(max=top).amax(2)
    if tile:
        tiles = -(-m // BLOCK)
        largest = torch.nn.functional.pad(largest, (0, 0, 0, tiles * BLOCK - m)).view(tiles, BLOCK, blocks).amax(1)
        largest = largest.repeat_interleave(BLOCK, 0)[:m]
    e = (((largest.view(torch.int32) + 0x1FFFFF) >> 23) - 8).clamp(min=16)
    v = torch.where(finite, x.clamp(-top, top), math.nan) * _exp2(254 - e).unsqueeze(2)
    return v.to(torch.float8_e4m3fn), e


def _values(packed, c):
    codes, e = packed
    return (codes.float() * _exp2(e).unsqueeze(2)).flatten(1)[:, :c]


def _plain_checkpoint(s):
    x = s["x"]
    n, c, h, w = x.shape
    rows = x.permute(0, 2, 3, 1).reshape(-1, c)
    return _values(_pack(rows), c).to(x.dtype).view(n, h, w, c).permute(0, 3, 1, 2)


def _plain_product(s):
    case = s["case"]
    out = _values(s["a"], case["k"]) @ _values(s["b"], case["k"]).t()
    if s["bias"] is not None:
        out = out + s["bias"]
    if case["act"] != "none":
        out = torch.where(out > 0, out, out * (0.01 if case["act"] == "leaky_relu" else 0.0))
    return out.to(DTYPES[case["dtype"]])


def _plain_pointwise(s):
    x, dy, dt = s["x"], s["dy"], s["x"].dtype
    n, c, h, w = x.shape
    cout = dy.shape[1]
    x8 = _values(_pack(x.permute(0, 2, 3, 1).reshape(-1, c)), c)
    w8 = _values(_pack(s["w"].view(cout, c), tile=True), c)
    rows = dy.permute(0, 2, 3, 1).reshape(-1, cout)
    y = x8 @ w8.t() + s["b"]
    dx = _values(_pack(rows), cout) @ w8
    rows = rows.float()
    dw = rows.t() @ x8
    back = lambda t: t.to(dt).view(n, h, w, -1).permute(0, 3, 1, 2)  # noqa: E731
    return {"y": back(y), "dx": back(dx), "dw": dw.view(cout, c, 1, 1), "db": rows.sum(0)}


def _plain_tail(s):
    x, dt = s["x"], s["x"].dtype
    n, c, h, w = x.shape
    rows = x.permute(0, 2, 3, 1).reshape(-1, c)
    x8 = _values(_pack(rows), c)
    rows = rows.float()
    m = rows.shape[0]
    mean = rows.mean(0)
    var = (rows - mean).square().mean(0)
    rstd = torch.rsqrt(var + EPS)
    gain = s["w"].abs() + EPS
    y = (rows - mean) * (gain * rstd) + s["b"] + s["shortcut"].permute(0, 2, 3, 1).reshape(-1, c).float()
    y = torch.relu(y)
    s["mean"].mul_(1 - MOMENTUM).add_(mean, alpha=MOMENTUM)
    s["var"].mul_(1 - MOMENTUM).add_(var * (m / max(m - 1, 1)), alpha=MOMENTUM)
    dz = torch.where(y > 0, s["dy"].permute(0, 2, 3, 1).reshape(-1, c).float(), 0.0)
    xh = (x8 - mean) * rstd
    db, dg = dz.sum(0), (dz * xh).sum(0)
    dx = gain * rstd * (dz - db / m - xh * (dg / m))
    back = lambda t: t.to(dt).view(n, h, w, c).permute(0, 3, 1, 2)  # noqa: E731
    return {"y": back(y), "dx": back(dx), "ds": back(dz), "dw": dg * s["w"].sign(), "db": db}


# ---- the definition in 64 bits, apart from the plain forms -------------------------------------------------------------------------
def _exact_q8(x, tile=False):
    """the values that the packed form of x [M, C] stands for"""
    top = 1.875 * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = x.double()
    m, c = x.shape
    out = torch.empty_like(x)
    for k in range(0, c, BLOCK):
        v = x[:, k:k + BLOCK].clamp(-top, top)
        largest = v.abs().amax(1, keepdim=True)
        if tile:
            largest = torch.cat([largest[r:r + BLOCK].amax().expand(min(BLOCK, m - r), 1) for r in range(0, m, BLOCK)])
        f, p = torch.frexp(largest)             # largest = f 2^p with 0.5 <= f < 1; 448 = 0.875 * 2^9
        e = torch.where(largest > 0, p - 9 + (f > 0.875), -111).clamp(min=-111).double()
        v = v / torch.exp2(e)
        _, p = torch.frexp(v)
        step = torch.exp2((p - 1).clamp(min=-6).double() - 3)
        out[:, k:k + BLOCK] = torch.round(v / step) * step * torch.exp2(e)
    return out


def _rows64(t):
    return t.permute(0, 2, 3, 1).reshape(-1, t.shape[1])


def exact(case, seed):
    # (the inputs alone: nothing of the framework is called for them)
    kind = case["kind"]
    if kind == "product":
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        m, n, k = case["m"], case["n"], case["k"]
        a = torch.randn(m, k, generator=g, device="cuda")
        a *= torch.exp(torch.randn(k, generator=g, device="cuda"))
        w = torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)
        bias = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        out = _exact_q8(a.to(DTYPES[case["dtype"]])) @ _exact_q8(w, tile=True).t()
        if bias is not None:
            out = out + bias.double()
        if case["act"] != "none":
            out = torch.where(out > 0, out, out * (0.01 if case["act"] == "leaky_relu" else 0.0))
        return out
    s = prepare(case, seed)
    x = _rows64(s["x"].detach())
    n, c, h, w = s["x"].shape
    back = lambda t: t.view(n, h, w, -1).permute(0, 3, 1, 2)  # noqa: E731
    x8 = _exact_q8(x)
    if kind == "checkpoint":
        return back(x8)
    dy = _rows64(s["dy"])
    weight, bias = s["w"].detach().double(), s["b"].detach().double()
    if kind == "pointwise":
        w8 = _exact_q8(s["w"].detach().view(-1, c), tile=True)
        return {"y": back(x8 @ w8.t() + bias), "dx": back(_exact_q8(dy) @ w8), "dw": (dy.double().t() @ x8).view(-1, c, 1, 1), "db": dy.double().sum(0)}
    x, dy = x.double(), dy.double()
    mean, var = x.mean(0), x.var(0, unbiased=False)
    rstd, gain = (var + EPS) ** -0.5, weight.abs() + EPS
    y = gain * (x - mean) * rstd + bias + _rows64(s["shortcut"].detach()).double()
    dz = dy * (y > 0)
    xh = (x8 - mean) * rstd
    g1, g2 = dz.mean(0), (dz * xh).mean(0)
    return {"y": back(y.clamp(min=0)), "dx": back(gain * rstd * (dz - g1 - xh * g2)), "ds": back(dz), "dw": (dz * xh).sum(0) * weight.sign(), "db": dz.sum(0)}


def work(case):
    kind = case["kind"]
    size = 4 if case["dtype"] == "fp32" else 2
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = -(-k // BLOCK)
        return {"bytes": (m + n) * (k + blocks) + size * m * n + 4 * n * bool(case["bias"]), "flops": 2 * m * n * k}
    m, c = case["n"] * case["h"] * case["w"], case["c"]
    packed = m * (c + -(-c // BLOCK))
    if kind == "checkpoint":       # read x; write, and later read, its packed form; write x^
        return {"bytes": 2 * size * m * c + 2 * packed, "flops": 4 * m * c}
    if kind == "pointwise":        # forward: read x, write y and the packed x; backward: read dy and the packed x, write dx
        n = case["cout"]
        return {"bytes": 2 * size * m * (c + n) + 2 * packed + 8 * n * c, "flops": 6 * m * n * c}
    # tail forward: x for the statistics and again for the result, shortcut, y, packed x, mask; backward: mask, dy, packed x, the sums, dz, dx
    return {"bytes": size * m * c * 6 + 2 * packed + m * c // 4, "flops": 30 * m * c}
