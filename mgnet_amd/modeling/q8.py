"""8-bit activations and weights: e4m3 codes with one power-of-two scale per block of 128 (csrc/q8.hip).  The entry points are those of
`ops`: q8_pack / Q8Map, q8_matmul, conv1x1_q8, abn_add_relu_q8.  [HIP] only: a CPU tensor raises."""
import torch
import torch.distributed as dist
import torch.nn.functional as F

from .. import _C
from .ops import PaddedMap, _allreduce_sums, _dist_active, _pstats, _train_coef

__all__ = ["Q8Map", "q8_pack", "q8_matmul", "conv1x1_q8", "conv1x1_q8_supported", "conv1x1_q8_layer", "abn_add_relu_q8", "abn_add_relu_q8_supported"]

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CL = torch.channels_last


class Q8Map:
    """An [M, C] matrix, or the channels-last map [N, C, H, W] with M = N*H*W pixels, in 8 bits.  `buf` holds `codes`, uint8 [M, C rounded up
    to 16], and `scales`, uint8 [ceil(C / 128), M rounded up to 16] (exponent + 127 of block k of row r at [k, r]).  A block is 128
    neighbouring channels of a row; of a weight matrix packed with tile=True all 128 rows of a tile share a scale.  `dtype` is the source's."""

    __slots__ = ("buf", "shape", "dtype", "rows", "channels")

    def __init__(self, buf, shape, dtype):
        self.buf, self.shape, self.dtype, self.channels = buf, tuple(shape), dtype, shape[1]
        self.rows = shape[0] if len(shape) == 2 else shape[0] * shape[2] * shape[3]

    @property
    def device(self):
        return self.buf.device

    @property
    def codes(self):
        return self.buf[:_C.q8_code_bytes(self.rows, self.channels)].view(self.rows, -1) if self.rows else self.buf.view(0, (self.channels + 15) // 16 * 16)

    @property
    def scales(self):
        return self.buf[_C.q8_code_bytes(self.rows, self.channels):].view((self.channels + 127) // 128, -1)

    def nbytes(self):
        return self.buf.numel()

    def unpack(self, dtype=None):
        """the values, in the source's type (exact) or `dtype` (rounded once); maps come back channels-last"""
        dtype = self.dtype if dtype is None else dtype
        if dtype not in _FLOATS:
            raise ValueError(f"Q8Map.unpack: float32, bfloat16 or float16, got {dtype}")
        if _elsewhere(self.buf):
            with torch.cuda.device(self.buf.device):
                return self.unpack(dtype)
        if len(self.shape) == 2:
            out = torch.empty(self.shape, dtype=dtype, device=self.buf.device)
        else:
            out = torch.empty(self.shape, dtype=dtype, device=self.buf.device, memory_format=_CL)
        return _C.q8_unpack(self.buf, self.rows, self.channels, out)


def _elsewhere(t):
    """the tensor's device is not the current one: launches go to the tensor's own, so the caller enters it first"""
    return t.device.index != torch.cuda.current_device()


def _check_source(x, what):
    if not isinstance(x, torch.Tensor) or x.dim() not in (2, 4):
        raise ValueError(f"{what}: an [M, C] matrix or an [N, C, H, W] map, got {tuple(x.shape) if isinstance(x, torch.Tensor) else type(x).__name__}")
    if not x.is_cuda:
        raise RuntimeError(f"{what}: the 8-bit operators have HIP kernels only (no CPU form), got a {x.device} tensor")
    if x.dtype not in _FLOATS:
        raise ValueError(f"{what}: float32, bfloat16 or float16, got {x.dtype}")
    if x.shape[1] < 1:
        raise ValueError(f"{what}: no channels in {tuple(x.shape)}")


def _geometry(x):
    """x (or a copy with unit channel stride) and its (M, C, sn, sh, sw, H, W) as mgn_q8_pack takes them"""
    st = x.stride()
    if x.dim() == 2:
        M, C = x.shape
        if st[1] != 1 and C > 1:
            x = x.contiguous()
            return x, (M, C, C, 0, 0, 1, 1)
        return x, (M, C, st[0], 0, 0, 1, 1)
    N, C, H, W = x.shape
    if st[1] != 1 and C > 1:
        x = x.permute(0, 2, 3, 1).contiguous()
        return x, (N * H * W, C, C, 0, 0, 1, 1)
    return x, (N * H * W, C, st[0], st[2], st[3], H or 1, W or 1)


def q8_pack(x, tile=False):
    """x [M, C] or [N, C, H, W], float32 / bfloat16 / float16, any strides -> Q8Map.  value = code * 2^e with the smallest e >= -111 that
    keeps the block's largest finite magnitude within 448 * 2^e: relative error at most 2^-4 down to 2^-6 * 2^e, absolute 2^-10 * 2^e below;
    NaN and infinities become NaN.  tile: a weight matrix [N, K], one scale per 128 x 128 tile.  Not differentiable (conv1x1_q8 is)."""
    _check_source(x, "q8_pack")
    if tile and (x.dim() != 2 or 0 in x.shape):
        raise ValueError(f"q8_pack: tile scales are for a weight matrix [N, K], got {tuple(x.shape)}")
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return q8_pack(x, tile)
    if tile:
        return Q8Map(_C.q8_pack_weight(x), x.shape, x.dtype)
    rows, geometry = _geometry(x)
    return Q8Map(_C.q8_pack(rows, *geometry), x.shape, x.dtype)


_ACT = {"none": 0, "relu": 1, "leaky_relu": 2}


def q8_matmul(a, b, bias=None, act="none", slope=0.01, out_dtype=None):
    """act(a b^T + bias) of two packed matrices a [M, K] (or a map [N, K, H, W]: the result is the map [N, n, H, W]) and b [n, K]; products
    of codes scaled in the matrix cores, one rounding to out_dtype (default: a's source type).  The matrix cores cut the products of 8
    neighbouring k to 2^-13 of the largest one's binade before they join the fp32 sum: 1.3e-5 of a result, which a float32 one shows.  act: none | relu |
    leaky_relu (0 <= slope <= 1).  No gradient (conv1x1_q8 has one)."""
    if not (isinstance(a, Q8Map) and isinstance(b, Q8Map)):
        raise ValueError("q8_matmul: two Q8Map operands (ops.q8_pack)")
    if len(b.shape) != 2 or a.channels != b.channels:
        raise ValueError(f"q8_matmul: a [M, K] and b [n, K] with one K, got {a.shape} and {b.shape}")
    dev = a.buf.device
    if dev != b.buf.device or (bias is not None and bias.device != dev):
        raise ValueError("q8_matmul: operands on different devices")
    out_dtype = a.dtype if out_dtype is None else out_dtype
    if act not in _ACT or out_dtype not in _FLOATS or not 0 <= slope <= 1:
        raise ValueError(f"q8_matmul: act one of {sorted(_ACT)}, 0 <= slope <= 1, a float32 / bfloat16 / float16 result; got {act}, {slope}, {out_dtype}")
    n, M = b.rows, a.rows
    if n < 1:
        raise ValueError("q8_matmul: b has no rows")
    if _elsewhere(a.buf):
        with torch.cuda.device(dev):
            return q8_matmul(a, b, bias, act, slope, out_dtype)
    if bias is not None:
        if tuple(bias.shape) != (n,):
            raise ValueError(f"q8_matmul: bias [{n}], got {tuple(bias.shape)}")
        bias = _f32(bias)
    out = torch.empty((M, n), dtype=out_dtype, device=dev)
    _C.q8_matmul(a.buf, M, b.buf, n, a.channels, bias, _ACT[act], float(slope), out)
    if len(a.shape) == 2:
        return out
    N, _, H, W = a.shape
    return out.view(N, H, W, n).permute(0, 3, 1, 2)


def _f32(t):
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.detach().float().contiguous()


def _rows16(t, dtype):
    """a gradient or operand as 16-bit channels-last rows on a 16-byte boundary"""
    if t.dtype != dtype:
        t = t.to(dtype)
    if not t.is_contiguous(memory_format=_CL):
        t = t.contiguous(memory_format=_CL)
    return t.clone(memory_format=_CL) if t.data_ptr() % 16 else t


class _Conv1x1Q8Fn(torch.autograd.Function):
    """[HIP] csrc/q8.hip.  What waits for the backward pass is the packed input (1 byte a value instead of 2) and the packed transpose of
    the weights, in one buffer; the data gradient is the 8-bit product of the packed dy with it, the weight gradient multiplies dy in 16
    bits with the exact 16-bit value of the codes."""

    @staticmethod
    def forward(ctx, x, weight, bias, relu, grad):
        # grad: torch.is_grad_enabled() at the call (needs_input_grad goes by the inputs alone, and in here gradients are off)
        N, C, H, W = x.shape
        Cout = weight.shape[0]
        y = torch.empty((N, Cout, H, W), dtype=x.dtype, device=x.device, memory_format=_CL)
        rows, geometry = _geometry(x)
        w = weight.view(Cout, C) if weight.dtype in (torch.float32, x.dtype) and weight.is_contiguous() else weight.detach().float().reshape(Cout, C)
        need = [grad and n for n in ctx.needs_input_grad]
        buf, kept = _C.q8_conv1x1_fwd(rows, *geometry, w, Cout, None if bias is None else _f32(bias), int(relu), y, int(need[1] or need[2]))
        if need[0] or need[1] or need[2]:
            if buf.numel() - kept > N * H * W * C:      # (x was packed in a pass of its own, for this call alone: its codes do not wait)
                buf = buf[:kept].clone()
            ctx.save_for_backward(buf, y if relu else None)
            ctx.cfg = (x.shape, x.dtype, weight.dtype, weight.shape, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        buf, y = ctx.saved_tensors
        xshape, dtype, wdtype, wshape, bdtype = ctx.cfg
        C, Cout, dev = wshape[1], wshape[0], dy.device
        M = xshape[0] * xshape[2] * xshape[3]
        want_dx, want_dw, want_db = ctx.needs_input_grad[:3]
        want_db = want_db and bdtype is not None
        dx = torch.empty(xshape, dtype=dtype, device=dev, memory_format=_CL) if want_dx else None
        if M == 0:
            return dx, torch.zeros(wshape, dtype=wdtype, device=dev) if want_dw else None, torch.zeros(Cout, dtype=bdtype, device=dev) if want_db else None, None, None
        dy = _rows16(dy, dtype)
        if y is not None:
            # (a select either way: what is masked may be infinite)
            dy = _C.relu_mask_bwd(dy, y) if _C.elt_supported(y) and _C.elt_supported(dy) else _rows16(dy.masked_fill(~(y > 0), 0.0), dtype)
        dw = torch.empty((Cout, C, 1, 1), dtype=torch.float32, device=dev) if want_dw or want_db else None
        db = torch.empty(Cout, dtype=torch.float32, device=dev) if want_db else None
        _C.q8_conv1x1_bwd(dy, M, C, Cout, buf, dx, dw, db)
        if want_db and bdtype != torch.float32:
            db = db.to(bdtype)
        return dx, (dw if wdtype == torch.float32 else dw.to(wdtype)) if want_dw else None, db, None, None


def conv1x1_q8(x, weight, bias=None, relu=False):
    """A 1x1 convolution (stride 1) trained in 8 bits: y = q(x) q(W)^T + bias [-> ReLU], dx = q(dy) q(W), dW = dy^T q(x), db = sum dy, with
    q(.) the block format of q8_pack (x and dy per 128 channels of a pixel, W per 128 x 128 tile), sums as in
    q8_matmul (dW and db: fp32).  Of the input only its packed form is kept for the backward pass, and not that where no weight wants a gradient.
    x [N, C, H, W] bfloat16 / float16 (any strides; the result is channels-last), weight [Cout, C, 1, 1], bias [Cout] or None."""
    _check_source(x, "conv1x1_q8")
    C = x.shape[1]
    if x.dim() != 4 or x.dtype == torch.float32:
        raise ValueError(f"conv1x1_q8: a bfloat16 or float16 map [N, C, H, W], got {x.dtype} {tuple(x.shape)}")
    if weight.dim() != 4 or tuple(weight.shape[1:]) != (C, 1, 1) or not 1 <= weight.shape[0] <= 65536 or C > 65536 or weight.dtype not in _FLOATS:
        raise ValueError(f"conv1x1_q8: weights [Cout, {C}, 1, 1] with at most 65536 channels, got {weight.dtype} {tuple(weight.shape)}")
    if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.device != x.device):
        raise ValueError(f"conv1x1_q8: bias [{weight.shape[0]}] on {x.device}, got {tuple(bias.shape)} on {bias.device}")
    if weight.device != x.device:
        raise ValueError("conv1x1_q8: operands on different devices")
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return _Conv1x1Q8Fn.apply(x, weight, bias, relu, torch.is_grad_enabled())
    return _Conv1x1Q8Fn.apply(x, weight, bias, relu, torch.is_grad_enabled())


def conv1x1_q8_supported(x, conv):
    """a training call of an nn.Conv2d that conv1x1_q8 covers; vectors (1 x 1 maps) keep their 16 bits: nothing is saved there"""
    return (x.is_cuda and x.dtype in _C.H16 and x.dim() == 4 and conv.training and torch.is_grad_enabled() and conv.kernel_size == (1, 1)
            and conv.stride == (1, 1) and conv.padding == (0, 0) and conv.groups == 1 and conv.in_channels == x.shape[1]
            and x.shape[2] * x.shape[3] > 1 and x.shape[0] > 0)


def conv1x1_q8_layer(x, weight, bias=None, relu=False, keep_pad=False):
    """conv1x1_q8 behind ops.conv2d's interface: with keep_pad, output channels that are not a multiple of 32 come as the 32-padded PaddedMap"""
    Cout = weight.shape[0]
    pad = -Cout % 32
    if not (keep_pad and pad):
        return conv1x1_q8(x, weight, bias, relu)
    return PaddedMap(conv1x1_q8(x, F.pad(weight, (0, 0, 0, 0, 0, 0, 0, pad)), None if bias is None else F.pad(bias, (0, pad)), relu), Cout)


class _AbnAddReluQ8Fn(torch.autograd.Function):
    """[HIP] csrc/q8.hip: the residual block's tail relu(norm(x) + shortcut) as ops._AbnAddReluFn, with x kept for the backward pass in 8 bits
    (the norm's x_hat is recomputed from there) and the ReLU mask in one bit a value; y is not kept."""

    @staticmethod
    def forward(ctx, x, shortcut, weight, bias, running_mean, running_var, training, momentum, eps, group, pstats, grad):
        N, C, H, W = x.shape
        M = N * H * W
        x, shortcut = _rows16(x, x.dtype), _rows16(shortcut, x.dtype)
        w32, b32 = _f32(weight), _f32(bias)
        need = ctx.needs_input_grad
        buf = _C.q8_tail_buffer(M, C, x.device) if training and grad and (need[0] or need[1] or need[2] or need[3]) else None   # (grad: as above)
        y = torch.empty((N, C, H, W), dtype=x.dtype, device=x.device, memory_format=_CL)
        world = dist.get_world_size(group) if _dist_active(group) else 1
        if training and world == 1 and pstats is None:
            coef = torch.empty((4, C), dtype=torch.float32, device=x.device)
            _C.q8_tail_train_fwd(x, shortcut, M, C, w32, b32, eps, momentum, running_mean, running_var, coef, y, buf)
        else:
            if training:
                coef = _train_coef(x, M, C, w32, b32, eps, momentum, running_mean, running_var, world, group, pstats or _C.q8_tail_stats(x, M, C))
            else:
                coef = _C.iabn_eval_coeffs(w32, b32, running_mean, running_var, eps)
            _C.q8_tail_fwd(x, shortcut, coef, M, C, y, buf)
        ctx.save_for_backward(buf, w32 if w32 is weight else w32.detach(), coef)
        ctx.cfg = (x.shape, x.dtype, eps, group, world, weight.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        buf, w32, coef = ctx.saved_tensors
        shape, dtype, eps, group, world, wdtype = ctx.cfg
        if buf is None:
            raise NotImplementedError("backward through eval-mode InPlaceABNSync is not on the training path")
        C, M = shape[1], shape[0] * shape[2] * shape[3]
        g = _rows16(g, dtype)
        dz = torch.empty(shape, dtype=dtype, device=g.device, memory_format=_CL)
        dx = torch.empty(shape, dtype=dtype, device=g.device, memory_format=_CL) if ctx.needs_input_grad[0] else None
        if world == 1:
            out = _C.q8_tail_train_bwd(buf, g, coef, w32, eps, M, C, dz, dx)
        else:
            out = _C.q8_tail_bwd_reduce(buf, g, coef, w32, M, C, dz)
            sums = _allreduce_sums(out[:2].contiguous(), group)
            if dx is not None:
                _C.q8_tail_bwd_apply(buf, dz, coef, w32, sums, float(M) * world, eps, M, C, dx)
        dw, db = out[2], out[3]
        if wdtype != torch.float32:
            dw, db = dw.to(wdtype), db.to(wdtype)
        return dx, dz, dw, db, None, None, None, None, None, None, None, None


def abn_add_relu_q8(x, norm, shortcut):
    """`relu_(norm(x) + shortcut)` for an identity-activation InPlaceABNSync (ops.abn_add_relu) that keeps x in 8 bits for the backward pass:
    forward values are those of the 16-bit x (rounded once), the backward pass uses x_hat of the packed x.  x, shortcut [N, C, H, W]
    bfloat16 or float16, C % 8 == 0; the batch statistics are exchanged over norm.group as in every norm."""
    _check_source(x, "abn_add_relu_q8")
    C = x.shape[1]
    if x.dim() != 4 or x.dtype == torch.float32 or C % 8 or C > 8192 or x.numel() == 0:
        raise ValueError(f"abn_add_relu_q8: a non-empty bfloat16 or float16 map [N, C, H, W] with C % 8 == 0, got {x.dtype} {tuple(x.shape)}")
    if shortcut.shape != x.shape or shortcut.dtype != x.dtype or shortcut.device != x.device:
        raise ValueError("abn_add_relu_q8: the shortcut must match x in shape, type and device")
    w = norm.weight
    if norm.activation != "identity" or norm.num_features != C or w.device != x.device or norm.running_mean.dtype != torch.float32:
        raise ValueError(f"abn_add_relu_q8: an identity-activation norm of {C} channels on {x.device} with float32 statistics, got {norm.activation}, "
                         f"{norm.num_features}, {w.device}, {norm.running_mean.dtype}")
    args = (x, shortcut, w, norm.bias, norm.running_mean, norm.running_var, norm.training, norm.momentum, norm.eps, norm.group, _pstats(x), torch.is_grad_enabled())
    if _elsewhere(x):
        with torch.cuda.device(x.device):
            return _AbnAddReluQ8Fn.apply(*args)
    return _AbnAddReluQ8Fn.apply(*args)


def abn_add_relu_q8_supported(x, norm, shortcut):
    """a training call of a block tail that abn_add_relu_q8 covers"""
    return (x.is_cuda and x.dtype in _C.H16 and norm.training and torch.is_grad_enabled() and norm.activation == "identity" and x.shape[1] % 8 == 0
            and x.shape[1] <= 8192 and x.numel() > 0 and x.shape == shortcut.shape and x.dtype == shortcut.dtype
            and norm.running_mean.dtype == torch.float32)
