"""Group norm with an activation on channels-last tensors, forward and backward (csrc/group_norm.hip, include/m355.h
m355_group_norm_*) -- the batch-independent counterpart of gan_ops' fused batch norm, for training with few samples per GPU.

    y = act((x - mean_g) / sqrt(var_g + eps) * weight + bias) [+ res]

`group_norm_act` is the function, `GroupNorm2d` the conditional form behind `norm_g='group'` (gan.ConditionalBatchNorm2d) and
`GroupNormAct2d` the layer with its own affine (norm_d='group', ReconstructionNetwork(norm='group')).  No CPU or torch fallback: CPU
tensors raise."""
import torch
import torch.nn as nn

from . import _lib
from ._lib import launch, lib, ptr, stream

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # m355_dtype
ACTS = {"lrelu": 0, "silu": 1}


class _on:
    """launches go to the current stream of the tensor's device, whichever device is current"""

    def __new__(cls, t):
        return torch.cuda.device(t.device) if t.device.index != torch.cuda.current_device() else _NULL


class _Null:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_NULL = _Null()


def _ws(n, hw, c, groups, dt, backward, dev):
    nbytes = lib().m355_group_norm_ws_bytes(n, hw, c, groups, dt, backward)
    return torch.empty((nbytes,), dtype=torch.uint8, device=dev)


def _sizes(x):
    n, c = x.shape[0], x.shape[-1]
    return n, (x.numel() // (n * c) if x.numel() else 0), c


def _affine(t):
    """[C] or [N,C] fp32 with unit channel stride -> the tensor itself (a view of a batched GEMM's output is read in place)"""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _forward(x, weight, bias, res, groups, eps, act, slope, w_off, out_slope):
    n, hw, c = _sizes(x)
    dt = _DTYPES[x.dtype]
    y = torch.empty_like(x)
    stat = torch.empty((2, n, groups), dtype=torch.float32, device=x.device)
    if x.numel() == 0:
        return y, stat, weight, bias
    weight = None if weight is None else _affine(weight)
    bias = None if bias is None else _affine(bias)
    one = weight if weight is not None else bias
    stride = 0
    if one is not None and one.dim() == 2:
        stride = one.stride(0)
        if weight is not None and bias is not None and bias.stride(0) != stride:
            weight, bias = weight.contiguous(), bias.contiguous()
            stride = c
    res_w = 0
    if res is not None and res.shape != x.shape:
        res_w = x.shape[2]
    with _on(x):
        launch("group_norm_fwd", ptr(x), ptr(weight), ptr(bias), stride, w_off, ptr(res), res_w, ptr(y), stat.data_ptr(),
               stat.data_ptr() + 4 * n * groups, ptr(_ws(n, hw, c, groups, dt, 0, x.device)), n, hw, c, groups, eps, act, slope,
               out_slope, dt, stream())
    return y, stat, weight, bias


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, res, groups, eps, act, slope, w_off, out_slope):
        y, stat, w, b = _forward(x, weight, bias, res, groups, eps, act, slope, w_off, out_slope)
        ctx.save_for_backward(x, w, b, stat)
        ctx.cfg = (groups, act, slope, w_off, None if res is None else tuple(res.shape))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stat = ctx.saved_tensors
        groups, act, slope, w_off, res_shape = ctx.cfg
        n, hw, c = _sizes(x)
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        if dy.dtype != x.dtype:
            dy = dy.to(x.dtype)
        dy = dy.contiguous()
        dev = x.device
        dx = torch.empty_like(x) if need_x else None
        dw = torch.empty(weight.shape, dtype=torch.float32, device=dev) if need_w else None
        db = torch.empty(bias.shape, dtype=torch.float32, device=dev) if need_b else None
        half = res_shape is not None and res_shape != tuple(x.shape)
        dres = None
        if need_r:
            dres = torch.empty(res_shape, dtype=x.dtype, device=dev) if half else dy
        if x.numel() == 0:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        elif need_x or need_w or need_b or (half and need_r):
            one = weight if weight is not None else bias
            per_sample = one is not None and one.dim() == 2
            with _on(x):
                launch("group_norm_bwd", ptr(dy), ptr(x), ptr(weight), ptr(bias), one.stride(0) if per_sample else 0, w_off,
                       stat.data_ptr(), stat.data_ptr() + 4 * n * groups, ptr(dx), ptr(dw), ptr(db), int(per_sample),
                       ptr(dres) if half else None, x.shape[2] if half else 0, ptr(_ws(n, hw, c, groups, _DTYPES[x.dtype], 1, dev)),
                       n, hw, c, groups, act, slope, _DTYPES[x.dtype], stream())
        return dx, dw, db, dres, None, None, None, None, None, None


def _check_affine(t, name, n, c, x):
    if not torch.is_tensor(t) or not t.is_cuda or t.device != x.device:
        raise _lib.M355Error(f"group_norm_act: {name} must be a tensor on {x.device}")
    if tuple(t.shape) not in ((c,), (n, c)):
        raise ValueError(f"group_norm_act: {name} must be [{c}] or [{n}, {c}], got {list(t.shape)}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"group_norm_act: {name} must be float32, float16 or bfloat16, got {t.dtype}")
    return t if t.dtype == torch.float32 else t.float()


def _apply(x, num_groups, weight, bias, eps, act, slope, res, w_off, out_slope):
    if not torch.is_tensor(x) or not x.is_cuda:
        raise _lib.M355Error("group_norm_act: x must be a CUDA(HIP) tensor; there is no CPU implementation")
    if x.dtype not in _DTYPES:
        raise TypeError(f"group_norm_act: x must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"group_norm_act: x must be [N, ..., C], got {list(x.shape)}")
    n, c, groups = x.shape[0], x.shape[-1], int(num_groups)
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"group_norm_act: {c} channels in {num_groups} groups")
    if not float(eps) >= 0.0:
        raise ValueError(f"group_norm_act: eps={eps!r}")
    if act not in ACTS:
        raise ValueError(f"group_norm_act: act={act!r} (one of {sorted(ACTS)})")
    if weight is not None:
        weight = _check_affine(weight, "weight", n, c, x)
    if bias is not None:
        bias = _check_affine(bias, "bias", n, c, x)
    if weight is not None and bias is not None and weight.shape != bias.shape:
        raise ValueError(f"group_norm_act: weight {list(weight.shape)} and bias {list(bias.shape)} must have one shape")
    if res is not None:
        if not torch.is_tensor(res) or res.device != x.device or res.dtype != x.dtype:
            raise TypeError(f"group_norm_act: res must be {x.dtype} on {x.device}")
        if res.shape != x.shape and not (x.dim() == 4 and x.shape[1] % 2 == 0 and x.shape[2] % 2 == 0
                                         and tuple(res.shape) == (n, x.shape[1] // 2, x.shape[2] // 2, c)):
            raise ValueError(f"group_norm_act: res must have x's shape {list(x.shape)} or half its height and width, got {list(res.shape)}")
        res = res.contiguous()
    x = x.contiguous()
    args = (x, weight, bias, res, groups, float(eps), ACTS[act], float(slope), float(w_off), float(out_slope))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4]):
        return _GroupNormAct.apply(*args)
    return _forward(*args)[0]


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="lrelu", slope=1.0, res=None):
    """Group norm of a channels-last tensor with the activation behind it, one fused operator with its gradient.

    x [N, ..., C] float32 / float16 / bfloat16 (an NCHW tensor in torch's channels_last format is `x.permute(0, 2, 3, 1)`; other
    strides are copied); num_groups divides C; every (sample, group) is normalised by its own mean and biased variance, held in
    float32.  weight, bias: [C], or [N, C] (conditional norms: one affine per sample; rows of a larger matrix are read in place), or None
    (1 / 0).  act 'lrelu': LeakyReLU(slope) -- slope 1.0 is no activation, 0.0 is ReLU, the derivative at 0 is 1 -- or 'silu'.
    res: added after the activation; x's shape, or half of x's height and width, read through the nearest x2 upsample.
    Returns y of x's shape and type, rounded once.  Gradients reach x, weight, bias and res; the results do not depend on the run."""
    return _apply(x, num_groups, weight, bias, eps, act, slope, res, 0.0, 1.0)


def _groups_for(ch, groups):
    if groups < 1 or ch % groups:
        raise ValueError(f"group norm: {ch} channels in {groups} groups")
    return groups


class GroupNorm2d(nn.Module):
    """Parameter-free group norm with gan_ops.BatchNorm2d's calling convention (norm_g='group'): LeakyReLU(GN(x) * (1 + gamma) + beta)
    [+ res] on NHWC activations, gamma / beta [N,C] per sample; training and evaluation are the same function."""

    def __init__(self, ch, num_groups=32, eps=1e-5):
        super().__init__()
        self.num_features, self.num_groups, self.eps = ch, _groups_for(ch, num_groups), eps

    def forward(self, x, gamma, beta, slope=1.0, res=None, out_slope=1.0, part=None):
        """out_slope != 1: a second LeakyReLU on the result whose BACKWARD IS LEFT TO THE CONSUMER (gan_ops.head_conv(in_slope=...));
        part (partial sums over the whole batch) is not used: these statistics are per sample"""
        return _apply(x, self.num_groups, gamma, beta, self.eps, "lrelu", slope, res, 1.0, out_slope)

    def extra_repr(self):
        return f"{self.num_features}, num_groups={self.num_groups}, eps={self.eps}"


class GroupNormAct2d(nn.Module):
    """nn.GroupNorm(num_groups, ch) (parameters `weight`, `bias`) + LeakyReLU(slope) [+ residual] on NHWC activations, fused"""

    def __init__(self, ch, num_groups=32, eps=1e-5):
        super().__init__()
        self.num_features, self.num_groups, self.eps = ch, _groups_for(ch, num_groups), eps
        self.weight = nn.Parameter(torch.ones(ch))
        self.bias = nn.Parameter(torch.zeros(ch))

    def forward(self, x, slope=0.0, res=None, out_slope=1.0):
        return _apply(x, self.num_groups, self.weight, self.bias, self.eps, "lrelu", slope, res, 0.0, out_slope)

    def extra_repr(self):
        return f"{self.num_features}, num_groups={self.num_groups}, eps={self.eps}"
