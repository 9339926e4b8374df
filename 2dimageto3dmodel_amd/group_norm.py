"""Group norm with an activation on channels-last tensors, forward and backward (csrc/group_norm.hip, include/m355.h
m355_group_norm_*) -- the batch-independent counterpart of gan_ops' fused batch norm, for training with few samples per GPU.

    y = act((x - mean_g) / sqrt(var_g + eps) * weight + bias) [+ res]

`group_norm_act` is the function, `GroupNorm2d` the conditional form behind `norm_g='group'` (gan.ConditionalBatchNorm2d) and
`GroupNormAct2d` the layer with its own affine (norm_d='group', ReconstructionNetwork(norm='group')).  No CPU or torch fallback: CPU
tensors raise."""
import ctypes
from math import gcd
from operator import index

import torch
import torch.autograd.forward_ad as fwad
import torch.nn as nn

from . import _lib
from ._lib import launch, lib, stream

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # m355_dtype
_F32 = torch.float32
ACTS = {"lrelu": 0, "silu": 1}
_get_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_is_tracing = getattr(torch._C, "_is_tracing", None) or torch.jit.is_tracing


class _Here:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def on_device(index):
    """launches go to the current stream of the tensors' device, whichever device is current"""
    return _HERE if index == _get_device() else torch.cuda.device(index)


class _Plan:
    """what a call's shapes, types, strides and constants decide: the checked descriptor and the workspace sizes"""
    __slots__ = ("desc", "at", "index", "stat", "ws", "ws_bwd", "half", "res_shape", "floats", "cast", "empty", "dtype", "shape", "device",
                 "aff_shape", "aff_strides", "grid")


_PLANS = {}   # by shapes, types, strides, devices and constants -- never by what the tensors hold or where they lie


def _reset():
    _PLANS.clear()


_lib._RESET_HOOKS.append(_reset)


def _check_affine(t, name, n, c, x):
    if not torch.is_tensor(t) or not t.is_cuda or t.device != x.device:
        raise _lib.M355Error(f"group_norm_act: {name} must be a tensor on {x.device}")
    if tuple(t.shape) not in ((c,), (n, c)):
        raise ValueError(f"group_norm_act: {name} must be [{c}] or [{n}, {c}], got {list(t.shape)}")
    if t.dtype not in _DTYPES:
        raise TypeError(f"group_norm_act: {name} must be float32, float16 or bfloat16, got {t.dtype}")


def _rows(aff, c):
    """floats between the rows of the affine's tensors as they lie in memory (0: one row for all samples), None: their values are not rows of
    unit stride, as far apart in one as in the other"""
    row = aff[0].stride(0) if aff and aff[0].dim() == 2 else 0
    for t in aff:
        if (t.stride(-1) != 1 and c != 1) or (t.dim() == 2 and t.stride(0) != row):
            return None
    return row


def _grid(c, groups, size):
    """bytes that the addresses of x, res and dy must be multiples of.  The kernels' vectors are at most 16 bytes, and what the channel count and
    every address are multiples of; a workgroup holds a group of at most 256 vectors (segments of them where vectors straddle groups).  0: no
    address is refused"""
    v = 1
    while v < 16 // size and c % (2 * v) == 0 and (c // groups) // gcd(v, c // groups) > 256:
        v *= 2
    return v * size if v > 1 else 0


def _on_grid(t, grid):
    """t, copied to an allocation of its own if a group of it were too wide from where it lies"""
    return t.clone() if t.data_ptr() % grid else t


def _make_plan(x, num_groups, weight, bias, eps, act, slope, res, w_off, out_slope):
    if not torch.is_tensor(x) or not x.is_cuda:
        raise _lib.M355Error("group_norm_act: x must be a CUDA(HIP) tensor; there is no CPU implementation")
    if x.dtype not in _DTYPES:
        raise TypeError(f"group_norm_act: x must be float32, float16 or bfloat16, got {x.dtype}")
    if x.dim() < 2:
        raise ValueError(f"group_norm_act: x must be [N, ..., C], got {list(x.shape)}")
    n, c, groups = x.shape[0], x.shape[-1], index(num_groups)
    if groups < 1 or c < 1 or c % groups:
        raise ValueError(f"group_norm_act: {c} channels in {num_groups} groups")
    if not float(eps) >= 0.0:
        raise ValueError(f"group_norm_act: eps={eps!r}")
    if act not in ACTS:
        raise ValueError(f"group_norm_act: act={act!r} (one of {sorted(ACTS)})")
    p = _Plan()
    p.cast = False
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check_affine(t, name, n, c, x)
            p.cast = p.cast or t.dtype != torch.float32
    one = weight if weight is not None else bias
    if weight is not None and bias is not None and weight.shape != bias.shape:
        raise ValueError(f"group_norm_act: weight {list(weight.shape)} and bias {list(bias.shape)} must have one shape")
    # rows of unit channel stride, as far apart in weight as in bias, are read in place (views of a batched GEMM's output)
    per_sample = one is not None and one.dim() == 2
    aff = [t for t in (weight, bias) if t is not None]
    row = None if p.cast else _rows(aff, c)
    p.floats, p.aff_shape = row is None, None if one is None else one.shape
    if row is None:
        row = c if per_sample else 0
    p.aff_strides = (row, 1) if per_sample else (1,)
    half = False
    if res is not None:
        if not torch.is_tensor(res) or res.device != x.device or res.dtype != x.dtype:
            raise TypeError(f"group_norm_act: res must be {x.dtype} on {x.device}")
        half = res.shape != x.shape
        if half and not (x.dim() == 4 and x.shape[1] % 2 == 0 and x.shape[2] % 2 == 0
                         and tuple(res.shape) == (n, x.shape[1] // 2, x.shape[2] // 2, c)):
            raise ValueError(f"group_norm_act: res must have x's shape {list(x.shape)} or half its height and width, got {list(res.shape)}")
    p.empty = x.numel() == 0
    p.half, p.res_shape = half, None if res is None else tuple(res.shape)
    p.index, p.dtype, p.shape, p.device = x.device.index, x.dtype, x.shape, x.device
    p.stat = 2 * n * groups
    p.grid = _grid(c, groups, x.element_size())
    p.desc = _lib.GnDesc(n, 0 if p.empty else x.numel() // (n * c), row, c, groups,
                         _DTYPES[x.dtype], ACTS[act], x.shape[2] if half else 0, int(per_sample), float(eps), float(slope),
                         float(out_slope), float(w_off))
    p.at = ctypes.addressof(p.desc)
    p.ws, p.ws_bwd = (0, 0) if p.empty else (lib().m355_group_norm_ws_bytes(p.at, 0), lib().m355_group_norm_ws_bytes(p.at, 1))
    if not p.empty and not p.ws_bwd:
        raise _lib.M355Error("group_norm_act: " + lib().m355_last_error().decode("utf-8", "replace"))
    return p


def _key(t):
    return None if t is None else (t.shape, t.dtype, t.device, t.stride())


def _forward(x, weight, bias, res, p):
    y = torch.empty_like(x)
    # (a small workspace lies behind the statistics: one allocation; a large one must not live as long as they do)
    small = p.ws <= 65536
    stat = torch.empty((p.stat + (-p.stat) % 4 + p.ws // 4 if small else p.stat,), dtype=torch.float32, device=x.device)
    if not p.empty:
        at = stat.data_ptr()
        ws = None if small else torch.empty((p.ws,), dtype=torch.uint8, device=x.device)
        with on_device(p.index):
            launch("group_norm_fwd", p.at, x.data_ptr(), None if weight is None else weight.data_ptr(),
                   None if bias is None else bias.data_ptr(), None if res is None else res.data_ptr(), y.data_ptr(), at,
                   at + 4 * (p.stat + (-p.stat) % 4) if small else ws.data_ptr(), stream())
    return y, stat


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, res, p):
        y, stat = _forward(x, weight, bias, res, p)
        ctx.save_for_backward(x, weight, bias, stat)
        ctx.p = p
        return y

    @staticmethod
    def backward(ctx, dy):
        if torch.is_grad_enabled():   # (create_graph)
            return _Once.apply(ctx.p, ctx.needs_input_grad, dy, *ctx.saved_tensors)
        return _backward(ctx.p, ctx.needs_input_grad, dy, *ctx.saved_tensors)


def _saved(p, x, weight, bias, stat):
    """the saved tensors as the kernels read them, and the descriptor for them.  A saved-tensor hook -- or an assignment to .data -- may bring
    a tensor back in another layout than the plan was made for: offloading makes a slice of a wide matrix dense"""
    dev = p.device
    changed = x.shape != p.shape or x.dtype is not p.dtype or x.device != dev or stat.dtype is not _F32 or stat.device != dev \
        or stat.numel() < p.stat
    moved = False
    for t in (weight, bias):
        if t is not None:
            changed = changed or t.shape != p.aff_shape or t.dtype is not _F32 or t.device != dev
            moved = moved or t.stride() != p.aff_strides
    if changed:
        raise RuntimeError("group_norm_act: a saved tensor has come back with another shape, type or device than it was saved with")
    desc = p.desc
    if moved:
        row = _rows([t for t in (weight, bias) if t is not None], p.shape[-1])
        if row is None:
            weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
            row = p.shape[-1] if len(p.aff_shape) == 2 else 0
        desc = _lib.GnDesc.from_buffer_copy(desc)
        desc.aff_stride = row
    return x.contiguous(), weight, bias, stat.contiguous(), desc


def _backward(p, needs, dy, x, weight, bias, stat):
    need_x, need_w, need_b, need_r, _ = needs
    x, weight, bias, stat, desc = _saved(p, x, weight, bias, stat)
    if dy.dtype != p.dtype:
        dy = dy.to(p.dtype)
    if not dy.is_contiguous():
        dy = dy.contiguous()
    dx = torch.empty_like(x) if need_x else None
    dw = torch.empty_like(weight, memory_format=torch.contiguous_format) if need_w else None
    db = torch.empty_like(bias, memory_format=torch.contiguous_format) if need_b else None
    dres = dy if need_r else None
    if p.grid:
        x, dy = _on_grid(x, p.grid), _on_grid(dy, p.grid)
    if need_r and p.half:
        dres = torch.empty(p.res_shape, dtype=p.dtype, device=x.device)
    if p.empty:
        for t in (dw, db):
            if t is not None:
                t.zero_()
    elif need_x or need_w or need_b or (need_r and p.half):
        ws = torch.empty((p.ws_bwd,), dtype=torch.uint8, device=x.device)
        with on_device(p.index):
            launch("group_norm_bwd", ctypes.addressof(desc), dy.data_ptr(), x.data_ptr(), None if weight is None else weight.data_ptr(),
                   None if bias is None else bias.data_ptr(), stat.data_ptr(), None if dx is None else dx.data_ptr(),
                   None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                   dres.data_ptr() if need_r and p.half else None, ws.data_ptr(), stream())
    return dx, dw, db, dres, None


class _Once(torch.autograd.Function):
    """the gradients of a backward pass that is itself recorded: whoever differentiates them -- by dy, x or the affine -- is told"""

    @staticmethod
    def forward(ctx, p, needs, dy, x, weight, bias, stat):
        return _backward(p, needs, dy, x, weight, bias, stat)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("group_norm_act can be differentiated once: no second derivatives")


def _has_tangent(t):
    return torch.is_tensor(t) and fwad.unpack_dual(t).tangent is not None


def _apply(x, num_groups, weight, bias, eps, act, slope, res, w_off, out_slope):
    if _is_tracing():   # (a trace records the result's allocation, not the launches; or the plan of the sizes it was made with)
        raise RuntimeError("group_norm_act cannot be traced")
    # (a tensor with a tangent need not require a gradient: it would take the way without autograd, and lose it)
    if fwad._current_level >= 0 and any(map(_has_tangent, (x, weight, bias, res))):
        raise RuntimeError("group_norm_act has no forward-mode derivative")
    try:
        key = (x.shape, x.dtype, x.device, index(num_groups), float(eps), act, float(slope), w_off, out_slope, _key(weight), _key(bias),
               None if res is None else (res.shape, res.dtype, res.device))
        p = _PLANS.get(key)
    except (AttributeError, TypeError, ValueError):   # (not tensors, not numbers: the checks say what)
        key = p = None
    if p is None:
        p = _make_plan(x, num_groups, weight, bias, eps, act, slope, res, w_off, out_slope)
        if len(_PLANS) >= 1024:
            _PLANS.clear()
        if key is not None:
            _PLANS[key] = p
    if p.floats:
        weight, bias = (None if t is None else t.float().contiguous() for t in (weight, bias))
    if not x.is_contiguous():
        x = x.contiguous()
    if res is not None and not res.is_contiguous():
        res = res.contiguous()
    if p.grid:
        x, res = _on_grid(x, p.grid), None if res is None else _on_grid(res, p.grid)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad) or (res is not None and res.requires_grad)):
        return _GroupNormAct.apply(x, weight, bias, res, p)
    return _forward(x, weight, bias, res, p)[0]


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="lrelu", slope=1.0, res=None):
    """Group norm of a channels-last tensor with the activation behind it, one fused operator with its gradient.

    x [N, ..., C] float32 / float16 / bfloat16 (an NCHW tensor in torch's channels_last format is `x.permute(0, 2, 3, 1)`; other
    strides are copied); num_groups divides C; every (sample, group) is normalised by its own mean and biased variance, held in
    float32 (a group of more channels than 256 vectors hold -- of 16 bytes, or the widest that C is a multiple of -- is refused).
    weight, bias: [C], or [N, C] (conditional norms: one affine per sample; rows of a larger matrix are read in place), or None
    (1 / 0).  act 'lrelu': LeakyReLU(slope) -- slope 1.0 is no activation, 0.0 is ReLU, the derivative at 0 is 1 -- or 'silu'.
    res: added after the activation; x's shape, or half of x's height and width, read through the nearest x2 upsample.
    Returns y of x's shape and type, rounded once.  Gradients reach x, weight, bias and res (first
    derivatives: differentiating them again raises, as do forward-mode tangents); it cannot be traced.  The results do not depend on the run."""
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
