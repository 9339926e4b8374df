"""Global norm of a list of gradients and clipping by it (csrc/grad_clip.hip, include/m355.h m355_grad_clip): two launches for a list of
any length up to 112 tensors, no host synchronisation, capturable.  No CPU or torch fallback: CPU tensors raise.

    norm = |scale| * sqrt(sum of squares),   out = g * scale * min(1, max_norm / (norm + 1e-6))

`clip_grad_norm_` takes parameters as torch.nn.utils.clip_grad_norm_ does, `clip_grads_` the gradient tensors themselves (in place, or
into `out` buffers with a scale: averaging a summed message and clipping it is one pass), `grad_norm` only measures."""
import ctypes

import torch

from . import _lib
from ._lib import launch, lib, ptr, stream
from .group_norm import _DTYPES, _on


def _flat(t):
    """the tensor's values lie in its memory without gaps, in whatever order (a permuted view counts)"""
    if t.is_contiguous():
        return True
    want = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _check(tensors, what):
    ts = [tensors] if torch.is_tensor(tensors) else list(tensors)
    dev = None
    for t in ts:
        if not torch.is_tensor(t) or not t.is_cuda:
            raise _lib.M355Error(f"{what}: gradients must be CUDA(HIP) tensors; there is no CPU implementation")
        if t.layout != torch.strided:
            raise TypeError(f"{what}: a gradient is {t.layout}: dense tensors only")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{what}: gradients must be float32, float16 or bfloat16, got {t.dtype}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{what}: gradients on {dev} and on {t.device}: clip each device's own list")
    return ts, dev


def _run(ts, outs, dev, max_norm, scale):
    n = len(ts)
    norm = torch.empty((), dtype=torch.float32, device=dev)
    with _on(norm):
        ws = torch.empty((lib().m355_grad_clip_ws_bytes(n),), dtype=torch.uint8, device=dev)
        args = [(ctypes.c_void_p * n)(*[t.data_ptr() for t in ts]),
                None if outs is None else (ctypes.c_void_p * n)(*[t.data_ptr() for t in outs]),
                (ctypes.c_longlong * n)(*[t.numel() for t in ts]), (ctypes.c_int * n)(*[_DTYPES[t.dtype] for t in ts])]
        launch("grad_clip", *args, n, float(scale), float(max_norm), ptr(norm), ptr(ws), stream())
    return norm


def grad_norm(grads, scale=1.0):
    """The 2-norm of all values of `grads` (a tensor or an iterable of tensors, float32 / float16 / bfloat16 mixed, one device), times
    |scale|: a 0-dimensional float32 tensor on their device.  Squares are added in 64 bits in a fixed order."""
    ts, dev = _check(grads, "grad_norm")
    if not ts:
        raise ValueError("grad_norm: no gradients")
    with torch.no_grad():
        return _run([t if _flat(t) else t.contiguous() for t in ts], None, dev, 0.0, scale)


def clip_grads_(grads, max_norm, out=None, scale=1.0):
    """Scale the gradient tensors so that their global 2-norm (of scale * gradients) is at most max_norm -> that norm before clipping, a
    0-dimensional float32 tensor on their device.

    In place, or -- out: as many tensors of the same shapes, types and strides -- written there, the gradients left as they were.
    max_norm >= 0, infinity never clips.  An infinite norm makes the finite gradients 0, a NaN makes all of them NaN (as
    torch.nn.utils.clip_grad_norm_): the returned norm says so.  Tensors that share memory (the same gradient twice) are refused."""
    ts, dev = _check(grads, "clip_grads_")
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads_: max_norm={max_norm!r}")
    if not ts:
        raise ValueError("clip_grads_: no gradients")
    outs = ts if out is None else _check(out, "clip_grads_")[0]
    if len(outs) != len(ts):
        raise ValueError(f"clip_grads_: {len(ts)} gradients, {len(outs)} outputs")
    for t, o in zip(ts, outs):
        if not _flat(t):
            raise ValueError(f"clip_grads_: a gradient of shape {list(t.shape)} and strides {list(t.stride())} has gaps or repeats")
        if o is not t and (o.device != dev or o.dtype != t.dtype or o.shape != t.shape
                           or (o.stride() != t.stride() and not (o.is_contiguous() and t.is_contiguous()))):
            raise ValueError("clip_grads_: an output must have its gradient's device, type, shape and strides")
    with torch.no_grad():
        norm = _run(ts, outs, dev, max_norm, scale)
        for o in outs:
            torch.autograd.graph.increment_version(o)
    return norm


def clip_grad_norm_(parameters, max_norm):
    """torch.nn.utils.clip_grad_norm_(parameters, max_norm) for the 2-norm: clip the .grad of the parameters in place -> the norm before
    clipping.  Parameters without a gradient are skipped; none with one: 0."""
    ps = [parameters] if torch.is_tensor(parameters) else list(parameters)
    grads = [p.grad for p in ps if p.grad is not None]
    if not grads:
        if not float(max_norm) >= 0.0:
            raise ValueError(f"clip_grad_norm_: max_norm={max_norm!r}")
        return torch.zeros((), device=ps[0].device) if ps else torch.zeros(())
    return clip_grads_(grads, max_norm)
