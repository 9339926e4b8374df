"""Global norm of a list of gradients and clipping by it (csrc/grad_clip.hip, include/m355.h m355_grad_clip): two launches for a list of
any length up to 112 tensors, no host synchronisation, capturable.  No CPU or torch fallback: CPU tensors raise.

    norm = |scale| * sqrt(sum of squares),   out = g * scale * min(1, max_norm / (norm + 1e-6))

`clip_grad_norm_` takes parameters as torch.nn.utils.clip_grad_norm_ does, `clip_grads_` the gradient tensors themselves (in place, or
into `out` buffers with a scale: averaging a summed message and clipping it is one pass), `grad_norm` only measures."""
from array import array

import torch
import torch.autograd.forward_ad as fwad

from . import _lib
from ._lib import launch, lib, stream
from .group_norm import _DTYPES, _has_tangent, _is_tracing, on_device

_strided, _same_size = torch.strided, torch.Tensor.is_same_size


def _flat(t):
    """the tensor's values lie in its memory without gaps, in whatever order (a permuted view counts)"""
    want = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _check(tensors, what):
    """-> the list, its device's index, how every tensor's values lie (2: in order, 1: without gaps, 0: otherwise), and the lists of addresses,
    counts and types"""
    ts = [tensors] if torch.is_tensor(tensors) else list(tensors)
    if not ts:
        raise ValueError(f"{what}: no gradients")
    if _is_tracing():   # (a trace records the norm's allocation, not the launches)
        raise RuntimeError(f"{what} cannot be traced")
    if fwad._current_level >= 0 and any(map(_has_tangent, ts)):
        raise RuntimeError(f"{what} has no forward-mode derivative")
    together, at, nums, kinds = 2, [], [], []
    try:
        index = ts[0].get_device()
        for t in ts:
            if t.get_device() != index or index < 0 or t.layout is not _strided:
                break
            kinds.append(_DTYPES[t.dtype])
            nums.append(t.numel())
            at.append(t.data_ptr())
            if together and not t.is_contiguous():
                together = 1 if _flat(t) or t.numel() == 0 else 0
        else:
            return ts, index, together, at, nums, kinds
    except (AttributeError, KeyError, RuntimeError, NotImplementedError):   # (not tensors, or not of this kind: said below)
        pass
    for t in ts:
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise _lib.M355Error(f"{what}: gradients must be CUDA(HIP) tensors; there is no CPU implementation")
        if t.layout is not _strided:
            raise TypeError(f"{what}: a gradient is {t.layout}: dense tensors only")
        if t.dtype not in _DTYPES:
            raise TypeError(f"{what}: gradients must be float32, float16 or bfloat16, got {t.dtype}")
        if t.device != ts[0].device:
            raise ValueError(f"{what}: gradients on {ts[0].device} and on {t.device}: clip each device's own list")
    raise _lib.M355Error(f"{what}: a gradient has no memory of its own ({type(ts[0])})")


def _run(dev, index, at, out, nums, kinds, max_norm, scale):
    n = len(at)
    with on_device(index):
        ws = torch.empty((lib().m355_grad_clip_ws_bytes(n),), dtype=torch.uint8, device=dev)
        norm = torch.empty((), dtype=torch.float32, device=dev)
        ptrs = array("Q", at)
        optr = ptrs if out is at or out is None else array("Q", out)
        nums, kinds = array("q", nums), array("i", kinds)
        launch("grad_clip", ptrs.buffer_info()[0], None if out is None else optr.buffer_info()[0], nums.buffer_info()[0],
               kinds.buffer_info()[0], n, scale, max_norm, norm.data_ptr(), ws.data_ptr(), stream())
    return norm


def grad_norm(grads, scale=1.0):
    """The 2-norm of all values of `grads` (a tensor or an iterable of tensors, float32 / float16 / bfloat16 mixed, one device), times
    |scale|: a 0-dimensional float32 tensor on their device.  Squares are added in 64 bits in a fixed order.  A measurement: no gradient
    flows back through it."""
    ts, index, together, at, nums, kinds = _check(grads, "grad_norm")
    if not together:
        with torch.no_grad():
            ts = [t.contiguous() for t in ts]
        at = [t.data_ptr() for t in ts]
    return _run(ts[0].device, index, at, None, nums, kinds, 0.0, float(scale))


def clip_grads_(grads, max_norm, out=None, scale=1.0):
    """Scale the gradient tensors so that their global 2-norm (of scale * gradients) is at most max_norm -> that norm before clipping, a
    0-dimensional float32 tensor on their device.

    In place, or -- out: as many tensors of the same shapes, types and strides -- written there, the gradients left as they were.
    max_norm >= 0.  A NaN makes all gradients NaN, whatever max_norm is; an infinite value makes the finite ones 0 (both as
    torch.nn.utils.clip_grad_norm_).  An infinite max_norm clips nothing else, an infinite norm included: the returned norm says so.
    (The factor comes from the 64-bit norm: one past float32's range is returned as infinity and still clips.)
    Tensors that share memory (the same gradient twice) are refused."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grads_: max_norm={max_norm!r}")
    ts, index, together, at, nums, kinds = _check(grads, "clip_grads_")
    if not together:
        raise ValueError("clip_grads_: a gradient's values have gaps or repeats between them (an expanded or sliced view)")
    outs, to = ts, at
    if out is not None:
        outs, o_index, o_together, to, o_nums, o_kinds = _check(out, "clip_grads_")
        if o_index != index or o_nums != nums or o_kinds != kinds:
            raise ValueError("clip_grads_: as many outputs as gradients, of their types and shapes, on their device")
        if not (all(map(_same_size, ts, outs)) and
                (together == o_together == 2 or all(t.is_contiguous() and o.is_contiguous() or t.stride() == o.stride() for t, o in zip(ts, outs)))):
            raise ValueError("clip_grads_: an output must have its gradient's shape and strides")
    norm = _run(ts[0].device, index, at, to, nums, kinds, max_norm, float(scale))
    torch.autograd.graph.increment_version(outs)
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
