"""GPU: calls of group norm and gradient clipping that programs make around the plain one -- saved tensors that were moved, tensors off the
vector grid, lists and maps larger than the memory-side cache."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, H, F = torch.bfloat16, torch.float16, torch.float32


def _spread(t):
    """the same values in rows that are further apart than they need be"""
    s = torch.zeros(t.shape[:-1] + (2 * t.shape[-1] + 3,), dtype=t.dtype, device=t.device)
    return s[..., :t.shape[-1]].copy_(t)


@pytest.mark.parametrize("shape,groups", [((16, 8, 4, 512), 32), ((4, 64, 32, 256), 32), ((1, 400, 301, 24), 3)], ids=str)
@pytest.mark.parametrize("affine", ["sliced", "layer"])
def test_saved_tensors_that_were_moved(pkg, shape, groups, affine):
    """offloading to the host and back, and other layouts from a hook: the bits of the plain backward.  (The affine as the generator passes
    it: slices of one wide matrix, rows far apart)"""
    n, c = shape[0], shape[-1]
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(shape, generator=g, device=DEV).to(BF)
    dy = (0.1 * torch.randn(shape, generator=g, device=DEV)).to(BF)
    wide = 0.3 * torch.randn(n, 3 * c, generator=g, device=DEV)
    w, b = (wide[:, c // 2:c // 2 + c], wide[:, 2 * c:]) if affine == "sliced" else (wide[0, :c], wide[0, c:2 * c])
    norm = pkg.GroupNorm2d(c, groups)

    def go(ctx=None):
        xs, ws, bs = x.detach().requires_grad_(), w.detach().requires_grad_(), b.detach().requires_grad_()
        f = (lambda: norm(xs, ws, bs, slope=0.2) if affine == "sliced" else pkg.group_norm_act(xs, groups, ws, bs, slope=0.2))
        if ctx is None:
            y = f()
        else:
            with ctx:
                y = f()
        return [y.detach()] + list(torch.autograd.grad(y, (xs, ws, bs), dy))
    want = go()
    hooks = torch.autograd.graph.saved_tensors_hooks
    for ctx in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True), hooks(_spread, lambda t: t),
                hooks(lambda t: t.transpose(0, -1).contiguous().transpose(0, -1), lambda t: t)):
        for a, k in zip(go(ctx), want):
            assert torch.equal(a, k)


def _off_grid(t, off):
    s = torch.empty(t.numel() + off, dtype=t.dtype, device=t.device)
    return s[off:].view(t.shape).copy_(t)


@pytest.mark.parametrize("c,groups,dtype", [(512, 1, BF), (640, 2, H), (1020, 2, BF), (1024, 1, F), (2048, 1, H)], ids=str)
@pytest.mark.parametrize("hw", [(4, 2), (40, 64)], ids=str)
def test_wide_groups_off_the_vector_grid(pkg, c, groups, dtype, hw):
    """x, the residual and the incoming gradient one element behind a vector's address, one at a time and together: taken as from an aligned
    one, with the same bits"""
    g = torch.Generator(device=DEV).manual_seed(c)
    x, res, dy = (torch.randn(3, *hw, c, generator=g, device=DEV).to(dtype) for _ in range(3))
    half = torch.randn(3, hw[0] // 2, hw[1] // 2, c, generator=g, device=DEV).to(dtype)
    w, b = 1 + 0.3 * torch.randn(c, generator=g, device=DEV), 0.2 * torch.randn(c, generator=g, device=DEV)

    def go(x, res, dy):
        ts = [t.detach().requires_grad_() for t in (x, w, b, res)]
        y = pkg.group_norm_act(ts[0], groups, ts[1], ts[2], slope=0.2, res=ts[3])
        return [y.detach()] + list(torch.autograd.grad(y, ts, dy))
    for r in (res, half):
        want = go(x, r, dy)
        for mask in range(1, 8):
            got = go(*(_off_grid(t, 1) if mask >> i & 1 else t for i, t in enumerate((x, r, dy))))
            assert all(torch.equal(a, k) for a, k in zip(got, want)), mask


@pytest.mark.parametrize("limit", [0.0, 1.0, float("inf")])
@pytest.mark.parametrize("form", ["in_place", "out"])
def test_a_nan_makes_every_gradient_nan(pkg, limit, form):
    """whatever the threshold, as torch.nn.utils.clip_grad_norm_; an infinite norm under an infinite threshold clips nothing"""
    for bad in (float("nan"), float("inf")):
        ts = [torch.ones(5000, device=DEV), torch.ones(77, dtype=BF, device=DEV), torch.ones(3, dtype=H, device=DEV)]
        ts[1][5] = bad
        out = None if form == "in_place" else [torch.zeros_like(t) for t in ts]
        before = [t.clone() for t in ts]
        n = pkg.clip_grads_(ts, limit, out=out)
        got = ts if out is None else out
        if bad != bad:
            assert torch.isnan(n) and all(torch.isnan(t).all() for t in got)
        elif limit == float("inf"):
            assert torch.isinf(n) and all(torch.equal(t, b) for t, b in zip(got, before))
        else:
            assert torch.isinf(n) and torch.isnan(got[1][5]) and float(got[0].abs().max()) == 0.0 and float(got[2].abs().max()) == 0.0


def test_a_norm_past_32_bits_still_clips(pkg):
    """1000 values of 3e38: the norm, 9.5e39, is returned as infinity, the factor is the 64-bit norm's"""
    t = torch.full((1000,), 3e38, device=DEV)
    factor = 1e30 / float((t.double() ** 2).sum() ** 0.5 + 1e-6)
    want = t.double() * factor
    assert torch.isinf(pkg.clip_grads_([t], 1e30)) and ((t.double() - want).abs() <= 2.0 ** -23 * want + 2.0 ** -24 * want).all()
