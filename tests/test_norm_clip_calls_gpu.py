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
