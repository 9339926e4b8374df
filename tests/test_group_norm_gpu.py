"""GPU: group norm with an activation, channels last (csrc/group_norm.hip), against the definition in 64 bits.

Tolerances.  u_t = eps(t) / 2 is the one rounding of a result to its type, u = 2^-24 a 32-bit rounding.  The statistics are joined
along a chain of at most CHAIN additions (a thread's few dozen loads, the trees over lanes, the ranges of a sample): relative to the
values' magnitude they are off by at most CHAIN u; a handful of further operations make a result of them.  So
    |y - y64|   <= u_t |y| + K u (|w| (|xhat| + M rstd) + |b| + |res|),       M = largest |x| of the group, K = 256 > CHAIN + 16
    |dx - dx64| <= u_t |dx| + K u rstd (|w dz| + A1 + |xhat| A2) (1 + M rstd),   A1 / A2 = group means of |w dz|, |w dz xhat|
    |dw - dw64| <= K u sum |dz| (|xhat| + M rstd),   |db - db64| <= K u sum |dz|
(M rstd: how much a 32-bit mean, off by K u M, moves xhat.)  SiLU's derivative changes by at most 0.5 per unit of z: the same order,
covered by |dy| in the place of |dz|.  A LeakyReLU's dz is not continuous at z = 0: no gradient arrives within 1e-3 of it."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
K, U = 256.0, 2.0 ** -24
EPS = 1e-5


def ut(dtype):
    return torch.finfo(dtype).eps / 2


def definition(x, groups, w, b, act, slope, res, eps=EPS):
    """64 bits, on the CPU: y, xhat, rstd and M as [N,HW,C]-shaped tensors (autograd through everything)"""
    n, c = x.shape[0], x.shape[-1]
    xg = x.reshape(n, -1, groups, c // groups)
    mu = xg.mean((1, 3), keepdim=True)
    rstd = ((xg - mu).pow(2).mean((1, 3), keepdim=True) + eps).rsqrt()
    xhat = ((xg - mu) * rstd).reshape(n, -1, c)
    shape = (lambda t: t[:, None, :] if t.dim() == 2 else t[None, None, :])
    z = xhat * (1.0 if w is None else shape(w)) + (0.0 if b is None else shape(b))
    y = torch.nn.functional.silu(z) if act == "silu" else torch.where(z >= 0, z, z * slope)
    r = 0.0
    if res is not None:
        r = res if res.shape == x.shape else res.repeat_interleave(2, 1).repeat_interleave(2, 2)
        y = y + r.reshape(n, -1, c)
    big = xg.abs().amax((1, 3), keepdim=True).expand_as(xg).reshape(n, -1, c)
    rs = rstd.expand_as(xg).reshape(n, -1, c)
    return y, z, xhat, rs, big


def make(shape, groups, dtype, act, slope, affine, res, seed=0, offset=0.4):
    n, c = shape[0], shape[-1]
    g = torch.Generator().manual_seed(seed + 7 * c + n)
    x = (torch.randn(shape, generator=g) * (0.5 + torch.rand(c, generator=g)) + offset * torch.randn(c, generator=g)).to(dtype)
    ws = {"none": None, "layer": (c,), "sample": (n, c)}[affine]
    w = None if ws is None else 1 + 0.3 * torch.randn(ws, generator=g)
    b = None if ws is None else 0.2 * torch.randn(ws, generator=g)
    r = None
    if res == "full":
        r = torch.randn(shape, generator=g).to(dtype)
    elif res == "half":
        r = torch.randn((n, shape[1] // 2, shape[2] // 2, c), generator=g).to(dtype)
    dy = (0.1 * torch.randn(shape, generator=g)).to(dtype)
    if act == "lrelu" and slope != 1.0:
        z = definition(x.double(), groups, None if w is None else w.double(), None if b is None else b.double(), act, slope, None)[1]
        dy[z.reshape(shape).abs() < 1e-3] = 0.0
    return x, w, b, r, dy


def run_and_check(pkg, x, groups, w, b, r, dy, act, slope, eps=EPS):
    dtype, n, c = x.dtype, x.shape[0], x.shape[-1]
    leaf = (lambda t: None if t is None else t.detach().double().requires_grad_())
    x6, w6, b6, r6 = leaf(x), leaf(w), leaf(b), leaf(r)
    y6, z6, xhat, rs, big = definition(x6, groups, w6, b6, act, slope, r6, eps)
    y6.backward(dy.double().reshape(y6.shape))
    dev = (lambda t: None if t is None else t.detach().to(DEV).requires_grad_())
    xd, wd, bd, rd = dev(x), dev(w), dev(b), dev(r)
    y = pkg.group_norm_act(xd, groups, wd, bd, eps=eps, act=act, slope=slope, res=rd)
    assert y.dtype == dtype and y.shape == x.shape
    y.backward(dy.to(DEV))
    with torch.no_grad():
        full = (lambda t, other: torch.full((1, 1, c), other, dtype=torch.float64) if t is None else
                (t[:, None, :] if t.dim() == 2 else t[None, None, :]).double())
        W, B = full(w, 1.0), full(b, 0.0)
        R = torch.zeros(()) if r is None else (r if r.shape == x.shape else r.repeat_interleave(2, 1).repeat_interleave(2, 2)).double().reshape(n, -1, c)
        move = 1 + big * rs
        tol = ut(dtype) * y6.abs() + K * U * (W.abs() * (xhat.abs() + big * rs) + B.abs() + R.abs()) + tiny(dtype)
        check("y", y.detach().cpu().double().reshape(y6.shape), y6, tol)
        D = dy.double().reshape(n, -1, c).abs() * (1.1 if act == "silu" else max(1.0, abs(slope)))
        gmean = (lambda t: t.reshape(n, -1, groups, c // groups).mean((1, 3), keepdim=True).expand(n, t.shape[1], groups, c // groups).reshape(t.shape))
        WD = W.abs() * D
        tol = ut(dtype) * x6.grad.reshape(n, -1, c).abs() + K * U * rs * (WD + gmean(WD) + xhat.abs() * gmean(WD * xhat.abs())) * move + tiny(dtype)
        check("dx", xd.grad.cpu().double().reshape(n, -1, c), x6.grad.reshape(n, -1, c), tol)
        if w is not None:
            s = (lambda t: t.sum(1) if w.dim() == 2 else t.sum((0, 1)))
            check("dw", wd.grad.cpu().double(), w6.grad, K * U * s(D * (xhat.abs() + move)))
            check("db", bd.grad.cpu().double(), b6.grad, K * U * s(D * move))
        if r is not None:
            tol = ut(dtype) * r6.grad.abs() + (0.0 if r.shape == x.shape else 1.0) * 4 * U * dy.double().abs().max() + tiny(dtype)
            check("dres", rd.grad.cpu().double(), r6.grad, tol)


def tiny(dtype):
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133   # half a step among the subnormal numbers


def check(what, got, want, tol):
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    bad = off > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / tol).max()):.2f} times the tolerance"


BF, H, F = torch.bfloat16, torch.float16, torch.float32
CASES = [
    # shape, groups, dtype, act, slope, affine, res
    ((16, 8, 4, 512), 32, BF, "lrelu", 0.2, "sample", "full"),
    ((2, 64, 32, 256), 32, BF, "lrelu", 0.2, "sample", "half"),
    ((2, 128, 64, 64), 32, BF, "lrelu", 0.2, "sample", "half"),
    ((3, 32, 32, 128), 32, BF, "lrelu", 0.0, "layer", "none"),
    ((3, 37, 29, 60), 12, F, "silu", 1.0, "layer", "none"),
    ((2, 24, 20, 320), 32, H, "silu", 1.0, "layer", "full"),
    ((1, 1, 1, 1), 1, F, "lrelu", 1.0, "layer", "none"),        # a group of one value: xhat = 0
    ((3, 1, 1, 32), 4, BF, "silu", 1.0, "sample", "none"),      # one pixel
    ((2, 5, 1, 7), 7, H, "lrelu", 0.2, "layer", "full"),        # one channel a group, an odd count
    ((2, 5, 3, 7), 1, F, "lrelu", 0.2, "sample", "none"),       # one group
    ((2, 3, 5, 24), 8, BF, "silu", 1.0, "none", "none"),        # vectors of eight over groups of three
    ((2, 2, 2, 100), 20, BF, "lrelu", 1.0, "layer", "half"),    # vectors of four over groups of five
    ((1, 6, 6, 4096), 32, BF, "lrelu", 0.2, "layer", "none"),   # channels of two slabs
    ((1, 4, 3, 1030), 10, H, "silu", 1.0, "sample", "full"),    # slabs of vectors of two over groups of 103, the last one short
    ((2, 3, 3, 520), 4, F, "lrelu", 0.2, "layer", "none"),
    ((1, 2, 2, 2048), 1, BF, "silu", 1.0, "layer", "none"),     # the widest group of a 16-bit type
    ((1, 16, 16, 1024), 32, BF, "lrelu", 0.2, "sample", "half"),   # one pass, rows of 64 bytes
    ((40, 16, 16, 1024), 32, BF, "lrelu", 0.2, "layer", "half"),   # one pass, rows of 128 bytes, 8 vectors a thread
    ((2, 32, 16, 256), 32, BF, "silu", 1.0, "layer", "full"),      # one pass, rows of 64 bytes, 8 vectors a thread
    ((2, 31, 17, 96), 3, H, "lrelu", 0.2, "layer", "none"),        # a slab of a whole group of 32
    ((257, 2, 1, 16), 2, BF, "lrelu", 0.2, "sample", "none"),   # many samples
    ((1, 300, 301, 6), 3, BF, "lrelu", 0.2, "layer", "none"),   # many ranges, the last one short
    ((1, 258, 130, 16), 2, F, "silu", 1.0, "layer", "half"),
    ((1, 100, 100, 96), 8, BF, "lrelu", 0.2, "layer", "none"),  # 64 ranges, joined by the second pass
    ((1, 120, 128, 64), 64, H, "silu", 1.0, "sample", "none"),  # the same, few lanes a group
    ((1, 400, 301, 24), 3, BF, "lrelu", 0.2, "layer", "full"),  # 177 ranges, joined between the passes
    ((2, 258, 260, 32), 4, H, "silu", 1.0, "sample", "half"),
]


@pytest.mark.parametrize("shape,groups,dtype,act,slope,affine,res", CASES, ids=lambda v: str(v).replace("torch.", ""))
def test_against_the_definition(pkg, shape, groups, dtype, act, slope, affine, res):
    x, w, b, r, dy = make(shape, groups, dtype, act, slope, affine, res)
    run_and_check(pkg, x, groups, w, b, r, dy, act, slope)


@pytest.mark.parametrize("shape,groups,dtype,affine", [
    ((2500, 48), 6, BF, "layer"),             # more partial rows than one workgroup adds, the last chunk short
    ((2048, 1, 1, 512), 32, BF, "layer"),     # samples of one pixel: slabs wider than 128 bytes
    ((1100, 1, 3, 320), 5, H, "sample"),      # the same, the channels no multiple of the wider slab
    ((1500, 2, 2, 96), 3, F, "layer"),
], ids=lambda v: str(v).replace("torch.", ""))
def test_many_small_samples(pkg, shape, groups, dtype, affine):
    x, w, b, _, dy = make(shape, groups, dtype, "silu", 1.0, affine, "none")
    run_and_check(pkg, x, groups, w, b, None, dy, "silu", 1.0)


def test_affine_gradients_of_large_samples(pkg):
    """more ranges a sample than one workgroup adds up: per-sample dw, db against 64-bit sums of the same terms.  A chain of additions is
    at most 64 loads of a thread, 8 lane joins, 9 rows of a chunk, 5 joins, 5 chunks and 5 joins: below K"""
    n, h, w_, c, groups = 2, 2100, 2100, 8, 4
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(n, h, w_, c, generator=g, device=DEV).to(BF)
    dy = (0.1 * torch.randn(n, h, w_, c, generator=g, device=DEV)).to(BF)
    w = torch.ones(n, c, device=DEV, requires_grad=True)
    b = torch.zeros(n, c, device=DEV, requires_grad=True)
    dw, db = torch.autograd.grad(pkg.group_norm_act(x, groups, w, b), (w, b), dy)
    for i in range(n):
        xs, ds = x[i].double().reshape(-1, c), dy[i].double().reshape(-1, c)
        xg = xs.reshape(-1, groups, c // groups)
        rstd = ((xg - xg.mean((0, 2), keepdim=True)).pow(2).mean((0, 2), keepdim=True) + EPS).rsqrt()
        xhat = ((xg - xg.mean((0, 2), keepdim=True)) * rstd).reshape(-1, c)
        big = (xs.abs().amax() * rstd.max())
        assert ((db[i] - ds.sum(0)).abs() <= K * U * ds.abs().sum(0)).all()
        assert ((dw[i] - (ds * xhat).sum(0)).abs() <= K * U * (ds.abs() * (xhat.abs() + big)).sum(0)).all()


@pytest.mark.parametrize("offset,outlier", [(1000.0, 0.0), (0.0, 1e4), (-30000.0, 0.0)])
def test_statistics_do_not_cancel(pkg, offset, outlier):
    """a mean far from zero, and one far value at the place a range starts: the variance keeps its digits (bf16-exact inputs keep
    the 64-bit statistics those of the same numbers)"""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 64, 64, 16, generator=g) + offset
    x[:, 0, 0, 0] += outlier
    w, b = torch.ones(16), torch.zeros(16)
    dy = 0.1 * torch.randn(x.shape, generator=g)
    run_and_check(pkg, x, 2, w, b, None, dy, "silu", 1.0)


def test_other_dimensions(pkg):
    """[N,C], [N,L,C] and [N,A,B,D,C] are the same operator on their values"""
    g = torch.Generator().manual_seed(1)
    for shape in ((4, 48), (2, 11, 48), (2, 3, 2, 5, 48)):
        x, dy = torch.randn(shape, generator=g), torch.randn(shape, generator=g)
        run_and_check(pkg, x, 6, torch.randn(48, generator=g), torch.randn(48, generator=g), None, dy, "silu", 1.0)


def test_values_that_are_not_finite_stay_in_their_group(pkg):
    g = torch.Generator().manual_seed(5)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.randn(3, 20, 20, 32, generator=g).to(BF)
        ok = pkg.group_norm_act(x.to(DEV), 4)
        x[1, 7, 3, 9] = bad    # sample 1, group 1
        y = pkg.group_norm_act(x.to(DEV), 4)
        hit = torch.zeros(x.shape, dtype=torch.bool)
        hit[1, :, :, 8:16] = True
        assert torch.isnan(y.cpu()[hit]).all() and torch.equal(y.cpu()[~hit], ok.cpu()[~hit])


def test_empty_batches(pkg):
    for shape in ((0, 4, 4, 16), (3, 0, 4, 16)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w, b = torch.ones(16, device=DEV, requires_grad=True), torch.zeros(16, device=DEV, requires_grad=True)
        y = pkg.group_norm_act(x, 4, w, b, slope=0.2)
        y.sum().backward()
        assert y.shape == x.shape and x.grad.shape == x.shape
        assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(b.grad, torch.zeros_like(b))


def test_refusals_on_the_device(pkg):
    """each refused by the host, before anything is launched"""
    x = torch.zeros(2, 6, 4, 12, device=DEV)
    row, rows = torch.ones(12, device=DEV), torch.ones(2, 12, device=DEV)
    f = pkg.group_norm_act
    for bad in (lambda: f(x, 5), lambda: f(x, 0), lambda: f(x, -3), lambda: f(x[0, 0, 0], 3), lambda: f(x, 3, row[:6]), lambda: f(x, 3, rows[:1]),
                lambda: f(x, 3, row, rows), lambda: f(x, 3, rows[:, None]), lambda: f(x, 3, eps=-1.0), lambda: f(x, 3, eps=float("nan")),
                lambda: f(x, 3, act="gelu"), lambda: f(x, 3, res=x[:, :3]), lambda: f(x, 3, res=x[:, :3, :2, :6]),
                lambda: f(x[:, :5], 3, res=x[:, :2, :2])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: f(x.double(), 3), lambda: f(x.int(), 3), lambda: f(x, 3, row.double()), lambda: f(x, 3, None, row.int()),
                lambda: f(x, 3, res=x.half()), lambda: f(x, 3, res=x.cpu()), lambda: f(x, 3.5), lambda: f(x, "3")):
        with pytest.raises(TypeError):
            bad()
    wide = torch.zeros(2, 3, 4096, device=DEV, dtype=BF)
    for bad in (lambda: f(x.cpu(), 3), lambda: f(x, 3, row.cpu()), lambda: f(x, 3, None, rows.cpu()), lambda: f(wide, 1),
                lambda: f(wide[..., :257], 1)):
        with pytest.raises(pkg._lib.M355Error):
            bad()
    assert torch.equal(f(x, 3, row, row), torch.ones_like(x))   # (the next call is not disturbed)


def test_strides_and_views(pkg):
    """a permuted NCHW tensor, a slice of channels, an affine read in place from a wide matrix, an expanded one, an expanded gradient
    and addresses off the vector grid: all the bits of the plain layout"""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 10, 14, 64, generator=g).to(BF).to(DEV)
    wide = (torch.randn(3, 200, generator=g) * 0.2).to(DEV)
    w, b = wide[:, 5:69], wide[:, 100:164]

    def go(xx, ww, bb, dy=None):
        xx, ww, bb = xx.detach().requires_grad_(), ww.detach().requires_grad_(), bb.detach().requires_grad_()
        y = pkg.group_norm_act(xx, 8, ww, bb, slope=0.2)
        (y.float().sum() if dy is None else (y * dy).float().sum()).backward()
        return y.detach(), xx.grad, ww.grad, bb.grad

    want = go(x, w.contiguous(), b.contiguous())
    nchw = x.permute(0, 3, 1, 2).contiguous()
    cl = nchw.contiguous(memory_format=torch.channels_last)
    for other in (nchw.permute(0, 2, 3, 1), cl.permute(0, 2, 3, 1), torch.cat((x, x), dim=3)[..., 64:]):
        for a, c in zip(go(other, w, b), want):
            assert torch.equal(a, c)
    one = go(x, w[:1].expand(3, -1), b[:1].expand(3, -1))
    two = go(x, w[:1].expand(3, -1).contiguous(), b[:1].expand(3, -1).contiguous())
    for a, c in zip(one, two):
        assert torch.equal(a, c)
    # a base address that is a multiple of one element only: other vectors, the same statistics to rounding, the same function
    store = torch.empty(x.numel() + 1, dtype=BF, device=DEV)
    odd = store[1:].view(x.shape).copy_(x)
    y = pkg.group_norm_act(odd, 8, w, b, slope=0.2)
    assert (y.float() - want[0].float()).abs().max() <= 2 * ut(BF) * want[0].float().abs().max()


def test_each_gradient_alone(pkg):
    """only the gradients that are asked for are made, each the same bits as with all of them"""
    x, w, b, r, dy = (t.to(DEV) for t in make((2, 12, 10, 48), 6, BF, "lrelu", 0.2, "layer", "half"))
    args = [x, w, b, r]
    every = None
    for mask in (15, 1, 2, 4, 8, 6):
        ts = [t.detach().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate(args)]
        pkg.group_norm_act(ts[0], 6, ts[1], ts[2], slope=0.2, res=ts[3]).backward(dy)
        if mask == 15:
            every = [t.grad for t in ts]
        for i, t in enumerate(ts):
            assert (t.grad is None) == (not mask >> i & 1)
            assert t.grad is None or torch.equal(t.grad, every[i])


def test_gradient_against_differences(pkg):
    """directional derivatives of sum(y * dy) along random directions.  Central differences with h = 1/64: the error is
    h^2 / 6 |third derivative| (below 1e-4 of the scale for these inputs of unit spread) plus the noise of the 32-bit y,
    2^-22 sqrt(n) |dy| / h = 2.4e-7 * 64 * 0.1 * sqrt(n) per evaluation"""
    x, w, b, r, dy = make((2, 6, 5, 24), 4, F, "silu", 1.0, "sample", "full", seed=4)
    x, w, b, r, dy = (t.to(DEV) for t in (x, w, b, r, dy))
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
    pkg.group_norm_act(leaves[0], 4, leaves[1], leaves[2], act="silu", res=leaves[3]).backward(dy)
    g = torch.Generator(device=DEV).manual_seed(8)
    h = 2.0 ** -6
    for i in range(4):
        v = torch.randn(leaves[i].shape, generator=g, device=DEV)
        side = []
        for s in (h, -h):
            t = [k.detach() for k in leaves]
            t[i] = t[i] + s * v
            side.append((pkg.group_norm_act(t[0], 4, t[1], t[2], act="silu", res=t[3]).double() * dy.double()).sum().item())
        got = (leaves[i].grad.double() * v.double()).sum().item()
        scale = (dy.double().abs() * 1.0).norm().item() * 2
        assert abs((side[0] - side[1]) / (2 * h) - got) < 2e-3 * scale + 2.4e-7 * 64 * 0.1 * dy.numel() ** 0.5, i


def test_same_bits_every_run_and_on_any_stream(pkg):
    for shape, groups in (((4, 64, 64, 64), 32), ((8, 8, 4, 512), 32)):
        x, w, b, r, dy = (t.to(DEV) for t in make(shape, groups, BF, "lrelu", 0.2, "sample", "half"))

        def go():
            ts = [t.detach().requires_grad_() for t in (x, w, b, r)]
            y = pkg.group_norm_act(ts[0], groups, ts[1], ts[2], slope=0.2, res=ts[3])
            y.backward(dy)
            return [y.detach()] + [t.grad for t in ts]
        want = go()
        side = torch.cuda.Stream()
        for _ in range(5):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                other = go()
            here = go()     # (both streams at once: every call has its own workspace)
            torch.cuda.synchronize()
            for a, c, d in zip(want, here, other):
                assert torch.equal(a, c) and torch.equal(a, d)


def test_two_threads_on_streams_of_their_own(pkg):
    """calls of both operators from two threads at once, each on its stream: the bits of one thread alone (one-pass, joined and finished
    statistics, shared and per-sample affines)"""
    import threading
    calls = []
    for i, (shape, groups, dtype, affine, res) in enumerate([((4, 8, 4, 64), 8, BF, "sample", "none"), ((2, 64, 32, 96), 12, H, "layer", "half"),
                                                             ((1, 400, 301, 24), 3, F, "sample", "full"), ((3, 37, 29, 60), 12, BF, "layer", "none")]):
        x, w, b, r, dy = (None if t is None else t.to(DEV) for t in make(shape, groups, dtype, "silu", 1.0, affine, res, seed=i))
        calls.append((x, groups, w, b, r, dy))

    def work(out):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(6):
                for x, groups, w, b, r, dy in calls:
                    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
                    it = iter(leaves)
                    xs, ws, bs, rs = (None if t is None else next(it) for t in (x, w, b, r))
                    y = pkg.group_norm_act(xs, groups, ws, bs, act="silu", res=rs)
                    g = torch.autograd.grad(y, leaves, dy)
                    clipped = [t.clone() for t in g]
                    out.append([y.detach(), *g, pkg.clip_grads_(clipped, 0.1), *clipped])
            torch.cuda.current_stream().synchronize()

    torch.cuda.synchronize()
    alone, outs, failed = [], [[], []], []
    work(alone)

    def guarded(out):
        try:
            work(out)
        except Exception as e:   # (a thread's exception does not reach the test by itself)
            failed.append(e)
    threads = [threading.Thread(target=guarded, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for o in outs:
        assert len(o) == len(alone) and all(torch.equal(p, q) for a, c in zip(alone, o) for p, q in zip(a, c))


def test_create_graph(pkg):
    """create_graph gives the same first gradients; a second derivative -- by x, the affine or dy -- is refused, not silently zero"""
    x, w, b, r, dy = (None if t is None else t.to(DEV) for t in make((2, 6, 4, 24), 4, F, "silu", 1.0, "layer", "half"))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    f = (lambda: pkg.group_norm_act(x, 4, w, b, act="silu", res=r))
    plain = torch.autograd.grad(f(), leaves, dy)
    again = torch.autograd.grad(f(), leaves, dy, create_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(plain, again))
    for t in again:
        with pytest.raises(RuntimeError, match="differentiated once"):
            t.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiated once"):
        penalty = torch.autograd.grad((f() ** 2).sum(), x, create_graph=True)[0]
        penalty.square().sum().backward()


def test_captured_forward_and_backward(pkg):
    """two graphs (their workspaces are their own), replayed with eager work between: every replay has the eager bits"""
    cases = []
    for shape, groups in (((4, 48, 32, 64), 32), ((8, 8, 4, 256), 32)):
        x, w, b, r, dy = (t.to(DEV) for t in make(shape, groups, BF, "lrelu", 0.2, "sample", "half"))
        ts = [t.detach().requires_grad_() for t in (x, w, b, r)]

        def go(ts=ts, groups=groups, dy=dy):
            y = pkg.group_norm_act(ts[0], groups, ts[1], ts[2], slope=0.2, res=ts[3])
            return [y.detach()] + list(torch.autograd.grad(y, ts, dy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go()
        cases.append((graph, out, ts, go))
    for k in range(4):
        for graph, out, ts, go in cases:
            with torch.no_grad():
                ts[0].copy_(torch.randn(ts[0].shape, device=DEV))
            for t in out:
                t.fill_(-7)
            graph.replay()
        torch.cuda.synchronize()
        for graph, out, ts, go in cases:
            for a, c in zip(out, go()):
                assert torch.equal(a, c), k


def test_offsets_past_32_bits(pkg):
    """a tensor of more than 2^31 values: the last sample's values are those of the sample alone"""
    n, hw, c = 33, 1 << 20, 64
    x = torch.empty((n, hw, c), dtype=BF, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    for i in range(n):
        x[i] = torch.randn((hw, c), generator=g, device=DEV)
    dy = x.flip(0)
    x.requires_grad_()
    y = pkg.group_norm_act(x, 32, slope=0.2)
    (dx,) = torch.autograd.grad(y, x, dy)
    for i in (0, n - 1):
        xi = x[i:i + 1].detach().clone().requires_grad_()
        yi = pkg.group_norm_act(xi, 32, slope=0.2)
        (di,) = torch.autograd.grad(yi, xi, dy[i:i + 1].clone())
        assert (yi.float() - y[i:i + 1].float()).abs().max() <= 2 * ut(BF) * yi.float().abs().max()
        assert (di.float() - dx[i:i + 1].float()).abs().max() <= 2 * ut(BF) * di.float().abs().max()
