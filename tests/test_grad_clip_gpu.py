"""GPU: global gradient norm and clipping (csrc/grad_clip.hip) against the definition in 64 bits.

Tolerances: the norm is a 64-bit sum rounded once to 32 bits (2^-24; 2^-23 leaves room for the 64-bit sum's 1e-12).  A clipped value
is g times a factor rounded to 32 bits, rounded to 32 bits, rounded to its type: u_t + 2 * 2^-24 relative, and half a step among the
subnormal numbers of the type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, H, F = torch.bfloat16, torch.float16, torch.float32


def make(sizes, dtypes, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(scale * torch.randn(s, generator=g)).to(dtypes[i % len(dtypes)]).to(DEV) for i, s in enumerate(sizes)]


def norm64(ts, scale=1.0):
    return abs(scale) * sum(float((t.double().cpu() ** 2).sum()) for t in ts) ** 0.5


def check(got, before, factor):
    want = before.double().cpu() * factor
    tiny = {F: 2.0 ** -150, BF: 2.0 ** -134, H: 2.0 ** -25}[before.dtype]
    tol = (torch.finfo(before.dtype).eps / 2 + 2.0 ** -23) * want.abs() + tiny
    assert ((got.double().cpu() - want).abs() <= tol).all()


LISTS = {
    "one value": ([1], [F]),
    "one tensor": ([4097], [BF]),
    "a network": ([(64, 8, 5, 5), 64, (128, 64, 4, 4), (256, 128, 4, 4), (1, 256, 5, 5), 1, (200, 256)], [F]),
    "mixed, empty, odd": ([0, 1, 2, 3, 5, 7, 8191, 8192, 8193, 0, 16385, (3, 1, 17)], [F, BF, H]),
    "two launches and more": ([1 + 37 * (i % 29) for i in range(250)], [F, H, BF]),
    "large": ([3000001, 5, 1 << 20], [F, BF]),
}


@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("ratio", [0.1, 3.0])
@pytest.mark.parametrize("scale", [1.0, -0.125])
def test_against_the_definition(pkg, name, ratio, scale):
    sizes, dtypes = LISTS[name]
    ts = make(sizes, dtypes, scale=0.3)
    want = norm64(ts, scale)
    max_norm = ratio * want
    factor = scale * min(1.0, max_norm / (want + 1e-6))
    before = [t.clone() for t in ts]
    n = pkg.grad_norm(ts, scale)
    assert n.dtype == F and n.dim() == 0 and n.device == ts[0].device and abs(float(n) - want) <= 2.0 ** -23 * want
    out = [torch.full_like(t, 9.0) for t in ts]
    m = pkg.clip_grads_(ts, max_norm, out=out, scale=scale)
    assert torch.equal(m, n) and all(torch.equal(t, c) for t, c in zip(ts, before))
    for o, c in zip(out, before):
        check(o, c, factor)
    assert torch.equal(pkg.clip_grads_(ts, max_norm, scale=scale), n)
    for t, o in zip(ts, out):
        assert torch.equal(t, o)     # in place: the bits of the other form


def test_thresholds(pkg):
    ts = make([1000, 77], [F, BF])
    before = [t.clone() for t in ts]
    assert abs(float(pkg.clip_grads_(ts, float("inf"))) - norm64(before)) <= 2.0 ** -23 * norm64(before)
    assert all(torch.equal(t, c) for t, c in zip(ts, before))
    pkg.clip_grads_(ts, 0.0)
    assert all(float(t.abs().max()) == 0.0 for t in ts)
    assert float(pkg.clip_grads_(ts, 1.0)) == 0.0                     # a zero gradient: nothing to divide by
    assert all(float(t.abs().max()) == 0.0 for t in ts)


@pytest.mark.parametrize("size", [1e-25, 1e25])
def test_squares_outside_the_32_bit_range(pkg, size):
    ts = [torch.full((1000,), size, device=DEV), torch.full((3,), -size, dtype=BF, device=DEV)]
    want = norm64(ts)
    before = [t.clone() for t in ts]
    assert abs(float(pkg.clip_grads_(ts, 1e20)) - want) <= 2.0 ** -23 * want
    for t, c in zip(ts, before):
        check(t, c, min(1.0, 1e20 / (want + 1e-6)))


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_values_that_are_not_finite_are_not_hidden(pkg, bad):
    """the rule of torch.nn.utils.clip_grad_norm_ on the same list"""
    ts = make([1000, 50], [F])
    ts[0][17] = bad
    ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t.clone()
    want = torch.nn.utils.clip_grad_norm_(ps, 1.0)
    got = pkg.clip_grads_(ts, 1.0)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    for p, t in zip(ps, ts):
        assert torch.equal(p.grad.isnan(), t.isnan()) and torch.equal(p.grad.nan_to_num(), t.nan_to_num())
    if bad == bad:
        t = torch.full((5,), bad, device=DEV)
        pkg.clip_grads_([t], float("inf"))     # an infinite threshold never clips
        assert torch.equal(t, torch.full((5,), bad, device=DEV))


def test_views_strides_and_alignment(pkg):
    g = torch.Generator().manual_seed(1)
    store = torch.randn(40000, generator=g).to(DEV)
    half = store.to(H)
    ts = [store[1:1001], store[1003:9001].view(-1, 31).t(), half[1:30], half[33:20001].view(2, -1, 8).permute(2, 0, 1)]
    before, rest, rest_h = [t.clone() for t in ts], store.clone(), half.clone()
    want = norm64(ts)
    pkg.clip_grads_(ts, 0.5 * want)
    for t, c in zip(ts, before):
        check(t, c, 0.5 * want / (want + 1e-6))
    for s, r, keep in ((store, rest, [(0, 1), (1001, 1003), (9001, 40000)]), (half, rest_h, [(0, 1), (30, 33), (20001, 40000)])):
        for a, b in keep:
            assert torch.equal(s[a:b], r[a:b])     # what lies between the tensors is left as it was
    gaps = store.view(200, 200)[:, :7]
    assert abs(float(pkg.grad_norm(gaps)) - norm64([gaps])) <= 2.0 ** -23 * norm64([gaps])
    assert abs(float(pkg.grad_norm([store[:1].expand(9)])) - norm64([store[:1]]) * 3) <= 2.0 ** -22 * norm64([store[:1]]) * 3
    assert float(pkg.grad_norm([store, store])) == pytest.approx(2 ** 0.5 * norm64([store]), rel=2.0 ** -23)


def test_parameters(pkg):
    lin = torch.nn.Linear(30, 20).to(DEV)
    lin(torch.randn(4, 30, device=DEV)).square().sum().backward()
    lin.register_parameter("unused", torch.nn.Parameter(torch.zeros(3, device=DEV)))
    before = {k: p.grad.clone() for k, p in lin.named_parameters() if p.grad is not None}
    want = norm64(before.values())
    versions = {k: p.grad._version for k, p in lin.named_parameters() if p.grad is not None}
    n = pkg.clip_grad_norm_(lin.parameters(), 0.25 * want)
    assert abs(float(n) - want) <= 2.0 ** -23 * want and lin.unused.grad is None
    for k, c in before.items():
        check(dict(lin.named_parameters())[k].grad, c, 0.25 * want / (want + 1e-6))
        assert dict(lin.named_parameters())[k].grad._version > versions[k]    # autograd knows of the write
    assert float(pkg.clip_grad_norm_([lin.unused], 1.0)) == 0.0
    one = torch.nn.Parameter(torch.zeros(5, device=DEV))
    one.grad = torch.ones(5, device=DEV)
    assert float(pkg.clip_grad_norm_(one, 1.0)) == pytest.approx(5 ** 0.5)


def test_refusals_on_the_device(pkg):
    a, b = torch.ones(100, device=DEV), torch.ones(100, device=DEV)
    for ts in ([a, a], [a, a[10:20]], [a[:60], a[40:]]):
        with pytest.raises(pkg._lib.M355Error, match="shares memory"):
            pkg.clip_grads_(ts, 1.0)
    with pytest.raises(pkg._lib.M355Error, match="shares memory"):
        pkg.clip_grads_([a, b], 1.0, out=[torch.empty_like(a), a])      # one's output over the other's input
    with pytest.raises(pkg._lib.M355Error, match="shares memory"):
        pkg.clip_grads_([a[:50]], 1.0, out=[a[10:60]])                  # its own input, shifted
    with pytest.raises(ValueError):
        pkg.clip_grads_([a.view(10, 10)[:, :3]], 1.0)                   # gaps
    with pytest.raises(ValueError):
        pkg.clip_grads_([a[:1].expand(4)], 1.0)
    for out in ([b.half()], [b.view(10, 10)], [torch.empty(200, device=DEV)[::2]], []):
        with pytest.raises(ValueError):
            pkg.clip_grads_([a], 1.0, out=out)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            pkg.clip_grads_([a], bad)
    with pytest.raises(pkg._lib.M355Error):
        pkg.clip_grads_([a], 1.0, scale=float("inf"))
    with pytest.raises(TypeError):
        pkg.clip_grads_([a.double()], 1.0)
    with pytest.raises(pkg._lib.M355Error):
        pkg.clip_grads_([a, torch.ones(3)], 1.0)
    assert torch.equal(a, torch.ones_like(a))


def test_same_bits_every_run_and_captured(pkg):
    ts = make([(256, 128, 3, 3), 77, (512, 512), 3], [F, BF])
    want = pkg.grad_norm(ts)
    outs = [torch.empty_like(t) for t in ts]
    max_norm = 0.3 * float(want)
    pkg.clip_grads_(ts, max_norm, out=outs)
    keep = [o.clone() for o in outs]
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = pkg.clip_grads_(ts, max_norm, out=outs)
    with torch.cuda.graph(other):
        m = pkg.grad_norm(ts)
    side = torch.cuda.Stream()
    for k in range(4):
        for o in outs:
            o.fill_(5.0)
        n.fill_(-1.0)
        graph.replay()
        other.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s = pkg.grad_norm(ts)
        e = pkg.grad_norm(ts)
        torch.cuda.synchronize()
        assert torch.equal(n, want) and torch.equal(m, want) and torch.equal(s, want) and torch.equal(e, want)
        assert all(torch.equal(o, c) for o, c in zip(outs, keep))
    with torch.no_grad():
        ts[0].mul_(2.0)          # (a replay reads what the tensors hold now)
    graph.replay()
    assert torch.equal(n, pkg.grad_norm(ts)) and not torch.equal(n, want)
