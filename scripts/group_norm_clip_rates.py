"""Group norm and gradient clipping: (1) the cases of perf/operators.py -- one call among others and the same call replayed from a hipGraph; (2)
where the host time of a small training call goes; (3) a GAN training cycle with batch norm, with group norm and with clipping."""
import importlib, os, sys, time
import torch
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT); sys.path.insert(0, os.path.join(ROOT, "tests"))
pkg = importlib.import_module("2dimageto3dmodel_amd")
gn = importlib.import_module("2dimageto3dmodel_amd.group_norm")
train = importlib.import_module("2dimageto3dmodel_amd.train")
from perf import operators as ops
ops.own = True


def timed(f, n):
    for _ in range(5): f()
    torch.cuda.synchronize()
    best = 1e9
    for _ in range(5):
        t0 = time.perf_counter()
        for _ in range(n): f()
        torch.cuda.synchronize()
        best = min(best, (time.perf_counter() - t0) / n)
    return best * 1e6


print("1. one call (us): among others | replayed from a graph of ten", flush=True)
for case in ops.listed():
    st = ops.prepare(case, 1)
    n = 200 if ops.work(case)["bytes"] < 2e8 else 30
    call = timed(lambda: ops.run(st), n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side): ops.run(st)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(10): keep = ops.run(st)
    print(f"   {case['name']:24s} {call:8.1f} | {timed(g.replay, max(3, n // 10)) / 10:8.1f}", flush=True)
    del st, g, keep
    torch.cuda.empty_cache()

print("2. host time (us) of a training call whose kernels take 11 us (16 x 8 x 4 x 512 bf16, residual)", flush=True)
st = ops.prepare([c for c in ops.listed() if c["name"] == "seed_block_train"][0], 1)
leaves = [st[k] for k in ("x", "weight", "bias", "res")]
args = (st["x"], 32, st["weight"], st["bias"], 1e-5, "lrelu", 0.2, st["res"])
p = [v for v in gn._PLANS.values() if v.shape == tuple(st["x"].shape) and v.res_shape == tuple(st["res"].shape)]


def host(f, n=300):
    for _ in range(20): f()
    best = 1e9
    for _ in range(7):
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        for _ in range(n): f()
        best = min(best, (time.perf_counter() - t0) / n)
    torch.cuda.synchronize()
    return best * 1e6


with torch.no_grad():
    a = host(lambda: pkg.group_norm_act(*args))
    x, w, b = (t.detach() for t in leaves[:3])
    y, stat = gn._forward(x, w, b, st["res"].detach(), p[0])
    body = host(lambda: gn._backward(p[0], (True, True, True, True, False), st["dy"], x, w, b, stat))
    alloc = host(lambda: (torch.empty_like(x), torch.empty_like(w), torch.empty_like(b), torch.empty((p[0].ws_bwd,), dtype=torch.uint8, device=x.device)))
    back = host(lambda: gn._saved(p[0], x, w, b, stat))
f = host(lambda: pkg.group_norm_act(*args))
whole = host(lambda: torch.autograd.grad(pkg.group_norm_act(*args), leaves, st["dy"]))
plain = host(lambda: torch.autograd.grad(leaves[0].add(leaves[3]), [leaves[0], leaves[3]], st["dy"]))
print(f"   forward without autograd {a:.1f}, recorded {f:.1f}; the backward's body {body:.1f}, of it allocations {alloc:.1f}, checking what was saved {back:.1f}")
print(f"   forward and backward {whole:.1f}: the engine's hand-over and bookkeeping {whole - f - body:.1f}; an addition of two tensors, forward and backward, {plain:.1f}", flush=True)
del st, leaves, args, x, w, b, y, stat

print("3. a GAN training cycle (1 generator step, 2 discriminator steps), 256 x 256, ms", flush=True)
import test_gan_modules as T
for B in (64, 16):
    batches = T._cycle_batches(B, 256, seed0=7300)
    for name, norms, kw in (("batch norm (the default)", {}, {}), ("clipping, both networks", {}, dict(max_grad_norm_g=1.0, max_grad_norm_d=1.0)),
                            ("group norm in the generator", dict(norm_g="group"), {}),
                            ("group norm in both", dict(norm_g="group", norm_d="group"), {}), ("batch norm, again", {}, {})):
        torch.manual_seed(733)
        tr = train.GanTrainer(T._trainer_args(texture_resolution=256, **norms), device="cuda:0", mesh_template=None, **kw)
        tr.train()

        def cycle():
            for bt, z in batches: tr.iteration(*bt, noise=z, epoch=0)
            tr.finish_pending()
        for _ in range(4): cycle()
        torch.cuda.synchronize()
        t = []
        for _ in range(12):
            t0 = time.perf_counter(); cycle(); torch.cuda.synchronize(); t.append(time.perf_counter() - t0)
        print(f"   batch {B}: {name:30s} {sorted(t)[len(t) // 2] * 1e3:7.2f}", flush=True)
        del tr
        torch.cuda.empty_cache()
    del batches
