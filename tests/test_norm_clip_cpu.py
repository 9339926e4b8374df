"""CPU: what group norm and gradient clipping refuse -- in Python and at the C entry points (which check before they launch)."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused(pkg):
    x = torch.zeros(2, 4, 4, 8)
    with pytest.raises(pkg._lib.M355Error):
        pkg.group_norm_act(x, 2)
    with pytest.raises(pkg._lib.M355Error):
        pkg.group_norm_act([1.0], 2)
    with pytest.raises(pkg._lib.M355Error):
        pkg.GroupNormAct2d(32)(x)
    for f in (pkg.grad_norm, lambda t: pkg.clip_grads_(t, 1.0)):
        with pytest.raises(pkg._lib.M355Error):
            f([x])
        with pytest.raises(ValueError):
            f([])
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(pkg.clip_grad_norm_([p], 1.0)) == 0.0 and float(pkg.clip_grad_norm_([], 1.0)) == 0.0
    with pytest.raises(ValueError):
        pkg.clip_grad_norm_([p], -1.0)
    p.grad = torch.ones(3)
    with pytest.raises(pkg._lib.M355Error):
        pkg.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError):
        pkg.GroupNorm2d(48, 32)
    with pytest.raises(ValueError):
        pkg.GroupNormAct2d(48, 0)


FAKE = ctypes.c_void_p(0x10000)     # device pointers are only looked at


def _desc(pkg, n=2, hw=16, c=8, g=2, dtype=2, act=0, res_w=0, stride=0, per_sample=0):
    return ctypes.byref(pkg._lib.GnDesc(n, hw, stride, c, g, dtype, act, res_w, per_sample, 1e-5, 0.2, 1.0, 0.0))


def _fwd(pkg, res=None, x=FAKE, y=ctypes.c_void_p(0x20000), ws=FAKE, **kw):
    return pkg._lib.lib().m355_group_norm_fwd(_desc(pkg, **kw), x, None, None, res, y, FAKE, ws, None)


def _bwd(pkg, dres=None, dy=FAKE, dx=ctypes.c_void_p(0x20000), **kw):
    return pkg._lib.lib().m355_group_norm_bwd(_desc(pkg, **kw), dy, ctypes.c_void_p(0x30000), None, None, FAKE, dx, None, None, dres, FAKE, None)


def test_group_norm_entry_points_check_their_arguments(pkg):
    L = pkg._lib.lib()
    for kw in (dict(n=-1), dict(hw=-1), dict(c=0), dict(g=0), dict(g=3), dict(dtype=3), dict(dtype=-1), dict(act=2), dict(n=1 << 31),
               dict(hw=1 << 40), dict(c=1 << 21, g=1 << 20), dict(stride=-1), dict(res_w=3), dict(res_w=-2),
               dict(res_w=16)):                                        # (one row: no half height)
        assert _fwd(pkg, res=FAKE, **kw) == -1 and L.m355_last_error()
        assert _bwd(pkg, dres=FAKE, **kw) == -1 and L.m355_last_error()
        assert L.m355_group_norm_ws_bytes(_desc(pkg, **kw), 1) == 0
    assert L.m355_group_norm_fwd(None, FAKE, None, None, None, FAKE, FAKE, FAKE, None) == -1
    assert _fwd(pkg, x=None) == -1 and b"null" in L.m355_last_error()
    assert _fwd(pkg, ws=None) == -1 and _fwd(pkg, y=FAKE) == -1
    assert _fwd(pkg, res=None, res_w=4) == -1
    assert _bwd(pkg, dres=FAKE, res_w=0) == -1
    assert _bwd(pkg, dy=None) == -1 and _bwd(pkg, dx=FAKE) == -1
    # a group wider than a workgroup: 257 odd channels, 4096 of a vector of eight
    for c, g, dtype in ((257, 1, 2), (771, 3, 0), (4096, 1, 2), (2056, 1, 2)):
        assert _fwd(pkg, c=c, g=g, dtype=dtype) == -2 and _bwd(pkg, c=c, g=g, dtype=dtype) == -2
    # nothing to do is no error, and launches nothing
    assert _fwd(pkg, n=0) == 0 and _fwd(pkg, hw=0) == 0 and _bwd(pkg, n=0) == 0 and _bwd(pkg, hw=0) == 0
    small, back = L.m355_group_norm_ws_bytes(_desc(pkg), 0), L.m355_group_norm_ws_bytes(_desc(pkg), 1)
    assert small >= 2 * 2 * 8 and back >= small + 2 * 2 * 8 * 4


def _clip(L, ins, outs, numel, dtype, scale=1.0, max_norm=1.0, norm=FAKE, ws=FAKE):
    n = len(numel)
    arr = (lambda v: None if v is None else (ctypes.c_void_p * n)(*v))
    return L.m355_grad_clip(arr(ins), arr(outs), (ctypes.c_longlong * n)(*numel), (ctypes.c_int * n)(*dtype), n, scale, max_norm, norm, ws, None)


def test_clip_entry_point_checks_its_arguments(pkg):
    L = pkg._lib.lib()
    a, b = 0x100000, 0x200000
    ok = dict(numel=[100, 100], dtype=[0, 0])
    for kw in (dict(scale=float("nan")), dict(scale=float("inf")), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(norm=None),
               dict(ws=None)):
        assert _clip(L, [a, b], [a, b], **ok, **kw) == -1 and L.m355_last_error()
    assert _clip(L, [a, b], [a, b], [100, -1], [0, 0]) == -1 and _clip(L, [a, b], [a, b], [100, 1 << 41], [0, 0]) == -1
    assert _clip(L, [a, b], [a, b], [100, 100], [0, 3]) == -1
    assert _clip(L, [a, None], [a, b], **ok) == -1 and _clip(L, [a, b], [a, None], **ok) == -1
    assert _clip(L, [a, b + 2], [a, b + 2], **ok) == -1 and _clip(L, [a, b], [a, b + 1], [100, 100], [0, 1]) == -1
    # memory that two tensors share: 100 floats are 400 bytes
    shared = [([a, a], [a, a]), ([a, a + 396], [a, a + 396]), ([a, b], [a, a + 4]), ([a, b], [b + 0x1000, a]), ([a, b], [a + 8, b]),
              ([a, b], [b, a]), ([a, b], [b + 0x1000, b + 0x1000])]
    for ins, outs in shared:
        assert _clip(L, ins, outs, **ok) == -1 and b"shares memory" in L.m355_last_error(), (ins, outs)
    assert L.m355_grad_clip_ws_bytes(-1) == 0
    assert L.m355_grad_clip_ws_bytes(0) == L.m355_grad_clip_ws_bytes(112) == 8 * 1024 and L.m355_grad_clip_ws_bytes(113) == 2 * 8 * 1024


def test_networks_take_group_norm(pkg):
    """construction, parameter names and refusals of the norm switches (no GPU: nothing runs)"""
    import argparse
    import importlib
    gan = importlib.import_module("2dimageto3dmodel_amd.gan")
    rec = importlib.import_module("2dimageto3dmodel_amd.reconstruction")
    kw = dict(conditional_class=True, conditional_color=False, conditional_text=False, n_classes=[5], texture_resolution=128, mask_output=True,
              num_discriminators=2, texture_only=False, text_embedding_dim=256)
    args = argparse.Namespace(norm_g="group", norm_d="group", **kw)
    G, D = gan.Generator(args, 64), gan.MultiScaleDiscriminator(args, 4)
    assert isinstance(G.blk1.norm1.norm, pkg.GroupNorm2d) and G.blk6.norm2.norm.num_groups == 32
    inst = gan.MultiScaleDiscriminator(argparse.Namespace(norm_g="batch", norm_d="instance", **kw), 4)
    assert list(D.state_dict()) == list(inst.state_dict())          # instance norm's names: weight, bias
    with pytest.raises(ValueError):
        gan.Generator(argparse.Namespace(norm_g="group", norm_d="none", norm_groups=48, **kw), 64)
    a, b = rec.ReconstructionNetwork(norm="group", norm_groups=16), rec.ReconstructionNetwork()
    assert [k for k, _ in a.named_parameters()] == [k for k, _ in b.named_parameters()]
    assert a.bn1e.num_groups == 16 and not [k for k in a.state_dict() if "running" in k]
    with pytest.raises(ValueError):
        rec.ReconstructionNetwork(norm="layer")
