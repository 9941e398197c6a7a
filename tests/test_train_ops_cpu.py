"""CPU: refusals of the training operators (before any launch), their C entries' argument checks, and the CPU forms."""
import math

import pytest
import torch

P, INV, WS = 0x1000, 1, 2                                  # dummy non-null "device pointer"; status codes


def test_group_norm_act_refusals():
    from pointnetgpd_amd.train_ops import group_norm_act
    x, w = torch.randn(2, 5, 12), torch.ones(12)
    with pytest.raises(ValueError, match="divide"):
        group_norm_act(x, 5)
    with pytest.raises(ValueError, match="divide"):
        group_norm_act(x, 0)
    with pytest.raises(ValueError, match="act"):
        group_norm_act(x, 3, act="tanh")
    with pytest.raises(ValueError, match="eps"):
        group_norm_act(x, 3, eps=-1.0)
    with pytest.raises(RuntimeError, match="shape"):
        group_norm_act(x[0, 0], 3)
    with pytest.raises(RuntimeError, match="weight"):
        group_norm_act(x, 3, w[:5])
    with pytest.raises(RuntimeError, match="bias"):
        group_norm_act(x, 3, w, torch.ones(1, 12))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_group_norm_act_cpu(act):
    from pointnetgpd_amd.train_ops import group_norm_act
    F = torch.nn.functional
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 7, 12, generator=g, dtype=torch.double, requires_grad=True)
    w = torch.randn(12, generator=g, dtype=torch.double, requires_grad=True)
    b = torch.randn(12, generator=g, dtype=torch.double, requires_grad=True)
    y = group_norm_act(x, 4, w, b, act=act)
    want = dict(none=lambda t: t, relu=F.relu, silu=F.silu, gelu=F.gelu)[act](
        F.group_norm(x.transpose(1, 2), 4, w, b)).transpose(1, 2)
    torch.testing.assert_close(y, want)
    dy = torch.randn(3, 7, 12, generator=g, dtype=torch.double)
    for p, q in zip(torch.autograd.grad(y, (x, w, b), dy), torch.autograd.grad(want, (x, w, b), dy)):
        torch.testing.assert_close(p, q)
    assert group_norm_act(torch.randn(2, 3, 4, 8).bfloat16(), 2, act=act).dtype == torch.bfloat16


def test_clip_grad_norm_cpu():
    from pointnetgpd_amd.optim import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(3))
    assert clip_grad_norm_([p], 1.0).item() == 0
    p.grad = torch.tensor([3.0, 4.0, 0.0])
    assert clip_grad_norm_(p, 1.0).item() == 5 and abs(p.grad.norm().item() - 1) < 1e-5
    for bad in (-0.1, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_([p], 1.0, 0.5)


def test_c_entries_check_their_arguments():
    import ctypes
    from pointnetgpd_amd import _lib
    lib = _lib.load()
    ptr, one = (ctypes.c_void_p * 2)(P, P + 64), (ctypes.c_longlong * 2)(4, 4)
    typ = (ctypes.c_int * 2)(0, 1)
    nb = lib.pngpd_grad_clip_workspace_bytes(2)
    assert nb > 0 and lib.pngpd_grad_clip_workspace_bytes(-1) == 0
    clip = lambda g=ptr, n=one, t=typ, k=2, kind=2, mx=1.0, tot=P, ws=P, b=nb: lib.pngpd_grad_clip(g, n, t, k, kind, mx, tot, ws, b, None)
    assert clip(g=None) == INV and clip(n=None) == INV and clip(k=-1) == INV and clip(tot=None) == INV
    assert clip(kind=3) == INV and clip(kind=-1) == INV and clip(mx=-1.0) == INV and clip(mx=math.nan) == INV
    assert clip(t=(ctypes.c_int * 2)(0, 7)) == INV and clip(n=(ctypes.c_longlong * 2)(4, -1)) == INV
    assert clip(g=(ctypes.c_void_p * 2)(P, None)) == INV and clip(g=(ctypes.c_void_p * 2)(P + 1, P + 64)) == INV
    assert clip(g=(ctypes.c_void_p * 2)(P + 2, P + 64)) == INV                           # float32 at a 2-byte address
    assert clip(g=(ctypes.c_void_p * 2)(P, P + 12)) == clip(g=(ctypes.c_void_p * 2)(P, P)) == 3    # they share memory
    assert clip(ws=None) == WS and clip(b=nb - 1) == WS and clip(ws=P + 4) == WS
    off = (ctypes.c_longlong * 1)(64)
    adam = lambda p=P, o=off, n=one, k=1, mx=1.0, tot=P, ws=P, b=nb, step=1.0: lib.pngpd_adam_flat_clip(
        p, P, P, P, o, n, k, 0.1, None, 0.9, 0.999, 1e-8, step, None, 1.0, None, mx, tot, ws, b, None)
    assert adam(p=None) == INV and adam(p=P + 4) == INV and adam(o=None) == INV and adam(k=0) == INV and adam(step=0.0) == INV
    assert adam(mx=-1.0) == INV and adam(tot=None) == INV and adam(ws=None) == WS and adam(b=8) == WS
    assert adam(o=(ctypes.c_longlong * 1)(2)) == INV and adam(n=(ctypes.c_longlong * 1)(0)) == INV
    fwd = lambda x=P, dt=0, B=2, N=3, C=8, G=2, wdt=0, eps=1e-5, act=1, y=P, st=P, ws=P, b=1 << 20: lib.pngpd_group_norm_fwd(
        x, dt, B, N, C, N * C, C, G, P, P, wdt, eps, act, y, st, ws, b, None)
    bwd = lambda x=P, dt=0, B=2, N=3, C=8, G=2, wdt=0, eps=1e-5, act=1, dy=P, st=P, ws=P, b=1 << 20: lib.pngpd_group_norm_bwd(
        x, dt, B, N, C, N * C, C, G, P, P, wdt, eps, act, st, dy, P, P, P, ws, b, None)
    for f in (fwd, bwd):
        assert f(x=None) == INV and f(dt=3) == INV and f(dt=-1) == INV and f(B=0) == INV and f(N=0) == INV and f(C=0) == INV
        assert f(G=0) == INV and f(G=3) == INV and f(wdt=1) == INV and f(dt=1, wdt=2) == INV and f(eps=-1.0) == INV
        assert f(eps=math.nan) == INV and f(act=4) == INV and f(act=-1) == INV and f(st=None) == INV
    assert fwd(y=None) == INV and bwd(dy=None) == INV and bwd(ws=None) == WS and bwd(b=0) == WS
    assert fwd(N=50000, ws=None) == WS and fwd(N=50000, b=0) == WS
    assert lib.pngpd_group_norm_workspace_bytes(2, 3, 8, 3, 0, 0, 0) == 0
    # every plan's workspace covers what it cuts: positive wherever the backward pass keeps per-sample sums
    for dt in (0, 1, 2):
        for B, N, C, G in [(1, 1, 1, 1), (3, 50000, 17, 1), (1024, 1024, 128, 32), (1, 50000, 1024, 32), (9, 77, 1000, 1)]:
            assert min(lib.pngpd_group_norm_workspace_bytes(B, N, C, G, dt, act, 1) for act in range(4)) >= B * C * 8


def test_command_refuses_a_negative_clip():
    from pointnetgpd_amd import mains
    with pytest.raises(SystemExit, match="clip-grad"):
        mains.run("1v", ["--mode", "train", "--clip-grad", "-1"])
