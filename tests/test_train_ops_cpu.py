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


def test_linear_cross_entropy_refusals():
    from pointnetgpd_amd.train_ops import linear_cross_entropy
    x, w, y, b = torch.randn(4, 8), torch.randn(5, 8), torch.tensor([0, 1, 2, 4]), torch.zeros(5)
    with pytest.raises(RuntimeError, match="do not fit"):
        linear_cross_entropy(x, w[:, :7], y)
    with pytest.raises(RuntimeError, match="do not fit"):
        linear_cross_entropy(x, w, y[:3])
    with pytest.raises(RuntimeError, match="shape"):
        linear_cross_entropy(x, w[0], y)
    with pytest.raises(RuntimeError, match="int64"):
        linear_cross_entropy(x, w, y.int())
    with pytest.raises(RuntimeError, match="bias"):
        linear_cross_entropy(x, w, y, bias=b[:4])
    with pytest.raises(RuntimeError, match="float64|float32"):
        linear_cross_entropy(x.double(), w, y)
    with pytest.raises(RuntimeError, match="no classes"):
        linear_cross_entropy(x, w[:0], y)
    with pytest.raises(ValueError, match="reduction"):
        linear_cross_entropy(x, w, y, reduction="batchmean")
    for bad in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="label_smoothing"):
            linear_cross_entropy(x, w, y, label_smoothing=bad)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_linear_cross_entropy_cpu(reduction):
    from pointnetgpd_amd.train_ops import linear_cross_entropy
    F = torch.nn.functional
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 6, 8, generator=g, dtype=torch.double, requires_grad=True)
    w, b = torch.randn(9, 8, generator=g, dtype=torch.double), torch.randn(9, generator=g, dtype=torch.double)
    y = torch.randint(0, 9, (2, 6), generator=g)
    y[0, 2] = -100
    got = linear_cross_entropy(x, w, y, bias=b, reduction=reduction, label_smoothing=0.1)
    want = F.cross_entropy(F.linear(x, w, b).flatten(0, 1), y.flatten(), reduction=reduction, label_smoothing=0.1).reshape(got.shape)
    torch.testing.assert_close(got, want)
    torch.testing.assert_close(torch.autograd.grad(got.sum(), x), torch.autograd.grad(want.sum(), x))
    assert linear_cross_entropy(x.detach().bfloat16(), w.bfloat16(), y).dtype == torch.float32


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


def test_loss_entries_check_their_arguments():
    import ctypes
    from pointnetgpd_amd import _lib
    lib = _lib.load()

    def args(**k):
        f = dict(x=256, w=256, target=256, ldx=8, ldw=8, ignore_index=-100, T=4, D=8, V=5, dtype=0, bias_dtype=0, reduction=1,
                 smoothing=0.0, stat=256, kept=256, loss=256, dloss=256, dx=256, dw=256, workspace=256, workspace_bytes=1 << 24)
        return _lib.LceArgs(**{**f, **k})
    for entry, own in ((lib.pngpd_lce_fwd, "loss"), (lib.pngpd_lce_bwd, "dloss")):
        def call(**k):
            a = args(**k)                                          # (lives until the entry has returned)
            return entry(ctypes.addressof(a), None)
        assert entry(None, None) == INV
        for bad in (dict(x=None), dict(w=None), dict(target=None), dict(T=0), dict(D=0), dict(V=0), dict(T=-1), dict(dtype=3),
                    dict(bias_dtype=1), dict(reduction=3), dict(smoothing=1.5), dict(smoothing=math.nan), dict(ldx=7), dict(ldw=7),
                    dict(stat=None), dict(kept=None), dict(rows=256), dict(T=512), {own: None},
                    dict(z=256), dict(z=264, D=128, ldx=128, ldw=128)):
            assert call(**bad) == INV, bad
        assert call(workspace=None) == WS and call(workspace_bytes=16) == WS and call(workspace=264) == WS
        assert call(D=(1 << 22) + 8, ldx=1 << 23, ldw=1 << 23) == 3
        assert call(T=1 << 30, rows=256) == call(V=1 << 30) == 3
    assert call(db=256) == INV                                                                  # a gradient of no bias
    assert lib.pngpd_lce_rows_ints(511) == 0 and lib.pngpd_lce_rows_ints(512) == 1025
    kept = lib.pngpd_lce_z_bytes                                   # float32 of whole 256 classes; 0: not kept
    assert kept(64, 256, 6500, 0) == 64 * 6656 * 4 and kept(64, 127, 6500, 0) == 0 == kept(8192, 1024, 40000, 0)
    assert kept(64, 256, 127, 0) == 0 and kept(64, 256, 128, 0) == 64 * 256 * 4                  # padding at most doubles them
    assert kept(9, 40, 300, 1) == 9 * 512 * 4 and kept(11, 40, 300, 1) == kept(0, 8, 8, 0) == kept(4, 256, 8, 3) == 0
    assert kept(8192, 1024, 32768, 0) == 1 << 30 and kept(512, 4096, 200000, 2) == 0
    a = args(T=0)
    assert lib.pngpd_lce_workspace_bytes(ctypes.addressof(a), 0) == 0
    # a piece's gradient of the logits is bounded: 256 MB, or 256 classes of all rows
    for T, V, D in ((8192, 100000, 1024), (100000, 100000, 64), (1, 1000000, 64)):
        a = args(T=T, V=V, D=D, ldx=D, ldw=D, dtype=1, bias_dtype=1, rows=256 if T >= 512 else None)
        n = lib.pngpd_lce_workspace_bytes(ctypes.addressof(a), 1)
        assert T * D * 2 < n < (256 << 20) + T * (256 + 128) * 2 + 16 * T * D * 4 + 1024 * 4 * D * 4 + (8 << 20) + 64 * V


def test_command_refuses_a_negative_clip():
    from pointnetgpd_amd import mains
    with pytest.raises(SystemExit, match="clip-grad"):
        mains.run("1v", ["--mode", "train", "--clip-grad", "-1"])


def test_gradients_with_gaps_that_share_memory():
    """The host's check: interleaved columns are apart, overlapping ones and a column of a listed buffer are not."""
    from pointnetgpd_amd.optim import _share_memory
    for dt in (torch.float32, torch.bfloat16):
        buf, other = torch.zeros(40, 12, dtype=dt), torch.zeros(7, dtype=dt)
        assert not _share_memory([buf[:, k] for k in range(12)] + [other])
        assert not _share_memory([buf[:, :5], buf[:, 5:8], buf[:, 9:], buf[3, 8:9], other[:0]])
        assert not _share_memory([buf[::2, :5], buf[1::2, 2:7], buf[::2, 5:], buf[1::2, 7:]])
        assert _share_memory([buf[:, 3], other, buf[:, 3]])
        assert _share_memory([buf[:, :5], buf[:, 4:8]])
        assert _share_memory([buf, buf[7:, 2]])
        assert _share_memory([other, buf[:, 6], buf[11]])
        wide = buf.view(20, 24)[:, ::5].t()                 # columns 0, 5, 10 of the even rows, 3 and 8 of the odd ones
    assert _share_memory([wide, buf[::3, 1:4]]) and not _share_memory([wide, buf[::3, 1:3]])


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_ignored_rows_hold_nothing_cpu(reduction):
    """What an ignored row holds reaches neither the loss nor a gradient; all rows ignored: no gradient."""
    from pointnetgpd_amd.train_ops import linear_cross_entropy
    g = torch.Generator().manual_seed(3)
    x, w, b = torch.randn(2, 6, 8, generator=g), torch.randn(9, 8, generator=g), torch.randn(9, generator=g)
    y = torch.randint(0, 9, (2, 6), generator=g)
    y[0, 2] = y[1, 3] = y[1, 5] = -100

    def run(x, y):
        ls = [t.clone().requires_grad_() for t in (x, w, b)]
        loss = linear_cross_entropy(ls[0], ls[1], y, bias=ls[2], reduction=reduction, label_smoothing=0.1)
        return loss.detach(), *torch.autograd.grad(loss, ls, torch.ones_like(loss))

    bad = x.clone()
    bad[0, 2], bad[1, 3] = math.nan, math.inf
    want, got = run(x, y), run(bad, y)
    assert all(torch.equal(u, v) for u, v in zip(want, got)) and not got[1][y == -100].any()
    loss, *grads = run(bad, torch.full_like(y, -100))
    assert loss.isnan() if reduction == "mean" else not loss.any()
    assert not any(t.any() for t in grads)


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspaces_of_the_loss_are_what_the_header_says(dtype):
    """Forward: 8 bytes a row and tile of classes (12 with smoothing), and the target's logit and the loss of a row, and a copy of
    many rows that span 4 GB; backward: a
    piece's gradient of the logits, x in its type and in float32 (64 MB at least), sums for the bias of a 32nd of the piece."""
    import ctypes
    from pointnetgpd_amd import _lib
    lib, es = _lib.load(), 4 if dtype == 0 else 2
    mb = 1 << 20
    for T in (1, 30, 64, 500, 1024, 5000, 8192, 40_000, 300_000, 1 << 20):
        for V in (2, 100, 3000, 33_000, 100_000):
            for D in (16, 256, 1024, 2048):
                for bias in (None, 256):
                    a = _lib.LceArgs(x=256, w=256, bias=bias, target=256, ldx=D, ldw=D, T=T, D=D, V=V, dtype=dtype, bias_dtype=0,
                                     reduction=1, stat=256, kept=256, rows=256 if T >= 512 else None)
                    for smoothing, size in ((0.0, 8), (0.1, 12)):
                        a.smoothing = smoothing
                        n = lib.pngpd_lce_workspace_bytes(ctypes.addressof(a), 0)
                        most = size * T * (V / 64 + 1) if T * V < 1 << 25 else size * T * (V / 128 + 1)
                        copy = T * D * es if T >= 512 and T * D * es >= 4e9 else 0
                        assert 0 < n <= most + copy + 8 * T + 2048, (T, V, D, n)
                    n = lib.pngpd_lce_workspace_bytes(ctypes.addressof(a), 1)
                    piece = max(1.25 * 1024 * mb, T * (256 + 128) * es)
                    assert n <= (1 + 1 / 16) * piece + T * D * (es + 4) + 4 * T + 72 * mb, (T, V, D, n)
                    if T * min(V, 256) * es <= 256 * mb and V * T * es <= 256 * mb:       # one piece: no more than its logits
                        assert n <= (1 + 1 / 16) * T * (V + 256 + 128) * es + T * D * (es + 4) + 4 * T + 72 * mb, (T, V, D, n)
