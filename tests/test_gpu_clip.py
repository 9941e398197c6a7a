"""The global gradient norm and clipping (optim.clip_grad_norm_, FlatAdam(max_grad_norm=)) against 64-bit arithmetic.

The norm is summed in float64 and rounded to float32 once: relative error 2^-24 (+ 2^-40 for the sums).  A clipped gradient
carries the rounding of the factor, of the norm in it, of the product and of the store: 3 * 2^-24 + finfo(type).eps / 2."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def make(shapes, dtypes, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps = []
    for i, s in enumerate(shapes):
        t = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.zeros(s, device="cuda", dtype=t))
        p.grad = (scale * torch.randn(s, generator=g, device="cuda")).to(t)
        ps.append(p)
    return ps


def norm64(grads, kind):
    v = torch.cat([g.double().reshape(-1) for g in grads]) if grads else torch.zeros(1)
    return torch.linalg.vector_norm(v, kind).item()


def check_clip(ps, max_norm, kind=2.0):
    from pointnetgpd_amd.optim import clip_grad_norm_
    before = [p.grad.clone() for p in ps]
    want = norm64(before, kind)
    versions = [p.grad._version for p in ps]
    got = clip_grad_norm_(ps, max_norm, kind)
    assert got.dtype == F32 and got.dim() == 0 and got.is_cuda
    assert abs(got.item() - want) <= 1.01 * U * want
    c = min(1.0, max_norm / (want + 1e-6)) if math.isfinite(max_norm) else 1.0
    for p, g, v in zip(ps, before, versions):
        assert p.grad._version > v
        if c == 1.0:
            assert torch.equal(p.grad, g)
        else:
            t = torch.finfo(g.dtype)
            w = g.double() * c
            off = (p.grad.double() - w).abs()
            assert (off <= (3.1 * U + t.eps / 2 * (1 + 4 * U)) * w.abs() + t.smallest_normal * t.eps).all()


RAGGED = [(1,), (3,), (8192,), (8193,), (16384,), (5, 7, 11), (300, 1000), (8191,), (100003,), (2, 2)]


@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=str)
@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
def test_ragged(dtypes, kind):
    check_clip(make(RAGGED, dtypes, 1), 0.37, kind)
    check_clip(make(RAGGED, dtypes, 1), 1e9, kind)                  # nothing to clip: not a bit changes
    check_clip(make(RAGGED, dtypes, 2), math.inf, kind)


def test_many_tensors():
    check_clip(make([(i % 17 + 1, 37) for i in range(700)], (F32, F16), 3), 1.0)


def test_one_large_tensor_and_alone():
    from pointnetgpd_amd.optim import clip_grad_norm_
    check_clip(make([(40_000_001,)], (BF16,), 4), 1.0)
    p = make([(1000,)], (F32,), 5)[0]
    n = clip_grad_norm_(p, 1e-3)                                    # a tensor in place of a list
    assert abs(norm64([p.grad], 2) - 1e-3) < 1e-6 and n > 1


def test_unaligned_views_and_gaps():
    """Gradients at odd addresses, permuted ones, and columns of a wider buffer; what lies between stays."""
    buf = torch.randn(200_001, device="cuda").to(BF16)
    wide = torch.randn(64, 50, device="cuda")
    keep = wide.clone()
    ps = [torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=BF16)) for n in (99_999, 70_000)]
    ps[0].grad, ps[1].grad = buf[1:100_000], buf[100_001:170_001]
    ps += [torch.nn.Parameter(torch.zeros(64, 7, device="cuda")), torch.nn.Parameter(torch.zeros(20, 30, 10, device="cuda"))]
    ps[2].grad = wide[:, 3:10]
    ps[3].grad = torch.randn(30, 10, 20, device="cuda").permute(2, 0, 1)
    tail = buf[[0, 100_000, 170_001, 200_000]].clone()
    check_clip(ps, 2.5)
    assert torch.equal(buf[[0, 100_000, 170_001, 200_000]], tail)
    assert torch.equal(wide[:, :3], keep[:, :3]) and torch.equal(wide[:, 10:], keep[:, 10:])


def test_range_of_the_squares():
    """Gradients whose squares leave float32 at either end."""
    for s in (1e25, 1e-25):
        check_clip(make([(5000,), (77,)], (F32, BF16), 6, scale=s), s)


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
def test_nonfinite(kind):
    from pointnetgpd_amd.optim import clip_grad_norm_
    for bad, norm in ((float("nan"), math.isnan), (float("inf"), math.isinf)):
        ps = make([(100,), (20000,)], (F32,), 7)
        ps[1].grad[12345] = bad
        before = [p.grad.clone() for p in ps]
        with pytest.raises(RuntimeError, match="norm of the gradients"):
            clip_grad_norm_(ps, 1.0, kind, error_if_nonfinite=True)
        assert torch.equal(ps[0].grad, before[0])                   # refused before anything was clipped
        assert norm(clip_grad_norm_(ps, math.inf, kind).item()) and torch.equal(ps[0].grad, before[0])
        assert norm(clip_grad_norm_(ps, 1.0, kind).item())
        ref = [torch.nn.Parameter(torch.zeros_like(p)) for p in ps]
        for r, g in zip(ref, before):
            r.grad = g.clone()
        torch.nn.utils.clip_grad_norm_(ref, 1.0, kind)
        assert all(torch.equal(p.grad.isnan(), r.grad.isnan()) for p, r in zip(ps, ref))


def test_nothing_and_empty():
    from pointnetgpd_amd.optim import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    assert clip_grad_norm_([p], 1.0).item() == 0 and clip_grad_norm_([], 1.0).item() == 0
    q = torch.nn.Parameter(torch.zeros(0, 4, device="cuda"))
    q.grad = torch.zeros(0, 4, device="cuda")
    assert clip_grad_norm_([p, q], 1.0).item() == 0
    p.grad = torch.zeros(3, device="cuda")
    assert clip_grad_norm_([p, q], 1.0).item() == 0 and not p.grad.any()
    p.grad = torch.tensor([3.0, 4.0, 0.0], device="cuda")
    assert clip_grad_norm_(iter([p, q]), 0.0).item() == 5 and not p.grad.any()


def test_refusals():
    from pointnetgpd_amd.optim import FlatAdam, clip_grad_norm_
    ps = make([(10,), (20,)], (F32,), 8)
    before = [p.grad.clone() for p in ps]
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip_grad_norm_(ps, bad)
        with pytest.raises(ValueError):
            FlatAdam([torch.nn.Parameter(torch.zeros(4, device="cuda"))], max_grad_norm=bad)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_(ps, 1.0, 3.0)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(ps + ps[:1], 1.0)
    ps[1].grad = ps[0].grad.new_zeros(1).expand(20)
    with pytest.raises(RuntimeError, match="expanded"):
        clip_grad_norm_(ps, 1.0)
    buf = torch.zeros(30, device="cuda")
    ps[0].grad, ps[1].grad = buf[:10], buf[5:25]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(ps, 1.0)
    q = torch.nn.Parameter(torch.zeros(2, device="cuda", dtype=torch.float64))
    q.grad = torch.zeros(2, device="cuda", dtype=torch.float64)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        clip_grad_norm_([q], 1.0)
    c = torch.nn.Parameter(torch.zeros(2))
    c.grad = torch.ones(2)
    with pytest.raises(RuntimeError, match="more than one device"):
        clip_grad_norm_([c, q], 1.0)
    ps[0].grad, ps[1].grad = before
    assert torch.equal(ps[0].grad, before[0])


def test_same_bits_and_graph():
    from pointnetgpd_amd.optim import clip_grad_norm_
    ps = make(RAGGED, (F32, BF16), 9)
    fresh = [p.grad.clone() for p in ps]
    n0 = clip_grad_norm_(ps, 0.5).clone()
    first = [p.grad.clone() for p in ps]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n1 = clip_grad_norm_(ps, 0.5)
    for k in range(4):
        for p, f in zip(ps, fresh):
            p.grad.copy_(f if k != 2 else f * 3)
        graph.replay()
        torch.cuda.synchronize()
        if k != 2:
            assert torch.equal(n1, n0) and all(torch.equal(p.grad, f) for p, f in zip(ps, first))
        else:
            assert n1 > 2.9 * n0


def adam_pair(max_norm, shapes=((300, 40), (7,), (1000, 33), (5,))):
    from pointnetgpd_amd.optim import FlatAdam
    g = torch.Generator(device="cuda").manual_seed(10)
    base = [torch.randn(s, generator=g, device="cuda") for s in shapes]
    opts = [FlatAdam([torch.nn.Parameter(b.clone()) for b in base], lr=0.01, max_grad_norm=m) for m in (max_norm, None)]
    return opts, g


def close(a, b, steps):
    """The clipped and the plain update of the same gradients.  The plain one has 1 - 0.9f (2.4e-7 off) and 1 - 0.999f
    (1.3e-5 off) for 1 - beta, which enter m and v as they are, and bias corrections 1 - beta^t in float32: 2^-23 of 1
    over 1 - 0.999^t, 1.2e-4 at t = 1, half of it under the root; an update is lr (about 1) at these steps."""
    assert (a.flat_m - b.flat_m).abs().max() <= steps * (2.4e-7 + 8 * U) * b.flat_m.abs().max()
    assert (a.flat_v - b.flat_v).abs().max() <= (1.4e-5 + steps * 8 * U) * b.flat_v.abs().max()
    assert (a.flat_p - b.flat_p).abs().max() <= steps * 0.01 * 2e-4


def test_adam_equals_clip_then_step():
    from pointnetgpd_amd.optim import clip_grad_norm_
    (a, b), g = adam_pair(0.7)
    for k in range(5):
        for pa, pb in zip(a._params, b._params):
            pa.grad.copy_(torch.randn(pa.shape, generator=g, device="cuda"))
            pb.grad.copy_(pa.grad)
        kept = a.flat_g.clone()
        a.step()
        n = clip_grad_norm_(b._params, 0.7)
        b.step()
        assert torch.equal(a.grad_norm, n) and torch.equal(a.flat_g, kept)
        close(a, b, k + 1)


def test_adam_unclipped_step_is_the_plain_one():
    (a, b), g = adam_pair(1e9)
    for k in range(3):
        for pa, pb in zip(a._params, b._params):
            pa.grad.copy_(torch.randn(pa.shape, generator=g, device="cuda"))
            pb.grad.copy_(pa.grad)
        a.step(); b.step()
        close(a, b, k + 1)


def test_adam_against_64_bits():
    """Ten clipped steps, host and device step counts: every state within float32 roundings of the formulas in 64 bits.
    A step rounds m, v, p and the factors about 8 times (8 U of each one's size); the division's 2.5 U and the square
    root's half of v's error go into an update of at most lr (1 + |m| / sqrt v); ten steps add up."""
    from pointnetgpd_amd.optim import FlatAdam
    for capturable in (False, True):
        g = torch.Generator(device="cuda").manual_seed(11)
        ps = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")) for s in ((201, 33), (5,))]
        opt = FlatAdam(ps, lr=0.01, max_grad_norm=0.5, capturable=capturable)
        state = [[p.detach().double().clone(), torch.zeros_like(p).double(), torch.zeros_like(p).double()] for p in ps]
        for t in range(1, 11):
            for p in ps:
                p.grad.copy_(torch.randn(p.shape, generator=g, device="cuda"))
            c = min(1.0, 0.5 / (norm64([p.grad for p in ps], 2) + 1e-6))
            for p, s in zip(ps, state):
                gg = p.grad.double() * c
                s[1] += (gg - s[1]) * (1 - 0.9)
                s[2] += (gg * gg - s[2]) * (1 - 0.999)
                s[0] -= 0.01 / (1 - 0.9 ** t) * s[1] / ((s[2] / (1 - 0.999 ** t)).sqrt() + 1e-8)
            opt.step()
        for p, s in zip(ps, state):
            top = [x.abs().max().item() for x in s]
            assert (p.detach().double() - s[0]).abs().max() <= 10 * 8 * U * (top[0] + 0.05)
            assert (opt.state[p]["exp_avg"].double() - s[1]).abs().max() <= 10 * 8 * U * top[1]
            assert (opt.state[p]["exp_avg_sq"].double() - s[2]).abs().max() <= 10 * 8 * U * top[2]


def test_adam_scaled_gradients():
    """grad_scale and grad_div come before the norm: sums over 8 samples clip as their mean does."""
    (a, b), g = adam_pair(0.3)
    b.max_grad_norm, b.grad_norm = 0.3, torch.zeros((), device="cuda")
    for pa, pb in zip(a._params, b._params):
        pa.grad.copy_(torch.randn(pa.shape, generator=g, device="cuda"))
        pb.grad.copy_(pa.grad * 8)
    a.step()
    b.step(grad_div=torch.tensor(16.0, device="cuda"), grad_scale=2.0)
    assert torch.equal(a.grad_norm, b.grad_norm) and torch.equal(a.flat_p, b.flat_p)


def test_adam_skipped_piece_does_not_count():
    """The stale slice of a fused piece that sat a step out is neither updated nor part of the norm."""
    (a, _), g = adam_pair(0.5)
    for p in a._params:
        p.grad.copy_(torch.randn(p.shape, generator=g, device="cuda"))
    a._grouped[2] = 1
    a._written[0] = 1
    p2 = a._params[2].detach().clone()
    want = norm64([p.grad for i, p in enumerate(a._params) if i != 2], 2)
    a.step()
    assert abs(a.grad_norm.item() - want) <= 1.01 * U * want and torch.equal(a._params[2].detach(), p2)


def test_classifier_step_eager_and_graphed():
    """The whole classifier's step with a clipped update: the captured one follows the eager one, and the clip is active."""
    import copy
    from pointnetgpd_amd.model.pointnet import PointNetCls
    from pointnetgpd_amd.optim import FlatAdam
    from pointnetgpd_amd.train import GraphedTrainStep, loss_backward
    torch.manual_seed(0)
    m0 = PointNetCls(num_points=128, input_chann=3, k=3).cuda().train()
    m1 = copy.deepcopy(m0)
    mk = lambda m, cap: FlatAdam(m.parameters(), lr=torch.tensor(0.002, device="cuda"), capturable=cap, max_grad_norm=0.05)
    o0, o1 = mk(m0, True), mk(m1, True)
    step = GraphedTrainStep(m1, 16, 128, optimizer=o1)
    g = torch.Generator(device="cuda").manual_seed(2)
    for k in range(4):
        x = 0.05 * torch.randn(16, 3, 128, generator=g, device="cuda")
        y = torch.randint(0, 3, (16,), generator=g, device="cuda")
        o0.zero_grad()
        l0, _, _ = m0.forward_loss(x, y)
        loss_backward(l0)
        o0.step()
        l1, _ = step(x, y)
        torch.cuda.synchronize()
        assert torch.equal(l0.detach(), l1) and torch.equal(o0.grad_norm, o1.grad_norm) and o0.grad_norm > 0.05
        assert torch.equal(o0.flat_p, o1.flat_p)


def test_gradients_with_gaps_that_overlap():
    """Views of one buffer as other tensor objects: refused before anything is written; columns that are apart are clipped."""
    from pointnetgpd_amd.optim import clip_grad_norm_
    buf = torch.randn(50, 9, device="cuda")
    want = buf.clone()
    ps = [torch.nn.Parameter(torch.zeros(50, device="cuda")) for _ in range(2)]
    ps[0].grad, ps[1].grad = buf[:, 4], buf[:, 4]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_(ps, 0.1)
    assert torch.equal(buf, want)
    ps[1].grad = buf[:, 5]
    norm = clip_grad_norm_(ps, 0.1)
    exact = want[:, 4:6].double().norm()
    assert abs(norm.double() - exact) <= 2.0 ** -23 * exact
    keep = [0, 1, 2, 3, 6, 7, 8]
    assert torch.equal(buf[:, keep], want[:, keep])
    scaled = want[:, 4:6].double() * (0.1 / (exact + 1e-6))             # the factor and the product are rounded once each, the norm too
    assert ((buf[:, 4:6].double() - scaled).abs() <= 2.0 ** -22 * scaled.abs()).all()


def test_adam_norms_of_several_steps():
    """What a step leaves in grad_norm stays that step's; with capturable there is one place, as a replay needs."""
    from pointnetgpd_amd.optim import FlatAdam
    for capturable in (False, True):
        g = torch.Generator(device="cuda").manual_seed(5)
        p = torch.nn.Parameter(torch.randn(300, generator=g, device="cuda"))
        opt = FlatAdam([p], max_grad_norm=0.5, capturable=capturable)
        held, want = [], []
        for k in range(3):
            p.grad.copy_((k + 1) * torch.randn(300, generator=g, device="cuda"))
            want.append(norm64([p.grad], 2))
            opt.step()
            held.append(opt.grad_norm)
        if capturable:
            assert len({t.data_ptr() for t in held}) == 1
            held, want = held[-1:], want[-1:]
        for n, v in zip(held, want):
            assert abs(n.item() - v) <= 1.01 * U * v
