"""Group norm + activation (train_ops.group_norm_act) against its formulas in 64 bits.

Bounds, elementwise, with u = 2^-24 (float32) and U = finfo(type).eps / 2 (one rounding to the output's type):
  z   = xh w + b in float32: the mean is rounded once (|mean| u), x - mean, the products and the sum once each, rstd once:
        ez = u (6 (|xh w| + |b|) + 2 |mean| rstd |w|)
  act : exp's argument carries |z| u, the hardware's exp and reciprocal 2^-23 each, Phi 1.5e-7 / 2 (the published bound of
        the polynomial): e_act = 2^-21 (|z| + z^2) for the value, 2^-20 (1 + |z| + z^2) for the slope; relu and none: 0
  y   : 1.2 ez + e_act + U |y|                                                  (slopes of the activations are below 1.2)
  dz  : |dy| (e_slope + 1.2 ez); relu's and none's slopes are exact                            (second derivatives below 1)
  sums: n terms one after the other in float32, n <= rows of a thread + 16: n u sum |.|
  dx  = rstd (w dz - S1 - xh S2): the parts' errors, 4 roundings of them, U |dx|
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
ACTS = ("none", "relu", "silu", "gelu")


def value_and_slope(z, act):
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        s = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * s, s + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return z, torch.ones_like(z)


def reference(x, dy, w, b, groups, act, eps=1e-5):
    """-> outputs and elementwise bounds of their errors (the output's own rounding left out)."""
    B, N, C = x.shape
    k = C // groups
    one, zero = torch.ones(C, device=x.device, dtype=torch.double), torch.zeros(C, device=x.device, dtype=torch.double)
    w, b = (one if w is None else w.double()), (zero if b is None else b.double())
    per_c = lambda t: t.repeat_interleave(k, 1).unsqueeze(1)                        # (B,G) -> (B,1,C)
    grp = lambda t: per_c(t.view(B, N, groups, k).sum((1, 3)) / (N * k))            # mean over the group, at every channel
    x, dy = x.double(), dy.double()
    mean = grp(x)
    var = grp((x - mean) ** 2)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    z = xh * w + b
    y, slope = value_and_slope(z, act)
    ez = U32 * (6 * ((xh * w).abs() + b.abs()) + 2 * mean.abs() * rstd * w.abs())
    smooth = act in ("silu", "gelu")
    e_act = 2.0 ** -21 * (z.abs() + z * z) if smooth else 0 * z
    e_slope = 2.0 ** -20 * (1 + z.abs() + z * z) + 1.2 * ez if smooth else 0 * z
    dz = dy * slope
    edz = dy.abs() * e_slope
    exh = U32 * (3 * xh.abs() + 2 * mean.abs() * rstd)
    n = N / 4 + 32
    S1, S2 = grp(w * dz), grp(w * dz * xh)
    eS1 = grp(w.abs() * (edz + n * U32 * dz.abs()))
    eS2 = grp(w.abs() * ((edz + n * U32 * dz.abs()) * xh.abs() + dz.abs() * exh))
    dx = rstd * (w * dz - S1 - xh * S2)
    edx = rstd * (w.abs() * edz + eS1 + xh.abs() * eS2 + exh * S2.abs()
                  + 4 * U32 * ((w * dz).abs() + S1.abs() + (xh * S2).abs()))
    db, dw = dz.sum((0, 1)), (dz * xh).sum((0, 1))
    edb = (edz + (n + 2) * U32 * dz.abs()).sum((0, 1))
    edw = ((edz + (n + 2) * U32 * dz.abs()) * xh.abs() + dz.abs() * exh).sum((0, 1))
    return dict(y=(y, 1.2 * ez + e_act), dx=(dx, edx), dw=(dw, edw), db=(db, edb))


def check(got, want, bound, what):
    assert got.shape == want.shape, what
    t = torch.finfo(got.dtype)
    tiny = t.smallest_normal * t.eps                                     # half a step of the subnormals is below this
    limit = bound + t.eps / 2 * (want.abs() + bound) + tiny
    off = (got.double() - want).abs()
    bad = ~(off <= limit)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, worst {(off / limit).nan_to_num(9e9).max().item():.3g} of the bound"


def run(x, w, b, groups, act, dy):
    from pointnetgpd_amd.train_ops import group_norm_act
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(*leaves[:1], groups, *leaves[1:], act=act)
    have = [t for t in leaves if t is not None]
    return dict(zip(["y"] + [n for n, t in zip(("dx", "dw", "db"), leaves) if t is not None],
                    [y.detach(), *torch.autograd.grad(y, have, dy)]))


def data(shape, dtype, seed, shift=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    B, N, C = shape
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = (r(B, N, C) + shift * r(C)).to(dtype)
    return x, (1 + 0.3 * r(C)).to(dtype), (0.3 * r(C)).to(dtype), r(B, N, C).to(dtype)


def compare(x, w, b, groups, act, dy):
    got = run(x, w, b, groups, act, dy)
    want = reference(x, dy, w, b, groups, act)
    for k, v in got.items():
        check(v, *want[k], k)
    return got


# (B, N, C, groups): one value; one row; narrow, odd and straddling groups; rows past a thread's; groups too wide or too
# long for one workgroup; a batch past 65535
SHAPES = [(1, 1, 1, 1), (2, 1, 8, 8), (3, 7, 12, 3), (2, 500, 64, 8), (4, 33, 226, 2), (2, 1000, 96, 32), (7, 1030, 6, 2),
          (2, 2049, 128, 32), (64, 75, 128, 16), (300, 2, 1040, 2), (1, 5000, 40, 5), (2, 9000, 33, 3), (1, 50000, 17, 1),
          (3, 260, 1024, 1), (70000, 1, 16, 4), (1, 20000, 256, 8), (2, 4097, 5, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("i", range(len(SHAPES)), ids=[str(s) for s in SHAPES])
def test_shapes(i, dtype):
    *shape, groups = SHAPES[i]
    x, w, b, dy = data(shape, dtype, i)
    compare(x, w, b, groups, ACTS[(i + 2) % 4], dy)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("shape", [(3, 50, 24, 4), (2, 3000, 136, 1)])
def test_activations(act, shape):
    for dtype in (torch.float32, torch.float16):
        x, w, b, dy = data(shape[:3], dtype, 5)
        compare(x, 4 * w, b, shape[3], act, dy)            # z out to where the exponentials under- and overflow


def test_relu_gradient_next_to_zero():
    """Slopes are settled in 64 bits: over six million values none takes the other side (float32 would flip some)."""
    x, w, b, dy = data((64, 750, 128), torch.float32, 3)
    compare(x, w, b, 16, "relu", dy)


@pytest.mark.parametrize("affine", ["none", "weight", "bias", "float32"])
def test_affine_parts(affine):
    x, w, b, dy = data((2, 70, 48), torch.bfloat16, 9)
    w, b = dict(none=(None, None), weight=(w, None), bias=(None, b), float32=(w.float(), b.float()))[affine]
    compare(x, w, b, 6, "silu", dy)


def test_strides():
    from pointnetgpd_amd.train_ops import group_norm_act
    g = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn(40, 6, 100, generator=g, device="cuda")
    w, b = torch.rand(33, device="cuda") + 0.5, torch.rand(33, device="cuda")
    for x in (big[:, :, 7:40], big[:, :, 7:40].transpose(0, 1), big[::3, 1:4, 60:93], big.permute(0, 2, 1)[:, :33, :][..., :6],
              big[:1, :, :33].expand(5, 6, 33)):
        C = x.shape[2]
        got = group_norm_act(x, 3, w[:C], b[:C], act="gelu")
        assert got.is_contiguous() and torch.equal(got, group_norm_act(x.contiguous(), 3, w[:C], b[:C], act="gelu"))
        compare(x, w[:C], b[:C], 3, "gelu", torch.randn(x.shape, generator=g, device="cuda"))
    x = big[..., :32].reshape(4, 10, 6, 32)                                    # positions of more than one dimension
    assert torch.equal(group_norm_act(x, 4).view(4, 60, 32), group_norm_act(x.reshape(4, 60, 32), 4))
    y = group_norm_act(big[0, :, :32], 4)                                      # (B, C): one position a sample
    assert torch.equal(y, group_norm_act(big[0, :, None, :32].contiguous(), 4)[:, 0])


def test_large_mean():
    """A mean 3000 times the spread: float32's E[x^2] - mean^2 would hold no digit of the variance."""
    x, w, b, dy = data((2, 600, 64), torch.float32, 2, shift=0.0)
    compare(x + 3000, w, b, 8, "none", dy)
    compare((x + 3000).repeat(1, 20, 1), w, b, 1, "silu", dy.repeat(1, 20, 1))


@pytest.mark.parametrize("shape,groups", [((2, 40, 32), 4), ((1, 30000, 64), 2)])
def test_nan_stays_in_its_group(shape, groups):
    x, w, b, dy = data(shape, torch.float32, 4)
    clean = run(x, w, b, groups, "gelu", dy)
    k = shape[2] // groups
    bad = x.clone()
    bad[0, 5, 1] = float("nan")
    bad[0, 6, 2] = float("inf")
    got = run(bad, w, b, groups, "gelu", dy)
    for n in ("y", "dx"):
        assert got[n][0, :, :k].isnan().all() and torch.equal(got[n][0, :, k:], clean[n][0, :, k:]), n
        assert torch.equal(got[n][1:], clean[n][1:])
    for n in ("dw", "db"):
        assert got[n][:k].isnan().all() and torch.equal(got[n][k:], clean[n][k:]), n


@pytest.mark.parametrize("shape,groups", [((922, 2, 8), 8), ((50, 1, 24), 12), ((300, 3, 40), 40)])
def test_groups_of_few_values(shape, groups):
    """Two or three values a group, some of them nearly equal: far from the mean's size, near each other."""
    x, w, b, dy = data(shape, torch.float32, 17)
    compare(x, w, b, groups, "none", dy)
    got = run(x, w, b, groups, "none", dy)
    want = reference(x, dy, w, b, groups, "none")
    # the differences x - mean are exact but for their own rounding, whatever the mean: 2^-21 covers eight of them
    assert (got["dw"].double() - want["dw"][0]).norm() <= 2.0 ** -21 * want["dw"][0].norm()
    assert (got["y"].double() - want["y"][0]).norm() <= 2.0 ** -21 * want["y"][0].norm()


def test_constant_group():
    """No spread: xh is 0, y is act(b), and the gradients are finite."""
    x = torch.full((2, 30, 16), 3.0, device="cuda")
    _, w, b, dy = data((2, 30, 16), torch.float32, 6)
    compare(x, w, b, 2, "relu", dy)


def test_empty():
    from pointnetgpd_amd.train_ops import group_norm_act
    w = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 5, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = group_norm_act(x, 2, w)
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert y.shape == x.shape and dx.shape == x.shape and not dw.any()


def test_gradient_against_differences():
    """<dx, v> + <dw, vw> + <db, vb> = df along (v, vw, vb), by central differences of the formulas in 64 bits."""
    x, w, b, dy = data((2, 90, 24), torch.float32, 7)
    g = torch.Generator(device="cuda").manual_seed(8)
    v, vw, vb = (torch.randn(t.shape, generator=g, device="cuda") for t in (x, w, b))
    for act in ("none", "silu", "gelu"):
        got = run(x, w, b, 4, act, dy)
        f = lambda h: (reference(x.double() + h * v, dy, w.double() + h * vw, b.double() + h * vb, 4, act)["y"][0] * dy).sum()
        h = 1e-5                                  # truncation h^2, rounding 1e-16 / h of sums of ~1e3: both below 1e-8
        want = (f(h) - f(-h)).item() / (2 * h)
        have = sum((got[k].double() * t).sum() for k, t in (("dx", v), ("dw", vw), ("db", vb))).item()
        size = sum((got[k].double() * t).abs().sum() for k, t in (("dx", v), ("dw", vw), ("db", vb))).item()
        assert abs(have - want) <= 2.0 ** -18 * size, (act, have, want)     # 64 roundings of every term


@pytest.mark.parametrize("shape,groups", [((8, 100, 64), 8), ((1, 30000, 64), 2)])
def test_same_bits_streams_and_graph(shape, groups):
    x, w, b, dy = data(shape, torch.bfloat16, 11)
    first = run(x, w, b, groups, "gelu", dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(x, w, b, groups, "gelu", dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first[k], other[k]) for k in first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(x, w, b, groups, "gelu", dy)
    for k in range(4):
        x.copy_(data(shape, torch.bfloat16, 20 + k)[0])
        graph.replay()
        eager = run(x, w, b, groups, "gelu", dy)
        torch.cuda.synchronize()
        assert all(torch.equal(held[n], eager[n]) for n in eager), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_small_values(dtype):
    """Features under the type's normal range (float16: 6e-5), where eps is what scales them."""
    x, w, b, dy = data((3, 200, 64), dtype, 18)
    compare((x.float() * 1e-5 + 3e-5).to(dtype), w, b, 8, "none", dy)
    compare((x.float() * 1e-5 + 3e-5).repeat(1, 40, 1).to(dtype), w, b, 1, "none", dy.repeat(1, 40, 1))


@pytest.mark.parametrize("shape,groups", [((4500, 1, 40), 5), ((8209, 3, 24), 2), ((5003, 1, 2000), 250), ((33001, 2, 6), 6),
                                          ((2100, 1, 5000), 1), ((9001, 1, 7), 1), ((4097, 40, 8), 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_samples_of_few_rows(shape, groups, dtype):
    """Samples share a workgroup, the last one has fewer, and a sample's NaN stays in it."""
    x, w, b, dy = data(shape, dtype, 31, shift=0.3)
    got = compare(x, w, b, groups, "silu", dy)
    at = shape[0] - 2
    x[at, 0, -1] = float("nan")
    bad = run(x, w, b, groups, "silu", dy)
    k = shape[2] // groups
    for name in ("y", "dx"):
        assert bad[name][at, :, -k:].isnan().all(), name
        rest = torch.ones(shape, dtype=torch.bool, device="cuda")
        rest[at, :, -k:] = False
        assert torch.equal(bad[name][rest], got[name][rest]), name
    for name in ("dw", "db"):
        assert bad[name][-k:].isnan().all() and torch.equal(bad[name][:-k], got[name][:-k]), name


# (B, N, C, groups): one row of groups of eight, four and two; several; a slab; cut along the rows
CLOSE = [(50, 1, 64, 8), (30, 1, 32, 8), (40, 1, 16, 8), (6, 10, 64, 4), (9, 3, 40, 5), (2, 500, 64, 8), (1, 20000, 64, 8),
         (9000, 2, 16, 2)]


@pytest.mark.parametrize("dtype,base", [(torch.float16, 1500.0), (torch.float16, 30.0), (torch.bfloat16, 200.0)])
@pytest.mark.parametrize("i", range(len(CLOSE)), ids=[str(s) for s in CLOSE])
def test_large_mean_of_16_bits(i, dtype, base):
    """A spread of one or a few units in the last place: the sums of squares have to hold every bit of them."""
    *shape, groups = CLOSE[i]
    x, w, b, dy = data(shape, torch.float32, 40 + i, shift=0.0)
    unit = base * torch.finfo(dtype).eps
    for spread in (1.0, 4.0):
        compare((base + spread * unit * x).to(dtype), w.to(dtype), b.to(dtype), groups, "none", dy.to(dtype))


@pytest.mark.parametrize("dtype,low,high", [(torch.float16, 2046.0, 2047.0), (torch.float16, 2047.0, 2050.0),
                                            (torch.bfloat16, 254.0, 255.0), (torch.bfloat16, 255.0, 258.0)])
@pytest.mark.parametrize("i", range(len(CLOSE)), ids=[str(s) for s in CLOSE])
def test_two_neighbouring_values(i, dtype, low, high):
    """Groups of two adjacent values of the type, also of two across a power of two; one odd one among equal ones in each
    fourth sample."""
    *shape, groups = CLOSE[i]
    x, w, b, dy = data(shape, dtype, 60 + i)
    pick = x > 0
    pick[::4] = False
    pick[::4, 0, ::shape[2] // groups] = True
    compare(torch.where(pick, high, low).to(dtype), w, b, groups, "silu", dy)


@pytest.mark.parametrize("size", [1e25, 1e-25])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,groups", [((3, 70, 48), 6), ((1, 20000, 64), 8), ((9000, 2, 16), 2)])
def test_spreads_whose_squares_leave_float32(shape, groups, dtype, size):
    """eps = 0: statistics of features of any size, and gradients of the inverse size."""
    from pointnetgpd_amd.train_ops import group_norm_act
    x, w, b, dy = data(shape, torch.float32, 80)
    x, w, b, dy = ((size * x).to(dtype), w.to(dtype), b.to(dtype), dy.to(dtype))
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(leaves[0], groups, *leaves[1:], eps=0.0, act="silu")
    got = dict(zip(("y", "dx", "dw", "db"), (y.detach(), *torch.autograd.grad(y, leaves, dy))))
    want = reference(x, dy, w, b, groups, "silu", eps=0.0)
    for k, v in got.items():
        check(v, *want[k], k)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_activations_relative_to_their_tails(act):
    """w = 0 makes z = b exactly and db = dy slope(z): values and slopes out to |z| = 12 with bounds that follow them.
    silu: the exponential's argument carries 2 |z| u, the exponential and the reciprocal 2^-23 each, products and sums one u
    each.  gelu: the published polynomial's own error there, in 64 bits, and of p(t) exp(-z^2/2): 2 z^2 u of the argument,
    2^-23 of the exponential and of the reciprocal, whose error the polynomial multiplies by its condition (below 8)."""
    C = 28_001
    z = torch.linspace(-12, 12, C, device="cuda")
    x = torch.randn(1, 1, C, generator=torch.Generator(device="cuda").manual_seed(90), device="cuda")
    dy = torch.linspace(0.5, 2.0, C, device="cuda").flip(0).view(1, 1, C)
    got = run(x, torch.zeros_like(z), z, 1, act, dy)
    z, dy = z.double(), dy.double().view(C)
    if act == "silu":
        y, slope = value_and_slope(z, act)
        s = torch.sigmoid(z)
        ey = U32 * (2 * z.abs() + 16) * y.abs()
        es = U32 * (2 * z.abs() + 16) * s * (1 + z.abs())
    else:
        e, v = torch.exp(-0.5 * z * z), z.abs() * math.sqrt(0.5)
        phi = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        y, slope = z * phi, phi + z * e / math.sqrt(2 * math.pi)
        t = 1 / (1 + 0.3275911 * v)
        poly = t * (0.254829592 + t * (-0.284496736 + t * (1.421413741 + t * (-1.453152027 + t * 1.061405429))))
        method = 0.5 * (torch.erfc(v) - poly * e).abs()
        assert method.max() <= 0.75e-7                                     # the published bound of it
        k = U32 * (2 * z * z + 64)
        tail = 0.5 * poly * e                                              # (above zero 1 - tail: one more u)
        ey = z.abs() * (method + k * tail + U32 * phi) + U32 * y.abs()
        es = method + k * (tail + z.abs() * e) + 2 * U32 * phi
    check(got["y"].view(C), y, ey, "y")
    check(got["db"], dy * slope, dy * es, "db")
    deep = z < -4                                                          # so a zero or a wrong sign would not pass
    assert (ey[deep] < 0.2 * y[deep].abs()).all() and (es[deep] < 0.2 * slope[deep].abs()).all()
