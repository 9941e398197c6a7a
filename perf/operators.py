"""What the training operators of pointnetgpd_amd are measured on: normalisation, loss and clipped update of a step.

* ``norm``  group norm with an activation over channels-last point features (B, N, C), forward and backward;
* ``loss``  softmax cross entropy of a linear classifier whose logits are never kept, forward and backward;
* ``clip``  the global gradient norm over many tensors and the clipping of them in place;
* ``adam``  the same norm and clipping inside the flat optimizer's update.

``run`` computes them in elementary torch operations, or, where ``own`` is set, through the package's entry points.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
BETA1, BETA2, ADAM_EPS, ADAM_LR, ADAM_STEP = 0.9, 0.999, 1e-8, 0.005, 10      # the training loop's Adam, ten steps in


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one cloud of a robot's scoring loop (N = 500), forward only: latency
        dict(name="norm_one_cloud", op="norm", B=1, N=500, C=64, G=8, dtype="fp32", act="relu", train=False),
        # the training recipe's batch (64 clouds of 750 points) behind the second layer
        dict(name="norm_recipe", op="norm", B=64, N=750, C=128, G=16, dtype="fp32", act="silu", train=True),
        # the benchmark's batch (1024 clouds of 1024 points) behind the second layer
        dict(name="norm_batch", op="norm", B=1024, N=1024, C=128, G=32, dtype="bf16", act="gelu", train=True),
        # one 50,000-point scene at the trunk's last width: one sample over the whole card
        dict(name="norm_scene", op="norm", B=1, N=50000, C=1024, G=32, dtype="fp16", act="silu", train=True),
        # one grasp against a codebook of 6500 grasps (a file's grasps), loss only: latency
        dict(name="loss_one_grasp", op="loss", T=1, D=256, V=6500, dtype="fp32", bias=True, smooth=0.0, ignored=0.0,
             reduction="mean", train=False),
        # the recipe's batch against the same codebook
        dict(name="loss_recipe", op="loss", T=64, D=256, V=6500, dtype="fp32", bias=True, smooth=0.0, ignored=0.0,
             reduction="mean", train=True),
        # pooled features of the benchmark's batch, one class for each point of a scene
        dict(name="loss_scene", op="loss", T=1024, D=1024, V=50000, dtype="bf16", bias=False, smooth=0.1, ignored=0.1,
             reduction="mean", train=True),
        # point features of several clouds against 100,000 candidates, a weight for each row's loss
        dict(name="loss_candidates", op="loss", T=8192, D=1024, V=100000, dtype="bf16", bias=True, smooth=0.0,
             ignored=0.2, reduction="none", train=True),
        # the gradients of the grasp classifier, clipped in place: latency of many small tensors
        dict(name="clip_classifier", op="clip", kind="classifier", scale=1, dtype="fp32", max_norm=1.0),
        # the gradients of a wide model in 16 bits, clipped in place
        dict(name="clip_wide", op="clip", kind="ragged", scale=192, dtype="bf16", max_norm=1.0),
        # the clipped Adam step of the classifier's head
        dict(name="adam_head", op="adam", kind="head", scale=1, dtype="fp32", max_norm=1.0),
        # the clipped Adam step of a wide model
        dict(name="adam_wide", op="adam", kind="ragged", scale=96, dtype="fp32", max_norm=1.0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "loss", "loss", "clip", "adam"))
    if op == "norm":
        G = rng.choice((1, 2, 4, 8, 16, 32))
        C = G * _spread(rng, 1, 1024 // G)
        B = _spread(rng, 1, 1024)
        N = _spread(rng, 1, max(1, min(50000, 64_000_000 // (B * C))))
        return dict(op=op, B=B, N=N, C=C, G=G, dtype=rng.choice(sorted(TYPES)),
                    act=rng.choice(("none", "relu", "silu", "gelu")), train=rng.random() < 0.75)
    if op == "loss":
        T, D = _spread(rng, 1, 8192), _spread(rng, 16, 2048)
        if rng.random() < 0.5:
            D = max(16, D // 16 * 16)
        V = _spread(rng, 2, min(100000, max(2, 200_000_000_000 // (T * D))))
        return dict(op=op, T=T, D=D, V=V, dtype=rng.choice(sorted(TYPES)), bias=rng.random() < 0.5,
                    smooth=rng.choice((0.0, 0.1)), ignored=rng.choice((0.0, 0.3)),
                    reduction=rng.choice(("none", "mean", "sum")), train=rng.random() < 0.75)
    if op == "clip":
        return dict(op=op, kind="ragged", scale=_spread(rng, 1, 128), dtype=rng.choice(sorted(TYPES)),
                    max_norm=rng.choice((0.5, 1.0, 1e6)))          # 1e6: a step whose gradients are not clipped
    return dict(op=op, kind="ragged", scale=_spread(rng, 1, 64), dtype="fp32", max_norm=rng.choice((0.5, 1.0, 1e6)))


def _shapes(case):
    """The tensors of a clip / adam case."""
    if case["kind"] == "classifier":        # two trunks of three layers, two heads of three, with their norms
        trunk = [(64, 3, 1), (64,), (128, 64, 1), (128,), (1024, 128, 1), (1024,), (64,), (64,), (128,), (128,), (1024,),
                 (1024,)]
        return trunk + _head(9) + trunk + _head(2)
    if case["kind"] == "head":
        return _head(2)
    s = case["scale"]                       # a wide model: two large matrices, ragged ones, vectors, a scalar
    return [(1024 * s, 512), (1024, 512 * s + 1), (257 * s, 129), (1000 * s + 7,), (1,), (33, 7, 5), (64 * s,), (3, 3),
            (2048, 31 * s), (5,)]


def _head(k):
    return [(512, 1024), (512,), (256, 512), (256,), (k, 256), (k,), (512,), (512,), (256,), (256,)]


# -------------------------------------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "norm":
        B, N, C = case["B"], case["N"], case["C"]
        # features with a mean and a spread of their own for each channel, as a linear layer leaves them
        x = _normal(g, B, N, C).mul_(0.5 + torch.rand(C, generator=g, device="cuda")).add_(_normal(g, C))
        s.update(x=x.to(t), w=(1 + 0.2 * _normal(g, C)).to(t), b=(0.2 * _normal(g, C)).to(t))
        if case["train"]:
            s["dy"] = _normal(g, B, N, C).to(t)
    elif case["op"] == "loss":
        T, D, V = case["T"], case["D"], case["V"]
        s.update(x=_normal(g, T, D).to(t), w=_normal(g, V, D).mul_(2.0 / math.sqrt(D)).to(t),
                 b=_normal(g, V).to(t) if case["bias"] else None)
        y = torch.randint(0, V, (T,), generator=g, device="cuda")
        drop = torch.rand(T, generator=g, device="cuda") < case["ignored"]
        drop[0] = False                                       # a mean over no row at all is no step anybody takes
        s["y"] = torch.where(drop, torch.full_like(y, -100), y)
        if case["train"] and case["reduction"] == "none":
            s["dloss"] = torch.rand(T, generator=g, device="cuda") / T
    else:
        shapes = _shapes(case)
        s["fresh"] = [_normal(g, *n).mul_(0.01).to(t) for n in shapes]      # what a backward pass leaves
        s["p"] = [torch.nn.Parameter(_normal(g, *n).mul_(0.05).to(t)) for n in shapes]
        if case["op"] == "clip":
            for p in s["p"]:
                p.grad = torch.empty_like(p)
        else:
            s["m"] = [_normal(g, *n).mul_(0.005) for n in shapes]
            s["v"] = [_normal(g, *n).mul_(0.01).square_() for n in shapes]
            s["step"] = ADAM_STEP
            if own:                                           # the optimizer that a training program keeps
                from pointnetgpd_amd.optim import FlatAdam
                o = s["opt"] = FlatAdam(s["p"], lr=ADAM_LR, betas=(BETA1, BETA2), eps=ADAM_EPS,
                                        max_grad_norm=case["max_norm"])
                o.load_state_dict(dict(state={i: dict(step=torch.tensor(float(ADAM_STEP)), exp_avg=m, exp_avg_sq=v)
                                              for i, (m, v) in enumerate(zip(s["m"], s["v"]))}, param_groups=[]))
                torch._foreach_copy_([p.grad for p in s["p"]], s["fresh"])
                s["m"], s["v"] = ([o.state[p][k] for p in s["p"]] for k in ("exp_avg", "exp_avg_sq"))
    return s


# ------------------------------------------------------------------------------------------------- the package's calls
def _own(s, case):
    if case["op"] == "norm":
        from pointnetgpd_amd.train_ops import group_norm_act
        x, w, b = (v.detach().requires_grad_(case["train"]) for v in (s["x"], s["w"], s["b"]))
        y = group_norm_act(x, case["G"], w, b, act=case["act"])
        if not case["train"]:
            return dict(y=y)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"])
        return dict(y=y.detach(), dx=dx, dw=dw, db=db)
    if case["op"] == "loss":
        from pointnetgpd_amd.train_ops import linear_cross_entropy
        leaves = [v.detach().requires_grad_(case["train"]) for v in (s["x"], s["w"], s["b"]) if v is not None]
        loss = linear_cross_entropy(leaves[0], leaves[1], s["y"], bias=leaves[2] if case["bias"] else None,
                                    reduction=case["reduction"], label_smoothing=case["smooth"])
        if not case["train"]:
            return dict(loss=loss)
        grads = torch.autograd.grad(loss, leaves, s.get("dloss"))
        return dict(zip(("loss", "dx", "dw", "db"), (loss.detach(),) + grads))
    if case["op"] == "clip":
        from pointnetgpd_amd.optim import clip_grad_norm_
        torch._foreach_copy_([p.grad for p in s["p"]], s["fresh"])
        norm = clip_grad_norm_(s["p"], case["max_norm"])
        return dict(norm=norm, grads=[p.grad for p in s["p"]])
    s["opt"].step()
    return dict(norm=s["opt"].grad_norm, p=[p.detach() for p in s["p"]], m=s["m"], v=s["v"])


# ------------------------------------------------------------------------------------------------------ the plain form
def _act(z, act):
    """The activation's value and its derivative."""
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "silu":
        e = 1 / (1 + torch.exp(-z))
        return z * e, e * (1 + z * (1 - e))
    if act == "gelu":
        e = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * e, e + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, torch.ones_like(z)


def _norm(s, case):
    B, N, C, G, t = case["B"], case["N"], case["C"], case["G"], s["x"].dtype
    # relu's slope jumps at 0: which side a value next to it is on is settled in 64 bits
    f = torch.float64 if case["act"] == "relu" and case["train"] else torch.float32
    x = s["x"].to(f).view(B, N, G, C // G)
    w, b = s["w"].to(f).view(G, C // G), s["b"].to(f).view(G, C // G)
    count = N * (C // G)
    d = x - x.sum((1, 3), keepdim=True) / count
    r = 1 / torch.sqrt(d.square().sum((1, 3), keepdim=True) / count + 1e-5)
    xh = d * r
    y, slope = _act(xh * w + b, case["act"])
    out = dict(y=y.reshape(B, N, C).to(t))
    if case["train"]:
        dz = s["dy"].to(f).view(B, N, G, C // G) * slope
        e = dz * w
        dx = r * (e - (e.sum((1, 3), keepdim=True) + xh * (e * xh).sum((1, 3), keepdim=True)) / count)
        out.update(dx=dx.reshape(B, N, C).to(t), dw=(dz * xh).sum((0, 1)).reshape(C).to(t),
                   db=dz.sum((0, 1)).reshape(C).to(t))
    return out


def _loss(s, case):
    V, eps, t = case["V"], case["smooth"], s["x"].dtype
    x, w, y = s["x"].float(), s["w"].float(), s["y"]
    z = x @ w.t()
    if case["bias"]:
        z = z + s["b"].float()
    z = z - z.max(1, keepdim=True).values
    e = torch.exp(z)
    total = e.sum(1)
    valid = y >= 0
    at = y.clamp_min(0).unsqueeze(1)
    hit = z.gather(1, at).squeeze(1)
    row = torch.log(total) - (1 - eps) * hit - eps * (z.sum(1) / V)
    row = torch.where(valid, row, torch.zeros_like(row))
    kept = valid.sum()
    loss = row if case["reduction"] == "none" else row.sum() if case["reduction"] == "sum" else row.sum() / kept
    out = dict(loss=loss)
    if case["train"]:
        c = s["dloss"] if case["reduction"] == "none" else torch.ones_like(row) / (kept if case["reduction"] == "mean" else 1)
        c = torch.where(valid, c, torch.zeros_like(c)).unsqueeze(1)
        p = e / total.unsqueeze(1) - eps / V
        p = p.scatter_add(1, at, torch.full_like(hit, eps - 1).unsqueeze(1)) * c
        out.update(dx=(p @ w).to(t), dw=(p.t() @ x).to(t))
        if case["bias"]:
            out["db"] = p.sum(0).to(t)
    return out


def _clip(s, case):
    torch._foreach_copy_([p.grad for p in s["p"]], s["fresh"])
    norm = torch.sqrt(sum(p.grad.float().square().sum() for p in s["p"]))
    c = (case["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    grads = [p.grad.copy_(p.grad.float() * c) for p in s["p"]]
    return dict(norm=norm, grads=grads)


def _adam_one(p, m, v, g, c, t):
    g = g * c
    m.copy_(m + (g - m) * (1 - BETA1))
    v.copy_(v * BETA2 + (1 - BETA2) * g * g)
    p.copy_(p - ADAM_LR / (1 - BETA1 ** t) * (m / (torch.sqrt(v) / math.sqrt(1 - BETA2 ** t) + ADAM_EPS)))
    return p


def _adam(s, case):
    s["step"] += 1
    norm = torch.sqrt(sum(g.square().sum() for g in s["fresh"]))
    c = (case["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    p = [_adam_one(p.detach(), m, v, g, c, s["step"]) for p, m, v, g in zip(s["p"], s["m"], s["v"], s["fresh"])]
    return dict(norm=norm, p=p, m=s["m"], v=s["v"])


def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return dict(norm=_norm, loss=_loss, clip=_clip, adam=_adam)[case["op"]](s, case)


# ------------------------------------------------------------------------------------------------------ cost and truth
def work(case):
    if case["op"] == "norm":
        n, e = case["B"] * case["N"] * case["C"], BYTES[case["dtype"]]
        # forward: x, y; with the backward pass dy and dx too
        return dict(bytes=n * e * (4 if case["train"] else 2) + 4 * case["C"] * e, flops=n * (25 if case["train"] else 10))
    if case["op"] == "loss":
        T, D, V, e = case["T"], case["D"], case["V"], BYTES[case["dtype"]]
        # the product; with the backward pass two more, and as many gradients as inputs
        return dict(bytes=(T * D + V * D) * e * (2 if case["train"] else 1) + 8 * T, flops=2 * T * D * V * (3 if case["train"] else 1))
    n = sum(math.prod(x) for x in _shapes(case))
    if case["op"] == "clip":
        return dict(bytes=2 * n * BYTES[case["dtype"]], flops=3 * n)
    return dict(bytes=7 * n * 4, flops=15 * n)                 # p, m, v read and written, the gradient read


def exact(case, seed):
    """The same from the definitions in 64 bits: autograd through torch's double-precision functions."""
    s = prepare(case, seed)
    F = torch.nn.functional
    if case["op"] == "norm":
        x, w, b = (s[k].double().requires_grad_(case["train"]) for k in ("x", "w", "b"))
        groups = x.unflatten(2, (case["G"], -1))
        var, mean = torch.var_mean(groups, (1, 3), correction=0, keepdim=True)
        z = ((groups - mean) * torch.rsqrt(var + 1e-5)).flatten(2) * w + b
        y = dict(none=lambda v: v.clone(), relu=F.relu, silu=F.silu, gelu=F.gelu)[case["act"]](z)
        if not case["train"]:
            return dict(y=y)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return dict(y=y.detach(), dx=dx, dw=dw, db=db)
    if case["op"] == "loss":
        leaves = [v.double().requires_grad_(case["train"]) for v in (s["x"], s["w"], s["b"]) if v is not None]
        z = F.linear(*leaves)
        loss = F.cross_entropy(z, s["y"], ignore_index=-100, reduction=case["reduction"], label_smoothing=case["smooth"])
        if not case["train"]:
            return dict(loss=loss)
        grads = torch.autograd.grad(loss, leaves, s["dloss"].double() if "dloss" in s else None)
        return dict(zip(("loss", "dx", "dw", "db"), (loss.detach(),) + grads))
    g = [v.double() for v in s["fresh"]]
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(v) for v in g]))
    c = min(1.0, case["max_norm"] / (float(norm) + 1e-6))
    g = [v * c for v in g]
    if case["op"] == "clip":
        return dict(norm=norm, grads=g)
    t = ADAM_STEP + 1
    m = [torch.lerp(g_, m_.double(), BETA1) for g_, m_ in zip(g, s["m"])]
    v = [BETA2 * v_.double() + (1 - BETA2) * g_ ** 2 for g_, v_ in zip(g, s["v"])]
    p = [p_.detach().double() - ADAM_LR * (m_ / (1 - BETA1 ** t)) / ((v_ / (1 - BETA2 ** t)).sqrt() + ADAM_EPS)
         for p_, m_, v_ in zip(s["p"], m, v)]
    return dict(norm=norm, p=p, m=m, v=v)
