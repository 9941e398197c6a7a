"""Operators for training grasp networks that are not the PointNet trunks: tensor-level functions with gradients.

* ``group_norm_act``       — group norm with an activation over channels-last point features.  The trunks' BatchNorm
                             (PointNetGPD/model/pointnet.py:29-31,144-147) needs two samples a rank and keeps statistics of
                             its replica; this one's are of each sample alone.

CUDA tensors run the HIP kernels of libpngpd (a missing library raises), CPU tensors the same formulas in ATen operations.
The gradients are those of the formulas; they are not differentiable again.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _call

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # PNGPD_F32, PNGPD_BF16, PNGPD_F16


def _dtype(t, name):
    if t.dtype not in DTYPES:
        raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return DTYPES[t.dtype]


def _bytes(dev, n):
    """Workspace of one call.  Taken from the caching allocator each time, never kept: two captured graphs must not
    share one, and the allocator orders its reuse by stream."""
    return torch.empty(max(int(n), 1), device=dev, dtype=torch.uint8)


def _same_device(ref, name, *others):
    for n, t in others:
        if t is not None and t.device != ref.device:
            raise RuntimeError(f"{name}: {n} is on {t.device}, the input on {ref.device}")


# --------------------------------------------------------------------------------------------- group norm + activation
class GroupNormActFn(torch.autograd.Function):
    """(B,N,C) with adjacent channels -> (B,N,C) contiguous."""

    @staticmethod
    def forward(ctx, x, w, b, groups, eps, act):
        B, N, C = x.shape
        y = torch.empty(B, N, C, device=x.device, dtype=x.dtype)
        ctx.groups, ctx.eps, ctx.act, ctx.has = groups, eps, act, (w is not None, b is not None)
        stats = torch.empty(B, groups, 2, device=x.device, dtype=torch.float64)
        w, b = (t.detach().contiguous() if t is not None else None for t in (w, b))
        if x.numel():
            dt = DTYPES[x.dtype]
            wdt = next((DTYPES[t.dtype] for t in (w, b) if t is not None), dt)
            nbytes = _lib.load().pngpd_group_norm_workspace_bytes(B, N, C, groups, dt, 0)
            _call("pngpd_group_norm_fwd", x, x.data_ptr(), dt, B, N, C, x.stride(0), x.stride(1), groups, w, b, wdt, eps,
                  act, y, stats, _bytes(x.device, nbytes), nbytes)
        ctx.save_for_backward(x, stats, *(t for t in (w, b) if t is not None))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, stats, *wb = ctx.saved_tensors
        w = wb.pop(0) if ctx.has[0] else None
        b = wb.pop(0) if ctx.has[1] else None
        B, N, C = x.shape
        need = ctx.needs_input_grad
        dx = torch.empty(B, N, C, device=x.device, dtype=x.dtype) if need[0] else None
        dw = torch.empty_like(w) if need[1] else None
        db = torch.empty_like(b) if need[2] else None
        if not x.numel():
            for t in (dw, db):
                if t is not None:
                    t.zero_()
            return dx, dw, db, None, None, None
        dt = DTYPES[x.dtype]
        wdt = next((DTYPES[t.dtype] for t in (w, b) if t is not None), dt)
        nbytes = _lib.load().pngpd_group_norm_workspace_bytes(B, N, C, ctx.groups, dt, 1)
        _call("pngpd_group_norm_bwd", x, x.data_ptr(), dt, B, N, C, x.stride(0), x.stride(1), ctx.groups, w, b, wdt,
              ctx.eps, ctx.act, stats, dy.contiguous(), dx, dw, db, _bytes(x.device, nbytes), nbytes)
        return dx, dw, db, None, None, None


def _group_norm_act_aten(x, groups, w, b, eps, act):
    v = x.float() if x.dtype in (torch.bfloat16, torch.float16) else x
    B, N, C = v.shape
    v = v.reshape(B, N, groups, C // groups)
    var, mean = torch.var_mean(v, (1, 3), correction=0, keepdim=True)
    z = ((v - mean) * torch.rsqrt(var + eps)).reshape(B, N, C)
    z = z if w is None else z * w.to(z.dtype)
    z = z if b is None else z + b.to(z.dtype)
    F = torch.nn.functional
    return {"none": lambda t: t, "relu": F.relu, "silu": F.silu, "gelu": F.gelu}[act](z).to(x.dtype)


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none"):
    """``act(group_norm(x))`` of channels-last features: x (B, ..., C), every sample's C channels in ``num_groups`` equal
    groups, mean and biased variance over a group's channels and all the positions between the first and the last
    dimension; weight / bias (C), each optional, of x's type or float32.  ``act``: "none", "relu", "silu" or "gelu" (the
    exact one, z * Phi(z)).  Returns a contiguous tensor of x's shape and type; statistics and arithmetic are float32 or
    wider.  Channels adjacent in memory are read in place with any strides of the samples and positions (positions that
    collapse into one stride); anything else is copied first."""
    if not isinstance(x, torch.Tensor) or x.dim() < 2:
        raise RuntimeError("group_norm_act: x must be a tensor of shape (B, ..., C)")
    if act not in ACTIVATIONS:
        raise ValueError(f"group_norm_act: act must be one of {sorted(ACTIVATIONS)}, got {act!r}")
    C, groups, eps = x.shape[-1], int(num_groups), float(eps)
    if groups < 1 or C < 1 or C % groups:
        raise ValueError(f"group_norm_act: {C} channels do not divide into {num_groups} groups")
    if not eps >= 0.0:
        raise ValueError(f"group_norm_act: eps must not be negative, got {eps}")
    for n, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (C,):
            raise RuntimeError(f"group_norm_act: {n} must have shape ({C},), got {tuple(t.shape)}")
    _same_device(x, "group_norm_act", ("weight", weight), ("bias", bias))
    N = 1
    for n in x.shape[1:-1]:
        N *= n
    v = x.reshape(x.shape[0], N, C)
    if not x.is_cuda:
        return _group_norm_act_aten(v, groups, weight, bias, eps, act).reshape(x.shape)
    _dtype(x, "group_norm_act: x")
    for n, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"group_norm_act: {n} must be of x's type ({x.dtype}) or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("group_norm_act: weight and bias must be of one type")
    if max(v.shape[:2]) >= 2 ** 31:
        raise RuntimeError("group_norm_act: more than 2^31 - 1 samples or positions")
    if v.stride(2) != 1 and C > 1:
        v = v.contiguous()
    return GroupNormActFn.apply(v, weight, bias, groups, eps, ACTIVATIONS[act]).view(x.shape)
