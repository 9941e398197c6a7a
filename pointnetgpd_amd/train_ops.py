"""Operators for training grasp networks that are not the PointNet trunks: tensor-level functions with gradients.

* ``group_norm_act``       — group norm with an activation over channels-last point features.  The trunks' BatchNorm
                             (PointNetGPD/model/pointnet.py:29-31,144-147) needs two samples a rank and keeps statistics of
                             its replica; this one's are of each sample alone.
* ``linear_cross_entropy`` — the loss of a linear classifier of any width, F.nll_loss(F.log_softmax(F.linear(...)))
                             (main_1v.py:73-74, pointnet.py:193-194), without its logits ever being kept: codebooks of
                             grasps, one class for each point of a scene.

CUDA tensors run the HIP kernels of libpngpd (a missing library raises), CPU tensors the same formulas in ATen operations.
The gradients are those of the formulas; they are not differentiable again.
"""
import ctypes

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


# ------------------------------------------------------------------------------------------------ linear cross entropy
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _lce_call(entry, a, ref, backward):
    """One C call on ``ref``'s device and current stream with a workspace of its own."""
    lib, dev = _lib.load(), ref.device
    ws = _bytes(dev, lib.pngpd_lce_workspace_bytes(ctypes.addressof(a), backward))
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    with _lib.device_guard(dev):
        _lib.check(getattr(lib, entry)(ctypes.addressof(a), torch.cuda.current_stream(dev).cuda_stream), entry)


class LinearCrossEntropyFn(torch.autograd.Function):
    """x (T,D), w (V,D), target (T) -> loss (T) or (); T, V, D > 0, channels adjacent."""

    @staticmethod
    def forward(ctx, x, w, bias, target, reduction, ignore_index, smoothing):
        dev, f32 = x.device, torch.float32
        T, D = x.shape
        bias = bias.detach().contiguous() if bias is not None else None
        stat, kept = torch.empty(T, 2, device=dev, dtype=f32), torch.empty((), device=dev, dtype=f32)
        loss = torch.empty((T,) if reduction == 0 else (), device=dev, dtype=f32)
        n = _lib.load().pngpd_lce_rows_ints(T)
        rows = torch.empty(n, device=dev, dtype=torch.int32) if n else None
        ctx.scalars = (reduction, ignore_index, smoothing)
        ctx.has = (bias is not None, rows is not None)
        ctx.save_for_backward(x, w, target, stat, kept, *(t for t in (bias, rows) if t is not None))
        a = LinearCrossEntropyFn._args(ctx.scalars, x, w, bias, target, stat, kept, rows)
        a.loss = loss.data_ptr()
        _lce_call("pngpd_lce_fwd", a, x, 0)
        return loss

    @staticmethod
    def _args(scalars, x, w, bias, target, stat, kept, rows):
        a = _lib.LceArgs()
        a.rows = None if rows is None else rows.data_ptr()
        a.x, a.w, a.target, a.stat, a.kept = (t.data_ptr() for t in (x, w, target, stat, kept))
        a.bias = None if bias is None else bias.data_ptr()
        (a.T, a.D), a.V = x.shape, w.shape[0]
        a.ldx, a.ldw = (t.stride(0) if t.shape[0] > 1 else t.shape[1] for t in (x, w))
        a.dtype = DTYPES[x.dtype]
        a.bias_dtype = a.dtype if bias is None else DTYPES[bias.dtype]
        a.reduction, a.ignore_index, a.smoothing = scalars
        return a

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        x, w, target, stat, kept, *more = ctx.saved_tensors
        bias = more.pop(0) if ctx.has[0] else None
        rows = more.pop(0) if ctx.has[1] else None
        need = ctx.needs_input_grad
        dloss = dloss.float().contiguous()
        dx = torch.empty(x.shape, device=x.device, dtype=x.dtype) if need[0] else None
        dw = torch.empty(w.shape, device=x.device, dtype=w.dtype) if need[1] else None
        db = torch.empty_like(bias) if bias is not None and need[2] else None
        a = LinearCrossEntropyFn._args(ctx.scalars, x, w, bias, target, stat, kept, rows)
        a.dloss = dloss.data_ptr()
        a.dx, a.dw, a.db = (None if t is None else t.data_ptr() for t in (dx, dw, db))
        _lce_call("pngpd_lce_bwd", a, x, 1)
        return dx, dw, db, None, None, None, None


def linear_cross_entropy(x, weight, target, bias=None, reduction="mean", ignore_index=-100, label_smoothing=0.0):
    """``F.cross_entropy(F.linear(x, weight, bias), target, ...)`` without the logits: x (..., D), weight (V, D), target
    (...) int64, bias (V) or None.  The forward pass reduces the logits tile by tile, the backward pass computes them again
    a piece of the classes at a time, so memory grows with the rows and not with rows x classes.

    Returns float32: a scalar for ``reduction`` "mean" (over the rows whose target is not ``ignore_index``; NaN if there is
    none, with zero gradients) or "sum", target's shape for "none".  Ignored rows have loss 0 and no gradient, whatever
    their x holds.  ``label_smoothing`` in [0, 1] as in ``F.cross_entropy``.  A target outside [0, V) gives a NaN loss
    and NaN gradients (there is no host check: it would wait for the device).  x and weight of one type, float32 (exact
    fp32 products), bfloat16 or float16 (fp32 accumulation; the logits' gradient is rounded once to that type before its
    two products); bias of the same type or float32.  A bias of -inf takes a class out.  Rows with adjacent channels are
    read in place where they start at 16-byte addresses, others through a copy."""
    if not (isinstance(x, torch.Tensor) and isinstance(weight, torch.Tensor)) or x.dim() < 1 or weight.dim() != 2:
        raise RuntimeError("linear_cross_entropy: x must have shape (..., D) and weight (V, D)")
    V, D = weight.shape
    if x.shape[-1] != D or tuple(target.shape) != tuple(x.shape[:-1]):
        raise RuntimeError(f"linear_cross_entropy: x {tuple(x.shape)}, weight {tuple(weight.shape)} and target "
                           f"{tuple(target.shape)} do not fit: expected (..., D), (V, D), (...)")
    if target.dtype != torch.int64:
        raise RuntimeError(f"linear_cross_entropy: target must be int64, got {target.dtype}")
    if bias is not None and tuple(bias.shape) != (V,):
        raise RuntimeError(f"linear_cross_entropy: bias must have shape ({V},), got {tuple(bias.shape)}")
    if reduction not in REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    label_smoothing, ignore_index = float(label_smoothing), int(ignore_index)
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"linear_cross_entropy: label_smoothing must be in [0, 1], got {label_smoothing}")
    if V < 1 or D < 1:
        raise RuntimeError("linear_cross_entropy: no classes or no channels")
    _same_device(x, "linear_cross_entropy", ("weight", weight), ("target", target), ("bias", bias))
    if x.dtype != weight.dtype:
        raise RuntimeError(f"linear_cross_entropy: x is {x.dtype}, weight {weight.dtype}")
    if not x.is_cuda or not target.numel():
        F = torch.nn.functional
        f32 = x.dtype in (torch.bfloat16, torch.float16)
        z = F.linear(*((t.float() if t is not None and f32 else t) for t in (x, weight, bias)))
        loss = F.cross_entropy(z.reshape(-1, V), target.reshape(-1), ignore_index=ignore_index, reduction=reduction,
                               label_smoothing=label_smoothing)
        return loss.reshape(target.shape) if reduction == "none" else loss
    _dtype(x, "linear_cross_entropy: x")
    if bias is not None and bias.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"linear_cross_entropy: bias must be of x's type ({x.dtype}) or float32, got {bias.dtype}")
    if max(V, D, target.numel()) >= 2 ** 31 - 256:
        raise RuntimeError("linear_cross_entropy: more than 2^31 - 257 rows, classes or channels")
    rows = [v if (v.shape[1] == 1 or v.stride(1) == 1) and (v.shape[0] == 1 or v.stride(0) >= v.shape[1]) else v.contiguous()
            for v in (x.reshape(-1, D), weight)]
    loss = LinearCrossEntropyFn.apply(rows[0], rows[1], bias, target.reshape(-1).contiguous(), REDUCTIONS[reduction],
                                      ignore_index, label_smoothing)
    return loss.reshape(target.shape) if reduction == "none" else loss
