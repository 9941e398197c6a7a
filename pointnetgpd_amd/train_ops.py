"""Operators for training grasp networks that are not the PointNet trunks: tensor-level functions with gradients.

* ``group_norm_act``       — group norm with an activation over channels-last point features.  The trunks' BatchNorm
                             (PointNetGPD/model/pointnet.py:29-31,144-147) needs two samples a rank and keeps statistics of
                             its replica; this one's are of each sample alone.
* ``linear_cross_entropy`` — the loss of a linear classifier of any width, F.nll_loss(F.log_softmax(F.linear(...)))
                             (main_1v.py:73-74, pointnet.py:193-194), without all rows x classes of logits in memory (what is
                             kept of them, and how not to: ``keep_logits``): codebooks of grasps, one class for each point of
                             a scene.

CUDA tensors run the HIP kernels of libpngpd (a missing library raises), CPU tensors the same formulas in ATen operations.
The gradients are those of the formulas; they are not differentiable again, and forward-mode derivatives raise on CUDA.
"""
import ctypes

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # PNGPD_F32, PNGPD_BF16, PNGPD_F16


def _dtype(t, name):
    if t.dtype not in DTYPES:
        raise RuntimeError(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return DTYPES[t.dtype]


def _bytes(dev, n):
    """Workspace of one call.  Taken from the caching allocator each time, never kept: two captured graphs must not
    share one, and the allocator orders its reuse by stream."""
    return torch.empty(n, device=dev, dtype=torch.uint8)


def _flat(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _same_device(ref, name, *others):
    index = ref.get_device()
    for n, t in others:
        if t is not None and t.get_device() != index:
            raise RuntimeError(f"{name}: {n} is on {t.device}, the input on {ref.device}")


# --------------------------------------------------------------------------------------------- group norm + activation
# The backward passes run on autograd's own thread, often on a far core: the same Python costs up to four times there what it
# costs in the forward pass.  So what a backward call needs besides addresses and strides is settled in the forward pass, and
# its node enters no context that it does not need (forward + backward of 64 rows against 6500 classes 175 -> 155 us with the
# thread on a far core, 102 -> 93 on a near one; a small group norm 134 -> 125 and 67 -> 65; without the context that
# call_on spares, 147 and 118 on a far core).
def _once(backward):
    """``once_differentiable(backward)`` where the call itself may be differentiated (create_graph), else ``backward``; an
    upstream gradient with a tangent is refused."""
    guarded = once_differentiable(backward)

    def call(ctx, g):
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(g).tangent is not None:
            raise NotImplementedError("the gradients of this operator have no jvp (forward-mode derivatives)")
        return (guarded if torch.is_grad_enabled() else backward)(ctx, g)
    return call


def _wants_node(*tensors):
    """Whether the call has to go through its autograd node: an input requires grad, or carries a tangent perhaps (forward-mode
    derivatives are not implemented, which the node says; past it they would vanish), or a trace is being recorded (of a node it
    holds the call, otherwise the empty outputs and no kernel)."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
            or forward_ad._current_level >= 0 or torch._C._get_tracing_state() is not None)


def _adjacent(x):
    """(B,N,C) with adjacent channels, as the kernels read it: x itself, or a copy."""
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _gn_call(fn, entry, dev, dims, nbytes, x, w, b, *ptrs):
    """One C call; ``dims``: see ``_gn_dims``; ``ptrs``: the pointers between act and the workspace."""
    dt, B, N, C, groups, wdt, eps, act = dims
    ws = _bytes(dev, nbytes) if nbytes else None      # held until the launches are queued: another thread may allocate meanwhile
    sB, sN, _ = x.stride()
    code = _lib.call_on(dev, fn, x.data_ptr(), dt, B, N, C, sB, sN, groups, None if w is None else w.data_ptr(),
                        None if b is None else b.data_ptr(), wdt, eps, act, *ptrs, None if ws is None else ws.data_ptr(), nbytes)
    if code:
        _lib.check(code, entry)


def _gn_dims(x, w, b, groups, eps, act):
    dt = DTYPES[x.dtype]
    return (dt, *x.shape, groups, DTYPES[w.dtype] if w is not None else DTYPES[b.dtype] if b is not None else dt, eps, act)


def _gn_workspace(dims, backward):
    dt, B, N, C, groups, _, _, act = dims
    return _lib.load().pngpd_group_norm_workspace_bytes(B, N, C, groups, dt, act, backward)


def _group_norm_fwd(x, w, b, dims):
    """(B,N,C) with adjacent channels -> y (B,N,C) contiguous, stats (B,G,2) float64."""
    dev = x.device
    y = torch.empty(x.shape, device=dev, dtype=x.dtype)
    stats = torch.empty((x.shape[0], dims[4], 2), device=dev, dtype=torch.float64)
    if x.numel():
        _gn_call(_lib.load().pngpd_group_norm_fwd, "group_norm_fwd", dev, dims, _gn_workspace(dims, 0), x, w, b, y.data_ptr(),
                 stats.data_ptr())
    return y, stats


def _group_norm_bwd(ctx, dy):
    x, w, b, stats = ctx.saved_tensors
    dims, nbytes, dev = ctx.call
    x, w, b, stats = _adjacent(x), _flat(w), _flat(b), _flat(stats)            # (a saved-tensor hook may have moved them)
    need = ctx.needs_input_grad
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    dw = torch.empty_like(w) if need[1] else None
    db = torch.empty_like(b) if need[2] else None
    if nbytes is not None:
        dy = _flat(dy)
        _gn_call(_lib.load().pngpd_group_norm_bwd, "group_norm_bwd", dev, dims, nbytes, x, w, b, stats.data_ptr(), dy.data_ptr(),
                 None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(),
                 None if db is None else db.data_ptr())
    else:
        for t in (dw, db):
            if t is not None:
                t.zero_()
    return dx, dw, db, None


class GroupNormActFn(torch.autograd.Function):
    """x (B,N,C) with adjacent channels, w, b (C) contiguous or None, ``_gn_dims``."""

    @staticmethod
    def forward(ctx, x, w, b, dims):
        y, stats = _group_norm_fwd(x, w, b, dims)
        ctx.call = (dims, _gn_workspace(dims, 1) if x.numel() else None, x.device)
        ctx.save_for_backward(x, w, b, stats)
        return y

    backward = staticmethod(_once(_group_norm_bwd))


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
    v = x if x.dim() == 3 else x.reshape(x.shape[0], N, C)
    if not x.is_cuda:
        return _group_norm_act_aten(v, groups, weight, bias, eps, act).reshape(x.shape)
    _dtype(x, "group_norm_act: x")
    for n, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"group_norm_act: {n} must be of x's type ({x.dtype}) or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("group_norm_act: weight and bias must be of one type")
    if v.shape[0] >= 2 ** 31 or max(N, C) > 2 ** 30:
        raise RuntimeError("group_norm_act: more than 2^31 - 1 samples, 2^30 positions or 2^30 channels")
    v, weight, bias = _adjacent(v), _flat(weight), _flat(bias)
    dims = _gn_dims(v, weight, bias, groups, eps, ACTIVATIONS[act])
    if _wants_node(v, weight, bias):
        y = GroupNormActFn.apply(v, weight, bias, dims)
    else:
        y = _group_norm_fwd(v, weight, bias, dims)[0]
    return y if y.shape == x.shape else y.view(x.shape)


# ------------------------------------------------------------------------------------------------ linear cross entropy
REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _lce_call(fn, entry, a, nbytes, dev):
    """One C call on ``dev`` and its current stream with a workspace of its own."""
    ws = _bytes(dev, nbytes)
    a.workspace, a.workspace_bytes = ws.data_ptr(), nbytes
    code = _lib.call_on(dev, fn, ctypes.addressof(a))
    if code:
        _lib.check(code, entry)


def _rows(v):
    """(rows, D) with adjacent channels, as the kernels read it: v itself, or a copy."""
    return v if (v.shape[1] == 1 or v.stride(1) == 1) and (v.shape[0] == 1 or v.stride(0) >= v.shape[1]) else v.contiguous()


def _where(x, w, bias, target, stat, rows, z):
    """Where tensors lie and how: a descriptor made for them holds as long as this is the same."""
    return (x.data_ptr(), x.stride(), w.data_ptr(), w.stride(), target.data_ptr(), target.stride(), stat.data_ptr(), stat.stride(),
            bias is None or (bias.data_ptr(), bias.stride()), rows is None or (rows.data_ptr(), rows.stride()),
            z is None or (z.data_ptr(), z.stride()))


def _lce_args(scalars, x, w, bias, target, stat, rows, z):
    (T, D), ld = x.shape, [t.stride(0) if t.shape[0] > 1 else t.shape[1] for t in (x, w)]
    dt, at = DTYPES[x.dtype], stat.data_ptr()
    reduction, ignore_index, smoothing = scalars
    return _lib.LceArgs(x=x.data_ptr(), w=w.data_ptr(), bias=None if bias is None else bias.data_ptr(), target=target.data_ptr(),
                        ldx=ld[0], ldw=ld[1], ignore_index=ignore_index, T=T, D=D, V=w.shape[0], dtype=dt,
                        bias_dtype=dt if bias is None else DTYPES[bias.dtype], reduction=reduction, smoothing=smoothing,
                        stat=at, kept=at + 8 * T, rows=None if rows is None else rows.data_ptr(),
                        z=None if z is None else z.data_ptr())


def _lce_fwd(x, w, bias, target, scalars, keep):
    """-> loss, what the backward pass reads (the logits among it where ``keep`` and they are few), the call's arguments."""
    lib, dev, T = _lib.load(), x.device, x.shape[0]
    stat = torch.empty(2 * T + 1, device=dev, dtype=torch.float32)             # (T,2), then the kept rows' number
    n = lib.pngpd_lce_rows_ints(T)
    rows = torch.empty(n, device=dev, dtype=torch.int32) if n else None
    n = lib.pngpd_lce_z_bytes(T, x.shape[1], w.shape[0], DTYPES[x.dtype]) if keep else 0
    z = torch.empty(n // 4, device=dev, dtype=torch.float32) if n else None
    loss = torch.empty((T,) if scalars[0] == 0 else (), device=dev, dtype=torch.float32)
    a = _lce_args(scalars, x, w, bias, target, stat, rows, z)
    a.loss = loss.data_ptr()
    _lce_call(lib.pngpd_lce_fwd, "pngpd_lce_fwd", a, lib.pngpd_lce_workspace_bytes(ctypes.addressof(a), 0), dev)
    return loss, (stat, rows, z), a


def _lce_bwd(ctx, dloss):
    saved = x, w, bias, target, stat, rows, z = ctx.saved_tensors
    made, where, nbytes, dev = ctx.call
    need = ctx.needs_input_grad
    dloss = _flat(dloss)
    if _where(*saved) == where:
        a = _lib.LceArgs.from_buffer_copy(made)                                # a copy: two threads may run one node
    else:                                                                      # saved tensors that a hook has moved
        x, w = _rows(x), _rows(w)
        bias, target, stat, rows, z = (_flat(t) for t in (bias, target, stat, rows, z))
        a = _lce_args(ctx.scalars, x, w, bias, target, stat, rows, z)
        nbytes = _lib.load().pngpd_lce_workspace_bytes(ctypes.addressof(a), 1)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format) if need[0] else None
    dw = torch.empty_like(w, memory_format=torch.contiguous_format) if need[1] else None
    db = torch.empty_like(bias) if need[2] else None
    a.dloss = dloss.data_ptr()
    a.dx, a.dw, a.db = (None if t is None else t.data_ptr() for t in (dx, dw, db))
    _lce_call(_lib.load().pngpd_lce_bwd, "pngpd_lce_bwd", a, nbytes, dev)
    return dx, dw, db, None, None, None


class LinearCrossEntropyFn(torch.autograd.Function):
    """x (T,D), w (V,D), target (T) -> loss (T) or (); T, V, D > 0, channels adjacent."""

    @staticmethod
    def forward(ctx, x, w, bias, target, scalars, keep):
        loss, made, a = _lce_fwd(x, w, bias, target, scalars, keep)
        saved = (x, w, bias, target, *made)
        ctx.scalars = scalars
        ctx.call = (a, _where(*saved), _lib.load().pngpd_lce_workspace_bytes(ctypes.addressof(a), 1), x.device)
        ctx.save_for_backward(*saved)
        return loss

    backward = staticmethod(_once(_lce_bwd))


def linear_cross_entropy(x, weight, target, bias=None, reduction="mean", ignore_index=-100, label_smoothing=0.0,
                         keep_logits=True):
    """``F.cross_entropy(F.linear(x, weight, bias), target, ...)`` without all of the logits: x (..., D), weight (V, D), target
    (...) int64, bias (V) or None.  The forward pass reduces the logits tile by tile, the backward pass computes them again
    a piece of the classes at a time.  Logits that are few are kept in float32 from the forward to the backward pass, since
    reading them is the faster way: up to 1 GB of float32 inputs', up to 256 MB of at most D / 4 rows of 16 bits.
    ``keep_logits=False`` keeps none: then a call holds 16 bytes a row until its backward pass, beside its inputs (or the
    copies that were needed of them).  Workspaces while a call runs: forward 8 bytes (12 with smoothing) for each row and tile
    of 256 classes, smaller tiles where there are few; backward the logits' gradient of a piece (320 MB at most, 1.25 GB where
    less would leave CUs idle, 256 classes where those take more) and copies of x in its type and in float32; both a copy of
    an operand whose rows are not whole 16-byte pieces at 16-byte addresses, forward also of 512 or more rows over 4 GB.

    Returns float32: a scalar for ``reduction`` "mean" (over the rows whose target is not ``ignore_index``; NaN if there is
    none, with zero gradients) or "sum", target's shape for "none".  Ignored rows have loss 0 and no gradient, whatever
    their x holds.  ``label_smoothing`` in [0, 1] as in ``F.cross_entropy``.  A target outside [0, V) gives a NaN loss
    and NaN gradients on the GPU (there is no host check: it would wait for the device), an IndexError on the CPU.  x and
    weight of one type, float32 (exact fp32 products), bfloat16 or float16 (fp32 accumulation; the logits' gradient is
    rounded once to that type before its two products, and not for the bias's); bias of the same type or float32.  float16
    holds that gradient over the largest row weight, so a row whose weight is less than 2^-20 of it loses digits of its
    dx.  A bias of -inf takes a class out.  Rows with adjacent channels are read in place where they start at 16-byte
    addresses, others through a copy."""
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
        x = torch.where((target == ignore_index).unsqueeze(-1), torch.zeros_like(x), x)       # an ignored row holds nothing
        z = F.linear(*((t.float() if t is not None and f32 else t) for t in (x, weight, bias)))
        loss = F.cross_entropy(z.reshape(-1, V), target.reshape(-1), ignore_index=ignore_index, reduction=reduction,
                               label_smoothing=label_smoothing)
        return loss.reshape(target.shape) if reduction == "none" else loss
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("linear_cross_entropy: on CUDA it cannot be recorded by torch.jit.trace")
    _dtype(x, "linear_cross_entropy: x")
    if bias is not None and bias.dtype not in (x.dtype, torch.float32):
        raise RuntimeError(f"linear_cross_entropy: bias must be of x's type ({x.dtype}) or float32, got {bias.dtype}")
    if max(V, target.numel()) >= 2 ** 30 or D > 2 ** 22:
        raise RuntimeError("linear_cross_entropy: more than 2^30 - 1 rows or classes, or 2^22 channels")
    rows, bias = [_rows(x.reshape(-1, D)), _rows(weight)], _flat(bias)
    target_rows, scalars = target.reshape(-1).contiguous(), (REDUCTIONS[reduction], ignore_index, label_smoothing)
    if _wants_node(*rows, bias):
        loss = LinearCrossEntropyFn.apply(*rows, bias, target_rows, scalars, bool(keep_logits))
    else:
        loss = _lce_fwd(*rows, bias, target_rows, scalars, False)[0]
    return loss.reshape(target.shape) if reduction == "none" else loss
