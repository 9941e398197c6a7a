"""``FlatAdam`` — ``torch.optim.Adam`` (the reference's optimizer, PointNetGPD/main_1v.py:61:
``optim.Adam(model.parameters(), lr=args.lr)`` with torch's defaults: betas (0.9, 0.999), eps 1e-8, no weight decay,
no amsgrad) over ONE flat HBM buffer.

The 44 parameters of a ``PointNetCls`` (1,604,363 values, 6.4 MB) are re-pointed at slices of a single buffer; their
gradients and the two Adam moments live in three more.  Consequences:

* ``step()`` is one launch (``pngpd_adam_flat``, 45 MB of streaming traffic) instead of torch's multi-tensor pair;
* the fused training entries (``train.FusedTrunkFn`` / ``FusedHeadFn``) write every parameter gradient straight
  into its slice of the gradient buffer — no per-parameter ``AccumulateGrad``, no ``zero_grad`` fills, and the exactly
  zero conv-bias gradients are written by the kernels;
* data-parallel training all-reduces slices of the SAME buffer (``ddp.GradAverager``): no gather / scatter copies,
  and the trunk gradients can leave while the rest of the backward still runs.

The update is torch's single-tensor Adam in fp32 (torch/optim/adam.py ``_single_tensor_adam``); per-parameter
``state`` entries (``step``, ``exp_avg``, ``exp_avg_sq``) are views of the flat moments, so ``state_dict()`` has the
layout of ``torch.optim.Adam``'s and checkpoints move between the two.
"""
import ctypes
import math
import weakref

import numpy as np
import torch
from torch.utils.weak import WeakIdKeyDictionary

from . import _lib

# parameter -> (gradient view, weakref to the owning FlatAdam, index in its parameter list).  Kept HERE and not as an
# attribute of the Parameter: instance attributes of a Parameter are pickled with it (a whole-module checkpoint would
# carry a second 6.4 MB buffer and come back with an orphaned view), and a registry entry dies with its optimizer.
_GRAD_VIEWS = WeakIdKeyDictionary()


def grad_view(param):
    """The flat-buffer gradient view the fused backward may write for ``param`` in place, or None: only while the
    owning FlatAdam is alive AND ``param.grad`` still IS that view (a ``zero_grad(set_to_none=True)`` of the module, a
    foreign optimizer, or a checkpoint round trip all break the identity and fall back to autograd's accumulation)."""
    e = _GRAD_VIEWS.get(param)
    if e is None:
        return None
    view, owner, _ = e
    if owner() is None or param.grad is not view:
        return None
    return view


class GradGroup:
    """The in-place gradient targets of ONE fused piece (a trunk's 12 parameters, an FC stack's 10): the flat
    optimizer's views in the piece's parameter order, resolved once and re-validated per step by identity checks only
    (the registry look-ups cost ~2 us per parameter — 0.1 ms per step at the reference's batch of 64, where the eager
    loop is host-bound)."""
    __slots__ = ("views", "params", "idx", "owner")

    def __init__(self, views, params, idx, owner):
        self.views, self.params, self.idx, self.owner = views, params, idx, owner

    def valid(self, params):
        if self.owner() is None or len(params) != len(self.params):
            return False
        for p, q, v in zip(params, self.params, self.views):
            if p is not q() or p.grad is not v:
                return False
        return True

    def mark_written(self):
        """Called by the fused backward after it has written the gradient slices of the piece in place."""
        opt = self.owner()
        if opt is None:
            return
        w = opt._written
        for i in self.idx:
            if w[i]:
                raise RuntimeError("FlatAdam: a gradient slice was written twice before step() — the fused backward "
                                   "OVERWRITES gradients (no accumulation over micro-batches or repeated module "
                                   "calls); use model.set_precision(sequencing='passes') or torch.optim.Adam for "
                                   "accumulation")
            w[i] = 1


_GROUPS = {}          # id(first parameter of the piece) -> GradGroup (validated by identity on every use)


def grad_group(params):
    """The GradGroup of a fused piece whose parameters ALL have live flat views (``grad_view``), None if none has one;
    a mix raises (the fused backward writes the whole piece's gradients in place)."""
    g = _GROUPS.get(id(params[0]))
    if g is not None and g.valid(params):
        return g
    entries = [_GRAD_VIEWS.get(p) for p in params]
    live = [e is not None and e[1]() is not None and p.grad is e[0] for e, p in zip(entries, params)]
    if not any(live):
        _GROUPS.pop(id(params[0]), None)
        return None
    if not all(live) or len({id(e[1]()) for e in entries}) != 1:
        raise RuntimeError("optim.FlatAdam must own all parameters of a trunk / FC stack or none of them "
                           "(the fused backward writes the whole piece's gradients in place)")
    g = GradGroup([e[0] for e in entries], [weakref.ref(p) for p in params], [e[2] for e in entries], entries[0][1])
    _GROUPS[id(params[0])] = g
    owner = entries[0][1]()
    for i in g.idx:
        owner._grouped[i] = 1     # these slices are OVERWRITTEN by a fused backward; all others accumulate via autograd
    return g


def ungroup(params):
    """Called by the NON-fused call paths (pass-by-pass sequencing, DEBUG_STASH) at forward time: their gradients
    arrive by autograd ACCUMULATION.  A slice a fused backward used to overwrite (``_grouped``) was exempt from
    ``zero_grad`` and may hold a stale gradient — zero it once and hand it back to the accumulate-and-clear regime."""
    for p in params:
        e = _GRAD_VIEWS.get(p)
        if e is None:
            continue
        view, owner, i = e
        opt = owner()
        if opt is not None and opt._grouped[i]:
            opt._grouped[i] = 0
            if not opt._written[i]:
                view.zero_()
    _GROUPS.pop(id(params[0]), None)


_NORM_KINDS = {2.0: 2, 1.0: 1, math.inf: 0}
_GRAD_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # PNGPD_F32, PNGPD_BF16, PNGPD_F16


def _dense(t):
    """Whether t's elements fill one range of memory, each once (a permutation of a contiguous tensor)."""
    want = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride != want:
            return False
        want *= size
    return True


class _Span:
    """t's addresses for numpy (which does not read them)."""

    def __init__(self, t):
        e = t.element_size()
        self.__array_interface__ = dict(version=3, typestr=f"|V{e}", data=(t.data_ptr(), False), shape=tuple(t.shape),
                                        strides=tuple(st * e for st in t.stride()))


def _share_memory(grads):
    """Whether two of the gradients, some with gaps, have an element in common (those without are compared by the C call)."""
    spans = []
    for g in grads:
        if g.numel():
            reach = sum(st * (n - 1) for st, n in zip(g.stride(), g.shape)) + 1
            spans.append((g.data_ptr(), g.data_ptr() + reach * g.element_size(), _dense(g), g))
    spans.sort(key=lambda s: s[:2])
    near = []                                  # those that reach past the start of the one at hand
    for s in spans:
        near = [o for o in near if o[1] > s[0]]
        for o in near:
            if not (o[2] and s[2]) and np.shares_memory(np.asarray(_Span(o[3])), np.asarray(_Span(s[3]))):
                return True
        near.append(s)
    return False


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """Clip the gradients of ``parameters`` (a tensor or an iterable of tensors; those without ``.grad`` are passed over)
    in place by their global norm, as ``torch.nn.utils.clip_grad_norm_`` does: the norm over every element of all of
    them as if one vector, then ``grad *= min(1, max_norm / (norm + 1e-6))``.  Returns the norm before clipping, a
    float32 scalar on the gradients' device that no host wait has touched.

    Gradients: float32, bfloat16 and float16, in any mix, on one device.  ``norm_type`` 2, 1 or ``math.inf``.  Two
    launches for up to 128 tensors (sums in float64, in a fixed order: the same gradients give the same bits).  A
    gradient reached twice (one parameter listed twice, views of one storage) is refused.  A NaN or infinite norm
    reaches the gradients through the factor, or raises with ``error_if_nonfinite`` (which waits for the device).
    ``max_norm=math.inf`` returns the norm and leaves the gradients alone.
    CPU gradients go to ``torch.nn.utils.clip_grad_norm_``.  With ``FlatAdam(max_grad_norm=...)`` no call is needed:
    the update clips."""
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    max_norm, norm_type = float(max_norm), float(norm_type)
    if not max_norm >= 0.0:
        raise ValueError(f"clip_grad_norm_: max_norm must not be negative, got {max_norm}")
    if norm_type not in _NORM_KINDS:
        raise ValueError(f"clip_grad_norm_: norm_type must be 2, 1 or inf, got {norm_type}")
    grads = [g for g in [p.grad for p in params] if g is not None]
    if not grads:
        return torch.tensor(0.0)
    index = grads[0].get_device()
    if index < 0:
        if any(g.get_device() >= 0 for g in grads):
            raise RuntimeError("clip_grad_norm_: the gradients are on more than one device")
        return torch.nn.utils.clip_grad_norm_(params, max_norm, norm_type, error_if_nonfinite)
    work, ptr, num, typ, gaps = [], [], [], [], False
    for g in grads:
        if g.get_device() != index:
            raise RuntimeError("clip_grad_norm_: the gradients are on more than one device")
        t = _GRAD_TYPES.get(g.dtype)
        if t is None or g.layout is not torch.strided:
            raise RuntimeError("clip_grad_norm_: expected dense float32, bfloat16 or float16 gradients, got "
                               f"{g.dtype}, {g.layout}")
        if not g.is_contiguous():
            if any(st == 0 and k > 1 for st, k in zip(g.stride(), g.shape)):
                raise RuntimeError("clip_grad_norm_: a gradient's elements share memory (an expanded tensor)")
            if not _dense(g):              # gaps (a column of a wider buffer): clipped in a copy and written back
                g = g.contiguous()
                gaps = True
        work.append(g)
        ptr.append(g.data_ptr()); num.append(g.numel()); typ.append(t)
    if gaps and _share_memory(grads):
        raise RuntimeError("clip_grad_norm_: two of the gradients share memory (a parameter listed twice?)")
    n, dev = len(work), grads[0].device
    lib = _lib.load()
    total = torch.empty((), device=dev, dtype=torch.float32)
    nbytes = lib.pngpd_grad_clip_workspace_bytes(n)
    ws = torch.empty(nbytes, device=dev, dtype=torch.uint8)
    ptr, num, typ = (ctypes.c_void_p * n)(*ptr), (ctypes.c_longlong * n)(*num), (ctypes.c_int * n)(*typ)
    stream = _lib.raw_stream(dev)
    with _lib.device_guard(dev):
        for bound in (math.inf, max_norm) if error_if_nonfinite else (max_norm,):       # inf: the norm alone
            code = lib.pngpd_grad_clip(ptr, num, typ, n, _NORM_KINDS[norm_type], bound, total.data_ptr(), ws.data_ptr(),
                                       nbytes, stream)
            if code == 3:                  # PNGPD_ERR_UNSUPPORTED
                raise RuntimeError("clip_grad_norm_: two of the gradients share memory (a parameter listed twice?)")
            _lib.check(code, "grad_clip")
            if error_if_nonfinite and not math.isfinite(float(total)):
                raise RuntimeError(f"clip_grad_norm_: the norm of the gradients is {float(total)}; nothing was clipped")
    for g, c in zip(grads, work):
        if c is not g:
            g.copy_(c)
    torch.autograd.graph.increment_version(grads)
    return total


class FlatAdam(torch.optim.Optimizer):
    """Bias correction uses ONE step count for the whole buffer (``_step``; torch.optim.Adam keeps one per parameter).
    They agree whenever every parameter takes part in every step — the case for a PointNetCls.  A fused piece that sat
    out k steps (its slices are skipped, as torch skips ``grad is None``) resumes with the GLOBAL count in its bias
    correction where torch would use its own smaller count: after the first few hundred steps the two corrections are
    both within 1e-3 of 1, before that the resumed piece takes slightly smaller steps than torch's would.

    ``max_grad_norm``: every step first clips the gradients it uses (after ``grad_scale`` / ``grad_div``) by their global
    2-norm, as ``clip_grad_norm_`` before the step would; the factor is applied inside the update, the gradient buffer
    keeps the unclipped values (bias corrections from float64: updates differ from the plain step's by up to 1e-4 of
    themselves in the first steps), and ``grad_norm`` holds the norm (a device scalar that no host wait has
    touched: each step's own tensor, but with ``capturable`` one that every step and replay overwrites).  The parameters a
    step leaves alone do not count."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, capturable=False, max_grad_norm=None):
        if max_grad_norm is not None and not float(max_grad_norm) >= 0.0:
            raise ValueError(f"FlatAdam: max_grad_norm must not be negative, got {max_grad_norm}")
        params = [p for p in params]
        if not params:
            raise ValueError("optimizer got an empty parameter list")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=float(eps)))
        ps = self.param_groups[0]["params"]
        dev = ps[0].device
        if dev.type != "cuda" or any(p.device != dev or p.dtype != torch.float32 for p in ps):
            raise RuntimeError("FlatAdam needs float32 parameters on one CUDA device (libpngpd has no CPU path)")
        self.device = dev
        # 256-byte aligned slices (the kernels write gradients with 16-byte stores) behind a 64-float header: slot 0 of
        # the GRADIENT buffer's header carries the kept-sample count of a data-parallel step, so that it travels in the
        # same all-reduce as the adjacent (first) gradient slice (ddp.GradAverager) — one collective fewer per step
        self.header = 64
        self.offsets, off = [], self.header
        for p in ps:
            self.offsets.append(off)
            off += (p.numel() + 63) // 64 * 64
        self.numel = off
        z = lambda: torch.zeros(off, device=dev, dtype=torch.float32)
        self.flat_p, self.flat_g, self.flat_m, self.flat_v = z(), z(), z(), z()
        self.capturable = bool(capturable)
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self.grad_norm = torch.zeros((), device=dev, dtype=torch.float32) if max_grad_norm is not None else None
        self._clip_ws = None
        # device-resident step count / learning rate for captured graphs (StepLR rewrites group["lr"] in place)
        self.step_dev = torch.zeros((), device=dev, dtype=torch.float32) if capturable else None
        self._step = 0
        self._views = []
        self._written = bytearray(len(ps))    # per parameter: slice written in place by the fused backward this step
        self._grouped = bytearray(len(ps))    # per parameter: owned by a fused piece (optim.GradGroup) — set on first use
        with torch.no_grad():
            for p, o in zip(ps, self.offsets):
                n = p.numel()
                self.flat_p[o:o + n].copy_(p.detach().reshape(-1))
                p.data = self.flat_p[o:o + n].view(p.shape)
                gv = self.flat_g[o:o + n].view(p.shape)
                p.grad = gv
                _GRAD_VIEWS[p] = (gv, weakref.ref(self), len(self._views))
                self._views.append(gv)
                self.state[p] = {"step": torch.tensor(0.0),
                                 "exp_avg": self.flat_m[o:o + n].view(p.shape),
                                 "exp_avg_sq": self.flat_v[o:o + n].view(p.shape)}
        self._params = ps

    # ---- gradient buffer -------------------------------------------------------------------------------------
    def segment(self, params):
        """(offset, length) of the smallest contiguous range of the flat buffers covering ``params``."""
        idx = [i for i, p in enumerate(self._params) if any(p is q for q in params)]
        lo = min(self.offsets[i] for i in idx)
        hi = max(self.offsets[i] + (self._params[i].numel() + 63) // 64 * 64 for i in idx)
        return lo, hi - lo

    def zero_grad(self, set_to_none=True):
        """The fused backward OVERWRITES the gradient slices of the pieces it owns (``optim.GradGroup``: the trunks and
        FC stacks), so those are never cleared (and the views are never dropped).  Every other parameter — a plain
        autograd parameter next to the fused pieces, e.g. a custom head on a ``PointNetfeat`` — receives its gradient by
        autograd ACCUMULATION into the same view and is zeroed here; with pass-by-pass / ATen sequencing that is every
        parameter (one fill of the whole buffer).  A slice written twice raises (``mark_written``)."""
        for p, gv in zip(self._params, self._views):
            if p.grad is not gv:
                p.grad = gv
        self._written[:] = bytes(len(self._written))
        if any(self._grouped):
            # ``_grouped`` is set when a fused piece registers (optim.grad_group) and cleared when the same parameters
            # go through a non-fused call path again (optim.ungroup): no process-global sequencing flag is consulted
            for i, gv in enumerate(self._views):
                if not self._grouped[i]:
                    gv.zero_()
            return
        # no fused piece has registered yet (first step, or a model without one): clear everything
        self.flat_g.zero_()

    def _settle_gradients(self):
        """Before the update: every parameter's gradient must be IN its slice.  A gradient autograd left elsewhere
        (``.grad`` re-pointed or dropped by foreign code) is copied in / zeroed.  Returns the indices of the parameters
        to leave untouched this step: slices of a fused piece that took no part in this step's backward (an unused or
        eval-mode sub-module) hold a STALE gradient — ``torch.optim.Adam`` skips a parameter whose ``.grad`` is None,
        and so does this update (no momentum-only drift).  Plain autograd parameters always update."""
        skip = []
        for i, (p, gv) in enumerate(zip(self._params, self._views)):
            g = p.grad
            if g is not gv:
                if g is None:
                    gv.zero_()
                else:
                    gv.copy_(g)
                p.grad = gv
            elif self._grouped[i] and not self._written[i] and any(self._written):
                skip.append(i)
        self._written[:] = bytes(len(self._written))
        return skip

    def _update_ranges(self, skip):
        """(offset, length) runs of the flat buffers to update = everything but the slices of ``skip``."""
        if not skip:
            return [(self.header, self.numel - self.header)]
        runs, lo = [], self.header
        for i in skip:
            o = self.offsets[i]
            if o > lo:
                runs.append((lo, o - lo))
            lo = o + (self._params[i].numel() + 63) // 64 * 64
        if self.numel > lo:
            runs.append((lo, self.numel - lo))
        return runs

    # ---- update ----------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None, grad_scale=1.0, grad_div=None):
        """``grad_scale``: host factor on the gradients; ``grad_div``: 0-dim float32 device tensor the gradients are
        divided by (max(., 1)) — the all-reduced global sample count of ``ddp.GradAverager.backward``."""
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        g = self.param_groups[0]
        lr, (b1, b2), eps = g["lr"], g["betas"], g["eps"]
        lib = _lib.load()
        stream = torch.cuda.current_stream(self.device).cuda_stream
        lr_dev = lr.data_ptr() if torch.is_tensor(lr) and lr.is_cuda else None
        lr_host = 0.0 if lr_dev else float(lr)
        runs = self._update_ranges(self._settle_gradients())      # one run (one launch) unless a fused piece sat out
        self._step += 1
        with _lib.device_guard(self.device):
            if self.step_dev is not None:
                _lib.check(lib.pngpd_adam_step_inc(self.step_dev.data_ptr(), stream), "adam_step_inc")
            if self.max_grad_norm is not None:
                if self.step_dev is None:                         # (a graph's replays write one place)
                    self.grad_norm = torch.empty((), device=self.device, dtype=torch.float32)
                k = len(runs)
                if self._clip_ws is None:                         # kept: two steps at once would race for the parameters too
                    n = lib.pngpd_grad_clip_workspace_bytes(len(self._params))         # (a run holds a parameter at least)
                    self._clip_ws = torch.empty(n, device=self.device, dtype=torch.uint8)
                ws = self._clip_ws
                _lib.check(lib.pngpd_adam_flat_clip(self.flat_p.data_ptr(), self.flat_g.data_ptr(), self.flat_m.data_ptr(),
                                                    self.flat_v.data_ptr(), (ctypes.c_longlong * k)(*[lo for lo, _ in runs]),
                                                    (ctypes.c_longlong * k)(*[n for _, n in runs]), k, lr_host, lr_dev,
                                                    float(b1), float(b2), float(eps), float(self._step),
                                                    self.step_dev.data_ptr() if self.step_dev is not None else None,
                                                    float(grad_scale), grad_div.data_ptr() if grad_div is not None else None,
                                                    self.max_grad_norm, self.grad_norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                                    stream), "adam_flat_clip")
                runs = []
            for lo, n in runs:
                h = lo * 4
                _lib.check(lib.pngpd_adam_flat(self.flat_p.data_ptr() + h, self.flat_g.data_ptr() + h,
                                               self.flat_m.data_ptr() + h, self.flat_v.data_ptr() + h,
                                               n, lr_host, lr_dev, float(b1), float(b2),
                                               float(eps), float(self._step),
                                               self.step_dev.data_ptr() if self.step_dev is not None else None,
                                               float(grad_scale), grad_div.data_ptr() if grad_div is not None else None,
                                               stream), "adam_flat")
        # the kernel rewrote every parameter behind autograd's back: version-keyed caches (the eval-mode fold cache)
        # must see it
        torch.autograd.graph.increment_version(self._params)
        return loss

    # ---- checkpoints (torch.optim.Adam layout) ------------------------------------------------------------------
    def state_dict(self):
        # a captured graph (train.GraphedTrainStep) advances only the device-resident counter: it is the truth then
        step = float(self.step_dev.item()) if self.step_dev is not None else float(self._step)
        self._step = int(step)
        for p in self._params:
            self.state[p]["step"] = torch.tensor(step)
        return super().state_dict()

    def load_state_dict(self, state_dict):
        sd = state_dict["state"]
        steps = [float(v["step"]) for v in sd.values() if "step" in v]
        with torch.no_grad():
            for i, p in enumerate(self._params):
                st = sd.get(i)
                if st is None:
                    continue
                self.state[p]["exp_avg"].copy_(st["exp_avg"])
                self.state[p]["exp_avg_sq"].copy_(st["exp_avg_sq"])
        self._step = int(max(steps)) if steps else 0
        if self.step_dev is not None:
            self.step_dev.fill_(float(self._step))
        for g, sg in zip(self.param_groups, state_dict["param_groups"]):
            for k, v in sg.items():
                if k == "params":
                    continue
                if k == "lr" and torch.is_tensor(g.get("lr")):
                    # a capturable optimizer's lr is a device tensor a captured graph reads: fill it, never replace it
                    g["lr"].fill_(float(v))
                else:
                    g[k] = v
