"""RAdamScheduleFree as ONE fused HIP kernel over the flat parameter buffer.

Restates schedulefree==1.4.1 `RAdamScheduleFree` (the optimizer of configs/jit/x-loss/config.yml:74-78,
selected through src/optimizer/util.py:5-31; not installed in the reference's environment here, so
parity is unpinned — the update below follows the published algorithm):

  k = step count, beta2_t = beta2^(k+1), bc2 = 1 - beta2_t
  rho_inf = 2/(1-beta2) - 1, rho_t = rho_inf - 2 (k+1) beta2_t / bc2
  rect = sqrt((rho_t-4)(rho_t-2) rho_inf / ((rho_inf-4)(rho_inf-2) rho_t)) if rho_t > 4
         else (0 if silent_sgd_phase else 1)
  lr_t = lr * rect ; scheduled_lr = lr_t ; lr_max = max(lr_max, lr_t)
  weight = (k+1)^r * lr_max^weight_lr_power ; weight_sum += weight ; ckp1 = weight / weight_sum (0 if 0/0)
  v = beta2 v + (1-beta2) g^2 ; g <- g / (sqrt(v / bc2) + eps)  (only when rho_t > 4)
  g += wd * y ; y <- lerp(y, z, ckp1) ; y <- y + lr_t (beta1 (1-ckp1) - 1) g ; z <- z - lr_t g
  (y is the bf16 parameter: rounded after the lerp and after the add, as the reference's two
  in-place foreach ops on a bf16 tensor round it)
and train()/eval() swap y <-> x via p.lerp_(z, 1-beta1) / p.lerp_(z, 1-1/beta1).

Differences from the reference by design: z and v are kept in f32 (the reference keeps them in the
parameter dtype, bf16), gradients arrive in f32, and the optional `grad_scale` folds the DDP mean.
The param_groups dicts carry the same keys as schedulefree (incl. "scheduled_lr", which
src/trainer/common.py:499-514 reads).
"""

from __future__ import annotations

import bisect
import math

import numpy as np
import torch

from . import ops


class RAdamScheduleFreeFlat:
    def __init__(self, params: torch.Tensor, grads: torch.Tensor, lr: float = 0.0025, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.0, r: float = 0.0, weight_lr_power: float = 2.0,
                 silent_sgd_phase: bool = True):
        if params.dtype != torch.bfloat16 or grads.dtype != torch.float32 or params.numel() != grads.numel():
            raise ValueError("flat bf16 params and f32 grads of equal size expected")
        self.params, self.grads = params, grads
        self.z = torch.empty(params.numel(), dtype=torch.float32, device=params.device)
        self.v = torch.empty_like(self.z)
        self._initialised = False
        self.param_groups = [dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, r=r, k=0,
                                  train_mode=False, weight_sum=0.0, lr_max=-1.0, scheduled_lr=0.0,
                                  weight_lr_power=weight_lr_power, silent_sgd_phase=silent_sgd_phase)]

    @torch.no_grad()
    def train(self):
        g = self.param_groups[0]
        if not g["train_mode"]:
            if self._initialised:
                ops.sf_lerp(self.params, self.z, 1.0 - g["betas"][0])
            g["train_mode"] = True

    @torch.no_grad()
    def eval(self):
        g = self.param_groups[0]
        if g["train_mode"]:
            if self._initialised:
                ops.sf_lerp(self.params, self.z, 1.0 - 1.0 / g["betas"][0])
            g["train_mode"] = False

    def scalars(self) -> dict:
        """Host-side scalar schedule for the next step (pure arithmetic, no device work)."""
        g = self.param_groups[0]
        beta1, beta2 = g["betas"]
        step = g["k"] + 1
        beta2_t = beta2 ** step
        bc2 = 1 - beta2_t
        rho_inf = 2 / (1 - beta2) - 1
        rho_t = rho_inf - 2 * step * beta2_t / bc2
        if rho_t > 4.0:
            rect = math.sqrt((rho_t - 4.0) * (rho_t - 2.0) * rho_inf / ((rho_inf - 4.0) * (rho_inf - 2.0) * rho_t))
        else:
            rect = float(not g["silent_sgd_phase"])
        lr = g["lr"] * rect
        lr_max = max(lr, g["lr_max"])
        weight = (step ** g["r"]) * (lr_max ** g["weight_lr_power"])
        weight_sum = g["weight_sum"] + weight
        ckp1 = weight / weight_sum if weight_sum != 0 else 0.0
        return dict(step=step, bc2=bc2, adam=rho_t > 4.0, lr=lr, lr_max=lr_max, weight_sum=weight_sum, ckp1=ckp1,
                    adaptive_y_lr=lr * (beta1 * (1 - ckp1) - 1), beta2=beta2)

    @torch.no_grad()
    def begin_step(self) -> dict:
        """Computes this step's scalars; the update itself is applied range by range (so each
        all-reduced gradient bucket can be stepped as soon as it lands) and closed by end_step."""
        g = self.param_groups[0]
        if not g["train_mode"]:
            raise RuntimeError("Optimizer was not in train mode when step is called. "
                               "Please insert .train() and .eval() calls on the optimizer.")
        if not self._initialised:
            ops.sf_init(self.params, self.z, self.v)
            self._initialised = True
        return self.scalars()

    @torch.no_grad()
    def apply_range(self, s: dict, lo: int, hi: int, grad_scale: float = 1.0, grad: torch.Tensor | None = None,
                    clip_coef: torch.Tensor | None = None, clip_value: float | None = None):
        """Steps parameters [lo, hi) from self.grads[lo:hi], or from `grad` (f32 or bf16, the range's
        all-reduced wire buffer) when given. clip_coef (device f32 scalar) / clip_value: gradient clipping
        (for_training.py:98-109) applied to grad_scale * grad inside the same kernel."""
        g = self.param_groups[0]
        if hi <= lo:
            return
        src = self.grads[lo:hi] if grad is None else grad
        ops.radam_sf_step(self.params[lo:hi], src, self.z[lo:hi], self.v[lo:hi], beta2=s["beta2"],
                          bias_correction2=s["bc2"], eps=g["eps"], ckp1=s["ckp1"], adaptive_y_lr=s["adaptive_y_lr"],
                          lr=s["lr"], decay=g["weight_decay"], grad_scale=grad_scale, adam=s["adam"],
                          clip_coef=clip_coef, clip_value=clip_value or 0.0)

    def end_step(self, s: dict):
        g = self.param_groups[0]
        g["scheduled_lr"] = s["lr"]
        g["lr_max"] = s["lr_max"]
        g["weight_sum"] = s["weight_sum"]
        g["k"] = g["k"] + 1

    @torch.no_grad()
    def step(self, grad_scale: float = 1.0):
        s = self.begin_step()
        self.apply_range(s, 0, self.params.numel(), grad_scale)
        self.end_step(s)

    def zero_grad(self, set_to_none: bool = False):
        self.grads.zero_()

    def state_dict(self) -> dict:
        return {"param_groups": [dict(g) for g in self.param_groups], "z": self.z, "v": self.v,
                "initialised": self._initialised}


# ----------------------------------------------------------------------------- clipping of many gradient tensors
_CLIP_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
_TINY = 2.0 ** -149  # the smallest f32 above 0, which would switch a limit off
_PIECE = np.dtype([("g", "<u8"), ("out", "<u8"), ("n", "<i4"), ("dtype", "<i4")])  # VptGradPiece
# Clipped copies: where gradients and copies are more than the 256-MB cache holds, copies left in it drive out the gradients
# still to be read, so they are stored past it. Cached : streamed, clipping and a pass over the copies: 95 MB of bf16
# gradients 83 : 87 us, 118 MB 101 : 104, 153 MB 147 : 142, 229 MB 236 : 226; f32 118 MB 96 : 99, 153 MB 137 : 129, 332 MB
# 340 : 330 (the clipping alone 214 : 187). In place the stores go to lines that were just read.
_CACHE = 256 << 20
_CAPTURED: list = []  # tables that captured graphs read at every replay: they stay when their handles go


def _dense(t: torch.Tensor) -> bool:
    """Whether t covers numel() consecutive elements, in whatever order of its dims."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        if stride != want:
            return False
        want *= size
    return True


def _span(t: torch.Tensor) -> tuple[int, int]:
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


class GradClip:
    """Global-norm and value clipping of a fixed list of gradient tensors, in two launches for any number of them
    (after_backward, src/models/for_training.py:98-109; torch.nn.utils.clip_grad_norm_ and clip_grad_value_).

    `grads`: dense GPU tensors of one device (bf16, f16 and f32 may be mixed; any dims, also transposed; empty ones too).
    `out`: tensors of the same types, shapes and strides for the clipped gradients; None: in place. What is written must not
    overlap. The handle keeps the tensors, their memory as it was then, and a table of it on the device: gradients that are new
    tensors every step (`zero_grad(set_to_none=True)`) go through clip_grad_norm_ instead, and a tensor that is given other
    memory (`t.data = ...`, `set_`) needs a new handle. Building it copies the table to the device, waiting for that, and is
    refused in a captured region; clip() and norm() are for one (their workspace is allocated per call, the table outlives
    the handle; the tensors are the graph's inputs and the caller's to keep), and may run on any stream."""

    def __init__(self, grads, out=None):
        self.grads = list(grads)
        self.out = self.grads if out is None else list(out)
        if len(self.out) != len(self.grads):
            raise ValueError(f"GradClip: {len(self.out)} outputs for {len(self.grads)} gradients")
        for g, o in zip(self.grads, self.out):
            if not isinstance(g, torch.Tensor) or not isinstance(o, torch.Tensor):
                raise ValueError("GradClip: tensors expected")
            if g.layout != torch.strided or g.dtype not in _CLIP_DTYPES:
                raise ValueError(f"GradClip: dense bf16, f16 or f32 gradients expected, got {g.dtype} {g.layout}")
            if not _dense(g):
                raise ValueError(f"GradClip: a gradient with gaps between its values (strides {tuple(g.stride())})")
            if o is not g and (o.dtype != g.dtype or o.shape != g.shape or o.stride() != g.stride()):
                raise ValueError("GradClip: an output of another type, shape or stride than its gradient")
        written = sorted(_span(o) for o in self.out if o.numel())
        if any(a[1] > b[0] for a, b in zip(written, written[1:])):
            raise ValueError("GradClip: the clipped gradients overlap (the same tensor twice?)")
        if out is not None:  # a gradient may share memory with its own output, all of it, and with no other
            spans = sorted((*_span(o), i) for i, o in enumerate(self.out) if o.numel())
            ends = [sp[1] for sp in spans]
            for i, g in enumerate(self.grads):
                if g.numel():
                    lo, hi = _span(g)
                    k = bisect.bisect_right(ends, lo)
                    if k < len(spans) and spans[k][0] < hi and spans[k] != (lo, hi, i):
                        raise ValueError("GradClip: an output overlaps another gradient, or its own in part")
        devs = {t.device for t in self.grads + self.out}
        if any(d.type != "cuda" for d in devs):
            raise ValueError("GradClip: GPU tensors expected")
        if len(devs) > 1:
            raise ValueError("GradClip: tensors on different devices")
        self.device = devs.pop() if devs else torch.device("cuda", torch.cuda.current_device())
        with ops._on(self.device.index):
            self._finish()

    def _finish(self):
        """The table of the checked tensors, and what it names: the memory stays this handle's, also when a tensor is given
        other memory meanwhile (`t.data = ...`)."""
        if ops._capturing():
            raise RuntimeError("GradClip: built inside a captured region (its table is copied from the host): build it before")
        self._memory = [t.untyped_storage() for t in self.grads]
        if self.out is not self.grads:
            self._memory += [t.untyped_storage() for t in self.out]
        self._table, self._count = self._pieces()
        self._captured = False
        self._stream = ops._raw_stream(self.device.index)
        self._parts = ops.call("vpt_grad_list_parts", self._count)
        size = sum(g.numel() * g.element_size() for g in self.grads)
        self._cached = int(2 * size <= _CACHE or all(o.data_ptr() == g.data_ptr() for g, o in zip(self.grads, self.out)))

    def _pieces(self):
        piece = ops.call("vpt_grad_list_piece")
        rows = [(g.data_ptr(), o.data_ptr(), g.numel(), _CLIP_DTYPES[g.dtype], g.element_size())
                for g, o in zip(self.grads, self.out) if g.numel()]
        if not rows:
            return None, 0
        ptr, outp, n, kind, size = (np.array(c, dtype=np.int64) for c in zip(*rows))
        cuts = -(-n // piece)
        first = np.cumsum(cuts) - cuts
        at = (np.arange(int(cuts.sum())) - np.repeat(first, cuts)) * piece  # each piece's first value in its tensor
        table = np.zeros(len(at), _PIECE)
        table["g"] = np.repeat(ptr, cuts) + at * np.repeat(size, cuts)
        table["out"] = np.repeat(outp, cuts) + at * np.repeat(size, cuts)
        table["n"] = np.minimum(np.repeat(n, cuts) - at, piece)
        table["dtype"] = np.repeat(kind, cuts)
        return torch.from_numpy(table.view(np.uint8)).to(self.device), len(at)

    def _run(self, max_norm: float, clip_value: float, count: int, want_norm: bool):
        with ops._on(self.device.index):
            st = ops._raw_stream(self.device.index)
            if self._table is not None:
                if ops._capturing():
                    if not self._captured:
                        self._captured = True
                        _CAPTURED.append(self._table)
                elif st != self._stream:
                    self._table.record_stream(torch.cuda.current_stream())
            table = None if self._table is None else self._table.data_ptr()
            if not want_norm:
                ops.call("vpt_grad_list_clip", table, count, self._cached, None, 0, 0.0, clip_value, None, st)
                return None
            ws = torch.empty(self._parts, dtype=torch.float64, device=self.device)
            norm = torch.empty((), dtype=torch.float32, device=self.device)
            ops.call("vpt_grad_list_norm", table, self._count, ws.data_ptr(), st)
            ops.call("vpt_grad_list_clip", table, count, self._cached, ws.data_ptr(), self._parts, max_norm, clip_value,
                     norm.data_ptr(), st)
            return norm

    @torch.no_grad()
    def clip(self, max_norm: float | None = None, clip_value: float | None = None) -> torch.Tensor | None:
        """out = clamp(min(1, max_norm / (norm + 1e-6)) * g, -clip_value, clip_value); returns the norm before it (f32, on the
        device, not synchronised; None without max_norm). A gradient that is not finite makes the norm, and with it the
        clipped gradients, what torch.nn.utils.clip_grad_norm_ makes of them."""
        if max_norm is not None and not max_norm >= _TINY:
            raise ValueError("max_norm must be > 0 (as f32)")
        if clip_value is not None and not clip_value >= _TINY:
            raise ValueError("clip_value must be > 0 (as f32)")
        if max_norm is None and clip_value is None:
            raise ValueError("clip: max_norm or clip_value")
        return self._run(float(max_norm or 0.0), float(clip_value or 0.0), self._count, max_norm is not None)

    @torch.no_grad()
    def norm(self) -> torch.Tensor:
        """The global L2 norm (f32, on the device); nothing is written."""
        return self._run(0.0, 0.0, 0, True)


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False, *,
                    clip_value: float | None = None) -> torch.Tensor:
    """torch.nn.utils.clip_grad_norm_ over parameters' .grad (its positions; norm_type 2 alone), then clip_grad_value_ when
    clip_value is given, in place. Parameters without a gradient are left out; error_if_nonfinite reads the norm back before
    anything is scaled. Every call builds the gradients' table (0.5 ms of the host for 226 of them, 2.1 ms for 1400) and copies
    it, which waits for all work queued on the device; torch's function does not wait. Gradients that stay where they are go
    through a GradClip kept over the steps, which neither builds nor waits."""
    if float(norm_type) != 2.0:
        raise ValueError(f"clip_grad_norm_: norm_type {norm_type}: the L2 norm (2.0) is the only one")
    params = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in params if p.grad is not None]
    if not grads:
        if not max_norm >= _TINY:
            raise ValueError("max_norm must be > 0 (as f32)")
        return torch.tensor(0.0)
    clipper = GradClip(grads)
    if error_if_nonfinite and not bool(torch.isfinite(clipper.norm())):
        raise RuntimeError("The total norm of the gradients is not finite, so it cannot be clipped.")
    return clipper.clip(max_norm, clip_value)
