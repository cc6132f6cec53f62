"""Training-step ops after the rasterizer (SURVEY.md §8f "next" rows 1-2), host side.

* ``l1_ssim_loss(image, gt, lambda_dssim)`` — the reference's loss
  ``(1 - l) * l1_loss(image, gt) + l * (1 - ssim(image, gt))`` (train.py:103-105,
  utils/loss_utils.py:17-108) as ONE HIP pass that also produces d loss / d image;
  the autograd backward only scales that map by the incoming gradient.
* ``FusedAdam`` — torch.optim.Adam's update (scene/gaussian_model.py:176-205: six
  groups, lr 0 default, eps 1e-15) in one HIP launch over every parameter; state
  (``exp_avg``, ``exp_avg_sq``, ``step``) kept like torch's.
* ``FusedAdamW`` — AdamW over any number of tensors, with its moments in 32 bits or in
  8 (``adamw_state`` / ``adamw_step``), and the gradients clipped by their global norm
  on the device (``grad_norm``).
* ``select_rows`` / ``take_rows`` — eviction to a budget by an accumulated weight: the
  rows that stay, and the rows of parameters and optimiser states gathered in one launch.
* ``densify_stats`` — train.py:126-127 + scene/gaussian_model.py:565-581
  (``max_radii2D``, ``xyz_gradient_accum``, ``denom``) in one HIP launch.
* ``dist_knn3`` — ``distCUDA2`` of the simple-knn submodule (scene/gaussian_model.py:
  153-155): mean squared distance to the 3 nearest other
  points, exact, through a uniform-grid HIP search.

All call libgsr.so through the C ABI (include/gsr.h) on the current HIP
stream; there is no CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes
import math
import struct

import numpy as np
import torch

from diff_gaussian_rasterization import _C


def _cuda(t: torch.Tensor, name: str):
    if not t.is_cuda:
        raise RuntimeError(f"{name}: tensors must be on the GPU (no CPU implementation)")
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name}: float32 expected, got {t.dtype}")


class _L1SSIM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, image, gt, lambda_dssim):
        lib = _C.load_library()
        _cuda(image, "l1_ssim_loss")
        _cuda(gt, "l1_ssim_loss")
        if image.shape != gt.shape or image.dim() != 3:
            raise RuntimeError(f"l1_ssim_loss: image {tuple(image.shape)} and gt {tuple(gt.shape)} must be equal [C,H,W]")
        x, y = image.contiguous(), gt.contiguous()
        C, H, W = x.shape
        # L1 alone (lambda 0): the loss here, its gradient in the backward from the
        # incoming dloss (gsr_l1_grad) — no map written here and scaled again there
        l1_only = float(lambda_dssim) == 0.0
        grad = None if l1_only else torch.empty_like(x)
        scratch = torch.empty(lib.gsr_l1_ssim_scratch_bytes(C, H, W), dtype=torch.uint8, device=x.device)
        out = torch.empty(3, dtype=torch.float32, device=x.device)
        _C._check(lib.gsr_l1_ssim(x.data_ptr(), y.data_ptr(), C, H, W, float(lambda_dssim),
                                  None if l1_only else grad.data_ptr(), scratch.data_ptr(), out.data_ptr(),
                                  _C._stream(x.device)), "gsr_l1_ssim")
        ctx.l1_only = l1_only
        ctx.save_for_backward(*((x, y) if l1_only else (grad,)))
        ctx.parts = out
        return out[0]

    @staticmethod
    def backward(ctx, g):
        if ctx.l1_only:
            x, y = ctx.saved_tensors
            lib = _C.load_library()
            grad = torch.empty_like(x)
            gd = g.detach().to(torch.float32).contiguous()
            _C._check(lib.gsr_l1_grad(x.data_ptr(), y.data_ptr(), x.numel(), gd.data_ptr(), grad.data_ptr(),
                                      _C._stream(x.device)), "gsr_l1_grad")
            return grad, None, None
        (grad,) = ctx.saved_tensors
        return grad * g, None, None


def l1_ssim_loss(image: torch.Tensor, gt: torch.Tensor, lambda_dssim: float = 0.2) -> torch.Tensor:
    """(1 - lambda) * L1 + lambda * (1 - SSIM) with the 11x11 sigma-1.5 window, mean over C*H*W."""
    return _L1SSIM.apply(image, gt, lambda_dssim)


class FusedAdam:
    """torch.optim.Adam (no weight decay, no amsgrad) over param groups, one launch per step.

    ``groups``: the reference's list of dicts (``params``, ``lr``, ``name``)."""

    def __init__(self, groups, lr: float = 0.0, betas=(0.9, 0.999), eps: float = 1e-15):
        self.param_groups = [dict(g) for g in groups]
        for g in self.param_groups:
            g.setdefault("lr", lr)
        if sum(len(g["params"]) for g in self.param_groups) > _C.ADAM_MAX_SEGS:
            raise ValueError(f"FusedAdam: at most {_C.ADAM_MAX_SEGS} tensors per launch")
        self.betas, self.eps = betas, eps
        self.state = {}

    @torch.no_grad()
    def step(self):
        """Validate every segment first, then advance the step counts and launch, so a
        rejected call leaves no parameter's state advanced."""
        lib = _C.load_library()
        segs = (_C.GsrAdamSegment * _C.ADAM_MAX_SEGS)()
        todo, grads = [], []
        for g in self.param_groups:
            for p in g["params"]:
                if p.grad is None:
                    continue
                _cuda(p, "FusedAdam")
                if not (p.is_contiguous() and p.grad.is_contiguous()):
                    raise RuntimeError("FusedAdam: parameters and gradients must be contiguous")
                if p.is_neg():
                    raise RuntimeError("FusedAdam: parameters must not be negated views")
                todo.append((g, p))
                grads.append(p.grad.resolve_neg())  # a complex number's backward may leave a negated view
        if len(todo) > _C.ADAM_MAX_SEGS:
            raise RuntimeError(f"FusedAdam: at most {_C.ADAM_MAX_SEGS} tensors per launch")
        steps = {self.state[p]["step"] if p in self.state else 0 for _, p in todo}
        if len(steps) > 1:
            raise RuntimeError("FusedAdam: parameters at different step counts")
        if not todo:
            return
        step = steps.pop() + 1
        for n, (g, p) in enumerate(todo):
            st = self.state.get(p)
            if st is None:
                st = self.state[p] = {"step": 0, "exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.zeros_like(p)}
            st["step"] = step
            segs[n] = _C.GsrAdamSegment(p.data_ptr(), grads[n].data_ptr(), st["exp_avg"].data_ptr(),
                                        st["exp_avg_sq"].data_ptr(), p.numel(), float(g["lr"]))
        _C._check(lib.gsr_adam_step(segs, len(todo), step, self.betas[0], self.betas[1], self.eps,
                                    _C._stream(todo[0][1].device)), "gsr_adam_step")

    def zero_grad(self, set_to_none: bool = True):
        for g in self.param_groups:
            for p in g["params"]:
                if set_to_none:
                    p.grad = None
                elif p.grad is not None:
                    p.grad.zero_()


# ------------------------------------------------------------------ AdamW, 32- or 8-bit states
SCALE_BLOCK = 64  # elements that share a scale in an 8-bit state
_KEYS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_scale", "exp_rms", "exp_rms_scale")}


_SAME = contextlib.nullcontext()
_F32, _CODE, _SCALE = torch.float32, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _on(device):
    """The launches of a call go to ``device``, whichever device is current."""
    return _SAME if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _raw_stream(index: int) -> int:
    """The current stream's handle on device ``index``: as _C._stream, without the 2 us of a
    torch.cuda.Stream object, a tenth of a small step."""
    return torch._C._cuda_getCurrentRawStream(index)


def adamw_state(param: torch.Tensor, state_bits: int = 32) -> dict:
    """The initial AdamW state of a tensor.  32 bits: ``exp_avg`` and ``exp_avg_sq`` in
    float32, as torch's.  8 bits: ``exp_avg`` and ``exp_rms`` (the root of exp_avg_sq) as
    float8_e4m3fn of the parameter's shape, with a float8_e8m0fnu scale for every 64
    elements of the flattened tensor each (``unpack_state8`` gives their values)."""
    if state_bits == 32:
        z = lambda: torch.zeros(param.shape, dtype=torch.float32, device=param.device)  # noqa: E731
        return {"step": 0, "exp_avg": z(), "exp_avg_sq": z()}
    if state_bits != 8:
        raise ValueError(f"adamw_state: state_bits must be 32 or 8 (got {state_bits})")
    nb = -(-param.numel() // SCALE_BLOCK)
    st = {"step": 0}
    for k in ("exp_avg", "exp_rms"):
        st[k] = torch.zeros(param.shape, dtype=torch.uint8, device=param.device).view(torch.float8_e4m3fn)
        st[k + "_scale"] = torch.zeros(nb, dtype=torch.uint8, device=param.device).view(torch.float8_e8m0fnu)
    return st


def unpack_state8(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The float32 values of an 8-bit state (``exp_avg`` with ``exp_avg_scale``, or ``exp_rms``
    with ``exp_rms_scale``), for inspection: torch operations, on any device."""
    b = scale.view(torch.uint8).to(torch.int32)
    s = torch.where(b > 0, b << 23, 0x400000).view(torch.float32).repeat_interleave(SCALE_BLOCK)[:codes.numel()]
    return (codes.reshape(-1).to(torch.float32) * s).view(codes.shape)


def _state_refuse(st: dict, p: torch.Tensor, who: str):
    bits = 32 if "exp_avg_sq" in st else 8
    n = p.numel()
    for k in _KEYS[bits]:
        t = st.get(k)
        scale = k.endswith("_scale")
        want = _F32 if bits == 32 else (_SCALE if scale else _CODE)
        if t is None or t.dtype is not want or t.numel() != (-(-n // SCALE_BLOCK) if scale else n) or \
                t.device != p.device or not t.is_contiguous() or t.is_neg():
            raise RuntimeError(f"{who}: state {k!r} must be contiguous {want} on {p.device}, no negated view, and fit "
                               f"its parameter of {tuple(p.shape)}" + ("" if t is None else
                               f" (got {t.dtype} {tuple(t.shape)} on {t.device})"))


def _state_ptrs(st: dict, p: torch.Tensor, n: int, who: str, raw: bool = True) -> tuple:
    """(bits, then exp_avg, exp_second and their scales' addresses) of a checked state of ``p``.
    ``raw``: its bytes are read (codes have no negated views: those come of complex numbers)."""
    at = p.get_device()
    v = st.get("exp_avg_sq")
    m = st.get("exp_avg")
    if v is not None:
        if m is None or not (m.dtype is v.dtype is _F32 and m.numel() == n == v.numel() and
                             m.get_device() == at == v.get_device() and m.is_contiguous() and v.is_contiguous()) or \
                raw and (m.is_neg() or v.is_neg()):
            _state_refuse(st, p, who)
        return 32, m.data_ptr(), v.data_ptr(), 0, 0
    r, ms, rs = st.get("exp_rms"), st.get("exp_avg_scale"), st.get("exp_rms_scale")
    if m is None or r is None or ms is None or rs is None or not (
            m.dtype is r.dtype is _CODE and ms.dtype is rs.dtype is _SCALE and
            m.numel() == n == r.numel() and ms.numel() == rs.numel() == -(-n // SCALE_BLOCK) and
            m.get_device() == r.get_device() == ms.get_device() == rs.get_device() == at and
            m.is_contiguous() and r.is_contiguous() and ms.is_contiguous() and rs.is_contiguous()):
        _state_refuse(st, p, who)
    return 8, m.data_ptr(), r.data_ptr(), ms.data_ptr(), rs.data_ptr()


def _per_tensor(x, n: int, name: str) -> list:
    if not isinstance(x, (list, tuple)):
        return [float(x)] * n
    if len(x) != n:
        raise ValueError(f"adamw_step: {len(x)} values of {name} for {n} tensors")
    return [float(v) for v in x]


def _adamw_refuse(p: torch.Tensor, g: torch.Tensor, dev):
    if not p.is_cuda:
        raise RuntimeError("adamw_step: tensors must be on the GPU (no CPU implementation)")
    if p.dtype not in _C.DTYPES or g.dtype is not p.dtype:
        raise RuntimeError(f"adamw_step: float32 or bfloat16 parameters with gradients of the same dtype "
                           f"expected, got {p.dtype} and {g.dtype}")
    if p.device != dev or g.device != dev:
        raise RuntimeError(f"adamw_step: tensors on {p.device} and {g.device}, expected {dev}")
    if g.shape != p.shape:
        raise RuntimeError(f"adamw_step: gradient {tuple(g.shape)} of a parameter {tuple(p.shape)}")
    if p.is_neg():
        raise RuntimeError("adamw_step: parameters must not be negated views")
    raise RuntimeError("adamw_step: parameters and gradients must be contiguous")


_ADAMW_MOST = 1 << 33  # elements of a tensor (include/gsr.h gsr_adamw_step)


def _adamw_refuse_count(count, size: int):
    if count is None or count < 0:
        raise RuntimeError(f"adamw_step: a state's step must be a count >= 0 (got {count!r})")
    raise RuntimeError(f"adamw_step: a tensor's size must be at most 2^33 elements (got {size})")


def adamw_step(params, grads, states, lr, weight_decay=0.0, betas=(0.9, 0.999), eps: float = 1e-15,
               grad_scale: torch.Tensor = None, seed: int = 0):
    """One AdamW step in place over lists of tensors of up to 2^33 elements: parameters, their
    gradients and their states (``adamw_state``; 32- and 8-bit ones may be mixed), in one launch
    for up to 40 tensors of a dtype and state width.

    ``lr`` and ``weight_decay``: a number, or one per tensor.  Each state's ``step`` counts
    its own tensor's steps and is advanced by one.  ``grad_scale``: a float32 scalar on the
    device that every gradient is multiplied by (``grad_norm``'s second result).  Parameters
    are float32 or bfloat16, gradients of the same dtype, all contiguous and on one device;
    parameters and states are no negated views.
    8-bit states and bfloat16 parameters are rounded stochastically, by a pure function of
    ``seed`` (an int of up to 64 bits), the tensor's step, its place in the list and the
    element: the same call gives the same bits.  ``eps``: 0, or 2^-126 and above.  Tensors must
    not overlap.  Step counts, rates and seed are host values and would be frozen in a captured
    graph: under capture this raises.

    Everything is validated before anything is launched and any count advanced."""
    lib = _C.load_library()
    n = len(params)
    if len(grads) != n or len(states) != n:
        raise ValueError(f"adamw_step: {n} parameters, {len(grads)} gradients, {len(states)} states")
    lrs, wds = _per_tensor(lr, n, "lr"), _per_tensor(weight_decay, n, "weight_decay")
    if not n:
        return
    dev, at = params[0].device, params[0].get_device()
    launches, seen, written, keep = {}, set(), 0, []
    for k, (p, g, st) in enumerate(zip(params, grads, states)):
        dt = p.dtype
        if at < 0 or dt not in _C.DTYPES or g.dtype is not dt or p.get_device() != at or g.get_device() != at or \
                not p.is_same_size(g) or not (p.is_contiguous() and g.is_contiguous()) or \
                dt is _F32 and p.is_neg():
            _adamw_refuse(p, g, dev)
        if dt is _F32 and g.is_neg():  # as a conjugated complex number's backward leaves it
            g = g.resolve_neg()
            keep.append(g)  # until the launch
        size = p.numel()
        bits, m, v, ms, vs = _state_ptrs(st, p, size, "adamw_step")
        count = st.get("step")
        if count is None or count < 0 or size > _ADAMW_MOST:  # what the library would refuse of a later launch
            _adamw_refuse_count(count, size)
        if not size:
            continue
        addr = p.data_ptr()
        written += 3 if bits == 32 else 5
        seen.update((addr, m, v) if bits == 32 else (addr, m, v, ms, vs))
        if len(seen) != written:
            raise RuntimeError("adamw_step: a parameter or a part of a state appears twice")
        launches.setdefault((dt, bits), []).extend((addr, g.data_ptr(), m, v, ms, vs, size, lrs[k], wds[k],
                                                    count + 1, k))
    if grad_scale is not None and (grad_scale.dtype is not torch.float32 or grad_scale.numel() != 1 or
                                   grad_scale.device != dev):
        raise RuntimeError(f"adamw_step: grad_scale must be a float32 scalar on {dev}")
    with _on(dev):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("adamw_step: step counts and rates are host values; not for graph capture")
        if grad_scale is not None:
            grad_scale = grad_scale.resolve_neg()
        stream, scale = _raw_stream(at), None if grad_scale is None else grad_scale.data_ptr()
        seed &= 0xFFFFFFFFFFFFFFFF
        tables = [(kind, struct.pack("7q2d2i" * (len(segs) // 11), *segs), len(segs) // 11)  # gsr_adamw_segment
                  for kind, segs in launches.items()]
        for (dt, bits), table, count in tables:
            _C._check(lib.gsr_adamw_step(table, count, _C.DTYPES[dt], bits, betas[0], betas[1], eps, scale, seed,
                                         stream), "gsr_adamw_step")
    for st in states:
        st["step"] += 1
    torch.autograd.graph.increment_version([p for p in params if not p.is_inference()])


def grad_norm(grads, max_norm: float = math.inf):
    """(norm, scale), two float32 scalars on the device: the 2-norm over all the tensors
    (float32 or bfloat16; squares and sums in 64 bits), and ``min(1, max_norm / (norm +
    1e-6))``, torch.nn.utils.clip_grad_norm_'s coefficient, which ``adamw_step`` takes as
    ``grad_scale`` (as torch's, NaN where the norm and ``max_norm`` are both infinite).  The gradients
    are not written and the host does not wait."""
    lib = _C.load_library()
    if not len(grads):
        raise ValueError("grad_norm: no gradients")
    dev, at = grads[0].device, grads[0].get_device()
    segs = []
    for g in grads:
        if g.get_device() != at or at < 0 or g.dtype not in _C.DTYPES or not g.is_contiguous():
            if not g.is_cuda:
                raise RuntimeError("grad_norm: tensors must be on the GPU (no CPU implementation)")
            if g.dtype not in _C.DTYPES:
                raise RuntimeError(f"grad_norm: float32 or bfloat16 expected, got {g.dtype}")
            raise RuntimeError(f"grad_norm: gradients must be contiguous and on one device ({dev})")
        segs += (g.data_ptr(), g.numel(), _C.DTYPES[g.dtype])
    count = len(grads)
    with _on(dev):
        out = torch.empty(2, dtype=torch.float32, device=dev)
        scratch = torch.empty(lib.gsr_grad_norm_scratch_bytes(count), dtype=torch.uint8, device=dev)
        _C._check(lib.gsr_grad_norm(struct.pack("3q" * count, *segs), count, float(max_norm), scratch.data_ptr(),
                                    out.data_ptr(), _raw_stream(at)), "gsr_grad_norm")
    return out.unbind()


def _adamw_options(groups, betas, eps) -> tuple:
    """(betas, eps) of the param groups, which share them (those given where a group has none); what a
    step would not do is refused."""
    got = set()
    for g in groups:
        for k in ("amsgrad", "maximize"):
            if g.get(k):
                raise ValueError(f"FusedAdamW: {k} is not implemented")
        if g["weight_decay"] and not g.get("decoupled_weight_decay", True):
            raise ValueError("FusedAdamW: weight decay is decoupled (a checkpoint of torch.optim.Adam's is not)")
        b1, b2 = g.get("betas", betas)
        got.add(((float(b1), float(b2)), float(g.get("eps", eps))))
    if len(got) > 1:
        raise ValueError(f"FusedAdamW: all groups have the same betas and eps (got {sorted(got)})")
    return got.pop() if got else (betas, eps)


class FusedAdamW:
    """AdamW over param groups (``params``, ``lr``, optionally ``weight_decay``, ``name``), with
    the moments in 32 bits or in 8 (``state_bits``), and gradients clipped to a global norm of
    ``max_norm`` (None: not clipped).  ``betas`` and ``eps`` stand in the groups, as torch's do, with
    the same values in all of them.  ``state[p]`` is ``adamw_state``'s dict: with 32 bits the
    names that code for torch's optimizer expects.  After each step ``grad_norm`` holds the
    norm before clipping (a device scalar; None without clipping)."""

    def __init__(self, groups, lr: float = 0.0, betas=(0.9, 0.999), eps: float = 1e-15, weight_decay: float = 0.0,
                 state_bits: int = 32, max_norm: float = None, seed: int = 0):
        if state_bits not in _KEYS:
            raise ValueError(f"FusedAdamW: state_bits must be 32 or 8 (got {state_bits})")
        self.param_groups = [dict(g) for g in groups]
        for g in self.param_groups:
            g.setdefault("lr", lr)
            g.setdefault("weight_decay", weight_decay)
            g.setdefault("betas", tuple(betas))
            g.setdefault("eps", eps)
        self._defaults = {"betas": tuple(betas), "eps": eps}
        self._options()
        self.state_bits, self.max_norm, self.seed = state_bits, max_norm, seed
        self.state = {}
        self.grad_norm = None

    def _options(self) -> tuple:
        return _adamw_options(self.param_groups, **self._defaults)

    def _set_option(self, key, value):
        for g in [self._defaults] + self.param_groups:
            g[key] = value

    betas = property(lambda self: self._options()[0], lambda self, b: self._set_option("betas", tuple(b)))
    eps = property(lambda self: self._options()[1], lambda self, e: self._set_option("eps", e))

    @torch.no_grad()
    def step(self):
        todo = [(g, p) for g in self.param_groups for p in g["params"] if p.grad is not None]
        if not todo:
            return
        betas, eps = self._options()
        params = [p for _, p in todo]
        grads = [p.grad for p in params]
        states = [self.state[p] if p in self.state else adamw_state(p, self.state_bits) for p in params]
        scale = norm = None
        if self.max_norm is not None:
            norm, scale = grad_norm(grads, self.max_norm)
        adamw_step(params, grads, states, [g["lr"] for g, _ in todo], [g["weight_decay"] for g, _ in todo],
                   betas, eps, scale, self.seed)
        self.grad_norm = norm
        self.state.update(zip(params, states))

    zero_grad = FusedAdam.zero_grad

    def state_dict(self) -> dict:
        """{"state": {place: state}, "param_groups": [...]} in torch.optim's form (the tensors
        themselves, not copies): place counts the parameters through the groups.  Beside them
        "seed", "max_norm" and "state_bits", so that a loaded optimiser continues bit for bit."""
        params = [p for g in self.param_groups for p in g["params"]]
        groups, at = [], 0
        for g in self.param_groups:
            groups.append({**g, "params": list(range(at, at + len(g["params"])))})
            at += len(g["params"])
        return {"state": {k: dict(self.state[p]) for k, p in enumerate(params) if p in self.state},
                "param_groups": groups, "seed": self.seed, "max_norm": self.max_norm, "state_bits": self.state_bits}

    def load_state_dict(self, d: dict):
        """Takes over ``state_dict``'s states (copied to their parameters' device), the groups' options
        (betas and eps among them) and what stands beside them; a dict of torch.optim.AdamW, which has
        no such things, leaves those as they are.  States of either width are taken as they are.
        Options that a step would not follow (amsgrad, maximize, betas by group) are refused."""
        if [len(g["params"]) for g in d["param_groups"]] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("FusedAdamW.load_state_dict: other param groups")
        groups = [{**g, **{n: x for n, x in h.items() if n != "params"}}
                  for g, h in zip(self.param_groups, d["param_groups"])]
        betas, eps = _adamw_options(groups, **self._defaults)
        state_bits = d.get("state_bits", self.state_bits)
        if state_bits not in _KEYS:
            raise ValueError(f"FusedAdamW.load_state_dict: state_bits must be 32 or 8 (got {state_bits})")
        params = [p for g in self.param_groups for p in g["params"]]
        state = {}
        for k, st in d["state"].items():
            p = params[k]
            st = {n: (x.to(p.device, copy=True) if isinstance(x, torch.Tensor) else x) for n, x in st.items()}
            st["step"] = int(st["step"])
            _state_ptrs(st, p, p.numel(), "FusedAdamW.load_state_dict")
            state[p] = st
        self.state, self.state_bits = state, state_bits
        self._defaults = {"betas": betas, "eps": eps}
        self.seed, self.max_norm = d.get("seed", self.seed), d.get("max_norm", self.max_norm)
        for g, h in zip(self.param_groups, groups):
            g.update(h)

    @torch.no_grad()
    def take_rows(self, rows: torch.Tensor, fresh: torch.Tensor = None) -> list:
        """Replaces every parameter by its rows ``rows`` (``take_rows``) and moves its state along;
        ``fresh`` (bool, one per row): those rows get the initial state (densified Gaussians:
        the parent's row, no history).  Returns the new parameters in the groups' order; they
        are leaves, without gradients.  All parameters must have the same number of rows."""
        params = [p for g in self.param_groups for p in g["params"]]
        have = [p for p in params if p in self.state]
        if fresh is None:
            new, states = take_rows(params, rows, [self.state[p] for p in have])
        else:
            if fresh.dtype is not torch.bool or fresh.shape != rows.shape:
                raise RuntimeError(f"FusedAdamW.take_rows: fresh must be {rows.numel()} bools, got {fresh.dtype} "
                                   f"{tuple(fresh.shape)}")
            new = take_rows(params, rows)
            _, states = take_rows([], torch.where(fresh, -1, rows), [self.state[p] for p in have])
        new = [torch.nn.Parameter(q, p.requires_grad) if isinstance(p, torch.nn.Parameter) else
               q.requires_grad_(p.requires_grad) for p, q in zip(params, new)]
        old = dict(zip(params, new))
        self.state = {old[p]: st for p, st in zip(have, states)}
        for g in self.param_groups:
            g["params"] = [old[p] for p in g["params"]]
        return new


# ------------------------------------------------------------------ eviction to a budget
def select_rows(score: torch.Tensor, budget: int, protect: torch.Tensor = None) -> torch.Tensor:
    """The rows that stay when a model is evicted to ``budget`` rows by an accumulated weight:
    the indices (int64, ascending) of the min(budget, P) largest of ``score`` ([P] or [P,1],
    float32).  Of equal scores the lowest index stays; NaN is below every number; rows with
    ``protect`` (bool, P of them) stay before all others.  The host does not wait."""
    lib = _C.load_library()
    _cuda(score, "select_rows")
    P = score.numel()
    if score.dim() not in (1, 2) or score.shape[0] != P:
        raise RuntimeError(f"select_rows: score must be [P] or [P,1], got {tuple(score.shape)}")
    if isinstance(budget, bool) or not isinstance(budget, int) or budget < 0:
        raise ValueError(f"select_rows: budget must be an int >= 0 (got {budget!r})")
    if P >= 1 << 31:
        raise RuntimeError(f"select_rows: at most 2^31 - 1 rows (got {P})")
    if protect is not None and (protect.dtype is not torch.bool or protect.numel() != P or
                                protect.device != score.device):
        raise RuntimeError(f"select_rows: protect must be {P} bools on {score.device}, got {protect.dtype} "
                           f"{tuple(protect.shape)} on {protect.device}")
    dev = score.device
    with _on(dev):
        s = score.resolve_neg().contiguous()
        pr = None if protect is None else protect.contiguous()
        rows = torch.empty(min(budget, P), dtype=torch.int64, device=dev)
        if rows.numel():
            scratch = torch.empty(lib.gsr_select_rows_scratch_bytes(P), dtype=torch.uint8, device=dev)
            _C._check(lib.gsr_select_rows(s.data_ptr(), None if pr is None else pr.data_ptr(), P, rows.numel(),
                                          rows.data_ptr(), scratch.data_ptr(), _raw_stream(dev.index)),
                      "gsr_select_rows")
    return rows


def take_rows(tensors, rows: torch.Tensor, states=None):
    """``[t[rows] for t in tensors]`` for tensors of any dtype, as new tensors of up to 2^34 bytes
    each (2^33 of an 8-bit state) without gradient history.  ``rows``: int64 [K], any order,
    repeats allowed; an index outside [0, P) gives a row of zeros (-1: a fresh row).  With
    ``states`` (AdamW state dicts of tensors with P rows, ``adamw_state``) returns (tensors,
    states): the states' rows, with ``step`` kept; 8-bit values are re-blocked under new scales,
    which changes a value only where it is below 2^-13 of its new block's largest.  One launch
    takes up to 40 tensors, where a state counts as two."""
    lib = _C.load_library()
    if rows.dtype is not torch.int64 or rows.dim() != 1 or not rows.is_cuda:
        raise RuntimeError(f"take_rows: rows must be an int64 vector on the GPU, got {rows.dtype} {tuple(rows.shape)} "
                           f"on {rows.device}")
    dev, at, K = rows.device, rows.get_device(), rows.numel()
    if K >= 1 << 31:
        raise RuntimeError(f"take_rows: at most 2^31 - 1 rows (got {K})")
    tensors, states = list(tensors), None if states is None else list(states)
    for t in tensors + [st["exp_avg"] for st in states or ()]:
        if t.dim():
            P = t.shape[0]
            break
    else:
        P = 0
    segs, keep, out, new_states = [], [], [], []

    def refuse(t):
        raise RuntimeError(f"take_rows: tensors must have the same number of rows and be on {dev}, got "
                           f"{tuple(t.shape)} on {t.device} beside {P} rows")

    def coded(codes, src, scale, src_scale, kind):
        s = codes.shape
        if codes.get_device() != at or not s or s[0] != P:
            refuse(codes)
        row = codes.numel() // P if P else math.prod(s[1:])
        new = codes.new_empty((K, *s[1:]))
        sc = scale.new_empty(-(-K * row // SCALE_BLOCK))
        segs.extend((src, new.data_ptr(), src_scale, sc.data_ptr(), row, kind))
        return new, sc

    with _on(dev):
        if not rows.is_contiguous():
            rows = rows.contiguous()
        plain = tensors
        for st in states or ():
            m = st["exp_avg"]
            bits, mp, vp, msp, vsp = _state_ptrs(st, m, m.numel(), "take_rows", raw=False)
            got = {"step": st["step"]}
            new_states.append(got)
            if bits == 32:
                plain = plain + [m, st["exp_avg_sq"]]
            else:
                got["exp_avg"], got["exp_avg_scale"] = coded(m, mp, st["exp_avg_scale"], msp, _C.ROWS_E4M3_SIGNED)
                got["exp_rms"], got["exp_rms_scale"] = coded(st["exp_rms"], vp, st["exp_rms_scale"], vsp, _C.ROWS_E4M3)
        for t in plain:
            s = t.shape
            if t.get_device() != at or not s or s[0] != P:
                refuse(t)
            if not t.is_contiguous() or t.is_conj() or t.is_neg():
                t = t.resolve_conj().resolve_neg().contiguous()
                keep.append(t)  # until the launch
            new = t.new_empty((K, *s[1:]))
            out.append(new)
            segs += (t.data_ptr(), new.data_ptr(), 0, 0, t.nbytes // P if P else math.prod(s[1:]) * t.element_size(),
                     _C.ROWS_PLAIN)
        moments = iter(out[len(tensors):])
        del out[len(tensors):]
        for got in new_states:
            if len(got) == 1:
                got["exp_avg"], got["exp_avg_sq"] = next(moments), next(moments)
        if K and segs:
            count = len(segs) // 6  # gsr_rows_segment's fields, the last two as one
            _C._check(lib.gsr_take_rows(struct.pack(f"{6 * count}q", *segs), count, P, rows.data_ptr(), K,
                                        _raw_stream(at)), "gsr_take_rows")
    return out if states is None else (out, new_states)


@torch.no_grad()
def densify_stats(radii: torch.Tensor, viewspace_grad: torch.Tensor, max_radii2D: torch.Tensor,
                  xyz_gradient_accum: torch.Tensor, denom: torch.Tensor):
    """In place, for radii > 0: max_radii2D = max(max_radii2D, radii); xyz_gradient_accum += |grad[:, :2]|;
    denom += 1 (train.py:126-127, scene/gaussian_model.py:565-581)."""
    lib = _C.load_library()
    for t, n in ((viewspace_grad, "viewspace_grad"), (max_radii2D, "max_radii2D"),
                 (xyz_gradient_accum, "xyz_gradient_accum"), (denom, "denom")):
        _cuda(t, f"densify_stats({n})")
    P = radii.shape[0]
    for t, n, shape in ((max_radii2D, "max_radii2D", (P,)), (xyz_gradient_accum, "xyz_gradient_accum", (P, 1)),
                        (denom, "denom", (P, 1))):
        # updated in place through their data pointers: a strided view would be misread
        if not t.is_contiguous() or t.dtype != torch.float32 or t.numel() != P:
            raise RuntimeError(f"densify_stats: {n} must be a contiguous float32 tensor of {P} elements "
                               f"(shape {shape}), got {tuple(t.shape)} {t.dtype}")
    vg = viewspace_grad.contiguous()
    _C._check(lib.gsr_densify_stats(P, radii.contiguous().data_ptr(), vg.data_ptr(), vg.shape[1],
                                    max_radii2D.data_ptr(), xyz_gradient_accum.data_ptr(), denom.data_ptr(),
                                    _C._stream(radii.device)), "gsr_densify_stats")


def dist_knn3(points: torch.Tensor) -> torch.Tensor:
    """distCUDA2(points): [P] mean of the squared distances from each point to its three
    nearest other points (FLT_MAX stands in for missing neighbours when P < 4)."""
    lib = _C.load_library()
    _cuda(points, "dist_knn3")
    if points.dim() != 2 or points.shape[1] != 3:
        raise RuntimeError(f"dist_knn3: points must be [P,3], got {tuple(points.shape)}")
    pts = points.detach().contiguous()
    P = pts.shape[0]
    out = torch.empty(P, dtype=torch.float32, device=pts.device)
    if P == 0:
        return out
    scratch = torch.empty(lib.gsr_knn_scratch_bytes(P), dtype=torch.uint8, device=pts.device)
    _C._check(lib.gsr_knn_mean_dist2(P, pts.data_ptr(), out.data_ptr(), scratch.data_ptr(), _C._stream(pts.device)),
              "gsr_knn_mean_dist2")
    return out


SH_C0 = 0.28209479177387814


def create_from_pcd(points, colors, max_sh_degree: int, device="cuda"):
    """GaussianModel.create_from_pcd (scene/gaussian_model.py:133-174) -> SynthGaussians:
    DC = RGB2SH(colors), higher SH zero, log scale = log(sqrt(max(dist_knn3, 1e-7))) x3,
    identity rotation, opacity = inverse_sigmoid(0.1)."""
    from synthetic import SynthGaussians

    xyz = torch.as_tensor(np.asarray(points), dtype=torch.float32).to(device)
    rgb = torch.as_tensor(np.asarray(colors), dtype=torch.float32).to(device)
    P = xyz.shape[0]
    M = (max_sh_degree + 1) ** 2
    features = torch.zeros((P, 3, M), dtype=torch.float32, device=device)
    features[:, :3, 0] = (rgb - 0.5) / SH_C0
    dist2 = torch.clamp_min(dist_knn3(xyz), 0.0000001)
    scales = torch.log(torch.sqrt(dist2))[..., None].repeat(1, 3)
    rots = torch.zeros((P, 4), device=device)
    rots[:, 0] = 1
    op = torch.full((P, 1), 0.1, dtype=torch.float32, device=device)
    opacities = torch.log(op / (1 - op))
    return SynthGaussians(xyz, features[:, :, 0:1].transpose(1, 2).contiguous(),
                          features[:, :, 1:].transpose(1, 2).contiguous(), scales, rots, opacities,
                          max_sh_degree, 0)
