"""Optimiser of a training step: AdamW over lists of tensors (one update launch for up to 384), and the norm of all gradients.

``adamw_step`` / ``grad_norm`` are the functional forms over lists of tensors; ``AdamW`` is the ``torch.optim.Optimizer`` on top of
them.  Everything a step depends on that changes from step to step (gradients, step counts, clipping factor, optionally the
learning rate) is read on the device, so a captured step replays correctly and nothing waits for the host.  The reference trains
its coefficients with torch.optim (modded-nanogpt/train_gpt2.py:354-372).

All tensors must be CUDA tensors: there is no CPU path.
"""
from __future__ import annotations

import ctypes
from array import array
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from . import kernels as K

BLOCK = _lib.ADAMW_BLOCK


def _uniform(what: str, ts: Sequence[torch.Tensor], dtypes, n: int, dev: int) -> torch.dtype:
    """The one type of a list of n contiguous CUDA tensors on device ``dev``; raises otherwise."""
    if len(ts) != n:
        raise RuntimeError(f"adamw_step: {n} params but {len(ts)} {what}")
    kinds = {t.dtype for t in ts}
    kind = next(iter(kinds))
    if len(kinds) != 1 or kind not in dtypes:
        raise RuntimeError(f"adamw_step: {what} must all have one type out of {sorted(str(d) for d in dtypes)}, got {sorted(str(d) for d in kinds)}")
    if {t.get_device() for t in ts} != {dev}:
        raise RuntimeError(f"adamw_step: {what} must live on cuda:{dev}")
    if False in [t.is_contiguous() for t in ts]:
        raise RuntimeError(f"adamw_step: {what} must be contiguous")
    return kind


_PARAM, _GRAD, _F32, _E4M3, _U8 = (torch.float32, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.float32,), (torch.float8_e4m3fn,), (torch.uint8,)


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps: Union[torch.Tensor, Sequence[torch.Tensor]], *,
               lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 1e-2, masters: Optional[Sequence[torch.Tensor]] = None,
               exp_avg_scales: Optional[Sequence[torch.Tensor]] = None, exp_avg_sq_scales: Optional[Sequence[torch.Tensor]] = None,
               seed: int = 0, grad_scale: Optional[torch.Tensor] = None) -> None:
    """One AdamW step over a list of contiguous tensors, in place (see rdb_adamw_step for the formula and the 8-bit formats).

    params      float32, or bfloat16 (all of one type); grads: float32 or bfloat16, same sizes.
    exp_avgs / exp_avg_sqs   float32 moments; or, with ``exp_avg_scales`` and ``exp_avg_sq_scales`` (float32, one per 256
                consecutive elements of a tensor), 8-bit moments: float8_e4m3fn and uint8 (no sign, 4 exponent and 4 mantissa bits).
    steps       float32 step counts on the device, raised by one here: one tensor with an element per param, or a list of
                one-element tensors.
    lr          a number, or a one-element float32 CUDA tensor that is read when the step runs.
    masters     float32 copies of bfloat16 params: they are updated, the params receive their rounding.
    seed        of the random rounding of the 8-bit second moments.
    grad_scale  one-element float32 CUDA tensor the gradients are multiplied with (the factor ``grad_norm`` returns).
    """
    if len(params) == 0:
        return
    state = _State(params, exp_avgs, exp_avg_sqs, steps, masters, exp_avg_scales, exp_avg_sq_scales)
    state.launch(params, grads, lr, betas, eps, weight_decay, seed, grad_scale, fresh=True)


class _State:
    """What a list of parameters keeps between steps, checked once: moments, scales, masters and counts."""

    def __init__(self, params, exp_avgs, exp_avg_sqs, steps, masters=None, exp_avg_scales=None, exp_avg_sq_scales=None):
        n = self.n = len(params)
        dev = self.dev = params[0].get_device()
        if dev < 0:
            raise RuntimeError("randumb_b200 kernels run on CUDA tensors only (no CPU implementation)")
        self.dtype = _uniform("params", params, _PARAM, n, dev)
        eight = self.eight = exp_avg_scales is not None or exp_avg_sq_scales is not None
        if eight and (exp_avg_scales is None or exp_avg_sq_scales is None):
            raise RuntimeError("adamw_step: 8-bit moments need exp_avg_scales and exp_avg_sq_scales")
        _uniform("exp_avgs", exp_avgs, _E4M3 if eight else _F32, n, dev)
        _uniform("exp_avg_sqs", exp_avg_sqs, _U8 if eight else _F32, n, dev)
        numels = self.numels = [t.numel() for t in params]
        lists = [("exp_avg", exp_avgs), ("exp_avg_sq", exp_avg_sqs)]
        if masters is not None:
            _uniform("masters", masters, _F32, n, dev)
            if self.dtype != torch.bfloat16:
                raise RuntimeError("adamw_step: masters are the float32 copies of bfloat16 params")
            lists.append(("master", masters))
        for what, ts in lists:
            if [t.numel() for t in ts] != numels:
                raise RuntimeError(f"adamw_step: {what}s and params differ in size")
        if eight:
            blocks = [-(-k // BLOCK) for k in numels]
            for what, ts in (("exp_avg_scale", exp_avg_scales), ("exp_avg_sq_scale", exp_avg_sq_scales)):
                _uniform(what + "s", ts, _F32, n, dev)
                if [t.numel() for t in ts] != blocks:
                    raise RuntimeError(f"adamw_step: scales hold one value per {BLOCK} elements of their tensor")
                lists.append((what, ts))
        if isinstance(steps, torch.Tensor):
            if steps.dtype != torch.float32 or steps.get_device() != dev or steps.numel() != n or not steps.is_contiguous():
                raise RuntimeError(f"adamw_step: steps must be {n} contiguous float32 counts on cuda:{dev}")
            at = steps.data_ptr()
            words = list(range(at, at + 4 * n, 4))
        else:
            _uniform("steps", steps, _F32, n, dev)
            if any([t.numel() != 1 for t in steps]):
                raise RuntimeError("adamw_step: every tensor has one step count")
            words = [t.data_ptr() for t in steps]
        counts = len(words)
        words += numels
        for _, ts in lists:
            words += [t.data_ptr() for t in ts]
        # every address once: two tensors in one place would be updated by two threads at a time
        at = words[:counts] + words[counts + n:]
        if len(set(at)) != len(at):
            empty = [k == 0 for k in numels]
            at = words[:counts] + [a for i, a in enumerate(words[counts + n:]) if not empty[i % n]]
            if len(set(at)) != len(at):
                raise RuntimeError("adamw_step: a step count, moment, scale or master is in the lists twice")
        self.names = ["step", "numel"] + [what for what, _ in lists]
        self.words = array("Q", words)                         # one list behind the other, in host memory
        self.keep = (steps, [ts for _, ts in lists])           # the tensors the addresses belong to
        self.masters = list(masters) if masters is not None else []
        self.some = sum(1 for k in numels if k)

    def launch(self, params, grads, lr, betas, eps, weight_decay, seed, grad_scale, fresh: bool = False) -> None:
        n, dev = self.n, self.dev
        if not fresh and (_uniform("params", params, _PARAM, n, dev) != self.dtype or [t.numel() for t in params] != self.numels):
            raise RuntimeError("adamw_step: params changed their type or size")
        gd = _uniform("grads", grads, _GRAD, n, dev)
        if [t.numel() for t in grads] != self.numels:
            raise RuntimeError("adamw_step: grads and params differ in size")
        pp = [t.data_ptr() for t in params]
        if len(set(pp)) != n and len({a for a, k in zip(pp, self.numels) if k}) != self.some:
            raise RuntimeError("adamw_step: a param is in the list twice")
        _one_float("grad_scale", grad_scale, dev)
        lr_dev = None
        if isinstance(lr, torch.Tensor):
            _one_float("lr", lr, dev)
            lr, lr_dev = 0.0, lr.data_ptr()
        pp += [t.data_ptr() for t in grads]
        moving = array("Q", pp)
        base, held = moving.buffer_info()[0], self.words.buffer_info()[0]
        arg = _lib.AdamwLists(n=n, param=base, grad=base + 8 * n, **{name: held + 8 * n * i for i, name in enumerate(self.names)})
        h = _lib.AdamwHyper(float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay), lr_dev, K._seed(seed))
        with K._on(dev):
            rc = _lib.lib().rdb_adamw_step(ctypes.byref(arg), K._dt(self.dtype), K._dt(gd), 8 if self.eight else 32, ctypes.byref(h),
                                           K._ptr(grad_scale), K._raw_stream(dev))
        _lib.check(rc, "rdb_adamw_step")
        # autograd learns that these were written: a graph that kept one refuses to run backward.  (Moments, scales and counts are in
        # no graph; raising theirs as well took a call with 93 tensors and 8-bit moments from 315 to 339 us.)
        torch.autograd.graph.increment_version([*params, *self.masters])


def _one_float(what: str, t: Optional[torch.Tensor], dev: int) -> None:
    if t is not None and (t.dtype != torch.float32 or t.numel() != 1 or t.get_device() != dev):
        raise RuntimeError(f"{what} must be a one-element float32 tensor on cuda:{dev}")


def grad_norm(grads: Sequence[torch.Tensor], max_norm: Optional[float] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(norm, factor): 2-norm over all gradients (float32 or bfloat16, contiguous, types may be mixed), and with ``max_norm`` the
    factor ``min(1, max_norm / (norm + 1e-6))`` to pass to ``adamw_step`` as ``grad_scale``.  Both are 0-d float32 tensors on the
    device; nothing is written to the gradients and nothing waits.  A gradient that holds a NaN or an infinity makes the norm
    one too, and the factor NaN or 0."""
    n = len(grads)
    if n == 0:
        raise RuntimeError("grad_norm: no gradients")
    dev = grads[0].get_device()
    if dev < 0:
        raise RuntimeError("randumb_b200 kernels run on CUDA tensors only (no CPU implementation)")
    if {t.get_device() for t in grads} != {dev}:
        raise RuntimeError("grad_norm: all gradients must live on the same device")
    if False in [t.is_contiguous() for t in grads]:
        raise RuntimeError("grad_norm: gradients must be contiguous")
    if max_norm is not None and not max_norm >= 0.0:
        raise RuntimeError(f"grad_norm: max_norm must not be negative, got {max_norm}")
    out = torch.empty((2,), dtype=torch.float32, device=grads[0].device)
    L = _lib.lib()
    ptrs, numels = array("Q", [t.data_ptr() for t in grads]), array("q", [t.numel() for t in grads])
    kinds = {d: K._dt(d) for d in {t.dtype for t in grads}}
    dtypes = array("i", [kinds[t.dtype] for t in grads])
    ws = K._workspace(L.rdb_grad_norm_workspace_bytes(n), out.device)
    clip = max_norm is not None
    with K._on(dev):
        rc = L.rdb_grad_norm(out.data_ptr(), out.data_ptr() + 4 if clip else None, ptrs.buffer_info()[0], numels.buffer_info()[0], dtypes.buffer_info()[0],
                             n, float(max_norm) if clip else 0.0, K._ptr(ws), ws.numel(), K._raw_stream(dev))
    _lib.check(rc, "rdb_grad_norm")
    return out[0], out[1] if clip else None


def second_moment_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float32 values of an 8-bit second moment (uint8 codes of ``adamw_step`` and their scales), laid out like ``codes``."""
    flat = _flat(codes)
    v = (flat.to(torch.int32) << 19).view(torch.float32) * 2.0 ** 112
    return _like(codes, v * scales.repeat_interleave(BLOCK)[:v.numel()].view(v.shape))


def first_moment_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float32 values of an 8-bit first moment (float8_e4m3fn codes of ``adamw_step`` and their scales), laid out like ``codes``."""
    v = _flat(codes).float()
    return _like(codes, v * scales.repeat_interleave(BLOCK)[:v.numel()].view(v.shape))


def _like(codes: torch.Tensor, values: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(codes, dtype=torch.float32)
    _flat(out).copy_(values)
    return out


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on two launches (step counts, update) per (parameter type, gradient type), group and 384 tensors, with 32-bit or
    8-bit moments.

    Args:
        params, lr, betas, eps, weight_decay: as torch.optim.AdamW; ``lr`` may be a one-element float32 CUDA tensor, read when the
            step runs (a schedule then works inside a captured step).
        state_bits: 32 or 8 (2 bytes and a little per element instead of 8; formats at ``adamw_step``).
        master_weights: keep a float32 copy of every bfloat16 parameter and update that (default True: with bfloat16 alone an
            update below 2^-9 of the weight is lost).  float32 parameters have none.
        max_grad_norm: clip the norm of all gradients of all groups to this value, without writing to the gradients.
        seed: of the random rounding of 8-bit second moments.

    ``step()`` returns the closure's loss; ``last_grad_norm`` holds the norm of the last step (a device tensor) with ``max_grad_norm``.
    The first step creates the state and cannot be captured (it raises); later ones can.
    """

    def __init__(self, params, lr: Union[float, torch.Tensor] = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = True, max_grad_norm: Optional[float] = None,
                 seed: int = 0):
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError(f"invalid learning rate: {lr}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"invalid betas: {betas}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError(f"invalid eps or weight_decay: {eps}, {weight_decay}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"invalid max_grad_norm: {max_grad_norm}")
        self.max_grad_norm, self.seed, self.last_grad_norm = max_grad_norm, int(seed), None
        self._lists: dict = {}                                      # (group, kind) -> state tensors of the parameters with a gradient, their lists
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, master_weights=master_weights))

    def add_param_group(self, param_group) -> None:
        _refuse_options({**self.defaults, **param_group})
        super().add_param_group(param_group)

    def _new_state(self, p: torch.Tensor, group: dict) -> dict:
        if p.dtype not in (torch.float32, torch.bfloat16) or not p.is_cuda:
            raise RuntimeError(f"AdamW takes float32 and bfloat16 CUDA parameters, got {p.dtype} on {p.device}")
        _flat(p)                                                    # refuses a parameter whose elements are not one block of memory
        st = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        if group["state_bits"] == 32:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        else:
            blocks = -(-p.numel() // BLOCK)
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.uint8).view(torch.float8_e4m3fn)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.uint8)
            st["exp_avg_scale"] = torch.zeros((blocks,), dtype=torch.float32, device=p.device)
            st["exp_avg_sq_scale"] = torch.zeros((blocks,), dtype=torch.float32, device=p.device)
        if p.dtype == torch.bfloat16 and group["master_weights"]:
            st["master"] = p.detach().float()
        return st

    def __getstate__(self) -> dict:                                 # copies and pickles; the lists are made again
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "seed": self.seed, "last_grad_norm": self.last_grad_norm}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        self._lists = {}

    def _state_of(self, key, params: list, group: dict, master: bool) -> _State:
        """The checked lists of these parameters' states; kept while the same parameters have gradients and the same tensors, in the
        same places, as state."""
        sts = [self.state[p] for p in params]
        have = self._lists.get(key)
        parts = [v for s in sts for v in s.values()]
        at = [t.data_ptr() for t in parts]
        if have is not None and at == have[2] and all([a is b for a, b in zip(have[0], parts)]):
            return have[1]
        eight = {}
        if group["state_bits"] == 8:
            eight = dict(exp_avg_scales=[s["exp_avg_scale"] for s in sts], exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in sts])
        made = _State([_flat(p) for p in params], [_flat(s["exp_avg"]) for s in sts], [_flat(s["exp_avg_sq"]) for s in sts], [s["step"] for s in sts],
                      [_flat(s["master"]) for s in sts] if master else None, **eight)
        self._lists[key] = (parts, made, at)
        return made

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        todo, all_grads = [], {}
        for gi, group in enumerate(self.param_groups):
            kinds: dict = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                st = self.state[p]
                if not st:
                    if g.is_sparse:
                        raise RuntimeError("AdamW does not take sparse gradients")
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: a parameter's first step creates its state and cannot be captured (a replay would begin again from "
                                           "zero): take one step first")
                    st.update(self._new_state(p, group))
                if p.is_contiguous() and g.is_contiguous() and g.dtype in _GRAD:
                    flat, g = p, g.detach()
                else:
                    if g.is_sparse:
                        raise RuntimeError("AdamW does not take sparse gradients")
                    if g.stride() != p.stride() or g.dtype not in _GRAD:
                        g = torch.empty_like(p).copy_(g)               # the parameter's own order of elements
                    flat, g = _flat(p), _flat(g)
                ps, flats, gs = kinds.setdefault((p.device, p.dtype, g.dtype, "master" in st), ([], [], []))
                ps.append(p)
                flats.append(flat)
                gs.append(g)
            for kind, (ps, flats, gs) in kinds.items():
                todo.append((gi, group, kind, ps, flats, gs))
                all_grads.setdefault(kind[0], []).extend(gs)
        scale = None
        if self.max_grad_norm is not None and all_grads:
            if len(all_grads) > 1:
                raise RuntimeError("max_grad_norm: the parameters must live on one device")
            self.last_grad_norm, scale = grad_norm(next(iter(all_grads.values())), self.max_grad_norm)
        for k, (gi, group, kind, ps, flats, gs) in enumerate(todo):
            self._state_of((gi,) + kind, ps, group, kind[3]).launch(flats, gs, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                                                                    self.seed + 0x632BE5AB * k, scale)
        return loss

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but every state tensor keeps its own type (moments and masters of a bfloat16 parameter are not bfloat16).  The
        groups' hyperparameters, ``state_bits`` and ``master_weights`` among them, become the checkpoint's; what a checkpoint of
        torch.optim.AdamW does not have keeps this optimiser's values, and its float32 moments load into 32-bit ones.  Options that
        this optimiser does not have (``maximize``, ``amsgrad``, ``differentiable``, torch.optim.Adam's weight decay) are refused.  A checkpoint that does not load
        changes nothing."""
        here = [dict(g) for g in self.param_groups]
        for group, old in zip(state_dict["param_groups"], here):
            _refuse_options({**old, **group})
        before = self.state, self.param_groups
        try:
            super().load_state_dict(state_dict)
            self._load_own(state_dict, here)
        except Exception:                                           # as it was
            self.state, self.param_groups = before
            raise
        finally:
            self._lists = {}

    def _load_own(self, state_dict, here: list) -> None:
        for group, old in zip(self.param_groups, here):
            for k in ("state_bits", "master_weights"):
                group.setdefault(k, old[k])
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        places = [(p, g) for g in self.param_groups for p in g["params"]]
        for i, (p, group) in zip(ids, places):
            if i not in state_dict["state"]:
                continue
            src, dst = state_dict["state"][i], self._new_state(p, group)
            if set(src) != set(dst):
                raise RuntimeError(f"AdamW: the checkpoint holds {sorted(src)} for a parameter whose state is {sorted(dst)}: other state_bits or masters")
            for k, t in dst.items():
                v = src[k] if isinstance(src[k], torch.Tensor) else torch.tensor(float(src[k]))
                if v.dtype != t.dtype or v.numel() != t.numel():
                    raise RuntimeError(f"AdamW: {k} is {v.dtype} of {v.numel()} in the checkpoint, {t.dtype} of {t.numel()} here")
                if "exp_avg_scale" in dst and v.dim() and not v.is_contiguous() == t.is_contiguous():
                    raise RuntimeError("AdamW: the checkpoint's parameter has its elements in another order, which 8-bit moments cannot follow")
                if t.dtype == torch.float8_e4m3fn:
                    t, v = t.view(torch.uint8), v.view(torch.uint8)
                t.copy_(v.reshape(t.shape))
            self.state[p] = dst


def _refuse_options(group: dict) -> None:
    """Raises for what torch's optimisers can do and ``step`` would leave undone."""
    for k in ("maximize", "amsgrad", "differentiable"):
        if group.get(k):
            raise ValueError(f"AdamW does not have the option {k}")
    if not group.get("decoupled_weight_decay", True) and group["weight_decay"] != 0:
        raise ValueError("AdamW's weight decay is decoupled from the gradient; the group asks for torch.optim.Adam's")
    if group["state_bits"] not in (8, 32):
        raise ValueError(f"state_bits must be 8 or 32, got {group['state_bits']}")


def _flat(t: torch.Tensor) -> torch.Tensor:
    """The elements of a dense tensor in memory order (any permutation of its dimensions)."""
    t = t.detach()
    if t.is_contiguous():
        return t
    acc = 1
    for size, stride in sorted(((n, st) for n, st in zip(t.shape, t.stride()) if n > 1), key=lambda x: x[1]):
        if stride != acc:
            raise RuntimeError("AdamW needs parameters whose elements are one block of memory")
        acc *= size
    return t.as_strided((t.numel(),), (1,))
