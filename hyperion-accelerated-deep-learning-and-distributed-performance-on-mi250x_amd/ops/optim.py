"""Fused multi-tensor Adam / AdamW on gfx950 (one launch for every parameter).

Reference optimizers: ``optim.Adam(lr=1e-3)`` in the baseline step benchmark
(``baseline_performance.ipynb:282``) and ``AdamW`` in every trainer (``distributed_utils.py:161,
232,334,503``).  torch's implementation launches a chain of ``_foreach_*`` kernels per parameter
group chunk; ``FusedAdam`` runs ``adam_mt_k`` once, reading step / loss-scale / found-inf from
device memory so the step can be captured in a hipGraph and skipped on overflow without a host
sync (GradScaler semantics).

Low-precision parameters (bf16/fp16 — "compute copies") get an fp32 master copy in the optimizer
state; the kernel updates the master and rewrites the compute copy in the same pass.  This lets a
model run its convolutions/GEMMs on bf16 weights directly (no per-forward autocast weight casts,
no bf16→fp32 grad casts in backward) while the optimizer math stays in fp32.

``state_bits=8`` holds the two moments in 8 bits (``csrc/kernels/adam8.hip``): 2 bytes and 8 bytes per
256 elements instead of 8 bytes a parameter.  Blocks of 256 elements share an fp32 scale, the block's
largest magnitude; the first moment is coded by the square root of its share of it, the second by the
fourth root.  Everything else (masters, scalars on the device, skipped steps, the deferred clip) is as
with 32 bits, and ``moment_vectors`` gives the values.

Also provides multi-tensor global-norm clipping that takes the norm over *all* gradient shards
(all-reduced when a process group is given) — the reference clipped only the local FSDP shard
(``distributed_utils.py:351,522``).
"""
from __future__ import annotations

import math
import weakref
from typing import Iterable, List, Optional, Tuple

import torch
import torch.distributed as dist

from . import _native
from .multi_tensor import TableCache


def grad_of(p: torch.Tensor) -> Optional[torch.Tensor]:
    """The gradient the optimizer should consume: ``p.main_grad`` (an fp32 reduced-gradient view
    that data-parallel wrappers attach to low-precision parameters, ``parallel/ddp.py``) when set,
    else ``p.grad``."""
    g = getattr(p, "main_grad", None)
    return g if g is not None else p.grad


def _dense(t: torch.Tensor) -> bool:
    return t.is_contiguous() or (t.dim() == 4 and t.is_contiguous(memory_format=torch.channels_last))


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Same element order in memory (strides of size-1 dims are irrelevant: a [K, C, 1, 1] weight is
    'contiguous' and 'channels-last' at once, and autograd may hand back either stride set)."""
    return a.shape == b.shape and all(sa == sb for sa, sb, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


# ---- 8-bit moments (state_bits=8): the PyTorch path and oracle of adam8.hip ------------------------
STATE_BLOCK = 256  # elements that share a scale (adam8.hip)
_STATE8 = ("exp_avg_q", "exp_avg_sq_q", "exp_avg_scale", "exp_avg_sq_scale")


def _channels_last(p: torch.Tensor) -> bool:
    return p.dim() == 4 and not p.is_contiguous() and p.is_contiguous(memory_format=torch.channels_last)


def _memory_order(t: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    """``t`` flat in the order that the blocks of ``like``'s moments follow: its memory order (channels-last
    4-D parameters), else row-major.  A view where the layout allows it."""
    return (t.permute(0, 2, 3, 1) if _channels_last(like) else t).reshape(-1)


def _in_blocks(x: torch.Tensor) -> torch.Tensor:
    return torch.nn.functional.pad(x, (0, -x.numel() % STATE_BLOCK)).view(-1, STATE_BLOCK)


def _unit(levels: int, second: bool) -> float:
    """What a block's largest magnitude is multiplied with: a product, as quotients by a number differ between CPU and GPU."""
    return 1.0 / float(levels) ** (4 if second else 2)


def _encode8(x: torch.Tensor, levels: int, second: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp64 [n] -> (codes [n], fp32 scales).  As in the kernel, the root only finds k = floor(r) and x is then compared
    with the border of k and k + 1, which itself belongs to k."""
    b = _in_blocks(x)
    s = b.abs().amax(1).float() if b.numel() else b.new_zeros(0).float()
    s = torch.where(s < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    s = torch.where(torch.isfinite(s), s, torch.full_like(s, math.nan))
    live = (s > 0)[:, None]
    unit = torch.where(live, s.double()[:, None] * _unit(levels, second), torch.zeros_like(b))
    r = torch.where(live, b.abs() / s.double()[:, None], torch.zeros_like(b)).sqrt()
    k = torch.floor((r.sqrt() if second else r) * levels).clamp(max=levels)
    h = (k + 0.5) * (k + 0.5) if second else k * k + k + 0.25
    q = torch.where(live, k + (b.abs() > unit * (h * h if second else h)), torch.zeros_like(b))
    if second:
        q = torch.where(live & (b > 0) & (q < 1), torch.ones_like(q), q)
    else:
        q = torch.where(b < 0, -q, q)
    return q.to(torch.uint8 if second else torch.int8).view(-1)[:x.numel()], s


def _decode8(q: torch.Tensor, s: torch.Tensor, levels: int, second: bool) -> torch.Tensor:
    b = _in_blocks(q.double())
    b = b * b * (b * b if second else torch.sign(b))
    return (b * (s.double() * _unit(levels, second))[:, None]).view(-1)[:q.numel()]


def _row_major(x: torch.Tensor, moved) -> torch.Tensor:
    """``x`` (dense moments) with the stretches of channels-last parameters put into row-major order, in place."""
    for a, (n, c, h, w) in moved:
        part = x[a:a + n * c * h * w]
        part.copy_(part.view(n, h, w, c).permute(0, 3, 1, 2).reshape(-1))
    return x


class FusedAdam(torch.optim.Optimizer):
    def __init__(
        self,
        params: Iterable,
        lr: float = 1e-3,
        betas=(0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 0.0,
        adamw: bool = False,
        zero_grad_in_step: bool = False,
        state_bits: int = 32,
    ):
        """``zero_grad_in_step``: the kernel writes zeros over each gradient as it consumes it, so
        ``zero_grad(set_to_none=False)`` before the next backward is free (one fill kernel per
        parameter saved — 256 launches per step for Llama LoRA under hipGraph capture).
        ``state_bits``: 32 (fp32 moments) or 8 (coded moments, module docstring)."""
        if state_bits not in (8, 32):
            raise ValueError(f"FusedAdam: state_bits must be 8 or 32, got {state_bits}")
        if state_bits == 8 and not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"FusedAdam: betas must be in [0, 1), got {betas}")
        self.state_bits = state_bits
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, adamw=adamw)
        super().__init__(params, defaults)
        self.zero_grad_in_step = zero_grad_in_step
        self._tables = TableCache()
        self._plan8 = None  # 8-bit states: (fingerprint, launches) of the last step that ran on the kernels alone
        self._fits8 = None  # 8-bit states: the parameters and states (fingerprint) that _check8 let pass last
        self._values8 = None  # (fingerprint, table, its key, elements, channels-last stretches) of moment_vectors
        self._step_t: Optional[torch.Tensor] = None
        self._host_step = 0
        # optional device scalars set by the AMP scaler
        self.inv_scale: Optional[torch.Tensor] = None
        self.found_inf: Optional[torch.Tensor] = None
        # a global-norm clip coefficient left for this step by clip_grad_norm_(defer_to=self): the
        # kernel applies it while it reads the gradients (no separate scaling pass); consumed by step()
        self.clip_coef: Optional[torch.Tensor] = None

    def _state(self, p: torch.Tensor):
        st = self.state[p]
        if not st and self.state_bits == 8:
            n, nb = p.numel(), -(-p.numel() // STATE_BLOCK)
            st["exp_avg_q"] = torch.zeros(n, dtype=torch.int8, device=p.device)
            st["exp_avg_sq_q"] = torch.zeros(n, dtype=torch.uint8, device=p.device)
            st["exp_avg_scale"] = torch.zeros(nb, dtype=torch.float32, device=p.device)
            st["exp_avg_sq_scale"] = torch.zeros(nb, dtype=torch.float32, device=p.device)
            st["channels_last"] = _channels_last(p)  # the order of the blocks
            if p.dtype != torch.float32:
                st["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format).clone()
        if not st:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
            if p.dtype != torch.float32:
                st["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format).clone()
        return st

    def zero_grad(self, set_to_none: bool = True) -> None:
        if self.zero_grad_in_step and not set_to_none:
            return  # the last step already zeroed every gradient it consumed
        super().zero_grad(set_to_none=set_to_none)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.state_bits == 8 and self._plan8 is not None and self._replay8():
            return loss
        if self.state_bits == 8:
            self._check8()
        self._host_step += 1
        launches = []  # 8-bit partitions; None once one of them took the reference path
        first = next((p for g in self.param_groups for p in g["params"] if grad_of(p) is not None), None)
        if first is None:
            return loss
        native = _native.use_native(first, op="adam")
        inv_scale = self.inv_scale
        if self.clip_coef is not None:
            inv_scale = self.clip_coef if inv_scale is None else self.clip_coef * inv_scale
            self.clip_coef = None
        if native:
            if self._step_t is None or self._step_t.device != first.device:
                self._step_t = torch.full((), float(self._host_step - 1), dtype=torch.float32, device=first.device)
            self._step_t.add_(1.0)
        for gi, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if grad_of(p) is not None]
            # partition by (param dtype, grad dtype): one launch per partition (an fp32 main_grad
            # of a bf16 parameter is its own partition: fp32 grads, bf16 params + fp32 masters)
            parts = {}
            for p in params:
                parts.setdefault((p.dtype, grad_of(p).dtype), []).append(p)
            for (pdt, gdt), ps in parts.items():
                sts = [self._state(p) for p in ps]
                gs = [grad_of(p) for p in ps]
                if self.state_bits == 8:
                    done = self._step8(f"adam8_{gi}_{pdt}_{gdt}", gi, ps, gs, sts, inv_scale, native)
                    launches = None if done is None or launches is None else launches + [done]
                    continue
                ms = [s["exp_avg"] for s in sts]
                vs = [s["exp_avg_sq"] for s in sts]
                masters = [s["master"] for s in sts] if pdt != torch.float32 else None
                ok = native and pdt in _native.DTYPE_CODE and gdt in _native.DTYPE_CODE and all(
                    (g.stride() == p.stride() and m.stride() == p.stride() and p.is_contiguous())  # fast path
                    or (_dense(p) and _dense(g) and _same_layout(p, g) and _same_layout(p, m))
                    for p, g, m in zip(ps, gs, ms)
                )
                if ok:
                    groups = [ps, gs, ms, vs] + ([masters] if masters is not None else [])
                    try:
                        tab = self._tables.get(f"adam{gi}_{pdt}_{gdt}", groups)
                    except ValueError:  # misaligned tensor -> reference path
                        ok = False
                if ok:
                    lr = group["lr"]
                    lr_t = lr if isinstance(lr, torch.Tensor) else None
                    b1, b2 = group["betas"]
                    _native.native().adam_mt(
                        tab.ptrs, tab.sizes, tab.blocks, tab.T, tab.chunk,
                        float(lr) if lr_t is None else 0.0, b1, b2, group["eps"], group["weight_decay"],
                        bool(group["adamw"]), lr_t, self._step_t, inv_scale, self.found_inf,
                        _native.DTYPE_CODE[gdt], _native.DTYPE_CODE[pdt], bool(self.zero_grad_in_step),
                    )
                else:
                    self._reference_step(group, ps, gs, ms, vs, masters, inv_scale)
                    if self.zero_grad_in_step:
                        for g in gs:
                            g.zero_()
        if self.state_bits == 8:
            self._plan8 = (self._fingerprint8(), launches) if launches else None
        return loss

    def _fingerprint8(self) -> bytes:
        return _native.native().optim_fingerprint(self.param_groups, self.state, _STATE8 + ("master",), True)

    def _replay8(self) -> bool:
        """The step from the last one's tables, where nothing that they depend on has changed: with hundreds of small
        tensors going through them in Python takes longer than the step."""
        launches = self._plan8[1]
        if _native.backend() == "torch" or "adam" in _native.torch_ops() or self._fingerprint8() != self._plan8[0]:
            return False
        if any(tab.key is not key for _, _, tab, key, _, _ in launches):
            return False  # re-pointed meanwhile
        self._host_step += 1
        inv_scale = self.inv_scale
        if self.clip_coef is not None:
            inv_scale = self.clip_coef if inv_scale is None else self.clip_coef * inv_scale
            self.clip_coef = None
        if self._step_t is None:
            self._step_t = torch.full((), float(self._host_step - 1), dtype=torch.float32, device=launches[0][2].ptrs.device)
        self._step_t.add_(1.0)
        capturing = torch.cuda.is_current_stream_capturing()
        for role, gi, tab, _, gdt, pdt in launches:
            if capturing:
                self._tables.pin(role, tab)
            self._launch8(gi, tab, gdt, pdt, inv_scale)
        return True

    def _launch8(self, gi, tab, gdt, pdt, inv_scale) -> None:
        group = self.param_groups[gi]
        lr = group["lr"]
        lr_t = lr if isinstance(lr, torch.Tensor) and lr.is_cuda else None
        b1, b2 = group["betas"]
        _native.count("adam8")
        _native.native().adam8_mt(
            tab.ptrs, tab.sizes, tab.blocks, tab.T, tab.chunk, float(lr) if lr_t is None else 0.0, b1, b2,
            group["eps"], group["weight_decay"], bool(group["adamw"]), lr_t, self._step_t, inv_scale, self.found_inf,
            _native.DTYPE_CODE[gdt], _native.DTYPE_CODE[pdt], bool(self.zero_grad_in_step))

    def _check8(self) -> None:
        """Refuses a step whose states do not fit the parameters, before anything of it has run: the kernels trust what
        the state says."""
        # (one pass in C++ where they are those of the last step that fitted)
        fingerprint = self._values_fingerprint() if self._step_t is not None else None
        if fingerprint is not None and fingerprint == self._fits8:
            return
        for group in self.param_groups:
            for p in group["params"]:
                st = self.state.get(p)
                if st and (st["exp_avg_q"].numel() != p.numel() or st["exp_avg_q"].device != p.device
                           or st["channels_last"] != _channels_last(p)):
                    if grad_of(p) is not None:
                        raise ValueError(f"FusedAdam(state_bits=8): a parameter (now {tuple(p.shape)}, strides {p.stride()}, "
                                         f"on {p.device}) changed its size, memory format or device after its first step")
                    fingerprint = None  # (not of this step)
        self._fits8 = fingerprint

    def _step8(self, role, gi, ps, gs, sts, inv_scale, native):
        """One partition (a parameter dtype and a gradient dtype) with 8-bit moments; the launch, or None where the
        reference path ran."""
        pdt, gdt = ps[0].dtype, gs[0].dtype
        tab = None
        if native and pdt in _native.DTYPE_CODE and gdt in _native.DTYPE_CODE and all(
                p.device == self._step_t.device and _dense(p) and _dense(g) and _same_layout(p, g)
                and (pdt == torch.float32 or _same_layout(p, st["master"])) for p, g, st in zip(ps, gs, sts)):
            groups = [ps, gs] + [[s[k] for s in sts] for k in _STATE8]
            if pdt != torch.float32:
                groups.append([s["master"] for s in sts])
            try:
                tab = self._tables.get(role, groups)
            except ValueError:  # misaligned tensor -> reference path
                pass
        if tab is not None:
            self._launch8(gi, tab, gdt, pdt, inv_scale)
            return role, gi, tab, tab.key, gdt, pdt
        self._reference_step8(self.param_groups[gi], ps, gs, sts, inv_scale)
        if self.zero_grad_in_step:
            for g in gs:
                g.zero_()
        return None

    def _reference_step8(self, group, ps, gs, sts, inv_scale=None):
        """PyTorch reference of the 8-bit step (CPU / fallback): moments and codes in fp64."""
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("FusedAdam: reference path reached during hipGraph capture (grad/param layouts "
                               "or dtypes outside the fused kernel's envelope)")
        if self.found_inf is not None and float(self.found_inf) != 0.0:
            return
        b1, b2 = group["betas"]
        lr, wd, eps = float(group["lr"]), group["weight_decay"], group["eps"]
        bc1, bc2_sqrt = 1 - b1**self._host_step, math.sqrt(1 - b2**self._host_step)
        inv = float(inv_scale) if inv_scale is not None else 1.0
        for p, g, st in zip(ps, gs, sts):
            w = st.get("master", p)
            flat = _memory_order(w, p).float()
            g = (_memory_order(g, p).float() * inv).double()
            if group["adamw"]:
                flat = flat * (1 - lr * wd)
            elif wd != 0:
                g = g + flat.double() * wd
            m = _decode8(st["exp_avg_q"], st["exp_avg_scale"], 127, False) * b1 + g * (1 - b1)
            v = _decode8(st["exp_avg_sq_q"], st["exp_avg_sq_scale"], 255, True) * b2 + g * g * (1 - b2)
            flat = (flat.double() - lr / bc1 * (m / (v.sqrt() / bc2_sqrt + eps))).float()
            for x, levels, second, key in ((m, 127, False, "exp_avg"), (v, 255, True, "exp_avg_sq")):
                q, s = _encode8(x, levels, second)
                st[key + "_q"].copy_(q)
                st[key + "_scale"].copy_(s)
            if _channels_last(p):
                flat = flat.view(p.shape[0], p.shape[2], p.shape[3], p.shape[1]).permute(0, 3, 1, 2)
            w.copy_(flat.view(p.shape) if not _channels_last(p) else flat)
            if w is not p:
                p.copy_(w)

    @torch.no_grad()
    def moment_vectors(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The first and second moments of every parameter that has been stepped, as two fp32 vectors: the
        parameters in order, each row-major (like ``torch.nn.utils.parameters_to_vector``)."""
        if self.state_bits == 8 and self._values8 is not None and _native.backend() != "torch":
            fingerprint, tab, key, total, moved = self._values8
            if tab.key is key and self._values_fingerprint() == fingerprint:
                return self._values_native(tab, total, moved)
        ps = [p for g in self.param_groups for p in g["params"] if self.state.get(p)]
        sts = [self.state[p] for p in ps]
        if not ps:
            return torch.zeros(0), torch.zeros(0)
        if self.state_bits == 32:
            return tuple(torch.cat([s[k].reshape(-1) for s in sts]) for k in ("exp_avg", "exp_avg_sq"))
        sizes = [p.numel() for p in ps]
        starts = [0]
        for n in sizes:
            starts.append(starts[-1] + n)
        moved = [(a, p.shape) for a, p in zip(starts, ps) if _channels_last(p)]  # coded in memory order
        tab = None
        if _native.use_native(*ps, op="adam") and all(p.device == ps[0].device for p in ps):
            try:
                tab = self._tables.get("adam8_values", [[s[k] for s in sts] for k in _STATE8])
            except ValueError:
                pass
        if tab is not None:
            if getattr(tab, "offs", None) is None:
                tab.offs = torch.tensor(starts[:-1]).to(ps[0].device)
            self._values8 = (self._values_fingerprint(), tab, tab.key, starts[-1], moved)
            return self._values_native(tab, starts[-1], moved)
        m = torch.cat([_decode8(s["exp_avg_q"], s["exp_avg_scale"], 127, False).float() for s in sts])
        v = torch.cat([_decode8(s["exp_avg_sq_q"], s["exp_avg_sq_scale"], 255, True).float() for s in sts])
        return _row_major(m, moved), _row_major(v, moved)

    def _values_fingerprint(self) -> bytes:
        return _native.native().optim_fingerprint(self.param_groups, self.state, _STATE8, False)

    def _values_native(self, tab, total, moved):
        if torch.cuda.is_current_stream_capturing():
            self._tables.pin("adam8_values", tab)
        m, v = _native.native().adam8_values(tab.ptrs, tab.sizes, tab.blocks, tab.offs, tab.T, tab.chunk, total)
        return _row_major(m, moved), _row_major(v, moved)

    def _reference_step(self, group, ps, gs, ms, vs, masters=None, inv_scale=None):
        """PyTorch reference (CPU / fallback); identical math to the kernel."""
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            # the host-side step count would be baked into the graph (frozen bias correction)
            raise RuntimeError("FusedAdam: reference path reached during hipGraph capture (grad/param layouts "
                               "or dtypes outside the fused kernel's envelope)")
        if self.found_inf is not None and float(self.found_inf) != 0.0:
            return
        b1, b2 = group["betas"]
        lr = float(group["lr"])
        wd = group["weight_decay"]
        step = self._host_step
        bc1 = 1 - b1**step
        bc2_sqrt = math.sqrt(1 - b2**step)
        inv = float(inv_scale) if inv_scale is not None else 1.0
        for i, (p, g, m, v) in enumerate(zip(ps, gs, ms, vs)):
            w = masters[i] if masters is not None else p
            g = g.float() * inv
            if group["adamw"]:
                w.mul_(1 - lr * wd)
            elif wd != 0:
                g = g.add(w, alpha=wd)
            m.mul_(b1).add_(g, alpha=1 - b1)
            v.mul_(b2).addcmul_(g, g, value=1 - b2)
            denom = (v.sqrt() / bc2_sqrt).add_(group["eps"])
            w.addcdiv_(m, denom, value=-lr / bc1)
            if masters is not None:
                p.copy_(w)

    def state_dict(self):
        sd = super().state_dict()
        sd["hyperion_step"] = self._host_step
        return sd

    def _check_state(self, st, p):
        """Refuses a saved state of the other kind, and 8-bit moments that do not fit: the kernels trust their
        types and sizes."""
        if self.state_bits == 32:
            if "exp_avg_q" in st:
                raise ValueError("FusedAdam(state_bits=32): the saved state has 8-bit moments (state_bits=8)")
            return
        if bool(st.get("channels_last", False)) != _channels_last(p):
            raise ValueError(f"FusedAdam(state_bits=8): the saved moments of a {tuple(p.shape)} parameter are coded in "
                             f"another memory format's order than the parameter's")
        n, nb = p.numel(), -(-p.numel() // STATE_BLOCK)
        want = {"exp_avg_q": (torch.int8, n), "exp_avg_sq_q": (torch.uint8, n),
                "exp_avg_scale": (torch.float32, nb), "exp_avg_sq_scale": (torch.float32, nb)}
        if p.dtype != torch.float32:
            want["master"] = (torch.float32, n)
        for k, (dt, size) in want.items():
            t = st.get(k)
            if not isinstance(t, torch.Tensor) or t.dtype != dt or t.numel() != size:
                raise ValueError(f"FusedAdam(state_bits=8): the saved state of a {tuple(p.shape)} {p.dtype} parameter needs "
                                 f"{k!r} with {size} elements of {dt}, got {None if t is None else (tuple(t.shape), t.dtype)}")

    def load_state_dict(self, state_dict):
        state_dict = dict(state_dict)
        host_step = int(state_dict.pop("hyperion_step", 0))
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        own = [p for g in self.param_groups for p in g["params"]]
        if len(saved) == len(own):  # (else the base class refuses)
            for i, p in zip(saved, own):
                if state_dict["state"].get(i):
                    self._check_state(state_dict["state"][i], p)
        super().load_state_dict(state_dict)
        self._host_step = host_step
        # the base class casts every state tensor to its parameter's dtype: moments and masters of bf16 / fp16
        # parameters are fp32, codes are integers, and the kernels read them as such
        for i, p in zip(saved, own):
            for k, t in state_dict["state"].get(i, {}).items():
                if k in _STATE8:
                    self.state[p][k] = t.detach().to(p.device).reshape(-1).clone()
                    self.state[p]["channels_last"] = _channels_last(p)
                elif k in ("exp_avg", "exp_avg_sq", "master"):
                    # (in the parameter's layout, which the kernels take them to have)
                    self.state[p][k] = torch.empty_like(p, dtype=torch.float32).copy_(t.detach().view(p.shape))
        self._step_t = None
        self._plan8 = self._fits8 = self._values8 = None
        # the table cache is kept: tables a captured graph uses stay pinned; new state tensors
        # simply key new tables


def FusedAdamW(params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
    return FusedAdam(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, adamw=True, state_bits=state_bits)


# clip tables per model: keyed (weakly) by the first parameter, so two same-shaped models never
# share -- and, once captured, never re-point -- each other's pointer table
# (a WeakKeyDictionary cannot hold tensors: its weakref keys compare their referents with the
# elementwise Tensor.__eq__ on a hash-bucket collision)
_clip_tables: "dict[int, tuple]" = {}


def _clip_cache(p0: torch.Tensor) -> TableCache:
    ent = _clip_tables.get(id(p0))
    if ent is None or ent[0]() is not p0:
        key = id(p0)
        ref = weakref.ref(p0, lambda _r, k=key: _clip_tables.pop(k, None))
        ent = (ref, TableCache())
        _clip_tables[key] = ent
    return ent[1]


@torch.no_grad()
def clip_grad_norm_(
    parameters: Iterable[torch.Tensor],
    max_norm: float,
    group: Optional["dist.ProcessGroup"] = None,
    sharded: bool = False,
    defer_to: Optional[FusedAdam] = None,
) -> torch.Tensor:
    """Clip by the global L2 norm.

    ``sharded=True``: each rank holds a disjoint shard of the gradients (FSDP); the squared norm
    is all-reduced over ``group`` before clipping — the reference's ``clip_grad_norm_`` on FSDP
    modules skipped this and clipped by the local shard norm.
    ``defer_to``: a FusedAdam whose next ``step()`` applies the clip coefficient as it reads the
    gradients (one pass over them fewer); the ``.grad`` tensors themselves are left unclipped.
    """
    params = [p for p in parameters if grad_of(p) is not None]
    grads: List[torch.Tensor] = [grad_of(p) for p in params]
    if not grads:
        return torch.zeros(())
    dev = grads[0].device
    native = _native.use_native(grads[0], op="clip") and all(_dense(g) and g.dtype == grads[0].dtype for g in grads)
    if native:
        try:
            tab = _clip_cache(params[0]).get("clip", [grads])
        except ValueError:
            native = False
    if native:
        code = _native.DTYPE_CODE[grads[0].dtype]
        total_sq = _native.native().sumsq_mt(tab.ptrs, tab.sizes, tab.blocks, tab.chunk, code)
    else:
        total_sq = torch.zeros(1, device=dev, dtype=torch.float32)
        for g in grads:
            total_sq += g.float().pow(2).sum()
    if sharded and dist.is_available() and dist.is_initialized():
        from ..train import segments as _seg

        _seg.eager(lambda: dist.all_reduce(total_sq, group=group))  # a hole of a segmented capture
    if defer_to is not None:
        defer_to.clip_coef = (max_norm / (total_sq.reshape(1).sqrt() + 1e-6)).clamp(max=1.0)
    elif native:
        _native.native().clip_mt(tab.ptrs, tab.sizes, tab.blocks, tab.chunk, total_sq, float(max_norm), code)
    else:
        coef = (max_norm / (total_sq.sqrt() + 1e-6)).clamp(max=1.0)
        for g in grads:
            g.mul_(coef.to(g.dtype))
    return total_sq.sqrt().reshape(())
