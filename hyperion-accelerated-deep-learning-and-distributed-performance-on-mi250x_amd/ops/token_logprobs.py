"""Log probabilities of given tokens, with each row's entropy and its most likely tokens.

The LM trainers' losses (:mod:`.cross_entropy`) are means over tokens; scoring needs the tokens
themselves: perplexities by position, preference and policy objectives, and the alternatives a
served token had.  ``token_logprobs`` returns them from one read of the logits
(``csrc/kernels/token_logprobs.hip``) and its backward takes the gradients of the log probabilities
and of the entropies to the logits in one more read and one write; no fp32 softmax is stored.

With ``y = logits / temperature``, ``p = softmax(y)``: ``logprobs = log p[target]``, ``entropy =
-sum p log p``, and the ``top_k`` largest logits of each row in falling order (equal ones by the
lower id) with their log probabilities.  Sums are fp32 whatever the logits' type.

* A row whose target is ``ignore_index`` gives 0 everywhere, ids -1 and a zero gradient.
* -inf logits (a masked vocabulary) have probability 0 and no gradient.  A row with nothing else has
  log probabilities -inf, entropy 0 and a zero gradient.
* A NaN or +inf logit makes its row's results and its whole gradient NaN.  A target outside the vocabulary
  makes its row's log probability and whole gradient NaN (masked logits among them, as does a NaN that comes
  back as the gradient of either result); the entropy and the alternatives do not depend on it.
"""
from __future__ import annotations

import math
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native

TOP_MAX = 32  # hyp::kTokenTopMax
TOP_VOCAB = 1 << 18  # hyp::kTokenTopVocab
FLOOR = -200 * math.log(2.0)  # hyp::kFloor as a natural logarithm: exp of it is 0 in fp32


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # fp32, the target's shape
    entropy: torch.Tensor  # fp32, the target's shape (nats)
    top_logprobs: Optional[torch.Tensor]  # fp32 [..., top_k]; None without top_k
    top_ids: Optional[torch.Tensor]  # int64 [..., top_k]; None without top_k


def _reference_fwd(z, target, k, ignore_index, inv_t):
    """PyTorch oracle of the forward kernel over [rows, V]: (logprobs, entropy, stats, top logprobs, top ids)."""
    V = z.shape[1]
    keep = target != ignore_index
    m = z.amax(1).float()
    empty = m == -math.inf  # (a NaN makes m NaN)
    # the difference first, as in the kernel: divided by the temperature, the type's lowest value would be -inf
    d = (z.float() - torch.where(empty, torch.zeros_like(m), m)[:, None]) * inv_t
    e = torch.exp(d)
    s = e.sum(1)
    logs = torch.where(empty, torch.full_like(s, math.inf), torch.log(s))
    u = torch.where(e == 0, torch.zeros_like(e), e * d).sum(1)
    h = torch.where(empty, torch.zeros_like(s), (logs - u / s)).clamp(min=0.0)
    inside = (target >= 0) & (target < V)
    lp = d.gather(1, torch.where(inside, target, torch.zeros_like(target))[:, None])[:, 0] - logs
    lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
    zero = torch.zeros_like(lp)
    ids = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :k]
    top = d.gather(1, ids) - logs[:, None]
    stats = torch.stack([torch.where(empty, torch.zeros_like(m), m), logs, h], dim=1)
    return (torch.where(keep, lp, zero), torch.where(keep, h, zero), stats,
            torch.where(keep[:, None], top, torch.zeros_like(top)), torch.where(keep[:, None], ids, torch.full_like(ids, -1)))


def _reference_bwd(z, target, stats, ignore_index, inv_t, dlogp, dent):
    V = z.shape[1]
    m, logs, h = stats[:, 0:1], stats[:, 1:2], stats[:, 2:3]
    live = (target != ignore_index)[:, None] & (logs != math.inf)
    inside = ((target >= 0) & (target < V))[:, None]
    zero = torch.zeros_like(h)
    wl = torch.where(live, zero if dlogp is None else dlogp[:, None], zero)
    wl = torch.where(live & ~inside, torch.full_like(wl, math.nan), wl)
    wh = torch.where(live, zero if dent is None else dent[:, None], zero)
    q = (z.float() - m) * inv_t - logs
    p = torch.exp(q)
    dz = -p * (wl + wh * (q.clamp(min=FLOOR) + h))  # (finite in a masked place: 0 unless the row's gradient is NaN)
    dz = dz.scatter_add(1, torch.where(inside[:, 0], target, torch.zeros_like(target))[:, None], wl)
    dz = torch.where((target != ignore_index)[:, None], dz * inv_t, torch.zeros_like(dz))
    return dz.to(z.dtype)


class _TokenLogprobsFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, target, k, ignore_index, inv_t, needs_grad):
        native = _native.use_native(logits, op="token_logprobs")
        if native:
            _native.count("token_logprobs")
            lp, h, stats, tl, ti = _native.native().token_logprobs_fwd(logits, target, k, ignore_index, inv_t,
                                                                             needs_grad)
        else:
            rows = logits.reshape(-1, logits.shape[-1])
            lp, h, stats, tl, ti = _reference_fwd(rows, target.reshape(-1), k, ignore_index, inv_t)
            lead = logits.shape[:-1]
            lp, h = lp.view(lead), h.view(lead)
            tl, ti = (tl.view(*lead, k), ti.view(*lead, k)) if k else (None, None)
        ctx.save_for_backward(logits, target, stats)
        ctx.cfg = (ignore_index, inv_t, native)
        if k:
            ctx.mark_non_differentiable(tl, ti)
        ctx.set_materialize_grads(False)
        return lp, h, tl, ti

    @staticmethod
    @once_differentiable
    def backward(ctx, dlogp, dent, _dtop, _dids):
        logits, target, stats = ctx.saved_tensors
        ignore_index, inv_t, native = ctx.cfg
        if dlogp is None and dent is None:
            return None, None, None, None, None, None
        dlogp = None if dlogp is None else dlogp.float().contiguous().view(-1)
        dent = None if dent is None else dent.float().contiguous().view(-1)
        if native:
            dz = _native.native().token_logprobs_bwd(logits, target, stats, ignore_index, inv_t, dlogp, dent)
        else:
            dz = _reference_bwd(logits.reshape(-1, logits.shape[-1]), target.reshape(-1), stats, ignore_index, inv_t,
                                dlogp, dent).view(logits.shape)
        return dz, None, None, None, None, None


def token_logprobs(logits: torch.Tensor, target: torch.Tensor, top_k: int = 0, ignore_index: int = -100,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Scores ``target`` [...] under ``logits`` [..., V] (bf16, fp16 or fp32).

    ``logprobs`` and ``entropy`` are differentiable in the logits (once); the ``top_k`` (at most 32, of at
    most 2^18 tokens) alternatives are not.  Logits whose rows have unit stride are read where they are, whatever the
    strides of their (at most two) leading dimensions: ``logits[:, :-1]`` is not copied."""
    if logits.dtype not in _native.DTYPE_CODE:
        raise TypeError(f"token_logprobs: logits must be fp32, bf16 or fp16, got {logits.dtype}")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"token_logprobs: logits must be [..., V] with V >= 1, got {tuple(logits.shape)}")
    if target.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"token_logprobs: target must hold int64 or int32 ids, got {target.dtype}")
    if target.shape != logits.shape[:-1]:
        raise ValueError(f"token_logprobs: target {tuple(target.shape)} does not match logits {tuple(logits.shape)}")
    if target.device != logits.device:
        raise ValueError(f"token_logprobs: target is on {target.device}, the logits are on {logits.device}")
    V = logits.shape[-1]
    if not 0 <= top_k <= min(TOP_MAX, V):
        raise ValueError(f"token_logprobs: top_k must be in [0, {min(TOP_MAX, V)}], got {top_k}")
    if top_k and V > TOP_VOCAB:
        raise ValueError(f"token_logprobs: alternatives are for at most {TOP_VOCAB} tokens, got {V}")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"token_logprobs: temperature must be in [1e-6, 1e6], got {temperature}")
    if logits.dim() > 3 or (logits.stride(-1) != 1 and V > 1):
        logits = logits.contiguous()
        if logits.dim() > 3:
            out = token_logprobs(logits.view(-1, V), target.reshape(-1), top_k, ignore_index, temperature)
            return TokenLogprobs(*(None if t is None else t.view(*target.shape, *t.shape[1:]) for t in out))
    needs_grad = logits.requires_grad and torch.is_grad_enabled()
    return TokenLogprobs(*_native.apply_fn(_TokenLogprobsFn, logits, target.long().contiguous(), int(top_k),
                                           int(ignore_index), 1.0 / float(temperature), needs_grad, needs_grad=needs_grad))
