"""token_logprobs in 64 bits on the CPU, row by row from its definition, with bounds on fp32's error."""
import math

import torch

EPS = 2.0 ** -24  # half a step of fp32


def oracle(logits, target, top_k=0, ignore_index=-100, temperature=1.0, dlogp=None, dent=None):
    """(logprobs, entropy, top_logprobs, top_ids, dlogits) over [rows, V], all in fp64 / int64."""
    z = logits.detach().cpu().double()
    t = target.cpu().long()
    R, V = z.shape
    lp, h = torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.float64)
    top, ids = torch.zeros(R, top_k, dtype=torch.float64), torch.full((R, top_k), -1)
    g = torch.zeros(R, V, dtype=torch.float64)
    for r in range(R):
        if t[r] == ignore_index:
            continue
        y = z[r] / temperature
        a = 0.0 if dlogp is None else float(dlogp[r])
        b = 0.0 if dent is None else float(dent[r])
        # falling order, NaN first, equal ones by the lower id
        ids[r] = torch.tensor(sorted(range(V), key=lambda j: (not math.isnan(z[r, j]), -z[r, j].nan_to_num(nan=0.0), j))[:top_k]
                              if torch.isnan(z[r]).any() else torch.sort(z[r], descending=True, stable=True)[1][:top_k].tolist())
        inside = 0 <= t[r] < V
        if (y == -math.inf).all():
            lp[r], top[r] = (-math.inf if inside else math.nan), -math.inf
            continue
        ls = y - y.max()  # the difference first: a row of the type's lowest value
        ls = ls - torch.logsumexp(ls, 0)
        if not torch.isfinite(y).logical_or(y == -math.inf).all():
            ls = torch.full_like(y, math.nan)
        p = ls.exp()
        h[r] = -torch.where(p == 0, torch.zeros_like(p), p * ls).sum()
        lp[r] = ls[t[r]] if inside else math.nan
        top[r] = ls[ids[r]]
        if not inside:
            a = math.nan
        g[r] = torch.where(p == 0, torch.zeros_like(p), -p * (a + b * (ls + h[r])))
        if inside:
            g[r, t[r]] += a
    return lp, h, top, ids, g / temperature


def bounds(logits, temperature, dlogp, dent, want):
    """How far fp32 may be: each exponent is rounded once (relative EPS, and c = log2(e) / T once), each of
    V / 256 + 64 additions of a sum once."""
    lp, h, top, ids, g = want
    V = logits.shape[1]
    n = V / 256 + 64
    fin = lambda x: torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x))  # noqa: E731
    y = logits.detach().cpu().double() / temperature
    y = torch.where(torch.isfinite(y), y, torch.zeros_like(y))
    y = y - y.amax(1, keepdim=True)
    y = y.clamp(min=-110.0)  # p is 0 in fp32 below
    span = (y.amax(1) - y.amin(1)) + math.log(V) + 1  # the largest |log p| of a row
    b_lp = EPS * (n + 8 * (fin(lp) + math.log(V) + 1))
    b_top = EPS * (n + 8 * (fin(top) + math.log(V) + 1))
    b_h = EPS * (n + 16) * (2 + 2 * math.log(V) + h.abs().nan_to_num())
    half = torch.finfo(logits.dtype).eps / 2
    a = torch.zeros_like(lp) if dlogp is None else dlogp.cpu().double().abs()
    b = torch.zeros_like(lp) if dent is None else dent.cpu().double().abs()
    weight = (a + b * (span + h.abs().nan_to_num()))[:, None] / temperature
    p_bound = EPS * (n + 8 * span[:, None])  # relative, of p
    p = torch.softmax(y, 1)
    b_g = (half * fin(g) * (1 + 1e-6) + weight * (p * p_bound + 4 * EPS * p) + 2 * EPS * a[:, None] / temperature * (g != 0)
           + {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -120}[logits.dtype])
    return b_lp, b_h, b_top, b_g


def check(got, want, bound):
    got, want = got.cpu().double(), want.double()
    assert got.shape == want.shape
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)])
    d = torch.where(odd, torch.zeros_like(want), (got - want).abs())
    assert bool((d <= bound).all()), f"off by {float((d - bound).max())} more than the bound"
