"""The operators of a memory-lean fine-tuning step, as cases that can be measured.

* ``logprobs``: log probabilities of given tokens with entropy and the top alternatives, and their
  gradient into the logits (``hyperion.ops.token_logprobs``);
* ``adamw8``: an AdamW step over many tensors whose moments are held in 8 bits
  (``hyperion.ops.FusedAdamW(state_bits=8)``);
* ``quantize`` / ``linear``: microscaled 4-bit floating point, quantisation and the products of a
  linear layer with a frozen 4-bit weight (``hyperion.ops.mxfp4``).

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own`` true
it makes the framework's calls.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
IGNORE = -100

LR, B1, B2, EPS, WD = 1e-3, 0.9, 0.999, 1e-8, 0.01
BLOCK = 256  # elements of a block of 8-bit moments
MX = 32  # elements of a block of 4-bit floating point


def listed():
    return [
        # one decoded token of the GPT-2-small LM: its log probability and twenty alternatives (latency)
        {"name": "score_token_top20", "op": "logprobs", "batch": 1, "seq": 1, "vocab": 50257, "dtype": "bf16",
         "top_k": 20, "train": False, "masked": 0.0, "temperature": 1.0},
        # a batch of served answers scored in fp32 with five alternatives, part of the vocabulary masked out
        {"name": "score_batch_masked", "op": "logprobs", "batch": 8, "seq": 33, "vocab": 32000, "dtype": "f32",
         "top_k": 5, "train": False, "masked": 0.4, "temperature": 0.7},
        # perplexity evaluation of the GPT-2-small LM at its training batch (forward only)
        {"name": "score_eval", "op": "logprobs", "batch": 16, "seq": 127, "vocab": 50257, "dtype": "bf16",
         "top_k": 0, "train": False, "masked": 0.0, "temperature": 1.0},
        # a policy objective over the LM-256 training batch: log probabilities, entropies and the logits' gradient
        {"name": "score_train", "op": "logprobs", "batch": 32, "seq": 127, "vocab": 50257, "dtype": "bf16",
         "top_k": 0, "train": True, "masked": 0.0, "temperature": 1.0},
        # the rank-16 adapters of four projections in 32 Llama layers: many small bf16 tensors with fp32 masters
        {"name": "adam_adapters", "op": "adamw8", "tensors": 256, "rows": 16, "cols": 4096, "extra": 0, "dtype": "bf16"},
        # a small fp32 language model: matrices and odd vectors
        {"name": "adam_small_lm", "op": "adamw8", "tensors": 26, "rows": 256, "cols": 1024, "extra": 771, "dtype": "f32"},
        # the projections of one Llama layer, trained in full
        {"name": "adam_layer", "op": "adamw8", "tensors": 4, "rows": 11008, "cols": 4096, "extra": 4096, "dtype": "bf16"},
        # a small odd fp32 matrix (tail blocks in every row)
        {"name": "quantize_odd", "op": "quantize", "rows": 1023, "cols": 500, "dtype": "f32"},
        # a Llama MLP weight, as an adapter's base is frozen
        {"name": "quantize_weight", "op": "quantize", "rows": 11008, "cols": 4096, "dtype": "bf16"},
        # one decoded token through an MLP projection (the weight's stream)
        {"name": "linear_token", "op": "linear", "m": 1, "n": 11008, "k": 4096, "dtype": "bf16", "train": False},
        # the LoRA step's 128 tokens through a projection, forward and data gradient
        {"name": "linear_lora_step", "op": "linear", "m": 128, "n": 4096, "k": 4096, "dtype": "bf16", "train": True},
        # a long prompt batch through an MLP projection, forward and data gradient
        {"name": "linear_long", "op": "linear", "m": 4064, "n": 11008, "k": 4096, "dtype": "bf16", "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "adamw8", "adamw8", "quantize", "linear", "linear", "linear"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 130000)
        rows = _log(rng, 1, max(1, min(4064, 4064 * 50257 // vocab)))
        batch = rng.choice([b for b in (1, 2, 3, 4, 8, 16) if b <= rows])
        train = rng.random() < 0.5
        top = 0 if train or rows > 512 else rng.choice([0, 1, 5, 20, 32])
        return {"op": op, "batch": batch, "seq": rows // batch, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])
                if rows * vocab < 100_000_000 else "bf16", "top_k": top, "train": train,
                "masked": rng.choice([0.0, 0.0, 0.3, 0.9]), "temperature": rng.choice([1.0, 1.0, 0.6, 1.5])}
    if op == "adamw8":
        total = _log(rng, 4096, 150_000_000)
        tensors = _log(rng, 1, min(256, max(1, total // 2048)))
        cols = rng.choice([c for c in (64, 100, 257, 768, 1024, 4096) if c * tensors <= total])
        return {"op": op, "tensors": tensors, "rows": max(1, total // (tensors * cols)), "cols": cols,
                "extra": rng.choice([0, 1, 255, 256, 1000]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "quantize":
        return {"op": op, "rows": _log(rng, 1, 11008), "cols": _log(rng, 16, 4096), "dtype": rng.choice(["bf16", "f16", "f32"])}
    m = _log(rng, 1, 4064)
    return {"op": op, "m": m, "n": rng.choice([64, 200, 256, 768, 1000, 2048, 4096, 8192, 11008]),
            "k": rng.choice([32, 100, 256, 768, 1024, 2048, 4096]),
            "dtype": rng.choice(["bf16", "bf16", "bf16", "f16", "f32"]) if m < 1500 else "bf16", "train": rng.random() < 0.5}


# ---- 8-bit moments, 4-bit weights: the codes and the values they stand for -------------------------
def _scale(top):
    """A block's scale as it is kept, in fp32: 0 below the smallest normal number, NaN where it is not finite."""
    s = top.float()
    s = torch.where(s < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    return torch.where(torch.isfinite(s), s, torch.full_like(s, math.nan))


def _ratio(x, s):
    """x / s in 64 bits (a code next to a border needs them), 0 in a block of zeros."""
    return torch.where(s > 0, x / s.double(), torch.zeros_like(x))


def _encode_m(m):
    """[blocks, 256] in 64 bits -> (int8 codes, scales)"""
    s = _scale(m.abs().amax(dim=1, keepdim=True))
    q = torch.round(torch.sqrt(_ratio(m.abs(), s)) * 127.0).clamp(0.0, 127.0)
    return torch.where(m < 0, -q, q).to(torch.int8), s


def _decode_m(q, s):
    q = q.double()
    return (q * q.abs()) * (s.double() / 16129.0)


def _encode_v(v):
    """[blocks, 256] in 64 bits -> (uint8 codes, scales)"""
    s = _scale(v.amax(dim=1, keepdim=True))
    q = torch.round(torch.sqrt(torch.sqrt(_ratio(v, s))) * 255.0).clamp(0.0, 255.0)
    q = torch.where((v > 0) & (s > 0) & (q < 1), torch.ones_like(q), q)
    return q.to(torch.uint8), s


def _decode_v(q, s):
    q = q.double() * q.double()
    return (q * q) * (s.double() / 4228250625.0)


def _blocks(tensors):
    """Every tensor in memory order, padded to whole blocks: [blocks, 256] in 64 bits."""
    return torch.cat([torch.nn.functional.pad(t.reshape(-1).double(), (0, -t.numel() % BLOCK)) for t in tensors]).view(-1, BLOCK)


def _tensors(blocks, like):
    """The inverse of _blocks: flat fp32 tensors with the sizes of `like`."""
    parts = blocks.float().reshape(-1).split([t.numel() + -t.numel() % BLOCK for t in like])
    return [p[:t.numel()] for p, t in zip(parts, like)]


def _mx_encode(x):
    """[rows, cols] -> (two codes a byte [rows, 16 blocks], exponents [rows, blocks]), cols padded to whole blocks"""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -cols % MX)).view(rows, -1, MX)
    amax = x.abs().amax(dim=2, keepdim=True)
    e = (torch.frexp(amax)[1] - 1 - 2).clamp(-127, 127)  # floor(log2(amax)) - 2
    e = torch.where(amax == 0, torch.full_like(e, -127), e)
    a = torch.ldexp(x.abs().double(), -e.double())
    # steps of the magnitudes 0, .5, 1, 1.5 | 2, 3 | 4, 6: 0.5 below 2, 1 below 4, 2 above; ties to the even code
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(0.0, 6.0)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(x).to(torch.uint8) << 3)
    scale = (e + 127).to(torch.uint8).squeeze(2)
    bad = ~torch.isfinite(amax).squeeze(2)
    scale = torch.where(bad, torch.full_like(scale, 255), scale)
    code = code.view(rows, -1, 2)
    return (code[..., 0] | (code[..., 1] << 4)), scale


def _mx_decode(codes, scales, cols):
    rows = codes.shape[0]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    q = torch.stack([codes & 15, codes >> 4], dim=-1).view(rows, -1, MX)
    s = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales.double() - 127).float()
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return (table[q.long()] * s[..., None]).view(rows, -1)[:, :cols]


# ---- inputs ----------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    dt = DTYPES.get(case["dtype"])
    st = {"case": case}
    if case["op"] == "logprobs":
        B, S, V = case["batch"], case["seq"], case["vocab"]
        z = randn(B, S, V).mul_(2.5)
        if case["masked"]:
            z = z.masked_fill_(torch.rand(V, generator=g, device=DEV) < case["masked"], -math.inf)
            z[..., 0] = 0.0
        st["logits"] = z.to(dt).requires_grad_(case["train"])
        t = torch.randint(V, (B, S), generator=g, device=DEV)
        if B * S > 8:  # a padded batch
            t = torch.where(torch.rand(B, S, generator=g, device=DEV) < 0.06, torch.full_like(t, IGNORE), t)
        if case["masked"]:  # given tokens are allowed ones
            t = torch.where((t >= 0) & (st["logits"].detach().gather(2, t.clamp(min=0)[..., None])[..., 0] == -math.inf), torch.zeros_like(t), t)
        st["target"] = t
        if case["train"]:
            st["w"], st["wh"] = randn(B, S) / (B * S), torch.full((B, S), -0.01 / (B * S), device=DEV)
        return st
    if case["op"] == "adamw8":
        shapes = [(case["rows"], case["cols"])] * case["tensors"] + [(case["extra"],)] * (case["tensors"] if case["extra"] else 0)
        # the parameters and the gradients are views of one buffer each, as a data-parallel program lays them out
        starts = [0]
        for s in shapes:
            starts.append(starts[-1] + -(-math.prod(s) // 64) * 64)
        st["flat"], grads = (randn(starts[-1]) * 0.02).to(dt), (randn(starts[-1]) * 1e-3).to(dt)
        st["params"] = [torch.nn.Parameter(st["flat"][a:a + math.prod(s)].view(s)) for a, s in zip(starts, shapes)]
        for p, a in zip(st["params"], starts):
            p.grad = grads[a:a + p.numel()].view(p.shape)
        st["master"] = [p.detach().float() for p in st["params"]]  # of fp32 parameters: themselves
        m = [randn(*s) * 3e-4 for s in shapes]
        v = [(randn(*s) * 1e-3).square_() for s in shapes]
        st["mq"], st["ms"] = _encode_m(_blocks(m))
        st["vq"], st["vs"] = _encode_v(_blocks(v))
        st["step"] = 100
        if own:
            st["opt"] = _optimizer(st)
        return st
    if case["op"] == "quantize":
        st["x"] = (randn(case["rows"], case["cols"]) * 0.02).to(dt)
        return st
    w = randn(case["n"], case["k"]) * 0.02
    st["codes"], st["scales"] = _mx_encode(w)
    st["x"] = randn(case["m"], case["k"]).to(dt).requires_grad_(case["train"])
    if case["train"]:
        st["dy"] = randn(case["m"], case["n"]).to(dt)
    if own:
        from hyperion.ops.mxfp4 import MXFP4Tensor

        st["weight"] = MXFP4Tensor(st["codes"], st["scales"], (case["n"], case["k"]))
    return st


def _optimizer(st):
    """The optimizer of a resumed run: 100 steps done, its 8-bit moments and fp32 masters in place."""
    from hyperion.ops import FusedAdamW

    opt = FusedAdamW(st["params"], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=8)
    sizes = [-(-p.numel() // BLOCK) for p in st["params"]]
    state = {}
    for i, (p, mq, ms, vq, vs) in enumerate(zip(st["params"], st["mq"].split(sizes), st["ms"].split(sizes),
                                                st["vq"].split(sizes), st["vs"].split(sizes))):
        n = p.numel()
        state[i] = {"exp_avg_q": mq.reshape(-1)[:n].clone(), "exp_avg_scale": ms.reshape(-1).clone(),
                    "exp_avg_sq_q": vq.reshape(-1)[:n].clone(), "exp_avg_sq_scale": vs.reshape(-1).clone()}
        if p.dtype != torch.float32:
            state[i]["master"] = st["master"][i].clone()
    sd = opt.state_dict()
    opt.load_state_dict({"state": state, "param_groups": sd["param_groups"], "hyperion_step": st["step"]})
    return opt


# ---- one pass --------------------------------------------------------------------------------------
def run(state):
    return {"logprobs": _run_logprobs, "adamw8": _run_adamw8, "quantize": _run_quantize, "linear": _run_linear}[state["case"]["op"]](state)


def _run_logprobs(state):
    c, z, t = state["case"], state["logits"], state["target"]
    if own:
        from hyperion.ops.token_logprobs import token_logprobs

        o = token_logprobs(z, t, top_k=c["top_k"], ignore_index=IGNORE, temperature=c["temperature"])
        out = {"logprobs": o.logprobs.detach(), "entropy": o.entropy.detach()}
        if c["top_k"]:
            out["top_logprobs"], out["top_ids"] = o.top_logprobs, o.top_ids
        if c["train"]:
            out["dlogits"], = torch.autograd.grad([o.logprobs, o.entropy], [z], [state["w"], state["wh"]])
        return out
    zd = z.detach()
    y = zd.float() * (1.0 / c["temperature"])
    valid = t != IGNORE
    m = y.amax(dim=-1, keepdim=True)
    d = y - m
    e = torch.exp(d)
    s = e.sum(dim=-1, keepdim=True)
    u = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(dim=-1, keepdim=True)
    logs = torch.log(s)
    h = logs - u / s
    tc = t.clamp(min=0)[..., None]
    lp = d.gather(-1, tc) - logs
    zero = torch.zeros((), device=y.device)
    out = {"logprobs": torch.where(valid, lp[..., 0], zero), "entropy": torch.where(valid, h[..., 0], zero)}
    if c["top_k"]:
        ids = torch.sort(zd, dim=-1, descending=True, stable=True)[1][..., :c["top_k"]]
        out["top_logprobs"] = torch.where(valid[..., None], d.gather(-1, ids) - logs, zero)
        out["top_ids"] = torch.where(valid[..., None], ids, torch.full_like(ids, -1))
    if c["train"]:
        w = torch.where(valid, state["w"], zero)[..., None]
        wh = torch.where(valid, state["wh"], zero)[..., None]
        p = e / s
        dz = torch.where(p > 0, -p * (w + wh * (d - logs + h)), zero)
        dz = dz.scatter_add(-1, tc, w)
        out["dlogits"] = (dz * (1.0 / c["temperature"])).to(z.dtype)
    return out


def _run_adamw8(state):
    params = state["params"]
    if own:
        state["opt"].step()
        m, v = state["opt"].moment_vectors()
        return {"params": state["flat"], "exp_avg": m, "exp_avg_sq": v}
    state["step"] += 1
    bc1, bc2 = 1 - B1 ** state["step"], math.sqrt(1 - B2 ** state["step"])
    g = _blocks([p.grad for p in params])
    w = _blocks(state["master"])
    m = _decode_m(state["mq"], state["ms"]) * B1 + g * (1 - B1)
    v = _decode_v(state["vq"], state["vs"]) * B2 + g * g * (1 - B2)
    w = w * (1 - LR * WD) - (m / (torch.sqrt(v) / bc2 + EPS)) * (LR / bc1)
    state["mq"], state["ms"] = _encode_m(m)
    state["vq"], state["vs"] = _encode_v(v)
    w = _tensors(w, params)
    torch._foreach_copy_([t.view(-1) for t in state["master"]], w)
    torch._foreach_copy_([p.detach().view(-1) for p in params], w)
    return {"params": state["flat"],
            "exp_avg": torch.cat(_tensors(_decode_m(state["mq"], state["ms"]), params)),
            "exp_avg_sq": torch.cat(_tensors(_decode_v(state["vq"], state["vs"]), params))}


def _run_quantize(state):
    x = state["x"]
    if own:
        from hyperion.ops.mxfp4 import quantize_mxfp4

        return quantize_mxfp4(x).dequantize(torch.float32)
    return _mx_decode(*_mx_encode(x), x.shape[1])


def _run_linear(state):
    c, x = state["case"], state["x"]
    if own:
        from hyperion.ops.mxfp4 import mxfp4_linear

        y = mxfp4_linear(x, state["weight"])
        return (y.detach(), torch.autograd.grad(y, x, state["dy"])[0]) if c["train"] else y
    w = _mx_decode(state["codes"], state["scales"], c["k"])
    y = (x.detach().float() @ w.t()).to(x.dtype)
    return (y, (state["dy"].float() @ w).to(x.dtype)) if c["train"] else y


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "logprobs":
        rows, n = case["batch"] * case["seq"], case["batch"] * case["seq"] * case["vocab"]
        out = rows * (16 + 12 * case["top_k"])
        return {"bytes": n * b * (2 if case["train"] else 1) + out + (8 * rows if case["train"] else 0),
                "flops": n * (14 if case["train"] else 6)}
    if case["op"] == "adamw8":
        n = case["tensors"] * (case["rows"] * case["cols"] + case["extra"])
        # gradient, master (and its low-precision copy), the codes in and out, the moments' values out
        per = b + 8 + (b if case["dtype"] != "f32" else 0) + 4 + 16 / BLOCK + 8
        return {"bytes": int(n * per), "flops": 40 * n}
    if case["op"] == "quantize":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (b + 4) + n * 17 // 32, "flops": 6 * n}
    m, n, k = case["m"], case["n"], case["k"]
    x = (m * k + m * n) * b
    return {"bytes": n * k * 17 // 32 + x * (2 if case["train"] else 1), "flops": 2 * m * n * k * (2 if case["train"] else 1)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        z, t = st["logits"].detach(), st["target"]
        ls = torch.log_softmax(z.double() / case["temperature"], dim=-1)
        keep = t != IGNORE
        lp = torch.where(keep, ls.gather(-1, t.clamp(min=0).unsqueeze(-1)).squeeze(-1), 0.0)
        p = ls.exp()
        h = -torch.nan_to_num(p * ls, nan=0.0).sum(-1)
        out = {"logprobs": lp, "entropy": torch.where(keep, h, 0.0)}
        if case["top_k"]:
            # the order of (value, lowest id): ids by a stable sort of the negated values
            ids = torch.argsort(-z.double(), dim=-1, stable=True)[..., :case["top_k"]]
            out["top_logprobs"] = torch.where(keep.unsqueeze(-1), ls.gather(-1, ids), 0.0)
            out["top_ids"] = torch.where(keep.unsqueeze(-1), ids, -1)
        if case["train"]:
            a, b = (torch.where(keep, st[k].double(), 0.0).unsqueeze(-1) for k in ("w", "wh"))
            hot = torch.zeros_like(p).scatter_(-1, t.clamp(min=0).unsqueeze(-1), 1.0)
            out["dlogits"] = (a * (hot - p) - b * p * (torch.nan_to_num(ls, neginf=0.0) + h.unsqueeze(-1))) / case["temperature"]
        return out
    if case["op"] == "adamw8":
        at, flat, n_steps = 0, st["flat"].double(), st["step"] + 1
        out = {"params": flat, "exp_avg": [], "exp_avg_sq": []}
        for p, w in zip(st["params"], st["master"]):
            n, nb, start = p.numel(), -(-p.numel() // BLOCK), p.storage_offset()
            mq, ms, vq, vs = (st[k][at:at + nb].double() for k in ("mq", "ms", "vq", "vs"))
            at += nb
            m = (mq.sign() * (mq / 127) ** 2 * ms).reshape(-1)[:n]
            v = ((vq / 255) ** 4 * vs).reshape(-1)[:n]
            grad = p.grad.double().reshape(-1)
            m = B1 * m + (1 - B1) * grad
            v = B2 * v + (1 - B2) * grad ** 2
            flat[start:start + n] = w.double().reshape(-1) * (1 - LR * WD) - LR * (m / (1 - B1 ** n_steps)) / ((v / (1 - B2 ** n_steps)).sqrt() + EPS)
            for x, levels, power, key in ((m, 127, 2, "exp_avg"), (v, 255, 4, "exp_avg_sq")):
                x = torch.cat([x, x.new_zeros(nb * BLOCK - n)]).view(nb, BLOCK)
                top = x.abs().amax(1, keepdim=True).float().double()  # the scale is a number of fp32
                code = torch.round(levels * (x.abs() / top) ** (1 / power)).clamp(max=levels)
                if power == 4:
                    code = torch.where(x > 0, code.clamp(min=1), code)
                out[key].append((x.sign() * (code / levels) ** power * top).reshape(-1)[:n])
        return {k: torch.cat(v) if k != "params" else v for k, v in out.items()}
    if case["op"] == "quantize":
        x = st["x"].double()
        rows, cols = x.shape
        x = torch.cat([x, x.new_zeros(rows, -cols % MX)], dim=1).view(rows, -1, MX)
        unit = 2.0 ** (torch.floor(torch.log2(x.abs().amax(2, keepdim=True).clamp(min=2.0 ** -125))) - 2)
        # the nearest of the eight magnitudes; a tie goes to the even one of its two neighbours
        grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
        mid = (grid[1:] + grid[:-1]) / 2
        a = x.abs() / unit
        up, down = torch.bucketize(a, mid, right=True), torch.bucketize(a, mid)  # they differ on a tie alone
        pick = torch.where(up % 2 == 0, up, down)
        return (x.sign() * grid[pick] * unit).reshape(rows, -1)[:, :cols]
    grid = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    grid = torch.tensor(grid + [-v for v in grid], dtype=torch.float64, device=DEV)
    codes = st["codes"].long()
    w = torch.stack((grid[codes % 16], grid[codes // 16]), dim=2).flatten(1)
    w = (w * torch.exp2(st["scales"].double() - 127).repeat_interleave(MX, dim=1))[:, :case["k"]]
    y = st["x"].detach().double() @ w.t()
    return (y, st["dy"].double() @ w) if case["train"] else y
