"""token_logprobs kernels against the 64-bit oracle: types, odd sizes, strides, masks, ties, graphs, streams."""
import math

import pytest
import torch

from hyperion.ops import _native
from hyperion.ops.token_logprobs import token_logprobs

from token_logprobs_oracle import bounds, check, oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows(R, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(R, V, generator=g) * 2.5).to(dtype)
    return z, torch.randint(V, (R,), generator=g), torch.randn(R, generator=g), torch.randn(R, generator=g)


def compare(z, t, dlogp, dent, k, temperature=1.0, ref=None):
    """`ref`: the oracle's rows where z is a view of another shape."""
    ref = z if ref is None else ref
    zd = z.detach().requires_grad_(True)
    n = _native.counters().get("token_logprobs", 0)
    out = token_logprobs(zd, t.to(DEV).view(z.shape[:-1]), top_k=k, temperature=temperature)
    assert _native.counters()["token_logprobs"] == n + 1
    g, = torch.autograd.grad([out.logprobs, out.entropy], [zd], [dlogp.to(DEV).view(z.shape[:-1]), dent.to(DEV).view(z.shape[:-1])])
    V = z.shape[-1]
    want = oracle(ref, t, k, -100, temperature, dlogp, dent)
    b = bounds(ref, temperature, dlogp, dent, want)
    check(out.logprobs.view(-1), want[0], b[0])
    check(out.entropy.view(-1), want[1], b[1])
    if k:
        assert torch.equal(out.top_ids.view(-1, k).cpu(), want[3])
        check(out.top_logprobs.view(-1, k), want[2], b[2])
    check(g.view(-1, V), want[4], b[3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (2, 7, 0), (5, 33, 32), (3, 509, 5), (4, 1000, 32), (2, 2049, 20),
                                   (3, 8193, 1), (2, 50257, 20), (1, 130001, 32), (530, 1003, 3), (520, 4, 0)])
def test_against_oracle(R, V, k, dtype):
    z, t, a, b = rows(R, V, dtype, R + V)
    if R > 2:
        t[1] = -100
    compare(z.to(DEV), t, a, b, k, temperature=1.0 if V % 2 else 0.7)


@pytest.mark.parametrize("V", [65, 9001])
def test_masked_empty_and_poisoned_rows(V):
    z, t, a, b = rows(9, V, torch.bfloat16)
    z[0] = -math.inf
    z[1, 3:] = -math.inf  # fewer tokens left than alternatives asked for
    t[1] = 40
    z[2, 7] = math.nan
    z[3, 9] = math.inf
    t[4] = V
    t[5] = -7
    z[6] = -math.inf
    z[6, 11] = 2.0
    t[6] = 11
    z[7] = torch.finfo(torch.bfloat16).min  # a mask of the type's lowest value everywhere
    z[8, ::2] = torch.finfo(torch.bfloat16).min
    compare(z.to(DEV), t, a, b, 8)


@pytest.mark.parametrize("R", [2, 515])
def test_ties_go_to_the_lowest_id(R):
    V = 9000
    z = torch.zeros(R, V, dtype=torch.bfloat16)
    z[0, 1::2] = -0.0
    z[1] = torch.arange(V) // 3 % 7
    t, a = torch.zeros(R, dtype=torch.long), torch.ones(R)
    compare(z.to(DEV), t, a, a, 32)


def test_more_candidates_than_fit():
    # most threads' largest logit is small and a few hold thousands of large ones: the bound passes them all
    V = 130000
    z = -torch.arange(V)[None] * 1e-6
    lot = torch.arange(V) // 8 % 1024 % 64 < 2
    z[0, lot] = 1 + torch.arange(V)[lot] % 997 * 1e-3
    compare(z.to(DEV), torch.tensor([5]), torch.ones(1), torch.ones(1), 32)


@pytest.mark.parametrize("value", [-math.inf, -1e9, 0.0])
@pytest.mark.parametrize("R", [2, 515])
def test_few_tokens_above_a_mask(R, value):
    # fewer tokens above the mask's value than alternatives, in one place, at both ends, and with a lower one
    V = 40000
    z = torch.full((R, V), value)
    z[0, 20000:20004] = torch.tensor([1.0, 3.0, 2.0, 3.0])
    z[1, [0, 7, V - 1]] = torch.tensor([5.0, 4.0, 6.0])
    if value != -math.inf:
        z[1, 3] = -math.inf
    t = torch.full((R,), 20001)
    t[1] = V - 1
    compare(z.to(DEV), t, torch.ones(R), torch.ones(R), 20)


def test_ties_with_the_bound_far_behind():
    # logits equal to the bound that the first ids do not hold
    V = 60000
    z = torch.full((1, V), -1.0)
    z[0, 30000:] = 2.0
    z[0, 59999] = 3.0
    compare(z.to(DEV), torch.tensor([1]), torch.ones(1), torch.ones(1), 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_largest_vocabulary_with_alternatives(dtype):
    z, t, a, b = rows(2, 1 << 18, dtype, 3)
    compare(z.to(DEV), t, a, b, 32)
    with pytest.raises(ValueError):
        token_logprobs(torch.zeros(1, (1 << 18) + 1, device=DEV), torch.zeros(1, dtype=torch.long, device=DEV), top_k=1)


@pytest.mark.parametrize("offset", range(8))
def test_every_alignment(offset):
    z, t, a, b = rows(1, 300 + offset, torch.bfloat16, offset)
    buf = torch.empty(400, dtype=torch.bfloat16, device=DEV)
    view = buf[offset:offset + 300 + offset].view(1, -1)
    view.copy_(z)
    compare(view, t, a, b, 7, ref=z)
    zs, ts, a, b = rows(1, 3, torch.bfloat16, offset)
    view = buf[offset:offset + 3].view(1, -1)
    view.copy_(zs)
    compare(view, ts, a, b, 3, ref=zs)


def test_strided_views_are_read_in_place():
    B, S, V = 3, 5, 501
    g = torch.Generator().manual_seed(1)
    full = (torch.randn(B, S, V + 3, generator=g) * 2).bfloat16().to(DEV)
    view = full[:, :-1, 1:V + 1]  # rows at odd elements, a gap after every batch entry
    t = torch.randint(V, (B * (S - 1),), generator=g)
    a, b = torch.randn(t.numel(), generator=g), torch.randn(t.numel(), generator=g)
    compare(view, t, a, b, 5, ref=view.reshape(-1, V))
    keep = full.clone()
    token_logprobs(view, t.to(DEV).view(B, S - 1))
    assert torch.equal(full, keep)
    swapped = full.transpose(0, 1)[..., :V]
    t2 = torch.randint(V, (S * B,), generator=g)
    a2 = torch.randn(S * B, generator=g)
    compare(swapped, t2, a2, a2, 3, ref=swapped.reshape(-1, V))
    column = full.permute(0, 2, 1)[:, :S, :]  # no unit stride in the last dimension: copied
    t3 = torch.randint(S, (B * S,), generator=g)
    compare(column, t3, a2[:B * S], a2[:B * S], 2, ref=column.reshape(-1, S))


def test_one_gradient_alone_and_none():
    z, t, a, _ = rows(4, 777, torch.float32)
    zd = z.to(DEV).requires_grad_(True)
    for pick in ("logprobs", "entropy"):
        o = token_logprobs(zd, t.to(DEV))
        g, = torch.autograd.grad(getattr(o, pick).sum(), zd)
        one, zero = torch.ones(4), torch.zeros(4)
        w = (one, zero) if pick == "logprobs" else (zero, one)
        want = oracle(z, t, 0, -100, 1.0, *w)
        check(g, want[4], bounds(z, 1.0, *w, want)[3])
    with torch.no_grad():
        assert not token_logprobs(zd, t.to(DEV)).logprobs.requires_grad
    empty = token_logprobs(zd[:0], t.to(DEV)[:0], top_k=2)
    assert empty.logprobs.shape == (0,) and torch.autograd.grad(empty.logprobs.sum(), zd)[0].abs().sum() == 0


def test_other_stream_and_graph_replays():
    z, t, a, b = rows(6, 50257, torch.bfloat16)
    zd, td, ad, bd = (x.to(DEV) for x in (z, t, a, b))

    def step(x):
        x = x.detach().requires_grad_(True)
        o = token_logprobs(x, td, top_k=5)
        return [o.logprobs.detach(), o.entropy.detach(), o.top_logprobs, o.top_ids,
                torch.autograd.grad([o.logprobs, o.entropy], [x], [ad, bd])[0]]

    want = step(zd)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(zd)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    static = zd.clone()
    with torch.cuda.stream(s):
        step(static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(3):
        static.copy_(torch.roll(zd, i, 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step(static)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,k", [(1, 1), (3, 3), (32, 32), (32, 5), (700, 32), (9001, 8)])
def test_nan_at_the_first_token(V, k, dtype):
    # alone, with others behind it, everywhere, with an infinity; as many alternatives as tokens among the sizes
    z, t, a, b = rows(5, V, dtype, V)
    z[0, 0] = math.nan
    z[1] = math.nan
    z[2, [0, V // 2, V - 1]] = math.nan
    z[3, 0], z[3, V - 1] = math.nan, math.inf
    compare(z.to(DEV), t, a, b, k)


@pytest.mark.parametrize("temperature", [0.5, 0.7, 1.3])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_logits_at_the_ends_of_their_type(dtype, temperature):
    z, t, a, b = rows(7, 65, dtype)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z[0] = low
    z[1] = low
    z[1, 3:] = -math.inf
    t[1] = 2
    z[2, 5:] = low
    t[2] = 1
    z[3] = high
    z[4, 7] = 0.8 * high  # one token is certain
    t[4] = 7
    z[5, 1::2] = low / 2
    t[5] = 4
    compare(z.to(DEV), t, a, b, 1, temperature)


def test_a_poisoned_row_has_no_gradient_but_nan():
    z, t, a, b = rows(3, 40, torch.float32)
    z[:, 20:] = -math.inf
    t[0], t[1], t[2] = 40, 3, 5
    b[1] = math.nan
    zd = z.to(DEV).requires_grad_(True)
    o = token_logprobs(zd, t.to(DEV), top_k=3)
    g, = torch.autograd.grad([o.logprobs, o.entropy], [zd], [a.to(DEV), b.to(DEV)])
    assert torch.isnan(o.logprobs[0]) and torch.isfinite(o.entropy).all() and torch.isfinite(o.top_logprobs).all()
    assert torch.isnan(g[:2]).all() and torch.isfinite(g[2]).all() and (g[2, 20:] == 0).all()


def test_longest_row():
    # 2^31 - 2 logits, the most that a row may have: equal but for the last two, one of which is the target
    V = (1 << 31) - 2
    z = torch.zeros(1, V, dtype=torch.bfloat16, device=DEV)
    z[0, V - 2:] = torch.tensor([15.0, 20.0])
    z.requires_grad_(True)
    o = token_logprobs(z, torch.tensor([V - 1], device=DEV))
    total = V - 2 + math.exp(15.0) + math.exp(20.0)
    want = 20.0 - math.log(total)
    # sums of whole powers of two up to 2^31 are exact, the others and the logarithm are rounded a few times
    assert abs(float(o.logprobs.detach()) - want) <= 16 * 2.0 ** -24 * math.log(total)
    g, = torch.autograd.grad(o.logprobs.sum(), z)
    p = torch.tensor([1.0, math.exp(15.0), math.exp(20.0)], dtype=torch.float64) / total
    got = torch.stack([g[0, :1].double().cpu()[0], *g[0, V - 2:].double().cpu()])
    expect = torch.stack([-p[0], -p[1], 1 - p[2]])
    # rounded to bf16 (2^-8); exponents of up to 31 are rounded a few times in fp32
    assert ((got - expect).abs() <= expect.abs() * (2.0 ** -8 + 256 * 2.0 ** -24) + 2.0 ** -22 * p[2]).all()
    assert bool((g[0, :V - 2] == g[0, 0]).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R", [3, 515])
def test_ties_at_the_last_places(R, dtype):
    """The k-th place is shared by logits anywhere in the row: behind the first ids, beside larger ones, at both ends."""
    V, k = 30011, 20
    g = torch.Generator().manual_seed(R)
    z = (torch.rand(R, V, generator=g) * 4 - 8).to(dtype)
    for r in range(R):
        n = r % (k + 1)  # this many above the tied ones
        at = torch.randperm(V, generator=g)[:n + 60]
        z[r, at[:n]] = torch.linspace(2, 6, max(n, 1))[:n].to(dtype)
        z[r, at[n:]] = 1.0
        if r % 3 == 0:
            z[r, V - 1] = 1.0
        if r % 3 == 1:
            z[r, 2000:] = torch.where(z[r, 2000:] < 0, torch.zeros((), dtype=dtype), z[r, 2000:])  # and a flood below
        if n and r % 2:
            z[r, (at[:n] + 1).clamp(max=V - 1)] = 1.0  # tied ones in the batches of larger ones
    t, a = torch.full((R,), 5), torch.ones(R)
    zd = z.to(DEV)
    out = token_logprobs(zd, t.to(DEV), top_k=k)
    assert torch.equal(out.top_ids.cpu(), torch.sort(z, dim=1, descending=True, stable=True)[1][:, :k])
    compare(zd[:3], t[:3], a[:3], a[:3], k)


@pytest.mark.parametrize("kind", ["any", "few allowed", "one of four masked"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives_do_not_sweep_ordinary_rows(kind, dtype):
    """Twenty alternatives of ordinary rows cost little more than none: a sweep for each was 10 to 50 times that."""
    z = torch.randn(520, 50257, device=DEV, generator=torch.Generator(DEV).manual_seed(1)) * 2.5
    if kind == "few allowed":
        z[:, :50250] = -math.inf
    elif kind == "one of four masked":
        z[:, ::4] = -math.inf
    z = z.to(dtype)
    t = torch.zeros(520, dtype=torch.long, device=DEV)

    def time(k):
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                token_logprobs(z, t, top_k=k)
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    assert time(20) < 4 * time(0)
