"""token_logprobs: the PyTorch path against the 64-bit oracle, its gradient against differences, refusals."""
import math

import pytest
import torch

from hyperion.ops.token_logprobs import TOP_MAX, token_logprobs

from token_logprobs_oracle import bounds, check, oracle


def rows(R, V, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(R, V, generator=g) * 2.5).to(dtype)
    return z, torch.randint(V, (R,), generator=g), torch.randn(R, generator=g), torch.randn(R, generator=g)


def compare(z, t, dlogp, dent, k, temperature=1.0):
    z = z.clone().requires_grad_(True)
    out = token_logprobs(z, t, top_k=k, temperature=temperature)
    g, = torch.autograd.grad([out.logprobs, out.entropy], [z], [dlogp, dent])
    want = oracle(z, t, k, -100, temperature, dlogp, dent)
    b = bounds(z, temperature, dlogp, dent, want)
    check(out.logprobs, want[0], b[0])
    check(out.entropy, want[1], b[1])
    if k:
        assert torch.equal(out.top_ids.cpu(), want[3])
        check(out.top_logprobs, want[2], b[2])
    check(g, want[4], b[3])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V", [1, 2, 33, 1000])
def test_against_oracle(V, dtype):
    z, t, a, b = rows(5, V, dtype, V)
    t[1] = -100
    compare(z, t, a, b, min(5, V), temperature=0.7)


def test_masked_empty_and_poisoned_rows():
    z, t, a, b = rows(7, 65, torch.float32)
    z[0] = -math.inf  # empty
    z[1, 3:] = -math.inf
    t[1] = 40  # a masked token
    z[2, 7] = math.nan
    z[3, 9] = math.inf
    t[4] = 65  # outside
    t[5] = -7
    z[6] = -math.inf
    z[6, 11] = 2.0  # one token left
    t[6] = 11
    compare(z, t, a, b, 4)


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
    compare(z, t, a, b, 1, temperature)


def test_a_poisoned_row_has_no_gradient_but_nan():
    z, t, a, b = rows(3, 40, torch.float32)
    z[:, 20:] = -math.inf
    t[0], t[1], t[2] = 40, 3, 5
    b[1] = math.nan
    zd = z.requires_grad_(True)
    o = token_logprobs(zd, t, top_k=3)
    g, = torch.autograd.grad([o.logprobs, o.entropy], [zd], [a, b])
    assert torch.isnan(o.logprobs[0]) and torch.isfinite(o.entropy).all() and torch.isfinite(o.top_logprobs).all()
    assert torch.isnan(g[:2]).all() and torch.isfinite(g[2]).all() and (g[2, 20:] == 0).all()


@pytest.mark.parametrize("V,k", [(1, 1), (3, 3), (32, 5)])
def test_nan_at_the_first_token(V, k):
    z, t, a, b = rows(4, V, torch.float32, V)
    z[0, 0] = math.nan
    z[1] = math.nan
    z[2, [0, V - 1]] = math.nan
    compare(z, t, a, b, k)


def test_gradient_against_differences():
    z, t, a, b = rows(3, 11, torch.float32)

    def f(x):  # the objective in 64 bits
        ls = torch.log_softmax(x / 1.3, 1)
        return float((a * ls.gather(1, t[:, None])[:, 0]).sum() - (b * (ls.exp() * ls).sum(1)).sum())

    zr = z.clone().requires_grad_(True)
    o = token_logprobs(zr, t, temperature=1.3)
    g, = torch.autograd.grad([o.logprobs, o.entropy], [zr], [a, b])
    zd, e = z.double(), 1e-5
    for r in range(3):
        for j in range(11):
            d = torch.zeros_like(zd)
            d[r, j] = e
            # a central difference is off by e^2 / 6 of the third derivative (at most about 10 here)
            assert abs((f(zd + d) - f(zd - d)) / (2 * e) - float(g[r, j])) < 1e-6


def test_shapes_and_broadcast_gradients():
    z = torch.randn(2, 3, 4, 9, requires_grad=True)
    t = torch.randint(9, (2, 3, 4), dtype=torch.int32)
    o = token_logprobs(z, t, top_k=2)
    assert o.logprobs.shape == (2, 3, 4) and o.top_ids.shape == (2, 3, 4, 2) and not o.top_logprobs.requires_grad
    o.logprobs.sum().backward()  # an expanded gradient
    want = torch.autograd.grad(torch.log_softmax(z, -1).gather(-1, t.long()[..., None]).sum(), z)[0]
    torch.testing.assert_close(z.grad, want, atol=1e-6, rtol=1e-5)
    one = token_logprobs(z[0, 0, 0].detach(), torch.tensor(3), top_k=9)
    assert one.logprobs.shape == () and one.top_ids.shape == (9,)
    none = token_logprobs(torch.zeros(0, 5), torch.zeros(0, dtype=torch.long), top_k=1)
    assert none.logprobs.shape == (0,) and none.top_ids.shape == (0, 1)


def test_refusals():
    z, t = torch.randn(3, 40), torch.zeros(3, dtype=torch.long)
    for bad in (dict(logits=z.double()), dict(target=t.float())):
        with pytest.raises(TypeError):
            token_logprobs(**{"logits": z, "target": t, **bad})
    for bad in (dict(target=t[:2]), dict(top_k=-1), dict(top_k=TOP_MAX + 1), dict(logits=z[:, :4], top_k=5),
                dict(temperature=0.0), dict(temperature=math.nan), dict(logits=z[:, :0])):
        with pytest.raises(ValueError):
            token_logprobs(**{"logits": z, "target": t, **bad})
