"""MXFP4: the PyTorch path against the 64-bit oracle, the layer and its refusals."""
import math

import pytest
import torch
import torch.nn as nn

from hyperion.ops.mxfp4 import MXFP4Linear, MXFP4Tensor, mxfp4_linear, quantize_mxfp4

from mxfp4_oracle import decoded, product_bound, quantized_values

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (3, 31), (2, 64), (5, 100)])
def test_quantize_against_oracle(R, K, dtype):
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(K)).to(dtype)
    q = quantize_mxfp4(x)
    assert q.nbytes == R * 17 * -(-K // 32)
    assert torch.equal(q.dequantize(torch.float32).double(), quantized_values(x))
    assert torch.equal(decoded(q.codes, q.scales, K), quantized_values(x))


def test_quantize_edges():
    x = torch.zeros(6, 64)
    x[0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 4.0])
    x[1, 3], x[1, 40] = math.nan, 1.0
    x[2, 3], x[2, 40] = -math.inf, 1.0
    x[3] = torch.linspace(0, 3e38, 64)
    x[4] = torch.linspace(0, 3e-44, 64)
    x[5, 0] = -0.0
    got = quantize_mxfp4(x).dequantize(torch.float32).double()
    want = quantized_values(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert torch.isnan(got[1, :32]).all() and torch.isfinite(got[1, 32:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_and_its_gradient(dtype):
    g = torch.Generator().manual_seed(2)
    w = quantize_mxfp4(torch.randn(20, 70, generator=g))
    x = torch.randn(3, 4, 70, generator=g).to(dtype).requires_grad_(True)
    b = torch.randn(20, generator=g).requires_grad_(True)
    dy = torch.randn(3, 4, 20, generator=g).to(dtype)
    y = mxfp4_linear(x, w, b)
    assert y.dtype == dtype and y.shape == (3, 4, 20)
    dx, db = torch.autograd.grad(y, [x, b], dy)
    W = decoded(w.codes, w.scales, 70)
    x2, d2 = x.detach().double().view(12, 70), dy.double().view(12, 20)
    want = x2 @ W.t() + b.detach().double()
    bound = product_bound(x2, W.t(), dtype) + (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * (b.detach().double().abs() + want.abs())
    assert ((y.detach().double().view(12, 20) - want).abs() <= bound).all()
    assert ((dx.double().view(12, 70) - d2 @ W).abs() <= product_bound(d2, W, dtype)).all()
    torch.testing.assert_close(db, d2.sum(0).float(), atol=1e-5, rtol=1e-5)


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    w = quantize_mxfp4(torch.randn(5, 33, generator=g))
    x = torch.randn(2, 33, generator=g)
    xr = x.clone().requires_grad_(True)
    mxfp4_linear(xr, w).square().sum().backward()
    W = w.dequantize(torch.float32).double()
    for i, j in ((0, 0), (1, 32), (0, 17)):
        e = torch.zeros(2, 33, dtype=torch.float64)
        e[i, j] = 1e-3
        f = lambda t: float((t @ W.t()).square().sum())  # noqa: E731 - quadratic: central differences are exact
        d = (f(x.double() + e) - f(x.double() - e)) / 2e-3
        assert abs(d - float(xr.grad[i, j])) < 1e-4 * (1 + abs(d))


def test_layer_state_dict_and_casts():
    lin = nn.Linear(40, 6)
    m = MXFP4Linear.from_linear(lin)
    assert m.bias is lin.bias and not hasattr(m, "weight_orig")
    x = torch.randn(2, 40)
    torch.testing.assert_close(m(x), nn.functional.linear(x, m.weight.dequantize(torch.float32), lin.bias), atol=1e-5, rtol=1e-5)
    fresh = MXFP4Linear(40, 6)
    fresh.load_state_dict(m.state_dict())
    assert torch.equal(fresh(x), m(x))
    m.to(torch.bfloat16)
    assert m.weight_codes.dtype == torch.uint8 and m(x.bfloat16()).dtype == torch.bfloat16
    assert mxfp4_linear(x[:0], fresh.weight).shape == (0, 6)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert mxfp4_linear(x, fresh.weight).dtype == torch.bfloat16


@pytest.mark.parametrize("M,N,K", [(0, 4, 40), (3, 0, 40), (3, 4, 0), (0, 0, 0)])
def test_empty_sizes(M, N, K):
    w = quantize_mxfp4(torch.randn(N, K, device="cpu"))
    assert w.dequantize().shape == (N, K)
    x, b = torch.randn(M, K, device="cpu", requires_grad=True), torch.randn(N, device="cpu", requires_grad=True)
    y = mxfp4_linear(x, w, b)
    assert torch.equal(y, b.detach().expand(M, N))  # sums over nothing
    dx, db = torch.autograd.grad(y.sum(), [x, b])
    assert dx.shape == x.shape and (N or not dx.any())
    assert torch.equal(db, torch.full_like(b, M))


def test_refusals():
    q = quantize_mxfp4(torch.randn(4, 40))
    x = torch.randn(2, 40)
    for bad in (lambda: quantize_mxfp4(x.double()), lambda: mxfp4_linear(x.double(), q), lambda: q.dequantize(torch.float64),
                lambda: mxfp4_linear(x, q.codes), lambda: mxfp4_linear(x, quantize_mxfp4(torch.randn(2, 3, 40))),
                lambda: MXFP4Tensor(q.codes.int(), q.scales, q.shape)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: quantize_mxfp4(torch.tensor(1.0)), lambda: mxfp4_linear(x[:, :39], q),
                lambda: mxfp4_linear(x, q, torch.zeros(5)), lambda: MXFP4Tensor(q.codes, q.scales, (4, 65)),
                lambda: MXFP4Tensor(q.codes[:3], q.scales, q.shape), lambda: mxfp4_linear(x, q, torch.zeros(4, dtype=torch.long))):
        with pytest.raises(ValueError):
            bad()


def test_a_weight_loaded_before_the_backward_is_noticed():
    m = MXFP4Linear.from_linear(nn.Linear(64, 8))
    other = MXFP4Linear.from_linear(nn.Linear(64, 8))
    x = torch.randn(3, 64, requires_grad=True)
    y, z = m(x), other(x)
    m.load_state_dict(other.state_dict())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z.sum().backward()
    assert x.grad is not None


def test_a_weight_quantised_in_inference_mode_trains():
    with torch.inference_mode():
        w = quantize_mxfp4(torch.randn(8, 64))
    x = torch.randn(3, 64, requires_grad=True)
    mxfp4_linear(x, w).sum().backward()
    torch.testing.assert_close(x.grad, w.dequantize(torch.float32).sum(0).expand(3, 64), atol=1e-5, rtol=1e-5)
