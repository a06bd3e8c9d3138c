"""MXFP4 kernels against the 64-bit oracle: types, odd sizes, strides, edges, both products, graphs, streams."""
import math

import pytest
import torch
import torch.nn as nn

from hyperion.ops import _native
from hyperion.ops.mxfp4 import MXFP4Linear, MXFP4Tensor, mxfp4_linear, quantize_mxfp4

from mxfp4_oracle import decoded, product_bound, quantized_values

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def same(got, want):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,K", [(1, 1), (3, 31), (2, 64), (5, 100), (1023, 500), (70, 4096)])
def test_quantize_against_oracle(R, K, dtype):
    x = torch.randn(R, K, generator=torch.Generator().manual_seed(K)).to(dtype)
    q = quantize_mxfp4(x.to(DEV))
    want = quantized_values(x)
    same(q.dequantize(torch.float32), want)
    same(q.dequantize(torch.bfloat16), want)
    same(q.dequantize(torch.float16), want.half().double())
    assert torch.equal(decoded(q.codes, q.scales, K), want)
    ref = quantize_mxfp4(x)
    assert torch.equal(q.codes.cpu(), ref.codes) and torch.equal(q.scales.cpu(), ref.scales)


def test_quantize_edges_and_strides():
    x = torch.zeros(7, 64)
    x[0, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, 4.0])
    x[1, 3], x[1, 40] = math.nan, 1.0
    x[2, 3], x[2, 40] = -math.inf, 1.0
    x[3] = torch.linspace(0, 3e38, 64)
    x[4] = torch.linspace(0, 3e-38, 64)
    x[5, 0] = -0.0
    x[6] = torch.linspace(0, 3e-44, 64)
    same(quantize_mxfp4(x.to(DEV)).dequantize(torch.float32), quantized_values(x))
    y = torch.randn(9, 77, generator=torch.Generator().manual_seed(1)).bfloat16()
    yd = y.to(DEV)
    same(quantize_mxfp4(yd[:, 3:70]).dequantize(torch.float32), quantized_values(y[:, 3:70]))  # rows at odd elements
    same(quantize_mxfp4(yd.t()).dequantize(torch.float32), quantized_values(y.t()))
    same(quantize_mxfp4(yd[None, ::2]).dequantize(torch.float32)[0], quantized_values(y[::2]))
    assert quantize_mxfp4(yd[:0]).dequantize().shape == (0, 77)


def check_linear(M, N, K, dtype, bias, seed=0, view=lambda t: t):
    g = torch.Generator().manual_seed(seed + M + N + K)
    w = quantize_mxfp4(torch.randn(N, K, generator=g).to(DEV))
    x = view(torch.randn(M, K, generator=g).to(dtype).to(DEV)).detach().requires_grad_(True)
    b = torch.randn(N, generator=g).to(DEV).requires_grad_(True) if bias else None
    dy = torch.randn(x.shape[0], N, generator=g).to(dtype).to(DEV)
    y = mxfp4_linear(x, w, b)
    dx = torch.autograd.grad(y, x, dy)[0]
    # the oracle's products run on the device in fp64
    W = decoded(w.codes, w.scales, K).to(DEV)
    xd, dd = x.detach().double(), dy.double()
    want, bound = xd @ W.t(), product_bound(xd, W.t(), dtype)
    if bias:
        want = want + b.detach().double()
        bound = bound + (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * (b.detach().double().abs() + want.abs())
    assert y.dtype == dtype and ((y.detach().double() - want).abs() <= bound).all()
    assert dx.dtype == dtype and ((dx.double() - dd @ W).abs() <= product_bound(dd, W, dtype)).all()
    return w, x, dy, y, dx


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 16, 32), (1, 1, 1), (3, 7, 33), (16, 100, 1000), (17, 200, 129), (40, 24, 64),
                                   (64, 50, 4096), (65, 100, 100), (130, 257, 500), (300, 1000, 768), (1, 4096, 4096)])
def test_linear_against_oracle(M, N, K, dtype):
    check_linear(M, N, K, dtype, bias=M % 2 == 1)


@pytest.mark.parametrize("M", [1, 5, 96])
def test_strided_activations(M):
    check_linear(M, 40, 96, torch.bfloat16, True, view=lambda t: torch.cat([t, t], 1)[:, 1:97])
    check_linear(96, 40, M, torch.bfloat16, False, view=lambda t: t.t().contiguous().t())


@pytest.mark.parametrize("M,N,K", [(1, 100, 160), (33, 300, 96), (70, 72, 384), (200, 264, 1056), (5, 1030, 2048), (40, 128, 128)])
def test_every_tile_gives_the_same_product(M, N, K):
    C = _native.native()
    g = torch.Generator().manual_seed(M)
    w = quantize_mxfp4(torch.randn(N, K, generator=g).to(DEV))
    W = decoded(w.codes, w.scales, K).to(DEV)
    b = torch.randn(N, generator=g).to(DEV)
    for dtype in DTYPES:
        x, dy = torch.randn(M, K, generator=g).to(dtype).to(DEV), torch.randn(M, N, generator=g).to(dtype).to(DEV)
        xd, dd = x.double(), dy.double()
        want = xd @ W.t() + b.double()
        bound = product_bound(xd, W.t(), dtype) + (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * (b.double().abs() + want.abs())
        lds = [] if w.scales.shape[1] % 4 else [(9, 1), (9, 2), (9, 4), (10, 2), (10, 4), (18, 8), (20, 8)]
        for mt, nt in [(0, 0), (1, 1), (2, 4)] + lds:
            y = C.mx_linear(x, w.codes, w.scales, b, 16 * mt + nt)
            assert ((y.double() - want).abs() <= bound).all(), (mt, nt)
        for mt in [0, 1] + ([9, 10, 18, 20] if lds else []):
            dx = C.mx_linear_dgrad(dy, w.codes, w.scales, K, mt)
            assert ((dx.double() - dd @ W).abs() <= product_bound(dd, W, dtype)).all(), mt


def test_batches_are_rows():
    w, x, dy, y, dx = check_linear(65, 64, 96, torch.bfloat16, False)
    assert torch.equal(mxfp4_linear(x.view(1, 65, 96), w)[0], y)
    assert torch.equal(mxfp4_linear(x[3], w), mxfp4_linear(x[3:4], w)[0])


def test_non_finite_activations_and_weights():
    g = torch.Generator().manual_seed(5)
    wv = torch.randn(32, 64, generator=g)
    wv[3, 40] = math.nan
    w = quantize_mxfp4(wv.to(DEV))
    for dtype in DTYPES:
        for M in (2, 70):
            x = torch.randn(M, 64, generator=g).to(dtype)
            x[1, 5] = math.inf
            y = mxfp4_linear(x.to(DEV), w).cpu()
            want = x.double() @ decoded(w.codes, w.scales, 64).t()
            assert torch.equal(torch.isfinite(y), torch.isfinite(want))
            assert torch.isnan(y[0, 3]) and torch.isfinite(y[0, 4])


def test_misaligned_codes_are_taken():
    q = quantize_mxfp4(torch.randn(8, 64, device=DEV))
    buf = torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device=DEV)
    buf[1:] = q.codes.view(-1)
    m = MXFP4Tensor(buf[1:].view(8, 32), q.scales, q.shape)
    x = torch.randn(3, 64, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(mxfp4_linear(x, m), mxfp4_linear(x, q))
    q = quantize_mxfp4(torch.randn(8, 128, device=DEV))
    buf = torch.empty(q.scales.numel() + 1, dtype=torch.uint8, device=DEV)
    buf[1:] = q.scales.view(-1)
    x = torch.randn(3, 128, device=DEV, dtype=torch.bfloat16)
    assert torch.equal(mxfp4_linear(x, MXFP4Tensor(q.codes, buf[1:].view(8, 4), q.shape)), mxfp4_linear(x, q))


@pytest.mark.parametrize("M", [3, 200])
def test_other_stream_and_graph_replays(M):
    w = quantize_mxfp4(torch.randn(320, 512, device=DEV) * 0.05)
    x = torch.randn(M, 512, device=DEV, dtype=torch.bfloat16)
    dy = torch.randn(M, 320, device=DEV, dtype=torch.bfloat16)

    def step(t):
        t = t.detach().requires_grad_(True)
        y = mxfp4_linear(t, w)
        return [y.detach(), torch.autograd.grad(y, t, dy)[0], quantize_mxfp4(t).codes]

    want = step(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(x)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(3):
        static.copy_(torch.roll(x, i, 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(static)))


def test_kernels_are_reached():
    w = quantize_mxfp4(torch.randn(64, 64, device=DEV))
    _native.reset_counters()
    x = torch.randn(4, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    mxfp4_linear(x, w).sum().backward()
    assert _native.counters() == {"mxfp4_linear": 1, "mxfp4_dgrad": 1}


@pytest.mark.parametrize("M,N,K", [(0, 4, 40), (3, 0, 40), (3, 4, 0), (0, 0, 0)])
def test_empty_sizes(M, N, K):
    w = quantize_mxfp4(torch.randn(N, K, device="cuda"))
    assert w.dequantize().shape == (N, K)
    x, b = torch.randn(M, K, device="cuda", requires_grad=True), torch.randn(N, device="cuda", requires_grad=True)
    y = mxfp4_linear(x, w, b)
    assert torch.equal(y, b.detach().expand(M, N))  # sums over nothing
    dx, db = torch.autograd.grad(y.sum(), [x, b])
    assert dx.shape == x.shape and (N or not dx.any())
    assert torch.equal(db, torch.full_like(b, M))


@pytest.mark.parametrize("M,N,K,dtype", [(700, 4096, 4096, torch.bfloat16), (333, 2049, 1024, torch.bfloat16),
                                         (600, 2048, 1152, torch.float32), (1500, 1000, 2048, torch.float16),
                                         (4096, 4096, 1024, torch.bfloat16)])
def test_many_rows(M, N, K, dtype):
    """The planned products of longer batches against the oracle, eager and replayed."""
    g = torch.Generator().manual_seed(M + N)
    w = quantize_mxfp4(torch.randn(N, K, generator=g).to(DEV))
    W = decoded(w.codes, w.scales, K).to(DEV)
    x, dy = torch.randn(M, K, generator=g).to(DEV, dtype), torch.randn(M, N, generator=g).to(DEV, dtype)

    def step(t):
        t = t.detach().requires_grad_(True)
        y = mxfp4_linear(t, w)
        return [y.detach(), torch.autograd.grad(y, t, dy)[0]]

    y, dx = step(x)
    assert ((y.double() - x.double() @ W.t()).abs() <= product_bound(x.double(), W.t(), dtype)).all()
    assert ((dx.double() - dy.double() @ W).abs() <= product_bound(dy.double(), W, dtype)).all()
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(3):
        static.copy_(torch.roll(x, i, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(static)))


def test_a_weight_loaded_before_the_backward_is_noticed():
    m = MXFP4Linear.from_linear(nn.Linear(64, 8).to(DEV))
    other = MXFP4Linear.from_linear(nn.Linear(64, 8).to(DEV))
    x = torch.randn(3, 64, device=DEV, requires_grad=True)
    y, z = m(x), other(x)
    m.load_state_dict(other.state_dict())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    z.sum().backward()
    assert x.grad is not None


def test_outputs_of_more_than_2_32_elements():
    # the pieces' products of fp32 activations, joined: rows on both sides of element 2^32
    M, N, K = 1 << 19, 8200, 32
    g = torch.Generator().manual_seed(8)
    w = quantize_mxfp4(torch.randn(N, K, generator=g).to(DEV))
    x = torch.randn(64, K, generator=g).to(DEV).repeat(M // 64, 1)
    y = mxfp4_linear(x, w)
    W = decoded(w.codes, w.scales, K).to(DEV)
    want = x[:64].double() @ W.t()
    bound = product_bound(x[:64].double(), W.t(), torch.float32)
    at = (1 << 32) // N // 64 * 64
    for r in (0, at - 64, at, at + 64, M - 64):
        assert ((y[r:r + 64].double() - want).abs() <= bound).all(), r
    assert bool((y.view(-1, 64, N) == y[:64]).all())
