"""FusedAdam with 8-bit moments on the CPU path: the oracle's steps, layouts, checkpoints, refusals."""
import copy

import numpy as np
import pytest
import torch

from hyperion.ops import FusedAdam, FusedAdamW

import adam8_oracle as o


def run_against_oracle(shapes, dtype, dev, steps=4, adamw=True, wd=0.1, scale=1.0, gdtype=None, seed=0, layout=None):
    """Steps an optimizer and the oracle side by side from the optimizer's own codes; checks every step."""
    rng = np.random.default_rng(seed)
    lr, b1, b2, eps = 1e-2, 0.9, 0.999, 1e-8
    ps = [torch.nn.Parameter(torch.tensor(rng.normal(size=s), dtype=torch.float32).to(dtype).to(dev)) for s in shapes]
    if layout is not None:
        for p in ps:
            if p.dim() == 4:
                p.data = p.data.contiguous(memory_format=layout)
    opt = FusedAdam(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, adamw=adamw, state_bits=8)
    if scale != 1.0:
        opt.inv_scale = torch.tensor([scale], device=dev)
    flat = lambda t, p: (t.permute(0, 2, 3, 1) if p.dim() == 4 and layout is not None else t).reshape(-1)  # noqa: E731
    for t in range(1, steps + 1):
        before = []
        for p in ps:
            g = torch.tensor(rng.normal(size=p.shape) * 10.0 ** rng.uniform(-6, 0, size=p.shape), dtype=torch.float32)
            g[rng.random(p.shape) < 0.1] = 0.0
            p.grad = torch.empty_like(p).copy_(g.to(gdtype or dtype))
            st = opt.state[p]
            w = flat(st.get("master", p).detach().float(), p).cpu().numpy().copy() if st else flat(p.detach().float(), p).cpu().numpy().copy()
            m = o.decode(st["exp_avg_q"].cpu().numpy(), st["exp_avg_scale"].cpu().numpy(), False) if st else np.zeros(p.numel())
            v = o.decode(st["exp_avg_sq_q"].cpu().numpy(), st["exp_avg_sq_scale"].cpu().numpy(), True) if st else np.zeros(p.numel())
            before.append((w, flat(p.grad.float(), p).cpu().numpy(), m, v))
        opt.step()
        vm, vv = opt.moment_vectors()
        at = 0
        for p, (w, g, m, v) in zip(ps, before):
            n = p.numel()
            w1, m1, v1 = o.step(w, g, m, v, t, lr, b1, b2, eps, wd, adamw, scale)
            st = opt.state[p]
            for x, key, second in ((m1, "exp_avg", False), (v1, "exp_avg_sq", True)):
                q, s = o.encode(x, second)
                got = st[key + "_q"].cpu().numpy().astype(np.float64)
                np.testing.assert_array_equal(got, q)
                # 0.9 S + 0.1 g = S + (g - S) / 10 lies exactly halfway between two fp32 numbers where (g - S) is 5
                # modulo 10 steps of that grid, which is common; fp64, whose 0.9 and 0.1 are off by 2^-54, then
                # rounds it either way: a scale may be one step of fp32 (2^-23) off
                np.testing.assert_allclose(st[key + "_scale"].cpu().numpy(), s, rtol=2.0 ** -23, atol=0)
                value = o.decode(got, st[key + "_scale"].cpu().numpy(), second)
                vec = (vm, vv)[second][at:at + n].cpu()
                vec = flat(vec.view(p.shape), p).numpy()
                np.testing.assert_allclose(vec, value, rtol=2.0 ** -23, atol=0)
            at += n
            got = flat(st.get("master", p).detach(), p).cpu().numpy()
            # the parameter: a few fp32 roundings of it, and of an update of at most lr * |u|
            upd = np.abs(w1 - w)
            np.testing.assert_array_less(np.abs(got - w1), 2.0 ** -22 * np.abs(w1) + 2.0 ** -20 * upd + 1e-30)
            if "master" in st:
                assert torch.equal(p.detach(), st["master"].to(dtype))
    return ps, opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("adamw", [True, False])
def test_steps_against_oracle(dtype, adamw):
    run_against_oracle([(3, 5), (256,), (257,), (1,), (40, 33)], dtype, "cpu", adamw=adamw)


def test_channels_last_is_coded_in_memory_order():
    ps, opt = run_against_oracle([(5, 7, 3, 3), (4, 4)], torch.float32, "cpu", layout=torch.channels_last)
    assert opt.moment_vectors()[0].numel() == 5 * 63 + 16


def test_tracks_the_32_bit_optimizer():
    torch.manual_seed(0)
    w = torch.randn(64, 64)
    a, b = torch.nn.Parameter(w.clone()), torch.nn.Parameter(w.clone())
    o32, o8 = FusedAdamW([a], lr=1e-2), FusedAdamW([b], lr=1e-2, state_bits=8)
    for i in range(20):
        g = torch.randn(64, 64)
        a.grad, b.grad = g.clone(), g.clone()
        o32.step(), o8.step()
    m32, v32 = o32.moment_vectors()
    m8, v8 = o8.moment_vectors()
    # a code is off by at most half a level each step and the errors decay by b1 (b2): levels are
    # 2 q / 127^2 (4 q^3 / 255^4) of a block's largest apart, at most 1.6% of it
    top = m32.abs().max()
    assert float((m8 - m32).abs().max()) < 0.5 * 0.016 * 10 * float(top)
    assert float((v8 - v32).abs().max()) < 0.5 * 0.016 * 20 * float(v32.max())
    assert (v8[v32 > 0] > 0).all()


def test_zero_and_non_finite_blocks():
    p = torch.nn.Parameter(torch.ones(600))
    opt = FusedAdamW([p], lr=0.1, state_bits=8, weight_decay=0.0)
    p.grad = torch.zeros(600)
    p.grad[300] = float("inf")
    p.grad[599] = 1e-30  # its square is below the smallest number
    opt.step()
    m, v = opt.moment_vectors()
    assert (m[:256] == 0).all() and torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
    assert m[599] != 0 and v[599] == 0 and (v[512:] == 0).all()
    assert torch.isfinite(p.detach()[:256]).all() and torch.isfinite(p.detach()[301:]).all()


def test_skipped_step_and_empty_parameters():
    p, e = torch.nn.Parameter(torch.ones(10)), torch.nn.Parameter(torch.ones(0))
    opt = FusedAdamW([p, e], state_bits=8)
    opt.found_inf = torch.ones(1)
    p.grad, e.grad = torch.ones(10), torch.ones(0)
    opt.step()
    assert (p == 1).all() and (opt.moment_vectors()[0] == 0).all()
    assert FusedAdam([p], state_bits=8).moment_vectors()[0].numel() == 0


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoint_continues_exactly(bits, tmp_path):
    torch.manual_seed(1)
    p = torch.nn.Parameter(torch.randn(300).bfloat16())
    opt = FusedAdamW([p], lr=1e-2, state_bits=bits)
    grads = [torch.randn(300).bfloat16() for _ in range(6)]
    for g in grads[:3]:
        p.grad = g.clone()
        opt.step()
    torch.save({"o": opt.state_dict(), "p": p.detach()}, tmp_path / "c.pt")
    doc = torch.load(tmp_path / "c.pt", weights_only=True)
    p2 = torch.nn.Parameter(doc["p"].clone())
    opt2 = FusedAdamW([p2], lr=1e-2, state_bits=bits)
    opt2.load_state_dict(doc["o"])
    assert opt2.state[p2]["master"].dtype == torch.float32
    for g in grads[3:]:
        p.grad, p2.grad = g.clone(), g.clone()
        opt.step(), opt2.step()
    assert torch.equal(p, p2) and torch.equal(opt.state[p]["master"], opt2.state[p2]["master"])
    assert all(torch.equal(a, b) for a, b in zip(opt.moment_vectors(), opt2.moment_vectors()))


def test_refusals():
    p = torch.nn.Parameter(torch.randn(300))
    for bad in (dict(state_bits=4), dict(state_bits=8, betas=(0.9, 1.0)), dict(state_bits=8, betas=(-0.1, 0.9))):
        with pytest.raises(ValueError):
            FusedAdam([p], **bad)
    p.grad = torch.randn(300)
    o8, o32 = FusedAdam([p], state_bits=8), FusedAdam([p])
    o8.step(), o32.step()
    sd8, sd32 = o8.state_dict(), o32.state_dict()
    with pytest.raises(ValueError, match="8-bit"):
        FusedAdam([p]).load_state_dict(sd8)
    with pytest.raises(ValueError, match="exp_avg_q"):
        FusedAdam([p], state_bits=8).load_state_dict(sd32)
    for key, value in (("exp_avg_scale", torch.zeros(1)), ("exp_avg_q", torch.zeros(299, dtype=torch.int8)),
                       ("exp_avg_sq_q", torch.zeros(300))):
        bad = copy.deepcopy(sd8)
        bad["state"][0][key] = value
        with pytest.raises(ValueError, match=key):
            FusedAdam([p], state_bits=8).load_state_dict(bad)


def test_memory_format_changes():
    torch.manual_seed(2)
    w = torch.randn(5, 7, 3, 3)

    def stepped(fmt, bits, dtype=torch.float32):
        p = torch.nn.Parameter(w.to(dtype, memory_format=fmt))
        opt = FusedAdamW([p], state_bits=bits)
        p.grad = torch.ones_like(p)
        opt.step()
        return p, opt

    p, opt = stepped(torch.channels_last, 8)
    other = torch.nn.Parameter(w.clone())
    with pytest.raises(ValueError, match="memory format"):
        FusedAdamW([other], state_bits=8).load_state_dict(opt.state_dict())
    same = torch.nn.Parameter(w.to(memory_format=torch.channels_last))
    FusedAdamW([same], state_bits=8).load_state_dict(opt.state_dict())
    p.data = p.data.contiguous()
    p.grad = torch.ones(5, 7, 3, 3)
    with pytest.raises(ValueError, match="memory format"):
        opt.step()
    p.data, p.grad = torch.randn(9), torch.randn(9)
    with pytest.raises(ValueError, match="size"):
        opt.step()
    # 32 bits: the moments and masters take the parameter's layout, whatever the saved one
    p, opt = stepped(torch.channels_last, 32, torch.bfloat16)
    q = torch.nn.Parameter(w.bfloat16())
    o2 = FusedAdamW([q])
    o2.load_state_dict(opt.state_dict())
    for k in ("exp_avg", "exp_avg_sq", "master"):
        assert o2.state[q][k].stride() == q.stride() and torch.equal(o2.state[q][k], opt.state[p][k])


def at_the_borders(dev):
    """One step with betas of 1/2 from nothing, whose moments lie exactly on the borders between two codes."""
    k = torch.arange(127.0)
    g = torch.zeros(4, 256)
    g[0, :127], g[0, 127] = (k + 0.5) ** 2, 127.0 ** 2  # m' = g / 2: the border of k and k + 1 under S = 127^2 / 2
    g[1] = -g[0]
    g[2, 0], g[2, 1:6] = 1.0, torch.tensor([0.25, -0.25, 0.25 + 2.0 ** -25, 0.25 - 2.0 ** -25, 0.0])  # v' / S = 1 / 16
    g[3, :3] = torch.tensor([1.0, 0.25, 0.0])  # m' / S = 1 / 4: 63.5
    p = torch.nn.Parameter(torch.zeros(4, 256, device=dev))
    opt = FusedAdam([p], betas=(0.5, 0.5), state_bits=8)
    p.grad = g.to(dev)
    opt.step()
    st = opt.state[p]
    return st["exp_avg_q"].view(4, 256).cpu(), st["exp_avg_sq_q"].view(4, 256).cpu(), st


def check_borders(dev):
    m, v, _ = at_the_borders(dev)
    k = torch.arange(127)
    assert torch.equal(m[0, :127].long(), k) and m[0, 127] == 127  # a half goes to the lower code
    assert torch.equal(m[1, :127].long(), -k) and m[1, 127] == -127
    assert m[3, 1] == 63
    assert v[2, :6].tolist() == [255, 127, 127, 128, 127, 0]


def test_borders_between_two_codes():
    check_borders("cpu")


def run_main_grads(dtype, dev, adamw):
    """fp32 gradients (``main_grad``) of low-precision parameters with masters, step by step against the oracle."""
    rng = np.random.default_rng(11)
    lr, b1, b2, eps, wd = 1e-2, 0.9, 0.999, 1e-8, 0.1
    ps = [torch.nn.Parameter(torch.tensor(rng.normal(size=s), dtype=torch.float32).to(dtype).to(dev))
          for s in ((3, 5), (257,), (2, 8193))]
    opt = FusedAdam(ps, lr=lr, betas=(b1, b2), eps=eps, weight_decay=wd, adamw=adamw, state_bits=8)
    ws = [p.detach().double().reshape(-1).cpu().numpy() for p in ps]
    ms, vs = [np.zeros(p.numel()) for p in ps], [np.zeros(p.numel()) for p in ps]
    for t in range(1, 4):
        for p in ps:
            g = rng.normal(size=p.shape) * 10.0 ** rng.uniform(-6, 0, size=p.shape)
            p.main_grad = torch.tensor(g, dtype=torch.float32).to(dev)  # (most have more digits than dtype holds)
        opt.step()
        for i, p in enumerate(ps):
            g = p.main_grad.reshape(-1).cpu().numpy()
            w1, m1, v1 = o.step(ws[i].astype(np.float32), g, ms[i], vs[i], t, lr, b1, b2, eps, wd, adamw)
            st = opt.state[p]
            for x, key, second, into in ((m1, "exp_avg", False, ms), (v1, "exp_avg_sq", True, vs)):
                q, s = o.encode(x, second)
                got, scale = st[key + "_q"].cpu().numpy().astype(np.float64), st[key + "_scale"].cpu().numpy()
                np.testing.assert_array_equal(got, q)
                np.testing.assert_allclose(scale, s, rtol=2.0 ** -23, atol=0)  # (one step of fp32, as above)
                into[i] = o.decode(got, scale, second)
            # the master: a few fp32 roundings of it, and of its update
            got = st["master"].reshape(-1).double().cpu().numpy()
            np.testing.assert_array_less(np.abs(got - w1), 2.0 ** -22 * np.abs(w1) + 2.0 ** -20 * np.abs(w1 - ws[i]) + 1e-30)
            assert st["master"].dtype == torch.float32 and torch.equal(p.detach(), st["master"].to(dtype))
            ws[i] = got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("adamw", [True, False])
def test_fp32_gradients_of_low_precision_parameters(dtype, adamw):
    run_main_grads(dtype, "cpu", adamw)


def check_refused_step(dev):
    torch.manual_seed(7)
    p, q = torch.nn.Parameter(torch.randn(300, device=dev)), torch.nn.Parameter(torch.randn(5, 7, 3, 3, device=dev))
    opt = FusedAdamW([p, q], state_bits=8)
    for x in (p, q):
        x.grad = torch.randn_like(x)
    opt.step()
    before, saved = p.detach().clone(), copy.deepcopy(opt.state_dict())
    q.data = q.data.contiguous(memory_format=torch.channels_last)
    with pytest.raises(ValueError, match="memory format"):
        opt.step()
    assert torch.equal(p, before) and opt.state_dict()["hyperion_step"] == saved["hyperion_step"] == 1
    for k in ("exp_avg_q", "exp_avg_sq_q", "exp_avg_scale", "exp_avg_sq_scale"):
        assert torch.equal(opt.state[p][k], saved["state"][0][k])
    held, q.grad = q.grad, None
    opt.step(), opt.step()  # q takes no part
    q.grad = held
    with pytest.raises(ValueError, match="memory format"):
        opt.step()
    q.data = q.data.contiguous()
    opt.step()
    assert opt.state_dict()["hyperion_step"] == 4


def test_a_refused_step_changes_nothing():
    check_refused_step("cpu")
