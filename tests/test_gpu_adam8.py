"""adam8 kernels against the 64-bit oracle: types, odd sizes, layouts, skipped steps, graphs, streams."""
import pytest
import torch

from hyperion.ops import FusedAdam, FusedAdamW, _native, clip_grad_norm_

from test_adam8_cpu import at_the_borders, check_borders, check_refused_step, run_against_oracle, run_main_grads

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(3, 5), (256,), (257,), (1,), (40, 33), (8192,), (8193,), (130, 777), (2047,)]


@pytest.mark.parametrize("gdtype", [None, torch.float32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("adamw", [True, False])
def test_steps_against_oracle(dtype, gdtype, adamw):
    _native.reset_counters()
    if gdtype is None:
        run_against_oracle(SHAPES, dtype, DEV, adamw=adamw)
    else:  # gradients scaled by the loss scaler's factor
        run_against_oracle(SHAPES, dtype, DEV, adamw=adamw, scale=2.0 ** -7)
    assert _native.counters()["adam8"] == 4


def test_without_weight_decay_and_channels_last():
    run_against_oracle([(5, 7, 3, 3), (64, 64, 3, 3), (9,)], torch.float32, DEV, adamw=False, wd=0.0, layout=torch.channels_last)


def test_same_codes_as_the_cpu():
    torch.manual_seed(0)
    w = torch.randn(100, 300)
    ps = [torch.nn.Parameter(w.clone().to(d)) for d in ("cpu", DEV)]
    opts = [FusedAdamW([p], lr=1e-2, state_bits=8) for p in ps]
    for _ in range(5):
        g = torch.randn(100, 300)
        for p, o in zip(ps, opts):
            p.grad = g.to(p.device)
            o.step()
        a, b = (o.state[p] for p, o in zip(ps, opts))
        for k in ("exp_avg_q", "exp_avg_sq_q", "exp_avg_scale", "exp_avg_sq_scale"):
            assert torch.equal(a[k], b[k].cpu()), k


def test_zero_and_non_finite_blocks():
    p = torch.nn.Parameter(torch.ones(600, device=DEV))
    opt = FusedAdamW([p], lr=0.1, state_bits=8, weight_decay=0.0)
    p.grad = torch.zeros(600, device=DEV)
    p.grad[300] = float("inf")
    p.grad[599] = 1e-30
    opt.step()
    m, v = opt.moment_vectors()
    assert (m[:256] == 0).all() and torch.isnan(m[256:512]).all() and torch.isnan(v[256:512]).all()
    assert m[599] != 0 and v[599] == 0 and (v[512:] == 0).all()
    assert torch.isfinite(p.detach()[:256]).all() and torch.isfinite(p.detach()[301:]).all()


def test_skipped_step_zeroed_gradients_and_deferred_clip():
    p = torch.nn.Parameter(torch.ones(1000, device=DEV))
    opt = FusedAdamW([p], state_bits=8)
    opt.zero_grad_in_step = True
    opt.found_inf = torch.ones(1, device=DEV)
    p.grad = torch.ones(1000, device=DEV)
    opt.step()
    assert (p == 1).all() and (p.grad == 0).all() and (opt.moment_vectors()[0] == 0).all()
    opt.found_inf = torch.zeros(1, device=DEV)
    p.grad.fill_(2.0)
    clip_grad_norm_([p], 1.0, defer_to=opt)
    opt.step()
    want = 0.1 * 2.0 / (2.0 * 1000 ** 0.5 + 1e-6)
    assert (p.grad == 0).all()
    torch.testing.assert_close(opt.moment_vectors()[0], torch.full((1000,), want, device=DEV), rtol=1e-5, atol=0)


def test_misaligned_parameters_take_the_torch_path():
    buf = torch.randn(301, device=DEV)
    p = torch.nn.Parameter(buf[1:])
    q = torch.nn.Parameter(buf[1:].clone())
    a, b = FusedAdamW([p], state_bits=8), FusedAdamW([q], state_bits=8)
    for _ in range(3):
        g = torch.randn(300, device=DEV)
        p.grad, q.grad = g.clone(), g.clone()
        a.step(), b.step()
    assert all(torch.equal(a.state[p][k], b.state[q][k]) for k in ("exp_avg_q", "exp_avg_sq_q"))
    torch.testing.assert_close(p, q, rtol=1e-6, atol=1e-7)


def test_other_stream_and_graph_replays():
    torch.manual_seed(2)
    ws = [torch.randn(300, 70, device=DEV).bfloat16(), torch.randn(9001, device=DEV).bfloat16()]
    grads = [[torch.randn_like(w) for w in ws] for _ in range(7)]
    pairs = []
    for _ in range(2):
        ps = [torch.nn.Parameter(w.clone()) for w in ws]
        for p in ps:
            p.grad = torch.zeros_like(p)
        pairs.append((ps, FusedAdamW(ps, lr=1e-2, state_bits=8)))

    def load(ps, i):
        for p, g in zip(ps, grads[i]):
            p.grad.copy_(g)

    (pa, oa), (pb, ob) = pairs
    s = torch.cuda.Stream()
    for i in range(2):
        load(pa, i)
        oa.step()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            load(pb, i)
            ob.step()
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
        values = ob.moment_vectors() if "adam8_values" in ob._tables._tables else None
    for i in range(2, 7):
        load(pa, i)
        oa.step()
        load(pb, i)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(pa, pb))
        assert all(torch.equal(x, y) for x, y in zip(oa.moment_vectors(), ob.moment_vectors()))
    assert values is None


def test_many_small_tensors_in_one_launch():
    run_against_oracle([(17, i % 9 + 1) for i in range(120)], torch.bfloat16, DEV, steps=2)


def test_tables_follow_what_changes_between_steps():
    """Steps replay the last one's tables where nothing changed: new gradients, frozen and thawed parameters, replaced
    state, a loaded checkpoint, main_grad and new hyperparameters are all noticed."""
    torch.manual_seed(3)
    ws = [torch.randn(400, device=DEV), torch.randn(31, 9, device=DEV)]
    native = [torch.nn.Parameter(w.clone()) for w in ws]
    plain = [torch.nn.Parameter(w.cpu()) for w in ws]
    a, b = FusedAdamW(native, lr=1e-2, state_bits=8), FusedAdamW(plain, lr=1e-2, state_bits=8)

    def step(which=(0, 1), main=False, keep=False):
        for i, (p, q) in enumerate(zip(native, plain)):
            if i not in which:
                p.grad = q.grad = None
                continue
            g = torch.randn(q.shape)
            if main:
                p.main_grad, q.main_grad = g.to(DEV), g.clone()
            elif keep and p.grad is not None:
                p.grad.copy_(g), q.grad.copy_(g)
            else:
                p.grad, q.grad = g.to(DEV), g.clone()
        a.step(), b.step()
        for p, q in zip(native, plain):
            for k in ("exp_avg_q", "exp_avg_sq_q", "exp_avg_scale", "exp_avg_sq_scale"):
                assert torch.equal(a.state[p][k].cpu(), b.state[q][k]) if a.state.get(p) else not b.state.get(q)
            torch.testing.assert_close(p.detach().cpu(), q.detach(), rtol=1e-6, atol=1e-7)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(a.moment_vectors(), b.moment_vectors()))

    step(which=(0,))
    for _ in range(3):
        step(keep=True)
    held = [p.grad for p in native]
    step()
    step(which=(1,))
    step(keep=True)
    for o, ps in ((a, native), (b, plain)):
        o.state[ps[0]]["exp_avg_q"] = torch.full_like(o.state[ps[0]]["exp_avg_q"], 5)
        o.param_groups[0]["lr"] = 3e-2
        o.param_groups[0]["weight_decay"] = 0.2
    step(keep=True)
    sa, sb = a.state_dict(), b.state_dict()
    step(keep=True)
    a.load_state_dict(sa), b.load_state_dict(sb)
    step(keep=True)
    step(main=True)
    step(main=True)
    for p, q in zip(native, plain):
        del p.main_grad, q.main_grad
    step(keep=True)
    assert held


def test_steps_without_changes_do_not_walk_the_tensors(monkeypatch):
    ps = [torch.nn.Parameter(torch.randn(64, device=DEV)) for _ in range(4)]
    for p in ps:
        p.grad = torch.randn_like(p)
    opt = FusedAdamW(ps, state_bits=8)
    opt.step(), opt.moment_vectors()
    monkeypatch.setattr(opt, "_step8", None)
    monkeypatch.setattr(opt._tables, "get", None)
    opt.step(), opt.moment_vectors()


def test_learning_rates_as_tensors():
    grads = [torch.randn(500, device="cuda") for _ in range(3)]
    results = []
    for lr in (0.01, torch.tensor(0.01), torch.tensor(0.01, device="cuda")):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 500, device="cuda"))
        opt = FusedAdamW([p], lr=lr, state_bits=8)
        for g in grads:
            p.grad = g
            opt.step()
        results.append(p.detach().clone())
    assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])


def test_scales_at_exact_halves():
    """0.9 S + 0.1 g is halfway between two fp32 numbers for many g a few steps from S: CPU and GPU round alike, also in the
    PyTorch path on the GPU."""
    n = 2048
    S = 1 + torch.arange(n) / n
    g = torch.zeros(n, 256)
    g[:, 7] = S * (1 + 2.0 ** -23 * (torch.arange(n) % 31))
    state = {"exp_avg_q": torch.zeros(n, 256, dtype=torch.int8), "exp_avg_sq_q": torch.zeros(n, 256, dtype=torch.uint8),
             "exp_avg_scale": S.clone(), "exp_avg_sq_scale": S.square()}
    state["exp_avg_q"][:, 7], state["exp_avg_sq_q"][:, 7] = 127, 255
    results = []
    for dev, backend in (("cpu", "hyperion"), (DEV, "hyperion"), (DEV, "torch")):
        p = torch.nn.Parameter(torch.zeros(n, 256, device=dev))
        opt = FusedAdamW([p], lr=1e-3, state_bits=8)
        opt.load_state_dict({"state": {0: {k: v.reshape(-1).to(dev) for k, v in state.items()}}, "hyperion_step": 5,
                             "param_groups": opt.state_dict()["param_groups"]})
        p.grad = g.to(dev)
        with pytest.MonkeyPatch.context() as mp:
            mp.setenv("HYPERION_KERNELS", backend)
            opt.step()
        results.append({k: opt.state[p][k].cpu() for k in state})
    for other in results[1:]:
        for k in state:
            assert torch.equal(results[0][k], other[k]), k


def test_borders_between_two_codes():
    check_borders(DEV)
    a, b = at_the_borders("cpu")[2], at_the_borders(DEV)[2]
    for k in ("exp_avg_q", "exp_avg_sq_q", "exp_avg_scale", "exp_avg_sq_scale"):
        assert torch.equal(a[k], b[k].cpu()), k


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("adamw", [True, False])
def test_fp32_gradients_of_low_precision_parameters(dtype, adamw):
    _native.reset_counters()
    run_main_grads(dtype, DEV, adamw)
    assert _native.counters()["adam8"] == 3


def test_captured_moment_vectors():
    torch.manual_seed(5)
    ws = [torch.randn(300, 70, device=DEV).bfloat16(), torch.randn(9001, device=DEV).bfloat16()]
    grads = [[torch.randn_like(w) for w in ws] for _ in range(6)]
    pairs = []
    for _ in range(2):
        ps = [torch.nn.Parameter(w.clone()) for w in ws]
        for p in ps:
            p.grad = torch.zeros_like(p)
        pairs.append((ps, FusedAdamW(ps, lr=1e-2, state_bits=8)))

    def load(ps, i):
        for p, g in zip(ps, grads[i]):
            p.grad.copy_(g)

    (pa, oa), (pb, ob) = pairs
    for ps, opt in pairs:
        load(ps, 0)
        opt.step(), opt.moment_vectors()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ob.step()
        captured = ob.moment_vectors()
    held = []
    for i in range(1, 6):
        load(pa, i), load(pb, i)
        oa.step()
        graph.replay()
        torch.cuda.synchronize()
        want = oa.moment_vectors()
        assert all(torch.equal(x, y) for x, y in zip(captured, want))
        # an eager call on other state gets a table of its own and leaves the graph's as it is
        other = {k: v.clone() for k, v in ob.state[pb[0]].items() if isinstance(v, torch.Tensor)}
        own = dict(ob.state[pb[0]])
        ob.state[pb[0]].update(other)
        held.append(other)
        assert all(torch.equal(x, y) for x, y in zip(ob.moment_vectors(), want))
        ob.state[pb[0]].update(own)


def test_a_refused_step_changes_nothing():
    check_refused_step(DEV)
