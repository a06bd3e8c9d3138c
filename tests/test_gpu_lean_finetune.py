"""LoRA on a 4-bit base, token log probabilities and 8-bit AdamW together, on the kernels."""
import pytest
import torch

from hyperion.ops import _native

from lean_finetune import adapters, batch, build, check_step, loss_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-4), (torch.bfloat16, 0.06)])
def test_step_against_the_dequantised_model(dtype, tol):
    # bf16: about 10 roundings of 2^-8 in a row through two layers, against fp32 throughout
    _native.reset_counters()
    check_step("cuda", dtype, tol)
    n = _native.counters()
    # the first layer's q, k and v read what no adapter precedes: they need no data gradient
    assert n["mxfp4_linear"] == 14 and n["mxfp4_dgrad"] == 14 - 3 and n["token_logprobs"] == 1 and n["adam8"] >= 1


def test_captured_step_follows_the_eager_one():
    from hyperion.ops import FusedAdamW

    runs = []
    for _ in range(2):
        m = build("cuda", torch.bfloat16)
        ps = list(adapters(m).values())
        for p in ps:
            p.grad = torch.zeros_like(p)
        runs.append((m, ps, FusedAdamW(ps, lr=1e-2, state_bits=8)))
    data = batch("cuda")

    def step(m, ps, opt):
        for p in ps:
            p.grad.zero_()
        loss, _ = loss_of(m, *data)
        loss.backward()
        opt.step()
        return loss.detach()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for r in runs:
            for _ in range(2):
                step(*r)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*runs[1])
    for _ in range(4):
        want = step(*runs[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)
        assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


def test_trainer_graphed_and_eager_agree(tmp_path):
    from hyperion.models.llama import LlamaConfig
    from hyperion.train.distributed import RunOptions, train_llama_fsdp

    losses = []
    for graph in (False, True):
        opts = RunOptions(dataset_size=64, max_steps_per_epoch=6, num_workers=0, log=lambda s: None, graph=graph, save=False)
        r = train_llama_fsdp(0, 1, epochs=1, base_dir=str(tmp_path / str(graph)), lora=True, batch_size=2, progress_every=0,
                             opts=opts, config=LlamaConfig.tiny(num_hidden_layers=1), base_format="mxfp4", state_bits=8)
        losses.append(r["history"][0]["loss"])
    # the dropout streams differ between the two; the losses are those of six small steps from one start
    assert abs(losses[0] - losses[1]) < 0.05 * losses[0]


def test_forward_mode_is_refused_not_lost():
    from torch.autograd import forward_ad as fw

    from hyperion.ops.layernorm import layer_norm
    from hyperion.ops.mxfp4 import mxfp4_linear, quantize_mxfp4
    from hyperion.ops.token_logprobs import token_logprobs

    w = quantize_mxfp4(torch.randn(16, 64, device="cuda"))
    x, b = torch.randn(3, 64, device="cuda"), torch.randn(16, device="cuda")
    scale = torch.ones(64, device="cuda")
    t = torch.zeros(3, dtype=torch.long, device="cuda")
    calls = [lambda d: mxfp4_linear(d, w, b), lambda d: mxfp4_linear(x, w, d[0, :16]), lambda d: token_logprobs(d, t)]
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        for call in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call(d)
        with torch.no_grad(), pytest.raises(NotImplementedError):
            layer_norm(d.bfloat16(), scale.bfloat16(), scale.bfloat16(), 1e-5)
        assert torch.equal(mxfp4_linear(x, w, b), mxfp4_linear(d.detach().clone(), w, b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapter_is_added_with_one_rounding(dtype):
    from test_lean_finetune_cpu import check_one_rounding

    check_one_rounding("cuda", dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lead", [(0,), (2, 0)])
def test_a_layer_without_rows(lead, dtype):
    from test_lean_finetune_cpu import check_no_rows

    check_no_rows("cuda", dtype, lead)


def test_scores_of_single_tokens():
    m = build("cuda", torch.bfloat16)
    ids = torch.tensor([[3], [5]], device="cuda")
    out = m.token_logprobs(ids, ids, top_k=2)  # nothing precedes them
    assert out.logprobs.shape == (2, 0) and out.top_ids.shape == (2, 0, 2)
