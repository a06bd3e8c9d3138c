"""LoRA on a 4-bit base, token log probabilities and 8-bit AdamW together, on the CPU paths."""
import pytest
import torch

from hyperion.models.lora import LoRALinear, apply_lora, load_adapter, merge_lora, quantize_base, save_adapter
from hyperion.models.llama import LlamaConfig, LlamaForCausalLM
from hyperion.ops.mxfp4 import MXFP4Linear

from lean_finetune import batch, build, check_step, dequantized


def test_step_against_the_dequantised_model():
    # fp32 on both sides: sums of up to 512 terms in two orders, through two layers
    check_step("cpu", torch.float32, 1e-4)


def test_keys_adapters_and_merge(tmp_path):
    m = build("cpu", torch.float32)
    keys = set(m.state_dict())
    assert "model.layers.0.self_attn.q_proj.base_layer.weight_codes" in keys and "lm_head.weight" in keys
    assert "model.layers.0.mlp.up_proj.weight_scales" in keys
    save_adapter(m, str(tmp_path))
    plain = apply_lora(LlamaForCausalLM(LlamaConfig.tiny(num_key_value_heads=1)), r=8, alpha=16, dropout=0.0)
    load_adapter(plain, str(tmp_path))  # the adapter files are those of any base
    for a, b in zip([x for x in m.modules() if isinstance(x, LoRALinear)], [x for x in plain.modules() if isinstance(x, LoRALinear)]):
        assert torch.equal(a.lora_B["default"].weight, b.lora_B["default"].weight)
    ids, mask, _, _ = batch("cpu")
    m.eval()
    want = m(ids, mask).logits
    merged = merge_lora(m)
    assert not any(isinstance(x, LoRALinear) for x in merged.modules())
    torch.testing.assert_close(merged(ids, mask).logits, want, atol=1e-4, rtol=1e-4)


def test_dropout_and_refusals():
    m = build("cpu", torch.float32)
    layer = next(x for x in m.modules() if isinstance(x, LoRALinear))
    layer.p = 0.5
    x = torch.randn(4, 128)
    torch.manual_seed(0)
    a = layer.train()(x)
    assert not torch.equal(a, layer.eval()(x))
    with pytest.raises(ValueError):
        apply_lora(LlamaForCausalLM(LlamaConfig.tiny()), base_format="int3")
    trainable = LlamaForCausalLM(LlamaConfig.tiny())
    assert not any(isinstance(x, MXFP4Linear) for x in quantize_base(trainable).modules())
    assert dequantized(m) is not m


def test_quantised_first_and_other_models():
    m = LlamaForCausalLM(LlamaConfig.tiny(num_key_value_heads=1)).bfloat16()
    for p in m.parameters():
        p.requires_grad_(False)
    apply_lora(quantize_base(m), r=4)
    layers = [x for x in m.modules() if isinstance(x, LoRALinear)]
    assert len(layers) == 8 and all(isinstance(x.base_layer, MXFP4Linear) for x in layers)
    assert all(x.lora_A["default"].weight.dtype == torch.bfloat16 for x in layers)
    from hyperion.models.transformer import create_custom_transformer

    torch.manual_seed(0)
    t = create_custom_transformer().eval()
    for p in t.parameters():
        p.requires_grad_(False)
    x = torch.randn(2, 5, 512)
    before = t(x)
    n = sum(isinstance(c, MXFP4Linear) for c in quantize_base(t).modules())
    assert n > 0 and t(x).shape == before.shape and torch.isfinite(t(x)).all()


def test_trainer_with_a_4_bit_base(tmp_path):
    from hyperion.train.distributed import train_llama_fsdp
    from test_trainers_cpu import _opts

    r = train_llama_fsdp(0, 1, epochs=1, base_dir=str(tmp_path), lora=True, batch_size=2, progress_every=0, opts=_opts(),
                         config=LlamaConfig.tiny(num_hidden_layers=1), base_format="mxfp4", state_bits=8)
    assert r["history"][0]["steps"] == 2 and r["mode"].endswith("mxfp4")
    with pytest.raises(ValueError, match="base_format"):
        train_llama_fsdp(0, 1, base_dir=str(tmp_path), lora=False, base_format="mxfp4")


def test_forward_mode_on_the_cpu_paths():
    from torch.autograd import forward_ad as fw

    from hyperion.ops.mxfp4 import mxfp4_linear, quantize_mxfp4
    from hyperion.ops.token_logprobs import token_logprobs

    torch.manual_seed(4)
    w, x, dx = quantize_mxfp4(torch.randn(16, 64)), torch.randn(3, 64), torch.randn(3, 64)
    t = torch.tensor([1, 2, 63])
    with fw.dual_level():
        d = fw.make_dual(x, dx)
        y = fw.unpack_dual(mxfp4_linear(d, w)).tangent
        torch.testing.assert_close(y, dx @ w.dequantize(torch.float32).t(), atol=1e-5, rtol=1e-5)
        lp = fw.unpack_dual(token_logprobs(d, t).logprobs).tangent
    want = (dx.gather(1, t[:, None])[:, 0] - (torch.softmax(x, 1) * dx).sum(1))
    torch.testing.assert_close(lp, want, atol=1e-5, rtol=1e-5)


def test_quantised_layers_keep_their_places_and_hooks():
    class Two(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.a = torch.nn.Linear(64, 64)
            self.b = self.a
            self.rest = torch.nn.ModuleList([self.a, torch.nn.Linear(64, 8)])
            self.normed = torch.nn.utils.weight_norm(torch.nn.Linear(8, 8))

        def forward(self, x):
            return self.normed(self.rest[1](self.rest[0](self.b(self.a(x)))))

    m = Two().eval()
    for p in m.parameters():
        p.requires_grad_(False)
    seen = []
    handles = [m.a.register_forward_pre_hook(lambda mod, args, kwargs: seen.append("pre"), with_kwargs=True),
               m.a.register_forward_hook(lambda mod, args, y: y + 1.0),
               m.a.register_full_backward_hook(lambda mod, gi, go: seen.append("grad"))]
    normed = m.normed
    quantize_base(m)
    assert isinstance(m.a, MXFP4Linear) and m.b is m.a and m.rest[0] is m.a and isinstance(m.rest[1], MXFP4Linear)
    assert m.normed is normed and not m.a.training
    x = torch.randn(3, 64, requires_grad=True)
    w = m.a.weight.dequantize(torch.float32)
    torch.testing.assert_close(m.a(x), x @ w.t() + m.a.bias + 1.0, atol=1e-5, rtol=1e-5)
    m(x).sum().backward()
    assert seen.count("pre") == 4 and seen.count("grad") == 3
    for h in handles:
        h.remove()
    torch.testing.assert_close(m.a(x), x @ w.t() + m.a.bias, atol=1e-5, rtol=1e-5)
    assert seen.count("pre") == 4


def test_merged_layers_are_the_frameworks_own():
    from hyperion.ops.linear import Linear

    m = build("cpu", torch.float32).eval()
    base = m.model.layers[0].self_attn.q_proj.base_layer
    calls = []
    handle = base.register_forward_hook(lambda mod, args, y: calls.append(mod))
    kinds = {n: type(x) for n, x in LlamaForCausalLM(LlamaConfig.tiny()).named_modules() if n.endswith("_proj")}
    merge_lora(m)
    for n, x in m.named_modules():
        if n.endswith(("q_proj", "k_proj", "v_proj", "o_proj")):
            assert type(x) is kinds[n] is Linear and not x.training and not x.weight.requires_grad, n
    ids, mask, _, _ = batch("cpu")
    m(ids, mask)
    assert calls == [m.model.layers[0].self_attn.q_proj]
    handle.remove()
    m(ids, mask)
    assert len(calls) == 1


def check_one_rounding(dev, dtype):
    torch.manual_seed(6)
    layer = LoRALinear(MXFP4Linear.from_linear(torch.nn.Linear(96, 64, device=dev)), r=7, alpha=12, dropout=0.0, dtype=dtype).eval()
    torch.nn.init.normal_(layer.lora_B["default"].weight)
    x = torch.randn(50, 96, device=dev).to(dtype).requires_grad_(True)
    y = layer(x)
    with torch.no_grad():
        base = layer.base_layer(x)
        u = layer.lora_B["default"](layer.lora_A["default"](x)) if dev == "cpu" else None
        if u is None:
            from hyperion.ops.linear import linear

            u = linear(linear(x, layer.lora_A["default"].weight), layer.lora_B["default"].weight)
    want = base.double() + 12 / 7 * u.double()
    # one rounding to dtype, and two of fp32 (the scaling and the sum) of at most |base| + 12 / 7 |u|
    bound = torch.finfo(dtype).eps / 2 * want.abs() * (1 + 1e-6) + 2.0 ** -22 * (base.double().abs() + 2 * u.double().abs())
    assert y.dtype == dtype and bool(((y.detach().double() - want).abs() <= bound).all())
    dy = torch.randn(50, 64, device=dev).to(dtype)
    gb, = torch.autograd.grad(y, layer.lora_B["default"].weight, dy)
    want = (12 / 7 * dy.double()).t() @ layer.lora_A["default"](x).detach().double()
    # dy scaled and rounded, the product's operand and result rounded
    scale = (12 / 7 * dy.double()).abs().t() @ layer.lora_A["default"](x).detach().double().abs()
    assert bool(((gb.double() - want).abs() <= 4 * torch.finfo(dtype).eps * scale).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_adapter_is_added_with_one_rounding(dtype):
    check_one_rounding("cpu", dtype)


def _ddp_on_a_4_bit_base(rank, world):
    from hyperion.parallel import DDP, ddp

    m = build("cpu", torch.float32, seed=rank)
    m.register_buffer("running", torch.full((3,), float(rank)))
    sent = []
    flat_broadcast = ddp._flat_broadcast

    def spy(ts, *args):
        sent.append(sum(t.numel() * t.element_size() for t in ts))
        flat_broadcast(ts, *args)

    ddp._flat_broadcast = spy
    d = DDP(m)
    ids, mask, _, _ = batch("cpu")
    m.running += rank
    first = d(ids, mask, return_logits=True).logits
    second = d(ids.flip(1), mask, return_logits=True).logits  # before the first one's backward
    with d.no_sync():
        first.square().mean().backward()
    second.square().mean().backward()
    codes = [b.clone() for n, b in m.named_buffers() if n.endswith(("weight_codes", "weight_scales"))]
    return {"sent": sent, "codes": codes, "running": m.running.clone(),
            "grads": [p.grad.clone() for p in m.parameters() if p.grad is not None]}


def test_ddp_broadcasts_a_4_bit_base_once():
    from dist_utils import run_world

    res = run_world(_ddp_on_a_4_bit_base, 2)
    a, b = res[0], res[1]
    whole = sum(c.numel() for c in a["codes"])
    assert len(a["codes"]) == 2 * 14 and all(torch.equal(x, y) for x, y in zip(a["codes"], b["codes"]))
    assert a["sent"][0] > whole and a["sent"][1:] == [12, 12]  # then the running statistics alone
    assert torch.equal(a["running"], torch.zeros(3)) and torch.equal(b["running"], torch.zeros(3))
    assert len(a["grads"]) > 0 and all(torch.equal(x, y) for x, y in zip(a["grads"], b["grads"]))


def check_no_rows(dev, dtype, lead):
    layer = LoRALinear(MXFP4Linear.from_linear(torch.nn.Linear(128, 64, device=dev)), r=8, dropout=0.1, dtype=dtype).train()
    x = torch.zeros(*lead, 128, device=dev, dtype=dtype, requires_grad=True)
    y = layer(x)
    assert y.shape == (*lead, 64) and y.dtype == dtype
    grads = torch.autograd.grad(y.sum(), [x, layer.lora_A["default"].weight, layer.lora_B["default"].weight])
    assert grads[0].shape == x.shape and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("lead", [(0,), (2, 0)])
def test_a_layer_without_rows(lead):
    check_no_rows("cpu", torch.float32, lead)
