"""A memory-lean fine-tuning step on a tiny Llama: LoRA on a 4-bit base, a policy objective over token log
probabilities, AdamW with 8-bit moments.  Shared by the CPU and GPU tests."""
import torch

from hyperion.models.llama import LlamaConfig, LlamaForCausalLM
from hyperion.models.lora import LoRALinear, apply_lora
from hyperion.ops import FusedAdamW
from hyperion.ops.mxfp4 import MXFP4Linear


def build(dev, dtype, seed=0):
    torch.manual_seed(seed)
    m = LlamaForCausalLM(LlamaConfig.tiny(num_key_value_heads=1)).to(dtype)
    apply_lora(m, r=8, alpha=16, dropout=0.0, base_format="mxfp4")
    for mod in m.modules():
        if isinstance(mod, LoRALinear):  # B starts at zero, which would hide A's gradient
            torch.nn.init.normal_(mod.lora_B["default"].weight, std=0.05)
    return m.to(dev)


def dequantized(m):
    """The same model with plain linear layers of the 4-bit values (fp32)."""
    ref = build("cpu", torch.float32)
    ref.load_state_dict({k: v.float().cpu() if v.is_floating_point() else v.cpu() for k, v in m.state_dict().items()})
    for mod in list(ref.modules()):
        for name, child in list(mod.named_children()):
            if isinstance(child, MXFP4Linear):
                lin = torch.nn.Linear(child.in_features, child.out_features, bias=False)
                lin.weight.data.copy_(child.weight.dequantize(torch.float32))
                lin.weight.requires_grad_(False)
                setattr(mod, name, lin)
    return ref


def batch(dev):
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(1, 512, (3, 12), generator=g)
    mask = torch.ones_like(ids)
    mask[1, 8:] = 0
    labels = ids.masked_fill(mask == 0, -100)
    advantage = torch.randn(3, 11, generator=g)
    return ids.to(dev), mask.to(dev), labels.to(dev), advantage.to(dev)


def loss_of(model, ids, mask, labels, advantage):
    out = model.token_logprobs(ids, labels, mask, top_k=3)
    n = (labels[:, 1:] != -100).sum()
    return -(advantage * out.logprobs + 0.01 * out.entropy).sum() / n, out


def reference_loss(model, ids, mask, labels, advantage):
    logits = model(ids, mask, return_logits=True).logits[:, :-1].float()
    ls = torch.log_softmax(logits, -1)
    keep = labels[:, 1:] != -100
    lp = ls.gather(-1, labels[:, 1:].clamp(min=0)[..., None])[..., 0]
    h = -(ls.exp() * ls).sum(-1)
    return -((advantage * lp + 0.01 * h) * keep).sum() / keep.sum()


def adapters(model):
    return {n: p for n, p in model.named_parameters() if p.requires_grad}


def check_step(dev, dtype, tol):
    """One step together: the loss and every adapter's gradient against the dequantised model in fp32 on the CPU."""
    m = build(dev, dtype)
    assert sum(isinstance(x, MXFP4Linear) for x in m.modules()) == 2 * 7
    ref = dequantized(m)
    ps = adapters(m)
    opt = FusedAdamW(ps.values(), lr=1e-2, state_bits=8)
    loss, out = loss_of(m, *batch(dev))
    loss.backward()
    want = reference_loss(ref, *batch("cpu"))
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= tol * (1 + abs(float(want.detach())))
    assert out.top_ids.shape == (3, 11, 3) and (out.top_ids[1, 8:] == -1).all()
    for n, p in adapters(ref).items():
        d = (ps[n].grad.float().cpu() - p.grad).norm() / p.grad.norm()
        assert d <= tol, (n, float(d))
    before = {n: p.detach().clone() for n, p in ps.items()}
    opt.step()
    assert all((p != before[n]).any() for n, p in ps.items())
    m_vec, v_vec = opt.moment_vectors()
    assert m_vec.numel() == sum(p.numel() for p in ps.values()) and torch.isfinite(m_vec).all() and (v_vec >= 0).all()
    return m, opt
