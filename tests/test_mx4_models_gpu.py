"""LoRA models on a 4-bit base: quantise, look up, multiply, attend, and the loss in pieces, run together on the GPU."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def _build(kind, dtype, device, seed=3):
    from mobilefinetuner_amd.models.gemma3 import Gemma3Config, Gemma3Model
    from mobilefinetuner_amd.models.gpt2 import GPT2Config, GPT2Model
    if kind == "gpt2":
        return GPT2Model(GPT2Config.preset("gpt2-tiny"), dtype=dtype, device=device, seed=seed)
    return Gemma3Model(Gemma3Config.preset("gemma3-tiny"), dtype=dtype, device=device, seed=seed)


def _inject(m, kind):
    from mobilefinetuner_amd.peft.lora import LoraSpec, inject_gemma, inject_gpt2
    if kind == "gpt2":
        inject_gpt2(m, LoraSpec(rank=8, alpha=16, targets=["AttnQKV", "AttnProj", "MlpFcIn", "MlpFcOut"]))
    else:
        inject_gemma(m, LoraSpec(rank=8, alpha=16, init="peft", targets=["q_proj", "v_proj", "o_proj", "gate_proj", "down_proj"]))
    with torch.no_grad():
        for mod in m.modules():
            for sl in getattr(mod, "lora_slices", []):
                sl.B.copy_(torch.randn(sl.B.shape, generator=torch.Generator().manual_seed(sl.ncols)) * 0.05)


def _values_in_place(m, kind):
    """The base weights rounded to the 4-bit grid, kept in the model's own type."""
    with torch.no_grad():
        ws = [lin.weight for lin in m.linear_modules().values()] + [m.wte if kind == "gpt2" else m.embed]
        for w in ws:
            w.copy_(ref.values(*ref.quantize(w.data)).to(w.dtype))


@pytest.mark.parametrize("kind", ["gpt2", "gemma"])
def test_training_step_matches_dense_model_of_the_same_values(kind):
    """fp32 on the host with the 4-bit values is the truth; the dense bf16 model with the same values and the 4-bit model
    both round activations to bf16 in the same places, the 4-bit one once more per adapter (the base product, then the
    adapter's update) -- at most twice as many roundings."""
    from mobilefinetuner_amd.peft.lora import lora_parameters
    from mobilefinetuner_amd.peft.mx4 import quantize_base
    from mobilefinetuner_amd.utils.params import FlatParams
    ids = torch.randint(0, 900, (4, 65), generator=torch.Generator().manual_seed(5))
    out = {}
    for name in ("host", "dense", "mx4"):
        m = _build(kind, torch.float32 if name == "host" else torch.bfloat16, "cpu" if name == "host" else DEV)
        if name == "host":  # the bf16 models' weights are rounded to bf16 before they are quantised
            with torch.no_grad():
                for p in m.parameters():
                    if p.dim() == 2:
                        p.copy_(p.bfloat16().float())
        if name != "mx4":
            _values_in_place(m, kind)
        _inject(m, kind)
        if name == "mx4":
            quantize_base(m)
        flat = FlatParams(lora_parameters(m), "cpu" if name == "host" else DEV, shadow=name != "host")
        dev = "cpu" if name == "host" else DEV
        loss = m(ids[:, :-1].to(dev), ids[:, 1:].to(dev))
        loss.backward()
        out[name] = (loss.item(), flat.grad.cpu().double())
    truth, g = out["host"]
    err = {n: ((out[n][1] - g).norm() / g.norm()).item() for n in ("dense", "mx4")}
    assert abs(out["mx4"][0] - truth) <= 2 * abs(out["dense"][0] - truth) + 2.0 ** -10 * truth, out
    assert err["mx4"] <= 2 * err["dense"] + 2.0 ** -8, err


@pytest.mark.parametrize("kind", ["gpt2", "gemma"])
def test_evaluation_matches_dense_model(kind):
    from mobilefinetuner_amd.peft.mx4 import quantize_base
    a, b = _build(kind, torch.bfloat16, DEV), _build(kind, torch.bfloat16, DEV)
    _values_in_place(b, kind)
    quantize_base(a)
    ids = torch.randint(0, 900, (3, 40), generator=torch.Generator().manual_seed(6)).to(DEV)
    with torch.no_grad():
        (sa, na), (sb, nb) = a.nll(ids[:, :-1], ids[:, 1:]), b.nll(ids[:, :-1], ids[:, 1:])
        la, lb = a.logits(ids).float(), b.logits(ids).float()
    # the same exact weights; hidden states differ by bf16 roundings of sums in another order (2^-8 each, a dozen layers' worth)
    assert na.item() == nb.item() and abs(sa.item() - sb.item()) <= 2.0 ** -8 * sb.item()
    assert ((la - lb).norm() / lb.norm()).item() <= 12 * 2.0 ** -8


def test_captured_training_steps():
    """The training engine captures the 4-bit step into a graph; its losses follow the eager steps' (the same kernels; the
    adapters' gradients are summed by fp32 atomics, so later steps may differ in their last bits)."""
    from mobilefinetuner_amd.optim.adamw import FusedAdamW
    from mobilefinetuner_amd.peft.lora import lora_parameters
    from mobilefinetuner_amd.peft.mx4 import quantize_base
    from mobilefinetuner_amd.train.engine import TrainStep
    from mobilefinetuner_amd.utils.params import FlatParams
    losses = {}
    ids = torch.randint(0, 900, (4, 65), generator=torch.Generator().manual_seed(7)).to(DEV)
    for graph in (False, True):
        m = _build("gpt2", torch.bfloat16, DEV)
        _inject(m, "gpt2")
        quantize_base(m)
        flat = FlatParams(lora_parameters(m), DEV)
        opt = FusedAdamW(flat, lr=1e-3)
        step = TrainStep(m, flat, opt, use_graph=graph)
        losses[graph] = [float(step([(ids[:, :-1].contiguous(), ids[:, 1:].contiguous())]).item()) for _ in range(6)]
    assert losses[True][0] == losses[False][0]
    assert all(abs(a - b) <= 2.0 ** -8 * b for a, b in zip(losses[True], losses[False])), losses
