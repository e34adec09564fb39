"""LoRA models on a 4-bit base (peft.mx4.quantize_base): wiring, refusals and CLIs on host tensors (oracle ops)."""
import os

import pytest
import torch

CPU = ["--device", "cpu", "--dtype", "fp32", "--random_init", "--synthetic_data", "--synthetic_tokens", "20000"]


def _model(kind, quantize=True, lora=True):
    from mobilefinetuner_amd.peft.lora import LoraSpec, inject_gemma, inject_gpt2
    from mobilefinetuner_amd.peft.mx4 import quantize_base
    if kind == "gpt2":
        from mobilefinetuner_amd.models.gpt2 import GPT2Config, GPT2Model
        m = GPT2Model(GPT2Config.preset("gpt2-tiny"), dtype=torch.float32, device="cpu", seed=1)
        if lora:
            inject_gpt2(m, LoraSpec(rank=8, alpha=16))
    else:
        from mobilefinetuner_amd.models.gemma3 import Gemma3Config, Gemma3Model
        m = Gemma3Model(Gemma3Config.preset("gemma3-tiny"), dtype=torch.float32, device="cpu", seed=1)
        if lora:
            inject_gemma(m, LoraSpec(rank=8, alpha=16, targets=["q_proj", "down_proj"], init="peft"))
    if quantize:
        quantize_base(m)
    return m


@pytest.mark.parametrize("kind", ["gpt2", "gemma"])
def test_quantized_model_equals_its_values(kind):
    """Every base weight is the MX4Weight of the original one, and the model computes with its values: close to the fp32
    model that holds them (the lookup's bf16 rounding and the bf16 that follows it on the host, 2^-8 a rounding)."""
    from mobilefinetuner_amd.models.layers import mx4_weights
    from mobilefinetuner_amd.ops import functional as Fx
    a, b = _model(kind), _model(kind, quantize=False)
    assert len(mx4_weights(a)) == len(a.linear_modules()) + 1
    assert a.num_parameters() == b.num_parameters()
    name = "wte" if kind == "gpt2" else "embed"
    with torch.no_grad():
        for (n, la), (_, lb) in zip(a.linear_modules().items(), b.linear_modules().items()):
            want = Fx.mx4_quantize(lb.weight.data)
            assert torch.equal(la.weight.codes, want.codes) and torch.equal(la.weight.scales, want.scales), n
            lb.weight.copy_(want.dequantize())
        getattr(b, name).copy_(Fx.mx4_quantize(getattr(b, name).data).dequantize())
    ids = torch.randint(0, 500, (2, 33), generator=torch.Generator().manual_seed(0))
    la, lb = a(ids[:, :-1], ids[:, 1:]), b(ids[:, :-1], ids[:, 1:])
    assert abs(la.item() - lb.item()) < 2.0 ** -7 * lb.item()
    la.backward()
    assert all(p.grad is not None for p in a.parameters() if p.requires_grad)
    with torch.no_grad():
        assert a.logits(ids[:, :4]).shape == b.logits(ids[:, :4]).shape
        s, n = a.nll(ids[:, :-1], ids[:, 1:])
        assert n.item() == 64 and abs(s.item() / 64 - la.item()) < 1e-4


def test_refusals():
    from mobilefinetuner_amd.models import hf_io
    from mobilefinetuner_amd.parallel.sharder import shard_gpt2
    from mobilefinetuner_amd.peft.lora import merge_all
    from mobilefinetuner_amd.peft.mx4 import is_quantized, quantize_base
    m = _model("gpt2")
    assert is_quantized(m)
    with pytest.raises(RuntimeError, match="already"):
        quantize_base(m)
    with pytest.raises(RuntimeError, match="4-bit base"):
        merge_all(m)
    with pytest.raises(RuntimeError, match="4-bit base"):
        m.set_full_finetune()
    with pytest.raises(RuntimeError, match="4-bit base"):
        hf_io.export_gpt2_state(m)
    with pytest.raises(RuntimeError, match="4-bit base"):
        hf_io.load_gpt2_state(m, {})
    with pytest.raises(RuntimeError, match="4-bit base"):
        shard_gpt2(m, 1 << 20)
    full = _model("gpt2", quantize=False, lora=False)
    full.set_full_finetune()
    with pytest.raises(RuntimeError, match="trainable"):
        quantize_base(full)


def test_clis(tmp_path):
    from mobilefinetuner_amd.cli import eval_ppl, gpt2_lora_finetune, train_lora_gemma
    out = str(tmp_path / "lora.safetensors")
    tr = gpt2_lora_finetune.main(["--model", "gpt2-tiny", *CPU, "--base_mx4", "--steps", "3", "--batch_size", "2",
                                  "--seq_len", "32", "--lora_out", out, "--eval_interval", "3", "--eval_batches", "1"])
    assert len(tr.history) == 3 and os.path.exists(out)
    tr = train_lora_gemma.main(["--model", "gemma3-tiny", *CPU, "--base_mx4", "--max_steps", "2", "--batch", "2",
                                "--seq_len", "32", "--output_dir", str(tmp_path), "--targets", "full"])
    assert len(tr.history) == 2
    eval_ppl.main(["--model", "gpt2-tiny", *CPU, "--base_mx4", "--seq_len", "32", "--max_batches", "2", "--lora_path", out])


@pytest.mark.parametrize("kind", ["gpt2", "gemma"])
def test_state_dict_holds_the_4_bit_base(kind):
    from mobilefinetuner_amd.models.layers import mx4_weights
    a, b = _model(kind), _model(kind)
    for w in mx4_weights(b):
        w.codes.fill_(0x11), w.scales.fill_(100)
    sd = a.state_dict()
    assert sum(k.endswith("_codes") for k in sd) == sum(k.endswith("_scales") for k in sd) == len(mx4_weights(a))
    b.load_state_dict(sd)
    for wa, wb in zip(mx4_weights(a), mx4_weights(b)):
        assert torch.equal(wa.codes, wb.codes) and torch.equal(wa.scales, wb.scales)
    name = ("wte" if kind == "gpt2" else "embed") + "_codes"
    with pytest.raises(RuntimeError, match="Missing key"):
        b.load_state_dict({k: v for k, v in sd.items() if k != name})
    with pytest.raises(RuntimeError, match=f"{name}: "):
        b.load_state_dict({**sd, name: sd[name][1:]})
    with pytest.raises(RuntimeError, match="Unexpected key"):
        _model(kind, quantize=False).load_state_dict(sd)


@pytest.mark.parametrize("kind", ["gpt2", "gemma"])
def test_the_4_bit_base_moves_with_its_model(kind):
    from mobilefinetuner_amd.models.layers import mx4_weights
    m = _model(kind)
    before = [(w.codes.clone(), w.scales.clone()) for w in mx4_weights(m)]
    m.double()  # a change of type is the parameters' alone
    assert all(torch.equal(w.codes, c) and torch.equal(w.scales, s) for w, (c, s) in zip(mx4_weights(m), before))
    m.to("meta")
    assert len(mx4_weights(m)) == len(before) and all(w.device.type == "meta" for w in mx4_weights(m))


@pytest.mark.parametrize("cli", ["eval_ppl", "eval_mmlu"])
def test_evaluation_says_that_a_4_bit_base_is_not_merged(cli, capsys):
    import importlib
    from mobilefinetuner_amd.cli import common
    parser = importlib.import_module(f"mobilefinetuner_amd.cli.{cli}").build_parser()
    need = ["--mmlu_root", "x"] if cli == "eval_mmlu" else []
    assert not common.merge_adapter(parser.parse_args([*need, "--base_mx4"]))
    assert "--lora_merge does not apply with --base_mx4" in capsys.readouterr().out
    assert common.merge_adapter(parser.parse_args(need))
    assert not common.merge_adapter(parser.parse_args([*need, "--base_mx4", "--lora_merge", "0"]))
    assert capsys.readouterr().out == ""


@pytest.mark.parametrize("kind", ["gpt2", "gemma"])
def test_zero3_refuses_a_4_bit_base(kind):
    from mobilefinetuner_amd.parallel.zero3 import attach_zero3
    with pytest.raises(RuntimeError, match="ZeRO-3: not on a 4-bit base"):
        attach_zero3(_model(kind), torch.device("cpu"))
