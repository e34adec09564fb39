"""4-bit frozen weights: the definition itself, the container's refusals, and host calls (no GPU)."""
import pytest
import torch

from oracle import mx4 as ref


def _fx():
    from mobilefinetuner_amd.ops import functional as Fx
    return Fx


def test_oracle_grid_and_ties():
    x = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0] * 4])
    codes, scales = ref.quantize(x)
    assert scales.item() == 127
    assert ref.values(codes, scales)[0, :8].tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0]


def test_oracle_scale_choice():
    x = torch.zeros(7, 32)
    x[:, 3] = torch.tensor([7.0, 7.0625, 4.0, 3.75, 3.5, 2.0 ** -140, 0.0])
    assert ref.quantize(x)[1].flatten().tolist() == [127, 128, 127, 127, 126, 2, 2]


def test_container():
    Fx = _fx()
    u8 = torch.uint8
    w = Fx.MX4Weight(torch.zeros(5, 48, dtype=u8), torch.zeros(5, 3, dtype=u8))
    assert w.shape == (5, 96) and w.nbytes == 5 * 51 and w.numel() == 480 and not w.requires_grad
    for codes, scales in ((torch.zeros(5, 48), torch.zeros(5, 3, dtype=u8)),
                          (torch.zeros(5, 40, dtype=u8), torch.zeros(5, 3, dtype=u8)),
                          (torch.zeros(5, 48, dtype=u8), torch.zeros(5, 4, dtype=u8)),
                          (torch.zeros(5, 48, dtype=u8), torch.zeros(4, 3, dtype=u8)),
                          (torch.zeros(5, 0, dtype=u8), torch.zeros(5, 0, dtype=u8)),
                          (torch.zeros(48, dtype=u8), torch.zeros(3, dtype=u8)),
                          (torch.zeros(48, 5, dtype=u8).t(), torch.zeros(5, 3, dtype=u8)),
                          (torch.zeros(5 * 48 + 1, dtype=u8)[1:].view(5, 48), torch.zeros(5, 3, dtype=u8))):
        with pytest.raises(ValueError, match="MX4Weight"):
            Fx.MX4Weight(codes, scales)


def test_host_calls_go_to_the_oracle():
    Fx = _fx()
    w = torch.randn(48, 64, generator=torch.Generator().manual_seed(0))
    w4 = Fx.mx4_quantize(w)
    v = ref.values(w4.codes, w4.scales)
    assert torch.equal(w4.dequantize().double(), v)
    x = torch.randn(3, 64, requires_grad=True)
    y = Fx.linear(x, w4)
    assert torch.equal(y, Fx.mx4_linear(x, w4)) and (y.double() - x.double() @ v.t()).abs().max() < 1e-4
    y.sum().backward()
    assert (x.grad.double() - v.sum(0)).abs().max() < 1e-4
    ids = torch.tensor([[1, 5], [47, 0]])
    assert torch.equal(Fx.embedding(ids, w4, None, 2.0).double(), 2.0 * v[ids.reshape(-1)])


def test_no_kernel_call_on_host_tensors():
    from mobilefinetuner_amd._ext import native
    C = native()
    u8 = torch.uint8
    codes, scales = torch.zeros(4, 16, dtype=u8), torch.zeros(4, 1, dtype=u8)
    with pytest.raises(RuntimeError, match="GPU"):
        C.mx4_linear(torch.zeros(2, 32, dtype=torch.bfloat16), codes, scales, None)
    with pytest.raises(RuntimeError, match="GPU"):
        C.mx4_dgrad(torch.zeros(2, 4, dtype=torch.bfloat16), codes, scales)
    with pytest.raises(RuntimeError, match="GPU"):
        C.mx4_dequantize(codes, scales)
    with pytest.raises(RuntimeError):
        C.mx4_quantize(torch.zeros(4, 32))
