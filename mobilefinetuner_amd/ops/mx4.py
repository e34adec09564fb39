"""Frozen weights in 4 bits.

``MX4Weight`` holds a matrix W [N, K] as e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two
per byte with the even column in the low half, and one power-of-two scale per 32 columns of a row
(2 ** (byte - 127); byte 255 reads as NaN): 4.25 bits a weight.  Sign, 1-bit mantissa and a power-of-two
scale make every weight exact in bf16, so products with it round nothing but their result.  ``mx4_quantize``
writes bytes 2 to 252; in weights made elsewhere bytes 0 and 1 give denormal bf16 numbers, exact as well, and
under bytes 253 and 254 a number past bf16's largest one reads as an infinity.

It stands where a frozen weight tensor stands: ``Linear.weight``, a model's vocabulary table, and the
``w`` of ``ops.functional``'s linear, LoRA, embedding and LM-head loss ops.
"""
from __future__ import annotations

import torch

GROUP = 32


class MX4Weight:
    __slots__ = ("codes", "scales", "shape")

    requires_grad = False        # a frozen weight: no gradient, no fp32 master, no shadow
    dtype = torch.bfloat16       # of its values, and of the activations it multiplies
    grad = None

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError(f"MX4Weight: codes [N, K / 2] and scales [N, K / 32] are 2-D uint8 tensors, got "
                             f"{codes.dtype} {tuple(codes.shape)} and {scales.dtype} {tuple(scales.shape)}")
        n, half = codes.shape
        if half % 16 or half == 0 or scales.shape != (n, half // 16):
            raise ValueError(f"MX4Weight: codes [N, K / 2] with K a multiple of {GROUP} and scales [N, K / 32], got "
                             f"{tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"MX4Weight: codes on {codes.device}, scales on {scales.device}")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.data_ptr() % 16:
            raise ValueError("MX4Weight: codes and scales are contiguous, codes at a 16-byte boundary")
        self.codes, self.scales, self.shape = codes, scales, torch.Size((n, 2 * half))

    @property
    def device(self):
        return self.codes.device

    @property
    def is_cuda(self):
        return self.codes.is_cuda

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def numel(self):
        return self.shape[0] * self.shape[1]

    def dim(self):
        return 2

    def to(self, device):
        return MX4Weight(self.codes.to(device), self.scales.to(device))

    def dequantize(self) -> torch.Tensor:
        """The values, bf16 [N, K]."""
        from .functional import mx4_dequantize
        return mx4_dequantize(self.codes, self.scales)

    def __repr__(self):
        return f"MX4Weight({self.shape[0]} x {self.shape[1]}, {self.device})"
