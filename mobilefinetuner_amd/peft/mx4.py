"""A LoRA model on a 4-bit frozen base.

``quantize_base`` replaces a model's frozen projection weights and its vocabulary table (embedding and tied LM
head) by ``ops.mx4.MX4Weight``: 4.25 bits a weight instead of 16 (Gemma-3 270M: 0.54 GB -> 0.14 GB of base
weights).  Adapters, norms, biases and position tables stay as they are.  The model then runs forward and
backward through ops.functional's mx4 ops, its loss through lm_head_cross_entropy_pieces.
"""
from __future__ import annotations

import torch

from ..ops import functional as Fx
from ..ops.mx4 import GROUP, MX4Weight


def is_quantized(model) -> bool:
    return isinstance(_table(model)[1], MX4Weight)


def _table(model):
    name = "wte" if hasattr(model, "wte") else "embed"
    return name, getattr(model, name)


@torch.no_grad()
def quantize_base(model) -> int:
    """Quantise the base of a GPT-2 or Gemma-3 model in place (after its weights are loaded; adapters may come
    before or after).  Returns the bytes that the base weights now take.  A trainable, sharded or partitioned
    base is refused, and so is a width that is no multiple of 32."""
    if is_quantized(model):
        raise RuntimeError("quantize_base: the base is in 4 bits already")
    if getattr(model, "sharder", None) is not None or getattr(model, "zero3", None) is not None:
        raise RuntimeError("quantize_base: not with parameter sharding or ZeRO-3: the 4-bit base is resident")
    name, table = _table(model)
    mods = model.linear_modules()
    for what, w in [(name, table)] + [(n, m.weight) for n, m in mods.items()]:
        if w.requires_grad:
            raise RuntimeError(f"quantize_base: {what} is trainable; a 4-bit base is frozen (LoRA)")
        if getattr(w, "shadow", None) is not None:
            raise RuntimeError(f"quantize_base: {what} has an fp32 master; a 4-bit base is frozen (LoRA)")
        if w.shape[1] % GROUP:
            raise RuntimeError(f"quantize_base: {what} has {w.shape[1]} inputs, not a multiple of {GROUP}")
    total = 0
    for m in mods.values():
        w4 = Fx.mx4_quantize(m.weight.data)
        Fx.drop_weight_t(m.weight)
        m.__dict__.pop("_waug", None)
        del m.weight
        m.weight = w4
        total += w4.nbytes
    w4 = Fx.mx4_quantize(table.data)
    delattr(model, name)
    setattr(model, name, w4)
    return total + w4.nbytes
