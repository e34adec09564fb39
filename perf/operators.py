"""The 4-bit frozen-base operators and the vocabulary-piece loss: cases, inputs, plain forms, exact values.

A 4-bit weight W [N, K] is held as two tensors: ``codes`` uint8 [N, K / 2] (two e2m1 numbers a byte, the
even column in the low half) and ``scales`` uint8 [N, K / 32] (2 ** (byte - 127) for 32 neighbouring
columns of a row).  e2m1 holds 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives.
"""
import math

import torch

own = False

GROUP = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------- cases
def listed():
    return [
        # a 4-bit base is made once when a model is loaded: one projection of the 124M model ...
        {"name": "quantize 2304x768", "op": "quantize", "n": 2304, "k": 768, "dtype": "bf16"},
        # ... and the vocabulary table of the 270M model, from an fp32 checkpoint
        {"name": "quantize 262144x640", "op": "quantize", "n": 262144, "k": 640, "dtype": "f32"},
        # one token through a projection with its bias: the call's latency
        {"name": "linear 1 row", "op": "linear", "m": 1, "n": 2304, "k": 768, "bias": True},
        # the next-token logits of one answer choice each over the whole vocabulary of the 1B model
        {"name": "linear 4 rows to vocabulary", "op": "linear", "m": 4, "n": 262144, "k": 1152, "bias": False},
        # a ragged handful of rows (last positions of an evaluation batch) through a long reduction
        {"name": "linear 37 rows", "op": "linear", "m": 37, "n": 1152, "k": 6912, "bias": False},
        # a training step's two directions: the micro-batch of 4 x 128 tokens through the fused q|k|v of the 124M model
        {"name": "linear step 512 rows", "op": "linear_step", "m": 512, "n": 2304, "k": 768, "bias": True},
        # a ragged batch through the 1.5B model's projection
        {"name": "linear step 1999 rows", "op": "linear_step", "m": 1999, "n": 6400, "k": 1600, "bias": True},
        # 128 x 256 tokens through gate|up of the 1B model: the largest product of its step
        {"name": "linear step 32768 rows", "op": "linear_step", "m": 32768, "n": 13824, "k": 1152, "bias": False},
        # token + position lookup of a micro-batch
        {"name": "embedding 4x128", "op": "embedding", "b": 4, "s": 128, "v": 50257, "c": 768, "scale": 1.0, "pos": True},
        # scaled lookup of a whole step's tokens
        {"name": "embedding 256x256", "op": "embedding", "b": 256, "s": 256, "v": 262144, "c": 640, "scale": 25.25, "pos": False},
        # the loss of a micro-batch against a dense table with an odd number of rows
        {"name": "loss 512 rows dense", "op": "loss", "m": 512, "v": 50257, "c": 768, "table": "bf16"},
        # the loss of 64 x 256 tokens against the 4-bit table of the 270M model
        {"name": "loss 16384 rows 4-bit", "op": "loss", "m": 16384, "v": 262144, "c": 640, "table": "mx4"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear_step", "linear_step", "embedding", "loss", "loss"])
    k = GROUP * _log(rng, 2, 216)
    if op == "quantize":
        return {"op": op, "n": _log(rng, 1, 167_000_000 // k), "k": k, "dtype": rng.choice(["bf16", "f32"])}
    if op == "linear":
        n = _log(rng, 16, min(262144, 302_000_000 // k))
        return {"op": op, "m": _log(rng, 1, 256), "n": n, "k": k, "bias": rng.random() < 0.5}
    if op == "linear_step":
        n = _log(rng, 64, min(13824, 15_900_000 // k))
        return {"op": op, "m": _log(rng, 64, min(32768, 520_000_000_000 // (n * k))), "n": n, "k": k, "bias": rng.random() < 0.5}
    if op == "embedding":
        c = GROUP * _log(rng, 2, 50)
        pos = rng.random() < 0.5
        return {"op": op, "b": _log(rng, 1, 256), "s": _log(rng, 1, 256), "v": _log(rng, 256, 104_000_000 // c), "c": c,
                "scale": round(rng.uniform(0.5, 40.0), 3), "pos": pos}
    c = GROUP * _log(rng, 4, 50)
    v = _log(rng, 1000, min(262144, 167_000_000 // c))
    return {"op": op, "m": _log(rng, 1, min(16384, 2_700_000_000_000 // (v * c))), "v": v, "c": c,
            "table": rng.choice(["bf16", "mx4"])}


# ---------------------------------------------------------------- 4-bit weights, plainly
def _quantize(w):
    """(codes, scales) of w: per 32 columns a power of two under which the largest value lies in [3.5, 7]
    (over 6 saturates: off by at most 1, half a step at that size), then nearest e2m1, ties to even."""
    n, k = w.shape
    x = w.float().view(n, k // GROUP, GROUP)
    bits = x.abs().amax(-1).view(torch.int32)
    byte = (bits >> 23) - 2 + ((bits & 0x7FFFFF) > 0x600000).int()
    byte = byte.clamp(2, 252)
    x = x * ((254 - byte) << 23).view(torch.float32).unsqueeze(-1)
    a = x.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = (torch.round(a / step) * step).clamp(max=6.0)
    # 0, .5, 1, 1.5, 2, 3, 4, 6 -> 0 .. 7
    code = torch.where(q < 2, q * 2, torch.where(q < 4, q + 2, q / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(x).to(torch.uint8) << 3)).view(n, k)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte.to(torch.uint8)


def _values(codes, scales, dtype):
    n, half = codes.shape
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=dtype, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).view(n, half * 2 // GROUP, GROUP)
    return (grid[c.int()] * torch.exp2(scales.to(dtype) - 127.0).unsqueeze(-1)).view(n, half * 2)


def _loss(h, w, labels, vdim):
    """Mean NLL over the rows whose label is not -100, and its gradient for h; h, w in the wanted precision."""
    valid = labels >= 0
    at = labels.clamp(min=0).unsqueeze(1)
    logits = torch.mm(h, w.t())
    top = logits.amax(1, keepdim=True)
    picked = logits.gather(1, at)
    logits.sub_(top).exp_()
    total = logits.sum(1, keepdim=True)
    share = valid.to(h.dtype) / valid.sum().clamp(min=1)
    loss = ((top + total.log() - picked).squeeze(1) * share).sum()
    logits.div_(total)
    logits.scatter_add_(1, at, torch.full_like(picked, -1.0))
    dh = torch.mm(logits, w) * share.unsqueeze(1)
    return loss, dh


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _weight(g, n, k, std):
    """Trained weights: normal, with some input columns several times larger than the others."""
    w = _randn(g, n, k) * std
    return w * torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 6.0, 1.0)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = {"case": case}
    if op == "quantize":
        w = _weight(g, case["n"], case["k"], 0.02)
        s["w"] = w if case["dtype"] == "f32" else w.bfloat16()
    elif op in ("linear", "linear_step"):
        m, n, k = case["m"], case["n"], case["k"]
        s["codes"], s["scales"] = _quantize(_weight(g, n, k, k ** -0.5))
        s["x"] = _randn(g, m, k).bfloat16()
        s["bias"] = (_randn(g, n) * 0.1).bfloat16() if case["bias"] else None
        if op == "linear_step":
            s["x"].requires_grad_(True)
            s["dy"] = (_randn(g, m, n) / m).bfloat16()
    elif op == "embedding":
        s["codes"], s["scales"] = _quantize(_weight(g, case["v"], case["c"], 0.02))
        # token ranks of text: few ids make up most of it
        u = torch.rand(case["b"], case["s"], device="cuda", generator=g, dtype=torch.float64)
        s["ids"] = (torch.exp(u * math.log(case["v"])) - 1).long().clamp(0, case["v"] - 1)
        s["wpe"] = (_randn(g, max(case["s"], 128), case["c"]) * 0.02).bfloat16() if case["pos"] else None
    else:
        m, v, c = case["m"], case["v"], case["c"]
        w = _weight(g, v, c, c ** -0.5)
        labels = torch.randint(0, v, (m,), device="cuda", generator=g)
        if case["table"] == "mx4":
            s["codes"], s["scales"] = _quantize(w)
            rows = _values(s["codes"][labels], s["scales"][labels], torch.float32)
        else:
            s["w"] = w.bfloat16()
            rows = s["w"][labels].float()
        # hidden states that lean towards their label, as a trained model's do: some rows are sure of it
        lean = torch.rand(m, 1, device="cuda", generator=g) * 12.0
        s["h"] = (_randn(g, m, c) + lean * rows / rows.norm(dim=1, keepdim=True)).bfloat16().requires_grad_(True)
        if m > 1:  # padding of ragged sequences
            labels[torch.rand(m, device="cuda", generator=g) < 0.1] = -100
        s["labels"] = labels
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from mobilefinetuner_amd.ops import functional as Fx
    c = s["case"]
    op = c["op"]
    if op == "quantize":
        w4 = Fx.mx4_quantize(s["w"])
        return w4.dequantize(), w4.scales
    if op == "loss":
        table = Fx.MX4Weight(s["codes"], s["scales"]) if c["table"] == "mx4" else s["w"]
        loss = Fx.lm_head_cross_entropy_pieces(s["h"], table, s["labels"], c["v"])
        return loss.detach(), torch.autograd.grad(loss, s["h"])[0]
    w4 = Fx.MX4Weight(s["codes"], s["scales"])
    if op == "embedding":
        return Fx.mx4_embedding(s["ids"], w4, s["wpe"], c["scale"])
    y = Fx.mx4_linear(s["x"], w4, s["bias"])
    if op == "linear":
        return y
    return y.detach(), torch.autograd.grad(y, s["x"], s["dy"])[0]


@torch.no_grad()
def _run_plain(s):
    c = s["case"]
    op = c["op"]
    if op == "quantize":
        codes, scales = _quantize(s["w"])
        return _values(codes, scales, torch.float32).bfloat16(), scales
    if op == "loss":
        w = _values(s["codes"], s["scales"], torch.float32) if c["table"] == "mx4" else s["w"].float()
        loss, dh = _loss(s["h"].float(), w, s["labels"], c["v"])
        return loss, dh.bfloat16()
    if op == "embedding":
        ids = s["ids"].reshape(-1)
        out = _values(s["codes"][ids], s["scales"][ids], torch.float32) * c["scale"]
        if c["pos"]:
            out = (out.view(c["b"], c["s"], -1) + s["wpe"][: c["s"]].float()).view(ids.numel(), -1)
        return out.bfloat16()
    w = _values(s["codes"], s["scales"], torch.float32)
    y = torch.mm(s["x"].float(), w.t())
    if c["bias"]:
        y = y + s["bias"].float()
    y = y.bfloat16()
    if op == "linear":
        return y
    return y, torch.mm(s["dy"].float(), w).bfloat16()


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "quantize":
        n, k = case["n"], case["k"]
        # the matrix read, its values in bf16 and the scales written
        return {"bytes": n * k * (4 if case["dtype"] == "f32" else 2) + n * k * 2 + n * k // GROUP, "flops": 4 * n * k}
    if op in ("linear", "linear_step"):
        m, n, k = case["m"], case["n"], case["k"]
        ways = 2 if op == "linear_step" else 1
        return {"bytes": ways * (n * k * 17 // 32 + 2 * m * k + 2 * m * n) + (2 * n if case["bias"] else 0),
                "flops": ways * 2 * m * n * k}
    if op == "embedding":
        m, c = case["b"] * case["s"], case["c"]
        return {"bytes": m * (8 + c * 17 // 32 + 2 * c) + (case["s"] * c * 2 if case["pos"] else 0), "flops": 2 * m * c}
    m, v, c = case["m"], case["v"], case["c"]
    return {"bytes": (v * c * 17 // 32 if case["table"] == "mx4" else 2 * v * c) + 4 * m * c + 8 * m, "flops": 4 * m * v * c}


# ---------------------------------------------------------------- in 64 bits
def _exact_values(codes, scales):
    """From the definition: sign, two exponent bits (bias 1, 0 = subnormal), one mantissa bit, times 2 ** (byte - 127)."""
    c = torch.stack((codes.long() % 16, codes.long() // 16), -1).flatten(1)
    e, f = c // 2 % 4, (c % 2).double()
    v = torch.where(e == 0, f * 0.5, (1.0 + 0.5 * f) * torch.ldexp(torch.ones_like(f), e - 1))
    v = torch.where(c >= 8, -v, v)
    return v * torch.ldexp(torch.ones_like(v), (scales.long() - 127).repeat_interleave(GROUP, 1))


def _exact_quantize(w):
    n, k = w.shape
    x = w.double().view(n, k // GROUP, GROUP)
    frac, e = torch.frexp(x.abs().amax(-1))  # max = frac * 2 ** e, frac in [0.5, 1)
    e = torch.where(frac > 0.875, e - 2, e - 3).clamp(-125, 125)
    x = torch.ldexp(x, -e.unsqueeze(-1))
    mag = x.abs()
    # nearest of the grid; at a border the neighbour with the even mantissa bit
    edges = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    out = torch.zeros_like(mag)
    for i, b in enumerate(edges):
        over = mag >= b if i % 2 else mag > b
        out = torch.where(over, GRID[i + 1], out)
    return torch.ldexp(torch.copysign(out, x), e.unsqueeze(-1)).view(n, k)


@torch.no_grad()
def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "quantize":
        w = s["w"]
        return torch.cat([_exact_quantize(p) for p in w.split(max(1, 32_000_000 // w.shape[1]))]), None
    if op == "embedding":
        ids = s["ids"].reshape(-1)
        out = _exact_values(s["codes"][ids], s["scales"][ids]) * case["scale"]
        if case["pos"]:
            out = out + s["wpe"].double()[torch.arange(ids.numel(), device=ids.device) % case["s"]]
        return out
    if op == "loss":
        m, v, c = case["m"], case["v"], case["c"]
        h, labels = s["h"].double(), s["labels"]
        valid = labels != -100
        part = max(256, min(v, 800_000_000 // max(1, m)))

        def table(i):
            return _exact_values(s["codes"][i:i + part], s["scales"][i:i + part]) if case["table"] == "mx4" else s["w"][i:i + part].double()

        lse = torch.full((m,), -math.inf, dtype=torch.float64, device=h.device)
        for i in range(0, v, part):
            lse = torch.logaddexp(lse, torch.logsumexp(h @ table(i).t(), 1))
        dh = torch.zeros_like(h)
        picked = torch.zeros_like(lse)
        for i in range(0, v, part):
            w = table(i)
            p = h @ w.t()
            here = torch.nonzero(valid & (labels >= i) & (labels < i + w.shape[0])).squeeze(1)
            picked[here] = p[here, labels[here] - i]
            p = torch.exp(p - lse.unsqueeze(1))
            p[here, labels[here] - i] -= 1.0
            dh += p @ w
        count = max(1, int(valid.sum()))
        return ((lse - picked) * valid).sum() / count, dh * (valid.double() / count).unsqueeze(1)
    w = _exact_values(s["codes"], s["scales"])
    y = s["x"].double() @ w.t()
    if case["bias"]:
        y = y + s["bias"].double()
    return y if op == "linear" else (y, s["dy"].double() @ w)
