"""4-bit frozen weights on the GPU (kernels/mx4.hip) against their definition in 64 bits.

Tolerances.  Weights and activations are exact bf16 numbers, a product of two is exact in fp32, a sum of n of
them in fp32 is off by at most n * 2^-23 of the sum of their magnitudes (2^-24 a step, twice that for an adder
that cuts off), and the result is rounded once to bf16: half a step, 2^-8 of the value."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu


def _fx():
    from mobilefinetuner_amd.ops import functional as Fx
    return Fx


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight(n, k, seed=0, std=0.05):
    w = torch.randn(n, k, device="cuda", generator=_gen(seed)) * std
    return _fx().mx4_quantize(w.bfloat16())


def _check(got, want, mag, terms):
    got, want = got.double().cpu(), want.cpu()
    off = (got - want).abs() - (want.abs() * 2.0 ** -8 + mag.cpu() * (terms + 2) * 2.0 ** -23 + 2.0 ** -133)
    assert not torch.isnan(got).any() and off.max().item() <= 0, (off.max().item(), (got - want).abs().max().item())


# ---------------------------------------------------------------- quantise
def _hard_rows():
    """Rows of one group: every border of the grid, saturation, ties, zeros of both signs, tiny and huge values."""
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 7.0])
    near = torch.cat([edges, edges * (1 + 2.0 ** -7), edges * (1 - 2.0 ** -8)])
    rows = []
    for top in (3.75, 4.0, 6.0, 7.0):
        r = torch.cat([near.clamp(max=top), torch.tensor([top, -top])])
        rows += [r * 2.0 ** e for e in (0, -1, -60, -110, -124, -126, 60, 124)]
    rows.append(torch.zeros(32))
    rows.append(-torch.zeros(32))
    rows.append(torch.full((32,), 2.0 ** -126))
    rows.append(torch.full((32,), 2.0 ** -133))
    rows.append(torch.full((32,), torch.finfo(torch.bfloat16).max))
    one = torch.zeros(32)
    one[17] = -1.0
    rows.append(one)
    return torch.stack(rows)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_matches_definition_on_hard_values(dtype):
    w = _hard_rows().to(dtype).cuda()
    w4 = _fx().mx4_quantize(w)
    codes, scales = ref.quantize(w)
    assert torch.equal(w4.scales.cpu(), scales)
    got, want = ref.values(w4.codes, w4.scales), ref.values(codes, scales)
    bad = (got != want).any(1).nonzero().flatten().tolist()
    assert not bad, (bad, w[bad[0]].tolist(), got[bad[0]].tolist(), want[bad[0]].tolist())
    assert torch.equal(w4.dequantize().double().cpu(), want)


@pytest.mark.parametrize("n,k,dtype", [(1, 32, torch.bfloat16), (3, 64, torch.float32), (257, 96, torch.bfloat16),
                                       (1000, 768, torch.float32), (77, 6912, torch.bfloat16)])
def test_quantize_random(n, k, dtype):
    g = _gen(n + k)
    w = torch.randn(n, k, device="cuda", generator=g) * torch.exp(3 * torch.randn(n, 1, device="cuda", generator=g))
    w = w.to(dtype)
    w4 = _fx().mx4_quantize(w)
    codes, scales = ref.quantize(w)
    assert w4.shape == (n, k) and torch.equal(w4.scales.cpu(), scales) and torch.equal(w4.codes.cpu(), codes)
    assert torch.equal(w4.dequantize().double().cpu(), ref.values(codes, scales))
    # the format's promise: off by at most half a step of the grid around 4 .. 6 (1.0) times the scale
    step = torch.pow(2.0, scales.double() - 127).repeat_interleave(32, 1)
    assert ((ref.values(codes, scales) - w.double().cpu()).abs() <= step).all()


def test_quantize_strided_unaligned_and_empty():
    big = torch.randn(40, 200, device="cuda", generator=_gen(1)).bfloat16()
    for w in (big[3:30, 5:69], big.t()[:64, :32], big[:0, :64]):
        w4 = _fx().mx4_quantize(w)
        codes, scales = ref.quantize(w) if w.shape[0] else (w4.codes.cpu(), w4.scales.cpu())
        assert w4.shape == w.shape and torch.equal(w4.codes.cpu(), codes) and torch.equal(w4.scales.cpu(), scales)


def test_nonfinite_group_reads_as_nan_and_no_other():
    w = torch.randn(4, 96, device="cuda", generator=_gen(2))
    w[1, 40], w[2, 0], w[2, 95] = float("inf"), float("nan"), float("-inf")
    w4 = _fx().mx4_quantize(w)
    nan = torch.isnan(w4.dequantize()).cpu()
    want = torch.zeros(4, 96, dtype=torch.bool)
    want[1, 32:64] = want[2, :32] = want[2, 64:] = True
    assert torch.equal(nan, want) and torch.equal(w4.scales.cpu() == 255, want[:, ::32])
    x = torch.randn(3, 96, device="cuda", generator=_gen(3)).bfloat16()
    y = _fx().mx4_linear(x, w4)
    assert torch.equal(torch.isnan(y).cpu(), torch.tensor([[False, True, True, False]] * 3))
    e = _fx().mx4_embedding(torch.tensor([[0, 1, 2, 3]], device="cuda"), w4)
    assert torch.equal(torch.isnan(e).cpu(), want)


# ---------------------------------------------------------------- products
SIZES = [(1, 1, 32), (1, 16, 64), (1, 2304, 768), (2, 15, 96), (5, 130, 160), (16, 64, 128), (17, 33, 224), (37, 1152, 6912),
         (64, 100, 128), (65, 257, 320), (100, 48, 32), (129, 128, 256), (300, 520, 1600), (512, 768, 640), (1000, 96, 1152),
         (2049, 264, 192), (3000, 1003, 96)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("with_bias", [False, True])
def test_linear_forward(m, n, k, with_bias):
    w4 = _weight(n, k, seed=m)
    x = torch.randn(m, k, device="cuda", generator=_gen(n)).bfloat16()
    b = torch.randn(n, device="cuda", generator=_gen(k)).bfloat16() if with_bias else None
    y = _fx().mx4_linear(x, w4, b)
    v, xd = ref.values(w4.codes, w4.scales).cuda(), x.double()
    want, mag = xd @ v.t(), xd.abs() @ v.abs().t()
    if with_bias:
        want, mag = want + b.double(), mag + b.double().abs()
    assert y.shape == (m, n) and y.dtype == torch.bfloat16
    _check(y, want, mag, k)


@pytest.mark.parametrize("m,n,k", SIZES)
def test_linear_gradient(m, n, k):
    w4 = _weight(n, k, seed=m + 1)
    x = torch.randn(m, k, device="cuda", generator=_gen(n)).bfloat16().requires_grad_(True)
    dy = torch.randn(m, n, device="cuda", generator=_gen(k)).bfloat16()
    y = _fx().mx4_linear(x, w4)
    (dx,) = torch.autograd.grad(y, x, dy)
    v = ref.values(w4.codes, w4.scales).cuda()
    assert dx.shape == x.shape and dx.dtype == torch.bfloat16
    _check(dx, dy.double() @ v, dy.double().abs() @ v.abs(), n)


def test_linear_gradient_against_differences():
    """y is linear in x: with small whole numbers (exact sums) <dy, y(x + d) - y(x - d)> / 2 equals <dx, d>; only the
    roundings of y and dx (2^-8 of their values) stand between the two."""
    g = _gen(9)
    w4 = _weight(48, 64, seed=4, std=1.0)
    x = torch.randint(-3, 4, (5, 64), device="cuda", generator=g).bfloat16().requires_grad_(True)
    d = torch.randint(-2, 3, (5, 64), device="cuda", generator=g).bfloat16()
    dy = torch.randint(-2, 3, (5, 48), device="cuda", generator=g).bfloat16()
    Fx = _fx()
    (dx,) = torch.autograd.grad(Fx.mx4_linear(x, w4), x, dy)
    with torch.no_grad():
        up, down = Fx.mx4_linear(x + d, w4).double(), Fx.mx4_linear(x - d, w4).double()
    lhs = (dy.double() * (up - down)).sum().item() / 2
    rhs = (dx.double() * d.double()).sum().item()
    room = 2.0 ** -8 * ((dy.double().abs() * (up.abs() + down.abs())).sum() / 2 + (dx.double() * d.double()).abs().sum()).item()
    assert abs(lhs - rhs) <= room, (lhs, rhs, room)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_linear_takes_views(m):
    """Row strides, unaligned starts, transposed and expanded activations and gradients, more dimensions, one."""
    Fx = _fx()
    k, n = 96, 72
    w4 = _weight(n, k)
    v = ref.values(w4.codes, w4.scales).cuda()
    big = torch.randn(m, 2 * k + 3, device="cuda", generator=_gen(m)).bfloat16()
    tall = torch.randn(k, m, device="cuda", generator=_gen(m + 1)).bfloat16()
    for x in (big[:, :k], big[:, 3:3 + k], tall.t(), big[:1, :k].expand(m, k), big[:, :k].reshape(1, m, 1, k)):
        x = x.detach().requires_grad_(True)
        y = Fx.mx4_linear(x, w4)
        assert y.shape == (*x.shape[:-1], n)
        xd = x.detach().double()
        _check(y.detach(), xd @ v.t(), xd.abs() @ v.abs().t(), k)
        for dy in (torch.ones(1, 1, device="cuda").bfloat16().expand(m, n), big[:, 1:1 + n], big[:, :n], tall[:n].t()):
            (dx,) = torch.autograd.grad(y, x, dy.reshape(y.shape), retain_graph=True)
            _check(dx.reshape(m, k), dy.double() @ v, dy.double().abs() @ v.abs(), n)
    y = Fx.mx4_linear(big[0, :k], w4)
    assert y.shape == (n,)
    _check(y, v @ big[0, :k].double(), v.abs() @ big[0, :k].double().abs(), k)
    assert Fx.mx4_linear(big[:0, :k], w4).shape == (0, n)


@pytest.mark.parametrize("m", [3, 40, 600])
def test_linear_nonfinite_rows_stay_their_own(m):
    Fx = _fx()
    n, k = 130, 160
    w4 = _weight(n, k)
    x = torch.randn(m, k, device="cuda", generator=_gen(5)).bfloat16()
    y0 = Fx.mx4_linear(x, w4)
    bad = x.clone()
    bad[1, k - 1] = float("nan")
    bad[2, 0] = float("inf")
    y = Fx.mx4_linear(bad, w4)
    keep = torch.ones(m, dtype=torch.bool)
    keep[1] = keep[2] = False
    assert torch.equal(y[keep.cuda()], y0[keep.cuda()])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[2][ref.values(w4.codes, w4.scales)[:, 0].cuda() != 0]).any()
    dy = torch.randn(m, n, device="cuda", generator=_gen(6)).bfloat16()
    C = __import__("mobilefinetuner_amd._ext", fromlist=["native"]).native()
    d0 = C.mx4_dgrad(dy, w4.codes, w4.scales)
    dy[1, n - 1] = float("nan")
    d = C.mx4_dgrad(dy, w4.codes, w4.scales)
    keep[2] = True
    assert torch.equal(d[keep.cuda()], d0[keep.cuda()]) and torch.isnan(d[1]).all()


def test_bias_gradient():
    Fx = _fx()
    w4 = _weight(64, 64)
    x = torch.randn(50, 64, device="cuda", generator=_gen(1)).bfloat16()
    b = torch.zeros(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(50, 64, device="cuda", generator=_gen(2)).bfloat16()
    (gb,) = torch.autograd.grad(Fx.mx4_linear(x, w4, b), b, dy)
    _check(gb, dy.double().sum(0), dy.double().abs().sum(0), 50)


# ---------------------------------------------------------------- embedding
@pytest.mark.parametrize("b,s,v,c", [(1, 1, 1, 32), (2, 3, 50, 96), (4, 128, 1001, 768), (3, 77, 300, 640)])
@pytest.mark.parametrize("scale", [1.0, 25.25])
@pytest.mark.parametrize("pos", [False, True])
def test_embedding(b, s, v, c, scale, pos):
    Fx = _fx()
    w4 = _weight(v, c, seed=v)
    ids = torch.randint(0, v, (b, s), device="cuda", generator=_gen(c))
    wpe = torch.randn(s + 5, c, device="cuda", generator=_gen(7)).bfloat16() if pos else None
    out = Fx.mx4_embedding(ids, w4, wpe, scale)
    want = ref.values(w4.codes, w4.scales)[ids.reshape(-1).cpu()] * float(torch.tensor(scale, dtype=torch.float32))
    mag = want.abs()
    if pos:
        p = wpe[:s].double().cpu().repeat(b, 1)
        want, mag = want + p, mag + p.abs()
    assert out.shape == (b * s, c)
    _check(out, want, mag, 2)
    assert torch.equal(out, Fx.embedding(ids, w4, wpe, scale))


def test_embedding_ids_outside_the_table_are_nan():
    w4 = _weight(10, 64)
    ids = torch.tensor([[0, -1, 9, 10, 1 << 40]], device="cuda")
    out = _fx().mx4_embedding(ids, w4)
    assert torch.isnan(out).all(1).tolist() == [False, True, False, True, True]
    assert not torch.isnan(out[0]).any() and not torch.isnan(out[2]).any()


# ---------------------------------------------------------------- streams, graphs
@pytest.mark.parametrize("m", [1, 48, 700])
def test_captured_and_replayed(m):
    """Forward and gradient in one graph, replayed with new inputs between eager work, equal to the eager calls."""
    Fx = _fx()
    w4 = _weight(136, 192)
    C = __import__("mobilefinetuner_amd._ext", fromlist=["native"]).native()
    x = torch.zeros(m, 192, device="cuda", dtype=torch.bfloat16)
    dy = torch.zeros(m, 136, device="cuda", dtype=torch.bfloat16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        Fx.mx4_linear(x, w4), C.mx4_dgrad(dy, w4.codes, w4.scales)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = Fx.mx4_linear(x, w4), C.mx4_dgrad(dy, w4.codes, w4.scales)
    for r in range(4):
        x.copy_(torch.randn(m, 192, device="cuda", generator=_gen(r)).bfloat16())
        dy.copy_(torch.randn(m, 136, device="cuda", generator=_gen(r + 10)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, Fx.mx4_linear(x, w4)) and torch.equal(dx, C.mx4_dgrad(dy, w4.codes, w4.scales))


def test_two_streams_at_once():
    Fx = _fx()
    w4 = _weight(2304, 768)
    xs = [torch.randn(m, 768, device="cuda", generator=_gen(m)).bfloat16() for m in (1, 700)]
    want = [Fx.mx4_linear(x, w4) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(Fx.mx4_linear(xs[i], w4))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


# ---------------------------------------------------------------- refusals
def test_refusals():
    Fx = _fx()
    w4 = _weight(64, 64)
    x = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="bf16"):
        Fx.mx4_linear(x.float(), w4)
    with pytest.raises(RuntimeError, match="expected"):
        Fx.mx4_linear(x[:, :32], w4)
    with pytest.raises(RuntimeError, match="bias"):
        Fx.mx4_linear(x, w4, torch.zeros(63, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="bias"):
        Fx.mx4_linear(x, w4, torch.zeros(64, device="cuda"))
    with pytest.raises(RuntimeError, match="GPU"):
        Fx.mx4_linear(x, w4.to("cpu"))
    with pytest.raises(RuntimeError, match="multiple of 32"):
        Fx.mx4_quantize(torch.zeros(4, 48, device="cuda"))
    with pytest.raises(RuntimeError, match="fp32 or bf16"):
        Fx.mx4_quantize(torch.zeros(4, 32, device="cuda", dtype=torch.float16))
    with pytest.raises(RuntimeError, match="int64"):
        Fx.mx4_embedding(torch.zeros(1, 2, device="cuda", dtype=torch.int32), w4)
    with pytest.raises(RuntimeError, match="wpe"):
        Fx.mx4_embedding(torch.zeros(1, 2, device="cuda", dtype=torch.long), w4,
                         torch.zeros(1, 64, device="cuda", dtype=torch.bfloat16))
    p = torch.zeros(2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="position table"):
        Fx.mx4_embedding(torch.zeros(1, 2, device="cuda", dtype=torch.long), w4, p)


# ---------------------------------------------------------------- every tile shape, split and the bf16 copy
SHAPES = [(7295, 1056, 128), (8664, 199, 128), (9432, 65, 1824), (8352, 395, 128), (8800, 386, 3456), (16, 16, 1344), (699, 16, 1504),
          (147, 5450, 128), (18, 2706, 2592), (1438, 16, 2016), (33, 2815, 2720), (570, 6695, 160), (261, 7211, 3712),
          (6788, 192, 1184), (599, 16, 3456), (65, 2470, 3808), (9817, 16, 1280), (6995, 3264, 544), (17, 717, 128),
          (16, 1530, 1472), (33, 3015, 352), (34, 1067, 2720), (5415, 6592, 160), (4099, 2304, 768), (4190, 16, 160),
          (2085, 5696, 160), (8236, 192, 1536), (5402, 22, 704)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_large_and_ragged_products(m, n, k):
    w4 = _weight(n, k, seed=m)
    x = torch.randn(m, k, device="cuda", generator=_gen(n)).bfloat16().requires_grad_(True)
    b = torch.randn(n, device="cuda", generator=_gen(k)).bfloat16()
    dy = torch.randn(m, n, device="cuda", generator=_gen(k + 1)).bfloat16()
    y = _fx().mx4_linear(x, w4, b)
    (dx,) = torch.autograd.grad(y, x, dy)
    v, xd, dd = ref.values(w4.codes, w4.scales).cuda(), x.detach().double(), dy.double()
    _check(y.detach(), xd @ v.t() + b.double(), xd.abs() @ v.abs().t() + b.double().abs(), k)
    _check(dx, dd @ v, dd.abs() @ v.abs(), n)


@pytest.mark.parametrize("m", [2, 40, 4100])
def test_bias_at_any_address(m):
    """A contiguous bias that starts inside a 16-byte word."""
    n, k = 13824 if m == 2 else 1024, 512
    w4 = _weight(n, k)
    x = torch.randn(m, k, device="cuda", generator=_gen(1)).bfloat16()
    long = torch.randn(n + 3, device="cuda", generator=_gen(2)).bfloat16()
    for o in (1, 2, 3):
        assert torch.equal(_fx().mx4_linear(x, w4, long[o:o + n]), _fx().mx4_linear(x, w4, long[o:o + n].clone()))


def test_one_weight_twice_in_a_graph():
    """A weight used by two products of one graph, and a graph walked twice: the gradients add, nothing is kept."""
    Fx = _fx()
    w4 = _weight(96, 96)
    x = torch.randn(70, 96, device="cuda", generator=_gen(3)).bfloat16().requires_grad_(True)
    dy = torch.randn(70, 96, device="cuda", generator=_gen(4)).bfloat16()
    y = Fx.mx4_linear(Fx.mx4_linear(x, w4), w4)
    (a,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    (b,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    assert torch.equal(a, b)
    (c,) = torch.autograd.grad(y, x, dy + dy)
    assert torch.equal(c, a + a)


def test_training_on_two_streams_at_once():
    Fx = _fx()
    w4 = _weight(2304, 768)
    g = _gen(5)
    xs = [torch.randn(m, 768, device="cuda", generator=g).bfloat16().requires_grad_(True) for m in (100, 1500)]
    dys = [torch.randn(x.shape[0], 2304, device="cuda", generator=g).bfloat16() for x in xs]
    want = [torch.autograd.grad(Fx.mx4_linear(x, w4), x, dy)[0] for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(8):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(torch.autograd.grad(Fx.mx4_linear(xs[i], w4), xs[i], dys[i])[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(d, want[i]) for d in got[i])


def test_codes_past_4_gib():
    """2,097,180 x 4,128: codes of 4.3 GB.  Its last rows give what they give as a weight of their own."""
    Fx = _fx()
    n, k, last = 2097180, 4128, 60
    codes = torch.zeros(n, k // 2, device="cuda", dtype=torch.uint8)
    scales = torch.full((n, k // 32), 127, device="cuda", dtype=torch.uint8)
    codes[-last:] = torch.randint(0, 256, (last, k // 2), device="cuda", generator=_gen(6)).to(torch.uint8)
    scales[-last:] = torch.randint(118, 122, (last, k // 32), device="cuda", generator=_gen(7)).to(torch.uint8)
    w4, end = Fx.MX4Weight(codes, scales), Fx.MX4Weight(codes[-last:].clone(), scales[-last:].clone())
    v = ref.values(end.codes, end.scales).cuda()
    for m in (1, 8, 40):
        x = torch.randn(m, k, device="cuda", generator=_gen(m)).bfloat16().requires_grad_(True)
        y = Fx.mx4_linear(x, w4)
        xd = x.detach().double()
        _check(y.detach()[:, -last:], xd @ v.t(), xd.abs() @ v.abs().t(), k)
        assert y.detach()[:, :-last].abs().max().item() == 0.0
        dy = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
        dy[:, -last:] = torch.randn(m, last, device="cuda", generator=_gen(m + 1)).bfloat16()
        (dx,) = torch.autograd.grad(y, x, dy)
        d = dy[:, -last:].double()
        _check(dx, d @ v, d.abs() @ v.abs(), last)
    ids = torch.tensor([[n - 1, n - last, 0]], device="cuda")
    out = Fx.mx4_embedding(ids, w4)
    assert torch.equal(out[0], v[-1].bfloat16()) and torch.equal(out[1], v[0].bfloat16()) and out[2].abs().max().item() == 0.0
    assert torch.equal(Fx.mx4_quantize(end.dequantize()).dequantize(), end.dequantize())


@pytest.mark.parametrize("m,n,k", [(5000, 1603, 1600), (8236, 195, 1536), (700, 1001, 512), (20, 13001, 256), (3, 13003, 128), (50, 2047, 96)])
def test_widths_that_are_no_multiple_of_8(m, n, k):
    """Odd result rows, and the gradient of one that starts at an odd address in a larger tensor, as a copy gives it."""
    Fx = _fx()
    w4 = _weight(n, k, seed=m)
    x = torch.randn(m, k, device="cuda", generator=_gen(n)).bfloat16().requires_grad_(True)
    b = torch.randn(n, device="cuda", generator=_gen(k)).bfloat16()
    big = torch.randn(m, n + 5, device="cuda", generator=_gen(k + 1)).bfloat16()
    y = Fx.mx4_linear(x, w4, b)
    dy = big[:, 3:3 + n]
    (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    (again,) = torch.autograd.grad(y, x, dy.contiguous())
    v, xd, dd = ref.values(w4.codes, w4.scales).cuda(), x.detach().double(), dy.double()
    _check(y.detach(), xd @ v.t() + b.double(), xd.abs() @ v.abs().t() + b.double().abs(), k)
    _check(dx, dd @ v, dd.abs() @ v.abs(), n)
    assert torch.equal(dx, again)


# ---------------------------------------------------------------- rows that repeat or overlap, at sizes of the bf16 copy
@pytest.mark.parametrize("m,n,k", [(9000, 6400, 1600), (600, 136, 192), (7, 96, 64)])
@pytest.mark.parametrize("stride", [0, 8])
def test_rows_that_repeat_or_overlap(m, n, k, stride):
    """x and dy whose rows are all one row (an expanded one) or start 8 elements apart, and the gradient that a sum over the
    rows hands back, strides (0, 1)."""
    Fx = _fx()
    w4 = _weight(n, k, seed=m)
    v = ref.values(w4.codes, w4.scales).cuda()

    def rows(width, seed):
        flat = torch.randn((m - 1) * stride + width, device="cuda", generator=_gen(seed)).bfloat16()
        return flat.as_strided((m, width), (stride, 1))
    x = rows(k, n).detach().requires_grad_(True)
    xd = x.detach().double()
    y = Fx.mx4_linear(x, w4)
    _check(y.detach(), xd @ v.t(), xd.abs() @ v.abs().t(), k)
    dy = rows(n, k)
    (dx,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    _check(dx, dy.double() @ v, dy.double().abs() @ v.abs(), n)
    g = torch.randn(n, device="cuda", generator=_gen(11)).bfloat16()
    (dx,) = torch.autograd.grad(y.sum(0), x, g)
    want = (g.double() @ v).expand(m, k)
    _check(dx, want, (g.double().abs() @ v.abs()).expand(m, k), n)


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode_derivatives_are_refused(grad):
    """A dual tensor's tangent is not dropped without a word, whether or not a gradient is tracked as well."""
    import torch.autograd.forward_ad as fw
    Fx = _fx()
    w4 = _weight(64, 64)
    ids = torch.zeros(1, 2, device="cuda", dtype=torch.long)
    labels = torch.zeros(2, device="cuda", dtype=torch.long)
    plain = torch.ones(2, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.ones(64, 64, device="cuda", dtype=torch.bfloat16)
    with fw.dual_level():
        x = fw.make_dual(plain.clone().requires_grad_(grad), torch.ones_like(plain))
        b = fw.make_dual(torch.ones_like(plain[0]), torch.ones_like(plain[0]))
        t = fw.make_dual(table.clone(), torch.ones_like(table))
        for call in (lambda: Fx.mx4_linear(x, w4), lambda: Fx.mx4_linear(plain, w4, b), lambda: Fx.linear(x, w4),
                     lambda: Fx.mx4_embedding(ids, w4, t), lambda: Fx.lm_head_cross_entropy_pieces(x, w4, labels, 64),
                     lambda: Fx.lm_head_cross_entropy_pieces(x, table, labels, 64), lambda: Fx.lm_head_token_nll(x, w4, labels, 64),
                     lambda: Fx.lm_head_cross_entropy_pieces(plain, t, labels, 64)):
            with pytest.raises(RuntimeError, match="forward-mode|jvp"):
                call()


# ---------------------------------------------------------------- scale bytes that the quantiser does not write
def test_every_scale_byte_and_code():
    """Bytes 0 and 1 (bf16 denormals), 253 and 254 (what is past bf16's largest number is an infinity), 255 (NaN), in weights
    from elsewhere: each of the 16 codes under each of the 256 bytes."""
    Fx = _fx()
    c = torch.arange(16, dtype=torch.uint8)
    codes = (c | ((c + 1) % 16) << 4).repeat(256, 1).cuda()
    w4 = Fx.MX4Weight(codes, torch.arange(256, dtype=torch.uint8).view(256, 1).cuda())
    want = ref.values(w4.codes, w4.scales).bfloat16()
    ids = torch.arange(256, device="cuda").view(1, 256)
    for got in (w4.dequantize(), Fx.mx4_embedding(ids, w4)):
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu()[:255], want[:255])


@pytest.mark.parametrize("m,n", [(1, 64), (40, 64), (4, 13000), (300, 512), (9000, 6400)])
@pytest.mark.parametrize("byte", [0, 1, 2])
def test_smallest_scales_in_products(m, n, byte):
    """Denormal bf16 weights reach the products of every route: one times 2^100, exact."""
    from mobilefinetuner_amd._ext import native
    Fx = _fx()
    k = 128
    codes = torch.zeros(n, k // 2, dtype=torch.uint8, device="cuda")
    codes[:, 0] = 0x21  # 0.5 and 1
    w4 = Fx.MX4Weight(codes, torch.full((n, k // 32), byte, dtype=torch.uint8, device="cuda"))
    x = torch.zeros(m, k, device="cuda", dtype=torch.bfloat16)
    x[:, :2] = 2.0 ** 100
    dy = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    dy[:, 0] = 2.0 ** 100
    scale = 2.0 ** (byte - 27)
    assert (Fx.mx4_linear(x, w4).double() == 1.5 * scale).all()
    dx = native().mx4_dgrad(dy, w4.codes, w4.scales).double()
    assert (dx[:, 0] == 0.5 * scale).all() and (dx[:, 1] == scale).all() and (dx[:, 2:] == 0).all()


SPLIT_16 = [(31, 403, 3680), (17, 28, 9088)]  # tiles of 16 rows that share out their reduction


@pytest.mark.parametrize("m,n,k", SPLIT_16)
def test_small_tiles_that_split(m, n, k):
    test_large_and_ragged_products(m, n, k)
