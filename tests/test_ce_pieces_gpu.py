"""LM-head cross entropy in pieces of the vocabulary (kernels/ce_pieces.hip) against the formula in 64 bits.

Tolerances.  Loss: a logit is an fp32 sum of K exact products (off by at most K 2^-23 sum|h w|), the exponentials and
logarithms of the softmax add a few 2^-23 of values up to |lse|.  Gradient of a row: the softmax numbers pass
through bf16 (half a step, 2^-8 of each: 2^-8 sum_v p_v |W_v|), a logit's error multiplies its softmax number,
the sums are fp32, and the result is rounded once (2^-8)."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu


def _fx():
    from mobilefinetuner_amd.ops import functional as Fx
    return Fx


def _case(m, k, v, table, seed=0, rows=None, lean=8.0, ignore=0.2, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(rows or v, k, device="cuda", generator=g) * k ** -0.5
    labels = torch.randint(0, v, (m,), device="cuda", generator=g)
    if table == "mx4":
        w = _fx().mx4_quantize(w)
        wd = ref.values(w.codes, w.scales).cuda()
    else:
        w = w.bfloat16()
        wd = w.double()
    pick = wd[labels]
    lean = torch.rand(m, 1, device="cuda", generator=g, dtype=torch.float64) * lean
    h = (torch.randn(m, k, device="cuda", generator=g) * scale + lean * pick / pick.norm(dim=1, keepdim=True)).bfloat16()
    labels[torch.rand(m, device="cuda", generator=g) < ignore] = -100
    return h, w, wd[:v], labels


def _exact(h, wd, labels):
    v = wd.shape[0]
    hd = h.double()
    valid = (labels >= 0) & (labels < v)
    n = max(1, int(valid.sum()))
    logits = hd @ wd.t()
    lse = torch.logsumexp(logits, 1)
    lab = torch.where(valid, labels, 0)
    rows = torch.where(valid, lse - logits.gather(1, lab[:, None])[:, 0], 0.0)
    p = torch.exp(logits - lse[:, None])
    mag_logit = (hd.abs() @ wd.abs().t()).amax(1)
    err_logit = 2.0 ** -23 * (h.shape[1] + 4) * mag_logit + 2.0 ** -20 * (1 + lse.abs())
    d = p.clone()
    d.scatter_add_(1, lab[:, None], torch.full_like(p[:, :1], -1.0))
    dh = (d @ wd) * valid[:, None] / n
    off_label = p.scatter(1, lab[:, None], 0.0)
    spread = off_label @ wd.abs() + (p.gather(1, lab[:, None]) * wd[lab].abs())
    room = (off_label @ wd.abs()) * 2.0 ** -8 + spread * (4 * err_logit[:, None] + 2.0 ** -18)
    room = room * valid[:, None] / n + dh.abs() * 2.0 ** -8 + 2.0 ** -133
    loss_room = (err_logit * valid).sum().item() / n * 2 + 2.0 ** -23 * 8 * (rows.sum().item() / n)
    return rows.sum() / n, dh, room, loss_room


def _run(h, w, labels, v, piece=None):
    x = h.detach().requires_grad_(True)
    loss = _fx().lm_head_cross_entropy_pieces(x, w, labels, v, piece)
    (dh,) = torch.autograd.grad(loss, x)
    return loss.detach(), dh


def _check(h, w, wd, labels, v, piece=None):
    loss, dh = _run(h, w, labels, v, piece)
    want, dwant, room, loss_room = _exact(h, wd, labels)
    assert abs(loss.item() - want.item()) <= loss_room, (loss.item(), want.item(), loss_room)
    over = (dh.double() - dwant).abs() - room
    assert not torch.isnan(dh).any() and over.max().item() <= 0, over.max().item()
    ignored = ~((labels >= 0) & (labels < v))
    assert dh[ignored].abs().sum().item() == 0.0
    with torch.no_grad():
        assert _fx().lm_head_cross_entropy_pieces(h, w, labels, v, piece).item() == loss.item()
    return loss, dh


# m, k, v, piece: one row to many, one piece to many, ragged last pieces (of one column too), K not a multiple of 64
SIZES = [(1, 64, 300, None), (1, 128, 1000, 256), (2, 96, 257, 256), (3, 64, 1, None), (7, 32, 64, 256), (17, 160, 4097, 1024),
         (64, 640, 5000, 512), (100, 768, 50257, None), (129, 64, 2304, 768), (255, 1152, 3001, 2048), (257, 320, 8192, 4096),
         (300, 768, 50257, 8192), (520, 1600, 1999, 512), (1025, 128, 2049, 1024), (2100, 640, 20000, 4096)]


@pytest.mark.parametrize("m,k,v,piece", SIZES)
@pytest.mark.parametrize("table", ["bf16", "mx4"])
def test_loss_and_gradient(m, k, v, piece, table):
    h, w, wd, labels = _case(m, k, v, table, seed=m + v)
    _check(h, w, wd, labels, v, piece)


def test_narrow_table_of_a_multiple_of_8():
    h, w, wd, labels = _case(33, 72, 700, "bf16")
    _check(h, w, wd, labels, 700, 256)


def test_padded_table_rows_do_not_count():
    """A table with rows past the vocabulary (a padded embedding): whatever finite values they hold."""
    h, w, wd, labels = _case(200, 128, 1000, "bf16", rows=1088)
    w[1000:] = 50.0
    _check(h, w, wd, labels, 1000, 512)
    w[1000:] = 0
    _check(h, w, wd, labels, 1000)


@pytest.mark.parametrize("piece", [None, 256, 1024])
def test_large_logits_and_sure_rows(piece):
    """Logits of about +-100 and rows that are sure of their label (p = 1 - tiny): the small gradient that is left
    keeps its precision, because the label's own softmax number never passes through bf16."""
    h, w, wd, labels = _case(300, 256, 3000, "bf16", lean=0.0, scale=25.0)
    _check(h, w, wd, labels, 3000, piece)
    h, w, wd, labels = _case(300, 256, 3000, "mx4", lean=14.0, scale=0.3)
    _check(h, w, wd, labels, 3000, piece)


def test_growing_and_falling_maxima():
    """The running maximum moves up in each piece, or was in the first one, hundreds above the rest."""
    g = torch.Generator(device="cuda").manual_seed(3)
    v, k = 2048, 64
    w = torch.randn(v, k, device="cuda", generator=g) * 0.05
    w[:, 0] = torch.linspace(0, 4, v, device="cuda")
    h = torch.randn(40, k, device="cuda", generator=g)
    h[:20, 0], h[20:, 0] = 60.0, -60.0
    labels = torch.randint(0, v, (40,), device="cuda", generator=g)
    h, w = h.bfloat16(), w.bfloat16()
    _check(h, w, w.double(), labels, v, 256)


@pytest.mark.parametrize("labels", ["none", "out of range", "edges"])
def test_labels(labels):
    h, w, wd, lab = _case(50, 64, 700, "mx4", ignore=0.0)
    if labels == "none":
        lab[:] = -100
    elif labels == "out of range":
        lab[::3], lab[1::3] = 700, -1
        lab[5] = 1 << 40
    else:
        lab[:] = torch.tensor([0, 255, 256, 511, 512, 699], device="cuda").repeat(9)[:50]
    loss, dh = _check(h, w, wd, lab, 700, 256)
    if labels == "none":
        assert loss.item() == 0.0 and dh.abs().sum().item() == 0.0


def test_gradient_against_differences():
    """Central differences of the loss along a random direction.  The loss is off by at most loss_room, so the
    quotient is off by loss_room / eps and by eps^2 / 6 of the third derivative (at most 6 max|<w, d>|^3 for a softmax);
    <dh, d> is off by sum room |d|."""
    h, w, wd, labels = _case(40, 128, 900, "bf16", lean=3.0)
    _, dh = _run(h, w, labels, 900, 256)
    _, _, room, loss_room = _exact(h, wd, labels)
    g = torch.Generator(device="cuda").manual_seed(8)
    eps = 2.0 ** -2
    # a step that bf16 h takes exactly: whole multiples of 2^-2 around values under 8 (8 bits)
    base = (h.float() * 16).round().clamp(-127, 127) / 16
    d = torch.randint(-1, 2, h.shape, device="cuda", generator=g).float()
    hb, up, down = base.bfloat16(), (base + eps * d).bfloat16(), (base - eps * d).bfloat16()
    d = (up.double() - down.double()) / (2 * eps)  # what was really taken
    mid = ((up.double() + down.double()) / 2 == hb.double()).all(1)
    labels = torch.where(mid, labels, -100)
    _, dh = _run(hb, w, labels, 900, 256)
    _, _, room, loss_room = _exact(hb, wd, labels)
    with torch.no_grad():
        lu, ld = (_fx().lm_head_cross_entropy_pieces(t, w, labels, 900, 256).double().item() for t in (up, down))
    slope = (dh.double() * d).sum().item()
    third = 6 * (d @ wd.t()).abs().max().item() ** 3
    tol = (room * d.abs()).sum().item() + loss_room / eps + eps ** 2 / 6 * third
    assert abs((lu - ld) / (2 * eps) - slope) <= tol, ((lu - ld) / (2 * eps), slope, tol)


def test_scaled_loss_scales_the_gradient():
    h, w, wd, labels = _case(64, 128, 500, "mx4")
    x = h.detach().requires_grad_(True)
    (a,) = torch.autograd.grad(_fx().lm_head_cross_entropy_pieces(x, w, labels, 500) * 4.0, x)
    _, b = _run(h, w, labels, 500)
    assert torch.equal(a, b * 4.0)


def test_pieces_and_reruns_agree():
    """The same call gives the same bits; another piece width only reorders fp32 sums and bf16 roundings."""
    h, w, wd, labels = _case(300, 256, 5000, "mx4", seed=5)
    a, b = _run(h, w, labels, 5000, 1024), _run(h, w, labels, 5000, 1024)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for piece in (256, 2048, None):
        _check(h, w, wd, labels, 5000, piece)


def test_views_and_other_shapes():
    Fx = _fx()
    h, w, wd, labels = _case(60, 128, 900, "bf16")
    big = torch.zeros(60, 300, device="cuda", dtype=torch.bfloat16)
    want = _run(h, w, labels, 900, 512)
    for c0 in (0, 8, 3):
        big[:, c0:c0 + 128] = h
        got = _run(big[:, c0:c0 + 128], w, labels, 900, 512)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.zeros(900, 200, device="cuda", dtype=torch.bfloat16)
    for c0 in (0, 3):
        wide[:, c0:c0 + 128] = w
        got = _run(h, wide[:, c0:c0 + 128], labels, 900, 512)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = _run(h, w, labels.view(6, 10), 900, 512)
    assert torch.equal(got[0], want[0])
    strided = torch.stack([labels, labels], 1)[:, 0]
    assert torch.equal(_run(h, w, strided, 900, 512)[1], want[1])
    empty = Fx.lm_head_cross_entropy_pieces(h[:0].requires_grad_(True), w, labels[:0], 900)
    assert empty.item() == 0.0


def test_nan_row_stays_its_own():
    h, w, wd, labels = _case(70, 128, 900, "mx4", ignore=0.0)
    _, want = _run(h, w, labels, 900, 256)
    h[3, 5] = float("nan")
    loss, dh = _run(h, w, labels, 900, 256)
    assert torch.isnan(loss) and torch.isnan(dh[3]).all()
    keep = torch.arange(70, device="cuda") != 3
    assert torch.equal(dh[keep], want[keep])


def test_evaluation_sums_take_the_4_bit_table():
    Fx = _fx()
    h, w, wd, labels = _case(90, 128, 900, "mx4")
    total, n = Fx.lm_head_token_nll(h, w, labels, 900)
    want, _, _, room = _exact(h, wd, labels)
    assert n.item() == (labels >= 0).sum().item()
    assert abs(total.item() / n.item() - want.item()) <= room
    assert Fx.lm_head_cross_entropy(h, w, labels, 900).item() == Fx.lm_head_cross_entropy_pieces(h, w, labels, 900).item()


@pytest.mark.parametrize("table", ["bf16", "mx4"])
def test_captured_and_replayed(table):
    h, w, wd, labels = _case(300, 128, 1999, table)
    C = __import__("mobilefinetuner_amd._ext", fromlist=["native"]).native()

    def call():
        mx = table == "mx4"
        return C.lm_head_ce_pieces(h, None if mx else w, w.codes if mx else None, w.scales if mx else None, labels, 1999, 512, True)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for r in range(4):
        h2, _, _, l2 = _case(300, 128, 1999, table, seed=r + 20)
        h.copy_(h2), labels.copy_(l2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_refusals():
    Fx = _fx()
    h, w, _, labels = _case(8, 64, 300, "bf16")
    w4 = Fx.mx4_quantize(w)
    with pytest.raises(RuntimeError, match="bf16"):
        Fx.lm_head_cross_entropy_pieces(h.float(), w, labels, 300)
    with pytest.raises(RuntimeError, match="multiple of 256"):
        Fx.lm_head_cross_entropy_pieces(h, w, labels, 300, piece=100)
    with pytest.raises(RuntimeError, match="vocab_size"):
        Fx.lm_head_cross_entropy_pieces(h, w, labels, 301)
    with pytest.raises(RuntimeError, match="vocab_size"):
        Fx.lm_head_cross_entropy_pieces(h, w4, labels, 301)
    with pytest.raises(RuntimeError, match="vocab_size"):
        Fx.lm_head_cross_entropy_pieces(h, w, labels, 0)
    with pytest.raises(RuntimeError, match="labels"):
        Fx.lm_head_cross_entropy_pieces(h, w, labels[:7], 300)
    with pytest.raises(RuntimeError, match="labels"):
        Fx.lm_head_cross_entropy_pieces(h, w, labels.int(), 300)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        Fx.lm_head_cross_entropy_pieces(h[:, :20], w[:, :20], labels, 300)
    with pytest.raises(RuntimeError, match="frozen"):
        Fx.lm_head_cross_entropy_pieces(h, w.clone().requires_grad_(True), labels, 300)


@pytest.mark.parametrize("m,k,v,piece", [(200, 128, 1000, None), (40, 64, 1000, None), (40, 96, 1001, 512), (300, 768, 50257, 8192),
                                         (2100, 256, 9999, None)])
def test_memory_after_the_vocabulary_is_not_used(m, k, v, piece):
    """The table ends inside a 64-row block: what lies after its rows, NaN here, reaches neither loss nor gradient."""
    h, w, wd, labels = _case(m, k, v, "bf16", seed=9)
    buf = torch.full((v + 300, k), float("nan"), device="cuda", dtype=torch.bfloat16)
    buf[:v] = w
    loss, dh = _check(h, buf[:v], wd, labels, v, piece)
    again, dh2 = _run(h, buf, labels, v, piece)
    assert torch.equal(loss, again) and torch.equal(dh, dh2)


@pytest.mark.parametrize("table", ["bf16", "mx4"])
def test_piece_past_32_bits(table):
    """16,640 rows x 262,144 columns in one piece: 4.36e9 exponentials.  The last rows against the formula."""
    m, k, v, last = 16640, 128, 262144, 40
    h, w, wd, labels = _case(m, k, v, table, seed=12)
    x = h.requires_grad_(True)
    loss = _fx().lm_head_cross_entropy_pieces(x, w, labels, v, v)
    (dh,) = torch.autograd.grad(loss, x)
    n, n_last = int((labels >= 0).sum()), int((labels[-last:] >= 0).sum())
    _, want, room, _ = _exact(h.detach()[-last:], wd, labels[-last:])
    over = (dh[-last:].double() - want * (n_last / n)).abs() - room * (n_last / n)
    assert over.max().item() <= 0, over.max().item()
    assert dh[labels < 0].abs().max().item() == 0.0


def test_two_streams_at_once():
    cases = [_case(m, 128, 3000, "mx4", seed=m) for m in (30, 700)]
    want = [_run(h, w, labels, 3000, 512) for h, w, _, labels in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_run(cases[i][0], cases[i][1], cases[i][3], 3000, 512))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_backward_twice():
    h, w, _, labels = _case(90, 128, 1000, "mx4")
    x = h.requires_grad_(True)
    loss = _fx().lm_head_cross_entropy_pieces(x, w, labels, 1000)
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    (b,) = torch.autograd.grad(loss, x)
    assert torch.equal(a, b)


@pytest.mark.parametrize("m", [1, 5, 300])
@pytest.mark.parametrize("table", ["bf16", "mx4"])
@pytest.mark.parametrize("stride", [0, 8])
def test_rows_that_repeat_or_overlap(m, table, stride):
    """h whose rows are all one row or start 8 elements apart (a one-row h with a row stride below its width, too), and a
    bf16 table whose rows overlap."""
    k, v = 128, 900
    g = torch.Generator(device="cuda").manual_seed(m + stride)
    _, w, wd, labels = _case(m, k, v, table, seed=m, ignore=0.0)
    h = torch.randn((m - 1) * stride + k, device="cuda", generator=g).bfloat16().as_strided((m, k), (stride, 1))
    _check(h, w, wd, labels, v, 512)
    if table == "bf16" and stride:
        w = (torch.randn((v - 1) * stride + k, device="cuda", generator=g) * k ** -0.5).bfloat16().as_strided((v, k), (stride, 1))
        _check(h, w, w.double(), labels, v, 512)


@pytest.mark.parametrize("m,piece", [(6, None), (300, None), (300, 256)])
@pytest.mark.parametrize("table", ["bf16", "mx4"])
def test_sure_rows_of_large_logits(m, piece, table):
    """Rows whose label lies at a logit of 1040, 10 to 22 above every other: the gradient that is left, about 5e-4, keeps its
    precision although an fp32 number of that size has steps of 1.2e-4.  Every number is a small multiple of a power of two,
    so the logits are exact, and what remains of the room is
    - off the label: p rounded to bf16 (2^-8), the exponential of a difference up to 32 (2^-17), the fp32 sum (v 2^-23);
    - at the label 1 - p = 1 - 1 / S: S = 1 + the others' sum, with fewer than 64 additions to a partial sum of about 1 (2^-18);
    - one rounding of the result (2^-8)."""
    k, v = 128, 1500
    g = torch.Generator(device="cuda").manual_seed(m)
    sign = torch.randint(0, 2, (v, k), device="cuda", generator=g) * 2.0 - 1.0
    w = 0.5 * sign
    w[:, 0] = 4.0
    labels = torch.randint(0, v, (m,), device="cuda", generator=g)
    h = (0.25 * sign[labels]).bfloat16()
    h[:, 0] = 256.0
    wd = w.double()
    w = _fx().mx4_quantize(w) if table == "mx4" else w.bfloat16()
    if table == "mx4":
        assert torch.equal(w.dequantize().double(), wd)
    loss, dh = _run(h, w, labels, v, piece)
    logits = h.double() @ wd.t()
    top = logits.gather(1, labels[:, None])
    off = torch.exp(logits - top).scatter(1, labels[:, None], 0.0)
    tail = off.sum(1, keepdim=True)
    assert (tail < 1e-2).all() and (top > 1030).all()
    p, rest = off / (1 + tail), tail / (1 + tail)
    want = (p @ wd - rest * wd[labels]) / m
    room = ((p @ wd.abs()) * (2.0 ** -8 + 2.0 ** -17 + v * 2.0 ** -23) + wd[labels].abs() * (2.0 ** -18 + rest * 2.0 ** -16)) / m
    over = (dh.double() - want).abs() - (room + want.abs() * 2.0 ** -8 + 2.0 ** -133)
    assert over.max().item() <= 0, over.max().item()
    nll = torch.log1p(tail).mean().item()
    assert abs(loss.item() - nll) <= 2.0 ** -18 + 2.0 ** -16 * nll, (loss.item(), nll)


def test_statistics_past_2_gib():
    """300,000 rows x 262,144 columns in one piece, the loss alone: 2.4 GB of tile statistics if the piece stays whole.
    The loss of the last rows, the others being ignored, against the formula."""
    m, k, v, last = 300000, 128, 262144, 40
    h, w, wd, labels = _case(m, k, v, "bf16", seed=14, ignore=0.0)
    labels[:-last] = -100
    loss = _fx().lm_head_cross_entropy_pieces(h, w, labels, v, v)
    want, _, _, room = _exact(h[-last:], wd, labels[-last:])
    assert abs(loss.item() - want.item()) <= room, (loss.item(), want.item(), room)
