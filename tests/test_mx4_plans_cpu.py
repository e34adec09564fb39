"""Which kernel, tile shape and split the sizes of test_mx4_gpu.py reach (no GPU): a refit of the cost model that leaves one of
them without a test shows here."""
import pytest

from test_mx4_gpu import SHAPES, SIZES, SPLIT_16

TILES = [(128, 4), (128, 2), (64, 4), (64, 2), (64, 1), (32, 2), (32, 1)]


@pytest.mark.parametrize("dgrad", [False, True])
def test_every_kernel_has_a_size(dgrad):
    from mobilefinetuner_amd._ext import native
    seen = set()
    for m, n, k in SHAPES + SIZES + SPLIT_16:
        bm, tn, splits, dense = native().mx4_plan(m, n, k, dgrad)
        seen.add("few rows" if bm < 0 else "bf16 copy" if dense else "narrow" if k < 128 else (bm, tn, splits > 1))
    want = {(*t, split) for t in TILES + ([] if dgrad else [(16, 1)]) for split in (False, True)} | {"bf16 copy", "narrow"}
    assert want - seen == set()
    assert dgrad or "few rows" in seen


def test_the_streaming_kernel_has_a_size():
    from mobilefinetuner_amd._ext import native
    assert native().mx4_plan(3, 13003, 128, False)[0] == native().mx4_plan(1, 2097180, 4128, False)[0] == -2
