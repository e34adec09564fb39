"""The columns of a piece of lm_head_cross_entropy_pieces (no GPU)."""
import itertools

import pytest

VOCABULARIES = (1, 257, 50257, 262144, 40_000_000, (1 << 30) - 1)
PIECES = (0, 256, 4096, 262144, 1 << 24, (1 << 30) - 256)


@pytest.mark.parametrize("m", [1, 2, 191, 4096, 300000, 1 << 24])
def test_pieces_fit_the_kernels_offsets(m):
    """E rows at most 2^21 columns (256 of them, and 32-bit byte offsets inside, stay under 2 GiB) and the statistics of all
    rows, 8 bytes a 256-column tile, under 2 GiB; never wider than asked for or than the vocabulary."""
    from mobilefinetuner_amd._ext import native
    for v, piece in itertools.product(VOCABULARIES, PIECES):
        w = native().lm_head_ce_pieces_width(m, v, piece)
        assert w >= 256 and w % 256 == 0 and w <= (v + 255) // 256 * 256, (v, piece, w)
        assert w <= 1 << 21 and m * (w // 256) * 8 < 1 << 31, (v, piece, w)
        if piece:
            assert w <= piece, (v, piece, w)
            if piece <= 1 << 21 and m * (piece // 256) * 8 < 1 << 31:
                assert w == min(piece, (v + 255) // 256 * 256), (v, piece, w)
