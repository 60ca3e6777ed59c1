"""Sizes of the streamed loss's slots: a part of a cut output tile is 256 x 256 fp32 numbers, what a pair of CTAs accumulates."""
import pytest

import _native as N

SLOT = 256 * 256


@pytest.mark.parametrize('rows,V,d,piece,dh,dw', [
    (1, 32000, 768, 32000 // 256 * 256 + 256, 72, 0),     # dh: one row tile x 3 column tiles, 24 parts each; dw: one k-block, not cut
    (32768, 32000, 768, 16384, 70, 220),                  # two pieces: the larger need of the two
    (7, 32000, 768, 1 << 20, 72, 0),
])
def test_slots_hold_every_part_of_a_cut_tile(rows, V, d, piece, dh, dw):
    count = lambda a, b: N.lib().ulm_streamed_ce_slots(rows, V, d, piece, a, b)          # noqa: E731
    assert count(0, 0) == 0
    for want, n in ((dh, count(1, 0)), (dw, count(0, 1)), (dh + dw, count(1, 1))):
        assert n % SLOT == 0 and n // SLOT == want
