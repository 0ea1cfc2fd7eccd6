"""The plan of a product's tiles (csrc/nt_plan.hpp), on the CPU: what it promises of every size, and that the sizes of the
GPU tests take every tile, split and cut there is."""
import random

import pytest

from tests import test_int8_gpu, test_readout_train_gpu
from tests.tile_plan import LARGE, MEDIUM, SMALL, int8_product, plan, readout, whole_rounds

ROWS = {SMALL: 64, MEDIUM: 128, LARGE: 256}
COLS = {SMALL: 128, MEDIUM: 128, LARGE: 256}


def sizes(n, seed):
    rng = random.Random(seed)
    size = lambda most: int(2 ** rng.uniform(0, most))  # noqa: E731
    return [(size(16), size(18), 16 * size(13)) for _ in range(n)]


def test_splits_cover_k():
    for m, n, kb in sizes(3000, 1):
        for split in (False, True):
            _, per, splits = plan(m, n, kb, split)
            assert per % 64 == 0 and 1 <= splits <= 64
            assert splits * per >= kb > (splits - 1) * per or splits == 1
            assert splits == 1 or (split and per >= 512)


def test_few_tiles_are_split():
    """Where a product's tiles are a sixteenth of the CUs and less, k of 2048 bytes or more is split: as many parts as have
    512 bytes, at most 64 and four workgroups a CU, or fewer."""
    seen = 0
    for m, n, kb in sizes(20000, 2):
        tiles = -(-m // 64) * -(-n // 128)
        if tiles <= 16 and kb >= 2048:
            _, _, splits = plan(m, n, kb, True)
            assert 2 <= splits <= kb // 512, (m, n, kb, splits)
            seen += 1
    assert seen > 200
    for m, n, k in ((64, 1000, 8192), (16, 256, 16384), (5, 40, 20000), (64, 2048, 4096)):
        assert int8_product(m, n, k)[1] >= 8


def test_whole_rounds_leave_a_rest():
    for m, n, kb in sizes(3000, 3):
        c = whole_rounds(m, n, kb)
        assert c == 0 or (0 < c < n and c % 256 == 0 and plan(m, n, kb, False)[0] == LARGE)


def test_int8_sizes_take_every_plan():
    taken = {(size, splits > 1) for size, splits in (int8_product(*p) for p in test_int8_gpu.PLANS)}
    assert taken == {(t, s) for t in (SMALL, MEDIUM, LARGE) for s in (False, True)}
    assert any(m % ROWS[LARGE] and n % COLS[LARGE] and int8_product(m, n, k) == (LARGE, 1) for m, n, k in test_int8_gpu.PLANS)


def test_readout_sizes_take_every_plan():
    logits, hidden, weight, cuts = set(), set(), set(), set()
    for rows, V, d, _, layout, _ in test_readout_train_gpu.PLANS:
        l, h, w = readout(rows, V, d, layout)
        logits.add(l[0])
        hidden.add((h[0], h[1] > 1))
        weight.add((w[0], w[1] > 1))
        if w[2]:
            cuts.add(layout)
    both = {(t, s) for t in (SMALL, MEDIUM, LARGE) for s in (False, True)}
    assert logits == {SMALL, MEDIUM, LARGE} and hidden == both and weight == both and cuts == {"dv", "vd"}


@pytest.mark.parametrize("rows,V,d,few", test_readout_train_gpu.TILES_OF_ROWS)
def test_rows_compared_are_scored_by_different_tiles(rows, V, d, few):
    full, part = readout(rows, V, d, "vd")[0], readout(few, V, d, "vd")[0]
    assert full != part, (full, part)
