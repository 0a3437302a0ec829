"""A schedule of units keeps min_chunk_keys: no request is cut into shorter items."""
import random

import numpy as np
import pytest

from test_serving_cpu import _lib, _units


def _cuts_hold(items, iptr, lens, least):
    for b, n in enumerate(lens):
        rows = items[iptr[b]:iptr[b + 1]]
        sizes = rows[:, 2] - rows[:, 1]
        assert sizes.sum() == n
        assert len(rows) == 0 or sizes.min() >= min(least, n), (b, n, sizes.tolist())


@pytest.mark.parametrize("seed", range(60))
def test_units_keep_the_least_item(seed):
    ffi, lib = _lib()
    g = random.Random(seed)
    page, hkv = g.choice([16, 32, 64, 128, 256]), g.choice([1, 2, 8, 40, 400])
    least, top = g.choice([65, 100, 500, 3000, 8192]), g.choice([300, 5000, 30000, 200000])
    lens = [0 if g.random() < 0.1 else g.randint(1, top) for _ in range(g.choice([1, 2, 5, 40, 300]))]
    items, iptr = _units(ffi, lib, lens, page, hkv, 0, least)
    _cuts_hold(items, iptr, lens, least)
    units = int((items[:, 3] > 0).sum())
    first = items[:units, 3] - 1
    for lo, hi in zip(first, np.append(first[1:], len(items))):
        assert 1 <= hi - lo <= 32
        assert sum((r[2] - 1) // page - r[1] // page + 1 for r in items[lo:hi]) <= 1024


@pytest.mark.parametrize("page", [16, 64])
def test_units_of_long_items(page):
    """The schedule that the long-ring test on the GPU runs: over a hundred stages."""
    ffi, lib = _lib()
    lens = [9000, 13011, 77, 4032]
    items, iptr = _units(ffi, lib, lens, page, 2, 0, 8192)
    _cuts_hold(items, iptr, lens, 8192)
    stages = -(-(items[:, 2] - items[:, 1]) // 64)
    assert stages.max() >= 200
