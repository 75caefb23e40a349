"""Groups of a batch that shares its beginnings, as many as there may be, where some lanes of a wave have no row of theirs:
which group a row is of is looked up in all lanes."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8
from test_gpu_attention_shared import attend, batch, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [64, 65, 100, 129, 190])
@pytest.mark.parametrize("kind,heads,n_kv,d", [(F16, 3, 1, 64), (F16, 2, 2, 128), (Q8, 3, 3, 64), (Q8, 6, 1, 128)])
def test_as_many_groups_as_there_may_be(gpu, rows, kind, heads, n_kv, d):
    """Of one row and more, also of rows that have not all of the pages; then the same groups named by others before them."""
    rng = np.random.default_rng(rows + d)
    sizes = np.bincount(np.r_[np.arange(64), rng.integers(0, 64, rows - 64)], minlength=64)
    groups = [(1 + g % 4, [None if (g + i) % 9 == 8 else (g * 7 + i * 5) % 60 for i in range(n)]) for g, n in enumerate(sizes)]
    pages, lens, starts, shared = batch(rng, kind, n_kv, d, 16, groups)
    q = rng.normal(0, 1.2, (rows, heads, d)).astype(np.float32)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    check(got, pages, lens, q)
    # group 0 of no rows in front: numbers move by one, and the last group's rows are by themselves
    check(attend(gpu, kv, table, lens, [0] + starts[:64], [9] + shared[:63], q), pages, lens, q)
