"""Whether a batch shares its beginnings, at the border that callers get and at borders of any size: told by a page out of
range in the table of a row that is not its group's first, which is looked at only where rows are by themselves."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8, Pages, attention_within
from test_gpu_attention_shared import attend

pytestmark = pytest.mark.gpu


def behind(rng, kind, n_kv, d, page, n):
    """Two sequences of the same n pages, of a few physical ones again and again; the second's table without its fourth."""
    pages = Pages(rng, kind, n_kv, d, page, [5 * page], spare=0)
    pages.fill_random(rng, [5 * page])
    pages.table = np.repeat(pages.table[0][rng.integers(0, 5, n)][None], 2, 0)
    good = pages.table[0].copy()
    pages.table[1, 3] = -1
    return pages, good


@pytest.mark.parametrize("padding", [0, 30])
@pytest.mark.parametrize("kind,enough", [(F16, lambda rows: 144 + rows), (Q8, lambda rows: -((144 + rows << 20) // -540672))])
def test_the_default_border(gpu, kind, enough, padding):
    """144 MB and one for each row, padding too, of pages of 1 MB (fp16) or 540672 bytes (8 bits: 256 positions of 8 heads'
    keys and values of 128 + 4)."""
    rng = np.random.default_rng(padding)
    n_kv, heads, d, page = 8, 16, 128, 256
    rows = 2 + padding
    for n, together in ((enough(rows), True), (enough(rows) - 1, False)):
        pages, good = behind(rng, kind, n_kv, d, page, n)
        kv, table = pages.device(gpu)
        q = rng.normal(0, 1, (rows, heads, d)).astype(np.float32)
        got = attend(gpu, kv, table, [n * page] * rows, [0, 2], [n], q, seq_ids=[0, 1] + [-1] * padding, fill=7.0, least=-1)
        assert np.all(got[2:] == 7)
        assert np.all(np.isfinite(got[0])) and np.all(np.isfinite(got[1]) if together else np.isnan(got[1])), n
        pos, h = np.arange(n * page), 5
        p, s = good[pos // page], pos % page
        k, v = ((x[p, h, s].view(np.float16).astype(np.float64) if kind == F16 else
                 x[p, h, s].astype(np.float64) * sc[p, h, s].astype(np.float64)[:, None])
                for x, sc in ((pages.k, pages.ks), (pages.v, pages.vs)))
        for r in range(2 if together else 1):
            want, limit = attention_within(q[r, 2 * h:2 * h + 2], k[:, None], v[:, None], kind)
            assert (np.abs(got[r, 2 * h:2 * h + 2] - want) / limit).max() <= 1, (n, r)


@pytest.mark.parametrize("rows", [4097, (1 << 19) + 1])
def test_borders_past_32_bits(gpu, rows):
    """As many rows by 8192 pages of 4 KB: a border of just what they save, a byte more, and any that is larger."""
    rng = np.random.default_rng(rows)
    n, page, d = 8192, 16, 64
    pages, _ = behind(rng, F16, 1, d, page, n + 10)
    kv, table = pages.device(gpu)
    q = rng.normal(0, 1, (rows, 1, d)).astype(np.float32)
    lens = np.full(rows, 1)
    lens[:2] = n * page
    saving = (rows - 1) * n * 4096
    for least, together in ((saving, True), (saving + 1, False), ((1 << 63) - 1, False), (saving - 1, True)):
        got = attend(gpu, kv, table, lens, [0, rows], [n], q, seq_ids=np.arange(rows) % 2, least=least)
        assert np.isfinite(got[1]).all() == together and np.isfinite(got[2:]).all() and np.isfinite(got[0]).all(), least
