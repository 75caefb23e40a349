"""Attention of a batch whose sequences share their beginnings refuses on the host what it cannot serve: no GPU needed."""
from __future__ import annotations

import pytest

FAR = [(i + 1) << 40 for i in range(12)]


@pytest.fixture(scope="module")
def ops():
    from rpgbarenginecuda_amd import ops as o

    o.load_library()
    return o


def call(ops, kv=None, table=None, **change):
    kv = kv or ops.GpuPagedKv(FAR[0], FAR[1], shape=(10, 8, 16, 128), kv_type=0)
    table = table or ops.GpuPageTable(FAR[2], shape=(4, 5))
    a = {**dict(lens=FAR[3], rows=FAR[4], pages=FAR[5], q=FAR[6], heads=16, n=3, out=FAR[7], work=FAR[8], seq=None,
                nbytes=1 << 32, groups=2), **change}
    ops.GpuAttentionPagedShared(kv, table, a["lens"], a["rows"], a["pages"], a["q"], a["heads"], a["n"], a["out"], a["work"],
                                seq_ids=a["seq"], workspace_bytes=a["nbytes"], n_groups=a["groups"])


@pytest.mark.parametrize("change,text", [
    (dict(groups=65), "65 groups"), (dict(groups=-1), "-1 groups"), (dict(rows=None), "null groups"),
    (dict(pages=None), "null groups"), (dict(rows=FAR[4] + 2), "4-byte"), (dict(pages=FAR[5] + 1), "4-byte"),
    (dict(heads=15), "15 query heads"), (dict(heads=0), "0 query heads"), (dict(n=-1), "-1 rows"),
    (dict(n=5), "5 rows without seq_ids"), (dict(lens=None), "null"), (dict(q=None), "null"), (dict(out=None), "null"),
    (dict(work=None), "null"), (dict(q=FAR[6] + 4), "16-byte"), (dict(out=FAR[7] + 8), "16-byte"),
    (dict(lens=FAR[3] + 1), "4-byte"), (dict(seq=FAR[9] + 2), "4-byte"), (dict(out=FAR[6] + 16), "must not overlap q"),
    (dict(work=FAR[8] + 16), "256-byte"), (dict(nbytes=1 << 20), "workspace of"), (dict(nbytes=-1), "negative size"),
    (dict(work=FAR[6]), "workspace must not overlap"), (dict(work=FAR[7] - (1 << 20)), "workspace must not overlap"),
    (dict(groups=None), "raw groups need n_groups"), (dict(nbytes=None), "needs workspace_bytes"),
])
def test_refusals(ops, change, text):
    with pytest.raises(ops.RpgError, match=text):
        call(ops, **change)


def test_caches_that_cannot_be_addressed_are_refused(ops):
    for name, value, text in (("head_dim", 96, "neither 64 nor 128"), ("page_size", 8, "power of two"), ("n_pages", 0, "0 pages"),
                              ("k", None, "null")):
        kv = ops.GpuPagedKv(FAR[0], FAR[1], shape=(10, 8, 16, 128), kv_type=0)
        setattr(kv.c, name, value)
        with pytest.raises(ops.RpgError, match=text):
            call(ops, kv)


def test_too_much_for_one_call_is_refused(ops):
    """2^31 units of work that the tables have room for."""
    table = ops.GpuPageTable(FAR[2], shape=(1 << 20, 1 << 24))
    with pytest.raises(ops.RpgError, match="too many for one call"):
        call(ops, table=table, n=3000, nbytes=1 << 38)


def test_no_rows_is_no_work(ops):
    call(ops, n=0)
    call(ops, n=0, groups=0, rows=None, pages=None)


def test_workspace_sizes(ops):
    sizes = [ops.GpuAttentionPagedSharedWorkspace(16, 8, d, n) for d in (64, 128) for n in (0, 1, 100)]
    assert sizes[0] < sizes[1] < sizes[2] and all(s % 16 == 0 for s in sizes)
    assert sizes[3] > ops.GpuAttentionPagedWorkspace(16, 8, 128)
    for heads, kv, d, n in ((16, 8, 96, 1), (16, 0, 128, 1), (15, 8, 128, 1), (0, 8, 128, 1), (16, 8, 128, -1),
                            (16, 8, 128, 1 << 40)):
        with pytest.raises(ops.RpgError):
            ops.GpuAttentionPagedSharedWorkspace(heads, kv, d, n)
