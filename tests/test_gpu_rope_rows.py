"""Rotation of rows at any positions on the GPU against 64 bits: every form, sizes that the vector path takes and ones that
it does not, positions in any order and out of range, in place, captured."""
from __future__ import annotations

import numpy as np
import pytest

from batch_ref import frequencies, rope

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def host(t):
    import torch

    torch.cuda.synchronize()
    return t.cpu().numpy()


def check(got, x, pos, rot, inter, table):
    """Against the rotation by the table's own numbers: two products and a sum, each rounded: 3 units of |a cos| + |b sin|
    (twice the largest of the pair's, rounded up by 1.5 units of each). Copied elements are equal."""
    x = x.astype(np.float64)
    co, si = table[pos, None, :rot // 2].astype(np.float64), table[pos, None, rot // 2:].astype(np.float64)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if inter else (slice(0, rot // 2), slice(rot // 2, rot))
    for at, want, size in ((a, x[..., a] * co - x[..., b] * si, np.abs(x[..., a] * co) + np.abs(x[..., b] * si)),
                           (b, x[..., b] * co + x[..., a] * si, np.abs(x[..., b] * co) + np.abs(x[..., a] * si))):
        assert np.all(np.abs(got[..., at] - want) <= 3 * U * size + 1e-44)
    assert np.array_equal(got[..., rot:], x[..., rot:].astype(np.float32))


CASES = [
    # rows, heads, kv, d, rot, interleaved
    (1, 16, 8, 128, 128, False),
    (1, 1, 0, 8, 8, True),
    (5, 3, 1, 64, 64, True),
    (33, 16, 8, 128, 64, False),
    (33, 16, 8, 128, 64, True),
    (7, 5, 2, 96, 96, False),
    (7, 5, 2, 96, 32, True),
    (9, 4, 4, 128, 8, False),
    (700, 33, 5, 128, 128, True),     # 38 heads: the last group is not whole
    (2811, 16, 8, 128, 128, False),
    (3000, 9, 2, 64, 32, True),
    (2, 2, 1, 1024, 1000, False),
    (4, 3, 2, 128, 2, False),         # from here on one element after the other
    (4, 3, 2, 128, 126, True),
    (31, 3, 2, 62, 62, False),
    (31, 7, 0, 5, 4, True),
    (1000, 3, 1, 100, 50, False),
    (3, 2, 2, 2, 2, True),
    (3, 2, 2, 1023, 1022, True),
]


@pytest.mark.parametrize("n,heads,kv,d,rot,inter", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rows(gpu, n, heads, kv, d, rot, inter, in_place):
    import torch

    rng = np.random.default_rng(n + heads + d + rot)
    rows = 500
    table = gpu.build_rope_table_scaled(rot, 1e4, rows, "yarn", 2.0, 100)
    pos = rng.integers(0, rows, n)
    q = rng.normal(0, 1, (n, heads, d)).astype(np.float32)
    k = (rng.normal(0, 1, (n, kv, d)) * 10.0 ** rng.integers(-3, 4, (n, kv, 1))).astype(np.float32)
    qd, kd = dev(q), dev(k) if kv else None
    qo, ko = (qd, kd) if in_place else (torch.full_like(qd, 7.0), torch.full_like(kd, 7.0) if kv else None)
    gpu.GpuRopeRows(qd, kd, heads, kv, d, rot, inter, dev(table), rows, dev(pos, np.int32), n, qo, ko)
    check(host(qo), q, pos, rot, inter, table)
    if kv:
        check(host(ko), k, pos, rot, inter, table)
        if not in_place:
            assert np.array_equal(host(kd), k)


def test_addresses_that_are_not_16_byte_aligned(gpu):
    import torch

    rng = np.random.default_rng(3)
    n, heads, kv, d, rows = 6, 4, 2, 64, 50
    table = gpu.build_rope_table(d, 1e4, rows)
    pos = rng.integers(0, rows, n)
    q, k = (rng.normal(0, 1, (n, h, d)).astype(np.float32) for h in (heads, kv))
    for at in range(1, 4):
        room = [torch.full((q.size + 8,), 7.0, device="cuda"), torch.full((k.size + 8,), 7.0, device="cuda")]
        qo, ko = room[0][at:at + q.size], room[1][4:4 + k.size]
        gpu.GpuRopeRows(dev(q), dev(k), heads, kv, d, d, True, dev(table), rows, dev(pos, np.int32), n, qo, ko)
        check(host(qo).reshape(q.shape), q, pos, d, True, table)
        check(host(ko).reshape(k.shape), k, pos, d, True, table)
        assert np.all(host(room[0])[:at] == 7) and np.all(host(room[0])[at + q.size:] == 7)


@pytest.mark.parametrize("rot,d", [(64, 128), (126, 130)])
def test_positions_out_of_range(gpu, rot, d):
    """NaN in what would be rotated, there alone; what is copied is copied."""
    rng = np.random.default_rng(4)
    rows = 20
    pos = np.array([0, 19, 20, -1, 2 ** 31 - 1, -2 ** 31, 7])
    fine = (pos >= 0) & (pos < rows)
    table = gpu.build_rope_table(rot, 1e4, rows)
    q = rng.normal(0, 1, (7, 3, d)).astype(np.float32)
    qd = dev(q)
    gpu.GpuRopeRows(qd, None, 3, 0, d, rot, False, dev(table), rows, dev(pos, np.int32), 7, qd, None)
    got = host(qd)
    check(got[fine], q[fine], pos[fine], rot, False, table)
    assert np.all(np.isnan(got[~fine][..., :rot])) and np.array_equal(got[~fine][..., rot:], q[~fine][..., rot:])


def test_half_layout_has_the_one_conversation_operators_bits(gpu):
    rng = np.random.default_rng(5)
    n, heads, d, first = 50, 16, 128, 30
    table = dev(gpu.build_rope_table(d, 1e6, 100))
    a = dev(rng.normal(0, 1, (n, heads, d)).astype(np.float32))
    b = a.clone()
    gpu.GpuRope(a, heads, d, table, first, n)
    gpu.GpuRopeRows(b, None, heads, 0, d, d, False, table, 100, dev(np.arange(first, first + n), np.int32), n, b, None)
    assert np.array_equal(host(a), host(b))


@pytest.mark.parametrize("kind,factor,original", [("none", 1.0, 0), ("linear", 8.0, 0), ("ntk", 4.0, 0), ("yarn", 4.0, 16384)])
@pytest.mark.parametrize("inter", [False, True])
def test_far_positions_of_scaled_frequencies(gpu, kind, factor, original, inter):
    """From the formulas on: the table's entries are off by half a step, and by their angles' last bits."""
    rng = np.random.default_rng(6)
    rows, d, rot = 40000, 128, 96
    table = gpu.build_rope_table_scaled(rot, 1e6, rows, kind, factor, original)
    pos = np.concatenate([[0, 1, rows - 1], rng.integers(0, rows, 40)])
    n = len(pos)
    q = rng.normal(0, 1, (n, 4, d)).astype(np.float32)
    qd = dev(q)
    gpu.GpuRopeRows(qd, None, 4, 0, d, rot, inter, dev(table), rows, dev(pos, np.int32), n, qd, None)
    f, by = frequencies(rot, 1e6, kind, factor, original)
    want = rope(q, pos[:, None] * f, by, rot, inter)
    assert np.all(np.abs(host(qd) - want) <= by * np.abs(q).max() * (8 * U + 16 * 2.0 ** -52 * rows))


def test_infinities_stay_in_their_pair(gpu):
    q = np.ones((2, 2, 64), np.float32)
    q[0, 1, 3] = np.inf
    q[1, 0, 5] = np.nan
    qd = dev(q)
    gpu.GpuRopeRows(qd, None, 2, 0, 64, 64, False, dev(gpu.build_rope_table(64, 1e4, 9)), 9, dev([3, 5], np.int32), 2, qd, None)
    bad = ~np.isfinite(host(qd))
    assert set(zip(*np.nonzero(bad))) == {(0, 1, 3), (0, 1, 35), (1, 0, 5), (1, 0, 37)}


def test_captured(gpu):
    """Positions and rows are read at replay."""
    import torch

    rng = np.random.default_rng(7)
    n, heads, kv, d, rows = 12, 8, 2, 64, 300
    table = gpu.build_rope_table(d, 1e4, rows)
    tab, pos = dev(table), torch.zeros(n, dtype=torch.int32, device="cuda")
    q, k = torch.zeros(n, heads, d, device="cuda"), torch.zeros(n, kv, d, device="cuda")
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        gpu.GpuRopeRows(q, k, heads, kv, d, d, False, tab, rows, pos, n, qo, ko)
    for _ in range(4):
        at = rng.integers(0, rows, n)
        x, y = (rng.normal(0, 1, (n, h, d)).astype(np.float32) for h in (heads, kv))
        for t, a in ((pos, at.astype(np.int32)), (q, x), (k, y)):
            t.copy_(dev(a))
        graph.replay()
        check(host(qo), x, at, d, False, table)
        check(host(ko), y, at, d, False, table)
