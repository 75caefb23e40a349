"""Attention of a batch whose sequences share their beginnings, on the GPU against 64 bits (the bound is paged_ref.bound's:
queries count to 2^-22 of each element and weights to 2^-22 of theirs, less than what it allows for either)."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8, Pages, attention, attention_within, bound

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def host(t):
    import torch

    torch.cuda.synchronize()
    return t.cpu().numpy()


def workspace(gpu, heads, n_kv, d, rows):
    import torch

    return torch.zeros(gpu.GpuAttentionPagedSharedWorkspace(heads, n_kv, d, rows), dtype=torch.uint8, device="cuda")


def batch(rng, kind, n_kv, d, page, groups, k_amp=1.0):
    """Groups of (shared pages, own lengths): pages, lengths, where groups begin, what they share. A length of None is a
    row of no positions at all."""
    lens, starts, shared = [], [0], []
    for pages_of, own in groups:
        lens += [0 if n is None else pages_of * page + n for n in own]
        starts.append(len(lens))
        shared.append(pages_of)
    p = Pages(rng, kind, n_kv, d, page, lens, width=1 + max([1] + [-(-n // page) for n in lens]))
    for g, n in enumerate(shared):
        held = [r for r in range(starts[g], starts[g + 1]) if lens[r] >= n * page and n]
        for r in held[1:]:
            p.table[r, :n] = p.table[held[0], :n]
    p.fill_random(rng, lens, k_amp)
    return p, lens, starts, shared


def attend(gpu, kv, table, lens, starts, shared, q, work=None, seq_ids=None, fill=np.nan, least=0):
    import torch

    n, heads, d = q.shape
    out = torch.full((n, heads, d), fill, dtype=torch.float32, device="cuda")
    work = workspace(gpu, heads, kv.n_kv_heads, d, n) if work is None else work
    gpu.GpuAttentionPagedShared(kv, table, dev(lens, np.int32), dev(starts, np.int32), dev(shared, np.int32), dev(q), heads,
                                n, out, work, seq_ids=None if seq_ids is None else dev(seq_ids, np.int32), least_saving=least)
    return host(out)


def check(got, pages, lens, q, seqs=None, look=None):
    for r in range(len(lens)) if look is None else look:
        seq, n = r if seqs is None else seqs[r], lens[r]
        if n == 0:
            assert np.all(got[r] == 0), r
            continue
        want, smag, vmax = attention(q[r], pages.rows("k", seq, n), pages.rows("v", seq, n))
        err = np.abs(got[r] - want).max(-1)
        limit = bound(pages.d, n, smag, vmax)
        assert np.all(err <= limit), (r, n, float((err / limit).max()))


OWN = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, None, 255, 300]
CASES = [
    # kind, heads, n_kv, d, page, groups of (shared pages, own lengths)
    (F16, 16, 8, 128, 16, [(1, [0, 1])]),
    (F16, 16, 8, 128, 16, [(24, [116, 3])]),
    (Q8, 16, 8, 128, 16, [(24, [116, 3])]),
    (F16, 2, 2, 64, 16, [(7, [5])]),                      # one row, one column
    (F16, 32, 4, 64, 16, [(63, OWN)]),                    # 144 columns: a second tile of 16
    (Q8, 32, 8, 128, 64, [(5, OWN)]),                     # 72
    (F16, 16, 8, 128, 32, [(9, OWN)]),                    # 36
    (Q8, 8, 8, 64, 256, [(3, OWN[:15])]),                 # 15
    (F16, 4, 4, 128, 128, [(2, OWN)]),                    # 18
    (Q8, 15, 3, 128, 16, [(8, OWN), (1, OWN[::-1])]),     # groups of 5 heads, 90 columns
    (F16, 33, 1, 128, 16, [(11, OWN[:7])]),               # 231
    (Q8, 24, 2, 64, 16, [(65, OWN)]),
    (F16, 7, 1, 64, 32, [(3, [9]), (4, [0]), (1, [None]), (10, [70, 0, 5])]),
    (Q8, 4, 2, 128, 32, [(0, [40, 3]), (2, [10, 11]), (7, [1] * 5)]),   # a group that shares nothing
    (F16, 8, 2, 128, 16, [(1 + g % 9, [g % 40, (3 * g) % 50][:1 + g % 2]) for g in range(64)]),
    (Q8, 2, 1, 64, 16, [(40, [(7 * i) % 90 for i in range(300)])]),     # 600 columns
    (F16, 4, 4, 64, 32, [(20, [(5 * i) % 33 for i in range(130)]), (0, [9] * 80), (33, [None, 4] * 20)]),
    (F16, 4, 2, 128, 64, [(300, [10, 400, 0])]),          # 19200 positions: many parts of a tile
    (Q8, 32, 8, 128, 64, [(120, [5, 700, 64, 0])]),
    (Q8, 1, 1, 128, 256, [(100, [1, 2])]),
    (F16, 8, 1, 64, 16, [(2001, [3] * 9)]),
]


@pytest.mark.parametrize("kind,heads,n_kv,d,page,groups", CASES)
def test_against_64_bits(gpu, kind, heads, n_kv, d, page, groups):
    rng = np.random.default_rng(heads * 100 + d + len(groups))
    pages, lens, starts, shared = batch(rng, kind, n_kv, d, page, groups)
    q = rng.normal(0, 1.5, (len(lens), heads, d)).astype(np.float32)
    kv, table = pages.device(gpu)
    work = workspace(gpu, heads, n_kv, d, len(lens))
    got = attend(gpu, kv, table, lens, starts, shared, q, work)
    assert np.all(np.isfinite(got))
    look = None if sum(lens) <= 150_000 else sorted({0, len(lens) - 1, *(int(r) for r in rng.choice(len(lens), 12))})
    check(got, pages, lens, q, look=look)
    assert np.array_equal(got, attend(gpu, kv, table, lens, starts, shared, q, work))  # parts are joined in one order


def test_without_groups_it_is_the_other_operator(gpu):
    import torch

    rng = np.random.default_rng(1)
    pages, lens, _, _ = batch(rng, F16, 2, 128, 16, [(3, [5, 6, 100])])
    q = rng.normal(0, 1, (3, 4, 128)).astype(np.float32)
    kv, table = pages.device(gpu)
    out = torch.zeros(3, 4, 128, device="cuda")
    work = workspace(gpu, 4, 2, 128, 3)
    gpu.GpuAttentionPaged(kv, table, dev(lens, np.int32), dev(q), 4, 3, out, work)
    want = host(out)
    assert np.array_equal(attend(gpu, kv, table, lens, [0], [], q, work), want)
    # groups in which no row takes part
    for starts, shared in (([0, 3], [0]), ([0, 3], [-1]), ([0, 3], [99]), ([0, 3], [2 ** 31 - 1]), ([0, 0], [2]),
                           ([3, 3], [2]), ([2, 1], [2]), ([5, 9], [2]), ([-9, 0], [2]), ([0, 3], [pages.table.shape[1]])):
        assert np.array_equal(attend(gpu, kv, table, lens, starts, shared, q, work), want), (starts, shared)


@pytest.mark.parametrize("kind,d", [(F16, 128), (F16, 64), (Q8, 128), (Q8, 64)])
def test_rows_and_groups_out_of_range(gpu, kind, d):
    """Padding, rows that do not reach behind the shared pages or lie in no group, bad lengths and sequences, a group's
    first rows among them; groups that overlap or reach past the rows."""
    rng = np.random.default_rng(2)
    n_kv, heads, page = 2, 6, 16
    pages, lens, _, _ = batch(rng, kind, n_kv, d, page, [(6, [30, 40, 50, 60]), (4, [33, 0, 8])])
    high, low = 2 ** 31 - 1, -2 ** 31
    # rows ask for these sequences and lengths
    seqs = [-1, 99, 0, 1, 2, 3, 0, low, 3, 4, 5, 6, 4, high, 1]
    ask = [50, 50, 90, -1, lens[2], 96, 96 + 30, 50, high, 64 + 33, 64, 0, 63, 5, 96 + 40]
    want = ["pad", "nan", "good", "nan", "good", "good", "good", "pad", "nan", "good", "good", "good", "good", "nan", "good"]
    kv, table = pages.device(gpu)
    n = len(seqs)
    q = rng.normal(0, 1, (n, heads, d)).astype(np.float32)
    work = workspace(gpu, heads, n_kv, d, n)
    for starts, shared in (([0, 9, 14], [6, 4]), ([-5, 9, 14, 90], [6, 4, 6]), ([0, 9, 9, 14, 15], [6, 3, 4, 6]),
                           ([1, 7, 13, 20], [6, 0, 6]), ([0, 5, 9, 3], [6, 6, 4])):
        got = attend(gpu, kv, table, ask, starts, shared, q, work, seqs, fill=7.0)
        for r in range(n):
            if want[r] == "pad":
                assert np.all(got[r] == 7), r
            elif want[r] == "nan":
                assert np.all(np.isnan(got[r])), r
            else:
                check(got[r:r + 1], pages, ask[r:r + 1], q[r:r + 1], seqs[r:r + 1])


def test_a_row_of_several_groups_is_of_the_first(gpu):
    rng = np.random.default_rng(3)
    pages, lens, _, _ = batch(rng, F16, 1, 64, 16, [(5, [9, 10, 11, 12])])
    q = rng.normal(0, 1, (4, 2, 64)).astype(np.float32)
    kv, table = pages.device(gpu)
    # group 1 is rows [2, 2): none; group 2 begins inside group 0
    got = attend(gpu, kv, table, lens, [0, 4, 2, 4], [5, 3, 3], q)
    check(got, pages, lens, q)
    assert np.array_equal(got, attend(gpu, kv, table, lens, [0, 4], [5], q))


@pytest.mark.parametrize("kind,d", [(F16, 128), (F16, 64), (Q8, 128), (Q8, 64)])
def test_bad_pages(gpu, kind, d):
    """Among the shared ones: NaN for the group; behind them: for the row. Nothing is read there."""
    rng = np.random.default_rng(4)
    n_kv, heads, page = 2, 4, 16
    pages, lens, starts, shared = batch(rng, kind, n_kv, d, page, [(20, [30, 5, 0]), (12, [9, 40, 20]), (3, [8, 9])])
    keep = pages.table.copy()
    for bad in (-1, pages.n_pages, 2 ** 31 - 1, -2 ** 31):
        pages.table = keep.copy()
        pages.table[0:3, 13] = bad
        pages.table[4, 13] = bad   # the second page that is row 4's own
        kv, table = pages.device(gpu)
        q = rng.normal(0, 1, (len(lens), heads, d)).astype(np.float32)
        got = attend(gpu, kv, table, lens, starts, shared, q)
        assert np.all(np.isnan(got[[0, 1, 2, 4]]))
        check(got[[3, 5, 6, 7]], pages, [lens[r] for r in (3, 5, 6, 7)], q[[3, 5, 6, 7]], [3, 5, 6, 7])


def test_a_group_reads_its_first_rows_table(gpu):
    """The tables of the others are not looked at where they name the shared pages: they may hold anything there."""
    rng = np.random.default_rng(5)
    pages, lens, starts, shared = batch(rng, Q8, 2, 64, 16, [(9, [None, 20, 30, 40])])
    q = rng.normal(0, 1, (4, 4, 64)).astype(np.float32)
    good = pages.table.copy()
    pages.table[2:, :9] = -7
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    pages.table = good
    check(got, pages, lens, q)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_where_sharing_does_not_pay(gpu, kind):
    """Where not even a full table would save what is asked for, the call is that of rows by themselves; where the groups do
    not, which the device finds, their rows are by themselves; a byte less asked for, and they share, which shows in what
    pages out of range reach."""
    import torch

    rng = np.random.default_rng(12)
    n_kv, d, page, heads = 2, 64, 16, 4
    cell = 2 * n_kv * page * (2 * d if kind == F16 else d + 4)
    pages, lens, starts, shared = batch(rng, kind, n_kv, d, page, [(9, [20, 30, 40]), (5, [7, 60])])
    q = rng.normal(0, 1, (5, heads, d)).astype(np.float32)
    saving = (2 * 9 + 1 * 5) * cell
    good = pages.table.copy()
    pages.table[1, 3] = pages.table[4, 2] = -1
    kv, table = pages.device(gpu)
    out = torch.zeros(5, heads, d, device="cuda")
    gpu.GpuAttentionPaged(kv, table, dev(lens, np.int32), dev(q), heads, 5, out, workspace(gpu, heads, n_kv, d, 5))
    alone = host(out)
    assert np.isnan(alone[[1, 4]]).all() and np.isfinite(alone[[0, 2, 3]]).all()
    for least in (-1, 1 << 62):
        assert np.array_equal(attend(gpu, kv, table, lens, starts, shared, q, least=least), alone, equal_nan=True), least
    found = attend(gpu, kv, table, lens, starts, shared, q, least=saving + 1)
    together = attend(gpu, kv, table, lens, starts, shared, q, least=saving)
    pages.table = good
    assert np.array_equal(np.isnan(found), np.isnan(alone))
    check(found, pages, lens, q, look=[0, 2, 3])
    check(together, pages, lens, q)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_magnitudes(gpu, kind):
    """Queries and keys that make one position take everything, or all count alike, on either side of where the shared part
    ends; tiny, huge and zero queries; each element held to the weighted magnitudes that it is made of."""
    rng = np.random.default_rng(6)
    n_kv, d, page, heads = 2, 128, 32, 4
    pages, lens, starts, shared = batch(rng, kind, n_kv, d, page, [(9, [40, 300, 1, 0, 64, 100])], k_amp=3.0)
    for i, pos in enumerate(rng.permutation(288)[:100]):
        pages.put(0, pos, rng.normal(0, 1, (n_kv, d)).astype(np.float32),
                  rng.normal(0, 10.0 ** (i % 7 - 4), (n_kv, d)).astype(np.float32))
    q = rng.normal(0, 1, (6, heads, d)).astype(np.float32)
    q[0] *= 20
    q[1] *= np.float32(1e-42)
    q[2] = 0
    q[3] *= np.float32(1e-20)
    q[3, 1, :] = 0
    q[3, 1, 7] = 5
    q[4, :, ::2] *= np.float32(1e-6)
    q[5, 2] *= np.float32(1e4) if kind == Q8 else 200
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    check(got, pages, lens, q)
    for r in range(6):
        if r == 1 or (r == 5 and kind == Q8):
            continue  # subnormal queries count relative to the smallest number; scores of 10^5 are off by whole units
        want, limit = attention_within(q[r], pages.rows("k", r, lens[r]), pages.rows("v", r, lens[r]), kind)
        assert np.all(np.abs(got[r] - want) <= limit), (r, float((np.abs(got[r] - want) / limit).max()))


@pytest.mark.parametrize("d", [64, 128])
def test_value_scales_of_any_size(gpu, d):
    """8-bit value rows from 1e-30 to 1e30, and keys: three terms of a weight times its row's scale have fp32's range."""
    rng = np.random.default_rng(7)
    page = 16
    pages, lens, starts, shared = batch(rng, Q8, 1, d, page, [(12, [30, 5]), (4, [0, 70]), (4, [3, 3])])
    for g, amp in ((0, None), (2, 1e-30), (4, 1e30)):
        for pos in range(lens[g + 1] if g == 0 else lens[g]):
            a = 10.0 ** rng.integers(-30, 30) if amp is None else amp
            pages.put(g, pos, rng.normal(0, 1, (1, d)).astype(np.float32), (a * rng.normal(0, 1, (1, d))).astype(np.float32))
    pages.put(2, 63, rng.normal(0, 1, (1, d)).astype(np.float32), np.zeros((1, d), np.float32))
    q = rng.normal(0, 1, (6, 2, d)).astype(np.float32)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    for r in range(6):
        want, limit = attention_within(q[r], pages.rows("k", r, lens[r]), pages.rows("v", r, lens[r]), Q8)
        assert np.all(np.abs(got[r] - want) <= limit), (r, float((np.abs(got[r] - want) / limit).max()))


@pytest.mark.parametrize("kind", [F16, Q8])
def test_what_is_no_number(gpu, kind):
    """In a query: its head's. In a shared row: whoever attends to it. In slots that nobody has: nobody's."""
    rng = np.random.default_rng(8)
    d, page = 128, 16
    pages, lens, starts, shared = batch(rng, kind, 2, d, page, [(9, [20, 21]), (3, [1, 0])])
    q = rng.normal(0, 1, (4, 4, d)).astype(np.float32)
    q[0, 1, 5] = np.inf
    q[1, 2, 6] = np.nan
    bad = np.ones((2, d), np.float32)
    bad[1, 3] = np.nan
    pages.put(2, 40, np.ones((2, d), np.float32), bad)  # values of the second kv head
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    assert np.all(np.isnan(got[0, 1])) and np.all(np.isfinite(got[0, [0, 2, 3]]))
    assert np.all(np.isnan(got[1, 2])) and np.all(np.isfinite(got[1, [0, 1, 3]]))
    assert np.all(np.isfinite(got[2:, :2])) and np.all(np.isnan(got[2:, 2:, 3]))
    if kind == F16:
        assert np.all(np.isfinite(np.delete(got[2:, 2:], 3, 2)))
    for r, h in ((0, 0), (0, 3), (1, 0), (1, 3)):
        want, smag, vmax = attention(q[r], pages.rows("k", r, lens[r]), pages.rows("v", r, lens[r]))
        assert np.all(np.abs(got[r, h] - want[h]) <= bound(d, lens[r], smag, vmax)[h])


def test_keys_of_minus_infinite_score(gpu):
    """Of every shared position, with the row's own to attend to, and without (nothing to attend to: NaN)."""
    rng = np.random.default_rng(9)
    d, page = 64, 16
    pages, lens, starts, shared = batch(rng, F16, 1, d, page, [(9, [20, 0, 4])])
    for pos in range(9 * page):
        p, s = pages.slot(0, pos)
        pages.k.view(np.float16)[p, 0, s] = 0
        pages.k.view(np.float16)[p, 0, s, 3] = np.float16(-65504)
    q = np.zeros((3, 1, d), np.float32)
    q[:, :, 3] = 1e36
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    assert np.all(np.isnan(got[1]))
    for r in (0, 2):
        k, v = (pages.rows(name, r, lens[r])[9 * page:] for name in "kv")
        best = k[:, 0, 3].argmax()  # scores of 10^35 apart: one takes all
        assert np.all(got[r, 0] == v[best, 0].astype(np.float32))


def test_own_keys_of_minus_infinite_score(gpu):
    """Of every own position: what is shared is attended to alone; with no weight in either, NaN."""
    rng = np.random.default_rng(13)
    d, page = 64, 16
    pages, lens, starts, shared = batch(rng, F16, 1, d, page, [(9, [20, 0, 200])])
    for r in (0, 2):
        for pos in range(9 * page, lens[r]):
            p, s = pages.slot(r, pos)
            pages.k.view(np.float16)[p, 0, s] = 0
            pages.k.view(np.float16)[p, 0, s, 3] = -np.inf
    q = np.abs(rng.normal(0, 1, (3, 2, d))).astype(np.float32) + np.float32(0.01)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, starts, shared, q)
    check(got, pages, [9 * page] * 3, q)
    pages.k[pages.table[0, :9]] = pages.k[pages.table[0, 9]][:, :1]
    kv, table = pages.device(gpu)
    assert np.all(np.isnan(attend(gpu, kv, table, lens, starts, shared, q)))


@pytest.mark.parametrize("kind,d", [(F16, 128), (Q8, 64)])
def test_captured(gpu, kind, d):
    """A captured call holds for any groups, lengths and rows at replay; eager calls between the replays agree."""
    import torch

    rng = np.random.default_rng(10)
    n_kv, heads, page = 2, 8, 32
    pages, lens0, _, _ = batch(rng, kind, n_kv, d, page, [(40, [700, 300, 64, 100]), (10, [500, 0, 31])])
    kv, table = pages.device(gpu)
    n = len(lens0)
    work, other = workspace(gpu, heads, n_kv, d, n), workspace(gpu, heads, n_kv, d, n)
    lens, starts, shared = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (n, 3, 2))
    q, out = torch.zeros(n, heads, d, device="cuda"), torch.zeros(n, heads, d, device="cuda")
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        gpu.GpuAttentionPagedShared(kv, table, lens, starts, shared, q, heads, n, out, work, least_saving=0)
    for ask, where, what in ((lens0, [0, 4, 7], [40, 10]), (lens0, [0, 4, 7], [1, 2]), ([1] * n, [0, 4, 7], [40, 10]),
                             (lens0, [0, 2, 2], [33, 0]), ([0] * n, [0, 4, 7], [40, 10]), (lens0, [0, 4, 7], [40, 10])):
        x = rng.normal(0, 1, (n, heads, d)).astype(np.float32)
        for t, a in ((lens, np.int32(ask)), (starts, np.int32(where)), (shared, np.int32(what)), (q, x)):
            t.copy_(dev(a))
        eager = attend(gpu, kv, table, ask, where, what, x, other)
        graph.replay()
        got = host(out)
        check(got, pages, ask, x)
        assert np.array_equal(got, eager)


def test_pages_past_32_bit_offsets(gpu):
    """A group whose pages start past 2^32 elements of the pool; one of its sequences has two rows."""
    import torch

    rng = np.random.default_rng(30)
    n_kv, d, page, heads = 8, 128, 256, 16
    few, lens, starts, shared = batch(rng, Q8, n_kv, d, page, [(3, [5, 300])])
    n_pages = (1 << 32) // (n_kv * d * page) + few.n_pages
    far = n_pages - few.n_pages
    k, v = (torch.zeros((n_pages, n_kv, page, d), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((n_pages, n_kv, page), device="cuda") for _ in range(2))
    for big, small in ((k, few.k), (v, few.v), (ks, few.ks), (vs, few.vs)):
        big[far:] = dev(small)
    kv, table = gpu.GpuPagedKv(k, v, ks, vs), gpu.GpuPageTable(dev(few.table + far, np.int32))
    q = rng.normal(0, 1, (3, heads, d)).astype(np.float32)
    lens, seqs = [lens[0], lens[1], lens[1] - 7], [0, 1, 1]
    check(attend(gpu, kv, table, lens, [0, 3], shared, q, seq_ids=seqs), few, lens, q, seqs)


def test_two_streams_at_once(gpu):
    import torch

    rng = np.random.default_rng(11)
    heads, n_kv, d = 8, 4, 128
    pages, lens, starts, shared = batch(rng, Q8, n_kv, d, 32, [(100, [300, 1, 64]), (30, [5, 900])])
    kv, table = pages.device(gpu)
    n, a, b = dev(lens, np.int32), dev(starts, np.int32), dev(shared, np.int32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [dev(rng.normal(0, 1, (5, heads, d)).astype(np.float32)) for _ in streams]
    works = [workspace(gpu, heads, n_kv, d, 5) for _ in streams]
    outs = [[torch.zeros_like(qs[0]) for _ in range(4)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(4):
        for s, q, w, o in zip(streams, qs, works, outs):
            with gpu.ScopedEngineStream(s):
                gpu.GpuAttentionPagedShared(kv, table, n, a, b, q, heads, 5, o[i], w, least_saving=0)
    torch.cuda.synchronize()
    for q, o in zip(qs, outs):
        check(host(o[0]), pages, lens, host(q))
        assert all(np.array_equal(host(x), host(o[0])) for x in o)


def test_one_workspace_for_calls_of_all_sizes(gpu):
    """Between calls with fewer rows, other groups, and the plain operator's on the same workspace."""
    import torch

    rng = np.random.default_rng(12)
    heads, n_kv, d = 4, 2, 128
    work = workspace(gpu, heads, n_kv, d, 40)
    for groups in ([(50, [9] * 40)], [(3, [70])], [(200, [4, 3000])], [(0, [5])], [(7, [None, 3]), (90, [1] * 30)]):
        pages, lens, starts, shared = batch(rng, F16, n_kv, d, 16, groups)
        q = rng.normal(0, 1, (len(lens), heads, d)).astype(np.float32)
        kv, table = pages.device(gpu)
        check(attend(gpu, kv, table, lens, starts, shared, q, work), pages, lens, q)
        out = torch.zeros(len(lens), heads, d, device="cuda")
        gpu.GpuAttentionPaged(kv, table, dev(lens, np.int32), dev(q), heads, len(lens), out, work)
        check(host(out), pages, lens, q)
