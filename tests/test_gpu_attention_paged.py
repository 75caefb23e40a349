"""Attention of one token per row over the paged cache on the GPU, against 64 bits (the bound is derived at
paged_ref.bound)."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8, Pages, attention, bound

pytestmark = pytest.mark.gpu


def dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def host(t):
    import torch

    torch.cuda.synchronize()
    return t.cpu().numpy()


def workspace(gpu, heads, n_kv, d):
    import torch

    return torch.zeros(gpu.GpuAttentionPagedWorkspace(heads, n_kv, d), dtype=torch.uint8, device="cuda")


def attend(gpu, kv, table, lens, q, work=None, seq_ids=None, fill=np.nan):
    import torch

    n, heads, d = q.shape
    out = torch.full((n, heads, d), fill, dtype=torch.float32, device="cuda")
    work = workspace(gpu, heads, kv.n_kv_heads, d) if work is None else work
    gpu.GpuAttentionPaged(kv, table, dev(lens, np.int32), dev(q), heads, n, out, work,
                          seq_ids=None if seq_ids is None else dev(seq_ids, np.int32))
    return host(out)


def check(got, pages, lens, q, seqs=None):
    for r, n in enumerate(lens):
        seq = r if seqs is None else seqs[r]
        want, smag, vmax = attention(q[r], pages.rows("k", seq, n), pages.rows("v", seq, n))
        if n == 0:
            assert np.all(got[r] == 0), r
            continue
        err = np.abs(got[r] - want).max(-1)
        limit = bound(pages.d, n, smag, vmax)
        assert np.all(err <= limit), (r, n, float((err / limit).max()))


EDGES = [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 127, 128, 129, 0, 255, 256, 257, 700]
CASES = [
    # kind, heads, n_kv, d, page, lens
    (F16, 16, 8, 128, 16, [500]),
    (F16, 16, 8, 128, 32, EDGES),
    (Q8, 32, 8, 128, 64, EDGES),
    (Q8, 16, 8, 128, 16, EDGES),
    (F16, 32, 4, 64, 16, EDGES),
    (Q8, 8, 8, 64, 256, EDGES),              # a page longer than a step
    (Q8, 15, 3, 128, 32, [77, 1000]),        # groups of 5
    (F16, 9, 3, 64, 64, [77, 1000]),         # of 3
    (F16, 7, 1, 128, 128, [1, 300]),         # of 7
    (Q8, 24, 2, 64, 16, [513, 5, 64]),       # of 12: more than one tile of query heads
    (F16, 33, 1, 128, 16, [40, 200]),        # of 33, the last tile of one head
    (Q8, 16, 1, 128, 64, [1, 2000]),         # of 16
    (F16, 1, 1, 64, 16, [30000]),            # one head, one long row: many shares of it
    (Q8, 4, 4, 128, 64, [20011, 3]),
    (F16, 4, 2, 64, 32, [(7 * i) % 23 for i in range(700)]),  # more rows than a workgroup's threads, many of them empty
]


@pytest.mark.parametrize("kind,heads,n_kv,d,page,lens", CASES)
def test_attention_vs_f64(gpu, kind, heads, n_kv, d, page, lens):
    """Unused slots and pages hold NaN (fp16) or NaN scales, table entries past a row's pages -1."""
    rng = np.random.default_rng(heads * 100 + d + len(lens))
    pages = Pages(rng, kind, n_kv, d, page, lens).fill_random(rng, lens)
    q = rng.normal(0, 1.5, (len(lens), heads, d)).astype(np.float32)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, q)
    check(got, pages, lens, q)
    assert np.array_equal(got, attend(gpu, kv, table, lens, q))  # shares are joined in one order


# What follows is shared out otherwise: from 8192 units (of 32 positions for fp16 rows of 128, else 64) all workgroups get
# alike; a row in more than 32 parts is joined in two steps; above 64 rows a lane stands for several, above 4096 the search
# for a row has a step more.
SHARED = [
    # kind, heads, n_kv, d, page, lens
    (F16, 4, 2, 128, 64, [(0, 2000, 1999, 700)[i % 4] + i for i in range(120)]),
    (Q8, 5, 1, 64, 32, [(4100 if i % 5 else 0) - i for i in range(150)]),
    (Q8, 2, 2, 128, 64, [4000, 1, 0, 5000, 77] * 16),
    (Q8, 8, 1, 128, 256, [8190] * 66),
    (F16, 2, 1, 64, 16, [140000, 140001, 140002, 120000]),
    (Q8, 5, 1, 128, 64, [20000]),
    (F16, 2, 2, 128, 16, [12000, 0, 31]),
    (F16, 1, 1, 64, 16, [(11 * i) % 40 for i in range(5000)]),
    (Q8, 2, 2, 64, 16, [(11 * i) % 90 for i in range(5000)]),
]


@pytest.mark.parametrize("kind,heads,n_kv,d,page,lens", SHARED)
def test_ways_of_sharing_out(gpu, kind, heads, n_kv, d, page, lens):
    lens = [max(n, 0) for n in lens]
    rng = np.random.default_rng(heads * 1000 + len(lens))
    pages = Pages(rng, kind, n_kv, d, page, lens).fill_random(rng, lens)
    q = rng.normal(0, 1.5, (len(lens), heads, d)).astype(np.float32)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, q)
    n = len(lens)
    look = range(n) if sum(lens) <= 250_000 else sorted({0, n - 1, *(int(r) for r in rng.choice(n, 20))})
    check(got[list(look)], pages, [lens[r] for r in look], q[list(look)], list(look))
    assert np.all(np.isfinite(got))
    assert np.array_equal(got, attend(gpu, kv, table, lens, q))


@pytest.mark.parametrize("kind", [F16, Q8])
def test_magnitudes(gpu, kind):
    """Queries and keys that make one position take everything, or all count alike; tiny, huge and zero queries; value
    rows of very different size (each held relative to the largest, as the bound says)."""
    rng = np.random.default_rng(21)
    lens = [300] * 6
    n_kv, d, page, heads = 2, 128, 32, 4
    pages = Pages(rng, kind, n_kv, d, page, lens).fill_random(rng, lens, k_amp=3.0)
    for i, pos in enumerate(rng.permutation(300)[:100]):
        pages.put(5, pos, rng.normal(0, 1, (n_kv, d)).astype(np.float32),
                  rng.normal(0, 10.0 ** (i % 7 - 4), (n_kv, d)).astype(np.float32))
    q = rng.normal(0, 1, (6, heads, d)).astype(np.float32)
    q[0] *= 20
    q[1] *= np.float32(1e-42)
    q[2] = 0
    q[3] *= np.float32(1e-20)
    q[3, 1, :] = 0
    q[3, 1, 7] = 5
    q[4, :, ::2] *= np.float32(1e-6)
    kv, table = pages.device(gpu)
    check(attend(gpu, kv, table, lens, q), pages, lens, q)


def test_scales_of_any_size(gpu):
    """8-bit value rows from 1e-30 to 1e30: an output is as near as the largest row's step allows."""
    rng = np.random.default_rng(22)
    lens = [200, 64, 64]
    pages = Pages(rng, Q8, 1, 64, 16, lens).fill_random(rng, lens)
    for r, amp in ((0, None), (1, 1e-30), (2, 1e30)):
        for pos in range(lens[r]):
            a = 10.0 ** rng.integers(-30, 30) if amp is None else amp
            pages.put(r, pos, rng.normal(0, 1, (1, 64)).astype(np.float32), (a * rng.normal(0, 1, (1, 64))).astype(np.float32))
    pages.put(1, 63, rng.normal(0, 1, (1, 64)).astype(np.float32), np.zeros((1, 64), np.float32))
    q = rng.normal(0, 1, (3, 2, 64)).astype(np.float32)
    kv, table = pages.device(gpu)
    check(attend(gpu, kv, table, lens, q), pages, lens, q)


@pytest.mark.parametrize("kind,d", [(F16, 128), (Q8, 64), (Q8, 128)])
def test_rows_out_of_range(gpu, kind, d):
    """Padding leaves its row alone; a bad length, sequence or page gives NaN, in that row alone."""
    rng = np.random.default_rng(23)
    lens = [100, 90, 33, 64, 20]
    n_kv, heads, page = 2, 8, 16
    pages = Pages(rng, kind, n_kv, d, page, lens, width=7).fill_random(rng, lens)
    pages.table[1, 3] = -5               # in the middle of row 1
    pages.table[2, 2] = pages.n_pages    # row 2's last position
    kv, table = pages.device(gpu)
    low, high = -2 ** 31, 2 ** 31 - 1
    seqs = [0, -1, low, 5, high, 0, 0, 0, 1, 1, 2, 2, 3, 4, 0]
    ask = [100, 7, 7, 7, 7, -1, 113, high, 90, 48, 33, 32, 64, 0, 112]
    #     good, padding, seq out,  lens out of range, page, before it, page, before it, good, empty, past its pages
    want = ["good", "pad", "pad", "nan", "nan", "nan", "nan", "nan", "nan", "good", "nan", "good", "good", "good", "good"]
    n = len(seqs)
    pages.k[pages.table[0, 6], :, 4:] = 0  # row 0's last page has slots behind position 99, asked for by the last row
    if kind == F16:
        pages.v[pages.table[0, 6], :, 4:] = 0
    else:
        pages.ks[pages.table[0, 6], :, 4:] = pages.vs[pages.table[0, 6], :, 4:] = 0.5
    kv, table = pages.device(gpu)
    q = rng.normal(0, 1, (n, heads, d)).astype(np.float32)
    work = workspace(gpu, heads, n_kv, d)
    got = attend(gpu, kv, table, ask, q, work, seqs, fill=7.0)
    for r in range(n):
        if want[r] == "pad":
            assert np.all(got[r] == 7), r
        elif want[r] == "nan":
            assert np.all(np.isnan(got[r])), r
        else:
            check(got[r:r + 1], pages, ask[r:r + 1], q[r:r + 1], seqs[r:r + 1])
    again = attend(gpu, kv, table, ask, q, work, seqs, fill=7.0)
    assert np.array_equal(got, again, equal_nan=True)


@pytest.mark.parametrize("d", [64, 128])
def test_infinities_among_the_attended(gpu, d):
    """As the definition gives them: a key of minus infinite score counts nothing, one of plus infinite score or NaN
    makes the head NaN; an infinite value reaches the output of its element, with its sign."""
    rng = np.random.default_rng(24)
    lens = [150] * 5
    n_kv, heads = 1, 2
    pages = Pages(rng, F16, n_kv, d, 16, lens).fill_random(rng, lens)
    q = np.abs(rng.normal(0, 1, (5, heads, d))).astype(np.float32) + np.float32(0.01)
    q[:, 1, 3] = 1.0            # exactly one fp16 number
    inf = np.float32(np.inf)

    def change(r, pos, name, element, value):
        p, s = pages.slot(r, pos)
        getattr(pages, name).view(np.float16)[p, 0, s, element] = value

    change(0, 149, "k", 3, -inf)
    change(1, 20, "k", 3, inf)
    change(2, 21, "k", 3, np.nan)
    change(3, 100, "v", 5, inf)
    change(3, 101, "v", 6, -inf)
    change(4, 100, "v", 5, inf)
    change(4, 3, "v", 5, -inf)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, q)
    assert np.all(np.isnan(got[1])) and np.all(np.isnan(got[2]))
    for r in (0, 3, 4):
        want, smag, vmax = attention(q[r], pages.rows("k", r, 150), pages.rows("v", r, 150))
        if r == 0:
            k = np.delete(pages.rows("k", r, 150), 149, 0)
            v = np.delete(pages.rows("v", r, 150), 149, 0)
            want, smag, vmax = attention(q[r], k, v)
        fine = np.isfinite(want)
        assert np.array_equal(got[r][~fine], want[~fine], equal_nan=True), r
        limit = bound(d, 150, smag, np.full(heads, 6.0))[:, None] + 0 * want
        assert np.all(np.abs(got[r] - want)[fine] <= limit[fine]), r


def test_non_finite_queries_and_poisoned_rows(gpu):
    """A query of an infinity or a NaN gives NaN in its own head; an 8-bit row kept as NaN reaches who attends to it."""
    rng = np.random.default_rng(25)
    lens = [70, 70, 70]
    pages = Pages(rng, Q8, 2, 64, 16, lens).fill_random(rng, lens)
    pages.put(1, 40, np.full((2, 64), np.inf, np.float32), np.ones((2, 64), np.float32))
    bad = np.ones((2, 64), np.float32)
    bad[1, 3] = np.nan
    pages.put(2, 69, np.ones((2, 64), np.float32), bad)
    q = rng.normal(0, 1, (3, 4, 64)).astype(np.float32)
    q[0, 1, 5] = np.inf
    q[0, 2, 6] = np.nan
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, q)
    assert np.all(np.isnan(got[0, 1:3])) and np.all(np.isfinite(got[0, [0, 3]]))
    assert np.all(np.isnan(got[1]))
    assert np.all(np.isfinite(got[2, :2])) and np.all(np.isnan(got[2, 2:]))


@pytest.mark.parametrize("heads,d", [(8, 128), (5, 64), (7, 128)])
def test_more_than_four_heads_of_an_8_bit_cache(gpu, heads, d):
    """Two column tiles: large and small queries and values, and what is not a number in one head, row or page alone."""
    rng = np.random.default_rng(35)
    lens = [300, 250, 70, 130, 129, 64]
    pages = Pages(rng, Q8, 1, d, 16, lens).fill_random(rng, lens, k_amp=2.0)
    for pos in range(lens[1]):
        pages.put(1, pos, rng.normal(0, 1, (1, d)).astype(np.float32),
                  (10.0 ** rng.integers(-30, 30) * rng.normal(0, 1, (1, d))).astype(np.float32))
    pages.put(2, 40, np.full((1, d), np.nan, np.float32), np.ones((1, d), np.float32))
    pages.put(5, 63, np.ones((1, d), np.float32), np.full((1, d), np.inf, np.float32))
    pages.table[3, 4] = pages.n_pages
    q = rng.normal(0, 1, (6, heads, d)).astype(np.float32)
    q[0, 0] *= 30
    q[0, heads - 1] *= np.float32(1e-30)
    q[4, 1, 2] = np.nan
    q[4, heads - 1, 3] = -np.inf
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, q)
    assert np.all(np.isnan(got[[2, 3, 5]]))
    check(got[:2], pages, lens[:2], q[:2])
    fine = [h for h in range(heads) if h not in (1, heads - 1)]
    assert np.all(np.isnan(got[4][[1, heads - 1]]))
    check(got[4:5][:, fine], pages, lens[4:5], q[4:5][:, fine], [4])


def test_rows_may_share_a_sequence(gpu):
    """A turn of several tokens: each row sees its own length of the one sequence; rows in any order, pages shared."""
    rng = np.random.default_rng(26)
    pages = Pages(rng, F16, 2, 128, 16, [130, 60]).fill_random(rng, [130, 60])
    seqs = [0, 1, 0, 0, 1, 0]
    ask = [130, 60, 128, 1, 59, 129]
    q = rng.normal(0, 1, (6, 4, 128)).astype(np.float32)
    kv, table = pages.device(gpu)
    check(attend(gpu, kv, table, ask, q, seq_ids=seqs), pages, ask, q, seqs)


def test_one_workspace_serves_call_after_call(gpu):
    """Calls of other shapes in between leave a workspace ready; its size covers every shape of the same heads."""
    rng = np.random.default_rng(27)
    heads, n_kv, d = 8, 2, 128
    work = workspace(gpu, heads, n_kv, d)
    work.fill_(0x55)
    gpu.GpuAttentionPagedWorkspaceInit(work, work.numel())
    assert not bool(work.any())
    for kind, page, lens in ((F16, 16, [9000]), (Q8, 64, [5, 0, 700]), (F16, 32, [1] * 300), (Q8, 16, [4000, 4001]),
                             (F16, 16, [9000])):
        pages = Pages(rng, kind, n_kv, d, page, lens).fill_random(rng, lens)
        q = rng.normal(0, 1, (len(lens), heads, d)).astype(np.float32)
        kv, table = pages.device(gpu)
        check(attend(gpu, kv, table, lens, q, work), pages, lens, q)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_captured_attention_follows_its_arrays(gpu, kind):
    """A captured call, replayed with other lengths, queries and pages; eager calls on another workspace in between."""
    import torch

    rng = np.random.default_rng(28)
    heads, n_kv, d, page = 16, 4, 128, 16
    room = [2000, 300, 800]
    pages = Pages(rng, kind, n_kv, d, page, room).fill_random(rng, room)
    kv, table = pages.device(gpu)
    work, other = workspace(gpu, heads, n_kv, d), workspace(gpu, heads, n_kv, d)
    lens = dev([1, 1, 1], np.int32)
    q = dev(rng.normal(0, 1, (3, heads, d)).astype(np.float32))
    out = torch.zeros_like(q)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        gpu.GpuAttentionPaged(kv, table, lens, q, heads, 3, out, work)
    for ask in ([2000, 300, 800], [0, 17, 64], [65, 0, 799], [2000, 1, 1]):
        lens.copy_(dev(ask, np.int32))
        q.copy_(dev(rng.normal(0, 1, (3, heads, d)).astype(np.float32)))
        eager = attend(gpu, kv, table, ask, host(q), other)
        graph.replay()
        got = host(out)
        check(got, pages, ask, host(q))
        assert np.array_equal(got, eager)


def test_two_streams_at_once(gpu):
    """Calls on two streams, a workspace each."""
    import torch

    rng = np.random.default_rng(29)
    heads, n_kv, d = 8, 4, 64
    lens = [3000, 100, 1500]
    pages = Pages(rng, Q8, n_kv, d, 32, lens).fill_random(rng, lens)
    kv, table = pages.device(gpu)
    n = dev(lens, np.int32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    qs = [dev(rng.normal(0, 1, (3, heads, d)).astype(np.float32)) for _ in streams]
    works = [workspace(gpu, heads, n_kv, d) for _ in streams]
    outs = [[torch.zeros_like(qs[0]) for _ in range(4)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(4):
        for s, q, w, o in zip(streams, qs, works, outs):
            with gpu.ScopedEngineStream(s):
                gpu.GpuAttentionPaged(kv, table, n, q, heads, 3, o[i], w)
    for q, o in zip(qs, outs):
        first = host(o[0])
        check(first, pages, lens, host(q))
        assert all(np.array_equal(first, host(x)) for x in o)


def test_pages_past_32_bit_offsets(gpu):
    """A sequence whose pages start past 2^32 elements of the pool."""
    import torch

    rng = np.random.default_rng(30)
    n_kv, d, page, heads = 8, 128, 256, 16
    few = Pages(rng, Q8, n_kv, d, page, [600], spare=0).fill_random(rng, [600])
    n_pages = (1 << 32) // (n_kv * d * page) + 8
    far = np.arange(n_pages - few.n_pages, n_pages)
    k, v = (torch.zeros((n_pages, n_kv, page, d), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((n_pages, n_kv, page), device="cuda") for _ in range(2))
    for big, small in ((k, few.k), (v, few.v), (ks, few.ks), (vs, few.vs)):
        big[int(far[0]):] = dev(small)
    kv, table = gpu.GpuPagedKv(k, v, ks, vs), gpu.GpuPageTable(dev(far[few.table], np.int32))
    q = rng.normal(0, 1, (1, heads, d)).astype(np.float32)
    check(attend(gpu, kv, table, [600], q), few, [600], q)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_the_longest_row_there_is(gpu, kind):
    """2^31 - 1 positions: a table whose entries are all one page, but for the last, whose last slot holds NaN and is the
    one position that the length leaves out.

    Each of the 256 slots counts 2^23 times, but for 255 of the first page and all but one of the last. A lane adds up
    16 weights for each of its wave's 2^25 / 2048 units one after the other, in fp32, and outputs likewise: 2^18 roundings
    of half a step, of the sum of the weights and of the outputs, so 2 * 2^18 * 2^-24 of the largest value, beside which
    the bound of a short row is nothing."""
    rng = np.random.default_rng(34)
    d, page, n = 64, 256, 2 ** 31 - 1
    pages = Pages(rng, kind, 1, d, page, [2 * page], spare=0).fill_random(rng, [2 * page])
    main, last = pages.table[0]
    pages.put(0, 2 * page - 1, np.full((1, d), np.nan, np.float32), np.full((1, d), np.nan, np.float32))
    kv, _ = pages.device(gpu)
    table = np.full((1, 2 ** 23), main, np.int32)
    table[0, -1] = last
    q = rng.normal(0, 1, (1, 2, d)).astype(np.float32)
    got = attend(gpu, kv, gpu.GpuPageTable(dev(table)), [n], q)
    k, v = pages.rows("k", 0, 2 * page - 1)[:, 0], pages.rows("v", 0, 2 * page - 1)[:, 0]
    times = np.where(np.arange(2 * page - 1) < page, 2.0 ** 23 - 1, 1.0)
    s = q[0].astype(np.float64) @ k.T / np.sqrt(d)
    w = np.exp(s - s.max(-1, keepdims=True)) * times
    want = w @ v / w.sum(-1, keepdims=True)
    vmax = np.abs(v).max()
    assert np.all(np.abs(got[0] - want) <= 2.0 ** -5 * vmax + bound(d, 512, np.abs(s).max() * d, vmax))


@pytest.mark.parametrize("kind,n_kv,group,page", [(F16, 8, 2, 16), (Q8, 8, 4, 64), (F16, 2, 8, 32)])
def test_a_batch_is_served(gpu, ora, kind, n_kv, group, page):
    """Two prompts put into pages, one read back into the contiguous cache for its attention there; then steps of one
    token for both: norm, rotation and write, attention over the pages. The step's outputs are those of 64 bits, and
    with fp16 pages those of the contiguous operators within the two sides' bounds."""
    import torch

    rng = np.random.default_rng(31)
    heads, d, eps, room = n_kv * group, 128, 1e-6, 256
    prompts, steps = [90, 37], 3
    lens = [n + steps for n in prompts]
    pages = Pages(rng, kind, n_kv, d, page, lens)
    kv, table = pages.device(gpu)
    tab = dev(gpu.build_rope_table(d, 1e6, room))
    qw, kw = dev((1 + 0.3 * rng.normal(0, 1, (2, d))).astype(np.float32))
    work = workspace(gpu, heads, n_kv, d)

    def raw(n):
        return [dev(rng.normal(0, 1, (n, h, d)).astype(np.float32)) for h in (heads, n_kv, n_kv)]

    flat = [torch.zeros((2, n_kv, room, d), dtype=torch.int16, device="cuda") for _ in prompts]
    seq = dev(np.repeat([0, 1], prompts), np.int32)
    pos = dev(np.concatenate([np.arange(n) for n in prompts]), np.int32)
    q, k, v = raw(sum(prompts))
    out = torch.empty_like(q)
    gpu.GpuQkNormRopeKvPaged(kv, table, seq, pos, q, k, v, qw, kw, heads, tab, room, sum(prompts), eps, out)
    at = 0
    for i, n in enumerate(prompts):
        mine = slice(at, at + n)
        at += n
        gpu.GpuKvReadPaged(kv, table, seq[mine], pos[mine], n, flat[i][0], flat[i][1], d, room * d)
        got = torch.empty((n, heads, d), device="cuda")
        gpu.GpuAttentionFromCache(heads, n_kv, d, 0, out[mine].contiguous(), n, flat[i][0], flat[i][1], room, got)
        ref, smag, vmax = ora.attention_f64(host(out[mine]), host(flat[i][0]).reshape(-1).view(np.uint16),
                                            host(flat[i][1]).reshape(-1).view(np.uint16), room, heads, n_kv, d, 0, n)
        err = np.abs(host(got).astype(np.float64) - ref.reshape(n, heads, d)).max(-1)
        assert np.all(err <= bound(d, n, smag, vmax))
    for step in range(steps):
        q, k, v = raw(2)
        now = [n + step for n in prompts]
        rot, got = torch.empty_like(q), torch.empty_like(q)
        p = dev(now, np.int32)
        gpu.GpuQkNormRopeKvPaged(kv, table, None, p, q, k, v, qw, kw, heads, tab, room, 2, eps, rot)
        gpu.GpuAttentionPaged(kv, table, p + 1, rot, heads, 2, got, work)
        torch.cuda.synchronize()
        for name, t in zip(("k", "v", "ks", "vs"), kv.tensors):
            if t is not None:
                a = host(t)
                setattr(pages, name, a.view(np.uint16) if a.dtype == np.int16 else a)
        check(host(got), pages, [n + 1 for n in now], host(rot))
        if kind == F16:
            for i in range(2):
                qq, kk = q[i:i + 1].clone(), k[i:i + 1].clone()
                gpu.GpuQkNormRopeKv(qq, kk, v[i:i + 1].contiguous(), qw, kw, heads, n_kv, d, tab, room, now[i], 1, eps,
                                    flat[i][0], flat[i][1], room)
                other = torch.empty_like(qq)
                gpu.GpuAttentionFromCache(heads, n_kv, d, now[i], qq, 1, flat[i][0], flat[i][1], room, other)
                _, smag, vmax = attention(host(rot)[i], pages.rows("k", i, now[i] + 1), pages.rows("v", i, now[i] + 1))
                assert np.all(np.abs(host(other[0]) - host(got[i])).max(-1) <= 2 * bound(d, now[i] + 1, smag, vmax))


@pytest.mark.parametrize("kind", [F16, Q8])
def test_prompts_of_head_64_are_served_a_row_a_token(gpu, kind):
    """Heads of 64: a prompt and a later turn of two conversations written into pages, each token attending as a row of
    its own to the positions up to it (the contiguous attention serves heads of 128 alone)."""
    import torch

    rng = np.random.default_rng(37)
    heads, n_kv, d, eps, room = 8, 2, 64, 1e-6, 128
    turns = [([0, 0], [50, 33]), ([50, 33], [7, 20])]  # positions held before, and new ones
    pages = Pages(rng, kind, n_kv, d, 16, [57, 53])
    kv, table = pages.device(gpu)
    tab = dev(gpu.build_rope_table(d, 1e6, room))
    qw, kw = dev((1 + 0.3 * rng.normal(0, 1, (2, d))).astype(np.float32))
    work = workspace(gpu, heads, n_kv, d)
    for past, new in turns:
        seqs = np.repeat([0, 1], new)
        at = np.concatenate([p + np.arange(m) for p, m in zip(past, new)])
        n = len(at)
        q, k, v = (dev(rng.normal(0, 1, (n, h, d)).astype(np.float32)) for h in (heads, n_kv, n_kv))
        seq, pos, out = dev(seqs, np.int32), dev(at, np.int32), torch.empty_like(q)
        gpu.GpuQkNormRopeKvPaged(kv, table, seq, pos, q, k, v, qw, kw, heads, tab, room, n, eps, q)
        gpu.GpuAttentionPaged(kv, table, pos + 1, q, heads, n, out, work, seq_ids=seq)
        torch.cuda.synchronize()
        for name, t in zip(("k", "v", "ks", "vs"), kv.tensors):
            if t is not None:
                a = host(t)
                setattr(pages, name, a.view(np.uint16) if a.dtype == np.int16 else a)
        check(host(out), pages, list(at + 1), host(q), list(seqs))
    layer = torch.zeros((2, n_kv, room, d), dtype=torch.int16, device="cuda")
    with pytest.raises(gpu.RpgError, match="supports head_dim 128"):
        gpu.GpuAttentionFromCache(heads, n_kv, d, 0, q, n, layer[0], layer[1], room, out)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_captured_steps_of_a_batch(gpu, kind):
    """A step of a batch as one graph: norm, rotation and write, then attention, with positions and lengths counted up in
    it. Replays, with eager calls of the same operators on other buffers in between, give the eager steps' bits."""
    import torch

    rng = np.random.default_rng(33)
    heads, n_kv, d, eps, room = 10, 2, 128, 1e-6, 512
    had = [300, 15, 63, 0]
    n = len(had)
    lens = [h + 8 for h in had]
    pages = Pages(rng, kind, n_kv, d, 16, lens).fill_random(rng, had)
    tab = dev(gpu.build_rope_table(d, 1e6, room))
    qw, kw = dev((1 + 0.3 * rng.normal(0, 1, (2, d))).astype(np.float32))
    seq = dev([0, 1, 2, -1], np.int32)  # the last row is padding
    raw = [dev(rng.normal(0, 1, (8, n, h, d)).astype(np.float32)) for h in (heads, n_kv, n_kv)]

    class Side:
        def __init__(self):
            self.kv, self.table = pages.device(gpu)
            self.work = workspace(gpu, heads, n_kv, d)
            self.pos, self.lens = dev(had, np.int32), dev(had, np.int32)
            self.q, self.k, self.v = (torch.zeros_like(x[0]) for x in raw)
            self.out = torch.full_like(self.q, 7.0)

        def step(self):
            gpu.GpuQkNormRopeKvPaged(self.kv, self.table, seq, self.pos, self.q, self.k, self.v, qw, kw, heads, tab, room,
                                     n, eps, self.q)
            self.lens.copy_(self.pos + 1)
            gpu.GpuAttentionPaged(self.kv, self.table, self.lens, self.q, heads, n, self.out, self.work, seq_ids=seq)
            self.pos.add_(1)

        def take(self, i):
            for to, x in zip((self.q, self.k, self.v), raw):
                to.copy_(x[i])

    eager, replayed = Side(), Side()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        replayed.step()
    for i in range(8):
        eager.take(i)
        replayed.take(i)
        with gpu.ScopedEngineStream(torch.cuda.current_stream()):
            eager.step()
        graph.replay()
        want, got = host(eager.out), host(replayed.out)
        assert np.array_equal(got, want)
        assert np.all(want[3] == 7)
        for name, t in zip(("k", "v", "ks", "vs"), eager.kv.tensors):
            if t is not None:
                a = host(t)
                setattr(pages, name, a.view(np.uint16) if a.dtype == np.int16 else a)
        check(want[:3], pages, [h + i + 1 for h in had[:3]], host(eager.q)[:3])
        assert pages.same_as(replayed.kv)
