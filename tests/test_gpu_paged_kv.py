"""The paged cache's writers and reader on the GPU: codes, halves and read-back values bit for bit, the norm and
rotation within the roundings they make, and nothing touched that a row does not name."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8, U, Pages, quantise

pytestmark = pytest.mark.gpu

EPS = 1e-6


def dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def host(t):
    import torch

    torch.cuda.synchronize()
    return t.cpu().numpy()


def rows(rng, n, heads, d):
    x = rng.normal(0, 1, (n, heads, d)).astype(np.float32)
    return x * np.exp(rng.normal(0, 2, (n, heads, 1))).astype(np.float32)


def placed(rng, lens, news):
    """seq_ids and positions of the last news[i] positions of each sequence, in mixed order."""
    seq = np.concatenate([np.full(m, i) for i, m in enumerate(news)])
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, news)])
    mix = rng.permutation(len(seq))
    return seq[mix].astype(np.int32), pos[mix].astype(np.int32)


CASES = [
    # kind, n_kv, d, page, lens, new positions
    (F16, 8, 128, 16, [1], [1]),
    (Q8, 8, 128, 64, [1], [1]),
    (F16, 3, 64, 32, [33, 16, 70], [33, 1, 5]),
    (Q8, 1, 64, 16, [17, 1, 300], [17, 1, 299]),
    (Q8, 5, 128, 256, [257, 256, 1], [2, 256, 1]),
    (F16, 2, 128, 128, [129, 500], [128, 3]),
]


@pytest.mark.parametrize("kind,n_kv,d,page,lens,news", CASES)
def test_write_and_read_are_exact(gpu, kind, n_kv, d, page, lens, news):
    import torch

    rng = np.random.default_rng(len(lens) * 1000 + d + page)
    pages = Pages(rng, kind, n_kv, d, page, lens)
    kv, table = pages.device(gpu)
    seq, pos = placed(rng, lens, news)
    n = len(seq)
    k, v = rows(rng, n, n_kv, d), rows(rng, n, n_kv, d)
    gpu.GpuKvWritePaged(kv, table, dev(seq), dev(pos), dev(k), dev(v), n)
    for t in range(n):
        pages.put(seq[t], pos[t], k[t], v[t])
    assert pages.same_as(kv)  # the rows, and every other byte as it was
    for f32 in (True, False):
        wide = torch.full((2, n, n_kv, d + 8), 7.0, dtype=torch.float32 if f32 else torch.float16, device="cuda")
        gpu.GpuKvReadPaged(kv, table, dev(seq), dev(pos), n, wide[0], wide[1], n_kv * (d + 8), d + 8)
        got = host(wide)
        assert np.all(got[..., d:] == 7)
        for i, x in enumerate((k, v)):
            if kind == F16:
                want = x.astype(np.float16).astype(np.float32)
            else:
                code, s = quantise(x)
                want = code.astype(np.float32) * s[..., None]
            assert np.array_equal(got[i, ..., :d], want if f32 else want.astype(np.float16))


def test_read_into_the_contiguous_cache(gpu):
    """(head_dim, max_seq * head_dim) strides: what GpuKvWrite leaves there."""
    import torch

    rng = np.random.default_rng(5)
    n_kv, d, n, max_seq = 8, 128, 77, 100
    pages = Pages(rng, F16, n_kv, d, 32, [n])
    kv, table = pages.device(gpu)
    k, v = dev(rows(rng, n, n_kv, d)), dev(rows(rng, n, n_kv, d))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    seq = torch.zeros_like(pos)
    gpu.GpuKvWritePaged(kv, table, seq, pos, k, v, n)
    a, b = (torch.full((2, n_kv, max_seq, d), 0x1234, dtype=torch.int16, device="cuda") for _ in range(2))
    gpu.GpuKvWrite(k, v, n_kv, d, 0, n, a[0], a[1], max_seq)
    gpu.GpuKvReadPaged(kv, table, seq, pos, n, b[0], b[1], d, max_seq * d)
    assert torch.equal(a, b)


def test_read_into_one_buffer(gpu):
    """Keys and values of a token, or of a head, one behind the other in one buffer, or with as much room between."""
    import torch

    from test_paged_args import shifted_reads

    rng = np.random.default_rng(6)
    n_kv, d, n = 2, 64, 3
    pages = Pages(rng, F16, n_kv, d, 16, [n])
    kv, table = pages.device(gpu)
    k, v = rows(rng, n, n_kv, d), rows(rng, n, n_kv, d)
    pos, seq = dev(np.arange(n), np.int32), dev(np.zeros(n), np.int32)
    gpu.GpuKvWritePaged(kv, table, seq, pos, dev(k), dev(v), n)
    apart = [c for c in shifted_reads(d, n, n_kv) if not c[-1]]
    assert len(apart) > 100
    for shift, ts, hs, f32, _ in apart:
        dtype, size = (torch.float32, 4) if f32 else (torch.float16, 2)
        buf = torch.full((8192,), 7.0, dtype=dtype, device="cuda")
        at = [2048, 2048 + shift // size]
        gpu.GpuKvReadPaged(kv, table, seq, pos, n, buf[at[0]:], buf[at[1]:], ts, hs)
        want = np.full(8192, 7, np.float32)
        for x, first in zip((k, v), at):
            for t in range(n):
                for h in range(n_kv):
                    want[first + t * ts + h * hs:][:d] = x[t, h].astype(np.float16)
        assert np.array_equal(host(buf).astype(np.float32), want)


def test_values_at_the_ends_of_the_range(gpu):
    """Rows of zeros, of subnormals, of the largest numbers, with ties, infinities and NaN in them."""
    d = 64
    base = np.random.default_rng(3).normal(0, 1, (12, 1, d)).astype(np.float32)
    base[0] = 0
    base[1] *= np.float32(1e-39)
    base[2] = np.float32(1e-45)
    base[3] *= np.float32(1e37)
    base[4, 0, 5] = np.finfo(np.float32).max
    base[5, 0, 6] = np.inf
    base[6, 0, 7] = -np.inf
    base[7, 0, 63] = np.nan
    base[8] = np.float32(2.0) * (np.arange(d) % 2 * 2 - 1)                  # every value the largest
    base[9] = (np.arange(d) - 32 + np.float32(0.5)) * np.float32(1 / 128)   # ties
    base[9, 0, 0] = np.float32(127 / 128)
    base[10] = np.float32(127 * 2.0 ** -126) * np.sign(base[10])            # the smallest scale there is
    base[11] = np.float32(126 * 2.0 ** -126) * np.sign(base[11])            # and the first that is not
    n = len(base)
    for kind in (F16, Q8):
        pages = Pages(np.random.default_rng(1), kind, 1, d, 16, [n])
        kv, table = pages.device(gpu)
        seq, pos = np.zeros(n, np.int32), np.arange(n, dtype=np.int32)
        gpu.GpuKvWritePaged(kv, table, dev(seq), dev(pos), dev(base), dev(-base), n)
        for t in range(n):
            pages.put(0, t, base[t], -base[t])
        if kind == F16:
            got, want = host(kv.tensors[0]).view(np.float16), pages.k.view(np.float16)
            assert np.array_equal(got, want, equal_nan=True)
        else:
            for got, want in zip(kv.tensors, (pages.k, pages.v, pages.ks, pages.vs)):
                assert np.array_equal(host(got), want, equal_nan=True)
            back = dev(np.zeros((2, n, d), np.float32))
            gpu.GpuKvReadPaged(kv, table, dev(seq), dev(pos), n, back[0], back[1], d, d)
            back = host(back)
            assert np.all(np.isnan(back[:, 5:8])) and np.all(np.isfinite(np.delete(back, [5, 6, 7], 1)))


def norm_rope_f64(x, w, tab, pos):
    """RoPE(RMSNorm(x) * w) in 64 bits, and the sum of magnitudes |a c| + |b s| that its last addition joins."""
    x = x.astype(np.float64)
    d = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
    a, b = y[..., :d // 2], y[..., d // 2:]
    t = tab.astype(np.float64)[pos][:, None]
    c, s = t[..., :d // 2], t[..., d // 2:]
    return (np.concatenate([a * c - b * s, b * c + a * s], -1),
            np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)], -1))


@pytest.mark.parametrize("heads,kind,n_kv,d,page,lens,news", [(8 * 2, *CASES[0]), (4, *CASES[3]), (3, *CASES[2]),
                                                              (15, *CASES[4]), (2, *CASES[5])])
def test_norm_rope_write(gpu, heads, kind, n_kv, d, page, lens, news):
    """q_out and the cache against 64 bits. A normed and rotated value is 3 roundings of each of a and b (scale, times
    scale, times weight), one of each product and one of the sum: 5 units of 2^-24 of |a c| + |b s|, 5.01 with the
    products of errors. An 8-bit row's scale and reciprocal are 3 roundings more, so that a value is off by half a step
    and 127 codes' worth of them; a half by half its last place (2^-11), at least 2^-25."""
    import torch

    rng = np.random.default_rng(heads + d)
    pages = Pages(rng, kind, n_kv, d, page, lens)
    kv, table = pages.device(gpu)
    seq, pos = placed(rng, lens, news)
    n = len(seq)
    q, k, v = rows(rng, n, heads, d), rows(rng, n, n_kv, d), rows(rng, n, n_kv, d)
    qw, kw = (1 + 0.3 * rng.normal(0, 1, (2, d))).astype(np.float32)
    rope_rows = max(lens)
    tab = gpu.build_rope_table(d, 1e6, rope_rows)
    qd, kd, vd, out = dev(q), dev(k), dev(v), torch.full((n, heads, d), np.nan, device="cuda")
    args = (dev(qw), dev(kw), heads, dev(tab), rope_rows, n, EPS)
    gpu.GpuQkNormRopeKvPaged(kv, table, dev(seq), dev(pos), qd, kd, vd, *args, out)
    assert np.array_equal(host(qd), q) and np.array_equal(host(kd), k) and np.array_equal(host(vd), v)
    want, mag = norm_rope_f64(q, qw.astype(np.float64), tab, pos)
    assert np.all(np.abs(host(out) - want) <= 5.01 * U * mag)
    back = dev(np.zeros((2, n, n_kv, d), np.float32))
    gpu.GpuKvReadPaged(kv, table, dev(seq), dev(pos), n, back[0], back[1], n_kv * d, d)
    back = host(back).astype(np.float64)
    want, mag = norm_rope_f64(k, kw.astype(np.float64), tab, pos)
    if kind == F16:
        assert np.all(np.abs(back[0] - want) <= 5.01 * U * mag + np.maximum(2.0 ** -11 * np.abs(want) * 1.001, 2.0 ** -25))
        assert np.array_equal(back[1], v.astype(np.float16).astype(np.float64))
    else:
        step = np.abs(want).max(-1, keepdims=True) / 127
        assert np.all(np.abs(back[0] - want) <= 5.01 * U * mag + step * (0.5 + 127 * 10 * U))
        code, s = quantise(v)
        assert np.array_equal(back[1], (code.astype(np.float32) * s[..., None]).astype(np.float64))
    inplace = qd.clone()
    gpu.GpuQkNormRopeKvPaged(kv, table, dev(seq), dev(pos), inplace, kd, vd, *args, inplace)
    assert torch.equal(inplace, out)


@pytest.mark.parametrize("n", [1, 21, 700])
def test_same_bits_as_the_contiguous_operator(gpu, n):
    """At head_dim 128: GpuQkNormRopeKv's q and cache, whatever pages the rows go to."""
    import torch

    rng = np.random.default_rng(n)
    heads, n_kv, d, past, max_seq = 16, 8, 128, 37, 800
    pages = Pages(rng, F16, n_kv, d, 64, [past + n])
    kv, table = pages.device(gpu)
    q, k, v = (dev(rows(rng, n, h, d)) for h in (heads, n_kv, n_kv))
    qw, kw = dev((1 + 0.3 * rng.normal(0, 1, (2, d))).astype(np.float32))
    tab = dev(gpu.build_rope_table(d, 1e6, max_seq))
    pos = torch.arange(past, past + n, dtype=torch.int32, device="cuda")
    out, seq = torch.empty_like(q), torch.zeros_like(pos)
    gpu.GpuQkNormRopeKvPaged(kv, table, seq, pos, q, k, v, qw, kw, heads, tab, max_seq, n, EPS, out)
    a = torch.zeros((2, n_kv, max_seq, d), dtype=torch.int16, device="cuda")
    row = torch.empty((2, n, n_kv, d), dtype=torch.int16, device="cuda")
    gpu.GpuKvReadPaged(kv, table, seq, pos, n, row[0], row[1], n_kv * d, d)
    gpu.GpuQkNormRopeKv(q, k, v, qw, kw, heads, n_kv, d, tab, max_seq, past, n, EPS, a[0], a[1], max_seq)
    assert torch.equal(out, q)
    assert torch.equal(row, a[:, :, past:past + n].transpose(1, 2))


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_name_no_slot(gpu, kind, d):
    """Padding leaves everything alone; rows out of range store nothing and give NaN."""
    import torch

    rng = np.random.default_rng(9)
    n_kv, heads, page, rope_rows = 2, 4, 16, 40
    lens = [48, 20]
    pages = Pages(rng, kind, n_kv, d, page, lens, width=3)
    pages.table[1, 2] = pages.n_pages  # a page past the pool; its neighbour -1 is not a page either
    kv, table = pages.device(gpu)
    low, high = -2 ** 31, 2 ** 31 - 1
    #        good  pad    pad   seq  seq    pos     pos      page  page<0...     past the RoPE table  good
    seq = [0,      -1,    low,  2,   high,  0,      0,       1,    1,            0,                   1]
    pos = [3,      5,     high, 4,   4,     -1,     48,      33,   high,         45,                  19]
    fine = np.array([True, False, False, False, False, False, False, False, False, True, True])
    pad = np.array(seq) < 0
    n = len(seq)
    k, v, q = rows(rng, n, n_kv, d), rows(rng, n, n_kv, d), rows(rng, n, heads, d)
    s, p = dev(seq, np.int32), dev(pos, np.int32)
    gpu.GpuKvWritePaged(kv, table, s, p, dev(k), dev(v), n)
    for t in np.flatnonzero(fine):
        pages.put(seq[t], pos[t], k[t], v[t])
    assert pages.same_as(kv)
    back = torch.full((2, n, n_kv, d), 7.0, device="cuda")
    gpu.GpuKvReadPaged(kv, table, s, p, n, back[0], back[1], n_kv * d, d)
    got = host(back)
    assert np.all(got[:, pad] == 7) and np.all(np.isnan(got[:, ~fine & ~pad])) and np.all(np.isfinite(got[:, fine]))
    fused = fine & (np.array(pos) < rope_rows)
    other = Pages(np.random.default_rng(9), kind, n_kv, d, page, lens, width=3)
    other.table[1, 2] = other.n_pages
    kv2, table2 = other.device(gpu)
    out = torch.full((n, heads, d), 7.0, device="cuda")
    w = dev(np.ones((2, d), np.float32))
    gpu.GpuQkNormRopeKvPaged(kv2, table2, s, p, dev(q), dev(k), dev(v), w[0], w[1], heads,
                             dev(gpu.build_rope_table(d, 1e6, rope_rows)), rope_rows, n, EPS, out)
    got = host(out)
    assert np.all(got[pad] == 7) and np.all(np.isnan(got[~fused & ~pad])) and np.all(np.isfinite(got[fused]))
    pools = [host(t) for t in kv2.tensors if t is not None]
    before = [a for a in (other.k, other.v, other.ks, other.vs) if a is not None]
    written = np.zeros((other.n_pages, page), bool)
    for t in np.flatnonzero(fused):
        written[other.slot(seq[t], pos[t])] = True
    for a, b in zip(pools, before):
        a, b = (x.view(np.uint8).reshape(*x.shape, -1) for x in (a, b.view(a.dtype)))
        there = (a != b).reshape(*a.shape[:3], -1).any((1, 3))
        assert np.array_equal(there, written)


def test_default_seq_ids_and_one_row_per_sequence(gpu):
    import torch

    rng = np.random.default_rng(11)
    lens = [5, 40, 17]
    pages = Pages(rng, Q8, 2, 64, 16, lens)
    kv, table = pages.device(gpu)
    k, v = rows(rng, 3, 2, 64), rows(rng, 3, 2, 64)
    pos = dev([n - 1 for n in lens], np.int32)
    gpu.GpuKvWritePaged(kv, table, None, pos, dev(k), dev(v), 3)
    for t, n in enumerate(lens):
        pages.put(t, n - 1, k[t], v[t])
    assert pages.same_as(kv)
    a, b = (torch.zeros((2, 3, 2, 64), device="cuda") for _ in range(2))
    gpu.GpuKvReadPaged(kv, table, None, pos, 3, a[0], a[1], 128, 64)
    gpu.GpuKvReadPaged(kv, table, dev([0, 1, 2], np.int32), pos, 3, b[0], b[1], 128, 64)
    assert torch.equal(a, b) and bool(a.any())


def test_captured_writes_follow_their_arrays(gpu):
    """A captured write and read, replayed with other rows, positions and tables each time, on its own stream."""
    import torch

    rng = np.random.default_rng(13)
    heads, n_kv, d, page, n = 4, 2, 128, 16, 9
    lens = [30, 33]
    pages = Pages(rng, Q8, n_kv, d, page, lens)
    kv, table = pages.device(gpu)
    tab = dev(gpu.build_rope_table(d, 1e6, 64))
    w = dev(np.ones((2, d), np.float32))
    q, k, v = (dev(rows(rng, n, h, d)) for h in (heads, n_kv, n_kv))
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda")
    out, back = torch.zeros_like(q), torch.zeros((2, n, n_kv, d), device="cuda")

    def step(into, rows_back):
        gpu.GpuQkNormRopeKvPaged(kv, table, seq, pos, q, k, v, w[0], w[1], heads, tab, 64, n, EPS, into)
        gpu.GpuKvReadPaged(kv, table, seq, pos, n, rows_back[0], rows_back[1], n_kv * d, d)

    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        step(out, back)
    for i in range(3):
        s, p = placed(rng, lens, [4, 5])
        seq.copy_(dev(s))
        pos.copy_(dev(p) - i)
        q.copy_(dev(rows(rng, n, heads, d)))
        k.copy_(dev(rows(rng, n, n_kv, d)))
        table.pages.copy_(dev(rng.permutation(pages.n_pages)[:table.pages.numel()].reshape(table.pages.shape), np.int32))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want_q, want_back = torch.zeros_like(out), torch.zeros_like(back)
        step(want_q, want_back)
        assert torch.equal(out, want_q) and torch.equal(back, want_back) and bool(out.any())


def test_pools_past_32_bit_offsets(gpu):
    """Rows in pages that start past 2^32 elements of the pool."""
    import torch

    n_kv, d, page = 8, 128, 256
    n_pages = (1 << 32) // (n_kv * d * page) + 2
    k, v = (torch.zeros((n_pages, n_kv, page, d), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((n_pages, n_kv, page), device="cuda") for _ in range(2))
    kv = gpu.GpuPagedKv(k, v, ks, vs)
    table = gpu.GpuPageTable(dev([[0, n_pages - 1]], np.int32))
    rng = np.random.default_rng(17)
    x, y = rows(rng, 2, n_kv, d), rows(rng, 2, n_kv, d)
    seq, pos = dev([0, 0], np.int32), dev([3, page + 255], np.int32)
    gpu.GpuKvWritePaged(kv, table, seq, pos, dev(x), dev(y), 2)
    for t, at in ((0, (0, slice(None), 3)), (1, (n_pages - 1, slice(None), 255))):
        for pool, scale, z in ((k, ks, x), (v, vs, y)):
            code, s = quantise(z[t])
            assert np.array_equal(host(pool[at]), code) and np.array_equal(host(scale[at]), s)
    back = torch.zeros((2, 2, n_kv, d), device="cuda")
    gpu.GpuKvReadPaged(kv, table, seq, pos, 2, back[0], back[1], n_kv * d, d)
    code, s = quantise(x)
    assert np.array_equal(host(back[0]), code * s[..., None])
    assert int((ks != 0).sum()) == 2 * n_kv
