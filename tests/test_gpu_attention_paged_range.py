"""Attention over the paged cache where values differ widely in size: each output element is as near as the weighted sum
of magnitudes that it is made of allows (derived at paged_ref.attention_within), whatever other rows of the cache hold."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8, Pages, attention_within, quantise
from test_gpu_attention_paged import attend, dev

pytestmark = pytest.mark.gpu


def hold(pages, seq, k, v):
    """fp32 rows [n, n_kv, d] as positions 0 .. n - 1 of a sequence."""
    pos = np.arange(len(k))
    p, s = pages.table[seq, pos // pages.page], pos % pages.page
    for name, x in (("k", k), ("v", v)):
        x = np.asarray(x, np.float32)
        if pages.kind == F16:
            getattr(pages, name)[p, :, s] = x.astype(np.float16).view(np.uint16)
        else:
            getattr(pages, name)[p, :, s], getattr(pages, name + "s")[p, :, s] = quantise(x)


def check(gpu, kind, q, ks, vs, page=32, rows=None):
    """Rows q [n, heads, d] over sequences of keys ks[i] and values vs[i]: the outputs, held to attention_within."""
    lens = [len(k) for k in ks]
    d, n_kv = q.shape[-1], ks[0].shape[1]
    pages = Pages(np.random.default_rng(1), kind, n_kv, d, page, lens)
    for i, (k, v) in enumerate(zip(ks, vs)):
        hold(pages, i, k, v)
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, lens, q)
    for r, n in enumerate(lens):
        want, limit = attention_within(q[r], pages.rows("k", r, n), pages.rows("v", r, n), kind)
        err = np.abs(got[r] - want)
        assert np.all(err <= limit), (r, n, float((err / np.maximum(limit, 1e-300)).max()))
    return got


def scored(rng, q, scores):
    """Keys [n, 1, d] whose scores with q [d] are about `scores`: along q, and as much again at random across it."""
    d = len(q)
    q = q.astype(np.float64)
    k = np.outer(np.asarray(scores) * np.sqrt(d) / (q @ q), q)
    x = rng.normal(0, 0.3, k.shape)
    return (k + x - np.outer(x @ q / (q @ q), q))[:, None].astype(np.float32)


LENS = [1, 63, 64, 65, 300, 1000, 3001]


@pytest.mark.parametrize("sigma", [1.0, 2.0, 6.0])
@pytest.mark.parametrize("heads,n_kv,d", [(4, 1, 128), (8, 1, 128), (5, 1, 64), (4, 4, 64)])
def test_value_rows_of_spread_sizes(gpu, heads, n_kv, d, sigma):
    """Sizes spread log-normally, in rows of one wave and of many workgroups."""
    rng = np.random.default_rng(int(10 * sigma) + heads + d)
    ks = [rng.normal(0, 1, (n, n_kv, d)) for n in LENS]
    vs = [rng.normal(0, 1, (n, n_kv, d)) * np.exp(rng.normal(0, sigma, (n, n_kv, 1))) for n in LENS]
    check(gpu, Q8, rng.normal(0, 1, (len(LENS), heads, d)).astype(np.float32), ks, vs)


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("heads,d", [(4, 128), (8, 128), (3, 64), (7, 64)])
def test_a_large_row_of_no_weight(gpu, heads, d, kind):
    """One value row far larger than all others, of no weight or of a weight that makes it count as much as they do, in
    the first, a middle and the last position."""
    rng = np.random.default_rng(heads + d)
    cases = [(size, at, n) for size in (1e3, 1e6, 1e9, 1e30) for at in (0, 70, -1) for n in (128, 500)]
    if kind == F16:
        cases = [c for c in cases if c[0] == 1e3]
    q1 = rng.normal(0, 1, d).astype(np.float32)
    q = np.repeat(q1[None], len(cases), 0)[:, None] * (1 + 0.01 * rng.normal(0, 1, (len(cases), heads, 1)))
    for score in (-150.0, None):
        ks, vs = [], []
        for size, at, n in cases:
            s = rng.normal(0, 1, n)
            s[at] = -np.log(size) if score is None else score
            v = rng.normal(0, 1, (n, 1, d))
            v[at] *= size
            ks.append(scored(rng, q1, s))
            vs.append(v)
        check(gpu, kind, q.astype(np.float32), ks, vs)


@pytest.mark.parametrize("heads,d", [(4, 128), (6, 64)])
@pytest.mark.parametrize("exponent", [-119, -100, 60, 105])
def test_values_all_small_or_all_large(gpu, heads, d, exponent):
    """Rows whose scales all lie near one power of two, down to the smallest normal ones."""
    rng = np.random.default_rng(heads + 1000 + exponent)
    lens = [1, 100, 700]
    ks = [rng.normal(0, 1, (n, 1, d)) for n in lens]
    vs = [rng.normal(0, 1, (n, 1, d)) * 2.0 ** exponent for n in lens]
    got = check(gpu, Q8, rng.normal(0, 1, (3, heads, d)).astype(np.float32), ks, vs)
    assert np.all(np.abs(got).max(-1) > 0.02 * 2.0 ** exponent)


@pytest.mark.parametrize("heads,d", [(4, 128), (8, 128), (1, 64), (6, 64)])
def test_queries_and_keys_far_from_one(gpu, heads, d):
    """Queries of 2^e and 8-bit keys of 2^-e: scores of ordinary size, between queries whose products with one code pass
    fp32's range on either side."""
    rng = np.random.default_rng(heads * d + 3)
    exponents, n = [118, 100, 60, -100, -110, -125], 200
    ks = [rng.normal(0, 1, (n, 1, d)) * 2.0 ** -e for e in exponents]
    vs = [rng.normal(0, 1, (n, 1, d)) for _ in exponents]
    q = rng.normal(0, 1, (len(exponents), heads, d)) * 2.0 ** np.array(exponents, np.float64)[:, None, None]
    q[0, 0] = 0
    if heads > 1:
        q[1, 1] *= 2.0 ** -140  # beside heads of another size
    check(gpu, Q8, q.astype(np.float32), ks, vs)


@pytest.mark.parametrize("heads,d", [(2, 128), (8, 128), (1, 64), (5, 64)])
def test_large_queries_and_keys_in_elements_apart(gpu, heads, d):
    """Queries of 2^120 in one half of the elements and 8-bit keys of 2^100 in the other: every score is 0, every weight
    1 / n, and the outputs are the values' means to within n + 64 roundings and the values' own rounding to 2^-24."""
    rng = np.random.default_rng(heads + d + 4)
    n = 150
    k, q = np.zeros((n, 1, d)), np.zeros((1, heads, d), np.float32)
    k[:, :, d // 2:] = rng.normal(0, 1, (n, 1, d // 2)) * 2.0 ** 100
    q[:, :, :d // 2] = rng.normal(0, 1, (1, heads, d // 2)) * 2.0 ** 120
    pages = Pages(rng, Q8, 1, d, 16, [n])
    hold(pages, 0, k, rng.normal(0, 1, (n, 1, d)))
    kv, table = pages.device(gpu)
    got = attend(gpu, kv, table, [n], q)
    v = pages.rows("v", 0, n)[:, 0]
    assert np.all(np.abs(got[0] - v.mean(0)) <= (n + 64 + 2) * 2.0 ** -24 * np.abs(v).max(-1).mean())


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("heads,d", [(2, 128), (8, 128), (4, 64)])
def test_many_small_weights_beside_a_large_one(gpu, heads, d, kind):
    """Thousands of positions of weight 2^-27 to 2^-34 and one of weight 1, in elements of their own: the small ones'
    sum is there."""
    rng = np.random.default_rng(d + heads)
    q1 = rng.normal(0, 1, d).astype(np.float32)
    lens, at = [3000] * 4 + [40_000], [0, 1500, 2999, 64, 7]
    ks, vs = [], []
    for n, a in zip(lens, at):
        s = -np.log(2.0) * rng.uniform(27, 34, n)
        s[a] = 0
        v = np.zeros((n, 1, d))
        v[:, :, d // 2:] = rng.uniform(0.5, 1, (n, 1, d // 2))
        v[a] = np.concatenate([np.ones(d // 2), np.zeros(d // 2)])
        ks.append(scored(rng, q1, s))
        vs.append(v)
    got = check(gpu, kind, np.repeat(q1[None, None], len(lens), 0).repeat(heads, 1), ks, vs)
    assert np.all(got[..., d // 2:] > 2.0 ** -23)


@pytest.mark.parametrize("heads,d", [(4, 128), (8, 64)])
def test_scores_and_sizes_that_move_together(gpu, heads, d):
    """Scores that rise or fall along the row by 40, against value rows whose sizes fall or rise as much, or twice as
    much; rows of zeros first, last, and everywhere."""
    rng = np.random.default_rng(heads * d)
    q1 = rng.normal(0, 1, d).astype(np.float32)
    n = 900
    up = np.linspace(0, 40, n)
    ks, vs = [], []
    for s, by in ((up, -up), (up[::-1], -up[::-1]), (up, -2 * up), (up[::-1], up), (up, up), (up, 0 * up), (up[::-1], 0 * up)):
        ks.append(scored(rng, q1, s))
        vs.append(rng.normal(0, 1, (n, 1, d)) * np.exp(by)[:, None, None])
    for zero in (slice(0, 200), slice(700, n), slice(0, n)):
        v = rng.normal(0, 1, (n, 1, d))
        v[zero] = 0
        ks.append(scored(rng, q1, up / 10))
        vs.append(v)
    got = check(gpu, Q8, np.repeat(q1[None, None], len(ks), 0).repeat(heads, 1), ks, vs)
    assert np.all(got[-1] == 0)


@pytest.mark.parametrize("kind", [F16, Q8])
def test_the_longest_row_counts_what_it_should(gpu, kind):
    """2^31 - 1 positions of values around 4, over one page again and again, the last slot left out (a NaN).

    The row's 2^25 units of 64 are spread over at least 1024 waves. A lane adds up at most 16 weights of each of its 2^15
    units one after the other, in fp32: 2^19 roundings of half a step; of outputs at most 4 sums a unit: 2^17."""
    rng = np.random.default_rng(36)
    d, page, n = 64, 256, 2 ** 31 - 1
    pages = Pages(rng, kind, 1, d, page, [2 * page], spare=0)
    k, v = rng.normal(0, 1, (2 * page, 1, d)), 4 + 0.1 * rng.normal(0, 1, (2 * page, 1, d))
    v[:, :, ::2] *= -1
    k[-1] = v[-1] = np.nan
    hold(pages, 0, k, v)
    main, last = pages.table[0]
    table = np.full((1, 2 ** 23), main, np.int32)
    table[0, -1] = last
    kv, _ = pages.device(gpu)
    q = rng.normal(0, 1, (1, 2, d)).astype(np.float32)
    got = attend(gpu, kv, gpu.GpuPageTable(dev(table)), [n], q)
    k, v = pages.rows("k", 0, 2 * page - 1)[:, 0], pages.rows("v", 0, 2 * page - 1)[:, 0]
    s = q[0].astype(np.float64) @ k.T / np.sqrt(d)
    w = np.exp(s - s.max(-1, keepdims=True)) * np.where(np.arange(2 * page - 1) < page, 2.0 ** 23 - 1, 1.0)
    want = w @ v / w.sum(-1, keepdims=True)
    assert np.all(np.abs(want) > 3.5)
    assert np.all(np.abs(got[0] / want - 1) <= (2 ** 19 + 2 ** 17) * 2.0 ** -24)
