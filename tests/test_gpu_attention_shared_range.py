"""Attention of a batch that shares its beginnings, where values, scores, queries or keys differ widely in size: what the
operator over rows by themselves is held to (test_gpu_attention_paged_range.py), at shared positions."""
from __future__ import annotations

import numpy as np
import pytest

from paged_ref import F16, Q8, Pages, attention_within
from test_gpu_attention_paged_range import hold, scored
from test_gpu_attention_shared import attend

pytestmark = pytest.mark.gpu


def shared(gpu, kind, q, ks, vs, copies, page=16):
    """Rows q [n, heads, d] over sequences of keys ks[i] and values vs[i], each asked for `copies` times: a group of as many
    rows, which shares all whole pages. Outputs [n, copies, heads, d], and the pages."""
    lens = [len(k) for k in ks]
    n, d, n_kv = len(lens), q.shape[-1], ks[0].shape[1]
    pages = Pages(np.random.default_rng(1), kind, n_kv, d, page, lens)
    for i, (k, v) in enumerate(zip(ks, vs)):
        hold(pages, i, k, v)
    kv, table = pages.device(gpu)
    seqs = np.repeat(np.arange(n), copies)
    got = attend(gpu, kv, table, np.repeat(lens, copies), np.arange(n + 1) * copies, [m // page for m in lens],
                 np.repeat(np.asarray(q, np.float32), copies, 0), seq_ids=seqs)
    return got.reshape(n, copies, *q.shape[1:]), pages


def check(gpu, kind, q, ks, vs, copies, page=16):
    got, pages = shared(gpu, kind, q, ks, vs, copies, page)
    for r in range(len(ks)):
        n = len(ks[r])
        want, limit = attention_within(q[r], pages.rows("k", r, n), pages.rows("v", r, n), kind)
        worst = (np.abs(got[r] - want).max(0) / np.maximum(limit, 1e-300)).max()
        assert worst <= 1, (r, n)
    return got


# heads of one kv head, d, copies: tiles of up to 16, 32, 64 and 128 columns, of which a wave takes 32, 32, 64 and 128 keys of
# a step in turn
TILES = [(4, 128, 1), (4, 64, 8), (8, 128, 8), (8, 64, 16), (4, 128, 40)]


@pytest.mark.parametrize("d", [128, 64])
@pytest.mark.parametrize("rows,group", [(4, 4), (8, 4), (16, 4), (32, 4)])
def test_large_value_rows_of_early_keys(gpu, rows, group, d):
    """Value rows 2^R larger than the others, of scores R + 12 octaves lower, in every second step of 128 positions and in
    the first 32 positions of the others: they come first, and count for a 2^-12th. There are more units than workgroups, so
    that a wave meets steps of both kinds."""
    rng = np.random.default_rng(rows + d)
    n_kv, n, page = 64, 768, 16
    pages = Pages(rng, Q8, n_kv, d, page, [n], spare=0)
    pos = np.arange(n)
    early = (pos // 128 % 2 == 0) | (pos % 128 < 32)
    k, v = rng.normal(0, 0.1, (n, n_kv, d)), rng.normal(0, 1, (n, n_kv, d))
    k[early] = 0
    k[early, :, 0] = -1
    hold(pages, 0, k, v)
    p, s = pages.table[0, pos // page], pos % page
    ks, vs = pages.ks.copy(), pages.vs.copy()
    q = rng.normal(0, 0.1, (rows, n_kv * group, d)).astype(np.float32)
    q[:, :, 0] = 4
    for octaves in (0, 20, 28, 36, 44, 60):
        pages.ks, pages.vs = ks.copy(), vs.copy()
        pages.ks[p[early], :, s[early]] *= np.float32((octaves + 12) * np.log(2) * np.sqrt(d) / 4)
        pages.vs[p[early], :, s[early]] *= np.float32(2.0 ** octaves)
        kv, table = pages.device(gpu)
        got = attend(gpu, kv, table, [n] * rows, [0, rows], [n // page], q, seq_ids=[0] * rows)
        kk, vv = pages.rows("k", 0, n), pages.rows("v", 0, n)
        for h in (0, 7, 20, 41, 63):
            at = slice(h * group, (h + 1) * group)
            for r in (0, rows // 2, rows - 1):
                want, limit = attention_within(q[r, at], kk[:, h:h + 1], vv[:, h:h + 1], Q8)
                worst = (np.abs(got[r, at] - want) / limit).max()
                assert worst <= 1, (octaves, h, r)


@pytest.mark.parametrize("heads,d,copies", TILES)
def test_scores_and_sizes_that_move_together(gpu, heads, d, copies):
    """Scores that rise or fall along the row by 40, against value rows whose sizes fall or rise as much, or twice as
    much; rows of zeros first, last, and everywhere."""
    rng = np.random.default_rng(heads * d + copies)
    q1 = rng.normal(0, 1, d).astype(np.float32)
    n = 896
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
    got = check(gpu, Q8, np.repeat(q1[None, None], len(ks), 0).repeat(heads, 1), ks, vs, copies)
    assert np.all(got[-1] == 0)


@pytest.mark.parametrize("heads,d,copies", TILES)
def test_a_large_row_of_no_weight(gpu, heads, d, copies):
    """One value row far larger than all others, of no weight or of a weight that makes it count as much as they do, in
    the first, a middle and the last position."""
    rng = np.random.default_rng(heads + d + copies)
    cases = [(size, at, n) for size in (1e3, 1e6, 1e9, 1e30) for at in (0, 70, -1) for n in (128, 512)]
    q1 = rng.normal(0, 1, d).astype(np.float32)
    q = np.repeat(q1[None], len(cases), 0)[:, None] * (1 + 0.01 * rng.normal(0, 1, (len(cases), heads, 1)))
    for score in (-150.0, -60.0, None):
        ks, vs = [], []
        for size, at, n in cases:
            s = rng.normal(0, 1, n)
            s[at] = -np.log(size) if score is None else score
            v = rng.normal(0, 1, (n, 1, d))
            v[at] *= size
            ks.append(scored(rng, q1, s))
            vs.append(v)
        check(gpu, Q8, q.astype(np.float32), ks, vs, copies)


@pytest.mark.parametrize("heads,d,copies", TILES)
@pytest.mark.parametrize("exponent", [-119, -100, 60, 105])
def test_values_all_small_or_all_large(gpu, heads, d, copies, exponent):
    """Rows whose scales all lie near one power of two, down to the smallest normal ones."""
    rng = np.random.default_rng(heads + 1000 + exponent)
    lens = [16, 100, 704]
    ks = [rng.normal(0, 1, (n, 1, d)) for n in lens]
    vs = [rng.normal(0, 1, (n, 1, d)) * 2.0 ** exponent for n in lens]
    got = check(gpu, Q8, rng.normal(0, 1, (3, heads, d)).astype(np.float32), ks, vs, copies)
    assert np.all(np.abs(got).max(-1) > 0.02 * 2.0 ** exponent)


@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("heads,d,copies", TILES)
def test_scores_of_any_size(gpu, heads, d, copies, kind):
    """Scores of 2^23 to 2^100 octaves: every second key has the score S, of bits that are the same in all of them, the
    others S / 2. Those of the higher score count alike and the rest for nothing, so that the output is the mean of their
    values, to within n + 64 roundings, the weights' and values' own (8) and, over 8-bit pages, 2^-24 of what it is made of."""
    rng = np.random.default_rng(heads + d + copies)
    exponents = [23.0, 25.3, 26.6, 27.5, 28.2, 31.5, 40.0, 60.0, 100.0]
    k0 = rng.normal(0, 1, d).astype(np.float32)
    n, own = 384, 5
    odd = np.arange(n) % 2 == 1
    k = np.where(odd[:, None], k0, k0 / 2)[:, None]
    cases = []  # keys, values, the positions that count, the exponent
    for e in exponents:
        for sign, behind in ((1, 0), (-1, 0), (1, own), (-1, own)):
            best = np.flatnonzero(odd if sign > 0 else ~odd) if sign > 0 or not behind else np.arange(n, n + own)
            cases.append((np.concatenate([sign * k, np.zeros((behind, 1, d))]), rng.normal(0, 1, (n + behind, 1, d)), best, e))
    by = np.array([2.0 ** c[3] * np.sqrt(d) / (float(k0.astype(np.float64) @ k0) * np.log2(np.e)) for c in cases])
    q = by[:, None, None] * k0 * (1 + np.arange(heads)[:, None] / 16)
    got, pages = shared(gpu, kind, q, [c[0] for c in cases], [c[1] for c in cases], copies)
    for r, (k, v, best, e) in enumerate(cases):
        v = pages.rows("v", r, len(k))[best, 0]
        worst = np.abs(got[r] - v.mean(0)).max() / ((n + own + 64 + 8 + 1) * 2.0 ** -24 * np.abs(v).max(-1).mean())
        assert worst <= 1, (e, r % 4)


@pytest.mark.parametrize("exponent", [-30.4, -33.4, -35.6, -37.4])
@pytest.mark.parametrize("kind", [F16, Q8])
@pytest.mark.parametrize("heads,d,copies", TILES)
def test_small_weights_that_are_all_alike(gpu, heads, d, copies, kind, exponent):
    """One weight of 1 and all others of 2^exponent, in elements of their own: what is rounded in one is rounded in all."""
    q = np.zeros((2, heads, d), np.float32)
    q[..., 0] = np.sqrt(d)
    ks, vs = [], []
    for n in (128, 1024):
        k, v = np.zeros((n, 1, d)), np.zeros((n, 1, d))
        k[:, :, 0] = exponent * np.log(2)
        k[77] = 0
        v[:, :, d // 2:] = 1
        v[77] = np.concatenate([np.ones(d // 2), np.zeros(d // 2)])
        ks.append(k)
        vs.append(v)
    check(gpu, kind, q, ks, vs, copies)


@pytest.mark.parametrize("heads,d,copies", TILES)
def test_queries_and_keys_far_from_one(gpu, heads, d, copies):
    """Queries of 2^e and 8-bit keys of 2^-e, and down to 2^-20 of that: scores of ordinary size, between queries whose
    products with one code pass fp32's range on either side."""
    rng = np.random.default_rng(heads * d + 3)
    exponents, n = [118, 100, 60, -60, -80, -100, -110, -125], 208
    sizes = 2.0 ** rng.integers(-20, 1, (n, 1, 1))
    sizes[rng.permutation(n)[:60]] = 1
    ks = [rng.normal(0, 1, (n, 1, d)) * sizes ** (e < 0) * 2.0 ** -e for e in exponents]
    vs = [rng.normal(0, 1, (n, 1, d)) for _ in exponents]
    q = rng.normal(0, 1, (len(exponents), heads, d)) * 2.0 ** np.array(exponents, np.float64)[:, None, None]
    q[0, 0] = 0
    q[1, 1] *= 2.0 ** -140  # beside heads of another size
    check(gpu, Q8, q.astype(np.float32), ks, vs, copies)


@pytest.mark.parametrize("heads,d,copies", TILES)
@pytest.mark.parametrize("of_q,of_k", [(120, 100), (-10, 125), (-120, 125), (120, -100)])
def test_large_queries_and_keys_in_elements_apart(gpu, heads, d, copies, of_q, of_k):
    """Queries in one half of the elements and 8-bit keys in the other: every score is 0, every weight 1 / n, and the outputs
    are the values' means to within n + 64 roundings and the values' own rounding to 2^-24."""
    rng = np.random.default_rng(heads + d + 4)
    n = 144
    k, q = np.zeros((n, 1, d)), np.zeros((1, heads, d), np.float32)
    k[:, :, d // 2:] = rng.normal(0, 1, (n, 1, d // 2)) * 2.0 ** of_k
    q[:, :, :d // 2] = rng.normal(0, 1, (1, heads, d // 2)) * 2.0 ** of_q
    got, pages = shared(gpu, Q8, q, [k], [rng.normal(0, 1, (n, 1, d))], copies)
    v = pages.rows("v", 0, n)[:, 0]
    assert np.abs(got[0] - v.mean(0)).max() <= (n + 64 + 2) * 2.0 ** -24 * np.abs(v).max(-1).mean()
