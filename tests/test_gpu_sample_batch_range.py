"""The choice of a batch's next tokens where settings and logits lie far out: what the definition in 64 bits allows."""
from __future__ import annotations

import numpy as np
import pytest

from test_gpu_sample_batch import check, choose, settings

pytestmark = pytest.mark.gpu


def cut_anywhere(x, t, k, p, m, u):
    """What may come of a row, (token, probability), with every number of tokens that min-p may leave.

    Weights are within 2^-36 of their value, so that those within 2^-35 of min-p's border may be kept or not, the larger
    ones before the smaller; batch_ref.sample tries none, all, and what 64 bits say. (At a temperature of 10^27 a weight is
    less than 1 for every logit but the largest, and 1 in 64 bits for all of them: a min-p of 1 may leave any number.)"""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
    live = np.flatnonzero(x > -np.inf)
    ranked = live[np.argsort(-x[live], kind="stable")]
    ranked = ranked[:k] if k > 0 else ranked
    w = np.exp((x[ranked] - x.max()) / np.float64(t))
    near = len(x) * 2.0 ** -39 + (len(x) * 2.0 ** -52 + 2.0 ** -36) * w.sum()
    upto = np.cumsum(w)
    goals = np.float64(p) * upto[-1] + np.array([-near, 0, near]) if 0 < p < 1 else [np.inf]
    m = min(np.float64(m), 1.0) if m > 0 else 0.0
    for count in {min(len(w), 1 + int(np.searchsorted(upto, g))) for g in goals}:
        sure, most = (max(int((w[:count] >= m * (1 + by)).sum()), 1) for by in (2.0 ** -35, -2.0 ** -35))
        for j in range(sure, max(sure, most) + 1):
            at = np.argsort(ranked[:j])
            sums = np.cumsum(w[:j][at])
            for g in np.float64(u if u > 0 else 0.0) * sums[-1] + np.array([-near, 0, near]):
                i = min(int(np.searchsorted(sums, max(g, 0.0), side="right")), j - 1)
                yield int(ranked[:j][at][i]), w[:j][at][i] / sums[-1]


def check_far(got, x, how):
    """As `check`; rows that it does not take are held to cut_anywhere."""
    for r in range(len(x)):
        try:
            check(got, x, how, look=[r])
        except AssertionError:
            off = 2.0 ** -24 + x.shape[1] * 2.0 ** -39 + 2.0 ** -34
            assert how[0][r] > 0 and any(
                token == got[0][r] and abs(got[1][r] - share) <= share * off + 1e-44
                for token, share in cut_anywhere(x[r], *(v[r] for v in how))), (r, [v[r] for v in how])


@pytest.mark.parametrize("t", [1.0, 50.0, 1e3, 1e5, 1e7, 1e8])
@pytest.mark.parametrize("top", [0.0, -700.0, 3e5])
def test_min_p_next_to_one_at_high_temperatures(gpu, t, top):
    """The border lies among logits of 22 and less below the largest, at a share of it that nears 1 with the temperature."""
    rng = np.random.default_rng(int(t) + int(abs(top)))
    rows, n = 40, 5000
    x = (top - rng.uniform(0, 24, (rows, n))).astype(np.float32)
    m = np.exp(-rng.uniform(0.5, 21, rows) / t).astype(np.float32)
    p = np.where(np.arange(rows) % 3 == 0, 0.9, 1.0)
    k = np.where(np.arange(rows) % 4 == 1, rng.integers(1, n, rows), 0)
    how = settings(rows, t, k, p, m, rng.random(rows))
    check(choose(gpu, x, how), x, how)


def test_settings_of_any_size(gpu):
    """Temperatures of 1e-30 to 1e30 and infinite, top-p and min-p next to their ends, top-k of any number, over rows that
    are flat, steep, tied, masked or of a few values."""
    rng = np.random.default_rng(5)
    for n in (1, 3, 70, 1300, 9000):
        rows = 120
        t = 10.0 ** rng.uniform(-30, 30, rows)
        t[::3] = 10.0 ** rng.uniform(-3, 3, len(t[::3]))
        t[::17] = np.inf
        k = rng.choice([0, 0, 1, 2, n // 2, n, n + 1, 2 ** 31 - 1, -1, -2 ** 31], rows)
        p = rng.choice([1.0, 0.0, 1e-30, 1e-6, 0.3, 0.9, 1 - 2.0 ** -24, 2.0, -1.0, np.nan], rows)
        m = rng.choice([0.0, 0.0, 1e-40, 1e-30, 1e-3, 0.5, 1 - 2.0 ** -24, 1.0, 3.0, -1.0, np.nan], rows)
        x = rng.normal(0, 1, (rows, n)) * 10.0 ** rng.uniform(-20, 20, (rows, 1))
        x[::4] = rng.normal(0, 3, x[::4].shape)
        x[1::4] = np.round(rng.normal(0, 2, x[1::4].shape))
        x[rng.random(x.shape) < 0.02] = -np.inf
        x[5::11] = rng.choice([-np.inf, 0.0, -0.0, 1.0, np.nan, np.inf, -3.4e38, 3.4e38], x[5::11].shape)
        x = x.astype(np.float32)
        how = settings(rows, t, k, p, m, rng.choice([0.0, 0.999999, 1.0, 0.5, *rng.random(8)], rows))
        check_far(choose(gpu, x, how), x, how)
