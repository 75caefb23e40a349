"""The operators of a step of many conversations from their definitions, in 64 bits: what their tests compare with."""
from __future__ import annotations

import math

import numpy as np


def sample(x, t, k, p, m, u, exact_sums=False):
    """What may come of one row: a list of (token, probability).

    Weights are within 2^-36 of their value and rounded to units of 2^-38 of the largest: a sum of n is off by n 2^-39 and
    2^-36 of it at most, and the sums here by n 2^-52 of their value. Where a border is nearer than that, either side of it
    is allowed; exact_sums (for weights that are small whole numbers of a power of two) leaves no such room."""
    n = len(x)
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64)) + 0.0
    live = np.flatnonzero(x > -np.inf)
    if not len(live):
        return [(-1, 0.0)]
    top = x.max()
    ranked = live[np.argsort(-x[live], kind="stable")]
    if not t > 0:
        return [(int(ranked[0]), 1.0)]
    if k > 0:
        ranked = ranked[:k]
    with np.errstate(all="ignore"):
        w = np.exp(np.where(x[ranked] == top, 0.0, (x[ranked] - top) / np.float64(t)))
    w = np.where(np.isnan(w), 0.0, w)
    near = 0.0 if exact_sums else n * 2.0 ** -39 + (n * 2.0 ** -52 + 2.0 ** -36) * w.sum()
    upto = np.cumsum(w)
    counts = {len(w)}
    if 0 < p < 1:
        goal = np.float64(p) * upto[-1]
        counts = {min(len(w), 1 + int(np.searchsorted(upto, g))) for g in (goal - near, goal, goal + near)}
    least = {0.0}
    if m > 0:
        least = {min(np.float64(m), 1.0) * f for f in ((1.0,) if exact_sums else (1 - 2.0 ** -35, 1.0, 1 + 2.0 ** -35))}
        least = {min(v, 1.0) for v in least}
    found = []
    u = u if u > 0 else 0.0
    for count in counts:
        for v in least:
            kept = ranked[:count][w[:count] >= v]
            at = np.argsort(kept)
            tokens, mine = kept[at], w[:count][w[:count] >= v][at]
            sums = np.cumsum(mine)
            goal = np.float64(u) * sums[-1]
            for g in {goal - near, goal, goal + near}:
                last = int(np.flatnonzero(mine > 0)[-1])
                i = min(int(np.searchsorted(sums, max(g, 0.0), side="right")), last)
                if mine[i] == 0:  # a goal of 0 in front of weights of 0
                    i = int(np.flatnonzero(mine > 0)[0])
                found.append((int(tokens[i]), mine[i] / sums[-1]))
    return found


def rope(x, angles, by, rot, interleaved):
    """x [n, heads, d] with its first rot elements rotated by angles [n, rot / 2] and multiplied by `by`."""
    x = np.asarray(x, np.float64)
    out = x.copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    co, si = by * np.cos(angles)[:, None], by * np.sin(angles)[:, None]
    out[..., a] = x[..., a] * co - x[..., b] * si
    out[..., b] = x[..., b] * co + x[..., a] * si
    return out


def frequencies(rot, theta, kind, factor=1.0, original=0, fast=32.0, slow=1.0):
    """Angles a position of the rot / 2 pairs, and what cos and sin are multiplied by."""
    i = np.arange(rot // 2, dtype=np.float64)
    if kind == "ntk" and rot > 2:
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-2 * i / rot)
    if kind == "linear":
        return f / factor, 1.0
    if kind == "yarn":
        def pair(turns):
            return rot / 2 * math.log(original / (turns * 2 * math.pi)) / math.log(theta)

        lo, hi = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f * (ramp / factor + 1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0
