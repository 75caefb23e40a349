"""A paged KV cache on the host and the operators over it from their definitions, in 64 bits: what the tests of the
paged operators compare with."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24
F16, Q8 = "f16", "q8"


def quantise(x):
    """Codes and scales of fp32 rows, in the fp32 operations that define them."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        finite = np.isfinite(x).all(-1)
        top = np.where(finite, np.abs(x).max(-1), 0).astype(np.float32)
        s = (top * np.float32(1 / 127)).astype(np.float32)
        s = np.where(s < np.finfo(np.float32).tiny, np.float32(0), s)
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
        y = np.where(finite[..., None], x, np.float32(0)) * inv[..., None]
        code = np.clip(np.rint(y), -127, 127).astype(np.int8)
    return code, np.where(finite, s, np.float32(np.nan)).astype(np.float32)


class Pages:
    """Pools filled with `fill` bytes, and a table whose entries past each sequence's pages are `pad`."""

    def __init__(self, rng, kind, n_kv, d, page, lens, spare=3, pad=-1, width=None, fill=0x7F):
        held = [-(-max(n, 0) // page) for n in lens]
        self.kind, self.n_kv, self.d, self.page = kind, n_kv, d, page
        self.n_pages = max(1, sum(held) + spare)
        order = rng.permutation(self.n_pages).astype(np.int32)
        width = max([1] + held) if width is None else width
        self.table = np.full((len(lens), width), pad, np.int32)
        at = 0
        for i, n in enumerate(held):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.n_pages, n_kv, page, d)
        if kind == F16:  # 0x7F7F is a NaN
            self.k, self.v = (np.full(shape, fill * 0x0101, np.uint16) for _ in range(2))
            self.ks = self.vs = None
        else:
            self.k, self.v = (np.full(shape, fill, np.int8) for _ in range(2))
            self.ks, self.vs = (np.full(shape[:3], np.nan, np.float32) for _ in range(2))

    def slot(self, seq, pos):
        return self.table[seq, pos // self.page], pos % self.page

    def put(self, seq, pos, k, v):
        """fp32 rows [n_kv, d] of one position."""
        p, s = self.slot(seq, pos)
        for name, x in (("k", k), ("v", v)):
            if self.kind == F16:
                with np.errstate(over="ignore"):
                    getattr(self, name)[p, :, s] = x.astype(np.float16).view(np.uint16)
            else:
                getattr(self, name)[p, :, s], getattr(self, name + "s")[p, :, s] = quantise(x)

    def fill_random(self, rng, lens, k_amp=1.0):
        """Every held position of every sequence."""
        for i, n in enumerate(lens):
            n = max(n, 0)
            k = rng.normal(0, k_amp, (n, self.n_kv, self.d)).astype(np.float32)
            v = rng.normal(0, 1, (n, self.n_kv, self.d)).astype(np.float32)
            pos = np.arange(n)
            p, s = self.table[i, pos // self.page], pos % self.page
            if self.kind == F16:
                self.k[p, :, s] = k.astype(np.float16).view(np.uint16)
                self.v[p, :, s] = v.astype(np.float16).view(np.uint16)
            else:
                self.k[p, :, s], self.ks[p, :, s] = quantise(k)
                self.v[p, :, s], self.vs[p, :, s] = quantise(v)
        return self

    def rows(self, name, seq, n):
        """What positions [0, n) of a sequence stand for, [n, n_kv, d] float64."""
        pos = np.arange(n)
        p, s = self.table[seq, pos // self.page], pos % self.page
        x = getattr(self, name)[p, :, s]
        if self.kind == F16:
            return x.view(np.float16).astype(np.float64)
        return x.astype(np.float64) * getattr(self, name + "s")[p, :, s].astype(np.float64)[..., None]

    def device(self, ops):
        """(GpuPagedKv, GpuPageTable) on the GPU."""
        import torch

        def up(a):
            if a is None:
                return None
            return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()

        kv = ops.GpuPagedKv(up(self.k), up(self.v), up(self.ks), up(self.vs))
        return kv, ops.GpuPageTable(up(self.table))

    def same_as(self, kv):
        """Whether the device's pools hold these bytes."""
        import torch

        torch.cuda.synchronize()
        mine = [self.k, self.v, self.ks, self.vs]
        return all(a is None or np.array_equal(t.cpu().numpy().view(np.uint8).reshape(-1), a.view(np.uint8).reshape(-1))
                   for a, t in zip(mine, kv.tensors))


def attention(q, k, v):
    """One row: q [heads, d], k and v [n, n_kv, d] -> out [heads, d], and per head max_j sum_d |q_d k_jd| / sqrt(d) and
    max |v|."""
    heads, d = q.shape
    g = heads // k.shape[1]
    if not len(k):
        return np.zeros((heads, d)), np.zeros(heads), np.zeros(heads)
    kk, vv = np.repeat(k, g, 1), np.repeat(v, g, 1)
    q = q.astype(np.float64)
    with np.errstate(all="ignore"):
        s = (kk * q).sum(-1) / np.sqrt(d)
        w = np.exp(s - s.max(0))
        out = (w[..., None] * vv).sum(0) / w.sum(0)[:, None]
    return out, (np.abs(kk * q).sum(-1) / np.sqrt(d)).max(0), np.abs(vv).max((0, 2))


def bound(d, n, smag, vmax):
    """How far a row's output may be from attention()'s, per head.

    A score is an fp32 sum of d products, in which q counts to 2^-21 of each of its elements (two fp16 terms of 11 bits,
    the first cut off: 8 units of 2^-24), then scaled, and for 8-bit keys times the row's scale: an error of at most
    delta = (d + 12) 2^-24 smag. That changes each weight by a factor within e^(+-2 delta), so the output by at most
    (e^(2 delta) - 1) vmax. The exponentials, the weights' own two terms, and the sums over n positions and the merges of
    their shares add (n + 64) 2^-24 vmax. Wrong rows, heads or borders are off by orders of magnitude more."""
    delta = (d + 12) * U * smag
    return (np.expm1(2 * delta) + (n + 64) * U) * vmax + 1e-30


def attention_within(q, k, v, kind):
    """One row of at least one position: attention()'s output and how far from it each element may be, [heads, d] both.

    Weights first. A score is off by delta_j = (d + 12) 2^-24 sum_d |q_d k_jd| / sqrt(d) as at bound(), and by what is cut
    off of queries relative to their row's largest element: half a unit of whole numbers below 2^30, that is 2^-30 of it
    (fp16: below 2^-38), for every |k_jd|. So w_j = p_j / sum p counts for (1 + e_j) w_j, |e_j| <= e^delta_j - 1 and 4
    roundings. With E = sum_j w_j |e_j|: numerators are off by sum_j w_j |e_j v_jd|, the denominator by E, the quotient by
    (sum_j w_j |e_j v_jd| + E A_d) / (1 - E), A_d = sum_j w_j |v_jd|.

    Sums: at most n + 64 roundings of half a step of partial sums no larger than A_d.

    8-bit rows: p_j times the row's scale enters as a whole number whose unit is at most 2^-29 of the largest of its 64
    positions, so that each is off by 2^-30 of that: together 64 times that times a code of 127, for every 64 positions.
    With B = sum_j w_j max_d |v_jd|, of which the largest of 64 is a part: 64 2^-30 B = 2^-24 B. fp16 rows: p_j, at most
    1, enters as two fp16 terms of p_j 2^14, of which the second may end at 2^-24: n 2^-39 / sum p, times max |v|.

    Weights below 2^-126 of the largest (2^-120 with the lag of the maximum) may count as none: n 2^-120 max |v|."""
    heads, d = q.shape
    n, g = len(k), heads // k.shape[1]
    q = q.astype(np.float64)
    out, limit = np.zeros((heads, d)), np.zeros((heads, d))
    for h in range(heads):
        kk, vv = k[:, h // g], v[:, h // g]
        s = kk @ q[h] / np.sqrt(d)
        w = np.exp(s - s.max())
        w /= w.sum()
        a, b = w @ np.abs(vv), w @ np.abs(vv).max(-1)
        cut = 2.0 ** (-30 if kind == Q8 else -38) * np.abs(q[h]).max()
        delta = ((d + 12) * U * np.abs(kk) @ np.abs(q[h]) + cut * np.abs(kk).sum(-1)) / np.sqrt(d)
        we = w * np.expm1(delta)
        out[h] = w @ vv
        limit[h] = (we @ np.abs(vv) + we.sum() * a) / (1 - we.sum()) + (n + 64 + 8) * U * a
        vmax = np.abs(vv).max()
        limit[h] += n * 2.0 ** -120 * vmax + (2.0 ** -24 * b if kind == Q8 else n * 2.0 ** -39 * w.max() * vmax)
    return out, limit
