"""The choice of a batch's next tokens on the GPU against its definition in 64 bits (batch_ref.sample): sizes, settings,
ties, masks, random numbers at their ends, streams and graphs."""
from __future__ import annotations

import numpy as np
import pytest

from batch_ref import sample

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
LOW = -np.finfo(np.float32).max


def dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def host(t):
    import torch

    torch.cuda.synchronize()
    return t.cpu().numpy()


def workspace(gpu, rows, n):
    import torch

    return torch.full((gpu.GpuSampleBatchWorkspace(rows, n),), 255, dtype=torch.uint8, device="cuda")  # of any contents


def settings(rows, t=1.0, k=0, p=1.0, m=0.0, u=0.5):
    return [np.broadcast_to(np.asarray(v, kind), rows).copy()
            for v, kind in ((t, np.float32), (k, np.int32), (p, np.float32), (m, np.float32), (u, np.float32))]


def choose(gpu, x, how, work=None):
    """Tokens and probabilities of the rows of x (a device tensor or an array)."""
    import torch

    rows, n = x.shape
    t, k, p, m, u = (dev(v) for v in how)
    tokens = torch.full((rows + 2,), -77, dtype=torch.int32, device="cuda")
    probs = torch.full((rows + 2,), 77.0, device="cuda")
    xd = x if isinstance(x, torch.Tensor) else dev(x)
    gpu.GpuSampleBatch(xd, rows, n, u, tokens, workspace(gpu, rows, n) if work is None else work, t, k, p, m, probs)
    tokens, probs = host(tokens), host(probs)
    assert np.all(tokens[rows:] == -77) and np.all(probs[rows:] == 77)
    return tokens[:rows], probs[:rows]


def check(got, x, how, exact_sums=False, look=None):
    """A share is off by half a step of fp32, 2^-24, by what the sum of weights, which is at least 1, is (n 2^-39 + 2^-36, as
    batch_ref.sample says), and by the weight's own 2^-36."""
    for r in range(len(x)) if look is None else look:
        allowed = sample(x[r], *(v[r] for v in how), exact_sums=exact_sums)
        right = [p for token, p in allowed if token == got[0][r]]
        assert right, (r, int(got[0][r]), allowed, [v[r] for v in how])
        off = 2.0 ** -24 + x.shape[1] * 2.0 ** -39 + 2.0 ** -34
        assert any(abs(got[1][r] - p) <= p * off + 1e-44 for p in right), (r, float(got[1][r]), right)


MIX = [(0.7, 0, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 0.98, 0.0), (0.8, 40, 0.9, 0.0), (1.1, 0, 1.0, 0.05),
       (1.0, 0, 1.0, 0.0), (1.0, 5, 1.0, 0.0), (2.0, 1000, 0.5, 0.01), (0.3, 3, 0.999, 0.3), (1.0, 1, 1.0, 0.0),
       (5.0, 0, 0.9, 0.0), (1.0, 20000, 0.99, 0.0), (0.05, 0, 0.9, 0.0)]


def mixed(rng, rows, u=None):
    t, k, p, m = zip(*(MIX[i % len(MIX)] for i in range(rows)))
    return settings(rows, t, k, p, m, rng.random(rows).astype(np.float32) if u is None else u)


def logits(rng, rows, n, spread=2.2):
    x = rng.normal(0, spread, (rows, n)).astype(np.float32)
    for r in range(rows):
        at = rng.integers(0, n, min(n, 40))
        x[r, at] += rng.uniform(3, 9, len(at)).astype(np.float32)
        if r % 3 == 1:
            x[r, rng.random(n) < 0.05] = -np.inf
    return x


@pytest.mark.parametrize("n", [1, 2, 3, 5, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4095, 4096, 4097, 8191, 12289, 31999,
                               151936, 200003])
def test_sizes(gpu, n):
    rng = np.random.default_rng(n)
    rows = 26 if n < 100_000 else 13
    x, how = logits(rng, rows, n), mixed(rng, rows)
    got = choose(gpu, x, how)
    check(got, x, how)
    again = choose(gpu, x, how)
    assert np.array_equal(got[0], again[0]) and np.array_equal(got[1], again[1])


@pytest.mark.parametrize("n", [300_007, (1 << 22) - 1, 1 << 22])
def test_vocabularies_of_many_slices(gpu, n):
    """More slices than a wave has lanes, up to the largest vocabulary there is."""
    rng = np.random.default_rng(n)
    x, how = logits(rng, 13, n), mixed(rng, 13)
    check(choose(gpu, x, how), x, how)


@pytest.mark.parametrize("alike", [1, 2, 63, 64, 65, 1024, 1025, 8191, 8192, 8193])
def test_so_many_values_around_the_cut(gpu, alike):
    """From where a wave's lanes hold the values that lie between the cut's borders to where LDS no longer does: all within
    an eighth of an octave, every third with a double, beside others far below."""
    rng = np.random.default_rng(alike)
    rows, n = 26, 30_011
    x = rng.normal(-30, 1, (rows, n)).astype(np.float32)
    for r in range(rows):
        at = rng.permutation(n)[:alike]
        x[r, at] = rng.uniform(4.0, 4.03, alike).astype(np.float32)
        x[r, at[1::3]] = x[r, at[:len(at[1::3])]]
    p, k = (0.6, 1.0, 0.9, 0.03, 1.0), (0, 1 + alike // 2, 2 * alike // 3 + 1, 0, alike)
    how = settings(rows, 1.0, [k[r % 5] for r in range(rows)], [p[r % 5] for r in range(rows)],
                   [0.0 if r % 3 else 0.99 for r in range(rows)], rng.random(rows).astype(np.float32))
    check(choose(gpu, x, how), x, how)


def test_rows_past_32_bit_offsets(gpu):
    import torch

    rng = np.random.default_rng(21)
    n, stride = 5003, (1 << 30) + 77
    x, (t, k, p, m, u) = logits(rng, 2, n), mixed(rng, 2)
    far = torch.zeros(stride + n, device="cuda")
    far[:n], far[stride:] = dev(x[0]), dev(x[1])
    tokens, probs = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    gpu.GpuSampleBatch(far, 2, n, dev(u), tokens, workspace(gpu, 2, n), dev(t), dev(k), dev(p), dev(m), probs, row_stride=stride)
    check((host(tokens), host(probs)), x, (t, k, p, m, u))


@pytest.mark.parametrize("spread", [0.01, 1.0, 8.0])
def test_flat_and_steep(gpu, spread):
    """From where nearly every token is kept to where a few are."""
    rng = np.random.default_rng(int(spread * 100))
    n, rows = 50021, 26
    x = rng.normal(0, spread, (rows, n)).astype(np.float32)
    how = mixed(rng, rows)
    check(choose(gpu, x, how), x, how)


def test_many_random_numbers(gpu):
    """One row many times, over all of u's range: each token's share of the draws is its share of the weight."""
    rng = np.random.default_rng(2)
    n, rows = 4000, 2048
    x = np.repeat(logits(rng, 1, n), rows, 0)
    how = settings(rows, 0.9, 0, 0.9, 0.0, (np.arange(rows) + 0.5) / rows)
    got = choose(gpu, x, how)
    check(got, x, how, look=range(0, rows, 31))
    tokens, counts = np.unique(got[0], return_counts=True)
    assert np.all(np.diff(got[0]) >= 0)  # the index order of the walk
    for token, count in zip(tokens, counts):
        share = got[1][got[0] == token][0]
        assert abs(count / rows - share) <= 1.01 / rows


def test_random_numbers_at_their_ends(gpu):
    us = np.array([0.0, 2.0 ** -149, 2.0 ** -126, 1e-9, 1 - 2.0 ** -24, 1.0, 1.5, INF, -1.0, -INF, NAN, -0.0], np.float32)
    rng = np.random.default_rng(3)
    for n in (1, 7, 9000):
        x = np.repeat(logits(rng, 1, n), len(us), 0)
        x[:, 0] = -np.inf if n > 1 else 1.0
        for t, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (30.0, 0, 1.0, 0.2)):
            how = settings(len(us), t, k, p, m, us)
            inside = settings(len(us), t, k, p, m)
            inside[4] = np.array([0.0, 2.0 ** -149, 2.0 ** -126, 1e-9, 1 - 2.0 ** -24, *[1 - 2.0 ** -53] * 3, 0, 0, 0, 0])
            check(choose(gpu, x, how), x, inside)


# Weights of equal logits are 1 each, and sums of them exact: no room at the borders. u takes the last kept one.
TIES = [
    # values, t, k, p, m, kept indexes
    ([1, 1, 1, 1, 1, 1], 1.0, 0, 0.5, 0.0, [0, 1, 2]),
    ([1, 1, 1, 1, 1, 1], 1.0, 4, 0.5, 0.0, [0, 1]),
    ([1, 1, 1, 1, 1, 1], 1.0, 4, 1.0, 0.0, [0, 1, 2, 3]),
    ([0, 1, 0, 1, 1, 0], 1.0, 2, 1.0, 0.0, [1, 3]),
    ([0, 1, 0, 1, 1, 0], INF, 4, 1.0, 0.0, [0, 1, 3, 4]),
    ([0, 1, 0, 1, 1, 0], INF, 5, 1.0, 0.0, [0, 1, 2, 3, 4]),
    ([0, 1, 0, 1, 1, 0], INF, 5, 0.8, 0.0, [0, 1, 2, 3, 4]),  # fl(0.8) is above 0.8
    ([0, 1, 0, 1, 1, 0], INF, 5, 0.75, 0.0, [0, 1, 3, 4]),
    ([0, 1, 0, 1, 1, 0], 1.0, 0, 1.0, 1.0, [1, 3, 4]),
    ([0, 1, 0, 1, 1, 0], 1.0, 0, 1.0, 7.0, [1, 3, 4]),
    ([0.0, -0.0, 0.0, -0.0], 1.0, 2, 1.0, 0.0, [0, 1]),      # the zeros are alike
    ([-0.0, 0.0, -0.0, 0.0], 1.0, 0, 0.75, 0.0, [0, 1, 2]),
    ([-INF, 2, 2, -INF, 2, NAN], 1.0, 5, 0.6, 0.0, [1, 2]),
    ([5, 5, 5, 5], INF, 3, 1.0, 0.0, [0, 1, 2]),
    ([1, 2, 3, -INF], INF, 0, 1.0, 0.0, [0, 1, 2]),          # all of one weight
    ([LOW, LOW, LOW], 1.0, 0, 1.0, 0.0, [0, 1, 2]),          # a mask of the lowest value over everything
    ([LOW, 3, LOW, 3], 1.0, 0, 1.0, 0.0, [1, 3]),
    ([LOW, 3, LOW, 3], 1e30, 0, 1.0, 1e-5, [1, 3]),
    ([INF, 3, INF, NAN], 1.0, 0, 1.0, 0.0, [0, 2]),
    ([INF, -INF, INF, NAN], INF, 1, 1.0, 0.0, [0]),
    ([-INF, LOW, NAN], 0.5, 0, 0.5, 0.5, [1]),
    ([3, 3.0000002, 3], 1e-30, 0, 1.0, 0.0, [1]),
    ([1, 1, 1, 1], 1.0, 0, 1e-30, 0.0, [0]),
    ([1, 1, 1, 1], 1.0, 0, 2.0 ** -149, 0.0, [0]),
    ([1, 1, 1, 1], 1.0, 0, 0.0, 0.0, [0, 1, 2, 3]),           # out of (0, 1): off
    ([1, 1, 1, 1], 1.0, 0, NAN, NAN, [0, 1, 2, 3]),
    ([1, 1, 1, 1], 1.0, -3, -1.0, -1.0, [0, 1, 2, 3]),
    ([1, 1, 1, 1], 1.0, 2 ** 31 - 1, 2.0, 0.0, [0, 1, 2, 3]),
    ([1, 1, 1, 1], 1.0, -2 ** 31, 1.0, 0.0, [0, 1, 2, 3]),
    ([1, 4, 4], 0.0, 0, 1.0, 0.0, [1]),
    ([1, 4, 4], -2.0, 0, 1.0, 0.0, [1]),
    ([1, 4, 4], NAN, 0, 1.0, 0.0, [1]),
    ([1, 4, 4], -0.0, 0, 1.0, 0.0, [1]),
]


@pytest.mark.parametrize("stretch", [1, 700, 5000])
def test_ties_and_values_that_are_no_numbers(gpu, stretch):
    """Every u between two kept tokens; stretched rows have -inf in between, so that ties lie in parts far apart."""
    for values, t, k, p, m, kept in TIES:
        n = len(values) * stretch
        x = np.full((len(kept), n), -np.inf, np.float32)
        x[:, ::stretch] = np.array(values, np.float32)
        how = settings(len(kept), t, k, p, m, (np.arange(len(kept)) + 0.5) / len(kept))
        tokens, probs = choose(gpu, x, how)
        assert list(tokens) == [i * stretch for i in kept], (values, t, k, p, m)
        assert np.all(np.abs(probs - 1 / len(kept)) <= 2.0 ** -24), (values, probs)
        check((tokens, probs), x, how, exact_sums=True)


def test_ties_over_a_whole_vocabulary(gpu):
    """A few values only: every border lies among thousands that are alike."""
    rng = np.random.default_rng(8)
    n, rows = 60000, 39
    x = rng.integers(0, 5, (rows, n)).astype(np.float32)
    x[5] = 0
    how = mixed(rng, rows)
    how[1][:] = np.where(how[1] > 0, rng.integers(1, n, rows), 0)
    check(choose(gpu, x, how), x, how)


def test_rows_with_nothing_to_choose(gpu):
    x = np.full((4, 5000), -np.inf, np.float32)
    x[1] = NAN
    x[2, 4999] = -3.0
    x[3, ::2] = NAN
    for t in (1.0, 0.0):
        tokens, probs = choose(gpu, x, settings(4, t, 10, 0.9, 0.1))
        assert list(tokens) == [-1, -1, 4999, -1] and list(probs) == [0, 0, 1, 0]


def test_strides_odd_addresses_and_what_is_left_out(gpu):
    """Rows further apart than they are long, from any 4-byte address; settings not given; no probabilities."""
    import torch

    rng = np.random.default_rng(9)
    rows, n, stride = 5, 9001, 9010
    x = logits(rng, rows, n)
    for at in range(4):
        room = torch.full((rows * stride + 8,), 99.0, device="cuda")
        view = room[at:at + rows * stride].view(rows, stride)
        view[:, :n] = dev(x)
        how = settings(rows, 1.0, 0, 1.0, 0.0, rng.random(rows))
        tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        flat = room[at:at + (rows - 1) * stride + n]
        gpu.GpuSampleBatch(flat, rows, n, dev(how[4]), tokens, workspace(gpu, rows, n), row_stride=stride)
        allowed = [[a for a, _ in sample(x[r], *(v[r] for v in how))] for r in range(rows)]
        assert all(t in a for t, a in zip(host(tokens), allowed))


def test_one_workspace_for_calls_of_all_sizes(gpu):
    rng = np.random.default_rng(10)
    work = workspace(gpu, 30, 40000)
    for rows, n in ((30, 40000), (1, 5), (13, 39999), (30, 100), (2, 40000), (30, 40000)):
        x, how = logits(rng, rows, n), mixed(rng, rows)
        check(choose(gpu, x, how, work), x, how)


def test_two_streams_at_once(gpu):
    import torch

    rng = np.random.default_rng(11)
    rows, n = 16, 60001
    x, how = logits(rng, rows, n), mixed(rng, rows)
    want = choose(gpu, x, how)
    streams = [torch.cuda.Stream() for _ in range(2)]
    xs, works = [dev(x) for _ in streams], [workspace(gpu, rows, n) for _ in streams]
    hows = [[dev(v) for v in how] for _ in streams]
    outs = [[(torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")) for _ in range(4)]
            for _ in streams]
    torch.cuda.synchronize()
    for i in range(4):
        for s, xd, w, (t, k, p, m, u), o in zip(streams, xs, works, hows, outs):
            with gpu.ScopedEngineStream(s):
                gpu.GpuSampleBatch(xd, rows, n, u, o[i][0], w, t, k, p, m, o[i][1])
    torch.cuda.synchronize()
    for o in outs:
        for tokens, probs in o:
            assert np.array_equal(host(tokens), want[0]) and np.array_equal(host(probs), want[1])


def test_captured(gpu):
    """Logits, settings and random numbers are read at replay; replays and eager calls between them agree."""
    import torch

    rng = np.random.default_rng(12)
    rows, n = 13, 33333
    work, other = workspace(gpu, rows, n), workspace(gpu, rows, n)
    xd = torch.zeros(rows, n, device="cuda")
    held = [dev(v) for v in mixed(rng, rows)]
    tokens, probs = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
    t, k, p, m, u = held
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        gpu.GpuSampleBatch(xd, rows, n, u, tokens, work, t, k, p, m, probs)
    for i in range(6):
        x, how = logits(rng, rows, n, (2.2, 0.3)[i % 2]), mixed(rng, rows)
        how = [np.roll(v, i) if j < 4 else v for j, v in enumerate(how)]
        xd.copy_(dev(x))
        for a, b in zip(held, how):
            a.copy_(dev(b))
        graph.replay()
        got = host(tokens), host(probs)
        check(got, x, how)
        eager = choose(gpu, x, how, other)
        assert np.array_equal(got[0], eager[0]) and np.array_equal(got[1], eager[1])


def test_settings_of_the_one_row_sampler(gpu):
    """With the counter's random number and no ties, the token that GpuSampleToken takes."""
    import torch

    rng = np.random.default_rng(13)
    n, rows, seed = 151936, 6, 11
    x = logits(rng, rows, n)
    x[x == -np.inf] = -40.0
    us = np.array([gpu.DevCounterUniform(seed, c) for c in range(rows)], np.float32)
    how = settings(rows, 0.7, 0, 0.95, 0.0, us)
    got = choose(gpu, x, how)
    probs, idx = torch.zeros(n, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    for r in range(rows):
        gpu.GpuSampleToken(dev(x[r]), n, gpu.SampleOptions(0.7, 0, 0.95), seed, r, probs, idx)
        assert int(host(idx)[0]) == got[0][r]
