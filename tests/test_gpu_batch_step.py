"""A step of many conversations as a server runs it, every operator on what the one before it left: queries and keys rotated
at each row's position by a scaled table, keys and values into the pages, attention over shared and own pages, logits, the
next tokens, whose embeddings are the next step's input. Each stage is held to 64 bits from the bits that it was given."""
from __future__ import annotations

import numpy as np
import pytest

from batch_ref import sample
from paged_ref import F16, Q8, U, Pages, attention, bound, quantise

pytestmark = pytest.mark.gpu

HEADS, N_KV, VOCAB, WIDTH, FAR = 8, 2, 5003, 96, 4096


def dev(a, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype))).cuda()


def host(t):
    import torch

    torch.cuda.synchronize()
    return t.cpu().numpy()


class Server:
    """Four conversations behind a prompt of 6 pages, three behind another of 2, and a place of the batch that nobody has
    (its seq_id is negative). Conversations grow by a token a step."""

    def __init__(self, gpu, kind, d):
        import torch

        rng = np.random.default_rng(d)
        self.gpu, self.kind, self.d, self.page = gpu, kind, d, 16
        shared, own = [6] * 4 + [2] * 3, [15, 0, 40, 16, 1, 100, 31]
        self.lens = [s * self.page + n for s, n in zip(shared, own)]
        self.seq = [0, 1, 2, 3, -1, 4, 5, 6]
        self.room = [n + 8 for n in self.lens]
        self.pages = Pages(rng, kind, N_KV, d, self.page, self.room)
        for first, last, n in ((0, 4, 6), (4, 7, 2)):
            self.pages.table[first:last, :n] = self.pages.table[first, :n]
        self.pages.fill_random(rng, self.lens)
        self.kv, self.table = self.pages.device(gpu)
        self.n = len(self.seq)
        self.rope = dev(gpu.build_rope_table_scaled(d, 1e4, FAR, "yarn", 4.0, 128))
        normal = [rng.normal(0, 1, s).astype(np.float32) for s in ((VOCAB, WIDTH), (WIDTH, (HEADS + 2 * N_KV) * d), (HEADS * d, VOCAB))]
        self.embedding, self.qkv, self.head = dev(normal[0]), dev(normal[1] / 10), dev(normal[2] / 5)
        f, i = torch.float32, torch.int32
        self.x = torch.zeros(self.n, WIDTH, device="cuda")
        self.q, self.k, self.v = (torch.zeros(self.n, h, d, device="cuda") for h in (HEADS, N_KV, N_KV))
        self.out = torch.zeros(self.n, HEADS, d, device="cuda")
        self.logits = torch.zeros(self.n, VOCAB, device="cuda")
        self.tokens, self.probs = torch.zeros(self.n, dtype=i, device="cuda"), torch.zeros(self.n, device="cuda")
        self.seq_ids = dev(self.seq, np.int32)
        self.pos, self.len, self.u = (torch.zeros(self.n, dtype=t, device="cuda") for t in (i, i, f))
        self.starts, self.shared = dev([0, 4, 8], np.int32), dev([6, 2], np.int32)
        self.how = [dev([0.8, 1.0, 0, 1.3, 1, 0.5, 1, 2], np.float32), dev([0, 40, 0, 0, 5, 0, 1, 3000], np.int32),
                    dev([0.9, 1, 0.5, 0.95, 1, 0.8, 1, 0.99], np.float32), dev([0, 0, 0, 0.05, 0, 0, 0, 0], np.float32)]
        self.work = torch.zeros(gpu.GpuAttentionPagedSharedWorkspace(HEADS, N_KV, d, self.n), dtype=torch.uint8, device="cuda")
        self.sample_work = torch.empty(gpu.GpuSampleBatchWorkspace(self.n, VOCAB), dtype=torch.uint8, device="cuda")

    def project(self):
        """What a model's layers stand for here: torch's products, of this step's embeddings."""
        import torch

        all_of = torch.mm(self.x, self.qkv).view(self.n, HEADS + 2 * N_KV, self.d)
        for to, a, b in ((self.q, 0, HEADS), (self.k, HEADS, HEADS + N_KV), (self.v, HEADS + N_KV, HEADS + 2 * N_KV)):
            to.copy_(all_of[:, a:b])

    def attend(self):
        g = self.gpu
        g.GpuRopeRows(self.q, self.k, HEADS, N_KV, self.d, self.d, False, self.rope, FAR, self.pos, self.n, self.q, self.k)
        g.GpuKvWritePaged(self.kv, self.table, self.seq_ids, self.pos, self.k, self.v, self.n)
        g.GpuAttentionPagedShared(self.kv, self.table, self.len, self.starts, self.shared, self.q, HEADS, self.n, self.out,
                                  self.work, seq_ids=self.seq_ids, least_saving=0)

    def choose(self):
        t, k, p, m = self.how
        self.gpu.GpuSampleBatch(self.logits, self.n, VOCAB, self.u, self.tokens, self.sample_work, t, k, p, m, self.probs)

    def set(self, step, rng):
        """This step's places and random numbers."""
        at = [self.lens[s] + step if s >= 0 else 0 for s in self.seq]
        self.pos.copy_(dev(at, np.int32))
        self.len.copy_(dev(np.array(at) + 1, np.int32))
        self.u.copy_(dev(rng.random(self.n), np.float32))
        return at


def rotated(x, table, at):
    """By the table's own numbers, and how far three roundings may be off."""
    half = x.shape[-1] // 2
    x, co, si = x.astype(np.float64), table[at, None, :half].astype(np.float64), table[at, None, half:].astype(np.float64)
    a, b = x[..., :half], x[..., half:]
    size = np.abs(a * co) + np.abs(b * si), np.abs(b * co) + np.abs(a * si)
    return np.concatenate([a * co - b * si, b * co + a * si], -1), 3 * U * np.concatenate(size, -1) + 1e-44


@pytest.mark.parametrize("kind,d", [(F16, 128), (Q8, 128), (F16, 64), (Q8, 64)])
def test_steps(gpu, kind, d):
    import torch

    s = Server(gpu, kind, d)
    rng = np.random.default_rng(7)
    table = host(s.rope)
    s.x.copy_(s.embedding[torch.arange(s.n, device="cuda")])
    live = [r for r in range(s.n) if s.seq[r] >= 0]
    for step in range(8):
        at = s.set(step, rng)
        s.project()
        before = {name: host(getattr(s, name)).copy() for name in "qkv"}
        s.out.fill_(7.0)
        s.attend()
        q, k = host(s.q), host(s.k)
        for name, got in (("q", q), ("k", k)):
            want, off = rotated(before[name], table, at)
            assert np.all(np.abs(got - want) <= off)
        for r in live:
            s.pages.put(s.seq[r], at[r], k[r], before["v"][r])
        assert s.pages.same_as(s.kv)
        out = host(s.out)
        for r in range(s.n):
            if s.seq[r] < 0:
                assert np.all(out[r] == 7.0)
                continue
            want, smag, vmax = attention(q[r], s.pages.rows("k", s.seq[r], at[r] + 1), s.pages.rows("v", s.seq[r], at[r] + 1))
            assert np.all(np.abs(out[r] - want).max(-1) <= bound(d, at[r] + 1, smag, vmax))
        torch.mm(s.out.view(s.n, -1), s.head, out=s.logits)
        s.choose()
        logits, tokens, probs = host(s.logits), host(s.tokens), host(s.probs)
        for r in range(s.n):
            may = sample(logits[r], *(host(v)[r] for v in s.how), host(s.u)[r])
            assert any(t == tokens[r] and abs(p - probs[r]) <= 1e-6 * p for t, p in may), (step, r)
        s.x.copy_(s.embedding[s.tokens.long()])
    assert len(set(tokens[live])) > 1


@pytest.mark.parametrize("kind,d", [(F16, 128), (Q8, 64)])
def test_captured_steps(gpu, kind, d):
    """A step's operators in one graph, replayed for every step of a generation between another server's eager ones."""
    import torch

    a, b = Server(gpu, kind, d), Server(gpu, kind, d)
    stream, graph, tail = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream), gpu.ScopedEngineStream(stream):
        a.attend()
    with torch.cuda.graph(tail, stream=stream), gpu.ScopedEngineStream(stream):
        a.choose()
    for s in (a, b):
        s.x.copy_(s.embedding[torch.arange(s.n, device="cuda")])
    for step in range(8):
        for s in (a, b):
            s.set(step, np.random.default_rng(step))
            s.project()
        b.attend()
        graph.replay()
        for s in (a, b):
            torch.mm(s.out.view(s.n, -1), s.head, out=s.logits)
        tail.replay()
        b.choose()
        assert np.array_equal(host(a.out), host(b.out)) and np.array_equal(host(a.q), host(b.q))
        assert np.array_equal(host(a.tokens), host(b.tokens)) and np.array_equal(host(a.probs), host(b.probs))
        for s in (a, b):
            s.x.copy_(s.embedding[s.tokens.long()])
    for x, y in zip(a.kv.tensors, b.kv.tensors):
        assert x is None or np.array_equal(host(x).view(np.uint8), host(y).view(np.uint8))


@pytest.mark.parametrize("kind", [F16, Q8])
def test_scaled_tables_for_the_fused_writer(gpu, kind):
    """GpuQkNormRopeKvPaged takes a scaled table as any other: the bits of keys that it caches are those that the norms'
    rows, rotated by GpuRopeRows, would give within a few roundings."""
    import torch

    rng = np.random.default_rng(3)
    n, d, page = 37, 128, 32
    pages = Pages(rng, kind, N_KV, d, page, [FAR])
    kv, table = pages.device(gpu)
    rope = dev(gpu.build_rope_table_scaled(d, 1e4, FAR, "yarn", 4.0, 1024))
    pos = rng.permutation(FAR)[:n].astype(np.int32)
    q, k, v = (rng.normal(0, 1, (n, h, d)).astype(np.float32) for h in (HEADS, N_KV, N_KV))
    ones, eps = np.ones(d, np.float32), 1e-6
    seq, q_out = dev(np.zeros(n), np.int32), torch.zeros(n, HEADS, d, device="cuda")
    gpu.GpuQkNormRopeKvPaged(kv, table, seq, dev(pos), dev(q), dev(k), dev(v), dev(ones), dev(ones), HEADS, rope, FAR, n, eps,
                             q_out)

    def normed(x):
        x = x.astype(np.float64)
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)

    want, size = rotated(normed(q), host(rope), pos)
    # the norm: d products and sums (d / 2 units of the mean square at most, half of that of its root), and four roundings
    assert np.all(np.abs(host(q_out) - want) <= (d / 4 + 4) / 3 * size + size)
    want, size = rotated(normed(k), host(rope), pos)
    off = (d / 4 + 4) / 3 * size + size
    back = torch.zeros(2, n, N_KV, d, device="cuda")
    gpu.GpuKvReadPaged(kv, table, seq, dev(pos), n, back[0], back[1], N_KV * d, d)
    got_k, got_v = host(back)
    if kind == F16:
        assert np.all(np.abs(got_k - want) <= off + 2.0 ** -11 * (np.abs(want) + off) + 2.0 ** -25)
        assert np.array_equal(got_v, v.astype(np.float16).astype(np.float32))
    else:  # half a code and its scale's roundings
        top = np.abs(want).max(-1, keepdims=True) + off.max(-1, keepdims=True)
        assert np.all(np.abs(got_k - want) <= off + top / 127 * (0.5 + 127 * 4 * U))
        code, scale = quantise(v)
        assert np.array_equal(got_v, code * scale[..., None])


def test_tensors_of_another_device_are_refused(gpu, monkeypatch):
    import torch

    x, i = torch.zeros(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    work = torch.zeros(gpu.GpuSampleBatchWorkspace(4, 8), dtype=torch.uint8, device="cuda")
    monkeypatch.setattr(gpu, "_current_device", lambda: 1)
    with pytest.raises(gpu.RpgError, match="q is on cuda:0, which is not the current device"):
        gpu.GpuRopeRows(x, None, 1, 0, 8, 8, False, x, 4, i, 4, x, None)
    with pytest.raises(gpu.RpgError, match="logits is on cuda:0, which is not the current device"):
        gpu.GpuSampleBatch(x, 4, 8, x, i, work)
    far = 1 << 40
    with pytest.raises(gpu.RpgError, match="workspace is on cuda:0, which is not the current device"):
        gpu.GpuSampleBatch(far, 4, 8, far, far, work)
