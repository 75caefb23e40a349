"""The work that the operators of a paged key-value cache are timed on: many conversations served at once, each
with its history in fixed-size pages of a shared pool, held as fp16 or as 8-bit codes with a scale for each row.

  attn   one new token of each conversation attends to its cached history (ragged lengths, grouped query heads)
  qkv    queries and keys normed and rotated, the rotated queries written out, keys and values put into the pages
  put    keys and values put into the pages as they are
  get    cached keys and values read back, into the layout of the contiguous cache or as rows of tokens

A page table [sequences, pages] holds each sequence's pages in order; position p of a sequence is slot p % page of
its page number p // page. Pools are [pages, kv heads, page, head], scales [pages, kv heads, page]. An 8-bit row x is
held as code = round(x / s) with s = max|x| / 127, and stands for code * s; where 8-bit rows are written, what they
stand for is read back in the same pass.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # One conversation early in its course: the smallest attention, all latency.
        {"name": "attn_1x500_f16", "kind": "attn", "type": "f16", "rows": 1, "lo": 500, "hi": 500, "heads": 16, "kv": 8,
         "head": 128, "page": 16},
        # One conversation with a very long history, in 8 bits: few rows, so the length itself is split.
        {"name": "attn_1x32768_q8", "kind": "attn", "type": "q8", "rows": 1, "lo": 32768, "hi": 32768, "heads": 32,
         "kv": 8, "head": 128, "page": 64},
        # A served batch of ordinary conversations, from just begun to long.
        {"name": "attn_32x4096_f16", "kind": "attn", "type": "f16", "rows": 32, "lo": 1, "hi": 4096, "heads": 16,
         "kv": 8, "head": 128, "page": 32},
        # A full server: many conversations, 8-bit pages, four query heads to a kv head.
        {"name": "attn_128x8192_q8", "kind": "attn", "type": "q8", "rows": 128, "lo": 300, "hi": 8192, "heads": 32,
         "kv": 8, "head": 128, "page": 64},
        # Small heads in groups of eight, odd lengths, some rows of the batch still empty.
        {"name": "attn_24x1777_d64_f16", "kind": "attn", "type": "f16", "rows": 24, "lo": 0, "hi": 1777, "heads": 32,
         "kv": 4, "head": 64, "page": 16},
        # One conversation's new token: the smallest write, all latency.
        {"name": "qkv_1_f16", "kind": "qkv", "type": "f16", "rows": 1, "each": 1, "past": 700, "heads": 16, "kv": 8,
         "head": 128, "page": 16},
        # One new token of each conversation of a batch, quantised as it is written.
        {"name": "qkv_64x1_q8", "kind": "qkv", "type": "q8", "rows": 64, "each": 1, "past": 1500, "heads": 32, "kv": 8,
         "head": 128, "page": 64},
        # A long system prompt, quantised as it is written.
        {"name": "qkv_1x2811_q8", "kind": "qkv", "type": "q8", "rows": 1, "each": 2811, "past": 0, "heads": 16, "kv": 8,
         "head": 128, "page": 32},
        # Follow-up turns of odd length for several conversations, keys and values as they come.
        {"name": "put_5x333_f16", "kind": "put", "type": "f16", "rows": 5, "each": 333, "past": 100, "heads": 32,
         "kv": 4, "head": 64, "page": 16},
        # Many prompts put into an 8-bit cache at once.
        {"name": "put_8x1024_q8", "kind": "put", "type": "q8", "rows": 8, "each": 1024, "past": 0, "heads": 16, "kv": 8,
         "head": 128, "page": 128},
        # A long cached prompt taken back into the contiguous cache, for the next prompt's attention.
        {"name": "get_1x2811_q8", "kind": "get", "type": "q8", "rows": 1, "each": 2811, "past": 0, "heads": 16, "kv": 8,
         "head": 128, "page": 32, "to": "cache", "max_seq": 4096},
        # Pieces of several conversations read back as 32-bit rows.
        {"name": "get_6x700_f16", "kind": "get", "type": "f16", "rows": 6, "each": 700, "past": 45, "heads": 16, "kv": 8,
         "head": 128, "page": 16, "to": "rows"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "qkv", "qkv", "put", "get"])
    kv = rng.choice([1, 2, 4, 8, 8])
    case = {"kind": kind, "type": rng.choice(["f16", "q8"]), "kv": kv, "heads": kv * rng.choice([1, 2, 2, 4, 4, 5, 8]),
            "head": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128])}
    if kind == "attn":
        rows = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, min(32768, 260_000 // rows))
        return {**case, "rows": rows, "lo": rng.randint(0, hi), "hi": hi}
    rows = _log_int(rng, 1, 64)
    case.update(rows=rows, each=_log_int(rng, 1, max(1, 8192 // rows)), past=_log_int(rng, 1, 2000) - 1)
    if kind == "get":
        case["to"] = "rows"
        if rows == 1 and rng.random() < 0.7:
            case.update(to="cache", past=0, max_seq=case["each"] + rng.randint(0, 500))
    return case


def _lens(case):
    """The batch's lengths: spread evenly from lo to hi, in mixed order, the same ones for every seed."""
    n, lo, hi = case["rows"], case["lo"], case["hi"]
    got = [lo + round((hi - lo) * i / (n - 1)) if n > 1 else hi for i in range(n)]
    random.Random(n * 1_000_003 + hi).shuffle(got)
    return got


def _pages_of(case):
    """Pages that each sequence holds."""
    if case["kind"] == "attn":
        return [-(-n // case["page"]) for n in _lens(case)]
    return [-(-(case["past"] + case["each"]) // case["page"])] * case["rows"]


def _codes(x):
    """An 8-bit row's codes, as whole numbers in 32 bits, and its scale."""
    s = x.abs().amax(-1) / 127
    s = torch.where(s < torch.finfo(torch.float32).tiny, torch.zeros_like(s), s)
    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    return torch.round(x * inv[..., None]).clamp(-127, 127), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    h = random.Random(int(seed))
    dev = {"device": "cuda"}
    kv, d, page, rows = case["kv"], case["head"], case["page"], case["rows"]

    def normal(*shape):
        return torch.randn(shape, generator=g, **dev)

    # the pages of all sequences, in the order in which a busy pool gives them out; entries behind a sequence's last
    # page hold none
    held = _pages_of(case)
    n_pages = sum(held) + 3
    order = list(range(n_pages))
    h.shuffle(order)
    width = max(held) + 1
    at, table = 0, []
    for n in held:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    s = {"case": case, "table": torch.tensor(table, dtype=torch.int32, **dev)}
    pool = (n_pages, kv, page, d)
    if case["kind"] in ("attn", "get"):
        if case["type"] == "f16":
            s["k"], s["v"] = normal(*pool).half(), normal(*pool).half()
        else:
            s["k"], s["v"] = (torch.randint(-127, 128, pool, generator=g, dtype=torch.int8, **dev) for _ in range(2))
            s["ks"], s["vs"] = ((0.5 + torch.rand(pool[:3], generator=g, **dev)) / 50 for _ in range(2))
    else:
        kind = torch.half if case["type"] == "f16" else torch.int8
        s["k"], s["v"] = (torch.zeros(pool, dtype=kind, **dev) for _ in range(2))
        if case["type"] == "q8":
            s["ks"], s["vs"] = (torch.zeros(pool[:3], **dev) for _ in range(2))
    if case["kind"] == "attn":
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, **dev)
        s["q"] = 1.3 * normal(rows, case["heads"], d)
        s["out"] = torch.zeros_like(s["q"])
    else:
        each = case["each"]
        n = rows * each
        s["pos"] = (torch.arange(each, dtype=torch.int32, **dev) + case["past"]).repeat(rows)
        s["seq"] = torch.arange(rows, dtype=torch.int32, **dev).repeat_interleave(each)
    if case["kind"] in ("qkv", "put"):
        s["xk"], s["xv"] = 2 * normal(n, kv, d), normal(n, kv, d)
        if case["type"] == "q8":
            s["k_back"], s["v_back"] = (torch.zeros((n, kv, d), dtype=torch.half, **dev) for _ in range(2))
    if case["kind"] == "qkv":
        s["xq"] = 2 * normal(n, case["heads"], d)
        s["q_out"] = torch.zeros_like(s["xq"])
        s["q_norm"], s["k_norm"] = 1 + 0.2 * normal(d), 1 + 0.2 * normal(d)
        angle = torch.arange(case["past"] + each, dtype=torch.float64, **dev)[:, None] * THETA ** (
            -torch.arange(0, d, 2, dtype=torch.float64, **dev) / d)
        s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    if case["kind"] == "get":
        if case["to"] == "cache":
            s["k_out"], s["v_out"] = (torch.zeros((kv, case["max_seq"], d), dtype=torch.half, **dev) for _ in range(2))
        else:
            s["k_out"], s["v_out"] = (torch.zeros((n, kv, d), **dev) for _ in range(2))
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program keeps beside its tensors: the checked views of the pool and the table, and a workspace."""
    from rpgbarenginecuda_amd import ops

    c = s["case"]
    s["ops"] = ops
    s["pages"] = ops.GpuPagedKv(s["k"], s["v"], s.get("ks"), s.get("vs"))
    s["of"] = ops.GpuPageTable(s["table"])
    if c["kind"] == "attn":
        s["work"] = torch.zeros(ops.GpuAttentionPagedWorkspace(c["heads"], c["kv"], c["head"]), dtype=torch.uint8,
                                device="cuda")


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    c, ops = s["case"], s["ops"]
    if c["kind"] == "attn":
        ops.GpuAttentionPaged(s["pages"], s["of"], s["lens"], s["q"], c["heads"], c["rows"], s["out"], s["work"])
        return {"out": s["out"]}
    kv, d, n = c["kv"], c["head"], c["rows"] * c["each"]
    if c["kind"] == "get":
        strides = (d, c["max_seq"] * d) if c["to"] == "cache" else (kv * d, d)
        ops.GpuKvReadPaged(s["pages"], s["of"], s["seq"], s["pos"], n, s["k_out"], s["v_out"], *strides)
        return {"k": s["k_out"], "v": s["v_out"]}
    got = {}
    if c["kind"] == "qkv":
        ops.GpuQkNormRopeKvPaged(s["pages"], s["of"], s["seq"], s["pos"], s["xq"], s["xk"], s["xv"], s["q_norm"],
                                 s["k_norm"], c["heads"], s["rope"], s["rope"].shape[0], n, EPS, s["q_out"])
        got["q"] = s["q_out"]
    else:
        ops.GpuKvWritePaged(s["pages"], s["of"], s["seq"], s["pos"], s["xk"], s["xv"], n)
    if c["type"] == "f16":
        return {**got, "k": s["k"], "v": s["v"]}
    ops.GpuKvReadPaged(s["pages"], s["of"], s["seq"], s["pos"], n, s["k_back"], s["v_back"], kv * d, d)
    return {**got, "k": s["k_back"], "v": s["v_back"]}


def _slots(s):
    """Page and slot of each token."""
    page = s["case"]["page"]
    pos = s["pos"].long()
    return s["table"][s["seq"].long(), pos // page].long(), pos % page


def _norm_rope(x, w, rope, pos):
    """Each head's row over its root mean square, times w, rotated in pairs (i, i + half) by its position's angles."""
    d = x.shape[-1]
    mean = x.double().square().sum(-1, keepdim=True) / d
    y = x * (1 / (mean + EPS).sqrt()).float() * w
    a, b = y[..., :d // 2], y[..., d // 2:]
    t = rope[pos.long()][:, None]
    co, si = t[..., :d // 2], t[..., d // 2:]
    return torch.cat([a * co - b * si, b * co + a * si], -1)


def _put_plain(s, name, x):
    """Rows x into the pool `name`, and what then stands there: the pool itself, or the 8-bit rows' values."""
    page, slot = _slots(s)
    if s["case"]["type"] == "f16":
        s[name][page, :, slot] = x.half()
        return s[name]
    code, scale = _codes(x)
    s[name][page, :, slot] = code.to(torch.int8)
    s[name + "s"][page, :, slot] = scale
    return (s[name][page, :, slot].float() * s[name + "s"][page, :, slot][..., None]).half()


def _get_plain(s, name, out):
    page, slot = _slots(s)
    x = s[name][page, :, slot].float()
    if s["case"]["type"] == "q8":
        x = x * s[name + "s"][page, :, slot][..., None]
    if s["case"]["to"] == "cache":
        out[:, :x.shape[0]] = x.transpose(0, 1).to(out.dtype)
    else:
        out.copy_(x)
    return out


def _history(s, name):
    """Every sequence's rows in order, [sequences, kv heads, positions, head], in 32 bits; zeros where there is none."""
    c = s["case"]
    table = s["table"].long().clamp(min=0)
    x = s[name][table].float()
    if c["type"] == "q8":
        x = x * s[name + "s"][table][..., None]
    x = x.transpose(1, 2).reshape(c["rows"], c["kv"], -1, c["head"])
    there = torch.arange(x.shape[2], device=x.device) < s["lens"][:, None]
    return x.masked_fill(~there[:, None, :, None], 0), there


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "qkv":
        q = _norm_rope(s["xq"], s["q_norm"], s["rope"], s["pos"])
        k = _norm_rope(s["xk"], s["k_norm"], s["rope"], s["pos"])
        return {"q": q, "k": _put_plain(s, "k", k), "v": _put_plain(s, "v", s["xv"])}
    if c["kind"] == "put":
        return {"k": _put_plain(s, "k", s["xk"]), "v": _put_plain(s, "v", s["xv"])}
    if c["kind"] == "get":
        return {"k": _get_plain(s, "k", s["k_out"]), "v": _get_plain(s, "v", s["v_out"])}
    k, there = _history(s, "k")
    v, _ = _history(s, "v")
    q = s["q"].view(c["rows"], c["kv"], -1, c["head"])
    score = torch.matmul(q, k.transpose(2, 3)) / math.sqrt(c["head"])
    score = score.masked_fill(~there[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1, total)
    return {"out": out.reshape(c["rows"], c["heads"], c["head"])}


def work(case):
    kv, d, heads, rows = case["kv"], case["head"], case["heads"], case["rows"]
    cell = kv * (2 * d if case["type"] == "f16" else d + 4)  # one position's keys, or values
    if case["kind"] == "attn":
        total = sum(_lens(case))
        return {"bytes": 2 * total * cell + 2 * rows * heads * d * 4 + 4 * (rows + sum(_pages_of(case))),
                "flops": 4 * total * heads * d}
    n = rows * case["each"]
    index = 8 * n + 4 * sum(_pages_of(case))
    if case["kind"] == "get":
        return {"bytes": n * 2 * (cell + kv * d * (2 if case["to"] == "cache" else 4)) + index, "flops": 2 * n * kv * d}
    moved = n * 2 * (cell + kv * d * 4)
    if case["type"] == "q8":
        moved += n * 2 * kv * d * 2  # what the codes stand for, read back
    flops = 8 * n * kv * d
    if case["kind"] == "qkv":
        moved += 2 * n * heads * d * 4 + 4 * d * (case["past"] + case["each"] if rows == 1 else case["each"])
        flops += 8 * n * (heads + kv) * d
    return {"bytes": moved + index, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    kv, d, page, heads = case["kv"], case["head"], case["page"], case["heads"]
    table = s["table"].tolist()

    def rows_of(name, row, first, n):
        """Positions first .. first + n - 1 of a sequence, [positions, kv heads, head]."""
        held = torch.tensor(table[row][first // page:-(-(first + n) // page)], dtype=torch.long, device="cuda")
        x = s[name][held].double()
        if case["type"] == "q8":
            x = x * s[name + "s"][held].double().unsqueeze(3)
        return x.permute(0, 2, 1, 3).flatten(0, 1)[first % page:first % page + n]

    if case["kind"] == "attn":
        out = torch.zeros(case["rows"], heads, d, dtype=torch.float64, device="cuda")
        for row, n in enumerate(_lens(case)):
            if n:
                k, v = (rows_of(name, row, 0, n).repeat_interleave(heads // kv, 1) for name in "kv")
                w = torch.softmax((k * s["q"][row].double()).sum(-1) / d ** 0.5, 0)
                out[row] = (w.unsqueeze(2) * v).sum(0)
        return {"out": out}
    if case["kind"] == "get":
        got = {}
        for name in "kv":
            x = torch.cat([rows_of(name, row, case["past"], case["each"]) for row in range(case["rows"])])
            if case["to"] == "cache":
                full = torch.zeros(kv, case["max_seq"], d, dtype=torch.float64, device="cuda")
                full[:, :len(x)] = x.permute(1, 0, 2)
                x = full
            got[name] = x
        return got

    def turned(x, w):
        x = x.double()
        x = x / ((x * x).mean(-1, keepdim=True) + EPS).sqrt() * w.double()
        t = s["rope"].double()[s["pos"].long()].unsqueeze(1)
        z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * torch.complex(t[..., :d // 2], t[..., d // 2:])
        return torch.cat([z.real, z.imag], -1)

    new = {"k": s["xk"].double(), "v": s["xv"].double()}
    got = {}
    if case["kind"] == "qkv":
        got["q"] = turned(s["xq"], s["q_norm"])
        new["k"] = turned(s["xk"], s["k_norm"])
    for name, x in new.items():
        if case["type"] == "q8":
            step = x.abs().amax(-1, keepdim=True) / 127
            got[name] = (x / step).round() * step
        else:
            got[name] = torch.zeros(s[name].shape, dtype=torch.float64, device="cuda")
            for t, (row, p) in enumerate(zip(s["seq"].tolist(), s["pos"].tolist())):
                got[name][table[row][p // page], :, p % page] = x[t]
    return got
