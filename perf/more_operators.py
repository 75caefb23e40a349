"""The work that the operators of a step of many conversations are timed on, from the projections to the next tokens:

  attn    one new token of each conversation attends to its paged history, where groups of conversations have the same
          beginning (a world's description, a character's): its pages are attended to once for the group
  sample  the next token of every conversation, each with its own temperature, top-k, top-p and min-p, from given
          uniform random numbers
  rope    queries and keys rotated at any positions, in pairs (i, i + half) or (2 i, 2 i + 1), the whole of a head or its
          first part, with frequencies scaled for long contexts

Attention: pools are [pages, kv heads, page, head], fp16 or 8-bit codes with scales [pages, kv heads, page]; a page table
[sequences, pages] holds each sequence's pages in order, and the sequences of a group begin with the same pages.

Sampling, for a row x of logits: tokens in the order of falling x, of two that are alike the lower one first; with weights
exp((x - max x) / temperature), kept are the first top_k (0: all), of these the fewest first ones that hold top_p of their
weight (1: all), and of these those of at least min_p of the largest weight. The token is the first, in the order of the
vocabulary, up to which the kept ones' weights add up to more than u times their sum. At temperature 0 it is the first.
Given back with it is its share of the kept weight.
"""
from __future__ import annotations

import math
import random

import torch

own = False

THETA = 1e6


def listed():
    return [
        # Two conversations just begun behind a short common prompt: the smallest attention, all latency.
        {"name": "attn_2x384_f16", "kind": "attn", "type": "f16", "rows": 2, "groups": 1, "shared": 384, "lo": 1,
         "hi": 116, "idle": 0, "heads": 16, "kv": 8, "head": 128, "page": 16},
        # A batch of ordinary conversations behind one long prompt.
        {"name": "attn_32x2816_f16", "kind": "attn", "type": "f16", "rows": 32, "groups": 1, "shared": 2816, "lo": 1,
         "hi": 1024, "idle": 0, "heads": 16, "kv": 8, "head": 128, "page": 32},
        # A full server whose conversations all have one very long beginning, in 8 bits, four query heads to a kv head.
        {"name": "attn_128x8192_q8", "kind": "attn", "type": "q8", "rows": 128, "groups": 1, "shared": 8192, "lo": 1,
         "hi": 2048, "idle": 0, "heads": 32, "kv": 8, "head": 128, "page": 64},
        # A few conversations behind a whole book, in 8 bits: the prefix's length itself is split.
        {"name": "attn_8x32768_q8", "kind": "attn", "type": "q8", "rows": 8, "groups": 1, "shared": 32768, "lo": 1,
         "hi": 512, "idle": 0, "heads": 32, "kv": 8, "head": 128, "page": 64},
        # Small heads in groups of eight, three characters with a prompt each, odd lengths, some rows of the batch idle.
        {"name": "attn_24x1008_d64_f16", "kind": "attn", "type": "f16", "rows": 24, "groups": 3, "shared": 1008, "lo": 0,
         "hi": 333, "idle": 3, "heads": 32, "kv": 4, "head": 64, "page": 16},
        # One conversation's next token with the engine's usual settings: the smallest sampling, all latency.
        {"name": "sample_1x151936", "kind": "sample", "style": "nucleus", "rows": 1, "vocab": 151936},
        # A batch where every conversation has its own settings, some of them greedy.
        {"name": "sample_32x151936_mixed", "kind": "sample", "style": "mixed", "rows": 32, "vocab": 151936},
        # A full server at a high temperature, where the cut is far down.
        {"name": "sample_128x151936_hot", "kind": "sample", "style": "hot", "rows": 128, "vocab": 151936},
        # A smaller vocabulary of odd size with top-k and top-p.
        {"name": "sample_48x31999_topk", "kind": "sample", "style": "topk", "rows": 48, "vocab": 31999},
        # One conversation's new token far behind the length that the model was trained on.
        {"name": "rope_1_yarn", "kind": "rope", "rows": 1, "heads": 16, "kv": 8, "head": 128, "rot": 128,
         "inter": False, "scaling": "yarn", "factor": 4.0, "original": 16384, "far": 65536},
        # A long prompt of one conversation.
        {"name": "rope_2811_yarn", "kind": "rope", "rows": 2811, "heads": 16, "kv": 8, "head": 128, "rot": 128,
         "inter": False, "scaling": "yarn", "factor": 2.0, "original": 16384, "far": 32768},
        # Several prompts at once, neighbours in pairs, half of each head, positions divided.
        {"name": "rope_9001_inter_part", "kind": "rope", "rows": 9001, "heads": 32, "kv": 8, "head": 128, "rot": 64,
         "inter": True, "scaling": "linear", "factor": 8.0, "original": 4096, "far": 32768},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "sample", "sample", "rope"])
    if kind == "sample":
        vocab = rng.choice([151936, _log_int(rng, 2, 200_000)])
        return {"kind": kind, "style": rng.choice(["nucleus", "mixed", "mixed", "hot", "topk", "flat"]), "vocab": vocab,
                "rows": _log_int(rng, 1, max(1, min(128, 128 * 151936 // vocab)))}
    kv = rng.choice([1, 2, 4, 8, 8])
    heads = kv * rng.choice([1, 2, 2, 4, 4, 5, 8])
    if kind == "rope":
        head = rng.choice([64, 96, 128, 128])
        return {"kind": kind, "rows": _log_int(rng, 1, min(9000, 9000 * 40 // (heads + kv))), "heads": heads, "kv": kv, "head": head,
                "rot": rng.choice([head, head, head // 2, 2 * rng.randint(1, head // 2)]),
                "inter": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "ntk", "yarn"]),
                "factor": rng.choice([2.0, 4.0, 8.0, 3.5]), "original": rng.choice([4096, 16384, 32768]),
                "far": _log_int(rng, 64, 65536)}
    rows = _log_int(rng, 1, 128)
    head = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    shared = _log_int(rng, 1, min(32768, 128 * 8192 * 32 // (rows * heads)) // page) * page
    hi = _log_int(rng, 1, min(2048, 200_000 // rows))
    return {"kind": kind, "type": rng.choice(["f16", "q8"]), "rows": rows, "groups": rng.randint(1, min(4, rows)),
            "shared": shared, "lo": rng.randint(0, hi), "hi": hi, "idle": rng.randint(0, rows // 4), "heads": heads,
            "kv": kv, "head": head, "page": page}


# ------------------------------------------------------------------ what a program has in hand


def _batch(case):
    """Of each row its group and its length, of each group its first row and its shared pages: the same for every seed."""
    n, groups, lo, hi, page = (case[k] for k in ("rows", "groups", "lo", "hi", "page"))
    h = random.Random(n * 1_000_003 + hi)
    starts = [n * g // groups for g in range(groups + 1)]
    # the last group has all of the shared length, those before it less
    pages = [max(1, case["shared"] // page * (g + 2) // (groups + 1)) for g in range(groups)]
    group = [g for g in range(groups) for _ in range(starts[g], starts[g + 1])]
    own_len = [lo + round((hi - lo) * i / (n - 1)) if n > 1 else hi for i in range(n)]
    h.shuffle(own_len)
    idle = set(h.sample(range(n), case["idle"]))
    lens = [0 if r in idle else pages[group[r]] * page + own_len[r] for r in range(n)]
    return starts, pages, group, lens


def _prepare_attn(case, g, h):
    dev = {"device": "cuda"}
    kv, d, page, n = case["kv"], case["head"], case["page"], case["rows"]
    starts, shared, group, lens = _batch(case)
    held = [max(0, -(-lens[r] // page) - shared[group[r]]) for r in range(n)]
    n_pages = sum(shared) + sum(held) + 3
    order = list(range(n_pages))
    h.shuffle(order)
    width = max(shared) + max(held) + 1
    at, common, table = 0, [], []
    for c in shared:
        common.append(order[at:at + c])
        at += c
    for r in range(n):
        row = common[group[r]] + order[at:at + held[r]] if lens[r] else []
        at += held[r]
        table.append(row + [-1] * (width - len(row)))
    s = {"lens": torch.tensor(lens, dtype=torch.int32, **dev), "table": torch.tensor(table, dtype=torch.int32, **dev),
         "group_rows": torch.tensor(starts, dtype=torch.int32, **dev),
         "group_pages": torch.tensor(shared, dtype=torch.int32, **dev),
         "q": 1.3 * torch.randn((n, case["heads"], d), generator=g, **dev)}
    s["out"] = torch.zeros_like(s["q"])
    pool = (n_pages, kv, page, d)
    if case["type"] == "f16":
        s["k"], s["v"] = (torch.randn(pool, generator=g, **dev).half() for _ in range(2))
    else:
        s["k"], s["v"] = (torch.randint(-127, 128, pool, generator=g, dtype=torch.int8, **dev) for _ in range(2))
        s["ks"], s["vs"] = ((0.5 + torch.rand(pool[:3], generator=g, **dev)) / 50 for _ in range(2))
    return s


def _prepare_sample(case, g, h):
    """Logits with a broad body and some dozens of likely tokens, as a model's are; in some rows tokens are ruled out."""
    n, rows, dev = case["vocab"], case["rows"], {"device": "cuda"}
    x = (1.0 if case["style"] == "flat" else 2.2) * torch.randn((rows, n), generator=g, **dev)
    if case["style"] != "flat":
        likely = min(50, n)
        where = torch.randint(0, n, (rows, likely), generator=g, **dev)
        x.scatter_add_(1, where, 3 + 6 * torch.rand((rows, likely), generator=g, **dev))
    banned = torch.rand((rows, n), generator=g, **dev) < 0.03
    x[banned & (torch.arange(rows, **dev) % 3 == 1)[:, None]] = -math.inf
    per_row = []
    for _ in range(rows):
        style = h.choice(["greedy", "nucleus", "hot", "topk", "minp", "plain"]) if case["style"] == "mixed" else case["style"]
        per_row.append({"greedy": (0.0, 0, 1.0, 0.0), "nucleus": (0.7, 0, 0.95, 0.0), "hot": (1.3, 0, 0.98, 0.0),
                        "topk": (0.8, 40, 0.9, 0.0), "minp": (1.1, 0, 1.0, 0.05), "plain": (1.0, 0, 1.0, 0.0),
                        "flat": (1.0, 0, 0.95, 0.0)}[style])
    t, k, p, m = zip(*per_row)
    s = {"x": x, "u": torch.rand(rows, generator=g, **dev), "temperature": torch.tensor(t, **dev),
         "top_k": torch.tensor(k, dtype=torch.int32, **dev), "top_p": torch.tensor(p, **dev),
         "min_p": torch.tensor(m, **dev)}
    s["token"] = torch.zeros(rows, dtype=torch.int32, **dev)
    s["prob"] = torch.zeros(rows, **dev)
    return s


def _prepare_rope(case, g, h):
    n, d, dev = case["rows"], case["head"], {"device": "cuda"}
    first = h.randrange(0, max(1, case["far"] - n + 1))
    pos = (torch.arange(n, **dev) + first) % case["far"]
    s = {"pos": pos.int(), "q": 2 * torch.randn((n, case["heads"], d), generator=g, **dev),
         "k": 2 * torch.randn((n, case["kv"], d), generator=g, **dev)}
    s["q_out"], s["k_out"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    h = random.Random(int(seed))
    s = {"attn": _prepare_attn, "sample": _prepare_sample, "rope": _prepare_rope}[case["kind"]](case, g, h)
    s["case"] = case
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program keeps beside its tensors: checked views of the pages, a workspace, the table of rotations."""
    from rpgbarenginecuda_amd import ops

    c = s["case"]
    s["ops"] = ops
    if c["kind"] == "attn":
        s["pages"] = ops.GpuPagedKv(s["k"], s["v"], s.get("ks"), s.get("vs"))
        s["of"] = ops.GpuPageTable(s["table"])
        need = ops.GpuAttentionPagedSharedWorkspace(c["heads"], c["kv"], c["head"], c["rows"])
    elif c["kind"] == "sample":
        need = ops.GpuSampleBatchWorkspace(c["rows"], c["vocab"])
    else:
        tab = ops.build_rope_table_scaled(c["rot"], THETA, c["far"], c["scaling"], c["factor"], c["original"])
        s["rope"] = torch.from_numpy(tab).cuda()
        return
    s["work"] = torch.zeros(need, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------ one pass


def run(s):
    kind = s["case"]["kind"]
    if own:
        return {"attn": _own_attn, "sample": _own_sample, "rope": _own_rope}[kind](s)
    return {"attn": _plain_attn, "sample": _plain_sample, "rope": _plain_rope}[kind](s)


def _own_attn(s):
    c = s["case"]
    s["ops"].GpuAttentionPagedShared(s["pages"], s["of"], s["lens"], s["group_rows"], s["group_pages"], s["q"], c["heads"],
                                     c["rows"], s["out"], s["work"])
    return {"out": s["out"]}


def _own_sample(s):
    c = s["case"]
    s["ops"].GpuSampleBatch(s["x"], c["rows"], c["vocab"], s["u"], s["token"], s["work"], temperature=s["temperature"],
                            top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], probs=s["prob"])
    return {"token": s["token"], "prob": s["prob"]}


def _own_rope(s):
    c = s["case"]
    s["ops"].GpuRopeRows(s["q"], s["k"], c["heads"], c["kv"], c["head"], c["rot"], c["inter"], s["rope"], c["far"],
                         s["pos"], c["rows"], s["q_out"], s["k_out"])
    return {"q": s["q_out"], "k": s["k_out"]}


def _rows_plain(s, name, pages):
    """The rows of some pages in order, [..., kv heads, positions, head], in 32 bits."""
    x = s[name][pages].float()
    if s["case"]["type"] == "q8":
        x = x * s[name + "s"][pages][..., None]
    return x.transpose(-4, -3).flatten(-3, -2)


def _plain_attn(s):
    c = s["case"]
    kv, d, page = c["kv"], c["head"], c["page"]
    starts, shared, _, lens = _batch(c)
    out = torch.zeros_like(s["q"])
    for g, n_shared in enumerate(shared):
        a, b = starts[g], starts[g + 1]
        live = [r for r in range(a, b) if lens[r]]
        if not live:
            continue
        n = len(live)
        rows = torch.tensor(live, device="cuda")
        q = s["q"][rows].view(n, kv, -1, d)
        table = s["table"][rows].long()
        # the shared positions once, every conversation's queries over them
        k, v = (_rows_plain(s, name, table[0, :n_shared]) for name in "kv")
        flat = q.transpose(0, 1).reshape(kv, -1, d)
        first = torch.matmul(flat, k.transpose(1, 2)) / math.sqrt(d)
        first = first.view(kv, n, -1, first.shape[-1]).transpose(0, 1)
        # each one's own
        most = max(0, max(-(-lens[r] // page) for r in live) - n_shared)
        mine = table[:, n_shared:n_shared + most].clamp(min=0)
        k2, v2 = (_rows_plain(s, name, mine) for name in "kv")
        there = torch.arange(most * page, device="cuda") < (s["lens"][rows] - n_shared * page)[:, None]
        k2, v2 = (x.masked_fill(~there[:, None, :, None], 0) for x in (k2, v2))
        second = torch.matmul(q, k2.transpose(2, 3)) / math.sqrt(d)
        second = second.masked_fill(~there[:, None, None], -math.inf)
        top = first.amax(-1, keepdim=True)
        if most:
            top = torch.maximum(top, second.amax(-1, keepdim=True))
        p, p2 = torch.exp(first - top), torch.exp(second - top)
        o = torch.matmul(p.transpose(0, 1).reshape(kv, -1, p.shape[-1]), v).view(kv, n, -1, d).transpose(0, 1)
        o = (o + torch.matmul(p2, v2)) / (p.sum(-1, keepdim=True) + p2.sum(-1, keepdim=True))
        out[rows] = o.reshape(n, c["heads"], d)
    return {"out": out}


def _plain_sample(s):
    n = s["case"]["vocab"]
    t = s["temperature"].double()[:, None]
    greedy = t <= 0
    x, order = torch.sort(s["x"].double(), dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, 1, t))
    place = torch.arange(n, device="cuda")
    k = s["top_k"].long()[:, None]
    w = torch.where((k > 0) & (place >= k), 0, w)
    upto = w.cumsum(1)
    p = s["top_p"].double()[:, None]
    w = torch.where((p < 1) & (upto - w >= p * upto[:, -1:]), 0, w)
    w = torch.where(w < s["min_p"].double()[:, None], 0, w)
    w = torch.where(greedy & (place > 0), 0, w)
    kept = torch.zeros_like(w).scatter_(1, order, w)  # in the order of the vocabulary
    upto = kept.cumsum(1)
    token = (upto <= s["u"].double()[:, None] * upto[:, -1:]).sum(1, keepdim=True).clamp(max=n - 1)
    share = kept.gather(1, token) / upto[:, -1:]
    return {"token": token[:, 0].int(), "prob": share[:, 0].float()}


def _frequencies(c):
    """The angle of each pair a position, in 64 bits, and what the rotated elements are multiplied by."""
    rot, factor = c["rot"], c["factor"]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device="cuda")
    if c["scaling"] == "ntk" and rot > 2:
        return (THETA * factor ** (rot / (rot - 2))) ** (-i / rot), 1.0
    f = THETA ** (-i / rot)
    if c["scaling"] == "linear":
        return f / factor, 1.0
    if c["scaling"] == "yarn":
        # pairs that turn more than 32 times within the original length stay, those that turn less than once are slowed
        def pair(turns):
            return rot * math.log(c["original"] / (turns * 2 * math.pi)) / (2 * math.log(THETA))

        lo, hi = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1
    return f, 1.0


def _plain_rope(s):
    c = s["case"]
    rot = c["rot"]
    f, by = _frequencies(c)
    angle = s["pos"].double()[:, None] * f
    co, si = ((by * t).float()[:, None] for t in (angle.cos(), angle.sin()))
    got = {}
    for name in "qk":
        x = s[name]
        y = x.clone()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if c["inter"] else (slice(0, rot // 2), slice(rot // 2, rot))
        y[..., a] = x[..., a] * co - x[..., b] * si
        y[..., b] = x[..., b] * co + x[..., a] * si
        got[name] = y
    return got


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["kind"] == "sample":
        return {"bytes": case["rows"] * (4 * case["vocab"] + 28), "flops": 4 * case["rows"] * case["vocab"]}
    d, heads, kv, n = case["head"], case["heads"], case["kv"], case["rows"]
    if case["kind"] == "rope":
        return {"bytes": 8 * n * (heads + kv) * d + 4 * min(n, case["far"]) * case["rot"] + 4 * n,
                "flops": 3 * n * (heads + kv) * case["rot"]}
    _, shared, group, lens = _batch(case)
    cell = kv * (2 * d if case["type"] == "f16" else d + 4)  # one position's keys, or values
    live = [r for r in range(n) if lens[r]]
    held = sum(shared[g] for g in {group[r] for r in live})
    once = held * case["page"] + sum(lens[r] - shared[group[r]] * case["page"] for r in live)
    pages = held + sum(-(-lens[r] // case["page"]) - shared[group[r]] for r in live)
    return {"bytes": 2 * once * cell + 8 * n * heads * d + 4 * (pages + n + 2 * case["groups"] + 1),
            "flops": 4 * sum(lens) * heads * d}


# ------------------------------------------------------------------ from the definitions, in 64 bits


def _exact_attn(case, s):
    heads, kv, d, page = case["heads"], case["kv"], case["head"], case["page"]
    out = torch.zeros(case["rows"], heads, d, dtype=torch.float64, device="cuda")
    table = s["table"].tolist()
    for row, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        held = torch.tensor(table[row][:-(-n // page)], device="cuda")
        k, v = (s[name][held].double() for name in "kv")
        if case["type"] == "q8":
            k, v = k * s["ks"][held].double().unsqueeze(3), v * s["vs"][held].double().unsqueeze(3)
        k, v = (x.permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :n] for x in (k, v))
        for h in range(kv):
            mine = slice(h * (heads // kv), (h + 1) * (heads // kv))
            weight = torch.softmax(s["q"][row, mine].double() @ k[h].t().contiguous() / d ** 0.5, 1)
            out[row, mine] = weight @ v[h]
    return {"out": out}


def _exact_sample(case, s):
    import numpy as np

    x, u = s["x"].cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
    settings = zip(*(s[name].cpu().numpy().astype(np.float64) for name in ("temperature", "top_k", "top_p", "min_p")))
    tokens, probs = [], []
    for row, (t, k, p, m) in enumerate(settings):
        if t <= 0:
            tokens.append(int(x[row].argmax()))
            probs.append(1.0)
            continue
        ranked = np.argsort(-x[row], kind="stable")
        if k > 0:
            ranked = ranked[:int(k)]
        w = np.exp((x[row][ranked] - x[row].max()) / t)
        if p < 1:
            w = w[:1 + int(np.searchsorted(np.cumsum(w), p * w.sum()))]
        w = w[w >= m] if m > 0 else w
        by_token = np.argsort(ranked[:len(w)])
        mine, w = ranked[:len(w)][by_token], w[by_token]
        upto = np.cumsum(w)
        i = min(int(np.searchsorted(upto, u[row] * upto[-1], side="right")), len(w) - 1)
        tokens.append(int(mine[i]))
        probs.append(w[i] / upto[-1])
    return {"token": torch.tensor(tokens, dtype=torch.int32), "prob": torch.tensor(probs, dtype=torch.float64)}


def _exact_rope(case, s):
    rot, half = case["rot"], case["rot"] // 2
    by, speeds = 1.0, []
    for i in range(half):
        speed = THETA ** (-2 * i / rot)
        if case["scaling"] == "linear":
            speed /= case["factor"]
        elif case["scaling"] == "ntk" and rot > 2:
            speed = (THETA * case["factor"] ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif case["scaling"] == "yarn":
            by = 1 + math.log(case["factor"]) / 10
            lo, hi = (rot / 2 * math.log(case["original"] / turns / math.tau, THETA) for turns in (32, 1))
            lo, hi = max(0, math.floor(lo)), min(rot - 1, math.ceil(hi))
            slow = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            speed *= slow / case["factor"] + 1 - slow
        speeds.append(speed)
    angle = s["pos"].double().unsqueeze(1) * torch.tensor(speeds, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, by), angle).unsqueeze(1)
    got = {}
    for name in "qk":
        x = s[name].double()
        pairs = x[..., :rot].unflatten(-1, (half, 2) if case["inter"] else (2, half))
        dim = -1 if case["inter"] else -2
        z = torch.complex(*pairs.unbind(dim)) * turn
        got[name] = torch.cat([torch.stack([z.real, z.imag], dim).flatten(-2), x[..., rot:]], -1)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "sample": _exact_sample, "rope": _exact_rope}[case["kind"]](case, s)
