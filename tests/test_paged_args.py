"""The paged cache's operators refuse on the host what they cannot serve, before anything is launched: no GPU needed."""
from __future__ import annotations

import ctypes

import pytest

FAKE = 0x1000  # never dereferenced: every call here fails its checks, or has nothing to do


@pytest.fixture(scope="module")
def ops():
    from rpgbarenginecuda_amd import ops as o

    o.load_library()
    return o


def views(ops, kv_type=0, shape=(10, 8, 16, 128), table=(4, 5), **changes):
    kv = ops.GpuPagedKv(FAKE, FAKE, FAKE if kv_type else None, FAKE if kv_type else None, shape=shape, kv_type=kv_type)
    t = ops.GpuPageTable(FAKE, shape=table)
    for name, value in changes.items():
        setattr(kv.c if hasattr(kv.c, name) else t.c, name, value)
    return kv, t


BAD_CACHES = [
    (dict(type=2), "neither F16 nor Q8"), (dict(head_dim=96), "neither 64 nor 128"), (dict(head_dim=0), "neither 64"),
    (dict(n_kv_heads=0), "n_kv_heads 0"), (dict(page_size=8), "power of two"), (dict(page_size=48), "power of two"),
    (dict(page_size=512), "power of two"), (dict(page_size=-16), "power of two"), (dict(n_pages=0), "0 pages"),
    (dict(n_pages=1 << 31), "out of range"), (dict(n_seqs=0), "0 x 5"), (dict(max_pages=0), "4 x 0"),
    (dict(max_pages=-1), "out of range"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(pages=None), "null"),
    (dict(k=FAKE + 8), "16-byte aligned"), (dict(v=FAKE + 2), "16-byte aligned"), (dict(pages=FAKE + 2), "4-byte aligned"),
]


def calls(ops, kv, t, n=2):
    yield lambda: ops.GpuKvWritePaged(kv, t, FAKE, FAKE, FAKE, FAKE, n)
    yield lambda: ops.GpuQkNormRopeKvPaged(kv, t, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16, FAKE, 100, n, 1e-6, FAKE)
    yield lambda: ops.GpuKvReadPaged(kv, t, FAKE, FAKE, n, FAKE, FAKE, 1024, 128, out_f32=False)
    yield lambda: ops.GpuAttentionPaged(kv, t, FAKE, FAKE, 16, n, 1 << 40, 1 << 41, FAKE, workspace_bytes=1 << 30)


@pytest.mark.parametrize("changes,text", BAD_CACHES)
def test_caches_that_cannot_be_addressed_are_refused(ops, changes, text):
    kv, t = views(ops, **changes)
    for call in calls(ops, kv, t):
        with pytest.raises(ops.RpgError, match=text):
            call()


def test_8_bit_caches_need_their_scales(ops):
    for name in ("k_scale", "v_scale"):
        for value, text in ((None, "needs its scales"), (FAKE + 4, "16-byte aligned")):
            kv, t = views(ops, kv_type=1, **{name: value})
            for call in calls(ops, kv, t):
                with pytest.raises(ops.RpgError, match=text):
                    call()


def test_no_rows_is_no_work_and_fewer_are_refused(ops):
    kv, t = views(ops)
    for call in calls(ops, kv, t, n=0):
        call()
    for call in calls(ops, kv, t, n=-1):
        with pytest.raises(ops.RpgError, match="-1 (tokens|rows)"):
            call()


def test_more_rows_than_sequences_need_seq_ids(ops):
    kv, t = views(ops)  # 4 sequences
    for call in (lambda: ops.GpuKvWritePaged(kv, t, None, FAKE, FAKE, FAKE, 5),
                 lambda: ops.GpuQkNormRopeKvPaged(kv, t, None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16, FAKE, 100, 5, 1e-6,
                                                  FAKE),
                 lambda: ops.GpuKvReadPaged(kv, t, None, FAKE, 5, FAKE, FAKE, 1024, 128, out_f32=True),
                 lambda: ops.GpuAttentionPaged(kv, t, FAKE, FAKE, 16, 5, 1 << 40, 1 << 41, workspace_bytes=1 << 30)):
        with pytest.raises(ops.RpgError, match="5 (tokens|rows) without seq_ids, but 4 sequences"):
            call()


def test_write_refusals(ops):
    kv, t = views(ops)
    for args, text in (((FAKE, None, FAKE, FAKE), "null positions"), ((FAKE, FAKE, None, FAKE), "null pointer"),
                       ((FAKE, FAKE, FAKE, None), "null pointer"), ((FAKE, FAKE, FAKE + 4, FAKE), "aligned"),
                       ((FAKE, FAKE, FAKE, FAKE + 8), "aligned")):
        with pytest.raises(ops.RpgError, match=text):
            ops.GpuKvWritePaged(kv, t, *args, 2)


def test_fused_write_refusals(ops):
    kv, t = views(ops)
    far = 1 << 40
    good = dict(q=FAKE, k=FAKE, v=FAKE, qn=FAKE, kn=FAKE, heads=16, tab=FAKE, rows=100, n=2, out=far)
    for change, text in ((dict(heads=0), "n_heads 0"), (dict(rows=0), "RoPE table of 0"), (dict(q=None), "null"),
                         (dict(k=None), "null"), (dict(v=None), "null"), (dict(qn=None), "null"), (dict(kn=None), "null"),
                         (dict(tab=None), "null"), (dict(out=None), "null"), (dict(q=FAKE + 4), "aligned"),
                         (dict(tab=FAKE + 4), "aligned"), (dict(out=far + 4), "aligned"),
                         (dict(out=FAKE + 16), "q itself or apart"), (dict(out=FAKE + 2 * 16 * 512 - 16), "q itself or apart"),
                         (dict(out=FAKE - 16), "q itself or apart")):
        a = {**good, **change}
        with pytest.raises(ops.RpgError, match=text):
            ops.GpuQkNormRopeKvPaged(kv, t, FAKE, FAKE, a["q"], a["k"], a["v"], a["qn"], a["kn"], a["heads"], a["tab"],
                                     a["rows"], a["n"], 1e-6, a["out"])


@pytest.mark.parametrize("token,head,text", [
    (1024, 120, "at least head_dim"), (120, 1024, "at least head_dim"), (1028, 128, "multiples of 8"),
    (1024, 132, "multiples of 8"), (128, 128, "overlap"), (1016, 128, "overlap"), (128, 248, "overlap"),
    (-1024, 128, "at least head_dim"), (1 << 60, 128, "at least head_dim"), (128, 1 << 60, "at least head_dim"),
])
def test_read_refuses_strides_that_overlap(ops, token, head, text):
    kv, t = views(ops)
    with pytest.raises(ops.RpgError, match=text):
        ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 2, FAKE, FAKE, token, head, out_f32=False)


def test_read_refusals(ops):
    kv, t = views(ops)
    for k, v, text in ((None, FAKE, "null"), (FAKE, None, "null"), (FAKE + 8, FAKE, "aligned"), (FAKE, FAKE + 8, "aligned")):
        with pytest.raises(ops.RpgError, match=text):
            ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 2, k, v, 1024, 128, out_f32=False)
    with pytest.raises(ops.RpgError, match="out_f32"):
        ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 2, FAKE, FAKE, 1024, 128)


def test_read_refuses_other_types(ops):
    import torch

    kv, t = views(ops)
    for dtype, f32 in ((torch.int32, None), (torch.float64, None), (torch.bfloat16, False), (torch.float16, True),
                       (torch.float32, False)):
        out = torch.zeros(2, 8, 128, dtype=dtype)
        with pytest.raises(ops.RpgError, match="k_out is torch"):
            ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 2, out, out, 1024, 128, out_f32=f32)


def test_attention_refusals(ops):
    kv, t = views(ops)
    need = ops.GpuAttentionPagedWorkspace(16, 8, 128)
    far, work = 1 << 40, 1 << 41
    good = dict(lens=FAKE, q=FAKE, heads=16, n=2, out=far, work=work, bytes=need)
    for change, text in ((dict(heads=12), "12 query heads do not divide among 8"), (dict(heads=0), "do not divide"),
                         (dict(heads=-8), "do not divide"), (dict(lens=None), "null"), (dict(q=None), "null"),
                         (dict(out=None), "null"), (dict(work=None), "null"), (dict(q=FAKE + 4), "aligned"),
                         (dict(out=far + 8), "aligned"), (dict(out=FAKE), "overlap"), (dict(out=FAKE + 16), "overlap"),
                         (dict(bytes=need - 1), "workspace of"), (dict(work=work + 128), "workspace of"),
                         (dict(bytes=-1), "negative"), (dict(n=1 << 31), "rows")):
        a = {**good, **change}
        with pytest.raises(ops.RpgError, match=text):
            ops.GpuAttentionPaged(kv, t, a["lens"], a["q"], a["heads"], a["n"], a["out"], a["work"], seq_ids=FAKE,
                                  workspace_bytes=a["bytes"])


def test_calls_too_large_to_count(ops):
    """Head rows of a write or a read, and units of an attention call, are counted in 32 bits."""
    far = 1 << 62  # past whatever the counts below make of q
    kv, t = views(ops, n_seqs=1 << 30)
    for n in ((1 << 31) // 16, 1 << 40):
        with pytest.raises(ops.RpgError, match="too many for one call"):
            ops.GpuKvWritePaged(kv, t, FAKE, FAKE, FAKE, FAKE, n)
        with pytest.raises(ops.RpgError, match="too many for one call"):
            ops.GpuQkNormRopeKvPaged(kv, t, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 16, FAKE, 100, n, 1e-6, FAKE)
        with pytest.raises(ops.RpgError, match="too many for one call"):
            ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 2 * n, FAKE, far, 1024, 128, out_f32=False)
    need = ops.GpuAttentionPagedWorkspace(16, 8, 128)
    # 2^20 rows that may have 2^17 positions each: 2^12 units of 32 for 8 kv heads
    kv, t = views(ops, max_pages=1 << 13, n_seqs=1 << 20)
    with pytest.raises(ops.RpgError, match="too many for one call"):
        ops.GpuAttentionPaged(kv, t, FAKE, FAKE, 16, 1 << 20, far, 1 << 41, seq_ids=FAKE, workspace_bytes=need)


def test_buffers_that_overlap_or_lie_askew_are_refused(ops):
    kv, t = views(ops)
    far = 1 << 40
    for name in ("k", "v", "q_norm", "k_norm", "tab"):
        a = dict(q=far, k=1 << 41, v=1 << 42, q_norm=1 << 43, k_norm=1 << 44, tab=1 << 45, out=1 << 46)
        size = 2 * 16 * 128 * 4
        for out in (a[name], a[name] - size + 16):
            with pytest.raises(ops.RpgError, match="must not overlap k, v"):
                ops.GpuQkNormRopeKvPaged(kv, t, FAKE, FAKE, a["q"], a["k"], a["v"], a["q_norm"], a["k_norm"], 16, a["tab"],
                                         100, 2, 1e-6, out)
    with pytest.raises(ops.RpgError, match="k_out and v_out are the same"):
        ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 2, far, far, 1024, 128, out_f32=False)
    for seq, pos in ((FAKE + 2, FAKE), (FAKE, FAKE + 1), (None, FAKE + 3)):
        with pytest.raises(ops.RpgError, match="4-byte aligned"):
            ops.GpuKvWritePaged(kv, t, seq, pos, FAKE, FAKE, 2)
        with pytest.raises(ops.RpgError, match="4-byte aligned"):
            ops.GpuKvReadPaged(kv, t, seq, pos, 2, far, 1 << 41, 1024, 128, out_f32=False)
        with pytest.raises(ops.RpgError, match="4-byte aligned"):
            ops.GpuAttentionPaged(kv, t, pos, FAKE, 16, 2, far, 1 << 41, seq_ids=seq, workspace_bytes=1 << 30)
    need = ops.GpuAttentionPagedWorkspace(16, 8, 128)
    for q, out in ((far, (1 << 41) + need - 16 & ~15), (far, (1 << 41) - 16), ((1 << 41) + 256, far)):
        with pytest.raises(ops.RpgError, match="workspace must not overlap"):
            ops.GpuAttentionPaged(kv, t, FAKE, q, 16, 2, out, 1 << 41, seq_ids=FAKE, workspace_bytes=need)


def shifted_reads(d=64, n=3, n_kv=2):
    """(bytes from k_out to v_out, token and head stride in elements, fp32, whether two of their rows share an element) of
    outputs that lie in one another."""
    for ts, hs in ((n_kv * d, d), (2 * n_kv * d, d), (2 * n_kv * d, 2 * d), (d, 4 * d), (2 * d, 16 * d), (n_kv * d + 8, d)):
        rows = [t * ts + h * hs for t in range(n) for h in range(n_kv)]
        for f32 in (False, True):
            size = 4 if f32 else 2
            for apart in range(-(rows[-1] + 2 * d) * size, (rows[-1] + 2 * d) * size, 16):
                shift = apart // size
                if apart:
                    yield apart, ts, hs, f32, any(abs(a + shift - b) < d for a in rows for b in rows)


def test_read_refuses_outputs_whose_rows_overlap(ops):
    kv, t = views(ops, shape=(10, 2, 16, 64))
    far, seen = 1 << 40, 0
    for apart, ts, hs, f32, meet in shifted_reads():
        if meet:
            seen += 1
            with pytest.raises(ops.RpgError, match="rows of k_out and v_out overlap"):
                ops.GpuKvReadPaged(kv, t, FAKE, FAKE, 3, far, far + apart, ts, hs, out_f32=f32)
    assert seen > 500


def test_other_devices_are_refused(ops):
    import torch

    kv, t = views(ops)
    kv.device, kv.device_index, t.device_index = torch.device("cuda", 1), 1, 0
    for call in calls(ops, kv, t):
        with pytest.raises(ops.RpgError, match="page table on device 0"):
            call()
    t.device_index, kv.current_device = 1, lambda: 0
    for call in calls(ops, kv, t):
        with pytest.raises(ops.RpgError, match="not the current device"):
            call()


def test_workspace_sizes(ops):
    for heads, kv, d in ((1, 1, 64), (16, 8, 128), (64, 1, 128)):
        assert ops.GpuAttentionPagedWorkspace(heads, kv, d) > 0
    for heads, kv, d in ((16, 8, 96), (16, 0, 128), (15, 8, 128), (0, 8, 128)):
        with pytest.raises(ops.RpgError):
            ops.GpuAttentionPagedWorkspace(heads, kv, d)
    for ptr, n in ((None, 256), (FAKE + 16, 256), (FAKE, 0), (FAKE, 24), (FAKE, -16)):
        with pytest.raises(ops.RpgError):
            ops.GpuAttentionPagedWorkspaceInit(ptr, n)


def test_null_structs_are_refused(ops):
    f = ops.paged_ops()
    kv, t = views(ops)
    assert f.kv_write(None, t.ref, FAKE, FAKE, FAKE, FAKE, 1) < 0
    assert b"null paged cache" in ops.load_library().rpg_ops_last_error()
    assert f.kv_write(kv.ref, None, FAKE, FAKE, FAKE, FAKE, 1) < 0
    assert b"null page table" in ops.load_library().rpg_ops_last_error()


def test_python_views_check_their_tensors(ops):
    import torch

    k = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    for args, text in (((k, k[:3]), "alike"), ((k, k.to(torch.int16)), "alike"), ((k[0], k[0]), "alike"),
                       ((k.float(), k.float()), "16-bit or int8"), ((k.to(torch.int8), k.to(torch.int8)), "need k_scale"),
                       ((k, k, torch.zeros(4, 2, 16), None), "no scales"),
                       ((k.to(torch.int8), k.to(torch.int8), torch.zeros(4, 2), torch.zeros(4, 2, 16)), "k_scale"),
                       ((k, k), "not on the GPU")):
        with pytest.raises(ops.RpgError, match=text):
            ops.GpuPagedKv(*args)
    with pytest.raises(ops.RpgError, match="n_seqs, max_pages"):
        ops.GpuPageTable(torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ops.RpgError, match="not on the GPU"):
        ops.GpuPageTable(torch.zeros(4, 2, dtype=torch.int32))


def test_pages_are_all_tensors_or_all_raw_addresses(ops):
    import torch

    k = torch.zeros(4, 2, 16, 64, dtype=torch.int8)
    s = torch.zeros(4, 2, 16)
    for args in ((k, k, FAKE, FAKE), (k, k, s, FAKE), (k, FAKE, s, s), (FAKE, k, FAKE, FAKE), (FAKE, FAKE, s, s),
                 (FAKE, FAKE, FAKE, s), (k, None, s, s), (None, None)):
        for given in ({}, dict(shape=(4, 2, 16, 64), kv_type=ops.KV_Q8)):
            with pytest.raises(ops.RpgError, match="all tensors or all raw addresses"):
                ops.GpuPagedKv(*args, **given)


def test_pages_go_with_their_view(ops):
    """Nothing that a view holds holds the view: the pages' memory is free when it goes, without a collection."""
    import gc
    import weakref

    gc.disable()
    try:
        kv, t = views(ops)
        for call in calls(ops, kv, t, n=0):
            call()
        gone = [weakref.ref(kv), weakref.ref(t)]
        del kv, t, call
        assert [r() for r in gone] == [None, None]
    finally:
        gc.enable()


def test_table_of_functions_matches_its_header(ops):
    """The struct in include/rpg_paged.h and its Python mirror have the same entries, in order."""
    import os
    import re

    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "rpg_paged.h")).read()
    body = re.sub(r"/\*.*?\*/", "", text[text.index("int64_t size;"):text.index("} rpg_paged_ops_t;")], flags=re.S)
    assert re.findall(r"\(\*(\w+)\)\(", body) == [n for n, _ in ops.PagedOpsC._fields_[1:]]
    for (name, kind), args in zip(ops.PagedOpsC._fields_[1:], re.findall(r"\(\*\w+\)\(([^)]*)\)", body)):
        want = [ctypes.c_void_p if "*" in a else {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64,
                                                   "float": ctypes.c_float}[a.split()[0]] for a in args.split(",")]
        assert list(kind._argtypes_) == want, name
    assert ops.paged_ops().size == ctypes.sizeof(ops.PagedOpsC)
