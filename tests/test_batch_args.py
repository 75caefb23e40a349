"""The operators of a step of many conversations refuse on the host what they cannot serve, before anything is launched,
and their rotation tables hold what the formulas say: no GPU needed."""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np
import pytest

from batch_ref import frequencies

FAKE = 0x1000  # never dereferenced: every call here fails its checks, or has nothing to do
FAR = [(i + 1) << 40 for i in range(12)]


@pytest.fixture(scope="module")
def ops():
    from rpgbarenginecuda_amd import ops as o

    o.load_library()
    return o


def test_table_of_functions_matches_its_header(ops):
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "rpg_batch.h")).read()
    body = re.sub(r"/\*.*?\*/", "", text[text.index("int64_t size;"):text.index("} rpg_batch_ops_t;")], flags=re.S)
    assert re.findall(r"\(\*(\w+)\)\(", body) == [n for n, _ in ops.BatchOpsC._fields_[1:]]
    kinds = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float, "double": ctypes.c_double}
    for (name, kind), args in zip(ops.BatchOpsC._fields_[1:], re.findall(r"\(\*\w+\)\(([^)]*)\)", body)):
        assert list(kind._argtypes_) == [ctypes.c_void_p if "*" in a else kinds[a.split()[0]] for a in args.split(",")], name
    assert ops.batch_ops().size == ctypes.sizeof(ops.BatchOpsC)


# ---------------------------------------------------------------- rotation tables


@pytest.mark.parametrize("rot", [2, 6, 64, 128])
@pytest.mark.parametrize("kind,factor,original", [("none", 1.0, 0), ("linear", 4.0, 0), ("ntk", 8.0, 0), ("yarn", 4.0, 16384),
                                                  ("yarn", 1.0, 4096), ("yarn", 3.5, 7)])
def test_scaled_tables(ops, rot, kind, factor, original):
    """Entries of magnitude up to `by` are rounded once, half a step; angles are products of 64 bits, whose last bits count
    by their size: 2^-52 times the angle, a few roundings of which are in the frequency (8 units)."""
    n = 5000
    got = ops.build_rope_table_scaled(rot, 1e6, n, kind, factor, original)
    f, by = frequencies(rot, 1e6, kind, factor, original)
    angle = np.arange(n)[:, None] * f
    for mine, want in ((got[:, :rot // 2], by * np.cos(angle)), (got[:, rot // 2:], by * np.sin(angle))):
        assert np.all(np.abs(mine - want) <= 2.0 ** -24 * np.abs(want) + by * 8 * 2.0 ** -52 * (1 + angle))


def test_plain_table_has_the_other_tables_bits(ops):
    assert np.array_equal(ops.build_rope_table_scaled(128, 1e6, 9000), ops.build_rope_table(128, 1e6, 9000))


def test_yarn_between_its_ends(ops):
    """Pairs that turn often keep their frequency, slow ones have it divided: read off position 1 of the table."""
    tab = ops.build_rope_table_scaled(128, 1e6, 2, "yarn", 4.0, 32768, attention=1.0)
    f, _ = frequencies(128, 1e6, "none")
    angle = np.arctan2(tab[1, 64:].astype(np.float64), tab[1, :64])
    assert np.allclose(angle[:20], f[:20], rtol=1e-6) and np.allclose(angle[-20:], f[-20:] / 4, rtol=1e-6)
    assert np.all((angle <= f * (1 + 1e-6)) & (angle >= f / 4 * (1 - 1e-6)))


@pytest.mark.parametrize("change,text", [
    (dict(rot_dim=7), "even head size"), (dict(theta=0.0), "theta must be positive"), (dict(theta=float("nan")), "positive"),
    (dict(factor=0.5), "factor 0.5"), (dict(factor=float("nan")), "factor"), (dict(factor=float("inf")), "factor"),
    (dict(scaling="other"), "none of"), (dict(n_pos=0), "0 positions"), (dict(rot_dim=0), "positions of 0"),
    (dict(original_positions=0), "original number"), (dict(beta_slow=0.0), "beta_slow"), (dict(beta_fast=0.5), "beta_slow"),
    (dict(theta=1.0), "theta above 1"), (dict(attention=-1.0), "attention factor"),
    (dict(attention=float("nan")), "attention factor"),
])
def test_table_refusals(ops, change, text):
    a = {**dict(rot_dim=128, theta=1e6, n_pos=10, scaling="yarn", factor=4.0, original_positions=4096), **change}
    with pytest.raises(ops.RpgError, match=text):
        ops.build_rope_table_scaled(**a)


def test_table_refusals_of_the_c_entry(ops):
    f = ops.batch_ops()
    out = np.zeros((4, 8), np.float32)
    assert f.rope_table(8, 1e6, 4, None, out.ctypes.data) == 0 and np.all(out[:, 0] != 0)
    assert f.rope_table(8, 1e6, 4, None, None) < 0
    assert f.rope_table(8, 1e6, 0, None, out.ctypes.data) < 0
    assert f.rope_table(8, 1e6, 1 << 60, None, out.ctypes.data) < 0
    how = ops.RopeScalingC(4, 2.0, 0, 32.0, 1.0, 0.0)
    assert f.rope_table(8, 1e6, 4, ctypes.byref(how), out.ctypes.data) < 0
    assert b"none of plain" in ops.load_library().rpg_ops_last_error()


# ---------------------------------------------------------------- rotation


def rope_call(ops, **change):
    a = {**dict(q=FAR[0], k=FAR[1], heads=4, kv=2, d=64, rot=64, inter=False, tab=FAR[2], tab_rows=10, pos=FAR[3], n=3,
                q_out=FAR[4], k_out=FAR[5]), **change}
    ops.GpuRopeRows(a["q"], a["k"], a["heads"], a["kv"], a["d"], a["rot"], a["inter"], a["tab"], a["tab_rows"], a["pos"],
                    a["n"], a["q_out"], a["k_out"])


@pytest.mark.parametrize("change,text", [
    (dict(heads=0), "0 query heads"), (dict(kv=-1), "-1 kv heads"), (dict(heads=1 << 21), "query heads"),
    (dict(d=0), "head_dim 0"), (dict(d=1025), "head_dim 1025"), (dict(rot=0), "rot_dim 0"), (dict(rot=63), "rot_dim 63"),
    (dict(rot=66), "rot_dim 66"), (dict(tab_rows=0), "table of 0"), (dict(tab_rows=1 << 41), "RoPE table"),
    (dict(n=-1), "-1 rows"), (dict(n=1 << 30), "out of range"), (dict(q=None), "null"), (dict(k=None), "null"),
    (dict(q_out=None), "null"), (dict(k_out=None), "null"), (dict(tab=None), "null"), (dict(pos=None), "null"),
    (dict(q=FAR[0] + 2), "4-byte"), (dict(pos=FAR[3] + 1), "4-byte"), (dict(q_out=FAR[0] + 4), "q itself"),
    (dict(q_out=FAR[0] + 3 * 4 * 64 * 4 - 4), "q itself"), (dict(k_out=FAR[1] - 4), "k itself"),
    (dict(q_out=FAR[1]), "must not overlap"), (dict(k_out=FAR[0]), "must not overlap"),
    (dict(k_out=FAR[4] + 4), "must not overlap"), (dict(q_out=FAR[2]), "table or the positions"),
    (dict(k_out=FAR[3]), "table or the positions"),
])
def test_rope_refusals(ops, change, text):
    with pytest.raises(ops.RpgError, match=text):
        rope_call(ops, **change)


def test_rope_of_no_rows(ops):
    rope_call(ops, n=0)
    rope_call(ops, n=0, kv=0, k=None, k_out=None)


# ---------------------------------------------------------------- sampling


def sample_call(ops, **change):
    a = {**dict(x=FAR[0], rows=3, n=100, u=FAR[1], out=FAR[2], work=FAR[3], t=FAR[4], k=FAR[5], p=FAR[6], m=FAR[7],
                probs=FAR[8], stride=None, nbytes=1 << 30), **change}
    ops.GpuSampleBatch(a["x"], a["rows"], a["n"], a["u"], a["out"], a["work"], a["t"], a["k"], a["p"], a["m"], a["probs"],
                       a["stride"], a["nbytes"])


@pytest.mark.parametrize("change,text", [
    (dict(n=0), "0 logits"), (dict(n=(1 << 22) + 1), "limit"), (dict(rows=-1), "-1 rows"), (dict(rows=(1 << 20) + 1), "rows"),
    (dict(stride=99), "99 apart"), (dict(stride=-5), "apart"), (dict(stride=1 << 50), "apart"), (dict(x=None), "null"),
    (dict(u=None), "null"), (dict(out=None), "null"), (dict(work=None), "null"), (dict(x=FAR[0] + 2), "4-byte"),
    (dict(u=FAR[1] + 1), "4-byte"), (dict(probs=FAR[8] + 2), "4-byte"), (dict(t=FAR[4] + 1), "4-byte"),
    (dict(work=FAR[3] + 16), "256-byte"), (dict(nbytes=16), "workspace of"), (dict(nbytes=-1), "negative size"),
    (dict(out=FAR[1]), "settings or u"), (dict(probs=FAR[6]), "settings or u"), (dict(work=FAR[7]), "settings or u"),
    (dict(out=FAR[0] + 1196), "must not overlap"), (dict(probs=FAR[2] + 8), "must not overlap"),
    (dict(work=FAR[0]), "must not overlap"), (dict(out=FAR[3]), "must not overlap"),
])
def test_sample_refusals(ops, change, text):
    with pytest.raises(ops.RpgError, match=text):
        sample_call(ops, **change)


def test_sample_of_no_rows(ops):
    sample_call(ops, rows=0)
    with pytest.raises(ops.RpgError, match="needs workspace_bytes"):
        sample_call(ops, nbytes=None)


def test_sample_workspaces(ops):
    sizes = [ops.GpuSampleBatchWorkspace(r, n) for r, n in ((0, 1), (1, 1), (1, 151936), (128, 151936), (3, 1 << 22))]
    assert all(s > 0 and s % 16 == 0 for s in sizes) and sizes[2] <= sizes[3]
    for r, n in ((-1, 5), (1, 0), (1, (1 << 22) + 1), ((1 << 20) + 1, 5)):
        with pytest.raises(ops.RpgError):
            ops.GpuSampleBatchWorkspace(r, n)


def test_tensors_are_checked(ops):
    import torch

    x = torch.zeros(3, 100)
    with pytest.raises(ops.RpgError, match="not on the GPU"):
        sample_call(ops, x=x)
    with pytest.raises(ops.RpgError, match="not on the GPU"):
        rope_call(ops, q=x)
