"""Sizes that pass every limit of their own and that a launch has no room for are refused with the arguments, before anything
is launched: no GPU needed."""
from __future__ import annotations

import pytest

FAR = [(i + 1) << 44 for i in range(10)]


@pytest.fixture(scope="module")
def ops():
    from rpgbarenginecuda_amd import ops as o

    o.load_library()
    return o


@pytest.mark.parametrize("n,heads,kv,d,rot", [(1 << 28, 1, 0, 2, 2), (1 << 25, 6, 2, 4, 4), ((1 << 28) - 3, 1, 0, 20, 10),
                                              (1 << 26, 1, 0, 1024, 1024)])
def test_rotation(ops, n, heads, kv, d, rot):
    with pytest.raises(ops.RpgError, match="too many for one call"):
        ops.GpuRopeRows(FAR[0], FAR[1], heads, kv, d, rot, False, FAR[2], 10, FAR[3], n, FAR[0], FAR[1])


@pytest.mark.parametrize("n,heads,d", [(1 << 24, 16, 64), (1 << 24, 8, 128), ((1 << 27) - 1, 1, 128)])
def test_shared_attention(ops, n, heads, d):
    kv = ops.GpuPagedKv(FAR[0], FAR[1], shape=(10, 1, 16, d), kv_type=0)
    table = ops.GpuPageTable(FAR[2], shape=(n, 4))
    with pytest.raises(ops.RpgError, match="too many for one call"):
        ops.GpuAttentionPagedShared(kv, table, FAR[3], FAR[4], FAR[5], FAR[6], heads, n, FAR[7], FAR[8],
                                    workspace_bytes=1 << 40, n_groups=1, least_saving=0)


def test_sampling(ops):
    with pytest.raises(ops.RpgError, match="too many for one call"):
        ops.GpuSampleBatch(FAR[0], 1 << 20, 70_000, FAR[2], FAR[3], FAR[4], workspace_bytes=1 << 43)
