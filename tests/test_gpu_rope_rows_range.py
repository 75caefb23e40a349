"""Rotation of as many heads as a launch of single elements has room for."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_the_most_heads_of_single_elements(gpu):
    """2^28 - 4 heads of 2, in place: the last ones and some between are rotated, each product rounded by itself."""
    import torch

    n = (1 << 28) - 4
    table = gpu.build_rope_table_scaled(2, 1e4, 1000)
    q = torch.ones(n, 1, 2, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda").remainder_(1000).int()
    gpu.GpuRopeRows(q, None, 1, 0, 2, 2, False, torch.from_numpy(table).cuda(), 1000, pos, n, q, None)
    look = [0, 1, 999, n // 2, n // 2 + 1, n - 1000, n - 2, n - 1]
    got = q[torch.tensor(look, device="cuda"), 0].cpu().numpy()
    co, si = table[np.array(look) % 1000].T
    assert np.array_equal(got, np.stack([co - si, co + si], -1))
    assert bool((q[:, 0, 0] != 1).logical_or_(pos == 0).all())
