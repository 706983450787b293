"""Paged attention and eviction where numbers get large, small or strange: positions past 2^24, prefixes past 2^31,
budgets without a limit, scales of zero and below, capped scores over their whole range, sums that are not finite.

Bars as in test_gpu_paged.py unless a test derives its own."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from test_gpu_paged import ATTN_BAR, Cache, attend, check_prompt, evict_ref, i32, rel

pytestmark = pytest.mark.gpu


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda()


# ── positions ────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("new", [[4, 3], [60, 40]])
@pytest.mark.parametrize("window", [0, 30])
def test_prefix_past_31_bits(pkg, ctx, f16, new, window):
    """A prefix longer than any sequence: everything cached is seen in both directions."""
    for prefix in ([0xFFFFFFFF, 1 << 31], [(1 << 31) - 1, (1 << 31) + 50]):
        check_prompt(pkg, ctx, 8, 2, 64, f16, 16, new, [100, 90], prefix=prefix, window=window, seed=1)
