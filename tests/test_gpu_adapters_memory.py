"""Adapters that no GPU has the memory for: the load is refused, and nothing of
it is left for the calls behind it."""
import numpy as np
import pytest
import torch

import relpos_mhsa as M

pytestmark = pytest.mark.gpu


def test_a_load_without_memory_fails_alone():
    """4096 adapters of 128 x 2^21 bf16 would take 2 TiB."""
    n = 1 << 21
    x = torch.ones(3, 64, device="cuda")
    adapters = M.LowRankAdapters(64, n, 4096, 128)
    a, b = np.ones((1, 64), np.float32), np.ones((n, 1), np.float32)
    for _ in range(2):
        with pytest.raises(M.MhsaError):
            adapters.load(0, a, b)
        assert torch.isfinite(M.add_norm(x).out).all()
        with pytest.raises(M.MhsaError):
            adapters.load(0, a, b)
        assert float((x + 1).sum()) == 2 * 3 * 64
