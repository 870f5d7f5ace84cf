"""Adapters whose first load was refused on one GPU, loaded on another."""
import numpy as np
import pytest
import torch

import relpos_mhsa as M

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")]


def test_a_refused_load_binds_to_no_gpu():
    a, b = np.eye(4, 64, dtype=np.float32), np.eye(48, 4, dtype=np.float32)
    adapters = M.LowRankAdapters(64, 48, 1, 8)
    with torch.cuda.device(0), pytest.raises(M.MhsaError):
        adapters.load(0, np.full_like(a, np.inf), b)
    with torch.cuda.device(1):
        adapters.load(0, a, b)
        layer = M.Fp8Linear(64, 48)
        layer.load(np.zeros((48, 64), np.float32))
        x = torch.arange(64.0, device="cuda:1").expand(3, 64).contiguous()
        y = layer.forward(x, adapters=adapters, which=torch.zeros(3, dtype=torch.int32, device="cuda:1"))
        assert torch.equal(y[:, :4], x[:, :4]) and (y[:, 4:] == 0).all()
    with torch.cuda.device(0), pytest.raises(M.MhsaError):
        adapters.load(0, a, b)
