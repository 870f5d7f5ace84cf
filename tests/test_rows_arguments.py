"""Rows' shapes and adapters' numbers that are refused in Python, without a GPU."""
import numpy as np
import pytest
import torch

import relpos_mhsa as M


@pytest.mark.parametrize("shape", [(), (4,), (4.0, 64), ("a", 64), (-2, -2, 64), (4, -64), (4, 0), (None, 64)])
def test_shapes_of_rounded_rows(shape):
    codes, scales = torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8)
    with pytest.raises(M.MhsaError):
        M.Fp8Linear(64, 48).forward(M.Fp8Rows(codes, scales, shape))


def test_a_shape_that_is_none_is_named():
    codes, scales = torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8)
    for shape in ((), (4.0, 64), (-2, -2, 64)):
        with pytest.raises(M.MhsaError, match="shape"):
            M.Fp8Rows(codes, scales, shape).check()


def test_numbers_past_an_int32():
    a, b = np.zeros((4, 64), np.float32), np.zeros((48, 4), np.float32)
    adapters = M.LowRankAdapters(64, 48, 2, 8)
    for slot in (-1, 2, 1 << 32, (1 << 32) + 1, None, "0", 0.5):
        with pytest.raises(M.MhsaError, match="slot"):
            adapters.load(slot, a, b)
        with pytest.raises(M.MhsaError, match="slot"):
            adapters.clear(slot)
    for sizes in (((1 << 32) + 64, 48, 2, 8), (64, (1 << 32) + 48, 2, 8), (64, 48, (1 << 32) + 2, 8), (64, 48, 2, (1 << 32) + 8)):
        with pytest.raises(M.MhsaError):
            M.LowRankAdapters(*sizes)
