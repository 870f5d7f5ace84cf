"""sum_out without a delta is x, to the bit: zeros of both signs, infinities,
the smallest and the largest numbers among them."""
import pytest
import torch

import relpos_mhsa as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [1, 5, 8, 100, 1023, 9001, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, -0.5, 0.0])
def test_a_copy_is_a_copy(d, dtype, scale):
    info = torch.finfo(dtype)
    values = torch.tensor([-0.0, 0.0, 1.5, -2.5, info.min, info.max, info.tiny, -info.tiny, float("inf"), float("-inf"), 1e-3], dtype=dtype)
    x = values[torch.arange(6 * d) % len(values)].view(6, d).cuda()
    got = M.add_norm(x, scale=scale, sum_out=torch.empty_like(x)).sum
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(got.view(bits), x.view(bits))
    zeros = torch.full((3, d), -0.0, dtype=dtype, device="cuda")  # with a delta: the sum of two negative zeros is one
    assert torch.equal(M.add_norm(zeros, zeros).sum.view(bits), zeros.view(bits))
