"""Arguments that are not tensors, and numbers of choices that no row has, are
refused as any other wrong argument."""
import numpy as np
import pytest
import torch

import relpos_mhsa as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [[0.0] * 8, np.zeros(8, np.float32), 1.0])
def test_route_bias(bad):
    with pytest.raises(M.MhsaError):
        M.route(torch.zeros(3, 8, device="cuda"), 2, bias=bad)


@pytest.mark.parametrize("top_k", [-1, 0, 9, 1 << 31, 1 << 40])
def test_route_choices(top_k):
    """Refused before memory is taken for the results."""
    with pytest.raises(M.MhsaError):
        M.route(torch.zeros(30000, 8, device="cuda"), top_k)


@pytest.mark.parametrize("bad", [None, 3, [[0], [1]], np.zeros((2, 1), np.int32)])
def test_experts_arguments(bad):
    layer = M.ExpertFeedForward(2, 64, 64)
    layer.load(torch.zeros(2, 64, 64), torch.zeros(2, 64, 64))
    x = torch.zeros(2, 64, device="cuda")
    idx, w = torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.ones(2, 1, device="cuda")
    assert torch.equal(layer.forward(x, idx, w), x)
    for args in ((bad, idx, w), (x, bad, w), (x, idx, bad)):
        with pytest.raises(M.MhsaError):
            layer.forward(*args)
    if bad is not None:
        for kw in ({"residual": bad}, {"out": bad}):
            with pytest.raises(M.MhsaError):
                layer.forward(x, idx, w, **kw)


@pytest.mark.parametrize("bad", [None, 3, [[0.0] * 64], np.zeros((1, 64), np.float32)])
def test_linear_arguments(bad):
    layer = M.Fp8Linear(64, 64)
    layer.load(torch.zeros(64, 64))
    with pytest.raises(M.MhsaError):
        layer.forward(bad)
    if bad is not None:
        with pytest.raises(M.MhsaError):
            layer.forward(torch.zeros(1, 64, device="cuda"), out=bad)
