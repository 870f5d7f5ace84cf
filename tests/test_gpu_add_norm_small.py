"""A residual's addition with its norm of rows whose squares leave f32's range
below, with an eps as small or of 0, against the float64 oracle.

Tolerances as in test_gpu_add_norm: 96 steps of 2^-24 of what enters y (a power
of two that rows are multiplied by adds none). The layer norm's mean is an f32,
off by 2^-150 where it is below f32's smallest normal number, 2^-126.
"""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M
import rows_oracle as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = 2.0 ** -24
SIZES = [1e-8, 1e-15, 3e-16, 1e-17, 1e-19, 1e-20, 1e-22, 1e-25, 1e-30, 1e-37, 1e-40, 1e-43]


@pytest.mark.parametrize("d", [8, 100, 600, 2500, 9000, 20001])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("eps", [0.0, 1e-42, 1e-36, 1e-31, 1e-29])
def test_small_rows(d, kind, eps):
    rng = np.random.default_rng(d)
    w, b = np.exp(0.3 * rng.standard_normal(d)), 0.2 * rng.standard_normal(d)
    tw, tb = (torch.from_numpy(v).float().cuda() for v in (w, b))
    for dtype in ("f32", "bf16"):
        sizes = np.array(SIZES if dtype == "f32" else SIZES[:10])  # (bf16's smallest number is 2^-133)
        x = rng.standard_normal((len(sizes), d)) * sizes[:, None]
        t = torch.from_numpy(x).float().to(DTYPES[dtype]).cuda()
        got = M.add_norm(t, weight=tw, bias=tb, kind=kind, eps=eps, want="both", out_dtype=torch.float32)
        v = t.double().cpu().numpy()
        y, _, size = R.norm(v, None, 1.0, tw.double().cpu().numpy(), tb.double().cpu().numpy(), kind, eps)
        tol = 96 * STEP * size
        if kind == "layer":
            u = v - v.mean(-1, keepdims=True)
            r = 1.0 / np.sqrt((u * u).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
            tol = tol + 2 * 2.0 ** -150 * r * (np.abs(tw.double().cpu().numpy()) + np.abs(u) * r)
        out = got.out.double().cpu().numpy()
        assert np.isfinite(y).all()
        bad = ~(np.abs(out - y) <= tol)
        assert not bad.any(), (dtype, sorted({int(i) for i in np.argwhere(bad)[:, 0]}), out[bad][:4], y[bad][:4])
        assert not (F.VALUES[got.codes.codes.cpu().numpy()] != F.VALUES[got.codes.codes.cpu().numpy()]).any()  # no NaN


@pytest.mark.parametrize("d", [64, 700, 5000])
def test_one_small_value_in_a_row_and_rows_of_zeros(d):
    """One value of a row of zeros, at both ends of the row and of f32; y is the
    root of the row's length there, and 0 over 0 in a row of zeros."""
    values = [1.0, 2.0 ** -50, 2.0 ** -64, 2.0 ** -100, 2.0 ** -126, 2.0 ** -149]
    x = torch.zeros(2 * len(values) + 1, d)
    for i, v in enumerate(values):
        x[2 * i, 0], x[2 * i + 1, d - 1] = v, -v
    got = M.add_norm(x.cuda(), eps=0.0).out.double().cpu()
    for i in range(len(values)):
        for row, at, sign in ((2 * i, 0, 1.0), (2 * i + 1, d - 1, -1.0)):
            assert abs(float(got[row, at]) - sign * d ** 0.5) <= 96 * STEP * d ** 0.5
            got[row, at] = 0.0
            assert (got[row] == 0).all()
    assert torch.isnan(got[-1]).all()
    assert (M.add_norm(x[-1:].cuda(), eps=1e-45).out == 0).all()


def test_small_and_ordinary_rows_side_by_side():
    """Four rows share a workgroup: a small one leaves its neighbours' bits alone."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(64, 512, generator=g)
    want = M.add_norm(x.cuda(), eps=0.0).out
    x[::3] *= 1e-25
    got = M.add_norm(x.cuda(), eps=0.0).out
    keep = torch.arange(64) % 3 != 0
    assert torch.equal(got[keep.cuda()], want[keep.cuda()])
    assert torch.allclose(got, want, rtol=200 * STEP, atol=0)
