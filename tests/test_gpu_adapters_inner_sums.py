"""The adapters' inner sums t = s A x behind a bfloat16 result, seen through a
projection of zeros: y = B t.

Tolerances. y is rounded once, by 2^-8 of itself. t enters as two bf16 numbers:
its first 8 bits, whose remainder is under 2^-7 of it, and that remainder
rounded, by 2^-8 of itself, so 2^-15 of sum |b| |t|. The products are exact, the
sums f32: K + rank + 64 steps of 2^-24 of the magnitudes that pass through both.
"""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M
import rows_oracle as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def made(rng, k, n, ranks, gain=1.0):
    layer, adapters = M.Fp8Linear(k, n), M.LowRankAdapters(k, n, len(ranks), max(ranks))
    layer.load_codes(np.zeros((n, k), np.uint8), np.full((-(-n // 128), -(-k // 128)), 127, np.uint8), None)
    parts = []
    for i, r in enumerate(ranks):
        a = torch.from_numpy(gain * rng.standard_normal((r, k)) / np.sqrt(k)).bfloat16()
        b = torch.from_numpy(rng.standard_normal((n, r)) / np.sqrt(r)).bfloat16()
        s = float(np.float32(rng.uniform(0.5, 2)))
        adapters.load(i, a, b, s)
        parts.append((a.double().numpy(), b.double().numpy(), s))
    return layer, adapters, parts


def check(got, x, which, parts):
    want, through, inner = R.adapted(x, which, parts)
    steps = x.shape[1] + max(p[0].shape[0] for p in parts) + 64
    tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -15 * inner + steps * 2.0 ** -24 * through
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol + 1e-37)
    assert not bad.any(), (int(bad.sum()), got.size, np.argwhere(bad)[:4].tolist(), (np.abs(got - want) / (tol + 1e-37)).max())


@pytest.mark.parametrize("rows,k,n,ranks", [(1, 1024, 512, [16]), (4, 300, 200, [7, 128]), (3, 4096, 96, [16, 9]), (40, 640, 300, [16, 3]),
                                            (200, 512, 256, [64, 20, 33]), (900, 384, 640, [24, 16]), (3000, 512, 1100, [128, 5])])
@pytest.mark.parametrize("xd", ["f32", "bf16", "codes"])
def test_inner_sums_are_not_rounded_to_the_results_type(rows, k, n, ranks, xd):
    rng = np.random.default_rng(rows + k)
    layer, adapters, parts = made(rng, k, n, ranks)
    x = torch.from_numpy(rng.standard_normal((rows, k))).float().cuda()
    which = np.sort(rng.integers(-1, len(ranks), rows)).astype(np.int32)
    which[0] = 0
    ids = torch.from_numpy(which).cuda()
    if xd == "codes":
        r = M.add_norm(x, want="both")
        values, x = F.round_rows(r.out.double().cpu().numpy()), r.codes
    else:
        x = x.to(DTYPES[xd])
        values = x.double().cpu().numpy()
    got = layer.forward(x, out_dtype=torch.bfloat16, adapters=adapters, which=ids)
    assert got.dtype == torch.bfloat16
    check(got, values, which, parts)


@pytest.mark.parametrize("rows", [2, 30, 2000])
def test_inner_sums_that_cancel(rows):
    """y = t_1 - t_2 of two ranks whose sums share their first 8 bits."""
    k, n = 128, 64
    layer, adapters = M.Fp8Linear(k, n), M.LowRankAdapters(k, n, 1, 2)
    layer.load_codes(np.zeros((n, k), np.uint8), np.full((1, 1), 127, np.uint8), None)
    a = np.zeros((2, k), np.float32)
    a[0, 0] = a[1, 1] = 1.0
    adapters.load(0, a, np.tile([1.0, -1.0], (n, 1)).astype(np.float32), 1.0)
    x = np.zeros((rows, k), np.float32)
    x[:, 1] = 1.0
    x[:, 0] = 1.0 + 2.0 ** -10  # rounds to 1 in bf16, and is 8 + 8 bits exactly
    which = torch.zeros(rows, dtype=torch.int32, device="cuda")
    got = layer.forward(torch.from_numpy(x).cuda(), out_dtype=torch.bfloat16, adapters=adapters, which=which)
    assert torch.equal(got, torch.full((rows, n), 2.0 ** -10, dtype=torch.bfloat16, device="cuda"))
