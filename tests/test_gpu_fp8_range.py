"""The 8-bit block-scaled projection at the ends of its powers of two: scale
bytes that no weight of the usual size has, beside activations that bring the
results back into f32's range. The bounds are those of ordinary values: f32 sums
are off by at most K + 64 steps of 2^-24 of their terms' magnitudes, the fp8
matrix unit's by 7 * 2^-13 more, and a bf16 store by 2^-8 of the value."""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# one launch; tiles of 64, of 128, of 256 and of 192 rows
SIZES = [(5, 520, 300), (300, 200, 330), (1500, 520, 1500), (16300, 264, 2040), (8200, 390, 2000)]


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("low,high,power", [(228, 254, -100), (0, 26, 100), (0, 254, 0), (247, 247, -118)])
@pytest.mark.parametrize("yd", ["f32", "bf16"])
def test_weights_of_any_power(rows, k, n, low, high, power, yd):
    """Bytes of every size in a row: the blocks' sums are then of very different
    sizes, and the largest decides the bound."""
    rng = np.random.default_rng(rows + low)
    codes = rng.integers(0, 126, (n, k)).astype(np.uint8) | (rng.integers(0, 2, (n, k)) << 7).astype(np.uint8)
    codes[rng.random((n, k)) < 0.1] = 0
    scales = rng.integers(low, high + 1, (-(-n // 128), -(-k // 128))).astype(np.uint8)
    x = rng.standard_normal((rows, k))
    x[0] = 0.0
    if power == 0:  # every block's product near 1
        x *= np.repeat(np.ldexp(1.0, 127 - scales[0].astype(int)).clip(2.0 ** -110, 2.0 ** 115), 128)[:k]
        scales[:] = scales[0]
    x = torch.from_numpy((x * 2.0 ** power).astype(np.float32)).cuda()
    layer = M.Fp8Linear(k, n)
    layer.load_codes(codes, scales)
    got = layer.forward(x, out_dtype=DTYPES[yd])
    at = np.unique(np.concatenate([rng.integers(0, rows, 300), np.arange(min(rows, 100)), [rows - 1]]))
    want, mag = F.linear(x[at].double().cpu().numpy(), codes, scales)
    tol = (k + 64) * 2.0 ** -24 * mag + 2.0 ** -149
    if yd == "bf16":
        tol = tol + 7 * 2.0 ** -13 * mag + 2.0 ** -8 * np.abs(want)
    assert np.abs(want).max() < 2.0 ** 126
    got = got[at].double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])
