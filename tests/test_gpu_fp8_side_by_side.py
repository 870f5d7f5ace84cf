"""The 8-bit block-scaled projection from and into the columns of one buffer."""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k,n", [(1, 96, 40), (7, 200, 77), (300, 256, 96), (3000, 136, 264)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("out_first", [False, True])
def test_results_beside_their_rows(rows, k, n, dtype, out_first):
    rng = np.random.default_rng(rows)
    layer = M.Fp8Linear(k, n)
    layer.load_codes(*F.quantize_weight(rng.standard_normal((n, k)) / np.sqrt(k)))
    buf = torch.from_numpy(rng.standard_normal((rows, 3 + k + 5 + n)).astype(np.float32)).to(dtype).cuda()
    x, out = (buf[:, n + 5:n + 5 + k], buf[:, :n]) if out_first else (buf[:, 3:3 + k], buf[:, 3 + k + 5:])
    before, want = buf.clone(), layer.forward(x.contiguous())
    layer.forward(x, out=out)
    assert torch.equal(out, want)
    out.copy_(before[:, :n] if out_first else before[:, 3 + k + 5:])
    assert torch.equal(buf, before)


def test_rows_that_share_bytes_are_refused():
    k, n = 64, 48
    layer = M.Fp8Linear(k, n)
    layer.load_codes(np.zeros((n, k), np.uint8), np.full((1, 1), 127, np.uint8))
    buf = torch.zeros(20, k + n, device="cuda")
    for x, out in ((buf[:, :k], buf[:, k - 1:k - 1 + n]), (buf[:, n:], buf[:, 1:n + 1]), (buf[:, :k], buf[:, :n]),
                   (buf[1:, n - 1:n - 1 + k], buf[:-1, :n]),  # a row behind
                   (buf[:, n:], buf.view(-1)[:20 * n].view(20, n)),  # other distances
                   (buf[:8, :k], buf.view(torch.bfloat16)[4:12, :n])):
        with pytest.raises(M.MhsaError):
            layer.forward(x, out=out)
    layer.forward(buf[:10, :k], out=buf[10:, :n])
    layer.forward(buf[1:, :k], out=buf[:-1, k:])  # beside the row before
