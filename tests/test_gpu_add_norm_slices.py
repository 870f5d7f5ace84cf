"""A residual's addition with its norm of more rows than one launch takes (2^21):
rows on both sides of where one launch ends and the next begins are what the
same rows give in a call of their own, in every tensor that is read or written."""
import pytest
import torch

import relpos_mhsa as M

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [7, 8, 13, 520, 4104])  # one, two and sixteen waves a row
def test_rows_past_a_launch(d):
    rows, cut = (1 << 22) + 300, 1 << 21
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    delta = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    w, b = torch.rand(d, device="cuda", generator=g), torch.rand(d, device="cuda", generator=g)
    at = torch.cat([torch.arange(lo, hi, device="cuda") for lo, hi in
                    ((0, 70), (cut - 70, cut + 70), (2 * cut - 70, 2 * cut + 70), (rows - 70, rows))]
                   + [torch.randint(0, rows, (500,), device="cuda", generator=g)]).unique()
    want = M.add_norm(x[at], delta[at], w, b, kind="layer", want="both", scale=0.5)
    got = M.add_norm(x, delta, w, b, kind="layer", want="both", scale=0.5, sum_out=x, out=delta)
    assert torch.equal(x[at], want.sum) and torch.equal(delta[at], want.out)
    assert torch.equal(got.codes.codes[at], want.codes.codes) and torch.equal(got.codes.scales[at], want.codes.scales)
    del x, delta, got
    torch.cuda.empty_cache()
