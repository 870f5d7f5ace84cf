"""The operators on rows and the adapters past 2^31 elements and 2^32 bytes, and
calls at once on two streams: what is far is what the same rows give near."""
import pytest
import torch

import relpos_mhsa as M

pytestmark = pytest.mark.gpu


def test_norm_of_more_than_4_gib():
    rows, d = 280000, 8192
    x = torch.empty(rows, d, dtype=torch.bfloat16, device="cuda").normal_()
    got = M.add_norm(x, x, kind="layer", want="both")
    at = torch.cat([torch.arange(0, rows, 40009, device="cuda"), torch.arange(rows - 9, rows, device="cuda")])
    want = M.add_norm(x[at], x[at], kind="layer", want="both")
    assert torch.equal(got.out[at], want.out) and torch.equal(got.sum[at], want.sum)
    assert torch.equal(got.codes.codes[at], want.codes.codes) and torch.equal(got.codes.scales[at], want.codes.scales)


def test_logits_of_more_than_4_gib():
    for rows, v in ((36000, 65000), (2200000, 1025)):
        x = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda").normal_()
        tokens = (torch.arange(rows, device="cuda", dtype=torch.int32) * 7) % v
        got = M.token_log_probs(x, tokens, 3)
        at = torch.cat([torch.arange(0, rows, rows // 400 + 1, device="cuda"), torch.arange(rows - 600, rows, device="cuda")])
        want = M.token_log_probs(x[at], tokens[at], 3)  # (about 1000 rows: as many parts, one)
        for a, b in zip(got, want):
            assert torch.equal(a[at], b)
        del x, got


def test_the_last_of_many_adapters():
    """4096 adapters of rank 128: their matrices take 4 GiB each."""
    k, n, count = 4096, 4100, 4096
    layer, adapters = M.Fp8Linear(k, n), M.LowRankAdapters(k, n, count, 128)
    g = torch.Generator(device="cuda").manual_seed(1)
    layer.load(torch.randn(n, k, device="cuda", generator=g) / 64)
    few = M.LowRankAdapters(k, n, 2, 128)
    for i, slot in enumerate((0, count - 1)):
        a, b = torch.randn(100, k, device="cuda", generator=g) / 64, torch.randn(n, 100, device="cuda", generator=g) / 10
        adapters.load(slot, a, b)
        few.load(i, a, b)
    for rows in (1, 40, 3000):
        x = torch.randn(rows, k, device="cuda", generator=g).bfloat16()
        which = torch.randint(0, 2, (rows,), device="cuda", generator=g, dtype=torch.int32)
        assert torch.equal(layer.forward(x, adapters=adapters, which=which * (count - 1)),
                           layer.forward(x, adapters=few, which=which))


@pytest.mark.parametrize("rows", [2, 48, 2000])
def test_two_streams_at_once(rows):
    k, n = 512, 1200
    g = torch.Generator(device="cuda").manual_seed(rows)
    layer, adapters = M.Fp8Linear(k, n), M.LowRankAdapters(k, n, 3, 32)
    layer.load(torch.randn(n, k, device="cuda", generator=g) / 20)
    for i in range(3):
        adapters.load(i, torch.randn(32, k, device="cuda", generator=g) / 20, torch.randn(n, 32, device="cuda", generator=g) / 6)
    xs = [torch.randn(rows, k, device="cuda", generator=g) for _ in range(2)]
    ids = [torch.randint(-1, 3, (rows,), device="cuda", generator=g, dtype=torch.int32) for _ in range(2)]

    def step(i):
        r = M.add_norm(xs[i], xs[i], want="codes")
        y = layer.forward(r.codes, out_dtype=torch.float32, adapters=adapters, which=ids[i])
        return (y, layer.forward(xs[i], adapters=adapters, which=ids[i]), *M.token_log_probs(y, top_k=5)[1:])
    want = [step(0), step(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = step(i)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))
