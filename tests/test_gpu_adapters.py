"""Low-rank adapters beside the 8-bit projection, and the projection from
rounded rows, against the float64 oracle.

Tolerances. The projection's as in test_gpu_fp8_linear. The adapters' products
are exact (bf16 by bf16, f32 as three bf16 parts) but for what the parts lose
under 2^-24 of a value, and sums are f32: K + rank + 64 steps of 2^-24 of the
magnitudes that pass through both products. For a bf16 result the inner sums are
rounded to bf16, by at most 2^-8 of each, and the result by 2^-8 of itself.
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


def tensor(a, dtype):
    return torch.from_numpy(np.asarray(a, np.float32)).to(DTYPES[dtype]).cuda()


class Made:
    """A projection with adapters, and their oracle."""

    def __init__(self, rng, k, n, ranks, max_rank, bias=True, gain=1.0):
        self.codes, self.scales = F.quantize_weight(rng.standard_normal((n, k)) / np.sqrt(k))
        self.bias = (0.1 * rng.standard_normal(n)).astype(np.float32) if bias else None
        self.layer = M.Fp8Linear(k, n, bias)
        self.layer.load_codes(self.codes, self.scales, self.bias)
        self.adapters = M.LowRankAdapters(k, n, len(ranks), max_rank)
        self.parts = []
        for i, r in enumerate(ranks):
            a = torch.from_numpy(gain * rng.standard_normal((max(r, 1), k)) / np.sqrt(k)).float().bfloat16()
            b = torch.from_numpy(rng.standard_normal((n, max(r, 1))) / np.sqrt(max(r, 1))).float().bfloat16()
            s = float(np.float32(rng.uniform(-2, 2)))
            if r:
                self.adapters.load(i, a, b, s)
            else:
                s = 0.0
            self.parts.append((a.double().numpy(), b.double().numpy(), s))
        self.k, self.n = k, n

    def check(self, got, x, which, values=None):
        """x: as the adapters see it, values: as the projection does (None: x rounded)."""
        x = x.double().cpu().numpy()
        want, mag = F.linear(x if values is None else values, self.codes, self.scales, self.bias)
        if self.bias is not None:
            mag = mag + np.abs(self.bias)
        add, through, inner = R.adapted(x, which, self.parts)
        tol = (self.k + 64) * STEP * mag + (self.k + 128 + 64) * STEP * through
        want = want + add
        if got.dtype == torch.bfloat16:
            tol = tol + 7 * 2.0 ** -13 * mag + 2.0 ** -8 * inner + 2.0 ** -8 * np.abs(want)
        got = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(got), np.isnan(want))
        bad = np.abs(got - want) > tol + 1e-37
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), np.nanmax(np.abs(got - want) / (tol + 1e-37)))


def requests(rng, rows, n, count):
    """Adapters of rows in runs, some of none."""
    which = np.empty(rows, np.int32)
    ends = np.sort(rng.integers(0, rows + 1, count - 1)) if count > 1 else []
    for part in np.split(np.arange(rows), ends):
        which[part] = rng.integers(-1, n)
    return which


SHAPES = [  # rows, in, out, ranks, max_rank, requests
    (1, 1, 1, [1], 1, 1), (1, 1024, 512, [16, 8, 0], 16, 1), (3, 100, 33, [3, 5], 7, 3), (16, 129, 130, [17, 32, 1], 32, 16),
    (17, 512, 2048, [16] * 5, 16, 9), (33, 640, 1025, [64, 20], 64, 4), (64, 256, 300, [128, 100], 128, 64),
    (112, 512, 256, [16] * 8, 16, 8), (300, 1000, 333, [24, 16, 9], 24, 20), (257, 2176, 130, [33], 40, 5),
    (700, 384, 640, [16] * 40, 16, 300), (1500, 256, 1100, [32, 7, 0, 30], 32, 6), (4100, 640, 2049, [64] * 6, 64, 30)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s[:3])))
@pytest.mark.parametrize("xd,yd", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_against_oracle(shape, xd, yd):
    rows, k, n, ranks, max_rank, count = shape
    rng = np.random.default_rng(rows + k + n)
    made = Made(rng, k, n, ranks, max_rank, bias=(rows + k) % 2 == 0)
    x = tensor(rng.standard_normal((rows, k)) * np.exp(0.5 * rng.standard_normal(k)), xd)
    which = requests(rng, rows, len(ranks), count)
    got = made.layer.forward(x, out_dtype=DTYPES[yd], adapters=made.adapters, which=torch.from_numpy(which).cuda())
    assert got.shape == (rows, n) and got.dtype == DTYPES[yd]
    made.check(got, x, which)
    # of no adapter at all: the projection, to the bit
    none = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(made.layer.forward(x, out_dtype=DTYPES[yd], adapters=made.adapters, which=none),
                       made.layer.forward(x, out_dtype=DTYPES[yd]))


@pytest.mark.parametrize("rows,k,n,count", [(9001, 520, 2300, 70), (6200, 700, 1800, 6000), (16300, 300, 2040, 1)])
@pytest.mark.parametrize("yd", ["bf16", "f32"])
def test_many_rows(rows, k, n, count, yd):
    """Large tiles, several to a workgroup, one to many adapters to a tile:
    sampled rows, and the last ones."""
    rng = np.random.default_rng(rows)
    made = Made(rng, k, n, [32, 16, 9, 27, 1], 32)
    x = tensor(rng.standard_normal((rows, k)), "bf16")
    which = requests(rng, rows, 5, count)
    if count == 1:
        which[:] = 3
    got = made.layer.forward(x, out_dtype=DTYPES[yd], adapters=made.adapters, which=torch.from_numpy(which).cuda())
    at = np.unique(np.concatenate([rng.integers(0, rows, 400), np.arange(rows - 300, rows)]))
    made.check(got[at], x[at], which[at])


@pytest.mark.parametrize("rows,k,n,ranks", [(1100, 5, 40, [3, 16]), (1030, 1001, 96, [40, 7]), (1024, 520, 64, [100]),
                                            (6, 4100, 64, [16, 9, 2]), (203, 2600, 130, [60, 30, 5, 1])])
@pytest.mark.parametrize("xd,yd", [("bf16", "bf16"), ("f32", "f32")])
def test_requests_of_every_length(rows, k, n, ranks, xd, yd):
    """Adapters that change from row to row, and rows of no whole runs of 8, few and many."""
    rng = np.random.default_rng(rows + n)
    made = Made(rng, k, n, ranks, max(ranks))
    x = tensor(rng.standard_normal((rows, k)), xd)
    for which in (requests(rng, rows, len(ranks), rows), rng.integers(-1, len(ranks), rows).astype(np.int32)):
        got = made.layer.forward(x, out_dtype=DTYPES[yd], adapters=made.adapters, which=torch.from_numpy(which).cuda())
        made.check(got, x, which)


@pytest.mark.parametrize("rows,k,n", [(1, 128, 64), (5, 100, 40), (16, 1000, 130), (40, 512, 2048), (300, 384, 333), (3000, 512, 2050),
                                      (2, 2200, 96)])
@pytest.mark.parametrize("yd", ["bf16", "f32"])
@pytest.mark.parametrize("lora", [False, True])
def test_from_a_norm(rows, k, n, yd, lora):
    """The norm's codes through the projection: what the norm's f32 values give,
    to the bit, and with adapters on the codes' values within the bounds."""
    rng = np.random.default_rng(rows + k)
    made = Made(rng, k, n, [16, 5], 16)
    x, delta = tensor(rng.standard_normal((rows, k)), "bf16"), tensor(rng.standard_normal((rows, k)), "bf16")
    w = tensor(np.exp(0.5 * rng.standard_normal(k)), "f32")
    r = M.add_norm(x, delta, w, want="both", out_dtype=torch.float32)
    if not lora:
        assert torch.equal(made.layer.forward(r.codes, out_dtype=DTYPES[yd]), made.layer.forward(r.out, out_dtype=DTYPES[yd]))
        if yd == "bf16":
            out = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda")
            assert made.layer.forward(r.codes, out=out) is out and torch.equal(out, made.layer.forward(r.codes))
        return
    which = requests(rng, rows, 2, 5)
    got = made.layer.forward(r.codes, out_dtype=DTYPES[yd], adapters=made.adapters, which=torch.from_numpy(which).cuda())
    values = F.round_rows(r.out.double().cpu().numpy())
    made.check(got, torch.from_numpy(values), which, values)


def test_a_serving_step():
    """Norm, projection with adapters, scores, as a decoder's head runs them, on
    packed requests; captured and replayed with other rows and other adapters."""
    rng = np.random.default_rng(8)
    rows, k, n = 40, 640, 1025
    made = Made(rng, k, n, [16, 8, 12], 16)
    x, delta = tensor(rng.standard_normal((rows, k)), "bf16"), tensor(rng.standard_normal((rows, k)), "bf16")
    w = torch.ones(k, device="cuda")
    which = torch.from_numpy(requests(rng, rows, 3, 6)).cuda()
    tokens = torch.from_numpy(rng.integers(0, n, rows).astype(np.int32)).cuda()

    def step():
        r = M.add_norm(x, delta, w, want="codes")
        logits = made.layer.forward(r.codes, out_dtype=torch.float32, adapters=made.adapters, which=which)
        return (r.sum, logits, *M.token_log_probs(logits, tokens, top_k=4))
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        x.copy_(tensor(rng.standard_normal((rows, k)), "bf16"))
        which.copy_(torch.from_numpy(requests(rng, rows, 3, 6)).cuda())
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
        lp = torch.log_softmax(want[1].double(), -1)
        # 1025 / 64 + 66 sums' steps, and d and log S (up to 40) ten steps each at most
        assert (want[2].double() - lp.gather(1, tokens.long()[:, None])[:, 0]).abs().max() < 500 * STEP
        assert torch.equal(want[4].long(), torch.sort(want[1], dim=-1, descending=True, stable=True).indices[:, :4])


@pytest.mark.parametrize("rows", [4, 30, 300])
@pytest.mark.parametrize("yd", ["bf16", "f32"])
def test_infinities_stay_in_their_rows_and_any_index_is_one_or_none(rows, yd):
    rng = np.random.default_rng(rows)
    made = Made(rng, 200, 150, [8, 16], 16)
    x = rng.standard_normal((rows, 200))
    x[1, 5], x[2, 100] = np.inf, np.nan
    x = tensor(x, "f32")
    which = rng.integers(0, 2, rows).astype(np.int32)
    which[3] = -7
    which[0] = 1 << 30
    which[rows - 1] = -(1 << 31)
    got = made.layer.forward(x, out_dtype=DTYPES[yd], adapters=made.adapters, which=torch.from_numpy(which).cuda())
    assert torch.isnan(got[1:3]).all()
    keep = [r for r in range(rows) if r not in (1, 2)]
    made.check(got[keep], x[keep], which[keep])


def test_slots_are_replaced_and_emptied():
    rng = np.random.default_rng(1)
    made = Made(rng, 96, 80, [16, 4], 20)
    x = tensor(rng.standard_normal((10, 96)), "f32")
    which = np.arange(10).astype(np.int32) % 2
    ids = torch.from_numpy(which).cuda()
    a, b = rng.standard_normal((2, 96)).astype(np.float32), rng.standard_normal((80, 2)).astype(np.float32)
    made.adapters.load(0, a, b, 0.5)  # of a smaller rank, f32, from the host
    made.parts[0] = (torch.from_numpy(a).bfloat16().double().numpy(), torch.from_numpy(b).bfloat16().double().numpy(), 0.5)
    made.check(made.layer.forward(x, adapters=made.adapters, which=ids), x, which)
    bad = a.copy()
    bad[1, 3] = np.inf
    for args in ((0, bad, b), (0, a, np.full_like(b, 3.4e38)), (0, np.full_like(a, np.nan), b)):
        with pytest.raises(M.MhsaError):
            made.adapters.load(*args)
    made.check(made.layer.forward(x, adapters=made.adapters, which=ids), x, which)  # as before
    made.adapters.clear(0)
    made.parts[0] = (*made.parts[0][:2], 0.0)
    made.check(made.layer.forward(x, adapters=made.adapters, which=ids), x, which)


def test_strides_streams_and_shapes():
    rng = np.random.default_rng(2)
    for rows in (6, 400):
        made = Made(rng, 130, 70, [8], 8)
        buf = tensor(rng.standard_normal((rows, 300)), "bf16")
        before = buf.clone()
        which = requests(rng, rows, 1, 4)
        ids = torch.from_numpy(which).cuda()
        x, out = buf[:, 3:133], buf[:, 140:210]
        want = made.layer.forward(x.contiguous(), adapters=made.adapters, which=ids)
        made.layer.forward(x, out=out, adapters=made.adapters, which=ids)
        assert torch.equal(out, want)
        out.copy_(before[:, 140:210])
        assert torch.equal(buf, before)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            other = made.layer.forward(x, adapters=made.adapters, which=ids)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(other, want)
        cube = x.contiguous().view(2, rows // 2, 130)
        assert torch.equal(made.layer.forward(cube, adapters=made.adapters, which=ids.view(2, -1)).view(rows, 70), want)
    empty = made.layer.forward(torch.empty(0, 130, device="cuda"), adapters=made.adapters, which=ids[:0])
    assert empty.shape == (0, 70)


def test_refusals():
    rng = np.random.default_rng(3)
    made = Made(rng, 64, 48, [4], 8, bias=False)
    x = torch.zeros(5, 64, device="cuda")
    ids = torch.zeros(5, dtype=torch.int32, device="cuda")
    other, unloaded = M.LowRankAdapters(64, 49, 1, 8), M.LowRankAdapters(64, 48, 1, 8)
    r = M.add_norm(x, want="codes").codes
    narrow = M.add_norm(x[:, :32], want="codes").codes

    def go(t=x, **kw):
        return lambda: made.layer.forward(t, **{"adapters": made.adapters, "which": ids, **kw})
    for bad in (go(which=None), go(which=ids.long()), go(which=ids[:4]), go(which=ids.cpu()), go(which=ids[:, None]), go(adapters=None),
                go(adapters=other), go(adapters=unloaded), go(adapters=3), go(t=narrow), go(out=x[:, :48]), go(t=r, which=ids[:4]),
                go(t=x[:, :63]), go(t=x.half()), lambda: made.adapters.load(1, torch.zeros(4, 64), torch.zeros(48, 4)),
                lambda: made.adapters.load(0, torch.zeros(9, 64), torch.zeros(48, 9)), lambda: made.adapters.load(0, torch.zeros(4, 63), torch.zeros(48, 4)),
                lambda: made.adapters.load(0, torch.zeros(4, 64), torch.zeros(48, 5)), lambda: made.adapters.load(0, torch.zeros(4, 64), None),
                lambda: made.adapters.load(0, torch.zeros(4, 64), torch.zeros(48, 4).half()),
                lambda: made.adapters.load(0, torch.zeros(4, 64), torch.zeros(48, 4), float("nan")),
                lambda: made.adapters.load(0, None, None), lambda: made.adapters.clear(-1),
                lambda: M.LowRankAdapters(64, 48, 0, 8), lambda: M.LowRankAdapters(64, 48, 1, 129), lambda: M.LowRankAdapters(0, 48, 1, 8)):
        with pytest.raises(M.MhsaError):
            bad()
