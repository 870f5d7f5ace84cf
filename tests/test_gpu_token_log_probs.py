"""Log probabilities of tokens, entropy and the likeliest tokens against the
float64 oracle.

Tolerances, in steps of 2^-24 (half of f32's). d = (x - M) / T is off by 4 of
itself (the difference, the factor, the product), e^d by those and 2; the sums
of a row go through at most V / 64 + 64 additions of positive terms. So log S is
off by V / 64 + 66 + 4 E|d| + 2 |log S|, a log probability by that, 4 |d| and 4
of itself, and the entropy by the sums' steps of 1 + 2 E|d| + |log S| and, by
e^d's errors, 8 E d^2.
"""
import numpy as np
import pytest
import torch

import relpos_mhsa as M
import rows_oracle as R

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = 2.0 ** -24


def tensor(a, dtype):
    return torch.from_numpy(np.asarray(a, np.float32)).to(DTYPES[dtype]).cuda()


def f64(t):
    return t.double().cpu().numpy()


def close(got, want, tol):
    got = f64(got)
    off = ~np.isfinite(want)
    assert np.array_equal(got[off], want[off], equal_nan=True), (got[off], want[off])
    bad = np.abs(got[~off] - want[~off]) > np.broadcast_to(tol, want.shape)[~off]
    assert not bad.any(), (int(bad.sum()), got[~off][bad][:4], want[~off][bad][:4])


def check(x, tokens, top_k, temperature=1.0):
    """x [rows, V] on the GPU, tokens [rows, n] int32 (numpy)."""
    tok = torch.from_numpy(tokens).cuda()
    got = M.token_log_probs(x, tok, top_k, temperature)
    lp, h, idx, top, sizes = R.scores(f64(x), tokens, top_k, temperature)
    n = x.shape[1] / 64 + 66
    m1, m2, ls = sizes.T
    base = (n + 4 * m1 + 2 * ls)[:, None]
    assert got.log_probs.shape == tokens.shape and got.entropy.shape == (x.shape[0],)

    def tol(want):
        with np.errstate(invalid="ignore"):
            return STEP * (base + 4 * (np.abs(want) + ls[:, None]) + 4 * np.abs(want))
    close(got.log_probs, lp, tol(lp))
    close(got.entropy, h, STEP * (n * (1 + 2 * m1 + ls) + 8 * m2))
    if top_k:
        assert np.array_equal(got.top_indices.cpu().numpy(), idx)
        close(got.top_log_probs, top, tol(top))
    else:
        assert got.top_indices is None and got.top_log_probs is None


def logits(rng, rows, v, spread=3.0):
    return rng.standard_normal((rows, v)) * (0.2 + spread * rng.random((rows, 1)))


SIZES = [(1, 1), (1, 2), (3, 5), (2, 63), (5, 64), (4, 65), (1, 1025), (9, 1025), (6, 1024), (3, 2049), (2, 4096), (2, 4097),
         (5, 8193), (3, 16384), (1, 32768), (2, 50001), (1, 128000), (3, 100003), (520, 33000)]


@pytest.mark.parametrize("rows,v", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_against_oracle(rows, v, dtype):
    rng = np.random.default_rng(rows + v)
    for k in sorted({0, 1, min(5, v), min(32, v)}):
        tokens = rng.integers(-1, v + 1, (min(rows, 40), 1 + k % 3)).astype(np.int32)
        x = tensor(logits(rng, min(rows, 40), v), dtype)
        if rows > 40:  # sampled from a call of as many rows
            whole = x.repeat(-(-rows // 40), 1)[:rows]
            got, want = M.token_log_probs(whole, top_k=k), M.token_log_probs(whole[:40], top_k=k)
            assert torch.allclose(got.entropy, got.entropy[:40].repeat(-(-rows // 40))[:rows], rtol=0, atol=0)
            if k:
                assert torch.equal(got.top_indices[40:80], want.top_indices)
        check(x, tokens, k, [1.0, 0.5, 1.7][k % 3])


@pytest.mark.parametrize("v", [2049, 2052, 4095, 4097, 4104, 8192, 8193, 9002, 12301, 16384, 16391])
@pytest.mark.parametrize("rows", [6, 530])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ends_of_rows(rows, v, dtype):
    """The largest logits where a row, its waves' shares and their chunks begin and end."""
    rng = np.random.default_rng(v)
    few = logits(rng, 6, v)
    for i in range(6):
        for n, at in enumerate((v - 1, 0, v - 2 - i, v // 2 - i, v // 4 + i, 1024 + i, v - 9 - i)):
            few[i, at] = 40.0 + (n + i) % 7
    x = tensor(few, dtype)
    tokens = np.stack([np.full(6, v - 1), np.arange(6), v - 1 - np.arange(6), rng.integers(0, v, 6)], 1).astype(np.int32)
    if rows == 6:
        check(x, tokens, 9)
        check(x, tokens, 0)
        return
    whole = x.repeat(-(-rows // 6), 1)[:rows]
    got = M.token_log_probs(whole, torch.from_numpy(np.tile(tokens, (-(-rows // 6), 1))[:rows]).cuda(), 9)
    lp, h, idx, top, sizes = R.scores(f64(x), tokens, 9)
    # every logit is within 60 of the largest; as in check() otherwise
    n, (m1, m2, ls) = v / 64 + 66, sizes.T
    far = STEP * (n + 4 * m1 + 6 * ls + 8 * 60)[:, None]
    for i in (0, rows - rows % 6 - 6):
        assert np.array_equal(got.top_indices[i:i + 6].cpu().numpy(), idx)
        close(got.log_probs[i:i + 6], lp, far)
        close(got.top_log_probs[i:i + 6], top, far)
        close(got.entropy[i:i + 6], h, STEP * (n * (1 + 2 * m1 + ls) + 8 * m2))


@pytest.mark.parametrize("rows,v", [(2500, 1025), (1200, 5000)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(rows, v, dtype):
    g = torch.Generator(device="cuda").manual_seed(v)
    x = (3 * torch.randn(rows, v, device="cuda", generator=g)).to(DTYPES[dtype])
    tok = torch.randint(0, v, (rows,), device="cuda", generator=g, dtype=torch.int32)
    got = M.token_log_probs(x, tok, 8)
    want = torch.log_softmax(x.double(), -1)
    assert got.log_probs.shape == (rows,)
    assert (got.log_probs.double() - want.gather(1, tok.long()[:, None])[:, 0]).abs().max() < 400 * STEP
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[:, :8]
    assert torch.equal(got.top_indices.long(), order)
    assert (got.top_log_probs.double() - want.gather(1, order)).abs().max() < 400 * STEP


@pytest.mark.parametrize("v", [40, 1025, 5000, 40001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties_masks_and_extremes(v, dtype):
    rng = np.random.default_rng(v)
    low = float(torch.finfo(DTYPES[dtype]).min)
    x = logits(rng, 16, v)
    x[0] = 0.0                          # all alike
    x[1] = -np.inf                      # nothing is left
    x[2, rng.random(v) < 0.9] = -np.inf
    x[3] = -np.inf
    x[3, [v - 1, 3, v // 2]] = 1.0, -2.0, 1.0
    x[4] = low                          # all masked by the lowest value
    x[5] = low
    x[5, [v - 2, 7]] = 3.0, 4.0         # all but two
    x[6] = np.arange(v) * 1e-3          # each larger than the ones before
    x[7] = -np.arange(v) * 1e-3
    x[8] = rng.integers(0, 3, v)        # many ties
    x[9, ::2], x[9, 1::2] = 0.0, -0.0   # alike
    x[10, v // 3] = np.nan
    x[11, v - 1] = np.inf
    x[12] *= 1e30
    x[13] = -1e4
    x[13, v - 1] = 0.0                  # sure
    x[14, 0] = -low                     # the two ends in one row
    x[14, 1] = low
    x[15] = np.nan
    t = tensor(x, dtype)
    tokens = np.stack([np.full(16, 0), np.full(16, v - 1), np.full(16, -1), np.full(16, v), np.full(16, 3)], 1).astype(np.int32)
    for k in (0, 1, 3, 20, 32):
        check(t, tokens, k)


@pytest.mark.parametrize("v", [3000, 30000])
def test_candidates_in_every_order(v):
    """Rising, falling, best in one lane or one chunk, few alternatives left:
    lists that overflow, and ties at their border."""
    rng = np.random.default_rng(v)
    x = np.stack([np.arange(v), np.arange(v)[::-1], np.arange(v) // 70, np.arange(v)[::-1] // 70, rng.permutation(v),
                  np.where(np.arange(v) % 64 == 5, 100.0 + np.arange(v) % 7, 0.0), np.where(np.arange(v) > v - 40, 9.0, 0.0),
                  np.where(np.arange(v) < 40, 9.0, 0.0), rng.permutation(v) // 40]).astype(np.float64) / 256
    for dtype in ("f32", "bf16"):
        for k in (2, 17, 32):
            check(tensor(x, dtype), np.zeros((len(x), 1), np.int32), k)


def test_strides_shapes_and_odd_addresses():
    rng = np.random.default_rng(0)
    for dtype in ("f32", "bf16"):
        buf = tensor(logits(rng, 7, 1100), dtype)
        x = buf[:, 3:1028]
        tokens = rng.integers(0, 1025, (7, 2)).astype(np.int32)
        check(x, tokens, 6)
        cube = tensor(logits(rng, 6, 77), dtype).view(2, 3, 77)
        tok = torch.from_numpy(rng.integers(0, 77, (2, 3)).astype(np.int32)).cuda()
        got, flat = M.token_log_probs(cube, tok, 3), M.token_log_probs(cube.view(6, 77), tok.view(6), 3)
        assert got.log_probs.shape == (2, 3) and got.entropy.shape == (2, 3) and got.top_indices.shape == (2, 3, 3)
        assert torch.equal(got.log_probs.view(6), flat.log_probs) and torch.equal(got.top_indices.view(6, 3), flat.top_indices)
        one = M.token_log_probs(cube[0, 0])
        assert one.entropy.shape == () and one.log_probs is None


def test_no_rows():
    got = M.token_log_probs(torch.empty(0, 50, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), 4)
    assert got.log_probs.shape == (0,) and got.top_indices.shape == (0, 4)


@pytest.mark.parametrize("rows,v", [(3, 1025), (2, 60000)])
def test_streams_and_graphs(rows, v):
    x = torch.randn(rows, v, device="cuda")
    tok = torch.zeros(rows, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        M.token_log_probs(x, tok, 5)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = M.token_log_probs(x, tok, 5)
    for i in range(4):
        x.copy_(torch.randn(rows, v, device="cuda") * (i + 1))
        graph.replay()
        want = M.token_log_probs(x, tok, 5)
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    tok = torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: M.token_log_probs(x.cpu()), lambda: M.token_log_probs(x.half()), lambda: M.token_log_probs(None),
                lambda: M.token_log_probs(x, tok.long()), lambda: M.token_log_probs(x, tok[:3]), lambda: M.token_log_probs(x, tok.cpu()),
                lambda: M.token_log_probs(x, top_k=65), lambda: M.token_log_probs(x, top_k=33), lambda: M.token_log_probs(x, top_k=-1),
                lambda: M.token_log_probs(x, temperature=0.0), lambda: M.token_log_probs(x, temperature=float("nan")),
                lambda: M.token_log_probs(x, temperature=1e9), lambda: M.token_log_probs(x.t()),
                lambda: M.token_log_probs(x, tok[:, None].expand(4, 2)), lambda: M.token_log_probs(x[:, :0])):
        with pytest.raises(M.MhsaError):
            bad()


@pytest.mark.parametrize("rows,v", [(3, 5000), (520, 9848), (2, 40001)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_masks_that_leave_a_stretch(rows, v, dtype):
    """Some waves have no token at all, or fewer than are asked for."""
    rng = np.random.default_rng(v)
    few = logits(rng, 3, v)
    for i, (lo, hi) in enumerate(((0, v // 9), (v // 2 + 5, v // 2 + 12), (v - v // 7, v))):
        few[i, :lo] = few[i, hi:] = -np.inf
    x = tensor(few[:rows], dtype)
    tokens = rng.integers(-1, v, (len(x), 2)).astype(np.int32)
    check(x, tokens, 20)
    if rows > 3:
        whole = x.repeat(-(-rows // 3), 1)[:rows]
        got, want = M.token_log_probs(whole, top_k=20), M.token_log_probs(x, top_k=20)
        assert torch.equal(got.top_indices[-3 - rows % 3:][:3], want.top_indices)
