"""The experts' FeedForward against the float64 oracle.

The fp8 matrix unit's sums are off by at most 7 * 2^-13 of their terms'
magnitudes (it adds products in groups of 8 and drops, of each but the largest,
less than 2^-13 of the largest's power of two) beside f32 roundings; the oracle's bound carries that through silu, the codes a hidden value may then
round to, and the second product. f32 sums in the combination and the store add
64 steps of 2^-24, a bf16 store 2^-8 of the value. Beside that bound, which
assumes the worst of every value, the whole result is held in the 2-norm to
1e-2: half of that for the store (2^-8), the rest for hidden values at a
code's edge (0.4% of them a step of 2^-3 off give 6e-3).
"""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu
SUM = 7 * 2.0 ** -13 + 2.0 ** -14
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(rng, e, d, f, bias):
    lin1 = [F.quantize_weight(rng.standard_normal((f, d)) / np.sqrt(d)) for _ in range(e)]
    lin2 = [F.quantize_weight(rng.standard_normal((d, f)) / np.sqrt(f)) for _ in range(e)]
    b1 = (0.2 * rng.standard_normal((e, f))).astype(np.float32) if bias else None
    b2 = (0.2 * rng.standard_normal((e, d))).astype(np.float32) if bias else None
    layer = M.ExpertFeedForward(e, d, f, bias)
    layer.load_codes(*(np.stack([m[i] for m in lin]) for lin in (lin1, lin2) for i in (0, 1)), b1, b2)
    return layer, lin1, lin2, b1, b2


def choose(rng, rows, e, k, skew=0.0):
    """k experts a row, some rows none, some fewer, some one expert twice, some an index out of range."""
    g = rng.standard_normal((rows, e)) - skew * np.log1p(np.arange(e))
    idx = np.argsort(-g, axis=1)[:, :k].astype(np.int32)
    if k > e:
        idx = np.concatenate([idx, rng.integers(0, e, (rows, k - e)).astype(np.int32)], 1)
    if rows > 3:
        idx[rng.integers(0, rows)] = -1
        idx[rng.integers(0, rows), 0] = -1
        idx[rng.integers(0, rows), -1] = e
        idx[rng.integers(0, rows)] = rng.integers(0, e)
    return idx, rng.uniform(0.05, 1.0, (rows, k)).astype(np.float32)


def frames(rng, rows, d, dtype):
    return torch.from_numpy((rng.standard_normal((rows, d)) * np.exp(0.5 * rng.standard_normal(d))).astype(np.float32)).to(DTYPES[dtype]).cuda()


def host(t):
    return None if t is None else t.double().cpu().numpy()


def check(got, x, idx, w, parts, residual=None, res_scale=1.0):
    _, lin1, lin2, b1, b2 = parts
    want, bound = F.experts(host(x), idx, w, lin1, lin2, b1, b2, host(residual), res_scale, sum_err=SUM)
    tol = bound + 64 * 2.0 ** -24 * (np.abs(want) + bound / SUM)
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (np.abs(want) + bound)
    got = host(got)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > tol + 1e-30
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())
    norm = np.linalg.norm(want)
    assert np.linalg.norm(got - want) <= 1e-2 * norm, np.linalg.norm(got - want) / norm


CASES = [(1, 2, 64, 64, 1), (1, 8, 256, 512, 2), (3, 4, 192, 320, 4), (16, 2, 128, 128, 2), (31, 8, 256, 384, 2), (64, 3, 128, 256, 1),
         (70, 5, 192, 192, 1), (112, 32, 128, 256, 2), (200, 16, 64, 448, 3), (333, 4, 256, 512, 2), (500, 1, 320, 192, 1),
         (1000, 8, 128, 256, 4), (900, 2, 384, 640, 2), (3000, 3, 128, 320, 1), (40, 1, 128, 64, 5), (150, 400, 64, 64, 2)]


@pytest.mark.parametrize("rows,e,d,f,k", CASES)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_against_oracle(rows, e, d, f, k, dtype):
    rng = np.random.default_rng(rows + e + d)
    parts = make(rng, e, d, f, bias=rows % 2 == 1)
    x = frames(rng, rows, d, dtype)
    idx, w = choose(rng, rows, e, k, skew=0.5)
    got = parts[0].forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    check(got, x, idx, w, parts)
    r = frames(rng, rows, d, dtype)
    args = (x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    got = parts[0].forward(*args, residual=r, res_scale=0.5)
    check(got, x, idx, w, parts, r, 0.5)
    inplace = r.clone()
    assert parts[0].forward(*args, residual=inplace, res_scale=0.5, out=inplace) is inplace
    assert torch.equal(inplace, got)


@pytest.mark.parametrize("rows,e,d,f,k,skew", [(21000, 3, 256, 512, 2, 0.3), (30000, 9, 320, 192, 2, 1.5), (9000, 2, 192, 1088, 3, 0.0)])
def test_many_large_tiles(rows, e, d, f, k, skew):
    """Several tiles to a workgroup in both products, experts of very different
    numbers of frames: sampled frames, and the last ones."""
    rng = np.random.default_rng(rows)
    parts = make(rng, e, d, f, bias=True)
    x = frames(rng, rows, d, "bf16")
    idx, w = choose(rng, rows, e, k, skew=skew)
    got = parts[0].forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    at = np.unique(np.concatenate([rng.integers(0, rows, 500), np.arange(rows - 300, rows)]))
    check(got[at], x[at], idx[at], w[at], parts)
    again = parts[0].forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    assert torch.equal(got, again)


@pytest.mark.parametrize("rows,e,k", [(700, 150, 4), (3000, 512, 4), (1100, 256, 8), (4000, 70, 3), (129, 1, 2), (40, 1, 5),
                                      (1, 256, 8), (8, 100, 8), (9, 100, 8), (16, 64, 16), (63, 64, 4), (32, 33, 8)])
def test_few_rows_of_many_experts(rows, e, k):
    """Lists of pairs of several thousands, experts of fewer than 16 frames, of
    more and of none; one expert of all of them."""
    rng = np.random.default_rng(rows)
    parts = make(rng, e, 128, 128, bias=True)
    x = frames(rng, rows, 128, "bf16")
    idx, w = choose(rng, rows, e, k, skew=0.2)
    got = parts[0].forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    check(got, x, idx, w, parts)


@pytest.mark.parametrize("rows,e", [(1, 2), (14, 2), (60, 2), (250, 1), (900, 64)])
def test_few_rows_round_hidden_values_from_f32_sums(rows, e):
    """A second matrix of the identity returns the hidden values' codes: those
    of a value that is off by at most (K + 64) steps of 2^-24 of its sum's
    magnitudes (silu's slope is at most 1.1) and 8 of its own."""
    rng = np.random.default_rng(rows + e)
    d = 512
    lin1 = [F.quantize_weight(rng.standard_normal((d, d)) / np.sqrt(d)) for _ in range(e)]
    one = np.zeros((d, d), np.uint8)
    one[np.arange(d), np.arange(d)] = 0x38
    layer = M.ExpertFeedForward(e, d, d, False)
    layer.load_codes(np.stack([m[0] for m in lin1]), np.stack([m[1] for m in lin1]), np.stack([one] * e),
                     np.full((e, 4, 4), 127, np.uint8))
    x, idx = frames(rng, rows, d, "f32"), rng.integers(0, e, (rows, 1)).astype(np.int32)
    got = host(layer.forward(x, torch.from_numpy(idx).cuda(), torch.ones(rows, 1, device="cuda")))
    for k in range(e):
        at = idx[:, 0] == k
        h, mag = F.linear(host(x)[at], *lin1[k])
        v = h / (1 + np.exp(-h))
        err = 1.1 * (d + 64) * 2.0 ** -24 * mag + 8 * 2.0 ** -24 * np.abs(v)
        for c in range(0, d, 128):
            b, eb, y = v[:, c:c + 128], err[:, c:c + 128], got[at, c:c + 128]
            s = [F.scale_byte((np.abs(b) + i * eb).max(1, initial=0))[:, None] - 127 for i in (-1, 1)]
            same = (s[0] == s[1])[:, 0]  # (a largest value next to a power's edge may take either)
            lo, hi = (np.ldexp(F.VALUES[F.encode(np.clip(np.ldexp(b + i * eb, -s[0]), -448, 448))], s[0]) for i in (-1, 1))
            assert ((lo <= y) & (y <= hi))[same].all()


@pytest.mark.parametrize("rows", [2, 100, 2000])
def test_rows_without_experts_are_the_residual(rows):
    rng = np.random.default_rng(1)
    parts = make(rng, 4, 128, 256, True)
    x, r = frames(rng, rows, 128, "bf16"), frames(rng, rows, 128, "bf16")
    x[0] = float("nan")  # what a frame without an expert holds does not matter
    idx = torch.full((rows, 2), -1, dtype=torch.int32, device="cuda")
    w = torch.full((rows, 2), float("nan"), device="cuda")
    assert torch.equal(parts[0].forward(x, idx, w, residual=r), r)
    assert (parts[0].forward(x, idx, w) == 0).all()
    idx[1, 1], w[1, 1] = 2, 0.5
    got = parts[0].forward(x, idx, w, residual=r)
    assert torch.equal(got[0], r[0]) and torch.equal(got[2:], r[2:])
    check(got[1:2], x[1:2], idx[1:2].cpu().numpy(), np.nan_to_num(w[1:2].cpu().numpy()), parts, r[1:2])


@pytest.mark.parametrize("rows", [20, 400])
def test_nans_stay_in_their_rows(rows):
    rng = np.random.default_rng(2)
    parts = make(rng, 2, 128, 256, False)
    x = frames(rng, rows, 128, "bf16")
    idx, w = choose(np.random.default_rng(3), rows, 2, 2)
    idx[idx < 0] = 0
    idx[idx >= 2] = 0
    t = (torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda())
    clean = parts[0].forward(x, *t)
    x[4, 3] = float("inf")
    got = parts[0].forward(x, *t)
    assert torch.isnan(got[4]).all()
    keep = [i for i in range(rows) if i != 4]
    assert torch.equal(got[keep], clean[keep])


def test_floats_are_rounded_at_loading():
    rng = np.random.default_rng(4)
    e, d, f = 3, 192, 128
    w1 = torch.from_numpy((rng.standard_normal((e, f, d)) / 14).astype(np.float32)).bfloat16()
    w2 = torch.from_numpy((rng.standard_normal((e, d, f)) / 11).astype(np.float32)).bfloat16()
    b1, b2 = torch.randn(e, f).bfloat16(), torch.randn(e, d).bfloat16()
    lin1, lin2 = ([F.quantize_weight(m.double().numpy()) for m in w] for w in (w1, w2))
    x = frames(rng, 90, d, "f32")
    idx, w = choose(rng, 90, e, 2)
    outs = []
    for dev in ("cpu", "cuda"):
        layer = M.ExpertFeedForward(e, d, f, True)
        layer.load(w1.to(dev), w2.to(dev), b1.to(dev), b2.to(dev))
        outs.append(layer.forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()))
        check(outs[-1], x, idx, w, (layer, lin1, lin2, b1.float().numpy(), b2.float().numpy()))
    assert torch.equal(*outs)


def test_more_pairs_than_one_part_takes():
    """Rows run in parts of up to 2^18 pairs: the same rows in another part give
    the same bits, and sampled rows match the oracle."""
    rng = np.random.default_rng(5)
    parts = make(rng, 3, 64, 64, True)
    x = frames(rng, 1000, 64, "bf16").repeat(100, 1)
    idx, w = choose(rng, 1000, 3, 3)
    t = (torch.from_numpy(idx).cuda().repeat(100, 1), torch.from_numpy(w).cuda().repeat(100, 1))
    got = parts[0].forward(x, *t).view(100, 1000, 64)
    assert all(torch.equal(got[0], got[i]) for i in range(1, 100))
    check(got[99], x[:1000], idx, w, parts)


def test_empty_shapes_and_refusals():
    rng = np.random.default_rng(6)
    parts = make(rng, 3, 128, 64, False)
    layer, x = parts[0], frames(rng, 12, 128, "bf16")
    idx, w = choose(rng, 12, 3, 2)
    idx, w = torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()
    assert layer.forward(x[:0], idx[:0], w[:0]).shape == (0, 128)
    assert torch.equal(layer.forward(x.view(3, 4, 128), idx.view(3, 4, 2), w.view(3, 4, 2)).view(12, 128), layer.forward(x, idx, w))
    for args, kw in (((x, idx.long(), w), {}), ((x, idx, w.double()), {}), ((x, idx[:5], w), {}), ((x[:, :64], idx, w), {}),
                     ((x, idx, w), {"out": x}), ((x, idx, w), {"residual": x.float()}), ((x.half(), idx, w), {}),
                     ((x, idx[:, :0], w[:, :0]), {}), ((x, idx, w), {"out": torch.empty(24, 128, device="cuda", dtype=x.dtype)[::2]})):
        with pytest.raises(M.MhsaError):
            layer.forward(*args, **kw)
    buf = frames(rng, 24, 128, "bf16")
    with pytest.raises(M.MhsaError):  # out lies half over the residual
        layer.forward(x, idx, w, residual=buf[:12], out=buf[6:18])


def test_a_load_that_fails_halfway_leaves_no_mixture():
    rng = np.random.default_rng(11)
    parts = make(rng, 3, 128, 64, True)
    layer, x = parts[0], frames(rng, 4, 128, "bf16")
    idx, w = (torch.from_numpy(a).cuda() for a in choose(rng, 4, 3, 2))
    w1, w2, b1 = torch.randn(3, 64, 128), torch.randn(3, 128, 64), torch.zeros(3, 64)
    assert M.library().mhsa_experts_load(layer._h, M.F32, w1.data_ptr(), b1.data_ptr(), w2.data_ptr(), None) == M.MHSA_EINVAL
    with pytest.raises(M.MhsaError):
        layer.forward(x, idx, w)
    layer.load(w1, w2, b1, torch.zeros(3, 128))
    assert torch.isfinite(layer.forward(x, idx, w)).all()
    none = torch.zeros((), dtype=torch.int32, device="cuda")
    with pytest.raises(M.MhsaError):
        layer.forward(x[0], none, none.float())


def test_replayed_graphs_and_streams():
    rng = np.random.default_rng(7)
    parts = make(rng, 4, 128, 256, True)
    layer = parts[0]
    rows = (8, 60, 700)
    x = [frames(rng, 700, 128, "bf16") for _ in range(4)]
    picks = [tuple(torch.from_numpy(a).cuda() for a in choose(rng, 700, 4, 2)) for _ in range(4)]
    held = [(x[0][:r].clone(), picks[0][0][:r].clone(), picks[0][1][:r].clone()) for r in rows]
    layer.forward(*held[0])
    graphs, outs = [], []
    for t in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.forward(*t))
        graphs.append(g)
    for i in range(4):
        for r, t in zip(rows, held):
            for dst, src in zip(t, (x[i], *picks[i])):
                dst.copy_(src[:r])
        layer.forward(x[i], *picks[i])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for t, o in zip(held, outs):
            assert torch.equal(o, layer.forward(*t))
    want = [layer.forward(x[i], *picks[i]) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer.forward(x[i], *picks[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


@pytest.mark.parametrize("rows", [1, 14, 375])
def test_gate_routing_and_experts_as_a_half_step(rows):
    """The gate's logits, the choice and the experts' half step in a row, as a
    block's FeedForward sublayer uses them, in place."""
    rng = np.random.default_rng(8)
    e, d, f, k = 8, 256, 512, 2
    parts = make(rng, e, d, f, True)
    gate = M.Fp8Linear(d, e)
    gate.load(torch.from_numpy((rng.standard_normal((e, d)) / 16).astype(np.float32)))
    x, h = frames(rng, rows, d, "bf16"), frames(rng, rows, d, "bf16")
    bias = (0.1 * rng.standard_normal(e)).astype(np.float32)
    logits = gate.forward(h, out_dtype=torch.float32)
    if rows > 2:
        logits[-2:] = -float("inf")  # padding frames
    idx, w = M.route(logits, k, score="sigmoid", bias=torch.from_numpy(bias).cuda(), renormalize=True)
    codes, scales = gate.read_codes()
    want, mag = F.linear(host(h), codes, scales)
    live = rows - 2 if rows > 2 else rows
    assert (np.abs(host(logits) - want)[:live] <= (d + 64) * 2.0 ** -24 * mag[:live]).all()
    want_i, want_w = F.route(logits.cpu().numpy(), k, score="sigmoid", bias=bias, renormalize=True)
    assert np.array_equal(idx.cpu().numpy(), want_i) and np.allclose(w.cpu().numpy(), want_w, rtol=2.0 ** -23, atol=0)
    before = x.clone()
    parts[0].forward(h, idx, w, residual=x, res_scale=0.5, out=x)
    check(x, h, want_i, want_w, parts, before, 0.5)
    if rows > 2:
        assert torch.equal(x[-2:], before[-2:])
