"""Routing of frames to experts against the float64 oracle: indices equal,
weights within an f32 rounding (2^-24 relative) of a sum of 64-bit values."""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu


def check(logits, top_k, bias=None, **kw):
    idx, w = M.route(logits, top_k, bias=None if bias is None else torch.from_numpy(bias).cuda(), **kw)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32 and idx.shape == w.shape == (*logits.shape[:-1], top_k)
    want_i, want_w = F.route(logits.float().cpu().numpy().reshape(-1, logits.shape[-1]), top_k, bias=bias, **kw)
    assert np.array_equal(idx.cpu().numpy().reshape(-1, top_k), want_i)
    got = w.double().cpu().numpy().reshape(-1, top_k)
    assert (np.abs(got - want_w) <= 2.0 ** -24 * np.abs(want_w) * (1 + 1e-9) + 2.0 ** -149).all()
    return idx, w


CASES = [(1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (5, 8, 8, 1, 1), (7, 3, 2, 1, 1), (33, 60, 4, 1, 1), (64, 64, 6, 8, 3),
         (101, 65, 5, 1, 1), (40, 96, 8, 8, 2), (129, 128, 3, 2, 1), (50, 160, 6, 8, 3), (31, 256, 8, 8, 4), (9, 300, 32, 4, 4),
         (6, 512, 17, 64, 20), (12, 64, 8, 64, 8), (3, 257, 1, 1, 1)]


@pytest.mark.parametrize("rows,experts,top_k,groups,kept", CASES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_oracle(rows, experts, top_k, groups, kept, score, dtype):
    rng = np.random.default_rng(rows + experts)
    x = torch.from_numpy((2 * rng.standard_normal((rows, experts))).astype(np.float32)).to(dtype).cuda()
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    check(x, top_k, score=score, n_groups=groups, topk_groups=kept, renormalize=True, scale=2.5)
    check(x, top_k, bias=bias, score=score, n_groups=groups, topk_groups=kept, renormalize=rows % 2 == 0)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_ties_masks_and_extremes(score, groups, kept):
    rng = np.random.default_rng(5)
    x = rng.integers(-2, 3, (40, 64)).astype(np.float32)  # many ties
    x[1] = -np.inf  # nothing left
    x[2] = -np.inf
    x[2, 17] = 3.0  # one left
    x[3, ::2] = -np.inf
    x[4] = np.finfo(np.float32).min
    x[5, 10] = np.nan
    x[6] = np.nan
    x[7, 20], x[7, 40] = np.inf, np.inf
    x[8] = 0.0
    x[9, :32] = -np.inf
    x[10, 1:] = -1000.0
    x[11] = 1000.0
    x[12, 16:] = np.finfo(np.float32).min
    bias = np.zeros(64, np.float32)
    bias[::3] = 0.25
    hidden = bias.copy()
    hidden[5], hidden[33], hidden[34] = -np.inf, np.nan, np.inf
    for renorm in (False, True):
        for b in (None, bias, hidden):
            idx, w = check(torch.from_numpy(x).cuda(), 6, bias=b, score=score, n_groups=groups, topk_groups=kept, renormalize=renorm)
            assert (idx[1] == -1).all() and (w[1] == 0).all() and (idx[6] == -1).all()


ROWS_CASES = [(256, 8, 8, 4), (256, 8, 1, 1), (64, 4, 1, 1), (128, 6, 4, 2), (16, 2, 1, 1), (60, 4, 1, 1), (160, 6, 8, 3),
              (5, 3, 1, 1), (64, 16, 16, 8), (16, 3, 16, 5), (112, 9, 2, 1), (250, 16, 1, 1), (48, 17, 1, 1), (96, 4, 3, 2)]


@pytest.mark.parametrize("experts,top_k,groups,kept", ROWS_CASES)
@pytest.mark.parametrize("score,dtype", [("softmax", torch.float32), ("sigmoid", torch.bfloat16), ("sigmoid", torch.float32)])
def test_many_rows(experts, top_k, groups, kept, score, dtype):
    """6157 rows, at an odd distance: 300 of them and the last ones against the
    oracle, all against the same rows in smaller calls."""
    rng = np.random.default_rng(experts + top_k)
    wide = torch.from_numpy((2 * rng.standard_normal((6157, experts + 3))).astype(np.float32)).to(dtype).cuda()
    x = wide[:, 1:1 + experts]
    bias = (0.1 * rng.standard_normal(experts)).astype(np.float32)
    kw = dict(score=score, n_groups=groups, topk_groups=kept, renormalize=top_k % 2 == 0, scale=1.5)
    at = np.unique(np.concatenate([rng.integers(0, 6157, 300), np.arange(6130, 6157)]))
    for b in (None, bias):
        t = None if b is None else torch.from_numpy(b).cuda()
        idx, w = M.route(x, top_k, bias=t, **kw)
        want_i, want_w = F.route(x.float().cpu().numpy()[at], top_k, bias=b, **kw)
        assert np.array_equal(idx.cpu().numpy()[at], want_i)
        assert (np.abs(w.double().cpu().numpy()[at] - want_w) <= 2.0 ** -24 * np.abs(want_w) * (1 + 1e-9) + 2.0 ** -149).all()
        parts = [M.route(x[i:i + 2053], top_k, bias=t, **kw) for i in range(0, 6157, 2053)]
        assert torch.equal(idx, torch.cat([p[0] for p in parts]))
        # (sums of 64-bit scores in another order, so an f32 rounding may differ)
        assert ((w - torch.cat([p[1] for p in parts])).abs() <= 2.0 ** -23 * w.abs()).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2), (16, 7)])
def test_many_rows_with_ties_masks_and_extremes(score, groups, kept):
    rng = np.random.default_rng(6)
    x = rng.integers(-2, 3, (48, 64)).astype(np.float32)  # many ties
    x[1] = -np.inf
    x[2], x[2, 17] = -np.inf, 3.0
    x[3, ::2] = -np.inf
    x[4] = np.finfo(np.float32).min
    x[5, 10], x[6] = np.nan, np.nan
    x[7, 20], x[7, 40] = np.inf, np.inf
    x[8] = 0.0
    x[9, :32] = -np.inf
    x[10, 1:] = -1000.0
    x[11] = 1000.0
    x[12:16] = np.nextafter(np.float32(0.5), np.float32(1))  # next to 0.5: alike in f32, not in 64 bits
    x[12:16, 1::3] = 0.5
    hidden = np.zeros(64, np.float32)
    hidden[::3], hidden[5], hidden[33], hidden[34] = 0.25, -np.inf, np.nan, np.inf
    for b in (None, hidden):
        want_i, want_w = F.route(x, 4, bias=b, score=score, n_groups=groups, topk_groups=kept, renormalize=True)
        idx, w = M.route(torch.from_numpy(np.tile(x, (130, 1))).cuda(), 4, bias=None if b is None else torch.from_numpy(b).cuda(),
                         score=score, n_groups=groups, topk_groups=kept, renormalize=True)
        idx, w = idx.cpu().numpy().reshape(130, 48, 4), w.double().cpu().numpy().reshape(130, 48, 4)
        assert (idx == want_i).all()
        assert (np.abs(w - want_w) <= 2.0 ** -24 * np.abs(want_w) * (1 + 1e-9) + 2.0 ** -149).all()


def test_near_scores_are_told_apart():
    """Sigmoid scores whose difference f32 rounds away."""
    x = np.full((4, 16), 12.0, np.float32)
    for r in range(4):
        x[r, 3 + r] = np.nextafter(np.float32(12.0), np.float32(13.0))
    idx, _ = check(torch.from_numpy(x).cuda(), 2, score="sigmoid")
    assert idx[:, 0].tolist() == [3, 4, 5, 6]


def test_strided_rows_shapes_and_no_rows():
    rng = np.random.default_rng(7)
    wide = torch.from_numpy(rng.standard_normal((30, 50)).astype(np.float32)).cuda()
    a, b = M.route(wide[:, 5:45], 3), M.route(wide[:, 5:45].contiguous().view(2, 15, 40), 3)
    assert torch.equal(a[0], b[0].view(30, 3)) and torch.equal(a[1], b[1].view(30, 3))
    assert M.route(torch.empty(0, 8, device="cuda"), 2)[0].shape == (0, 2)
    with pytest.raises(M.MhsaError):
        M.route(wide, 3, bias=torch.zeros(49, device="cuda"))
    with pytest.raises(M.MhsaError):
        M.route(wide.T, 3)
    with pytest.raises(M.MhsaError):
        M.route(wide.half(), 3)


def test_refusals():
    x = torch.zeros(3, 8, device="cuda")
    for bad, kw in ((x[:, :0], {}), (x.double(), {}), (x.cpu(), {}), (x[0, 0], {}), (x, {"score": "tanh"}), (x, {"n_groups": 3}),
                    (x, {"bias": torch.zeros(7, device="cuda")}), (x, {"bias": torch.zeros(8)}), (x.T, {}), (x, {"scale": float("inf")})):
        with pytest.raises(M.MhsaError):
            M.route(bad, 2, **kw)
    for top_k in (0, -1, 9):
        with pytest.raises(M.MhsaError):
            M.route(x, top_k)


def test_replayed_graph():
    rng = np.random.default_rng(8)
    x = torch.from_numpy(rng.standard_normal((5, 77, 64)).astype(np.float32)).cuda()
    t = x[0].clone()
    M.route(t, 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        idx, w = M.route(t, 4, score="sigmoid", n_groups=4, topk_groups=2, renormalize=True)
    for i in range(5):
        t.copy_(x[i])
        g.replay()
        torch.cuda.synchronize()
        a, b = M.route(x[i], 4, score="sigmoid", n_groups=4, topk_groups=2, renormalize=True)
        assert torch.equal(a, idx) and torch.equal(b, w)
