"""The experts' FeedForward on f32 activations: exact products and f32 sums in
both matrix products, at the sizes of every kernel that a call can take.

Tolerances. Where all sums are whole numbers of a power of two and their partial
sums stay under 2^24 of it, an f32 sum in any order is exact, and results are
compared bit for bit. The fp8 matrix unit would not give them: beside a product
of 448 * 448 it drops what lies under 2^4 of the products that it adds with it.
Elsewhere a sum of K products is off by at most K + 64 steps of 2^-24 of their
magnitudes; the oracle carries that to the codes that a hidden value may take.
"""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu

# rows, experts, d_model, ff_dim, top_k: up to 16 pairs; up to 256 of up to 64
# experts and of more; up to 1024; a list of 16 pairs each; of 128; of 256 with
# 128 and with 256 columns of the second product; and in several tiles a workgroup
SIZES = [(1, 2, 128, 256, 2), (7, 3, 192, 320, 2), (16, 4, 256, 64, 1), (60, 5, 192, 192, 2), (100, 80, 128, 128, 2),
         (450, 64, 128, 192, 2), (1100, 70, 128, 128, 2), (333, 4, 256, 512, 2), (1500, 3, 320, 192, 1), (4100, 3, 1280, 192, 3),
         (9000, 2, 192, 1088, 3)]


def load(codes1, scales1, codes2, scales2, b1=None, b2=None):
    e, f, d = codes1.shape
    layer = M.ExpertFeedForward(e, d, f, b1 is not None)
    layer.load_codes(codes1, scales1, codes2, scales2, b1, b2)
    return layer


def code_of(v):
    return F.encode(np.asarray(v, np.float64))


def flat(e, n, k, byte=127):
    return np.full((e, -(-n // 128), -(-k // 128)), byte, np.uint8)


def choices(rng, rows, e, k):
    idx = np.stack([rng.permutation(e)[:k] if k <= e else rng.integers(0, e, k) for _ in range(rows)]).astype(np.int32)
    if rows > 2:
        idx[rows // 2, 0] = -1
        idx[rows // 3, -1] = e
    return idx


@pytest.mark.parametrize("rows,e,d,f,k", SIZES)
def test_second_product_is_exact(rows, e, d, f, k):
    """Hidden values from the bias alone (silu(v) = v in f32 from 20 on), two of
    them 448 with weights of 448 and -448, so that what is left is the small
    products' sum."""
    rng = np.random.default_rng(rows + f)
    h = rng.choice([20.0, 22.0, 24.0, 28.0, 32.0], (e, f))
    w2 = rng.choice([-0.5, -0.25, 0.25, 0.5], (e, d, f))
    for x in range(e):
        for i, j in rng.permutation(f)[:4].reshape(2, 2):
            h[x, i] = h[x, j] = 448.0
            w2[x, :, i], w2[x, :, j] = 448.0, -448.0
    b2 = rng.integers(-8, 9, (e, d)).astype(np.float32)
    layer = load(np.zeros((e, f, d), np.uint8), flat(e, f, d), code_of(w2), flat(e, d, f), h.astype(np.float32), b2)
    y = np.einsum("edf,ef->ed", w2, h) + b2
    idx, w = choices(rng, rows, e, k), rng.choice([0.5, 1.0, 2.0], (rows, k)).astype(np.float32)
    r = rng.integers(-64, 65, (rows, d)).astype(np.float32)
    there = (idx >= 0) & (idx < e)
    want = r + 0.5 * (np.where(there, w, 0.0)[..., None] * y[np.where(there, idx, 0)]).sum(1)
    x = torch.from_numpy(rng.standard_normal((rows, d)).astype(np.float32)).cuda()
    got = layer.forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda(), residual=torch.from_numpy(r).cuda(),
                        res_scale=0.5).cpu().numpy()
    bad = got != want
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), np.abs(got - want).max())


def hidden_codes(h, steps):
    """The least and the largest values that the codes of silu(h) may stand for
    when silu is off by `steps` of 2^-24, and the blocks whose power is certain."""
    v = F.silu(h)
    lo, hi, sure = np.empty_like(v), np.empty_like(v), np.empty(v.shape, bool)
    for c in range(0, v.shape[1], 128):
        b = v[:, c:c + 128]
        err = steps * 2.0 ** -24 * np.abs(b)
        s = [F.scale_byte((np.abs(b) + i * err).max(1, initial=0))[:, None] - 127 for i in (-1, 1)]
        sure[:, c:c + 128] = s[0] == s[1]
        lo[:, c:c + 128], hi[:, c:c + 128] = (
            np.ldexp(F.VALUES[F.encode(np.clip(np.ldexp(b + i * err, -s[0]), -448, 448))], s[0]) for i in (-1, 1))
    return lo, hi, sure


@pytest.mark.parametrize("rows,e,f", [(1, 2, 128), (11, 3, 192), (200, 4, 320), (700, 64, 128), (1100, 70, 192), (500, 6, 192),
                                      (1500, 3, 320), (4000, 2, 1280)])
def test_first_product_is_exact(rows, e, f):
    """A second matrix of the identity returns the hidden values' codes; silu is
    off by at most 8 steps."""
    rng = np.random.default_rng(rows + f)
    x, w1 = rng.integers(-4, 5, (rows, f)).astype(np.float64), rng.integers(-4, 5, (e, f, f)).astype(np.float64)
    for i, j in rng.permutation(f)[:6].reshape(3, 2):
        x[:, i] = x[:, j] = 448.0
        w1[:, :, i], w1[:, :, j] = 448.0, -448.0
    one = np.zeros((e, f, f), np.uint8)
    one[:, np.arange(f), np.arange(f)] = 0x38
    layer = load(code_of(w1), flat(e, f, f, 121), one, flat(e, f, f))
    idx = rng.integers(0, e, (rows, 1)).astype(np.int32)
    got = layer.forward(torch.from_numpy(x.astype(np.float32)).cuda(), torch.from_numpy(idx).cuda(),
                        torch.ones(rows, 1, device="cuda")).double().cpu().numpy()
    for k in range(e):
        at = idx[:, 0] == k
        lo, hi, sure = hidden_codes(x[at] @ w1[k].T / 64, 8)
        bad = ~((lo <= got[at]) & (got[at] <= hi)) & sure
        assert not bad.any(), (k, int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("rows,e,d,f,k", SIZES[:-2] + [(4100, 3, 640, 192, 3), (2500, 2, 192, 640, 3)])
def test_against_oracle(rows, e, d, f, k):
    rng = np.random.default_rng(rows + d)
    lin1 = [F.quantize_weight(rng.standard_normal((f, d)) / np.sqrt(d)) for _ in range(e)]
    lin2 = [F.quantize_weight(rng.standard_normal((d, f)) / np.sqrt(f)) for _ in range(e)]
    layer = load(*(np.stack([m[i] for m in lin]) for lin in (lin1, lin2) for i in (0, 1)))
    x = torch.from_numpy((rng.standard_normal((rows, d)) * np.exp(0.5 * rng.standard_normal(d))).astype(np.float32)).cuda()
    idx, w = choices(rng, rows, e, k), rng.uniform(0.05, 1.0, (rows, k)).astype(np.float32)
    got = layer.forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()).double().cpu().numpy()
    step = (max(d, f) + 64) * 2.0 ** -24
    want, bound = F.experts(x.double().cpu().numpy(), idx, w, lin1, lin2, sum_err=step)
    tol = bound + 64 * 2.0 ** -24 * (np.abs(want) + bound / step)
    bad = np.abs(got - want) > tol + 1e-30
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("rows", [5, 300, 3000])
def test_infinities_and_nans_stay_in_their_rows(rows):
    rng = np.random.default_rng(rows)
    lin = [[F.quantize_weight(rng.standard_normal(s) / 12) for _ in range(2)] for s in ((192, 256), (256, 192))]
    layer = load(*(np.stack([m[i] for m in part]) for part in lin for i in (0, 1)))
    x = torch.from_numpy(rng.standard_normal((rows, 256)).astype(np.float32)).cuda()
    idx = torch.from_numpy(rng.integers(0, 2, (rows, 1)).astype(np.int32)).cuda()
    w = torch.ones(rows, 1, device="cuda")
    clean = layer.forward(x, idx, w)
    x[1, 200], x[3, 5] = float("nan"), float("inf")
    got = layer.forward(x, idx, w)
    keep = [r for r in range(rows) if r not in (1, 3)]
    assert torch.isnan(got[[1, 3]]).all() and torch.equal(got[keep], clean[keep])
