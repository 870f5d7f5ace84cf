"""Every result of the experts' tiles, in both dtypes.

Whole numbers: activations and first weights of up to 8 have products that the
fp8 matrix unit adds exactly, so a hidden value is silu of a known number, off by
at most 8 steps of 2^-24, and its code is one of one or two. A second matrix with
a single 1 or -1 in each row returns it. A frame's sum of two and its store round
by at most half a step of the dtype.

Ordinary numbers: at most 1% of a frame's hidden values, each by a step of 2^-3 at
most, take a code beside their own, 1.25e-2 of their 2-norm; the second matrix
spreads that over all columns, so that 16 of them have 8 times their share in
none of the runs. One wrong run is off by its whole share.
"""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}

# pairs of each expert, d_model, ff_dim, top_k: lists of 16 pairs, tiles of 128 (by
# the mean, and because one block of inputs does not fill the large ones' ring), of
# 256 with 128 columns in the second product and with 256, several to a workgroup
COUNTS = {
    "16": ([1, 15, 16, 17, 31, 0, 8] * 15, 128, 192, 1),
    "128": ([129, 143, 128, 64, 1, 0, 257, 255], 192, 320, 1),
    "128 twice": ([129, 143, 128, 64, 2, 0, 257, 255], 256, 64, 2),
    "one block": ([257, 271, 500], 128, 320, 1),
    "256 x 128": ([257, 271, 511, 513], 192, 320, 1),
    "256 x 128 twice": ([257, 271, 511, 513], 320, 192, 2),
    "256 x 256": ([6001, 5121, 271, 0, 5007], 1280, 192, 1),
    "many hidden": ([6001, 5121, 271, 0, 5007], 192, 1280, 1),
}


def pairs_of(rng, counts, k):
    return rng.permutation(np.repeat(np.arange(len(counts)), counts)).astype(np.int32).reshape(-1, k)


def frames(a, dtype):
    return torch.from_numpy(np.asarray(a, np.float32)).to(DTYPES[dtype]).cuda()


def layer_of(w1, s1, w2, s2):
    e, f, d = w1.shape
    layer = M.ExpertFeedForward(e, d, f)
    layer.load_codes(w1, s1, w2, s2)
    return layer


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_whole_numbers(name, dtype):
    counts, d, f, k = COUNTS[name]
    rng = np.random.default_rng(len(name) + d)
    e, idx = len(counts), pairs_of(rng, counts, k)
    rows = len(idx)
    x, w1 = rng.integers(-8, 9, (rows, d)).astype(np.float64), rng.integers(-8, 9, (e, f, d)).astype(np.float64)
    s1 = rng.integers(117, 122, (e, -(-f // 128), -(-d // 128))).astype(np.uint8)
    s1[:] = s1[:, :, :1]  # (sums stay whole numbers of one power of two)
    pick, sign = rng.integers(0, f, (e, d)), rng.choice([-1.0, 1.0], (e, d))
    w2 = np.zeros((e, d, f))
    w2[np.arange(e)[:, None], np.arange(d), pick] = sign
    layer = layer_of(F.encode(w1), s1, F.encode(w2), np.full((e, -(-d // 128), -(-f // 128)), 127, np.uint8))
    w = rng.choice([0.5, 1.0, -2.0], (rows, k)).astype(np.float32)
    got = layer.forward(frames(x, dtype), torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()).double().cpu().numpy()
    low, high, sure = np.zeros((rows, d)), np.zeros((rows, d)), np.ones((rows, d), bool)
    for j in range(k):
        for c in range(e):
            at = np.nonzero(idx[:, j] == c)[0]
            power = np.repeat(np.ldexp(1.0, s1[c, :, 0].astype(int) - 127), 128)[:f]
            v = F.silu((x[at] @ w1[c].T) * power)
            lo, hi, ok = np.empty_like(v), np.empty_like(v), np.empty(v.shape, bool)
            for b in range(0, f, 128):
                t = v[:, b:b + 128]
                err = 8 * 2.0 ** -24 * np.abs(t)
                s = [F.scale_byte((np.abs(t) + i * err).max(1, initial=0))[:, None] - 127 for i in (-1, 1)]
                ok[:, b:b + 128] = s[0] == s[1]  # (a largest value next to a power's edge may take either)
                lo[:, b:b + 128], hi[:, b:b + 128] = (
                    np.ldexp(F.VALUES[F.encode(np.clip(np.ldexp(t + i * err, -s[0]), -448, 448))], s[0]) for i in (-1, 1))
            times = w[at, j][:, None].astype(np.float64) * sign[c]
            a, b = times * lo[:, pick[c]], times * hi[:, pick[c]]
            low[at] += np.minimum(a, b)
            high[at] += np.maximum(a, b)
            sure[at] &= ok[:, pick[c]]
    half = torch.finfo(DTYPES[dtype]).eps / 2 * np.maximum(np.abs(low), np.abs(high)) * (k > 1)
    bad = ~((low - half <= got) & (got <= high + half)) & sure
    assert sure.mean() > 0.9 and (low == high).mean() > 0.9
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("name", COUNTS)
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_runs_of_columns(name, dtype):
    counts, d, f, k = COUNTS[name]
    rng = np.random.default_rng(len(name) + f)
    e, idx = len(counts), pairs_of(rng, counts, k)
    rows = len(idx)
    lin1 = [F.quantize_weight(rng.standard_normal((f, d)) / np.sqrt(d)) for _ in range(e)]
    lin2 = [F.quantize_weight(rng.standard_normal((d, f)) / np.sqrt(f)) for _ in range(e)]
    layer = layer_of(*(np.stack([m[i] for m in lin]) for lin in (lin1, lin2) for i in (0, 1)))
    x, w = frames(rng.standard_normal((rows, d)), dtype), rng.uniform(0.5, 1.0, (rows, k)).astype(np.float32)
    got = layer.forward(x, torch.from_numpy(idx).cuda(), torch.from_numpy(w).cuda()).double().cpu().numpy()
    want, _ = F.experts(x.double().cpu().numpy(), idx, w, lin1, lin2)
    runs = (rows, d // 16, 16)
    share = np.linalg.norm(want, axis=1)[:, None] * np.sqrt(16 / d)
    off = np.linalg.norm((got - want).reshape(runs), axis=2)
    tol = 0.1 * share + torch.finfo(DTYPES[dtype]).eps / 2 * np.linalg.norm(want.reshape(runs), axis=2)
    bad = ~(off <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), (off / share).max())
