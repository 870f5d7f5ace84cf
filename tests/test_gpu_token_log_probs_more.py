"""Log probabilities of many tokens a row, at temperatures whose reciprocal is no
f32, over logits of the type's lowest value, and of more rows than one launch
takes.

Tolerances, in steps of 2^-24, as in test_gpu_token_log_probs but against the
definition, softmax(logits / temperature) for the f32 temperature: d is off by 5
of itself (the difference, log2 e, 1 / T, their product, the product), e^d by
those and 2; log S by V / 64 + 66 + 5 E|d| + 2 |log S|, a log probability by that,
5 |d| and 4 of itself, and the entropy by the sums' steps of 1 + 2 E|d| + |log S|
and, by e^d's errors, 10 E d^2.
"""
import numpy as np
import pytest
import torch

import relpos_mhsa as M

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
STEP = 2.0 ** -24


def oracle(x, temperature):
    """Log probabilities [rows, V] in 64 bits, entropy, and (E|d|, E d^2, log S)."""
    d = (x - x.max(-1, keepdims=True)) / np.float64(np.float32(temperature))
    e = np.exp(d)
    s = e.sum(-1, keepdims=True)
    p, ls = e / s, np.log(s)
    on = np.where(p > 0, d, 0.0)
    return d - ls, (ls[:, 0] - (p * on).sum(-1)), ((p * -on).sum(-1), (p * on * on).sum(-1), ls[:, 0])


def close(got, want, tol):
    with np.errstate(over="ignore"):
        f = want.astype(np.float32)  # what no f32 holds is -inf
    got = got.double().cpu().numpy()
    far = np.isinf(f)
    assert np.array_equal(got[far], f[far].astype(np.float64))
    bad = ~(np.abs(got - want) <= tol)[~far]
    assert not bad.any(), (int(bad.sum()), got[~far][bad][:4], want[~far][bad][:4])


def check(x, tokens, temperature, top_k):
    got = M.token_log_probs(x, torch.from_numpy(tokens).cuda(), top_k, temperature)
    f64 = x.double().cpu().numpy()
    lp, h, (m1, m2, ls) = oracle(f64, temperature)
    n = x.shape[1] / 64 + 66
    base = (n + 5 * m1 + 2 * ls)[:, None]

    def tol(want):
        size = np.where(np.abs(want) < 3.5e38, np.abs(want), 0.0)
        return STEP * (base + 5 * (size + ls[:, None]) + 4 * size)
    there = (tokens >= 0) & (tokens < x.shape[1])
    want = np.where(there, np.take_along_axis(lp, np.where(there, tokens, 0), 1), 0.0)
    assert (got.log_probs.cpu().numpy()[~there] == 0).all()
    close(got.log_probs, want, tol(want))
    close(got.entropy, h, STEP * (n * (1 + 2 * m1 + ls) + 10 * m2))
    if top_k:
        order = np.argsort(-f64, axis=-1, kind="stable")[:, :top_k]
        assert np.array_equal(got.top_indices.cpu().numpy(), order)
        want = np.take_along_axis(lp, order, 1)
        close(got.top_log_probs, want, tol(want))


@pytest.mark.parametrize("rows,v", [(5, 300), (9, 1025), (3, 9000), (2, 60000)])  # a wave, several, parts that are joined
@pytest.mark.parametrize("n", [63, 64, 65, 130, 1024])
def test_many_tokens(rows, v, n):
    rng = np.random.default_rng(v + n)
    x = torch.from_numpy(3 * rng.standard_normal((rows, v))).float().cuda()
    tokens = rng.integers(-2, v + 2, (rows, n)).astype(np.int32)
    tokens[:, -1], tokens[0, n // 2:] = v - 1, -1
    tokens[1, -2] = v
    check(x, tokens, 1.0, 3)


@pytest.mark.parametrize("rows,v", [(7, 5), (9, 1025), (3, 9000), (2, 60000)])
@pytest.mark.parametrize("temperature", [0.01, 0.07, 0.7, 1.3, 3.0, 100.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_temperatures(rows, v, temperature, dtype):
    rng = np.random.default_rng(v)
    x = torch.from_numpy(rng.standard_normal((rows, v)) * (0.2 + 3 * rng.random((rows, 1)))).to(DTYPES[dtype]).cuda()
    check(x, rng.integers(-1, v, (rows, 4)).astype(np.int32), temperature, 4)


@pytest.mark.parametrize("v", [40, 1025, 9000, 60000])
@pytest.mark.parametrize("temperature", [0.01, 0.5, 0.999, 1.0, 2.0])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_lowest_values_as_masks(v, temperature, dtype):
    """A finite logit whose distance over the temperature is no f32 has log p
    -inf; it takes no part in the sums, and no NaN comes of it."""
    rng = np.random.default_rng(v)
    low = float(torch.finfo(DTYPES[dtype]).min)
    x = rng.standard_normal((6, v))
    x[0, rng.random(v) < 0.9] = low
    x[0, 0] = 0.5
    x[1] = low                       # all alike
    x[2, 1:] = low                   # one left
    x[3, :v - 1] = low
    x[4] = low
    x[4, [2, v // 2]] = 0.1 * low    # far above the others, and below what is ordinary
    x[5, ::2] = low
    t = torch.from_numpy(x).to(DTYPES[dtype]).cuda()
    tokens = np.stack([np.full(6, 0), np.full(6, 1), np.full(6, v - 1), np.full(6, v // 2), np.full(6, -1)], 1).astype(np.int32)
    for k in (0, 3, 20):
        check(t, tokens, temperature, k)


def test_rows_past_a_launch():
    """More than 2^22 rows of a vocabulary that two waves take."""
    rows, v, cut = (1 << 22) + 300, 4100, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, v, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    tokens = torch.randint(-1, v, (rows, 2), device="cuda", generator=g, dtype=torch.int32)
    at = torch.cat([torch.arange(lo, hi, device="cuda") for lo, hi in ((0, 99), (cut - 99, cut + 99), (rows - 99, rows))]
                   + [torch.randint(0, rows, (500,), device="cuda", generator=g)]).unique()
    got, want = M.token_log_probs(x, tokens, 3), M.token_log_probs(x[at], tokens[at], 3)
    for a, b in zip(got, want):
        assert torch.equal(a[at], b)
    del x, got
    torch.cuda.empty_cache()
