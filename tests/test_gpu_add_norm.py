"""A residual's addition with its norm against the float64 oracle.

Tolerances, in steps of 2^-24 (half of f32's): v one; sums of squares or values
of a row, held by the lanes of up to 16 waves, go through at most 32 additions
in a lane, 6 in a wave and 16 between waves, and all squares are positive; the
mean's error is relative to the values' mean magnitude; the root halves the
sum's and adds two; three more products and a sum. 96 steps of what enters
cover these. bf16 results round by half a step more, 2^-8 of the value.
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


def f64(t):
    return t.double().cpu().numpy()


def near(got, want, tol):
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * np.abs(want)
    got = f64(got)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    bad = np.abs(got - want) > tol + 1e-37
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


def check_codes(rows, y):
    """rows: Fp8Rows of y (f32 as the kernel has it), to the bit."""
    d = y.shape[-1]
    kb = -(-d // 128)
    codes, scales = rows.codes.cpu().numpy(), rows.scales.cpu().numpy()
    assert codes.shape == (y.shape[0], kb * 128) and scales.shape == (y.shape[0], -(-kb // 4) * 4)
    assert (codes[:, d:] == 0).all() and (scales[:, kb:] == 127).all()
    for j in range(kb):
        b = y[:, 128 * j:128 * (j + 1)]
        s = F.scale_byte(F._finite_max(b, 1))
        assert np.array_equal(scales[:, j], s)
        want = F.VALUES[F.encode(np.ldexp(b, 127 - s[:, None]))]
        assert np.array_equal(F.VALUES[codes[:, 128 * j:128 * j + b.shape[1]]], want, equal_nan=True)


WIDTHS = [1, 7, 8, 64, 100, 128, 129, 500, 512, 513, 1000, 1024, 1025, 2048, 2056, 4096, 4100, 8192, 8200, 16385, 32768]


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("dtype,kind", [("f32", "rms"), ("f32", "layer"), ("bf16", "rms"), ("bf16", "layer")])
@pytest.mark.parametrize("rows", [1, 6, 37])
def test_against_oracle(rows, d, dtype, kind):
    rng = np.random.default_rng(d + rows)
    x = tensor(rng.standard_normal((rows, d)) * np.exp(rng.standard_normal((rows, 1))) + 0.3, dtype)
    delta = tensor(rng.standard_normal((rows, d)), dtype)
    w, b = tensor(np.exp(0.3 * rng.standard_normal(d)), "f32"), tensor(0.2 * rng.standard_normal(d), "f32")
    before = x.clone(), delta.clone()
    got = M.add_norm(x, delta, w, b, kind=kind, scale=0.3, want="both", out_dtype=torch.float32)
    y, v, size = R.norm(f64(x), f64(delta), 0.3, f64(w), f64(b), kind)
    assert got.sum.dtype == x.dtype and got.out.dtype == torch.float32
    near(got.out, y, 96 * STEP * size)
    near(got.sum, v, STEP * np.abs(v))
    check_codes(got.codes, f64(got.out))
    assert torch.equal(x, before[0]) and torch.equal(delta, before[1])
    plain = M.add_norm(x, kind=kind, out_dtype=torch.bfloat16, eps=0.5)
    y, _, size = R.norm(f64(x), kind=kind, eps=0.5)
    assert plain.sum is None and plain.codes is None
    near(plain.out, y, 96 * STEP * size)
    only = M.add_norm(x, delta, w, b, kind=kind, scale=0.3, want="codes")
    assert torch.equal(only.codes.codes, got.codes.codes) and torch.equal(only.codes.scales, got.codes.scales)
    assert torch.equal(only.sum, got.sum)


@pytest.mark.parametrize("rows,d", [(70000, 64), (40000, 520), (9000, 2100)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(rows, d, dtype):
    """More rows than a launch has workgroups: each row as in a call of its own."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, d, device="cuda", generator=g).to(DTYPES[dtype])
    delta = torch.randn(rows, d, device="cuda", generator=g).to(DTYPES[dtype])
    w = torch.rand(d, device="cuda", generator=g)
    got = M.add_norm(x, delta, w, kind="layer", want="both")
    at = torch.cat([torch.arange(0, rows, 997), torch.arange(rows - 70, rows)])
    one = M.add_norm(x[at], delta[at], w, kind="layer", want="both")
    assert torch.equal(got.out[at], one.out) and torch.equal(got.sum[at], one.sum)
    assert torch.equal(got.codes.codes[at], one.codes.codes) and torch.equal(got.codes.scales[at], one.codes.scales)
    y, _, size = R.norm(f64(x[at]), f64(delta[at]), 1.0, f64(w), None, "layer")
    near(one.out, y, 96 * STEP * size)


@pytest.mark.parametrize("d", [96, 1000, 3000, 9001])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_in_place(d, dtype):
    """Rows within a wider buffer, at odd addresses; sums and results over their
    inputs; what lies beside them stays."""
    rng = np.random.default_rng(d)
    rows = 11
    buf = tensor(rng.standard_normal((rows, 3 * d + 7)), dtype)
    before = buf.clone()
    x, delta, y = buf[:, 1:1 + d], buf[:, d + 2:2 * d + 2], buf[:, 2 * d + 5:3 * d + 5]
    want = M.add_norm(x.contiguous(), delta.contiguous(), want="both")
    got = M.add_norm(x, delta, out=y, sum_out=x, want="both")
    assert torch.equal(x, want.sum) and torch.equal(y, want.out) and torch.equal(got.codes.codes, want.codes.codes)
    x.copy_(before[:, 1:1 + d])
    y.copy_(before[:, 2 * d + 5:3 * d + 5])
    assert torch.equal(buf, before)
    M.add_norm(x, delta, out=x, sum_out=delta)  # both over their inputs
    assert torch.equal(x, want.out) and torch.equal(delta, want.sum)
    lead = before[:, 1:1 + d].contiguous().view(1, rows, 1, d)
    got = M.add_norm(lead, want="both")
    assert got.out.shape == lead.shape and got.codes.shape == lead.shape
    copy = torch.empty_like(lead)
    assert M.add_norm(lead, sum_out=copy).sum is copy and torch.equal(copy, lead)


@pytest.mark.parametrize("d", [100, 2500])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_values_at_the_ends(d, kind):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, d))
    x[0] = 0.0
    x[1, 3], x[2, d - 1], x[3, 0] = np.nan, np.inf, -np.inf
    x[4] *= 1e-30
    x[5] *= 1e15
    x[6] = 2.5
    w = np.ones(d)
    w[5] = 0.0
    t, tw = tensor(x, "f32"), tensor(w, "f32")
    got = M.add_norm(t, weight=tw, kind=kind, want="both")
    y, _, size = R.norm(f64(t), weight=f64(tw), kind=kind)
    assert torch.isnan(got.out[1]).all()
    fine = [0, 4, 5, 6, 7, 8]
    near(got.out[fine], y[fine], 96 * STEP * size[fine])
    assert torch.isnan(got.out[2:4]).any(1).all()  # infinity over infinity (rms: and zeros beside it)
    check_codes(got.codes, f64(got.out))


def test_no_rows_and_no_kept_state():
    x = torch.empty(0, 64, device="cuda")
    got = M.add_norm(x, x.clone(), want="both")
    assert got.out.shape == (0, 64) and got.codes.codes.shape == (0, 128) and got.sum.shape == (0, 64)


def test_streams_and_graphs():
    """On another stream and captured: replays with other inputs give what
    eager calls give."""
    x, delta = torch.randn(300, 1024, device="cuda"), torch.randn(300, 1024, device="cuda")
    w = torch.rand(1024, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        M.add_norm(x, delta, w, want="both")
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = M.add_norm(x, delta, w, want="both")
    for i in range(4):
        x.copy_(torch.randn(300, 1024, device="cuda") * (i + 1))
        graph.replay()
        want = M.add_norm(x, delta, w, want="both")
        torch.cuda.synchronize()
        assert torch.equal(held.out, want.out) and torch.equal(held.sum, want.sum)
        assert torch.equal(held.codes.codes, want.codes.codes) and torch.equal(held.codes.scales, want.codes.scales)


def test_refusals():
    x = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    buf = torch.zeros(5, 64, device="cuda")
    for bad in (lambda: M.add_norm(x.cpu()), lambda: M.add_norm(x.half()), lambda: M.add_norm(None), lambda: M.add_norm(x, x.bfloat16()),
                lambda: M.add_norm(x, x[:3]), lambda: M.add_norm(x, weight=w[:63]), lambda: M.add_norm(x, weight=w.bfloat16()),
                lambda: M.add_norm(x, bias=w.cpu()), lambda: M.add_norm(x, kind="batch"), lambda: M.add_norm(x, want="all"),
                lambda: M.add_norm(x, eps=-1.0), lambda: M.add_norm(x, eps=float("nan")), lambda: M.add_norm(x, x, scale=float("inf")),
                lambda: M.add_norm(x, want="codes", out=x), lambda: M.add_norm(x.t()), lambda: M.add_norm(x, out=x[:2]),
                lambda: M.add_norm(x, out=x, out_dtype=torch.bfloat16), lambda: M.add_norm(torch.zeros(2, 32769, device="cuda")),
                lambda: M.add_norm(x, x.clone(), sum_out=x, out=x), lambda: M.add_norm(buf[1:], out=buf[:4]),
                lambda: M.add_norm(buf[1:], buf[:4], sum_out=buf[1:], out=buf[:4], weight=buf[0]),
                lambda: M.add_norm(torch.zeros(3, 0, device="cuda"))):
        with pytest.raises(M.MhsaError):
            bad()
