"""The 8-bit block-scaled projection against the float64 oracle.

Tolerances. f32 out: products of two codes are exact in f32 and a sum of K of
them in any order is off by at most K steps of 2^-24 of the sum of their
magnitudes, the split sums, bias and store a few more. bf16 out: the fp8 matrix
unit adds products in groups of 8 and drops, of each but the largest, less than
2^-13 of the largest's power of two, so at most 7 * 2^-13 of the magnitudes'
sum; the store rounds by at most 2^-8 of the value.
"""
import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def make(rng, rows, k, n, bias=True, spread=0):
    x = rng.standard_normal((rows, k)) * np.exp(0.5 * rng.standard_normal(k))
    x *= 2.0 ** rng.integers(-spread, spread + 1, (rows, 1)) if spread else 1.0
    w = rng.standard_normal((n, k)) / np.sqrt(k)
    codes, scales = F.quantize_weight(w)
    return x, codes, scales, (0.1 * rng.standard_normal(n)).astype(np.float32) if bias else None


def on_gpu(x, dtype):
    return torch.from_numpy(np.asarray(x, np.float32)).to(DTYPES[dtype]).cuda()


def layer_of(k, n, codes, scales, bias):
    layer = M.Fp8Linear(k, n, bias is not None)
    layer.load_codes(codes, scales, bias)
    return layer


def check(got, x, codes, scales, bias, k):
    want, mag = F.linear(x.float().cpu().double().numpy(), codes, scales, bias)
    if bias is not None:
        mag = mag + np.abs(bias)
    tol = (k + 64) * 2.0 ** -24 * mag
    if got.dtype == torch.bfloat16:
        tol = tol + 7 * 2.0 ** -13 * mag + 2.0 ** -8 * np.abs(want)
    got = got.float().cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    bad = np.abs(got - want) > tol + 1e-38
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist(), np.nanmax(np.abs(got - want) / (mag + 1e-300)))


SHAPES = [(1, 1, 1), (1, 128, 16), (1, 100, 3), (2, 1024, 4096), (3, 5, 33), (16, 129, 130), (17, 256, 15), (33, 4096, 64),
          (64, 640, 1025), (65, 640, 1025), (66, 1, 1), (70, 127, 65), (113, 512, 2048), (300, 1000, 333), (257, 384, 256),
          (128, 2176, 128), (700, 513, 640), (1500, 256, 1100), (4100, 128, 2049)]


@pytest.mark.parametrize("rows,k,n", SHAPES)
@pytest.mark.parametrize("xd,yd", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
def test_against_oracle(rows, k, n, xd, yd):
    rng = np.random.default_rng(rows * 7 + k * 3 + n)
    x, codes, scales, bias = make(rng, rows, k, n, bias=(rows + k) % 2 == 0, spread=12)
    x = on_gpu(x, xd)
    got = layer_of(k, n, codes, scales, bias).forward(x, out_dtype=DTYPES[yd])
    assert got.shape == (rows, n) and got.dtype == DTYPES[yd]
    check(got, x, codes, scales, bias, k)


@pytest.mark.parametrize("rows,k,n", [(16300, 300, 2040), (9001, 129, 2304), (9001, 520, 2300), (6200, 700, 1800)])
@pytest.mark.parametrize("yd", ["bf16", "f32"])
def test_many_large_tiles(rows, k, n, yd):
    """Several tiles to a workgroup, of 256 and of 192 rows, with two stages and
    more: sampled rows, and the last ones."""
    rng = np.random.default_rng(rows + k)
    x, codes, scales, bias = make(rng, rows, k, n, spread=6)
    x = on_gpu(x, "bf16")
    got = layer_of(k, n, codes, scales, bias).forward(x, out_dtype=DTYPES[yd])
    at = np.unique(np.concatenate([rng.integers(0, rows, 400), np.arange(rows - 300, rows)]))
    check(got[at], x[at], codes, scales, bias, k)


@pytest.mark.parametrize("rows", [5, 200])
@pytest.mark.parametrize("xd", ["bf16", "f32"])
def test_activations_round_as_the_format_says(rows, xd):
    """Weights of the identity return the rounded activations, to the bit: rows
    of any magnitude, zeros, subnormals, steps halfway between codes."""
    rng = np.random.default_rng(3)
    k = 300
    x = rng.standard_normal((rows, k)) * 2.0 ** rng.integers(-130, 100, (rows, 1))
    x[0] = 0.0
    x[1] = 448.0
    x[1, ::2] = (F.POSITIVE[np.arange(150) % 126] + F.POSITIVE[np.arange(150) % 126 + 1]) / 2
    x[2, 128:256] = 2.0 ** -140
    x[3, 7] = 448.0 * 2.0 ** 3  # sets the scale, exactly at its edge
    x[4, 7] = 452.0 * 2.0 ** 3
    x = on_gpu(x, xd)
    codes = np.zeros((k, k), np.uint8)
    codes[np.arange(k), np.arange(k)] = 0x38
    layer = layer_of(k, k, codes, np.full((3, 3), 127, np.uint8), None)
    got = layer.forward(x, out_dtype=torch.float32).cpu().numpy()
    want = F.round_rows(x.double().cpu().numpy())
    # (the matrix cores may flush results under the smallest normal f32)
    assert np.array_equal(np.where(np.abs(want) < 2.0 ** -126, 0, got), np.where(np.abs(want) < 2.0 ** -126, 0, want))
    # (a bf16 out: the same values, exact in bf16)
    got = layer.forward(x, out_dtype=torch.bfloat16).double().cpu().numpy()
    assert np.array_equal(np.where(np.abs(want) < 2.0 ** -126, 0, got), np.where(np.abs(want) < 2.0 ** -126, 0, want))


@pytest.mark.parametrize("rows", [5, 300, 3000])
@pytest.mark.parametrize("yd", ["bf16", "f32"])
def test_tiny_rows_and_large_weights(rows, yd):
    """Rows about 2^-126 on weights about 2^40: an operand may lose what lies
    below 2^-133, so each product 2^-133 of the other's magnitude."""
    rng = np.random.default_rng(12)
    k, n = 520, 300
    x, codes, scales, _ = make(rng, rows, k, n, bias=False)
    x, scales = on_gpu(x * 2.0 ** -126, "f32"), scales + 40
    got = layer_of(k, n, codes, scales, None).forward(x, out_dtype=DTYPES[yd])
    want, mag = F.linear(x.double().cpu().numpy(), codes, scales)
    w = np.abs(F.weight_values(codes, scales)).sum(1)
    tol = (k + 64) * 2.0 ** -24 * mag + 2.0 ** -133 * (w + k * 2.0 ** -100)
    if yd == "bf16":
        tol = tol + 7 * 2.0 ** -13 * mag + 2.0 ** -8 * np.abs(want)
    bad = np.abs(got.double().cpu().numpy() - want) > tol
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4].tolist())


@pytest.mark.parametrize("rows", [4, 130])
def test_infinities_and_nans_stay_in_their_rows(rows):
    rng = np.random.default_rng(4)
    x, codes, scales, bias = make(rng, rows, 384, 200)
    x[1, 5], x[2, 200], x[3, 383] = np.inf, np.nan, -np.inf
    for xd in ("bf16", "f32"):
        t = on_gpu(x, xd)
        for yd in ("bf16", "f32"):
            got = layer_of(384, 200, codes, scales, bias).forward(t, out_dtype=DTYPES[yd])
            assert torch.isnan(got[1:4]).all()
            keep = [r for r in range(rows) if r not in (1, 2, 3)]
            check(got[keep], t[keep], codes, scales, bias, 384)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 257), (1025, 640)])
def test_loading_rounds_weights(dtype, n, k):
    rng = np.random.default_rng(n + k)
    w = torch.from_numpy((rng.standard_normal((n, k)) * 0.1).astype(np.float32)).to(dtype)
    bias = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).to(dtype)
    codes, scales = F.quantize_weight(w.double().numpy())
    x = on_gpu(rng.standard_normal((9, k)), "f32")
    for src in (w, w.cuda()):
        layer = M.Fp8Linear(k, n, True)
        layer.load(src, bias if src is w else bias.cuda())
        got = layer.read_codes()
        assert np.array_equal(got[1], scales) and np.array_equal(F.VALUES[got[0]], F.VALUES[codes])
        check(layer.forward(x), x, codes, scales, bias.float().numpy(), k)


def test_codes_from_host_and_gpu_and_nan_blocks():
    rng = np.random.default_rng(6)
    x, codes, scales, _ = make(rng, 7, 300, 260)
    scales[1, 2] = 255
    t = on_gpu(x, "f32")
    a = layer_of(300, 260, codes, scales, None)
    b = layer_of(300, 260, torch.from_numpy(codes).cuda().view(torch.float8_e4m3fn), torch.from_numpy(scales).cuda(), None)
    for rows in (t, t.repeat(20, 1)):
        u, v = a.forward(rows), b.forward(rows)
        assert torch.equal(u.view(torch.int32), v.view(torch.int32))
        assert torch.isnan(u[:, 128:256]).all() and not torch.isnan(u[:, :128]).any() and not torch.isnan(u[:, 256:]).any()
        assert torch.isnan(a.forward(rows, out_dtype=torch.bfloat16)[:, 128:256]).all()


@pytest.mark.parametrize("rows", [3, 129])
@pytest.mark.parametrize("yd", ["bf16", "f32"])
def test_strided_rows_leave_their_surroundings(rows, yd):
    rng = np.random.default_rng(8)
    k, n = 200, 77
    x, codes, scales, bias = make(rng, rows, k, n)
    wide = on_gpu(np.pad(x, ((0, 0), (3, 10)), constant_values=np.nan), "bf16")
    out = torch.full((rows + 2, n + 9), 7.0, device="cuda", dtype=DTYPES[yd])
    layer = layer_of(k, n, codes, scales, bias)
    view = out[1:-1, 4:4 + n]
    got = layer.forward(wide[:, 3:3 + k], out=view)
    assert got is view
    check(got, wide[:, 3:3 + k], codes, scales, bias, k)
    around = out.clone()
    around[1:-1, 4:4 + n] = 7.0
    assert (around == 7.0).all()
    with pytest.raises(M.MhsaError):
        layer.forward(wide.T[:, :1].expand(-1, k))  # rows that do not lie apart
    with pytest.raises(M.MhsaError):
        layer.forward(wide[:, 3:3 + k], out=wide[:, :n])  # overlaps x


def test_empty_and_leading_shapes():
    rng = np.random.default_rng(9)
    x, codes, scales, bias = make(rng, 12, 256, 96)
    layer = layer_of(256, 96, codes, scales, bias)
    assert layer.forward(torch.empty(0, 256, device="cuda")).shape == (0, 96)
    t = on_gpu(x, "f32")
    assert torch.equal(layer.forward(t.view(2, 6, 256)).view(12, 96), layer.forward(t))
    assert torch.equal(layer.forward(t[0]), layer.forward(t)[0])


def test_loading_again_replaces_the_weights():
    rng = np.random.default_rng(10)
    x, codes, scales, bias = make(rng, 100, 256, 96)
    layer = layer_of(256, 96, codes, scales, bias)
    t = on_gpu(x, "f32")
    layer.forward(t)
    _, codes, scales, bias = make(rng, 100, 256, 96)
    layer.load_codes(codes, scales, bias)
    check(layer.forward(t), t, codes, scales, bias, 256)


def test_replayed_graphs_and_streams():
    """Two captured calls of one layer with workspaces of their own, replayed
    with eager work between; and eager calls on two streams at once."""
    rng = np.random.default_rng(11)
    x, codes, scales, bias = make(rng, 600, 512, 300)
    layer = layer_of(512, 300, codes, scales, bias)
    ins = [on_gpu(x[:200], "bf16"), on_gpu(x[:9], "bf16")]
    layer.forward(ins[0])
    graphs, outs = [], []
    for t in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.forward(t))
        graphs.append(g)
    for rep in range(4):
        for i, t in enumerate(ins):
            t.copy_(on_gpu(x[rep * 100:rep * 100 + t.shape[0]], "bf16"))
        layer.forward(on_gpu(x, "f32"))  # a larger eager call between
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for t, o in zip(ins, outs):
            assert torch.equal(o, layer.forward(t))
    big = [on_gpu(x, "bf16"), on_gpu(-x, "bf16")]
    want = [layer.forward(t) for t in big]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer.forward(big[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_workspace_is_checked():
    rng = np.random.default_rng(12)
    x, codes, scales, bias = make(rng, 300, 256, 96)  # (up to 256 rows may need none)
    layer, lib = layer_of(256, 96, codes, scales, bias), M.library()
    t, out = on_gpu(x, "f32"), torch.empty(300, 96, device="cuda")
    need = lib.mhsa_fp8_linear_workspace(layer._h, 300)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")

    def call(ptr, size):
        return lib.mhsa_fp8_linear_forward(layer._h, t.data_ptr(), M.F32, 300, 256, out.data_ptr(), M.F32, 96, ptr, size, None)
    torch.cuda.synchronize()
    assert call(None, need) == call(ws.data_ptr(), need - 1) == call(ws.data_ptr() + 8, need) == M.MHSA_EINVAL
    assert call(t.data_ptr(), need) == M.MHSA_EINVAL
    assert call(ws.data_ptr(), need) == M.MHSA_OK
    torch.cuda.synchronize()
    check(out, t, codes, scales, bias, 256)
