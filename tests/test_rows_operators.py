"""The operators on rows and the adapters without a GPU: the oracle against
torch in 64 bits, and what the C ABI refuses before it touches a device."""
import ctypes

import numpy as np
import pytest
import torch

import relpos_mhsa as M
import rows_oracle as R

SOME = 1 << 20  # a plausible, aligned device address: no call here may get as far as using it


def test_oracle_norm_against_torch():
    rng = np.random.default_rng(0)
    x, d = rng.standard_normal((2, 5, 37))
    w, b = rng.standard_normal((2, 37))
    t = torch.from_numpy(x + 0.5 * d)
    y, v, _ = R.norm(x, d, 0.5, w, b, "layer", 1e-3)
    want = torch.nn.functional.layer_norm(t, (37,), torch.from_numpy(w), torch.from_numpy(b), float(np.float32(1e-3)))
    assert np.allclose(y, want.numpy(), rtol=1e-12, atol=1e-12) and np.array_equal(v, t.numpy())
    y, _, _ = R.norm(x, None, 1.0, w, None, "rms", 1e-3)
    want = torch.nn.functional.rms_norm(torch.from_numpy(x), (37,), torch.from_numpy(w), float(np.float32(1e-3)))
    assert np.allclose(y, want.numpy(), rtol=1e-12, atol=1e-12)


def test_oracle_scores_against_torch():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((6, 50))
    x[0, 5:] = -np.inf
    tokens = rng.integers(0, 50, (6, 2)).astype(np.int32)
    tokens[0], tokens[1, 0] = 3, -1
    lp, h, idx, top, _ = R.scores(x, tokens, 4, 0.5)
    want = torch.log_softmax(torch.from_numpy(x) / 0.5, -1)
    for r in range(6):
        for j in range(2):
            assert lp[r, j] == 0.0 if tokens[r, j] < 0 else np.isclose(lp[r, j], want[r, tokens[r, j]], rtol=1e-12)
    assert np.allclose(h, torch.special.entr(want.exp()).sum(-1).numpy())
    assert np.array_equal(idx, want.topk(4).indices.numpy()) and np.allclose(top, want.topk(4).values.numpy())


def test_add_norm_refuses():
    f = M.library().mhsa_add_norm
    good = dict(x=SOME, dt=M.F32, rows=4, dim=64, ldx=64, d=2 * SOME, ldd=64, a=1.0, s=3 * SOME, lds=64, kind=0, w=4 * SOME, b=None,
                eps=1e-5, o=5 * SOME, od=M.F32, ldo=64, c=None, sc=None)

    def call(**more):
        a = {**good, **more}
        return f(a["x"], a["dt"], a["rows"], a["dim"], a["ldx"], a["d"], a["ldd"], a["a"], a["s"], a["lds"], a["kind"], a["w"], a["b"],
                 a["eps"], a["o"], a["od"], a["ldo"], a["c"], a["sc"], None)
    for more in (dict(dt=M.F16), dict(od=M.F16), dict(kind=2), dict(dim=32769, ldx=32769, ldd=32769, lds=32769, ldo=32769),
                 dict(rows=(1 << 25) + 1), dict(ldx=(1 << 30) + 1), dict(ldo=(1 << 30) + 1)):
        assert call(**more) == M.MHSA_ENOTSUP, more
    for more in (dict(rows=-1), dict(dim=0), dict(eps=-1e-9), dict(eps=float("nan")), dict(eps=float("inf")), dict(a=float("nan")),
                 dict(x=None), dict(s=None, o=None), dict(ldx=63), dict(ldd=63), dict(lds=63), dict(ldo=63), dict(x=SOME + 2),
                 dict(d=2 * SOME + 1), dict(w=4 * SOME + 2), dict(b=SOME + 1), dict(c=6 * SOME), dict(sc=6 * SOME),
                 dict(c=6 * SOME + 8, sc=7 * SOME), dict(c=6 * SOME, sc=6 * SOME + 16), dict(c=SOME, sc=7 * SOME),
                 dict(c=6 * SOME, sc=4 * SOME), dict(s=SOME + 4), dict(o=SOME + 256), dict(o=3 * SOME), dict(o=2 * SOME + 4),
                 dict(s=4 * SOME), dict(o=4 * SOME - 4), dict(o=SOME, od=M.BF16), dict(s=SOME, lds=80)):
        assert call(**more) == M.MHSA_EINVAL, more
    assert call(rows=0, x=None, d=None, s=None, o=None) == M.MHSA_OK


def test_token_log_probs_refuses():
    lib = M.library()
    f = lib.mhsa_token_log_probs
    good = dict(x=SOME, dt=M.F32, rows=4, v=64, ld=64, t=1.0, tok=2 * SOME, n=1, lp=3 * SOME, h=4 * SOME, k=2, i=5 * SOME, tp=6 * SOME,
                ws=None, wn=0)

    def call(**more):
        a = {**good, **more}
        return f(a["x"], a["dt"], a["rows"], a["v"], a["ld"], a["t"], a["tok"], a["n"], a["lp"], a["h"], a["k"], a["i"], a["tp"], a["ws"],
                 a["wn"], None)
    for more in (dict(dt=M.F16), dict(v=(1 << 24) + 1, ld=1 << 25), dict(k=33), dict(n=1025), dict(rows=(1 << 25) + 1),
                 dict(ld=(1 << 30) + 1)):
        assert call(**more) == M.MHSA_ENOTSUP, more
    for more in (dict(rows=-1), dict(v=0), dict(k=-1), dict(k=65), dict(n=-1), dict(t=0.0), dict(t=-1.0), dict(t=0.009), dict(t=101.0),
                 dict(t=float("nan")), dict(t=float("inf")), dict(x=None), dict(tok=None), dict(lp=None), dict(i=None), dict(tp=None),
                 dict(x=SOME + 2), dict(tok=SOME + 1), dict(lp=3 * SOME + 2), dict(h=SOME + 3), dict(i=SOME + 1), dict(tp=SOME + 2),
                 dict(ld=63), dict(lp=SOME), dict(h=SOME + 1020), dict(i=2 * SOME), dict(tp=5 * SOME + 28), dict(h=3 * SOME + 12),
                 dict(v=100000, ld=100000), dict(v=100000, ld=100000, ws=7 * SOME, wn=16), dict(v=100000, ld=100000, ws=7 * SOME + 8, wn=1 << 20),
                 dict(v=100000, ld=100000, ws=SOME + 64, wn=1 << 20)):
        assert call(**more) == M.MHSA_EINVAL, more
    assert call(rows=0, x=None, tok=None, lp=None, h=None, i=None, tp=None) == M.MHSA_OK
    ws = lib.mhsa_token_log_probs_workspace
    for args in ((-1, 64, 1), (1, 0, 1), (1, (1 << 24) + 1, 1), (1, 64, -1), (1, 64, 33), ((1 << 25) + 1, 64, 1)):
        assert ws(*args) == -1
    assert ws(0, 1 << 20, 4) == 0 and ws(100, 1025, 4) == 0 and ws(1, 1 << 20, 4) > 0


@pytest.mark.parametrize("v,k", [(8193, 0), (20000, 1), (128000, 20), (1 << 24, 32)])
def test_token_log_probs_workspace_grows_with_the_rows(v, k):
    ws = M.library().mhsa_token_log_probs_workspace
    need = [ws(r, v, k) for r in list(range(1, 1500)) + [5000, 100000]]
    assert all(a <= b for a, b in zip(need, need[1:]))


def adapters(i=256, o=384, n=4, r=16):
    h = ctypes.c_void_p()
    assert M.library().mhsa_adapters_create(i, o, n, r, ctypes.byref(h)) == 0
    return h


def linear(i=256, o=384):
    h = ctypes.c_void_p()
    assert M.library().mhsa_fp8_linear_create(i, o, 0, ctypes.byref(h)) == 0
    return h


def test_adapters_create_and_load_refuse():
    lib, h = M.library(), ctypes.c_void_p()
    for args, code in (((0, 8, 1, 1), M.MHSA_EINVAL), ((8, 0, 1, 1), M.MHSA_EINVAL), ((8, 8, 0, 1), M.MHSA_EINVAL),
                       ((8, 8, 1, 0), M.MHSA_EINVAL), ((32769, 8, 1, 1), M.MHSA_ENOTSUP), ((8, (1 << 22) + 1, 1, 1), M.MHSA_ENOTSUP),
                       ((8, 8, 4097, 1), M.MHSA_ENOTSUP), ((8, 8, 1, 129), M.MHSA_ENOTSUP)):
        assert lib.mhsa_adapters_create(*args, ctypes.byref(h)) == code and not h.value
    assert lib.mhsa_adapters_create(8, 8, 1, 1, None) == M.MHSA_EINVAL
    h, w = adapters(), np.zeros((384, 256), np.float32)
    p = w.ctypes.data
    f = lib.mhsa_adapters_load
    assert f(None, 0, 4, M.F32, p, p, 1.0) == M.MHSA_EINVAL
    for args, code in (((-1, 4, M.F32, p, p, 1.0), M.MHSA_EINVAL), ((4, 4, M.F32, p, p, 1.0), M.MHSA_EINVAL),
                       ((0, 17, M.F32, p, p, 1.0), M.MHSA_EINVAL), ((0, -1, M.F32, p, p, 1.0), M.MHSA_EINVAL),
                       ((0, 4, M.F32, None, p, 1.0), M.MHSA_EINVAL), ((0, 4, M.F32, p, None, 1.0), M.MHSA_EINVAL),
                       ((0, 4, M.U32, p, p, 1.0), M.MHSA_ENOTSUP), ((0, 4, M.F32, p, p, float("inf")), M.MHSA_EINVAL)):
        assert f(h, *args) == code, args
    lib.mhsa_adapters_destroy(h)
    a = M.LowRankAdapters(256, 384, 2, 8)
    for args in ((0, w[:4], w[:, :5]), (0, w[:4, :255], w[:, :4]), (0, w[0], w[:, :4]), (0, [1.0], w), (0, w[:4], None),
                 (0, w[:4], w[:, :4].astype(np.float16)), (0, w[:9], w[:, :9]), (2, w[:4], w[:, :4]),
                 (0, w[:4].astype(np.float64), w[:, :4].astype(np.float64))):
        with pytest.raises(M.MhsaError):
            a.load(*args)


def test_adapted_forward_refuses():
    lib, h, ad, other = M.library(), linear(), adapters(), adapters(o=385)
    f = lib.mhsa_fp8_linear_forward_adapted
    assert f(None, SOME, M.F32, 1, 256, ad, SOME, 2 * SOME, M.F32, 384, None, 0, None) == M.MHSA_EINVAL
    for args in ((SOME, M.F16, 1, 256, ad, 3 * SOME, 2 * SOME, M.F32, 384), (SOME, M.F32, 1, 256, ad, 3 * SOME, 2 * SOME, M.U32, 384),
                 (SOME, M.F32, (1 << 25) + 1, 256, ad, 3 * SOME, 2 * SOME, M.F32, 384)):
        assert f(h, *args, None, 0, None) == M.MHSA_ENOTSUP
    for args in ((SOME, M.F32, -1, 256, ad, 3 * SOME, 2 * SOME, M.F32, 384), (None, M.F32, 1, 256, ad, 3 * SOME, 2 * SOME, M.F32, 384),
                 (SOME, M.F32, 2, 255, ad, 3 * SOME, 2 * SOME, M.F32, 384), (SOME, M.F32, 1, 256, ad, 3 * SOME, 2 * SOME, M.F32, 384)):
        assert f(h, *args, None, 0, None) == M.MHSA_EINVAL
    assert b"no weights" in lib.mhsa_last_error()
    assert f(h, None, M.F32, 0, 256, ad, None, None, M.F32, 384, None, 0, None) == M.MHSA_OK
    g = lib.mhsa_fp8_linear_forward_rounded
    for args in ((None, SOME, 1, None, None, 2 * SOME, M.F32, 384), (SOME, None, 1, None, None, 2 * SOME, M.F32, 384),
                 (SOME + 8, 3 * SOME, 1, None, None, 2 * SOME, M.F32, 384), (SOME, 3 * SOME + 4, 1, None, None, 2 * SOME, M.F32, 384),
                 (SOME, 3 * SOME, 1, None, None, None, M.F32, 384), (SOME, 3 * SOME, 1, None, None, 2 * SOME, M.F32, 383),
                 (SOME, 3 * SOME, -1, None, None, 2 * SOME, M.F32, 384), (SOME, 3 * SOME, 1, None, None, 2 * SOME, M.F32, 384)):
        assert g(h, *args, None, 0, None) == M.MHSA_EINVAL
    assert b"no weights" in lib.mhsa_last_error()
    assert g(h, SOME, 3 * SOME, 1, None, None, 2 * SOME, M.F16, 384, None, 0, None) == M.MHSA_ENOTSUP
    assert g(h, None, None, 0, None, None, None, M.F32, 384, None, 0, None) == M.MHSA_OK
    w = lib.mhsa_fp8_linear_adapted_workspace
    assert w(None, ad, 4) == -1 and w(h, None, 4) == -1 and w(h, ad, -1) == -1 and w(h, ad, (1 << 25) + 1) == -1 and w(h, ad, 0) == 0
    for x in (ad, other):
        lib.mhsa_adapters_destroy(x)
    lib.mhsa_fp8_linear_destroy(h)


@pytest.mark.parametrize("i,o,r", [(64, 64, 4), (1024, 4096, 16), (4096, 1024, 64), (300, 7000, 128)])
def test_adapted_workspace_grows_with_the_rows(i, o, r):
    lib, h, ad = M.library(), linear(i, o), adapters(i, o, 2, r)
    need = [lib.mhsa_fp8_linear_adapted_workspace(h, ad, n) for n in list(range(1, 400)) + [1000, 30000, 1 << 25]]
    plain = [lib.mhsa_fp8_linear_workspace(h, n) for n in list(range(1, 400)) + [1000, 30000, 1 << 25]]
    lib.mhsa_adapters_destroy(ad)
    lib.mhsa_fp8_linear_destroy(h)
    assert all(a <= b for a, b in zip(need, need[1:])) and all(a >= b for a, b in zip(need, plain))
