"""The 8-bit block-scaled projection, routing and the experts' FeedForward
without a GPU: the oracle's formats against torch's e4m3, and what the C ABI
refuses before it touches a device."""
import ctypes

import numpy as np
import pytest
import torch

import fp8_oracle as F
import relpos_mhsa as M

SOME = 1 << 20  # a plausible, aligned device address: no call here may get as far as using it


def test_code_values_are_e4m3():
    t = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(F.VALUES, t, equal_nan=True)


def test_encoding_rounds_to_nearest_even():
    rng = np.random.default_rng(0)
    v = np.concatenate([rng.uniform(-448, 448, 20000), rng.standard_normal(20000) * 2.0 ** rng.integers(-12, 6, 20000)])
    mid = (F.POSITIVE[1:] + F.POSITIVE[:-1]) / 2
    v = np.concatenate([v, mid, -mid, F.POSITIVE, [448.0, 0.0]]).astype(np.float32)
    want = torch.from_numpy(v).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(F.VALUES[F.encode(v)], F.VALUES[want])


@pytest.mark.parametrize("e", [-127, -60, 0, 1, 80])
def test_scale_byte_is_the_smallest(e):
    edge = 448.0 * 2.0 ** e
    assert F.scale_byte(edge) == e + 127
    assert F.scale_byte(np.nextafter(edge, np.inf)) == e + 128
    assert F.scale_byte(0.0) == 127 and F.scale_byte(2.0 ** -149) == 0


def linear(i=256, o=384, bias=0):
    h = ctypes.c_void_p()
    assert M.library().mhsa_fp8_linear_create(i, o, bias, ctypes.byref(h)) == 0
    return h


def experts(e=4, d=128, f=256, bias=0):
    h = ctypes.c_void_p()
    assert M.library().mhsa_experts_create(e, d, f, bias, ctypes.byref(h)) == 0
    return h


def test_create_refuses():
    lib, h = M.library(), ctypes.c_void_p()
    for args, code in (((0, 8, 0), M.MHSA_EINVAL), ((8, -1, 0), M.MHSA_EINVAL), ((32769, 8, 0), M.MHSA_ENOTSUP),
                       ((32768, 1 << 20, 0), M.MHSA_ENOTSUP), ((8, (1 << 22) + 1, 0), M.MHSA_ENOTSUP)):
        assert lib.mhsa_fp8_linear_create(*args, ctypes.byref(h)) == code and not h.value
    assert lib.mhsa_fp8_linear_create(8, 8, 0, None) == M.MHSA_EINVAL
    for args, code in (((0, 64, 64, 0), M.MHSA_EINVAL), ((2, 65, 64, 0), M.MHSA_EINVAL), ((2, 64, 0, 0), M.MHSA_EINVAL),
                       ((1025, 64, 64, 0), M.MHSA_ENOTSUP), ((2, 64, 32832, 0), M.MHSA_ENOTSUP)):
        assert lib.mhsa_experts_create(*args, ctypes.byref(h)) == code and not h.value
    assert lib.mhsa_experts_create(2, 64, 64, 0, None) == M.MHSA_EINVAL


def test_load_refuses():
    lib, h = M.library(), linear()
    w = np.zeros((384, 256), np.float32)
    assert lib.mhsa_fp8_linear_load(None, M.F32, w.ctypes.data, None) == M.MHSA_EINVAL
    assert lib.mhsa_fp8_linear_load(h, M.F32, None, None) == M.MHSA_EINVAL
    assert lib.mhsa_fp8_linear_load(h, M.U32, w.ctypes.data, None) == M.MHSA_ENOTSUP
    assert lib.mhsa_fp8_linear_load(h, M.F32, w.ctypes.data, w.ctypes.data) == M.MHSA_EINVAL  # created without a bias
    assert lib.mhsa_fp8_linear_load_codes(h, None, w.ctypes.data, None) == M.MHSA_EINVAL
    assert lib.mhsa_fp8_linear_load_codes(h, w.ctypes.data, None, None) == M.MHSA_EINVAL
    assert lib.mhsa_fp8_linear_read_codes(h, w.ctypes.data, w.ctypes.data) == M.MHSA_EINVAL  # nothing loaded
    lib.mhsa_fp8_linear_destroy(h)
    layer = M.Fp8Linear(256, 384, True)
    with pytest.raises(M.MhsaError):
        layer.load(w, np.zeros(384, np.float16))  # another dtype than the weight's
    for weight, bias in ((w.T, np.zeros(384, np.float32)), (w.astype(np.float64), np.zeros(384, np.float32)),
                         (w, np.zeros(383, np.float32)), (w, None)):
        with pytest.raises(M.MhsaError):
            layer.load(weight, bias)
    with pytest.raises(M.MhsaError):
        layer.load_codes(w, np.zeros((3, 2), np.uint8), np.zeros(384, np.float32))  # float codes
    with pytest.raises(M.MhsaError):
        layer.load_codes(np.zeros((384, 256), np.uint8), np.zeros((2, 3), np.uint8), np.zeros(384, np.float32))


def test_linear_forward_refuses():
    lib, h = M.library(), linear()
    f = lib.mhsa_fp8_linear_forward
    assert f(None, SOME, M.F32, 1, 256, SOME, M.F32, 384, None, 0, None) == M.MHSA_EINVAL
    for args in ((SOME, M.F16, 1, 256, SOME, M.F32, 384), (SOME, M.F32, 1, 256, SOME, M.U32, 384),
                 (SOME, M.F32, (1 << 25) + 1, 256, SOME, M.F32, 384), (SOME, M.F32, 2, (1 << 30) + 1, SOME, M.F32, 384),
                 (SOME, M.F32, 2, 256, SOME, M.F32, (1 << 30) + 1)):
        assert f(h, *args, None, 0, None) == M.MHSA_ENOTSUP
    for args in ((SOME, M.F32, -1, 256, SOME, M.F32, 384), (None, M.F32, 1, 256, SOME, M.F32, 384),
                 (SOME, M.F32, 1, 256, None, M.F32, 384), (SOME, M.F32, 2, 255, SOME, M.F32, 384),
                 (SOME, M.F32, 2, 256, SOME, M.F32, 383), (SOME + 2, M.F32, 1, 256, SOME, M.F32, 384),
                 (SOME, M.BF16, 1, 256, SOME + 1, M.BF16, 384), (SOME, M.F32, 1, 256, 2 * SOME, M.F32, 384)):
        assert f(h, *args, None, 0, None) == M.MHSA_EINVAL
    assert b"no weights" in lib.mhsa_last_error()
    assert f(h, None, M.F32, 0, 256, None, M.F32, 384, None, 0, None) == M.MHSA_OK  # no rows, nothing to do
    assert lib.mhsa_fp8_linear_workspace(h, -1) == -1 and lib.mhsa_fp8_linear_workspace(None, 4) == -1
    assert lib.mhsa_fp8_linear_workspace(h, 0) == 0
    assert lib.mhsa_fp8_linear_workspace(h, 1000) >= 1000 * 256 + 1000 * 2
    lib.mhsa_fp8_linear_destroy(h)


def test_route_refuses():
    f = M.library().mhsa_route
    good = dict(x=SOME, dt=M.F32, rows=4, e=64, ld=64, score=0, bias=None, g=8, kg=4, k=4, rn=1, s=1.0, i=2 * SOME, w=3 * SOME)

    def call(**more):
        a = {**good, **more}
        return f(a["x"], a["dt"], a["rows"], a["e"], a["ld"], a["score"], a["bias"], a["g"], a["kg"], a["k"], a["rn"],
                 a["s"], a["i"], a["w"], None)
    for more in (dict(dt=M.F16), dict(score=2), dict(e=520, ld=520, g=1, kg=1), dict(e=130, ld=130, g=65), dict(e=512, ld=512, g=1, kg=1, k=33),
                 dict(rows=(1 << 25) + 1), dict(ld=(1 << 30) + 1)):
        assert call(**more) == M.MHSA_ENOTSUP, more
    for more in (dict(rows=-1), dict(e=0), dict(g=0), dict(g=7), dict(kg=0), dict(kg=9), dict(k=0), dict(k=33), dict(ld=63),
                 dict(s=float("nan")), dict(s=float("inf")), dict(x=None), dict(i=None), dict(w=None), dict(x=SOME + 2),
                 dict(i=SOME + 1), dict(bias=SOME + 2), dict(i=SOME + 1020), dict(w=SOME), dict(w=2 * SOME + 60),
                 dict(bias=2 * SOME - 4), dict(bias=3 * SOME + 60)):
        assert call(**more) == M.MHSA_EINVAL, more
    assert call(rows=0, x=None, i=None, w=None) == M.MHSA_OK
    with pytest.raises(M.MhsaError):
        M.route(torch.zeros(2, 8), 2)  # a host tensor
    with pytest.raises(M.MhsaError):
        M.route(torch.zeros(2, 8), 2, score="relu")


def test_experts_forward_refuses():
    lib, h = M.library(), experts()
    f = lib.mhsa_experts_forward
    x, idx, w, r, out, ws = (SOME * i for i in range(1, 7))
    big = 1 << 19
    assert f(None, x, M.F32, 2, idx, w, 2, r, 1.0, out, ws, big, None) == M.MHSA_EINVAL
    assert f(h, x, M.F16, 2, idx, w, 2, r, 1.0, out, ws, big, None) == M.MHSA_ENOTSUP
    for args in ((x, M.F32, -1, idx, w, 2, r, 1.0, out), (x, M.F32, 2, idx, w, 0, r, 1.0, out), (x, M.F32, 2, idx, w, 33, r, 1.0, out),
                 (None, M.F32, 2, idx, w, 2, r, 1.0, out), (x, M.F32, 2, None, w, 2, r, 1.0, out), (x, M.F32, 2, idx, None, 2, r, 1.0, out),
                 (x, M.F32, 2, idx, w, 2, r, 1.0, None), (x + 4, M.F32, 2, idx, w, 2, r, 1.0, out), (x, M.F32, 2, idx, w, 2, r + 8, 1.0, out),
                 (x, M.F32, 2, idx + 2, w, 2, r, 1.0, out), (x, M.F32, 2, idx, w, 2, r, 1.0, out)):
        assert f(h, *args, ws, big, None) == M.MHSA_EINVAL, args
    assert b"no weights" in lib.mhsa_last_error()
    assert f(h, None, M.F32, 0, None, None, 2, None, 1.0, None, None, 0, None) == M.MHSA_OK
    assert f(h, x, M.F32, (1 << 25) + 1, idx, w, 2, r, 1.0, out, ws, big, None) == M.MHSA_ENOTSUP
    assert lib.mhsa_experts_workspace(h, (1 << 25) + 1, 2) == -1
    assert lib.mhsa_experts_workspace(h, 5, 0) == -1 and lib.mhsa_experts_workspace(h, -5, 2) == -1
    assert lib.mhsa_experts_workspace(h, 0, 2) == 0 and lib.mhsa_experts_workspace(h, 5, 2) > 0
    # rows run in parts, so the workspace stops growing
    assert lib.mhsa_experts_workspace(h, 1 << 20, 2) == lib.mhsa_experts_workspace(h, 1 << 24, 2)
    lib.mhsa_experts_destroy(h)
