"""Microscaled 4-bit formats and the RMS norm without a GPU: the reference's own
arithmetic, sizes, and the arguments that the entry points refuse before any
device work."""
import ctypes as C

import numpy as np
import pytest

import mx4_ref as R

P = 1 << 20  # a well aligned address that is never followed


@pytest.fixture(scope="module")
def nq():
    import nova_b200.capi as capi
    return capi


def test_e2m1_and_e4m3_roundings():
    x = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 100.0, 0.2501, -0.75, -5.0])
    assert R.e2m1(x).tolist() == [0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, 0.5, -1.0, -4.0]
    every = R.e4m3_of_byte(np.arange(127))
    assert every[-1] == 448.0 and every[1] == 2.0 ** -9
    assert np.array_equal(R.e4m3(every), every)
    mid = (every[1:] + every[:-1]) / 2
    assert np.array_equal(R.e4m3(mid), np.where(np.arange(126) % 2 == 0, every[:-1], every[1:]))


@pytest.mark.parametrize("fmt", [R.MX, R.NV])
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (130, 100), (257, 64)])
def test_reference_storage_round_trips(fmt, shape):
    x = np.random.default_rng(shape[1]).standard_normal(shape)
    q, s, g = R.quantize(x, fmt)
    codes, scales, rows = R.pack(x, fmt)
    v = (R.e2m1(q) * s[..., None]).reshape(shape[0], -1)[:, :shape[1]]
    assert np.array_equal(R.values(codes, scales, *shape, fmt), v)
    back = v if g is None else v * g[:, None]
    # a block's step is 1/6 (MX: at most 1/4, saturating from 7 to 6) of its largest value at most, half of it up or down
    top = np.repeat(np.abs(R.blocks(x, fmt)).max(-1), R.BLOCK[fmt], 1)[:, :shape[1]]
    assert np.all(np.abs(back - x) <= 0.25 * top + 1e-12)


def test_backward_reference_against_differences():
    rng = np.random.default_rng(0)
    h, w, dy = rng.standard_normal((4, 7)), rng.standard_normal(7), rng.standard_normal((4, 7))
    f = lambda h, w: (R.rmsnorm(h, w, 1e-3)[0] * R.rmsnorm(h, w, 1e-3)[1][:, None] * dy).sum()
    dx, dw = R.rmsnorm_backward(h, w, dy, None, 1e-3)
    e = 1e-6
    for i in np.ndindex(h.shape):
        d = np.zeros_like(h)
        d[i] = e
        assert abs((f(h + d, w) - f(h - d, w)) / (2 * e) - dx[i]) < 1e-8
    for j in range(7):
        d = np.zeros(7)
        d[j] = e
        assert abs((f(h, w + d) - f(h, w - d)) / (2 * e) - dw[j]) < 1e-8


def test_sizes(nq):
    for cols in (0, 1, 31, 32, 33, 8192, 2 ** 31 - 1):
        assert nq.mx4_row_bytes(cols) == R.pitch(cols)
    for rows, cols in ((0, 5), (1, 1), (128, 128), (129, 129), (28672, 8192), (2 ** 31 - 1, 1)):
        for fmt in (R.MX, R.NV):
            assert nq.mx4_scale_bytes(rows, cols, fmt) == (rows + 127) // 128 * R.words(cols, fmt) * 512
    assert nq.mx4_row_bytes(-1) == 0 and nq.mx4_scale_bytes(-1, 4, 0) == 0 and nq.mx4_scale_bytes(4, 4, 2) == 0


def test_quantize_refusals(nq):
    q = nq.quantize_rows_mx4.raw
    good = dict(src=P, dt=nq.BF16, ld=0, codes=P, bs=P, g=P, rows=4, cols=64, fmt=nq.NVFP4)
    call = lambda **k: q(*{**good, **k}.values(), None)
    for bad in (dict(src=None), dict(codes=None), dict(bs=None), dict(g=None), dict(rows=-1), dict(cols=-1), dict(fmt=2),
                dict(dt=nq.S8), dict(ld=63), dict(codes=P + 8), dict(bs=P + 4), dict(src=P + 1), dict(g=P + 2),
                dict(fmt=nq.MXFP4), dict(src=P + 2, dt=nq.F32)):
        assert call(**bad) == 1, bad
        assert b"nq_quantize_rows_mx4" in nq.lib.nq_last_error()
    assert call(cols=(1 << 30) + 1) == 2
    assert call(rows=0, src=None) == 0 and call(cols=0, src=None) == 0


def test_dequantize_refusals(nq):
    q = nq.dequantize_rows_mx4.raw
    good = dict(codes=P, bs=P, g=P, dst=P, dt=nq.BF16, rows=4, cols=64, fmt=nq.NVFP4)
    call = lambda **k: q(*{**good, **k}.values(), None)
    for bad in (dict(codes=None), dict(bs=None), dict(dst=None), dict(rows=-1), dict(cols=-1), dict(fmt=-1), dict(dt=nq.S32),
                dict(codes=P + 8), dict(bs=P + 8), dict(dst=P + 1), dict(g=P + 1)):
        assert call(**bad) == 1, bad
    assert call(rows=0, dst=None) == 0 and call(cols=0, dst=None) == 0


def test_gemm_refusals(nq):
    good = dict(a=P, sa=P, b=P, sb=P, out=P)

    def call(ptrs=(), **k):
        d = nq.make_mx4_desc(**{**dict(m=4, n=8, k=64), **k})
        return nq.gemm_mx4.raw(C.byref(d), *{**good, **dict(ptrs)}.values(), None)

    for bad in (dict(m=-1), dict(n=-1), dict(k=-1), dict(format=2), dict(out_dtype=nq.S8), dict(row_scale=P + 1),
                dict(col_scale=P + 2), dict(bias=P + 3)):
        assert call(**bad) == 1, bad
    for name in good:
        assert call({name: None}) == 1, name
    for name in ("a", "sa", "b", "sb"):
        assert call({name: P + 8}) == 1, name
    assert call({"out": P + 1}) == 1
    assert call(k=(1 << 30) + 1) == 2
    assert nq.gemm_mx4.raw(None, P, P, P, P, P, None) == 1
    assert call({"out": None}, m=0) == 0 and call({"out": None}, n=0) == 0


def norm_call(nq, four):
    good = dict(x=P, res=P + 4096, w=P, sum=P + 8192, y=P + 16384, codes=P, bs=P, g=P, fmt=nq.NVFP4 if four else nq.E4M3)
    if not four:
        del good["bs"]

    def call(ptrs=(), **k):
        d = nq.make_rmsnorm_desc(**{**dict(rows=4, cols=64), **k})
        fn = nq.rmsnorm_quantize_mx4.raw if four else nq.rmsnorm_quantize.raw
        return fn(C.byref(d), *{**good, **dict(ptrs)}.values(), None)

    return call


@pytest.mark.parametrize("four", [False, True])
def test_rmsnorm_refusals(nq, four):
    call = norm_call(nq, four)
    for bad in (dict(rows=-1), dict(cols=-1), dict(dtype=nq.S8), dict(weight_dtype=nq.S32), dict(eps=0.0), dict(eps=-1.0),
                dict(eps=float("nan")), dict(eps=float("inf")), dict(x_stride=63), dict(residual_stride=1)):
        assert call(**bad) == 1, bad
    for bad in (dict(x=None), dict(w=None), dict(codes=None), dict(g=None), dict(res=None), dict(fmt=7), dict(y=P),
                dict(y=P + 4096), dict(y=P + 8192), dict(x=P + 1), dict(res=P + 1), dict(sum=P + 1), dict(y=P + 1),
                dict(w=P + 1), dict(g=P + 2)):
        assert call(bad) == 1, bad
    assert call(dict(y=None, codes=None, g=None, **({"bs": None} if four else {}))) == 1   # no output at all
    assert call(dict(sum=P), x_stride=128) == 1                                             # in place of a strided tensor
    assert call(dict(sum=P + 4096), residual_stride=128) == 1
    if four:
        assert call(dict(bs=None)) == 1 and call(dict(codes=P + 8)) == 1 and call(dict(bs=P + 8)) == 1
        assert call(dict(fmt=nq.MXFP4)) == 1                                                # no row scales
    assert call(cols=(1 << 30) + 1) == 2
    assert call(dict(x=None), rows=0) == 0 and call(dict(x=None), cols=0) == 0


def test_rmsnorm_backward_refusals(nq):
    good = dict(h=P, w=P, dy=P + 4096, dsum=P + 8192, dx=P + 16384, dw=P + 32768)

    def call(ptrs=(), **k):
        d = nq.make_rmsnorm_desc(**{**dict(rows=4, cols=64), **k})
        return nq.rmsnorm_backward.raw(C.byref(d), *{**good, **dict(ptrs)}.values(), None)

    for bad in (dict(h=None), dict(w=None), dict(dy=None), dict(dx=None, dw=None), dict(dx=P), dict(dx=P + 4096), dict(dw=P),
                dict(dw=P + 16384), dict(dw=P + 2), dict(dx=P + 1), dict(h=P + 1), dict(dy=P + 1), dict(dsum=P + 1)):
        assert call(bad) == 1, bad
    for bad in (dict(rows=-1), dict(eps=0.0), dict(dtype=2), dict(x_stride=2)):
        assert call(**bad) == 1, bad
    assert call(dict(h=None), cols=0) == 0 and call(dict(h=None, dw=None), rows=0) == 0


def test_rmsnorm_eps_range(nq):
    """eps from FLT_MIN to FLT_MAX, as the header says: squares below fp32's range would count beside a smaller one."""
    smallest = float(np.finfo(np.float32).tiny)
    for eps in (smallest, 1e-5, 1.0, float(np.finfo(np.float32).max)):
        d = nq.make_rmsnorm_desc(0, 64, eps=eps)
        assert nq.rmsnorm_quantize.raw(C.byref(d), P, None, P, None, P + 4096, None, None, nq.E4M3, None) == 0
        assert nq.rmsnorm_quantize_mx4.raw(C.byref(d), P, None, P, None, P + 4096, None, None, None, nq.NVFP4, None) == 0
        assert nq.rmsnorm_backward.raw(C.byref(d), P, P, P, None, P + 4096, None, None) == 0
    for eps in (0.0, 1e-45, 1e-39, 0.5 * smallest):
        d = nq.make_rmsnorm_desc(4, 64, eps=eps)
        for call in (lambda: nq.rmsnorm_quantize.raw(C.byref(d), P, None, P, None, P + 4096, None, None, nq.E4M3, None),
                     lambda: nq.rmsnorm_quantize_mx4.raw(C.byref(d), P, None, P, None, P + 4096, None, None, None, nq.NVFP4, None),
                     lambda: nq.rmsnorm_backward.raw(C.byref(d), P, P, P, None, P + 4096, None, None)):
            assert call() == 1 and b"eps" in nq.lib.nq_last_error()
