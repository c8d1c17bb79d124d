"""Microscaled 4-bit quantize, dequantize and product on the GPU against 64-bit
references (tests/mx4_ref.py).

Tolerances:
- quantize: codes and scales are the correctly rounded ones, value for value.
- dequantize: exact products rounded to fp32 once (2^-24), to bf16 once more (2^-8 eps / 2).
- product: every product of two elements and two scales is exact; a group of 64
  is summed by one instruction and added to the fp32 accumulator, each to
  2^-22 of the sum of magnitudes at worst (a truncated fp32 addition is 2^-23),
  so |error| <= (groups + 2) 2^-22 sum |a b|, then at most four fp32
  roundings (scales, bias) and the output's."""
import ctypes as C

import numpy as np
import pytest

import mx4_ref as R

pytestmark = pytest.mark.gpu
FMTS = [R.MX, R.NV]


@pytest.fixture(scope="module")
def nq(cuda):
    import nova_b200.capi as capi
    return capi


def make(rows, cols, seed, bf16, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * scale
    return x.to(torch.bfloat16) if bf16 else x


def dtype_of(nq, t):
    import torch
    return nq.BF16 if t.dtype == torch.bfloat16 else nq.F32


def buffers(nq, rows, cols, fmt, guard=64):
    """Codes, scales and row scales filled with 0xAA, each with guard bytes behind."""
    import torch
    code_n, scale_n = rows * nq.mx4_row_bytes(cols), nq.mx4_scale_bytes(rows, cols, fmt)
    u8 = lambda n: torch.full((n + guard,), 0xAA, dtype=torch.uint8, device="cuda")
    return u8(code_n), u8(scale_n), torch.full((rows + 4,), -7.0, device="cuda") if fmt == R.NV else None


def quantize(nq, x, fmt, stride=0, stream=None):
    import torch
    rows, cols = x.shape
    codes, scales, g = buffers(nq, rows, cols, fmt)
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    nq.quantize_rows_mx4(x.data_ptr(), dtype_of(nq, x), stride, codes.data_ptr(), scales.data_ptr(),
                         g.data_ptr() if g is not None else 0, rows, cols, fmt, s)
    return codes, scales, g


def check_quantized(x, codes, scales, g, fmt):
    """Packed results (numpy, without guards) against the reference for doubles x."""
    rows, cols = x.shape
    q, s, gr = R.quantize(x, fmt)
    nb = (cols + R.BLOCK[fmt] - 1) // R.BLOCK[fmt]
    got_s = R.unpack_scales(scales, rows, cols, fmt)
    assert np.all(got_s[:, nb:] == (2.0 ** -127 if fmt == R.MX else 0.0)), "scales behind the last block"
    assert np.array_equal(got_s, s), "block scales"
    if fmt == R.NV:
        assert np.array_equal(g, gr.astype(np.float32)), "row scales"
    got = R.unpack_codes(codes, rows, cols)
    assert np.all(got[:, cols:] == 0), "codes behind the last column"
    w = q.shape[1] * q.shape[2]
    got = np.pad(got, ((0, 0), (0, max(0, w - got.shape[1]))))[:, :w].reshape(q.shape)
    assert np.array_equal(got, R.e2m1(q)), "codes"


SHAPES = [(1, 1), (1, 64), (70, 496), (900, 16), (700, 2064), (40, 512), (2, 15), (3, 16), (5, 17), (7, 33), (33, 128), (129, 130), (4, 1000), (300, 511), (64, 4096),
          (2, 8192), (3, 8200), (2, 16384), (2, 20008), (1, 40000), (3, 33001)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(nq, fmt, bf16, shape):
    import torch
    x = make(*shape, sum(shape), bf16)
    if shape[0] > 1:
        x[-1] = 0.0                     # a row of zeros
        x[0, : shape[1] // 2] *= 1e-4   # blocks far below the row's maximum
    codes, scales, g = quantize(nq, x, fmt)
    torch.cuda.synchronize()
    rows, cols = shape
    n, m = rows * nq.mx4_row_bytes(cols), nq.mx4_scale_bytes(rows, cols, fmt)
    codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
    assert np.all(codes[n:] == 0xAA) and np.all(scales[m:] == 0xAA)
    # bytes of rows behind the last one are left as they were
    used = np.zeros(m, bool)
    used[R.scale_index(rows, cols, fmt)] = True
    assert np.all(scales[:m][~used] == 0xAA)
    if g is not None:
        assert np.all(g[rows:].cpu().numpy() == -7.0)
        g = g[:rows].cpu().numpy()
    check_quantized(x.double().cpu().numpy(), codes[:n], scales[:m], g, fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_borders(nq, fmt):
    """Values on the borders of codes and scales: small integers, each ratio to the maximum many times."""
    import torch
    rng = np.random.default_rng(3)
    x = rng.integers(-255, 256, (200, 1600)).astype(np.float64) * np.ldexp(1.0, rng.integers(-6, 1, (200, 1600)))
    t = torch.from_numpy(x).cuda().to(torch.bfloat16)
    assert np.array_equal(t.double().cpu().numpy(), x)
    codes, scales, g = quantize(nq, t, fmt)
    n, m = 200 * nq.mx4_row_bytes(1600), nq.mx4_scale_bytes(200, 1600, fmt)
    check_quantized(x, codes[:n].cpu().numpy(), scales[:m].cpu().numpy(), None if g is None else g[:200].cpu().numpy(), fmt)


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_fp32_next_to_borders(nq, fmt):
    """fp32 values a step or two of 2^-24 from a border of their code, on either side and on it."""
    import torch
    rng = np.random.default_rng(5)
    rows, cols = 400, 640
    level = rng.uniform(1.0, 2.0, (rows, 1)).astype(np.float32).astype(np.float64)
    s = R.e4m3(rng.uniform(1.0, 448.0, (rows, cols // 16, 1)))
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    x = (rng.choice(mids, (rows, cols // 16, 16)) * s * level[..., None] / 2688.0).reshape(rows, cols).astype(np.float32)
    x = (x.view(np.int32) + rng.integers(-2, 3, x.shape, dtype=np.int32)).view(np.float32) * rng.choice([-1.0, 1.0], x.shape).astype(np.float32)
    x[:, ::16] = (s[..., 0] * level / 448.0).astype(np.float32)   # the blocks' maxima, near borders of the scales
    x[:, 0] = level[:, 0]
    t = torch.from_numpy(x).cuda()
    codes, scales, g = quantize(nq, t, fmt)
    n, m = rows * nq.mx4_row_bytes(cols), nq.mx4_scale_bytes(rows, cols, fmt)
    check_quantized(x.astype(np.float64), codes[:n].cpu().numpy(), scales[:m].cpu().numpy(), None if g is None else g[:rows].cpu().numpy(), fmt)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-33, 1e-20, 1e20, 3e37])
def test_quantize_extreme_magnitudes(nq, fmt, scale):
    import torch
    x = (make(9, 160, 11, False).clamp(-4, 4) * 0.25) * torch.tensor(scale, dtype=torch.float64, device="cuda").float()
    x[2, 7] = 3.4e38
    codes, scales, g = quantize(nq, x, fmt)
    n, m = 9 * nq.mx4_row_bytes(160), nq.mx4_scale_bytes(9, 160, fmt)
    check_quantized(x.double().cpu().numpy(), codes[:n].cpu().numpy(), scales[:m].cpu().numpy(),
                    None if g is None else g[:9].cpu().numpy(), fmt)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("bf16", [True, False])
def test_quantize_not_finite(nq, bad, bf16):
    import torch
    x = make(4, 100, 5, bf16)
    x[1, 40] = bad
    for fmt in FMTS:
        codes, scales, g = quantize(nq, x, fmt)
        c = R.unpack_codes(codes[:4 * nq.mx4_row_bytes(100)].cpu().numpy(), 4, 100)
        raw = scales[:nq.mx4_scale_bytes(4, 100, fmt)].cpu().numpy()[R.scale_index(4, 100, fmt)]
        if fmt == R.MX:
            assert raw[1, 1] == 255 and (raw == 255).sum() == 1 and np.all(c[1, 32:64] == 0)
        else:
            assert np.isnan(g[1].item()) and np.isfinite(g[[0, 2, 3]].cpu().numpy()).all()
            assert np.all(raw[1] == 0) and np.all(c[1] == 0)
        out = dequantize(nq, codes, scales, g, 4, 100, fmt, False)
        assert torch.isnan(out[1, 40]) and torch.isfinite(out[[0, 2, 3]]).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bf16", [True, False])
def test_quantize_strided_and_unaligned(nq, fmt, bf16):
    import torch
    big = make(40, 520, 21, bf16)
    for x, stride in ((big[:, :264], 520), (big[:, 8:8 + 96], 520), (big[:, 3:3 + 77], 520), (big[:, 1:1 + 512], 520)):
        codes, scales, g = quantize(nq, x, fmt, stride)
        cc, ss, gg = quantize(nq, x.contiguous(), fmt)
        n = 40 * nq.mx4_row_bytes(x.shape[1])
        assert torch.equal(codes[:n], cc[:n]) and torch.equal(scales, ss) and (g is None or torch.equal(g, gg))


def dequantize(nq, codes, scales, g, rows, cols, fmt, bf16, stream=None):
    import torch
    out = torch.full((rows * cols + 8,), 99.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    nq.dequantize_rows_mx4(codes.data_ptr(), scales.data_ptr(), g.data_ptr() if g is not None else 0, out.data_ptr(),
                           nq.BF16 if bf16 else nq.F32, rows, cols, fmt, s)
    assert torch.all(out[rows * cols:] == 99.0)
    return out[:rows * cols].view(rows, cols)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", [(1, 1), (5, 17), (129, 130), (300, 511), (64, 4096), (2, 20008), (260, 8)])
def test_dequantize(nq, fmt, bf16, shape):
    import torch
    rows, cols = shape
    x = np.random.default_rng(cols).standard_normal(shape)
    codes, scales, g = R.pack(x, fmt)
    dev = lambda a: torch.from_numpy(a).cuda()
    got = dequantize(nq, dev(codes), dev(scales), None if g is None else dev(g), rows, cols, fmt, bf16)
    ref = R.values(codes, scales, rows, cols, fmt) * (1.0 if g is None else g.astype(np.float64)[:, None])
    err = np.abs(got.double().cpu().numpy() - ref)
    assert np.all(err <= np.abs(ref) * (2.0 ** -24 + (2.0 ** -8 if bf16 else 0.0)))


def test_dequantize_every_scale_byte(nq):
    import torch
    for fmt, ref in ((R.MX, lambda b: np.where(b == 255, np.nan, np.ldexp(1.0, b - 127))), (R.NV, R.e4m3_of_byte)):
        n = R.BLOCK[fmt]
        codes = np.tile(np.array([0x10, 0x32, 0x54, 0x76, 0x98, 0xBA, 0xDC, 0xFE], np.uint8), 256 * n // 16)
        scales = np.zeros(R.words(256 * n, fmt) * 512, np.uint8)
        scales[R.scale_index(1, 256 * n, fmt)] = np.arange(256, dtype=np.uint8)[None]
        out = dequantize(nq, torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), None, 1, 256 * n, fmt, False)
        want = R.unpack_codes(codes, 1, 256 * n) * np.repeat(ref(np.arange(256)), n)[None]
        with np.errstate(over="ignore"):   # 6 * 2^127 is an infinity in fp32
            want = want.astype(np.float32).astype(np.float64)
        assert np.array_equal(out.double().cpu().numpy(), want, equal_nan=True)


# ---- the product ---------------------------------------------------------------------
def operand(rows, cols, fmt, seed, scale=1.0):
    """A quantized operand on the GPU and its doubles (without row scales)."""
    import torch
    x = np.random.default_rng(seed).standard_normal((rows, cols)) * scale
    codes, scales, g = R.pack(x, fmt)
    # rows of scales behind the last one hold what a NaN looks like: they must not matter
    used = np.zeros(scales.size, bool)
    used[R.scale_index(rows, cols, fmt)] = True
    scales[~used] = 0xFF if fmt == R.MX else 0x7F
    dev = lambda a: torch.from_numpy(a).cuda()
    return (dev(codes), dev(scales), None if g is None else dev(g)), R.values(codes, scales, rows, cols, fmt)


def product(nq, a, b, m, n, k, fmt, bf16, alpha=1.0, bias=None, out=None, stream=None):
    import torch
    out = torch.full((m * n + 16,), 99.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda") if out is None else out
    p = lambda t: 0 if t is None else t.data_ptr()
    d = nq.make_mx4_desc(m, n, k, fmt, nq.BF16 if bf16 else nq.F32, alpha, p(a[2]), p(b[2]), p(bias))
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    nq.gemm_mx4(C.byref(d), a[0].data_ptr(), a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(), out.data_ptr(), s)
    return out


def check_product(got, va, vb, a, b, k, bf16, alpha=1.0, bias=None):
    m, n = va.shape[0], vb.shape[0]
    f = alpha * (a[2].double().cpu().numpy()[:, None] if a[2] is not None else 1.0) * \
        (b[2].double().cpu().numpy()[None] if b[2] is not None else 1.0)
    ref = va @ vb.T * f
    tol = (np.abs(va) @ np.abs(vb).T) * np.abs(f) * ((k + 63) // 64 + 2) * 2.0 ** -22
    bb = 0.0 if bias is None else bias.double().cpu().numpy()[None]
    ref = ref + bb
    tol = tol + (np.abs(ref) + np.abs(bb)) * (4 * 2.0 ** -24 + (2.0 ** -8 if bf16 else 0.0)) + 1e-30
    err = np.abs(got[:m * n].view(m, n).double().cpu().numpy() - ref)
    assert np.all(err <= tol), f"worst {np.max(err / tol)} of the bound at {np.unravel_index(np.argmax(err / tol), err.shape)}"
    assert bool((got[m * n:] == 99.0).all()), "written behind the output"


GEMM_SHAPES = [(1, 1, 1), (1, 64, 32), (3, 5, 17), (16, 128, 64), (17, 130, 96), (33, 257, 100), (64, 512, 256),
               (65, 300, 320), (128, 128, 2048), (129, 129, 33), (200, 1000, 1111), (256, 256, 512), (300, 520, 1000),
               (257, 1024, 4096), (512, 96, 640), (1000, 300, 48), (2, 4096, 8192), (40, 8000, 5000), (130, 33, 20000),
               (16, 28672, 1024), (64, 16384, 1024), (600, 2304, 1536)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", GEMM_SHAPES)
def test_product(nq, fmt, bf16, shape):
    m, n, k = shape
    a, va = operand(m, k, fmt, m + k)
    b, vb = operand(n, k, fmt, n + k + 1, 0.05)
    got = product(nq, a, b, m, n, k, fmt, bf16)
    check_product(got, va, vb, a, b, k, bf16)
    assert nq.device_error_flags() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", [(20, 4096, 4096), (300, 700, 512)])
def test_product_epilogue(nq, fmt, shape):
    import torch
    m, n, k = shape
    a, va = operand(m, k, fmt, 1)
    b, vb = operand(n, k, fmt, 2)
    bias = torch.randn(n, device="cuda")
    rows, cols = torch.rand(m, device="cuda") + 0.5, torch.rand(n, device="cuda") + 0.5
    for sa, sb, bi in ((rows, None, None), (None, cols, bias), (rows, cols, bias), (None, None, bias), (None, None, None)):
        aa, bb = (a[0], a[1], sa), (b[0], b[1], sb)
        check_product(product(nq, aa, bb, m, n, k, fmt, False, -0.37, bi), va, vb, aa, bb, k, False, -0.37, bi)


def test_product_of_nothing_is_the_bias(nq):
    import torch
    bias = torch.randn(70, device="cuda")
    z = torch.zeros(512, dtype=torch.uint8, device="cuda")
    for fmt in FMTS:
        out = product(nq, (z, z, None), (z, z, None), 9, 70, 0, fmt, False, 1.0, bias)
        assert torch.equal(out[:630].view(9, 70), bias.expand(9, 70))


@pytest.mark.parametrize("shape", [(20, 4096, 4096), (300, 700, 512)])
def test_product_nan_stays_in_its_row(nq, shape):
    import torch
    m, n, k = shape
    for fmt in FMTS:
        a, _ = operand(m, k, fmt, 1)
        b, _ = operand(n, k, fmt, 2)
        a[1][R.scale_index(m, k, fmt)[7, 3]] = 0xFF if fmt == R.MX else 0x7F
        b[1][R.scale_index(n, k, fmt)[11, 0]] = 0xFF if fmt == R.MX else 0x7F
        out = torch.isnan(product(nq, a, b, m, n, k, fmt, False)[:m * n].view(m, n))
        want = torch.zeros(m, n, dtype=torch.bool, device="cuda")
        want[7], want[:, 11] = True, True
        assert torch.equal(out, want)


def test_product_unaligned_output(nq):
    import torch
    for m, n in ((20, 4096), (300, 704)):
        a, va = operand(m, 512, R.NV, 1)
        b, vb = operand(n, 512, R.NV, 2)
        for bf16 in (True, False):
            whole = torch.full((m * n + 17,), 99.0, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
            got = product(nq, a, b, m, n, 512, R.NV, bf16, out=whole[1:])
            check_product(got, va, vb, a, b, 512, bf16)
            assert whole[0] == 99.0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", [(16, 8192, 8192), (64, 28672, 2048), (700, 1024, 2048)])
def test_product_repeats_bit_for_bit(nq, fmt, shape):
    """Two streams at once, and the same call again: the order of the sums is fixed, and calls do not share state."""
    import torch
    m, n, k = shape
    a, _ = operand(m, k, fmt, 1)
    b, _ = operand(n, k, fmt, 2)
    first = product(nq, a, b, m, n, k, fmt, False)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(first) for _ in range(4)] for _ in streams]
    torch.cuda.synchronize()
    for i in range(4):
        for s, o in zip(streams, outs):
            o[i].fill_(99.0)  # on the current stream: ordered below
    torch.cuda.synchronize()
    for i in range(4):
        for s, o in zip(streams, outs):
            product(nq, a, b, m, n, k, fmt, False, out=o[i], stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for os in outs for o in os)
    assert nq.device_error_flags() == 0


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 16, 300])
def test_linear_captured_and_replayed(nq, fmt, m):
    """quantize -> product, eager, in a graph, and two graphs of the same buffers' shapes replayed at once."""
    import torch
    n, k = 8192, 4096
    b, _ = operand(n, k, fmt, 2)
    xs = [make(m, k, 30 + i, True) for i in range(3)]

    class Layer:
        def __init__(self):
            self.x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
            self.q = buffers(nq, m, k, fmt, 0)
            self.out = torch.full((m * n,), 99.0, dtype=torch.bfloat16, device="cuda")

        def run(self):
            s = torch.cuda.current_stream().cuda_stream
            g = self.q[2].data_ptr() if self.q[2] is not None else 0
            nq.quantize_rows_mx4(self.x.data_ptr(), nq.BF16, 0, self.q[0].data_ptr(), self.q[1].data_ptr(), g, m, k, fmt, s)
            product(nq, self.q, b, m, n, k, fmt, True, out=self.out)

    layers = [Layer(), Layer()]
    refs = []
    for x in xs:
        layers[0].x.copy_(x)
        layers[0].run()
        refs.append(layers[0].out.clone())
    torch.cuda.synchronize()
    graphs = []
    for l in layers:
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            l.run()
        graphs.append(gph)
    side = torch.cuda.Stream()
    for i in range(3):
        layers[0].x.copy_(xs[i])
        layers[1].x.copy_(xs[(i + 1) % 3])
        torch.cuda.synchronize()
        for _ in range(3):
            graphs[0].replay()
            with torch.cuda.stream(side):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(layers[0].out, refs[i]) and torch.equal(layers[1].out, refs[(i + 1) % 3])
    layers[0].x.copy_(xs[2])
    layers[0].run()
    torch.cuda.synchronize()
    assert torch.equal(layers[0].out, refs[2]) and nq.device_error_flags() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_shared_out_product_captured_and_replayed(nq, fmt):
    """Few rows against a long K (k-blocks of a unit on several CTAs, parts through a workspace): two graphs
    replayed at once beside eager calls give the eager result."""
    import torch
    m, n, k = 4, 4096, 28672
    w = make(n, k, 1, True, 0.02)
    b = buffers(nq, n, k, fmt, 0)
    x = make(m, k, 2, True)
    a = buffers(nq, m, k, fmt, 0)
    s = torch.cuda.current_stream().cuda_stream
    for t, q, rows in ((w, b, n), (x, a, m)):
        nq.quantize_rows_mx4(t.data_ptr(), nq.BF16, 0, q[0].data_ptr(), q[1].data_ptr(), q[2].data_ptr() if q[2] is not None else 0,
                             rows, k, fmt, s)
    a, b = [(q[0], q[1], None if q[2] is None else q[2][:r].contiguous()) for q, r in ((a, m), (b, n))]
    ref = product(nq, a, b, m, n, k, fmt, False)
    va, vb = (R.values(q[0].cpu().numpy(), q[1].cpu().numpy(), r, k, fmt) for q, r in ((a, m), (b, n)))
    check_product(ref, va, vb, a, b, k, False)
    outs = [torch.full_like(ref, 99.0) for _ in range(3)]
    graphs = []
    for o in outs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                product(nq, a, b, m, n, k, fmt, False, out=o)
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(4):
        for o in outs:
            o.fill_(99.0)
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        product(nq, a, b, m, n, k, fmt, False, out=outs[2])
        torch.cuda.synchronize()
        assert all(torch.equal(o, ref) for o in outs)
    assert nq.device_error_flags() == 0


@pytest.mark.parametrize("fmt", FMTS)
def test_quantize_past_32_bits(nq, fmt):
    """More than 2^32 bytes of input and 2^31 elements: the last rows equal the same rows quantized alone."""
    import torch
    rows, cols, tail = 36000, 65536, 300
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for r in range(0, rows, 4000):
        x[r:r + 4000] = make(min(4000, rows - r), cols, r, True)
    codes, scales, g = quantize(nq, x, fmt)
    first = rows // 128 * 128 - 256
    cc, ss, gg = quantize(nq, x[first:], fmt)
    n, pitch = rows - first, nq.mx4_row_bytes(cols)
    assert torch.equal(codes[first * pitch:rows * pitch], cc[:n * pitch])
    at = first // 128 * R.words(cols, fmt) * 512
    idx = torch.from_numpy(R.scale_index(n, cols, fmt)).cuda()
    assert torch.equal(scales[at:][idx], ss[idx])
    if g is not None:
        assert torch.equal(g[first:rows], gg[:n])
    out = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    nq.dequantize_rows_mx4(codes.data_ptr(), scales.data_ptr(), g.data_ptr() if g is not None else 0, out.data_ptr(), nq.BF16, rows, cols,
                           fmt, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(out[first:], dequantize(nq, cc, ss, gg, n, cols, fmt, True))
    assert (out[first:].float() - x[first:].float()).norm() < 0.2 * x[first:].float().norm()


def test_two_threads_at_once(nq):
    """Two host threads, each with its stream, buffers and shapes, through quantize and every kind of product."""
    import threading
    import torch
    jobs = [(R.NV, [(4, 4096, 14336), (300, 1000, 1024), (40, 2048, 512)]), (R.MX, [(16, 8192, 8192), (70, 700, 640), (2, 512, 16384)])]
    failed = []

    def work(fmt, shapes):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                layers = []
                for m, n, k in shapes:
                    w, x = make(n, k, m + n, True, 0.02), make(m, k, k, True)
                    b, a = buffers(nq, n, k, fmt, 0), buffers(nq, m, k, fmt, 0)
                    s = stream.cuda_stream
                    p = lambda t: t.data_ptr() if t is not None else 0
                    nq.quantize_rows_mx4(w.data_ptr(), nq.BF16, 0, p(b[0]), p(b[1]), p(b[2]), n, k, fmt, s)
                    layers.append((m, n, k, x, a, b, w))

                def step(m, n, k, x, a, b):
                    nq.quantize_rows_mx4(x.data_ptr(), nq.BF16, 0, p(a[0]), p(a[1]), p(a[2]), m, k, fmt, s)
                    return product(nq, a, b, m, n, k, fmt, False, stream=s)

                refs = []
                for l in layers:
                    refs.append(step(*l[:6]))
                    stream.synchronize()
                for _ in range(30):
                    outs = [step(*l[:6]) for l in layers]
                    stream.synchronize()
                    if not all(torch.equal(o, r) for o, r in zip(outs, refs)):
                        failed.append(fmt)
                for (m, n, k, x, _, _, w), r in zip(layers, refs):
                    want = x.double() @ w.double().t()
                    if ((r[:m * n].view(m, n) - want).norm() / want.norm()).item() > 0.25:
                        failed.append((m, n, k))
        except Exception as e:
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    torch.cuda.synchronize()
    assert not failed and nq.device_error_flags() == 0


FIRST_CALL = """
import ctypes as C, sys, torch
import nova_b200.capi as nq
x, w = torch.randn(600, 4096, device="cuda").bfloat16(), torch.randn(4096, device="cuda").bfloat16()
u8 = lambda n: torch.zeros(n, dtype=torch.uint8, device="cuda")
codes, scales, g = u8(600 * nq.mx4_row_bytes(16384)), u8(nq.mx4_scale_bytes(600, 16384, 1)), torch.ones(600, device="cuda")
out, dx, dw = torch.empty(600, 600, device="cuda"), torch.empty_like(x), torch.full((4096,), 7.0, device="cuda")
norm = nq.make_rmsnorm_desc(600, 4096, nq.BF16, nq.BF16, 1e-5)
gemm = nq.make_mx4_desc(4, 256, 16384, 1, nq.F32, 1.0)
p = lambda t: t.data_ptr()

def go():
    s = torch.cuda.current_stream().cuda_stream
    if sys.argv[1] == "norm":
        nq.rmsnorm_quantize_mx4(C.byref(norm), p(x), 0, p(w), 0, p(dx), p(codes), p(scales), p(g), 1, s)
    elif sys.argv[1] == "backward":
        nq.rmsnorm_backward(C.byref(norm), p(x), p(w), p(x), 0, p(dx), p(dw), s)
    elif sys.argv[1] == "quantize":
        nq.quantize_rows_mx4(p(x), nq.BF16, 0, p(codes), p(scales), p(g), 600, 4096, 1, s)
    else:
        nq.gemm_mx4(C.byref(gemm), p(codes), p(scales), p(codes), p(scales), p(out), s)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    go()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (codes, scales, g, out[:4], dx, dw)]
go()
torch.cuda.synchronize()
assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, (codes, scales, g, out[:4], dx, dw)))
assert nq.device_error_flags() == 0
print("captured")
"""


@pytest.mark.parametrize("what", ["norm", "backward", "quantize", "product"])
def test_first_call_of_a_process_captured(nq, what):
    """The library's first call may already be inside a capture (its pool is then created there)."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, what], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("m,n,k", [(300, 700, 512), (4, 4096, 28672), (8, 64, 64)])
def test_first_call_of_a_thread(nq, m, n, k):
    """A product as the first CUDA call that a host thread makes."""
    import threading
    import torch
    a, _ = operand(m, k, R.NV, 1)
    b, _ = operand(n, k, R.NV, 2)
    i8 = lambda r, c: torch.randint(-127, 128, (r, c), dtype=torch.int8, device="cuda")
    ia, ib = i8(m, k), i8(n, k)
    ref = product(nq, a, b, m, n, k, R.NV, False)
    outs = [torch.empty(m, n, device="cuda") for _ in range(2)]
    gemm = nq.make_desc(m, n, k, nq.INT8, nq.INT8, nq.B_NK, nq.F32, 1.0)
    eight = lambda o, s: nq.gemm(C.byref(gemm), ia.data_ptr(), ib.data_ptr(), o.data_ptr(), s)
    s = torch.cuda.current_stream().cuda_stream
    eight(outs[0], s)
    out = torch.full_like(ref, 99.0)
    torch.cuda.synchronize()
    failed = []

    def work(call):
        try:
            call()
        except Exception as e:
            failed.append(repr(e))

    for call in (lambda: product(nq, a, b, m, n, k, R.NV, False, out=out, stream=s), lambda: eight(outs[1], s)):
        t = threading.Thread(target=work, args=(call,))
        t.start()
        t.join(60)
    torch.cuda.synchronize()
    assert not failed and torch.equal(out, ref) and torch.equal(*outs)


def shared_out_operands(nq, m, n, k):
    """Quantized operands of a product whose k-blocks are shared out over the CTAs."""
    import torch
    ops = []
    for rows, seed in ((m, 2), (n, 1)):
        q = buffers(nq, rows, k, R.NV, 0)
        x = make(rows, k, seed, True, 0.1)
        nq.quantize_rows_mx4(x.data_ptr(), nq.BF16, 0, q[0].data_ptr(), q[1].data_ptr(), q[2].data_ptr(), rows, k, R.NV,
                             torch.cuda.current_stream().cuda_stream)
        ops.append((q[0], q[1], q[2][:rows].contiguous()))
    torch.cuda.synchronize()
    return ops


def test_shared_out_product_on_the_per_thread_stream(nq):
    """cudaStreamPerThread is one handle and another stream in every thread: two threads that pass it share no flags."""
    import threading
    import torch
    m, n, k = 4, 4096, 28672
    a, b = shared_out_operands(nq, m, n, k)
    ref = product(nq, a, b, m, n, k, R.NV, False)
    outs = [[torch.full_like(ref, 99.0) for _ in range(40)] for _ in range(2)]
    torch.cuda.synchronize()
    failed, both = [], threading.Barrier(2)

    def work(mine):
        try:
            both.wait(60)
            for o in mine:
                product(nq, a, b, m, n, k, R.NV, False, out=o, stream=2)   # cudaStreamPerThread
            torch.cuda.synchronize()
        except Exception as e:
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    torch.cuda.synchronize()
    assert not failed and all(torch.equal(o, ref) for mine in outs for o in mine)
    assert nq.device_error_flags() == 0


def test_shared_out_product_on_streams_without_end(nq):
    """Streams destroyed with their work in flight, whose handles come back: every one counts as a new one; behind the
    first thousand a launch brings its own flags."""
    import torch
    m, n, k = 2, 512, 16384
    a, b = shared_out_operands(nq, m, n, k)
    ref = product(nq, a, b, m, n, k, R.NV, False)
    outs = [torch.full_like(ref, 99.0) for _ in range(1200)]
    torch.cuda.synchronize()
    rt, handles = torch.cuda.cudart(), set()
    for o in outs:
        h = C.c_void_p()
        assert int(rt.cudaStreamCreate(C.addressof(h))) == 0
        handles.add(h.value)
        product(nq, a, b, m, n, k, R.NV, False, out=o, stream=h.value)
        assert int(rt.cudaStreamDestroy(h.value)) == 0
    torch.cuda.synchronize()
    assert len(handles) < len(outs)   # (handles did come back)
    assert all(torch.equal(o, ref) for o in outs) and nq.device_error_flags() == 0


# several 256 x 256 tiles a cluster (74 of them on 148 SMs): whole rounds and a tail of half tiles (171 tiles), a
# remainder of more than half the clusters (112, ragged, rows of the output not whole 16 bytes), more than one band of
# 32 row tiles (165), more than two rounds with a short K (285)
MANY_TILES = [(2304, 4864, 600), (1700, 4001, 2100), (8400, 1100, 320), (3700, 4700, 40)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", MANY_TILES)
def test_product_of_many_tiles(nq, fmt, bf16, shape):
    """Accumulators, scale words and stages handed from tile to tile; the same again, bit for bit."""
    import torch
    m, n, k = shape
    a, va = operand(m, k, fmt, m + k)
    b, vb = operand(n, k, fmt, n + k + 1, 0.05)
    bias = torch.randn(n, device="cuda")
    got = product(nq, a, b, m, n, k, fmt, bf16, 0.75, bias)
    check_product(got, va, vb, a, b, k, bf16, 0.75, bias)
    for _ in range(3):
        assert torch.equal(product(nq, a, b, m, n, k, fmt, bf16, 0.75, bias), got)
    plain = (a[0], a[1], None), (b[0], b[1], None)
    got = product(nq, *plain, m, n, k, fmt, bf16)
    check_product(got, va, vb, *plain, k, bf16)
    assert nq.device_error_flags() == 0
