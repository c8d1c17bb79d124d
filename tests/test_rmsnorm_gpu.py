"""RMS norm with the residual's addition and a quantized output, and its
gradient, against 64-bit references (tests/mx4_ref.py).

Tolerances (u = 2^-24, one fp32 rounding):
- h is one rounding of an exact sum: equal to the reference's.
- sum(h^2): products rounded once, added over at most cols / 32 + 32 additions
  in a thread, a warp and a block (all terms positive), so r is within
  R = (cols / 32 + 34) / 2 u + 2 u, and y = t r within R + 2 u, plus the
  type's rounding.
- 8-bit scales r T / qmax: R + 4 u.  A code is the nearest value of a quotient
  t qmax / T whose t, T and division are rounded, so its distance from the exact
  quotient is half a step plus 4 u |q|.  For bf16 tensors t is exact and the codes are the
  correctly rounded ones, value for value.
- NVFP4 codes are compared like those of fp32 values (scales 2^-20, codes 2^-17);
  t itself is a rounded product (u of it): 2^-19 and 2^-16 (|q| <= 9).
  MXFP4 codes of y: y within R + 2 u, so a border moves by 8 (R + 2 u), and a block's
  power of two may change where its maximum is that near one.
- gradients: g = dy w (u); mean(g h) has R' = (cols / 32 + 34) u of mean|g h|; each output
  few roundings: |error| <= 2 R' (|r g| + |h| r^3 mean|g h|) + 2 u |dsum|;
  the weight's: rows additions in at most rows / 1 + 64 roundings: (rows + 70 + 2 R / u) u sum|dy h r|."""
import ctypes as C

import numpy as np
import pytest

import mx4_ref as R

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
E4M3, E5M2, INT8 = 0, 1, 2
EPS = 1e-5


@pytest.fixture(scope="module")
def nq(cuda):
    import nova_b200.capi as capi
    return capi


def rand(rows, cols, seed, bf16, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, device="cuda", generator=g) * scale
    return x.to(torch.bfloat16) if bf16 else x


def ptr(t):
    return 0 if t is None else t.data_ptr()


def tol_r(cols):
    return (cols / 32 + 34) / 2 * U + 2 * U


def code_values(codes, fmt):
    import torch
    if fmt == INT8:
        return codes.view(torch.int8).double().cpu().numpy()
    return codes.view(torch.float8_e4m3fn if fmt == E4M3 else torch.float8_e5m2).double().cpu().numpy()


def half_step(q, fmt):
    """Half the distance between the codes around |q|."""
    if fmt == INT8:
        return 0.5
    bits, low = (3, -6) if fmt == E4M3 else (2, -14)
    _, e = np.frexp(np.maximum(np.abs(q), 2.0 ** low))
    return np.ldexp(0.5, e - 1 - bits)


def check_codes8(codes, scales, t, r, cols, fmt, exact=False):
    T = np.abs(t).max(1)
    level = np.maximum(T, 2.0 ** -110)
    want = np.where(T > 0, r * level / R.QMAX[fmt], 1.0)
    s = scales.double().cpu().numpy()
    assert np.all(np.abs(s - want) <= want * (tol_r(cols) + 4 * U))
    q = t * R.QMAX[fmt] / level[:, None]   # one rounding of exact products: borders stay borders
    got = code_values(codes, fmt)
    if exact:
        bits = {E4M3: (3, -6), E5M2: (2, -14)}
        if fmt == INT8:
            want_q = np.rint(q)
        else:
            mant, low = bits[fmt]
            _, e = np.frexp(np.maximum(np.abs(q), 2.0 ** low))
            s = np.ldexp(1.0, e - 1 - mant)
            want_q = np.rint(q / s) * s
        assert np.array_equal(got, want_q)
    # at the edge above a power of two the step doubles: take the wider one
    step = np.maximum(half_step(q, fmt), half_step(q * (1 + 8 * U), fmt))
    assert np.all(np.abs(got - q) <= step + 4 * U * np.abs(q))


def check_mx4(nq, buf, t, r, rows, cols, fmt):
    codes, scales, g = (None if b is None else b.cpu().numpy() for b in buf)
    s = R.unpack_scales(scales, rows, cols, fmt)
    got = R.unpack_codes(codes, rows, cols)
    assert np.all(got[:, cols:] == 0)
    rel = 8 * (tol_r(cols) + 2 * U)
    if fmt == R.MX:
        x = t * r[:, None]
        _, lo, _ = R.quantize(x * (1 - rel), fmt)
        _, hi, _ = R.quantize(x * (1 + rel), fmt)
        assert np.all((s == lo) | (s == hi))
        q, slack = R.blocks(x, fmt) / s[..., None], 8 * rel
    else:
        top = np.abs(R.blocks(t, fmt)).max(-1)
        level = np.maximum(top.max(1, keepdims=True), 2688.0 * 2.0 ** -110)
        v = 448.0 * top / level
        assert np.all((s == R.e4m3(v * (1 - 2.0 ** -19))) | (s == R.e4m3(v)) | (s == R.e4m3(v * (1 + 2.0 ** -19))))
        want = np.where(top.max(1) > 0, r * level[:, 0] / 2688.0, 1.0)
        assert np.all(np.abs(g - want) <= want * (tol_r(cols) + 4 * U))
        d = (s * level)[..., None]
        q, slack = np.where(d > 0, 2688.0 * R.blocks(t, fmt) / np.where(d > 0, d, 1.0), 0.0), 2.0 ** -16
    w = q.shape[1] * q.shape[2]
    got = np.pad(got, ((0, 0), (0, max(0, w - got.shape[1]))))[:, :w].reshape(q.shape)
    ok = (got == R.e2m1(q)) | (got == R.e2m1(q - slack)) | (got == R.e2m1(q + slack))
    assert ok.all()


def run(nq, x, res, w, fmt, four=False, sum=None, want_y=True, want_codes=True, xs=0, rs=0, stream=None):
    import torch
    rows, cols = x.shape
    bf = x.dtype == torch.bfloat16
    y = torch.full((rows * cols + 8,), 9.0, dtype=x.dtype, device="cuda") if want_y else None
    if four:
        u8 = lambda n: torch.full((n,), 0xAA, dtype=torch.uint8, device="cuda")
        codes, bs = u8(rows * nq.mx4_row_bytes(cols)), u8(nq.mx4_scale_bytes(rows, cols, fmt))
    else:
        codes, bs = torch.full((rows * cols + 8,), 0xAA, dtype=torch.uint8, device="cuda"), None
    g = torch.full((rows + 4,), -7.0, device="cuda") if not (four and fmt == R.MX) else None
    if not want_codes:
        codes = bs = g = None
    d = nq.make_rmsnorm_desc(rows, cols, nq.BF16 if bf else nq.F32, nq.BF16 if w.dtype == torch.bfloat16 else nq.F32, EPS, xs, rs)
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    if four:
        nq.rmsnorm_quantize_mx4(C.byref(d), ptr(x), ptr(res), ptr(w), ptr(sum), ptr(y), ptr(codes), ptr(bs), ptr(g), fmt, s)
    else:
        nq.rmsnorm_quantize(C.byref(d), ptr(x), ptr(res), ptr(w), ptr(sum), ptr(y), ptr(codes), ptr(g), fmt, s)
    torch.cuda.synchronize()
    if y is not None:
        assert torch.all(y[rows * cols:] == 9.0)
        y = y[:rows * cols].view(rows, cols)
    if codes is not None and not four:
        assert torch.all(codes[rows * cols:] == 0xAA)
        codes = codes[:rows * cols].view(rows, cols)
    if g is not None:
        assert torch.all(g[rows:] == -7.0)
        g = g[:rows]
    return y, codes, bs, g


def reference_h(x, res):
    h = x.double() if res is None else (x.double() + res.double())
    h = h.cpu().numpy()
    return R.bf16(h) if str(x.dtype) == "torch.bfloat16" and res is not None else h.astype(np.float32).astype(np.float64)


def check_y(y, t, r, cols):
    ref = t * r[:, None]
    half = 2.0 ** -8 if str(y.dtype) == "torch.bfloat16" else 0.0
    assert np.all(np.abs(y.double().cpu().numpy() - ref) <= np.abs(ref) * (tol_r(cols) + 2 * U + half) + 1e-44)


SHAPES = [(1, 1), (1, 8192), (2, 7), (3, 64), (5, 130), (9, 1000), (300, 1024), (7, 1032), (130, 2048), (3, 2051), (40, 4096),
          (200, 8192), (5, 16384), (2, 16392), (2, 40000), (3, 33001), (2000, 96)]


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_eight_bits(nq, bf16, shape):
    import torch
    rows, cols = shape
    x, res = rand(rows, cols, 1, bf16), rand(rows, cols, 2, bf16, 3.0)
    w = rand(1, cols, 3, bf16).view(-1) + 1.0
    if rows > 2:
        x[1], res[1] = 0.0, 0.0
    for fmt in (E4M3, E5M2, INT8):
        for r_ in (res, None):
            s = torch.empty_like(x) if r_ is not None else None
            y, codes, _, scales = run(nq, x, r_, w, fmt, sum=s)
            h = reference_h(x, r_)
            if s is not None:
                assert np.array_equal(s.double().cpu().numpy(), h)
            t, r = R.rmsnorm(h, w.double().cpu().numpy(), EPS)
            check_y(y, t, r, cols)
            check_codes8(codes, scales, t, r, cols, fmt, exact=bf16)


@pytest.mark.parametrize("fmt", [R.MX, R.NV])
@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_four_bits(nq, fmt, bf16, shape):
    import torch
    rows, cols = shape
    x, res = rand(rows, cols, 1, bf16), rand(rows, cols, 2, bf16, 3.0)
    w = rand(1, cols, 3, bf16).view(-1) + 1.0
    s = torch.empty_like(x)
    y, codes, bs, g = run(nq, x, res, w, fmt, four=True, sum=s)
    h = reference_h(x, res)
    assert np.array_equal(s.double().cpu().numpy(), h)
    t, r = R.rmsnorm(h, w.double().cpu().numpy(), EPS)
    check_y(y, t, r, cols)
    check_mx4(nq, (codes, bs, g), t, r, rows, cols, fmt)
    y2, codes2, bs2, g2 = run(nq, x, res, w, fmt, four=True, want_y=False)   # no sum, no y: the same codes
    assert torch.equal(codes, codes2) and torch.equal(bs, bs2) and (g is None or torch.equal(g, g2))


def test_outputs_one_by_one(nq):
    import torch
    for cols in (4096, 4097, 20000):
        x, res, w = rand(6, cols, 1, True), rand(6, cols, 2, True), rand(1, cols, 3, False).view(-1)   # fp32 weight, bf16 rows
        s = torch.empty_like(x)
        y, codes, _, scales = run(nq, x, res, w, E4M3, sum=s)
        y1, c1, _, _ = run(nq, x, res, w, E4M3, want_codes=False)
        assert c1 is None and torch.equal(y, y1)
        y2, c2, _, s2 = run(nq, x, res, w, E4M3, want_y=False)
        assert y2 is None and torch.equal(codes, c2) and torch.equal(scales, s2)
        # the sum in place of either input
        for k in range(2):
            a, b = x.clone(), res.clone()
            y3, c3, _, s3 = run(nq, a, b, w, E4M3, sum=(a, b)[k])
            assert torch.equal((a, b)[k], s) and torch.equal((b, a)[k], (res, x)[k])
            assert torch.equal(y, y3) and torch.equal(codes, c3) and torch.equal(scales, s3)


@pytest.mark.parametrize("bf16", [True, False])
def test_strided_and_unaligned_rows(nq, bf16):
    import torch
    big, rbig = rand(20, 2100, 4, bf16), rand(20, 2200, 5, bf16)
    wb = rand(1, 2100, 6, bf16).view(-1)
    for lo, cols in ((0, 1024), (8, 1024), (4, 520), (3, 1024), (1, 77)):
        x, res, w = big[:, lo:lo + cols], rbig[:, lo:lo + cols], wb[lo:lo + cols]
        a = run(nq, x, res, w, E4M3, xs=2100, rs=2200)
        b = run(nq, x.contiguous(), res.contiguous(), w.clone(), E4M3)
        assert torch.equal(a[1], b[1])                     # codes and y do not depend on the path beyond
        assert np.all(np.abs((a[3] / b[3] - 1).cpu().numpy()) <= 2 * tol_r(cols))
        t, r = R.rmsnorm(reference_h(x, res), w.double().cpu().numpy(), EPS)
        check_y(a[0], t, r, cols)


def test_not_finite_and_zero_rows(nq):
    import torch
    for cols in (1024, 1001, 20000):
        x, w = rand(5, cols, 1, True), rand(1, cols, 2, True).view(-1)
        x[1, 3], x[2, 5], x[3] = float("nan"), float("inf"), 0.0
        y, codes, _, scales = run(nq, x, None, w, E4M3)
        assert torch.isnan(scales[[1, 2]]).all() and scales[3] == 1.0 and torch.isfinite(scales[[0, 4]]).all()
        assert torch.all(codes[3] & 127 == 0) and torch.all(y[3] == 0) and torch.isnan(y[1]).all()
        for fmt in (R.MX, R.NV):
            y, codes, bs, g = run(nq, x, None, w, fmt, four=True)
            if fmt == R.NV:
                assert torch.isnan(g[[1, 2]]).all() and g[3] == 1.0 and torch.isfinite(g[[0, 4]]).all()
            c = R.unpack_codes(codes.cpu().numpy(), 5, cols)
            s = R.unpack_scales(bs.cpu().numpy(), 5, cols, fmt)
            assert np.all(c[3] == 0) and np.isfinite(s[[0, 3, 4]]).all()
            if fmt == R.MX:   # the row's y is NaN all over for a NaN, and at the infinity for an infinity
                assert np.isnan(s[1, :(cols + 31) // 32]).all() and np.isnan(s[2, 0])


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", [(1, 1), (1, 64), (3, 7), (130, 2051), (70, 1024), (33, 4096), (1000, 520), (5, 8192), (6, 16384),
                                   (3, 16392), (2, 33001), (3000, 96), (700, 2048)])
def test_backward(nq, bf16, shape):
    import torch
    rows, cols = shape
    h, w = rand(rows, cols, 1, bf16, 2.0), rand(1, cols, 2, bf16).view(-1) + 1.0
    dy, dsum = rand(rows, cols, 3, bf16, 0.1), rand(rows, cols, 4, bf16, 0.1)
    d = nq.make_rmsnorm_desc(rows, cols, nq.BF16 if bf16 else nq.F32, nq.BF16 if bf16 else nq.F32, EPS)
    s = torch.cuda.current_stream().cuda_stream
    n64 = lambda t: None if t is None else t.double().cpu().numpy()
    for ds in (dsum, None):
        dx = torch.full((rows * cols + 8,), 9.0, dtype=h.dtype, device="cuda")
        dw = torch.full((cols + 4,), -7.0, device="cuda")
        nq.rmsnorm_backward(C.byref(d), ptr(h), ptr(w), ptr(dy), ptr(ds), ptr(dx), ptr(dw), s)
        rx, rw = R.rmsnorm_backward(n64(h), n64(w), n64(dy), n64(ds), EPS)
        assert torch.all(dx[rows * cols:] == 9.0) and torch.all(dw[cols:] == -7.0)
        g, r = n64(dy) * n64(w), R.rmsnorm(n64(h), 1.0, EPS)[1][:, None]
        mean = np.abs(g * n64(h)).mean(1, keepdims=True)
        rp = (cols / 32 + 34) * U
        tol = 2 * rp * (np.abs(r * g) + np.abs(n64(h)) * r ** 3 * mean) + (0 if ds is None else 2 * U * np.abs(n64(ds))) + 1e-44
        tol = tol + np.abs(rx) * (2.0 ** -8 if bf16 else 2 * U)
        assert np.all(np.abs(dx[:rows * cols].view(rows, cols).double().cpu().numpy() - rx) <= tol)
        tol = np.abs(n64(dy) * n64(h) * r).sum(0) * (rows + 70 + 2 * tol_r(cols) / U) * U + 1e-44
        assert np.all(np.abs(dw[:cols].double().cpu().numpy() - rw) <= tol)
        # one at a time, and in place of the residual stream's gradient
        dx2, dw2 = torch.empty(rows, cols, dtype=h.dtype, device="cuda"), torch.empty(cols, device="cuda")
        nq.rmsnorm_backward(C.byref(d), ptr(h), ptr(w), ptr(dy), ptr(ds), ptr(dx2), 0, s)
        nq.rmsnorm_backward(C.byref(d), ptr(h), ptr(w), ptr(dy), ptr(ds), 0, ptr(dw2), s)
        assert torch.equal(dx2.view(-1), dx[:rows * cols]) and torch.equal(dw2, dw[:cols])
        if ds is not None:
            ds2 = ds.clone()
            nq.rmsnorm_backward(C.byref(d), ptr(h), ptr(w), ptr(dy), ptr(ds2), ptr(ds2), ptr(dw2), s)
            assert torch.equal(ds2, dx2) and torch.equal(dw2, dw[:cols])


def test_backward_of_no_rows_and_strides(nq):
    import torch
    s = torch.cuda.current_stream().cuda_stream
    dw = torch.full((40,), 3.0, device="cuda")
    d = nq.make_rmsnorm_desc(0, 40, nq.BF16, nq.BF16, EPS)
    nq.rmsnorm_backward(C.byref(d), 0, 0, 0, 0, 0, ptr(dw), s)
    assert torch.all(dw == 0.0)
    big, w = rand(50, 700, 1, True), rand(1, 512, 2, True).view(-1)
    dy = rand(50, 512, 3, True)
    for lo in (0, 8, 3):
        h = big[:, lo:lo + 512]
        out = []
        for t, stride in ((h, 700), (h.contiguous(), 0)):
            dx, dw = torch.empty(50, 512, dtype=torch.bfloat16, device="cuda"), torch.empty(512, device="cuda")
            d = nq.make_rmsnorm_desc(50, 512, nq.BF16, nq.BF16, EPS, stride)
            nq.rmsnorm_backward(C.byref(d), ptr(t), ptr(w), ptr(dy), 0, ptr(dx), ptr(dw), s)
            out.append((dx, dw))
        scale = (out[1][0].abs().max().item(), out[1][1].abs().max().item())
        assert (out[0][0].float() - out[1][0].float()).abs().max().item() <= scale[0] * 2.0 ** -7
        assert (out[0][1] - out[1][1]).abs().max().item() <= scale[1] * 1e-4


def test_backward_captured_beside_eager(nq):
    """A captured backward replays to the eager results, while eager calls go on with the same leaves."""
    import torch
    rows, cols = 600, 2048
    h, w = rand(rows, cols, 1, True), rand(1, cols, 2, True).view(-1)
    dy = rand(rows, cols, 3, True)
    d = nq.make_rmsnorm_desc(rows, cols, nq.BF16, nq.BF16, EPS)
    bufs = [(torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda"), torch.empty(cols, device="cuda")) for _ in range(3)]
    go = lambda b: nq.rmsnorm_backward(C.byref(d), ptr(h), ptr(w), ptr(dy), 0, ptr(b[0]), ptr(b[1]),
                                       torch.cuda.current_stream().cuda_stream)
    go(bufs[0])
    torch.cuda.synchronize()
    graphs = []
    for b in bufs[1:]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(b)
        graphs.append(g)
    side = torch.cuda.Stream()
    for _ in range(3):
        for b in bufs[1:]:
            b[0].zero_(), b[1].zero_()
        torch.cuda.synchronize()
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        go(bufs[0])
        torch.cuda.synchronize()
        for b in bufs[1:]:
            assert torch.equal(b[0], bufs[0][0]) and torch.equal(b[1], bufs[0][1])


@pytest.mark.parametrize("tokens", [1, 16, 300])
def test_norm_to_product_layer(nq, tokens):
    """norm -> 4-bit product and norm -> INT8 product back to back, against the same layers step by step and in 64 bits."""
    import torch
    H, N = 4096, 8192
    x, res = rand(tokens, H, 1, True), rand(tokens, H, 2, True, 2.0)
    w = rand(1, H, 3, True, 0.1).view(-1) + 1.0
    s = torch.cuda.current_stream().cuda_stream
    wt = rand(N, H, 4, True, 0.02)
    t, r = R.rmsnorm(reference_h(x, res), w.double().cpu().numpy(), EPS)
    y64 = torch.from_numpy(t * r[:, None]).cuda()
    exact = y64 @ wt.double().t()
    for fmt in (R.MX, R.NV):
        u8 = lambda n: torch.empty(n, dtype=torch.uint8, device="cuda")
        wq, wsc, wg = u8(N * nq.mx4_row_bytes(H)), u8(nq.mx4_scale_bytes(N, H, fmt)), torch.empty(N, device="cuda") if fmt else None
        nq.quantize_rows_mx4(ptr(wt), nq.BF16, 0, ptr(wq), ptr(wsc), ptr(wg), N, H, fmt, s)
        out = torch.empty(tokens, N, dtype=torch.bfloat16, device="cuda")
        d = nq.make_rmsnorm_desc(tokens, H, nq.BF16, nq.BF16, EPS)
        cq, csc, cg = u8(tokens * nq.mx4_row_bytes(H)), u8(nq.mx4_scale_bytes(tokens, H, fmt)), torch.empty(tokens, device="cuda") if fmt else None
        sm = torch.empty_like(x)
        gd = nq.make_mx4_desc(tokens, N, H, fmt, nq.BF16, 1.0, ptr(cg), ptr(wg))
        for _ in range(3):
            cq.zero_()
            nq.rmsnorm_quantize_mx4(C.byref(d), ptr(x), ptr(res), ptr(w), ptr(sm), 0, ptr(cq), ptr(csc), ptr(cg), fmt, s)
            nq.gemm_mx4(C.byref(gd), ptr(cq), ptr(csc), ptr(wq), ptr(wsc), ptr(out), s)
        deq = lambda c, b, g, rows: R.values(c.cpu().numpy(), b.cpu().numpy(), rows, H, fmt) * (1.0 if g is None else g.double().cpu().numpy()[:, None])
        va, vb = (torch.from_numpy(deq(*v)).cuda() for v in ((cq, csc, cg, tokens), (wq, wsc, wg, N)))
        ref, mag = va @ vb.t(), va.abs() @ vb.abs().t()
        tol = mag * ((H // 64 + 2) * 2.0 ** -22) + ref.abs() * (2.0 ** -8 + 4 * U)
        assert torch.all((out.double() - ref).abs() <= tol)
        # two operands with 4-bit noise (relative rms about 0.1 each): near the unquantized layer
        assert ((out.double() - exact).norm() / exact.norm()).item() < 0.25
    # INT8 codes straight into the INT8 product
    codes, scales = torch.empty(tokens, H, dtype=torch.int8, device="cuda"), torch.empty(tokens, device="cuda")
    wi, ws = torch.empty(N, H, dtype=torch.int8, device="cuda"), torch.empty(N, device="cuda")
    nq.quantize_rows(ptr(wt), nq.BF16, ptr(wi), ptr(ws), N, H, nq.INT8, s)
    nq.rmsnorm_quantize(C.byref(d), ptr(x), ptr(res), ptr(w), ptr(sm), 0, ptr(codes), ptr(scales), nq.INT8, s)
    g = nq.make_desc(tokens, N, H, nq.INT8, nq.INT8, nq.B_NK, nq.BF16, 1.0, ptr(scales), ptr(ws))
    nq.gemm(C.byref(g), ptr(codes), ptr(wi), ptr(out), s)
    ref = (codes.double() @ wi.double().t()) * scales.double()[:, None] * ws.double()   # the integer sums are exact
    assert torch.all((out.double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 4 * U) + 1e-30)
    assert ((out.double() - exact).norm() / exact.norm()).item() < 0.03
    assert nq.device_error_flags() == 0


def test_norm_past_32_bits(nq):
    """More than 2^31 elements: the last rows equal the same rows alone, forward and backward."""
    import torch
    rows, cols = 270000, 8192
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for r in range(0, rows, 30000):
        x[r:r + 30000] = rand(min(30000, rows - r), cols, r, True)
    w = rand(1, cols, 1, True).view(-1)
    last = slice(rows - 1000, rows)
    y, codes, _, scales = run(nq, x, None, w, E4M3, want_y=False)
    _, c, _, sc = run(nq, x[last], None, w, E4M3, want_y=False)
    assert torch.equal(codes[last], c) and torch.equal(scales[last], sc)
    del codes, scales
    dx = torch.empty_like(x)
    s = torch.cuda.current_stream().cuda_stream
    d = nq.make_rmsnorm_desc(rows, cols, nq.BF16, nq.BF16, EPS)
    nq.rmsnorm_backward(C.byref(d), ptr(x), ptr(w), ptr(x), 0, ptr(dx), 0, s)
    dx1 = torch.empty(1000, cols, dtype=torch.bfloat16, device="cuda")
    d = nq.make_rmsnorm_desc(1000, cols, nq.BF16, nq.BF16, EPS)
    xl = x[last].clone()
    nq.rmsnorm_backward(C.byref(d), ptr(xl), ptr(w), ptr(xl), 0, ptr(dx1), 0, s)
    assert torch.equal(dx[last], dx1)


@pytest.mark.parametrize("bf16", [True, False])
def test_dense_unaligned_base(nq, bf16):
    """Dense odd-width rows whose tensors start off a 16-byte boundary, all by the same or by different distances."""
    import torch
    rows, cols = 37, 1003
    n = rows * cols
    flat = lambda seed, off: rand(1, n + 8, seed, bf16).view(-1)[off:off + n].view(rows, cols)
    w = rand(1, cols, 9, bf16).view(-1)
    for offs in ((0, 0, 0), (3, 3, 3), (3, 1, 0), (8, 0, 5)):
        x, res = flat(1, offs[0]), flat(2, offs[1])
        whole = torch.full((n + 16,), 7.0, dtype=x.dtype, device="cuda")
        sm = whole[offs[2]:offs[2] + n].view(rows, cols)
        y, codes, _, scales = run(nq, x, res, w, E4M3, sum=sm)
        h = reference_h(x, res)
        assert np.array_equal(sm.double().cpu().numpy(), h)
        assert torch.all(whole[:offs[2]] == 7.0) and torch.all(whole[offs[2] + n:] == 7.0)
        t, r = R.rmsnorm(h, w.double().cpu().numpy(), EPS)
        check_y(y, t, r, cols)
        check_codes8(codes, scales, t, r, cols, E4M3)


def product32(h, w):
    """t = h w as fp32 rounds it (a double holds the exact product of two fp32 values)."""
    return (h * w).astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", [(9, 96), (9, 1024), (9, 1003), (700, 2048), (3, 40000), (2, 33001)])
@pytest.mark.parametrize("scale", [1e-36, 1e-30, 1e30, 3e37])
def test_eight_bits_of_extreme_weights(nq, bf16, shape, scale):
    """Finite rows of any magnitude of h w have the codes of t qmax / T: nothing on the way leaves fp32's range."""
    import torch
    rows, cols = shape
    x, w = rand(rows, cols, 1, bf16).clamp(-4, 4), (rand(1, cols, 2, False).view(-1).clamp(-2, 2) * scale)
    w = w.to(x.dtype)
    if scale < 1:   # a row of both ends
        x[:, 0], w[0] = 0.0, 1.0
        x[1, 0] = 1.0
    h, w64 = reference_h(x, None), w.double().cpu().numpy()
    t, r = product32(h, w64), R.rmsnorm(h, 1.0, EPS)[1]
    assert np.isfinite(t).all()
    for fmt in (E4M3, E5M2, INT8):
        _, codes, _, scales = run(nq, x, None, w, fmt, want_y=False)
        check_codes8(codes, scales, t, r, cols, fmt, exact=bf16)


def far_rows(x, scale):
    """Rows of finite values whose squares leave fp32's range: all of them, and one column alone."""
    x = x.clamp(-4, 4) * scale
    x[1] /= scale
    x[1, 3] = scale
    return x


# widths and heights of every forward kernel: a warp a row, a block a row, many rows, odd widths, wide ones
FAR_SHAPES = [(9, 96), (9, 77), (9, 1024), (9, 1003), (700, 2048), (3, 40000), (3, 33001)]


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", FAR_SHAPES)
@pytest.mark.parametrize("scale", [1e20, 1e30, 5e37])
def test_rows_whose_squares_overflow(nq, bf16, shape, scale):
    """sum(h^2) beyond fp32: r, y and the scales are those of the formula, for any finite row.

    Squares of h 2^-80: the same roundings as in range; a subnormal r (rms above 2^126) or y is off by 2^-150 more
    (2^-134 for a bf16 y)."""
    import torch
    rows, cols = shape
    x = far_rows(rand(rows, cols, 1, bf16), scale)
    res = rand(rows, cols, 2, bf16)
    w = (rand(1, cols, 3, False).view(-1).clamp(-0.4, 0.4) + 1.0).to(x.dtype)
    w64 = w.double().cpu().numpy()
    for r_, with_sum in ((None, False), (res, False), (res, True)):
        s = torch.empty_like(x) if with_sum else None
        h = reference_h(x, r_)
        t, r = product32(h, w64), R.rmsnorm(h, 1.0, EPS)[1]
        assert np.isfinite(t).all()
        for fmt in (E4M3, E5M2, INT8):
            y, codes, _, scales = run(nq, x, r_, w, fmt, sum=s)
            check_codes8(codes, scales, t, r, cols, fmt, exact=bf16)
            assert s is None or np.array_equal(s.double().cpu().numpy(), h)
        ref = t * r[:, None]
        half, low = (2.0 ** -8, 2.0 ** -134) if bf16 else (0.0, 2.0 ** -150)
        assert np.all(np.abs(y.double().cpu().numpy() - ref) <= np.abs(ref) * (tol_r(cols) + 2 * U + half) + 2 * low)
        for fmt in (R.MX, R.NV):
            _, codes, bs, g = run(nq, x, r_, w, fmt, four=True, sum=s, want_y=False)
            check_mx4(nq, (codes, bs, g), t, r, rows, cols, fmt)
    for bad in (float("inf"), float("nan")):   # a row that is not finite beside them
        x[2, 5] = bad
        y, codes, _, scales = run(nq, x, None, w, E4M3)
        assert torch.isnan(scales[2]) and torch.isfinite(scales[[0, 1]]).all() and torch.isnan(y[2, 5])


def check_backward(nq, h, w, dy, ds, eps):
    """Gradients against the formula's in 64 bits, within the roundings of the module's head."""
    import torch
    rows, cols = h.shape
    bf16 = h.dtype == torch.bfloat16
    dx, dw = torch.empty_like(h), torch.empty(cols, device="cuda")
    d = nq.make_rmsnorm_desc(rows, cols, nq.BF16 if bf16 else nq.F32, nq.BF16 if bf16 else nq.F32, eps)
    nq.rmsnorm_backward(C.byref(d), ptr(h), ptr(w), ptr(dy), ptr(ds), ptr(dx), ptr(dw), torch.cuda.current_stream().cuda_stream)
    n64 = lambda t: None if t is None else t.double().cpu().numpy()
    rx, rw = R.rmsnorm_backward(n64(h), n64(w), n64(dy), n64(ds), d.eps)
    g, r = n64(dy) * n64(w), R.rmsnorm(n64(h), 1.0, d.eps)[1][:, None]
    rp = (cols / 32 + 34) * U
    tol = 2 * rp * (np.abs(r * g) + np.abs(n64(h)) * r ** 3 * np.abs(g * n64(h)).mean(1, keepdims=True))
    tol = tol + (0 if ds is None else 2 * U * np.abs(n64(ds))) + np.abs(rx) * (2.0 ** -8 if bf16 else 2 * U)
    tol = tol + (2.0 ** -133 if bf16 else 2.0 ** -147)   # subnormal results and products
    assert np.all(np.abs(n64(dx) - rx) <= tol)
    tol = np.abs(n64(dy) * n64(h) * r).sum(0) * (rows + 70 + 2 * tol_r(cols) / U) * U + rows * 2.0 ** -147
    assert np.all(np.abs(n64(dw) - rw) <= tol)


# widths and heights of every gradient kernel
GRAD_SHAPES = [(9, 96), (9, 77), (200, 1024), (9, 1003), (5, 8192), (3, 16384), (3, 33001), (3, 40000)]


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", GRAD_SHAPES)
@pytest.mark.parametrize("scale,dscale,eps", [(1e18, 1e-6, EPS), (1e-19, 1e3, 1.1754944e-38), (0.0, 1e3, 1.1754944e-38)])
def test_backward_of_far_scales(nq, bf16, shape, scale, dscale, eps):
    """1 / rms^2 leaves fp32's range (or falls among its last bits) although no result does."""
    rows, cols = shape
    h, w = rand(rows, cols, 1, bf16, scale), rand(1, cols, 2, bf16).view(-1) + 1.0
    dy, ds = rand(rows, cols, 3, bf16, dscale), rand(rows, cols, 4, bf16, dscale / max(scale, 1e-19))
    for d in (None, ds):
        check_backward(nq, h, w, dy, d, eps)


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", GRAD_SHAPES)
@pytest.mark.parametrize("scale,dscale", [(1e20, 1.0), (1e30, 1e-3), (1e34, 1.0), (1e10, 1e30)])
def test_backward_of_rows_whose_sums_overflow(nq, bf16, shape, scale, dscale):
    """sum(h^2), or sum(g h) alone, beyond fp32: the gradients are the formula's."""
    rows, cols = shape
    h, w = far_rows(rand(rows, cols, 1, bf16), scale), rand(1, cols, 2, bf16).view(-1) + 1.0
    dy, ds = rand(rows, cols, 3, bf16, dscale), rand(rows, cols, 4, bf16, dscale / scale)
    for d in (None, ds):
        check_backward(nq, h, w, dy, d, EPS)


# many aligned rows: every block takes several of them through its ring
RING_SHAPES = [(True, 2500, 2048), (True, 1300, 8192), (True, 700, 1032), (True, 3000, 4096), (False, 1500, 1000),
               (False, 2000, 2048), (False, 700, 8192)]


@pytest.mark.parametrize("bf16,rows,cols", RING_SHAPES)
def test_many_rows(nq, bf16, rows, cols):
    """Every output of many aligned rows, with and without the residual, against the 64-bit reference."""
    import torch
    x, res = rand(rows, cols, 1, bf16), rand(rows, cols, 2, bf16, 3.0)
    w = rand(1, cols, 3, bf16).view(-1) + 1.0
    x[rows // 2], res[rows // 2] = 0.0, 0.0
    for r_ in (res, None):
        s = torch.empty_like(x) if r_ is not None else None
        h = reference_h(x, r_)
        t, r = R.rmsnorm(h, w.double().cpu().numpy(), EPS)
        for fmt in (E4M3, E5M2, INT8):
            y, codes, _, scales = run(nq, x, r_, w, fmt, sum=s)
            check_codes8(codes, scales, t, r, cols, fmt, exact=bf16)
            check_y(y, t, r, cols)
            assert s is None or np.array_equal(s.double().cpu().numpy(), h)
        for fmt in (R.MX, R.NV):
            y, codes, bs, g = run(nq, x, r_, w, fmt, four=True, sum=s)
            check_mx4(nq, (codes, bs, g), t, r, rows, cols, fmt)
            check_y(y, t, r, cols)
    assert nq.device_error_flags() == 0


@pytest.mark.parametrize("bf16,rows,cols", [(True, 2500, 2048), (True, 1300, 8192), (False, 2000, 2048)])
def test_many_rows_in_place_and_in_pieces(nq, bf16, rows, cols):
    """The sum written over an input while the rows behind it are on their way in; and the same rows in calls of a
    few hundred, which another kernel takes: equal codes (they do not depend on the order of a sum), scales within
    both sums' tolerance."""
    import torch
    x, res = rand(rows, cols, 1, bf16), rand(rows, cols, 2, bf16, 3.0)
    w = rand(1, cols, 3, bf16).view(-1) + 1.0
    s = torch.empty_like(x)
    y, codes, _, scales = run(nq, x, res, w, E4M3, sum=s)
    _, nv, nvb, nvg = run(nq, x, res, w, R.NV, four=True, sum=s)
    for k in range(2):
        a, b = x.clone(), res.clone()
        y2, c2, _, s2 = run(nq, a, b, w, E4M3, sum=(a, b)[k])
        assert torch.equal((a, b)[k], s) and torch.equal((b, a)[k], (res, x)[k])
        assert torch.equal(y2, y) and torch.equal(c2, codes) and torch.equal(s2, scales)
    pitch, words = nq.mx4_row_bytes(cols), R.words(cols, R.NV)
    for at in range(0, rows, 512):   # whole tiles of scales
        part = slice(at, min(rows, at + 512))
        n = part.stop - at
        ps = torch.empty_like(x[part])
        _, c2, _, s2 = run(nq, x[part], res[part], w, E4M3, sum=ps)
        assert torch.equal(c2, codes[part]) and torch.equal(ps, s[part])
        assert torch.all((s2.double() / scales[part].double() - 1).abs() <= 2 * tol_r(cols) + 8 * U)
        _, c4, b4, g4 = run(nq, x[part], res[part], w, R.NV, four=True)
        idx = torch.from_numpy(R.scale_index(n, cols, R.NV)).cuda()
        assert torch.equal(c4, nv[at * pitch:part.stop * pitch]) and torch.equal(b4[idx], nvb[at // 128 * words * 512:][idx])
        assert torch.all((g4.double() / nvg[part].double() - 1).abs() <= 2 * tol_r(cols) + 8 * U)
    assert nq.device_error_flags() == 0


@pytest.mark.parametrize("bf16", [True, False])
@pytest.mark.parametrize("shape", FAR_SHAPES)
def test_far_rows_in_place_and_rows_beside_them(nq, bf16, shape):
    """A row whose squares overflow with the sum over either input, or with a weight of the other type: the results of
    separate tensors; the rows beside it are those of a call without it."""
    import torch
    rows, cols = shape
    x, res = rand(rows, cols, 1, bf16), rand(rows, cols, 2, bf16)
    w = rand(1, cols, 3, not bf16).view(-1).clamp(-0.4, 0.4) + 1.0
    calm = run(nq, x, res, w, E4M3)
    x[rows - 1, 2:70] = 1e25
    s = torch.empty_like(x)
    far = run(nq, x, res, w, E4M3, sum=s)
    nv = run(nq, x, res, w, R.NV, four=True)
    mx = run(nq, x, res, w, R.MX, four=True)
    t, r = product32(reference_h(x, res), w.double().cpu().numpy()), R.rmsnorm(reference_h(x, res), 1.0, EPS)[1]
    check_codes8(far[1], far[3], t, r, cols, E4M3)
    check_mx4(nq, nv[1:], t, r, rows, cols, R.NV)
    check_mx4(nq, mx[1:], t, r, rows, cols, R.MX)
    for a, b in ((calm[0], far[0]), (calm[1], far[1]), (calm[3], far[3])):
        assert torch.equal(a[:rows - 1], b[:rows - 1])
    for k in range(2):
        a, b = x.clone(), res.clone()
        y, codes, _, scales = run(nq, a, b, w, E4M3, sum=(a, b)[k])
        assert torch.equal((a, b)[k], s) and torch.equal(y, far[0]) and torch.equal(codes, far[1]) and torch.equal(scales, far[3])
        for fmt, want in ((R.NV, nv), (R.MX, mx)):
            a, b = x.clone(), res.clone()
            y, codes, bs, g = run(nq, a, b, w, fmt, four=True, sum=(a, b)[k])
            assert torch.equal(y, want[0]) and torch.equal(codes, want[1]) and torch.equal(bs, want[2])
            assert g is None or torch.equal(g, want[3])
