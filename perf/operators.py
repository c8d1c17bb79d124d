"""What is measured of the RMS-norm and microscaled 4-bit operators.

Operators (the `op` of a case):
  norm       h = x + residual, RMS norm, 8-bit codes with a scale for each row
  norm_int8  the same with INT8 codes, through the INT8 linear layer behind it
  backward   gradients of the RMS norm (input and weight)
  roundtrip  microscaled 4-bit quantisation and back to values
  gemm       microscaled 4-bit product of two quantised operands
  linear     quantise the activations, then the product with quantised weights
  layer      h = x + residual, RMS norm with a 4-bit output, then the product

Formats: e4m3 / e5m2 (8 bits, a scale for each row); mx = MXFP4 (blocks of 32,
power-of-two scales), nv = NVFP4 (blocks of 16, E4M3 scales and one fp32 scale
for each row).
"""
import ctypes
import math

import torch

own = False

_QMAX = {"e4m3": 448.0, "e5m2": 57344.0, "int8": 127.0}
_F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_BLOCK = {"mx": 32, "nv": 16}
_T = {"bf16": torch.bfloat16, "f32": torch.float32}
_EPS = 1e-5


# ---- cases -----------------------------------------------------------------------
def listed():
    return [
        # one generated token through a block's norm, residual stream of 8192
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 8192, "dtype": "bf16", "fmt": "e4m3", "res": True},
        # a prompt of 16384 tokens
        {"name": "norm_prompt", "op": "norm", "rows": 16384, "cols": 8192, "dtype": "bf16", "fmt": "e4m3", "res": True},
        # odd width (no aligned rows), fp32 stream, gradients' format, first norm of a network (no residual yet)
        {"name": "norm_ragged", "op": "norm", "rows": 1021, "cols": 5003, "dtype": "f32", "fmt": "e5m2", "res": False},
        # a training step's norm
        {"name": "backward_batch", "op": "backward", "rows": 8192, "cols": 4096, "dtype": "bf16", "res": True},
        {"name": "backward_ragged", "op": "backward", "rows": 130, "cols": 2051, "dtype": "f32", "res": False},
        # an MLP weight quantised at load time and read back to check it
        {"name": "roundtrip_weight", "op": "roundtrip", "rows": 28672, "cols": 8192, "dtype": "bf16", "fmt": "mx"},
        # a ragged batch of activations
        {"name": "roundtrip_ragged", "op": "roundtrip", "rows": 257, "cols": 4111, "dtype": "f32", "fmt": "nv"},
        # the product alone, both operands quantised
        {"name": "gemm_square", "op": "gemm", "m": 4096, "n": 4096, "k": 4096, "fmt": "mx", "out": "bf16"},
        # up-projection of a prompt: activations quantised on the way
        {"name": "linear_prompt", "op": "linear", "m": 8192, "n": 14336, "k": 4096, "fmt": "nv", "out": "bf16"},
        # 16 sequences decoding: the weights' bytes count
        {"name": "linear_decode", "op": "linear", "m": 16, "n": 28672, "k": 8192, "fmt": "nv", "out": "bf16"},
        # every size ragged, fp32 out
        {"name": "gemm_ragged", "op": "gemm", "m": 300, "n": 1000, "k": 1111, "fmt": "mx", "out": "f32"},
        # 64 sequences decoding through norm and projection
        {"name": "layer_decode", "op": "layer", "m": 64, "n": 28672, "k": 8192, "fmt": "nv", "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_int8", "backward", "roundtrip", "gemm", "linear", "linear", "layer"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("norm", "backward", "roundtrip"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, min(65536, (1 << 26) // cols))
        c = {"op": op, "rows": rows, "cols": cols, "dtype": dtype}
        if op == "norm":
            c["fmt"] = rng.choice(["e4m3", "e5m2"])
        if op == "roundtrip":
            c["fmt"] = rng.choice(["mx", "nv"])
        else:
            c["res"] = rng.random() < 0.7
        return c
    m = _log(rng, 1, 8192)
    n, k = _log(rng, 64, 28672), _log(rng, 64, 14336)
    while m * n * k > 400_000_000_000:
        m = max(1, m // 2)
    if op == "norm_int8":  # the 8-bit product's aligned sizes
        return {"op": op, "m": m, "n": max(64, n // 16 * 16), "k": max(64, k // 16 * 16), "dtype": "bf16", "fmt": "int8"}
    if rng.random() < 0.6:
        n, k = max(64, n // 64 * 64), max(64, k // 64 * 64)
    c = {"op": op, "m": m, "n": n, "k": k, "fmt": rng.choice(["mx", "nv"]), "out": "bf16"}
    # fp32 out where 32 bits decide no rounding to 4 bits on the way: values next to a border would show in it
    if op == "gemm" or (op == "linear" and c["fmt"] == "mx"):
        c["out"] = rng.choice(["bf16", "f32"])
    return c


# ---- the 4-bit formats, in plain form -----------------------------------------------
def _e2m1_code(a):
    """Code 0..7 of |x| in 0, .5, 1, 1.5, 2, 3, 4, 6: nearest, ties to the even code, above 5 the largest."""
    c = (a > 0.25).to(torch.uint8)
    for t, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= t) if up else (a > t)
    return c


def _pitch(cols):
    return (cols + 31) // 32 * 16


def _scale_shape(rows, cols, fmt):
    return (rows + 127) // 128, ((cols + _BLOCK[fmt] - 1) // _BLOCK[fmt] + 3) // 4, 32, 4, 4


def _blocks(x, fmt):
    """x (fp32, rows x cols) in whole blocks: rows x blocks x block, zero behind the last column."""
    b = _BLOCK[fmt]
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % b)).view(rows, -1, b)


def _quantize(x, fmt):
    """Codes (rows x blocks x block, 0..15), the blocks' scale bytes and values, and the rows' scales (None for mx) of fp32 x."""
    v = _blocks(x, fmt)
    amax = v.abs().amax(-1)
    if fmt == "mx":
        byte = ((amax.view(torch.int32) >> 23) - 2).clamp_min(0)  # 2^(floor(log2 amax) - 2), biased by 127
        q = v * ((254 - byte) << 23).view(torch.float32).unsqueeze(-1)
        value = torch.exp2((byte - 127).double()).float()
        g = None
    else:
        # 64 bits: bf16 values often fall right on a border of the blocks' scales and codes
        v, amax = v.double(), amax.double()
        top = amax.amax(-1, keepdim=True)
        top = torch.where(top > 0, top.clamp_min(2688.0 * 2.0 ** -110), 2688.0)
        s8 = (amax * 448.0 / top).float().to(torch.float8_e4m3fn)
        byte, value = s8.view(torch.uint8), s8.float()
        g = (top / 2688.0).float().reshape(-1)
        unit = (value * top).unsqueeze(-1)
        q = torch.where(unit > 0, v * 2688.0 / unit, 0.0)
    return _e2m1_code(q.abs()) | (torch.signbit(q).to(torch.uint8) << 3), byte.to(torch.uint8), value, g


def _pack(code, byte, rows, cols, fmt):
    """Codes two to a byte in rows of whole 16 bytes, and the scale bytes in tiles of 128 rows x 4 blocks."""
    flat = torch.nn.functional.pad(code.reshape(rows, -1), (0, 2 * _pitch(cols) - code.shape[1] * code.shape[2]))
    packed = flat[:, 0::2] | (flat[:, 1::2] << 4)
    rb, kb = _scale_shape(rows, cols, fmt)[:2]
    t = torch.nn.functional.pad(byte, (0, kb * 4 - byte.shape[1], 0, rb * 128 - rows))
    return packed.contiguous(), t.view(rb, 4, 32, kb, 4).permute(0, 3, 2, 1, 4).contiguous()


def _value_of(device):
    v = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    return torch.tensor(v + [-x for x in v], device=device)


def _scale_values(tiles, rows, fmt):
    rb, kb = tiles.shape[:2]
    byte = tiles.permute(0, 3, 2, 1, 4).reshape(rb * 128, kb * 4)[:rows]
    return byte.view(torch.float8_e4m3fn).float() if fmt == "nv" else torch.exp2(byte.double() - 127).float()


def _unpack(packed, tiles, rows, cols, fmt):
    """fp32 values (without the rows' scales) of a packed operand."""
    code = torch.stack((packed & 15, packed >> 4), -1).view(rows, -1).int()
    s = _scale_values(tiles, rows, fmt).repeat_interleave(_BLOCK[fmt], 1)[:, :cols]
    return _value_of(packed.device)[code[:, :cols]] * s


# ---- inputs -----------------------------------------------------------------------
def _activations(rows, cols, gen, dtype):
    """A residual stream's values: normal, every 128th channel larger."""
    x = torch.randn(rows, cols, device="cuda", generator=gen)
    x[:, 5::128] *= 8.0
    return x.to(dtype)


def _operand(rows, cols, fmt, gen, scale):
    """A quantised rows x cols operand as a program keeps it: packed codes, scale tiles, rows' scales."""
    code, byte, _, g = _quantize(torch.randn(rows, cols, device="cuda", generator=gen) * scale, fmt)
    return (*_pack(code, byte, rows, cols, fmt), g)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("norm", "backward", "roundtrip"):
        rows, cols, dt = case["rows"], case["cols"], _T[case["dtype"]]
    else:
        rows, cols, dt = case["m"], case["k"], torch.bfloat16
    s.update(op=op, rows=rows, cols=cols, dt=dt)
    if op != "gemm":
        s["x"] = _activations(rows, cols, gen, dt)
    if op in ("norm", "norm_int8", "layer", "backward"):
        s["w"] = (1.0 + 0.1 * torch.randn(cols, device="cuda", generator=gen)).to(dt)
    if op in ("norm", "norm_int8", "layer"):
        res = case.get("res", True)
        s["res"] = torch.randn(rows, cols, device="cuda", generator=gen).mul_(2.0).to(dt) if res else None
        s["sum"] = torch.empty(rows, cols, dtype=dt, device="cuda") if res else None
    if op in ("norm", "norm_int8"):
        s["codes"] = torch.empty(rows, cols, dtype=_F8.get(case["fmt"], torch.int8), device="cuda")
        s["scales"] = torch.empty(rows, device="cuda")
    if op == "backward":
        s["dy"] = (0.01 * torch.randn(rows, cols, device="cuda", generator=gen)).to(dt)
        s["dsum"] = (0.01 * torch.randn(rows, cols, device="cuda", generator=gen)).to(dt) if case["res"] else None
        s["dx"] = torch.empty(rows, cols, dtype=dt, device="cuda")
        s["dw"] = torch.empty(cols, device="cuda")
    if op in ("roundtrip", "linear", "layer"):  # room for the quantised activations
        s["ac"] = torch.empty(rows, _pitch(cols), dtype=torch.uint8, device="cuda")
        s["as"] = torch.empty(_scale_shape(rows, cols, case["fmt"]), dtype=torch.uint8, device="cuda")
        s["ag"] = torch.empty(rows, device="cuda") if case["fmt"] == "nv" else None
    if op == "roundtrip":
        s["values"] = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    if op == "gemm":
        s["ac"], s["as"], s["ag"] = _operand(rows, cols, case["fmt"], gen, 1.0)
    if op in ("gemm", "linear", "layer"):
        s["bc"], s["bs"], s["bg"] = _operand(case["n"], cols, case["fmt"], gen, 0.02)
        s["out"] = torch.empty(rows, case["n"], dtype=_T[case["out"]], device="cuda")
    if op == "norm_int8":
        s["bc"] = torch.randint(-127, 128, (case["n"], cols), device="cuda", generator=gen, dtype=torch.int8)
        s["bg"] = torch.rand(case["n"], device="cuda", generator=gen) * 1e-3 + 1e-4
        s["out"] = torch.empty(rows, case["n"], dtype=torch.bfloat16, device="cuda")
    return s


# ---- plain forms --------------------------------------------------------------------
def _norm(s):
    """h = x + residual as stored, h times the weight, and 1 / rms of each row (fp32)."""
    h = s["x"] if s["res"] is None else (s["x"].float() + s["res"].float()).to(s["dt"])
    f = h.float()
    return h, f * s["w"].float(), torch.rsqrt(f.square().mean(-1, keepdim=True) + _EPS)


def _codes8(y, fmt):
    """Values that the 8-bit codes stand for (before the rows' scales), and those scales."""
    a = y.abs().amax(-1, keepdim=True)
    q = y * torch.where(a > 0, _QMAX[fmt] / a, 1.0)
    q = torch.round(q).clamp(-127.0, 127.0) if fmt == "int8" else q.clamp(-_QMAX[fmt], _QMAX[fmt]).to(_F8[fmt])
    return q, torch.where(a > 0, a / _QMAX[fmt], 1.0).reshape(-1)


def _product(s, a, ag, fmt):
    b = _unpack(s["bc"], s["bs"], s["out"].shape[1], s["cols"], fmt)
    out = a @ b.t()
    if fmt == "nv":
        out = out * ag[:, None] * s["bg"]
    return out.to(s["out"].dtype)


def _requantized(x, fmt, cols):
    """(values without the rows' scales, rows' scales) of fp32 x quantised to 4 bits."""
    code, _, value, g = _quantize(x, fmt)
    return (_value_of(x.device)[code.int()] * value.unsqueeze(-1)).view(x.shape[0], -1)[:, :cols], g


def _run_plain(s):
    op, case = s["op"], s["case"]
    if op == "norm":
        h, y, r = _norm(s)
        codes, scales = _codes8(y * r, case["fmt"])
        return (codes, scales) if s["res"] is None else (codes, scales, h)
    if op == "norm_int8":
        h, y, r = _norm(s)
        q, scales = _codes8(y * r, "int8")
        return ((q @ s["bc"].float().t()) * scales[:, None] * s["bg"]).to(torch.bfloat16), h
    if op == "backward":
        h, dy = s["x"].float(), s["dy"].float()
        r = torch.rsqrt(h.square().mean(-1, keepdim=True) + _EPS)
        n = h * r
        g = dy * s["w"].float()
        dx = r * (g - n * (g * n).mean(-1, keepdim=True))
        if s["dsum"] is not None:
            dx = dx + s["dsum"].float()
        return dx.to(s["dt"]), (dy * n).sum(0)
    fmt = case["fmt"]
    if op == "roundtrip":
        v, g = _requantized(s["x"].float(), fmt, s["cols"])
        return (v if g is None else v * g[:, None]).to(torch.bfloat16)
    if op == "gemm":
        return _product(s, _unpack(s["ac"], s["as"], s["rows"], s["cols"], fmt), s["ag"], fmt)
    if op == "linear":
        return _product(s, *_requantized(s["x"].float(), fmt, s["cols"]), fmt)
    h, y, r = _norm(s)
    if fmt == "mx":
        return _product(s, *_requantized(y * r, fmt, s["cols"]), fmt), h
    v, g = _requantized(y, fmt, s["cols"])  # a row's factor cancels in all but the row's scale
    return _product(s, v, g * r.reshape(-1), fmt), h


# ---- the framework's calls -----------------------------------------------------------
_nq = None


def _library():
    global _nq
    if _nq is None:
        import nova_b200.capi as _nq
    return _nq


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _plan(s, nq):
    """The descriptors that a program keeps, made in its first pass."""
    dt, op, case = nq.F32 if s["dt"] == torch.float32 else nq.BF16, s["op"], s["case"]
    if op in ("norm", "norm_int8", "layer", "backward"):
        s["norm"] = nq.make_rmsnorm_desc(s["rows"], s["cols"], dt, dt, _EPS)
    if op == "norm_int8":
        s["gemm"] = nq.make_desc(s["rows"], case["n"], s["cols"], nq.INT8, nq.INT8, nq.B_NK, nq.BF16, 1.0,
                                 s["scales"].data_ptr(), s["bg"].data_ptr())
    if op in ("gemm", "linear", "layer"):
        s["gemm"] = nq.make_mx4_desc(s["rows"], case["n"], s["cols"], nq.NVFP4 if case["fmt"] == "nv" else nq.MXFP4,
                                     nq.BF16 if case["out"] == "bf16" else nq.F32, 1.0, _ptr(s["ag"]), _ptr(s["bg"]))
    s["plan"] = True


def _run_own(s):
    nq = _library()
    if "plan" not in s:
        _plan(s, nq)
    op, case = s["op"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if op in ("norm", "norm_int8"):
        fmt = {"e4m3": nq.E4M3, "e5m2": nq.E5M2, "int8": nq.INT8}[case["fmt"]]
        nq.rmsnorm_quantize(ctypes.byref(s["norm"]), s["x"].data_ptr(), _ptr(s["res"]), s["w"].data_ptr(), _ptr(s["sum"]), 0,
                            s["codes"].data_ptr(), s["scales"].data_ptr(), fmt, stream)
        if op == "norm_int8":
            nq.gemm(ctypes.byref(s["gemm"]), s["codes"].data_ptr(), s["bc"].data_ptr(), s["out"].data_ptr(), stream)
            return s["out"], s["sum"]
        return (s["codes"], s["scales"]) if s["res"] is None else (s["codes"], s["scales"], s["sum"])
    if op == "backward":
        nq.rmsnorm_backward(ctypes.byref(s["norm"]), s["x"].data_ptr(), s["w"].data_ptr(), s["dy"].data_ptr(), _ptr(s["dsum"]),
                            s["dx"].data_ptr(), s["dw"].data_ptr(), stream)
        return s["dx"], s["dw"]
    fmt = nq.NVFP4 if case["fmt"] == "nv" else nq.MXFP4
    if op in ("roundtrip", "linear"):
        nq.quantize_rows_mx4(s["x"].data_ptr(), nq.F32 if s["dt"] == torch.float32 else nq.BF16, 0, s["ac"].data_ptr(),
                             s["as"].data_ptr(), _ptr(s["ag"]), s["rows"], s["cols"], fmt, stream)
    if op == "layer":
        nq.rmsnorm_quantize_mx4(ctypes.byref(s["norm"]), s["x"].data_ptr(), s["res"].data_ptr(), s["w"].data_ptr(),
                                s["sum"].data_ptr(), 0, s["ac"].data_ptr(), s["as"].data_ptr(), _ptr(s["ag"]), fmt, stream)
    if op == "roundtrip":
        nq.dequantize_rows_mx4(s["ac"].data_ptr(), s["as"].data_ptr(), _ptr(s["ag"]), s["values"].data_ptr(), nq.BF16,
                               s["rows"], s["cols"], fmt, stream)
        return s["values"]
    nq.gemm_mx4(ctypes.byref(s["gemm"]), s["ac"].data_ptr(), s["as"].data_ptr(), s["bc"].data_ptr(), s["bs"].data_ptr(),
                s["out"].data_ptr(), stream)
    return (s["out"], s["sum"]) if op == "layer" else s["out"]


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- the work that a pass cannot do without ----------------------------------------------
def _operand_bytes(rows, cols, fmt):
    return rows * (cols / 2 + cols / _BLOCK[fmt]) + (4 * rows if fmt == "nv" else 0)


def work(case):
    op = case["op"]
    if op in ("norm", "backward", "roundtrip"):
        rows, cols, e = case["rows"], case["cols"], 2 if case["dtype"] == "bf16" else 4
        n = rows * cols
        if op == "norm":
            return {"bytes": n * (e + 1 + (2 * e if case["res"] else 0)) + 4 * rows + cols * e, "flops": 6 * n}
        if op == "backward":
            return {"bytes": n * e * (4 if case["res"] else 3) + cols * (e + 4), "flops": 12 * n}
        return {"bytes": n * (e + 2) + _operand_bytes(rows, cols, case["fmt"]), "flops": 6 * n}
    m, n, k = case["m"], case["n"], case["k"]
    flops = 2.0 * m * n * k
    if op == "norm_int8":
        return {"bytes": m * k * 6 + 2 * k + n * k + 4 * n + 2 * m * n, "flops": flops}
    b = _operand_bytes(n, k, case["fmt"]) + m * n * (2 if case["out"] == "bf16" else 4)
    if op == "gemm":
        b += _operand_bytes(m, k, case["fmt"])
    elif op == "linear":
        b += 2 * m * k
    else:
        b += 6 * m * k + 2 * k
    return {"bytes": b, "flops": flops}


# ---- 64-bit values, from the definitions ----------------------------------------------------
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_e2m1(v):
    """Nearest E2M1 value of each double, ties to the even code, saturating."""
    a = v.abs()
    best = torch.zeros_like(a)
    for i in range(1, 8):
        mid = (_E2M1[i - 1] + _E2M1[i]) / 2
        best = torch.where((a > mid) | ((a == mid) & (i % 2 == 0)), _E2M1[i], best)
    return torch.copysign(best, v)


def _exact_e4m3(v):
    """Nearest E4M3 value of each non-negative double, ties to even, at most 448."""
    step = torch.exp2(torch.floor(torch.log2(v.clamp_min(2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp_max(448.0)


def _exact_mx4(x, fmt):
    """The doubles that a rows x cols matrix's 4-bit form stands for, row by row."""
    rows, cols = x.shape
    size = 32 if fmt == "mx" else 16
    whole = torch.zeros(rows, (cols + size - 1) // size * size, dtype=torch.float64, device=x.device)
    whole[:, :cols] = x
    blocks = whole.reshape(rows, -1, size)
    top = blocks.abs().amax(2, keepdim=True)
    if fmt == "mx":
        unit = torch.exp2((torch.frexp(top)[1].double() - 3).clamp_min(-127.0))
    else:
        row = top.amax(1, keepdim=True)
        row = torch.where(row > 0, row.clamp_min(2688.0 * 2.0 ** -110), 2688.0)
        level = _exact_e4m3(448.0 * top / row)
        near = torch.where(level > 0, 2688.0 * blocks / torch.where(level > 0, level * row, 1.0), 0.0)
        return (_exact_e2m1(near) * level * row / 2688.0).reshape(rows, -1)[:, :cols]
    return (_exact_e2m1(blocks / unit) * unit).reshape(rows, -1)[:, :cols]


def _exact_kept(codes, tiles, rows_scale, rows, cols, fmt):
    """The doubles of an operand that the program keeps packed."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), dtype=torch.float64, device=codes.device)
    out = torch.empty(rows, codes.shape[1] * 2, dtype=torch.float64, device=codes.device)
    out[:, 0::2] = table[(codes % 16).long()]
    out[:, 1::2] = table[(codes // 16).long()]
    size = 32 if fmt == "mx" else 16
    r = torch.arange(rows, device=codes.device)[:, None]
    b = (torch.arange(cols, device=codes.device) // size)[None, :]
    byte = tiles[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]
    unit = torch.exp2(byte.double() - 127.0) if fmt == "mx" else byte.view(torch.float8_e4m3fn).double()
    out = out[:, :cols] * unit
    return out if rows_scale is None else out * rows_scale.double()[:, None]


def _exact_norm(s):
    h = s["x"].double()
    if s["res"] is not None:
        h = (h + s["res"].double()).to(s["dt"]).double()
    return h, h * s["w"].double(), 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h, y, r = _exact_norm(s)
        y = y * r
        scale = y.abs().amax(1, keepdim=True) / _QMAX[case["fmt"]]
        scale = torch.where(scale > 0, scale, 1.0)
        codes = (y / scale).to(_F8[case["fmt"]]).double()
        return (codes, scale.reshape(-1)) if s["res"] is None else (codes, scale.reshape(-1), h)
    if op == "norm_int8":
        h, y, r = _exact_norm(s)
        y = y * r
        scale = y.abs().amax(1, keepdim=True) / 127.0
        q = torch.round(y / scale) * scale
        return q @ (s["bc"].double() * s["bg"].double()[:, None]).t(), h
    if op == "backward":
        x, w, dy = s["x"].double(), s["w"].double(), s["dy"].double()
        n = x.shape[1]
        norm = torch.sqrt((x * x).mean(1, keepdim=True) + _EPS)
        dx = dy * w / norm - x * (dy * w * x).sum(1, keepdim=True) / (n * norm ** 3)
        if s["dsum"] is not None:
            dx = dx + s["dsum"].double()
        return dx, (dy * x / norm).sum(0)
    fmt = case["fmt"]
    if op == "roundtrip":
        return torch.cat([_exact_mx4(x.double(), fmt) for x in s["x"].split(4096)])
    m, n, k = case["m"], case["n"], case["k"]
    h = None
    if op == "gemm":
        a = _exact_kept(s["ac"], s["as"], s["ag"], m, k, fmt)
    elif op == "linear":
        a = _exact_mx4(s["x"].double(), fmt)
    else:
        h, y, r = _exact_norm(s)
        a = _exact_mx4(y * r, fmt) if fmt == "mx" else _exact_mx4(y, fmt) * r
    out = torch.empty(m, n, dtype=torch.float64, device=a.device)
    for at in range(0, n, 8192):
        to = min(n, at + 8192)  # whole tiles of 128 rows of scales
        b = _exact_kept(s["bc"][at:to], s["bs"][at // 128:], None if s["bg"] is None else s["bg"][at:to], to - at, k, fmt)
        out[:, at:to] = a @ b.t()
    return out if h is None else (out, h)
