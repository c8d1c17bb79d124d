"""64-bit references of the microscaled 4-bit formats and the RMS norm, on numpy.

Everything is computed from the definitions in include/nova_q.h on doubles;
ratios of bf16 (or fp32) values that fall on a rounding border are kept exact:
the quotients are single correctly rounded divisions of exactly held operands."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
MX, NV = 0, 1
BLOCK = {MX: 32, NV: 16}
QMAX = {0: 448.0, 1: 57344.0, 2: 127.0}


def e2m1(v):
    """Nearest E2M1 value, ties to the even code, saturating."""
    a = np.abs(v)
    mids = (E2M1[1:] + E2M1[:-1]) / 2
    i = np.searchsorted(mids, a, side="left")         # mids[i-1] < a <= mids[i]
    tie = (i < 7) & (a == mids[np.minimum(i, 6)])
    i = i + (tie & (i % 2 == 1))                       # an odd lower neighbour goes up
    return np.copysign(E2M1[i], v)


def e4m3(v):
    """Nearest E4M3 value of non-negative doubles, ties to even, at most 448."""
    _, e = np.frexp(np.maximum(v, 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.minimum(np.rint(v / step) * step, 448.0)


def e4m3_of_byte(b):
    b = b.astype(np.int64)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.ldexp(1.0, (e - 10).astype(np.int32)))
    return np.where(b & 128, -v, v) + np.where((b & 127) == 127, np.nan, 0.0)


def pitch(cols):
    return (cols + 31) // 32 * 16


def words(cols, fmt):
    return ((cols + BLOCK[fmt] - 1) // BLOCK[fmt] + 3) // 4


def blocks(x, fmt):
    rows, cols = x.shape
    n = words(cols, fmt) * 4 * BLOCK[fmt]
    out = np.zeros((rows, n))
    out[:, :cols] = x
    return out.reshape(rows, -1, BLOCK[fmt])


def quantize(x, fmt):
    """(quotients q that E2M1 rounds, block scales, row scales or None) of finite doubles x.

    Blocks run to the end of the last word of four scales."""
    b = blocks(x, fmt)
    top = np.abs(b).max(-1)
    if fmt == MX:
        _, e = np.frexp(top)
        s = np.where(top > 0, np.ldexp(1.0, np.maximum(e - 3, -127)), 2.0 ** -127)
        return b / s[..., None], s, None
    row = top.max(1, keepdims=True)
    level = np.maximum(row, 2688.0 * 2.0 ** -110)
    s = e4m3(448.0 * top / level)
    d = (s * level)[..., None]
    q = np.where(d > 0, 2688.0 * b / np.where(d > 0, d, 1.0), 0.0)
    return q, s, np.where(row > 0, level / 2688.0, 1.0)[:, 0]


def scale_index(rows, cols, fmt):
    """Byte offsets of the block scales, rows x blocks (whole words)."""
    w = words(cols, fmt)
    r = np.arange(rows)[:, None]
    b = np.arange(4 * w)[None, :]
    return (r // 128 * w + b // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + b % 4


def unpack_codes(buf, rows, cols):
    """E2M1 values rows x (2 * pitch) of packed codes."""
    b = np.asarray(buf, np.uint8).reshape(rows, pitch(cols))
    c = np.stack((b & 15, b >> 4), -1).reshape(rows, -1)
    return np.where(c & 8, -1.0, 1.0) * E2M1[c & 7]


def unpack_scales(buf, rows, cols, fmt):
    b = np.asarray(buf, np.uint8)[scale_index(rows, cols, fmt)]
    if fmt == NV:
        return e4m3_of_byte(b)
    return np.where(b == 255, np.nan, np.ldexp(1.0, b.astype(np.int32) - 127))


def values(codes, scales, rows, cols, fmt):
    """Doubles (without row scales) of a packed operand."""
    v = unpack_codes(codes, rows, cols)[:, :cols]
    return v * np.repeat(unpack_scales(scales, rows, cols, fmt), BLOCK[fmt], 1)[:, :cols]


def pack(x, fmt):
    """Packed codes and scale bytes (uint8) and row scales (fp32 or None) of doubles x, for the product's tests."""
    rows, cols = x.shape
    q, s, g = quantize(x, fmt)
    v = e2m1(q).reshape(rows, -1)
    n = 2 * pitch(cols)
    v = v[:, :n] if v.shape[1] >= n else np.pad(v, ((0, 0), (0, n - v.shape[1])))
    code = np.searchsorted(E2M1, np.abs(v)).astype(np.uint8) | (np.signbit(v).astype(np.uint8) << 3)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    if fmt == MX:
        byte = (np.frexp(s)[1] + 126).astype(np.uint8)
    else:
        table = e4m3_of_byte(np.arange(127))
        byte = np.searchsorted(table, s).astype(np.uint8)
    buf = np.zeros(((rows + 127) // 128) * words(cols, fmt) * 512, np.uint8)
    buf[scale_index(rows, cols, fmt)] = byte
    return codes, buf, None if g is None else g.astype(np.float32)


def bf16(x):
    """Doubles or floats rounded to bf16 (via fp32), as doubles."""
    u = np.asarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return r.astype(np.float64)


def rmsnorm(h, w, eps):
    """(t, r) of doubles: t = h w, r = 1 / sqrt(mean(h^2) + eps)."""
    return h * w, 1.0 / np.sqrt((h * h).mean(1) + eps)


def rmsnorm_backward(h, w, dy, dsum, eps):
    n = h.shape[1]
    r = 1.0 / np.sqrt((h * h).mean(1, keepdims=True) + eps)
    g = dy * w
    dx = r * g - h * r ** 3 * (g * h).sum(1, keepdims=True) / n
    return dx + (0.0 if dsum is None else dsum), (dy * h * r).sum(0)
