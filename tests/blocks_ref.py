"""64-bit references of the 8-bit block operators and of the residual stream, on the CPU, for the tests."""
import numpy as np
import torch

FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0, 4, 3, 7), "e5m2": (torch.float8_e5m2, 57344.0, 5, 2, 15)}


def decode(format):
    """The value of every byte of a format, from its definition (sign, exponent, digits)."""
    _, largest, ebits, mbits, bias = FORMATS[format]
    b = np.arange(256)
    e, m = (b >> mbits) & ((1 << ebits) - 1), b & ((1 << mbits) - 1)
    v = np.where(e == 0, m * 2.0 ** (1 - bias - mbits), (1 + m / 2.0 ** mbits) * 2.0 ** (e.astype(float) - bias))
    if format == "e4m3":
        v = np.where((b & 127) == 127, np.nan, v)
    else:
        v = np.where(e == 31, np.where(m == 0, np.inf, np.nan), v)
    return np.where(b >= 128, -v, v)


def nearest(v, format):
    """Bytes of the nearest value of the format, ties to the even byte; |v| at most the largest."""
    table = decode(format)[:128]
    n = int(np.sum(np.isfinite(table)))
    table = table[:n]
    a = np.abs(v)
    hi = np.clip(np.searchsorted(table, a), 0, n - 1)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - table[lo], table[hi] - a
    pick = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return (pick | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def quantize(x, format, square=False):
    """Bytes [M,K] and scale bytes of a float64 array whose values are exact."""
    _, largest, _, _, _ = FORMATS[format]
    M, K = x.shape
    q, KB = np.zeros((M, K), np.uint8), -(-K // 128)
    rows = [(i, min(M, i + 128)) for i in range(0, M, 128)] if square else [(i, i + 1) for i in range(M)]
    s = np.zeros((len(rows), KB), np.uint8)
    for i, (r0, r1) in enumerate(rows):
        for j in range(KB):
            b = x[r0:r1, j * 128:(j + 1) * 128]
            fin = np.abs(b[np.isfinite(b)])
            a, e = (fin.max() if fin.size else 0.0), 0
            if a > 0:
                e = int(np.frexp(a)[1]) - int(np.frexp(largest)[1]) - 1
                while a > largest * 2.0 ** e:
                    e += 1
                e = max(e, -127)
            s[i, j] = e + 127
            safe = np.where(np.isfinite(b), b, 0.0)
            o = nearest(safe / 2.0 ** e, format)
            o = np.where(np.isnan(b), 0x7F, o)
            o = np.where(np.isinf(b), 0x7F if format == "e4m3" else np.where(b > 0, 0x7C, 0xFC), o)
            q[r0:r1, j * 128:(j + 1) * 128] = o
    return q, s


def same_bytes(got, want, format):
    """Equal bytes, any NaN standing for any other."""
    nan = np.isnan(decode(format))
    return bool(np.all((got == want) | (nan[got] & nan[want])))


def values(q, s, format):
    """What bytes [M,K] and scale bytes (rows or squares) stand for, in float64."""
    M, K = q.shape
    f = np.repeat(2.0 ** (s.astype(float) - 127), 128, axis=1)[:, :K]
    if s.shape[0] != M:
        f = np.repeat(f, 128, axis=0)[:M]
    return decode(format)[q] * f


def norm_forward(t, kind, eps, alpha, dtype):
    """t: float64 tensors y, residual, pre_weight, pre_bias, post_weight, post_bias, gate (None where absent).  r is rounded to dtype
    with the identity as its gradient."""
    def norm(v, w, b):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w
        return v if b is None else v + b
    u = t["y"] if t["post_weight"] is None else norm(t["y"], t["post_weight"], t["post_bias"])
    r = u if t["gate"] is None else u * t["gate"]
    if t["residual"] is not None:
        r = r + alpha * t["residual"]
    r = r + (r.detach().to(dtype).double() - r.detach())
    return r, None if t["pre_weight"] is None else norm(r, t["pre_weight"], t["pre_bias"])
