"""Plain 64-bit NumPy forms of the 8-bit floating-point Linear operators and of the sampler (cube_quant_fp8, cube_gemm_fp8,
cube_linear_fp8, cube_sample_rows): test infrastructure, never imported by the product."""
import numpy as np

BLOCK = 128


def e4m3_values():
    """value of every byte: sign, 4 exponent bits (bias 7), 3 fraction bits; 0x7f and 0xff are NaN."""
    b = np.arange(256)
    exp, frac = (b >> 3) & 15, (b & 7).astype(np.float64)
    v = np.where(exp == 0, frac * 2.0 ** -9, (1 + frac / 8) * 2.0 ** (exp - 7.0)) * np.where(b >> 7, -1.0, 1.0)
    v[(b & 127) == 127] = np.nan
    return v


def quant(x):
    """x [M, K] -> (values of the codes [M, KB*128], exponent bytes int [M, KB])."""
    x = np.asarray(x, dtype=np.float64)
    M, K = x.shape
    kb = -(-K // BLOCK)
    b = np.zeros((M, kb * BLOCK))
    b[:, :K] = x
    b = b.reshape(M, kb, BLOCK)
    a = np.where(np.isfinite(b), np.abs(b), 0.0).max(2) if M else np.zeros((0, kb))
    e = np.full(a.shape, -127)
    for i in range(-126, 128):
        e = np.where(a > 448.0 * 2.0 ** (i - 1), i, e)
    y = b * (2.0 ** -e.astype(np.float64))[:, :, None]
    fin = np.isfinite(y)
    with np.errstate(divide="ignore"):
        step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(np.where(fin, y, 1.0)), 2.0 ** -6))) - 3)
    v = np.where(fin, np.round(np.where(fin, y, 0.0) / step) * step, np.nan)
    return v.reshape(M, kb * BLOCK), e + 127


def unpack(q, scale, columns):
    """q uint8 [rows, KB*128], scale int32 [ceil(KB/4), rows] -> (code values, exponent bytes [rows, KB])."""
    kb = -(-columns // BLOCK)
    s = np.ascontiguousarray(scale.T).view(np.uint8).reshape(q.shape[0], -1)[:, :kb].astype(np.int64)
    return e4m3_values()[q], s


def pack(values, e_bytes):
    """the reverse of `unpack`, for building operands: code values must be e4m3 numbers."""
    tab = e4m3_values()
    order = np.argsort(tab[:127])
    codes = order[np.searchsorted(tab[:127][order], np.abs(values))].astype(np.uint8)
    q = np.where(np.signbit(values), codes | 128, codes).astype(np.uint8)
    rows, kb = e_bytes.shape
    s = np.zeros((rows, -(-kb // 4) * 4), dtype=np.uint8)
    s[:, :kb] = e_bytes
    return q, np.ascontiguousarray(s.view(np.int32).T)


def rows_value(values, e_bytes):
    return values * np.repeat(2.0 ** (e_bytes.astype(np.float64) - 127), BLOCK, axis=1)


def gemm(a, w, bias=None, act=None):
    """a [M, K], w [N, K] in float64 -> (result, sum of magnitudes per output: what rounding errors scale with)."""
    y = a @ w.T
    mag = np.abs(a) @ np.abs(w).T
    if bias is not None:
        y = y + bias
        mag = mag + np.abs(bias)
    if act == "tanh":
        y = np.tanh(y)
    elif act == "relu":
        y = np.where(np.isnan(y), y, np.maximum(y, 0.0))
    return y, mag


def candidates(z):
    """indices of a row's candidates in the sampler's order."""
    z = np.asarray(z, dtype=np.float64) + 0.0
    idx = np.flatnonzero(z > -np.inf)
    return idx[np.argsort(-z[idx], kind="stable")]


def sample_row(z, u, T=1.0, k=0, p=1.0, m=0.0):
    """-> (token, prob, distance of u * total from the nearest border relative to the total)."""
    z = np.asarray(z, dtype=np.float64) + 0.0
    order = candidates(z)
    if len(order) == 0:
        return -1, 0.0, 1.0
    if not T > 0:
        return int(order[0]), 1.0, 1.0
    top = z[order[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(z[order] == top, 0.0, (z[order] - top) / T)
    w = np.exp(x)
    if 0 < k < len(w):
        w = w[:k]
    c = np.cumsum(w)
    n = len(w)
    if p < 1:
        n = min(n, int(np.searchsorted(c, max(p, 0.0) * c[-1], side="left")) + 1)
    n = max(1, min(n, int((w >= min(m, 1.0)).sum())))
    c = c[:n]
    t = min(max(u, 0.0), 1.0) * c[-1]
    at = min(int(np.searchsorted(c, t, side="right")), int(np.flatnonzero(w[:n] > 0)[-1]))
    return int(order[at]), float(w[at] / c[-1]), float(np.abs(c - t).min() / c[-1])
