"""The 4-bit (MXFP4) K/V cache format restated in numpy, 64 bits, for the tests: quantisation, page layout, attention.

A block of 32 columns: 2^e with e = floor(log2(amax)) - 2 (+ 1 from 1.75 * 2^floor on), at least -126, byte e + 127; codes
0, 0.5, 1, 1.5, 2, 3, 4, 6, nearest with ties to the even code; byte 255 = the block held an infinity or a NaN."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """Codes ``[..., D]`` (0..15) and scale bytes ``[..., D / 32]`` of float64 rows."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    finite = np.isfinite(b).all(-1)
    amax = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0)).max(-1), 1.0)
    f, ex = np.frexp(amax)
    e = np.where(amax == 0, -126, np.maximum(ex - 3 + (f >= 0.875), -126))
    y = np.ldexp(np.abs(np.where(finite[..., None], b, 0)), -e[..., None])
    d = np.abs(y[..., None] - GRID)
    near = d.min(-1, keepdims=True)
    tie_rank = np.where(d == near, np.arange(8) % 2, 2)  # among the nearest the even code first
    code = tie_rank.argmin(-1).astype(np.uint8)
    code = np.where(finite[..., None], code | (np.signbit(b).astype(np.uint8) << 3), 0).astype(np.uint8)
    return code.reshape(x.shape), np.where(finite, e + 127, 255).astype(np.uint8)


def values(codes, scales):
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32) * s[..., None]).reshape(v.shape)


def _positions(heads, dim, page, is_v):
    t, h, d = np.ix_(np.arange(page), np.arange(heads), np.arange(dim))
    if is_v:
        n, w = 512 // dim, dim // 16
        byte = (((h * (page // n) + t // n) * 16 + d // w) * n + t % n) * (w // 2) + (d % w) // 2
    else:
        byte = (h * page + t) * (dim // 2) + d // 2
    t, h, s = np.ix_(np.arange(page), np.arange(heads), np.arange(dim // 32))
    scale = heads * page * dim // 2 + (h * (dim // 32) + s) * page + t
    return np.broadcast_to(byte, (page, heads, dim)), scale


def pack(codes, scales, is_v):
    """Pages ``[P, page bytes]`` of codes ``[P, page, heads, D]`` / scale bytes ``[P, page, heads, D / 32]``."""
    P, page, heads, dim = codes.shape
    byte, sc = _positions(heads, dim, page, is_v)
    raw = np.zeros((P, heads * page * (dim // 2 + dim // 32)), np.uint8)
    raw[:, byte[..., 0::2].ravel()] = (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(P, -1)
    raw[:, sc.ravel()] = scales.reshape(P, -1)
    return raw


def unpack(raw, heads, dim, page, is_v):
    """Values ``[P, page, heads, D]`` in float64 of raw pages."""
    P = raw.shape[0]
    byte, sc = _positions(heads, dim, page, is_v)
    b = raw[:, byte.ravel()].reshape(P, page, heads, dim)
    code = np.where(np.arange(dim) % 2, b >> 4, b & 15)
    return values(code, raw[:, sc.ravel()].reshape(P, page, heads, dim // 32))


def attention(q, k, v, scale, m):
    """Rows ``q [m, H, D]`` at the last m positions of keys ``k / v [n, Hkv, D]``: outputs, sum p |v|, and a bound of the
    error of a row's scores (see :func:`bound`).  Rows at negative positions: NaN."""
    n, hkv, dim = k.shape
    H = q.shape[1]
    o, av, ds = (np.full((m, H, dim), np.nan) for _ in range(3))
    for j in range(m):
        seen = n - m + 1 + j
        if seen <= 0:
            continue
        for h in range(H):
            kk, vv = k[:seen, h // (H // hkv)], v[:seen, h // (H // hkv)]
            with np.errstate(all="ignore"):
                s = kk @ q[j, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                o[j, h], av[j, h] = p @ vv, p @ np.abs(vv)
                ds[j, h] = scale * (dim + 8) * 2.0 ** -23 * (np.abs(kk) @ np.abs(q[j, h])).max()
    return o, av, ds


def bound(o, av, ds, n, half_step):
    """Error bound of an output.

    half_step |o|: its own rounding.  Times sum p |v|: the probabilities' two bf16 terms (2^-16), fp32 sums over n keys
    (each wave's accumulator adds a product of 32 keys every 128 keys; the sum over its pieces; 2^-23 each), and the
    scores' error ds: with scores off by at most ds every weight p_j / sum p is off by a factor between exp(-2 ds) and
    exp(2 ds), so the output by at most (exp(2 ds) - 1) sum p |v|.  ds is the rounding of an fp32 sum of dim
    exact products, (dim + 8) 2^-23 sum |q k|."""
    with np.errstate(over="ignore"):
        gamma = 2.0 ** -16 + (n / 64 + 64) * 2.0 ** -23 + np.expm1(2 * ds)
    return half_step * np.abs(o) + gamma * av + 1e-30
