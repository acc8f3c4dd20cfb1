"""8-bit rows in numpy and 64 bits, from their definition: what the kernels are compared with."""
import numpy as np

_C = np.arange(256)
_E, _F = (_C >> 3) & 15, _C & 7
TABLE = np.where(_E == 0, np.ldexp(_F.astype(np.float64), -9), np.ldexp(8.0 + _F, _E - 10)) * np.where(_C & 128, -1.0, 1.0)
TABLE[[0x7F, 0xFF]] = np.nan
_MAG = TABLE[:0x7F]  # magnitudes of the finite codes, ascending


def blocks(d):
    return (d + 127) // 128


def quantize(x):
    """(codes (n, whole blocks), scale exponents (n, blocks)) of rows of float64 that hold the caller's values exactly."""
    x = np.asarray(x, dtype=np.float64)
    n, d = x.shape
    nb = blocks(d)
    v = np.zeros((n, nb * 128))
    v[:, :d] = x
    v = v.reshape(n, nb, 128)
    with np.errstate(all="ignore"):
        bad = ~np.isfinite(v).all(axis=2)
        a = np.where(bad[..., None], 0.0, np.abs(v)).max(axis=2)
        m, e = np.frexp(a)                                     # a = m 2^e, 448 = 0.875 2^9
        s = np.where(a == 0, -127, np.maximum(e - 9 + (m > 0.875), -127))
        u = np.where(bad[..., None], 0.0, v) * np.ldexp(1.0, -s)[..., None]
        mag = np.abs(u)
        hi = np.clip(np.searchsorted(_MAG, mag), 0, 0x7E)      # first code >= mag
        lo = np.maximum(hi - 1, 0)
        dl, dh = mag - _MAG[lo], _MAG[hi] - mag
        up = (dh < dl) | ((dh == dl) & (hi % 2 == 0))          # ties to the even code
        c = np.where(up, hi, lo) | np.where(np.signbit(u), 128, 0)
    inside = (np.arange(nb * 128) < d).reshape(1, nb, 128)
    c = np.where(bad[..., None], np.where(inside, 0x7F, 0), c)
    return c.reshape(n, nb * 128).astype(np.uint8), np.where(bad, 255, s + 127).astype(np.uint8)


def values(codes, scales, d):
    n, nb = codes.shape[0], blocks(d)
    s = np.where(scales[:, :nb] == 255, np.nan, np.ldexp(1.0, scales[:, :nb].astype(np.int64) - 127))
    return (TABLE[codes].reshape(n, nb, 128) * s[..., None]).reshape(n, nb * 128)[:, :d]


def round_rows(x):
    return values(*quantize(x), np.asarray(x).shape[1])


def search(X, Q, k):
    """Top-k of the 64-bit products: score descending, ties by the lower id; NaN scores are no results.  X, Q: 64-bit values."""
    S = Q @ X.T
    D = np.full((len(Q), k), -np.finfo(np.float32).max, dtype=np.float32)
    I = np.full((len(Q), k), -1, dtype=np.int64)
    for i, s in enumerate(S):
        ids = np.flatnonzero(~np.isnan(s))
        if len(ids) > k:
            ids = ids[s[ids] >= np.partition(s[ids], len(ids) - k)[len(ids) - k]]   # (only what can be among them is sorted)
        order = ids[np.lexsort((ids, -s[ids]))][:k]
        D[i, :len(order)] = s[order].astype(np.float32)
        I[i, :len(order)] = order
    return D, I
