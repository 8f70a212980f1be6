"""The 8-bit moment storage in numpy, from its definition in include/anni_adam.h: tables of the
codes' values and a search between neighbours, in 64 bits."""
import numpy as np

BLOCK = 256
GOLD, MULT = 0x9E3779B9, 0xB7E15163


def _table(normals):
    """Magnitudes of the codes relative to 2^E: eight even steps at the bottom, then binades up to [1, 2)."""
    bottom = -(normals - 1)
    vals = [r * 2.0 ** (bottom - 3) for r in range(8)]
    for e in range(bottom, 1):
        vals += [(1 + r / 8) * 2.0 ** e for r in range(8)]
    return np.array(vals)


TABLE_M, TABLE_V = _table(15), _table(31)          # 128 and 256 codes; the last of each is never written


def dither(n, t, first=0):
    """(m's, v's) 16 random bits of the elements [first, first + n) at step t."""
    s = ((t * GOLD) & 0xFFFFFFFF) ^ (t >> 7)
    s = (s * MULT) & 0xFFFFFFFF
    s ^= s >> 16
    m32 = np.uint64(0xFFFFFFFF)
    x = ((np.arange(first, first + n, dtype=np.uint64) * np.uint64(GOLD)) + np.uint64(s)) & m32
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(MULT)) & m32
    x ^= x >> np.uint64(15)
    return (x & np.uint64(0xFFFF)).astype(np.float64), (x >> np.uint64(16)).astype(np.float64)


def _blocks(x):
    nb = (x.size + BLOCK - 1) // BLOCK
    full = np.zeros(nb * BLOCK, x.dtype)
    full[:x.size] = x
    return full.reshape(nb, BLOCK)


def exponents(x):
    """The exponent byte of each block of a float32 array."""
    out = []
    for row in _blocks(np.asarray(x, np.float32)):
        top = float(np.max(np.abs(row)))
        if not np.isfinite(top) or top > 1.75 * 2.0 ** 127:
            out.append(255)
            continue
        e = -127
        if top > 0:
            e = int(np.frexp(top)[1]) - 1
            if top > 1.75 * 2.0 ** e:
                e += 1
        out.append(max(e + 127, 0))
    return np.array(out, np.uint8)


def _scale(b, n):
    e = np.maximum(b.astype(np.int64), 1) - 127
    return np.repeat(2.0 ** e.astype(np.float64), BLOCK)[:n]


def encode(x, table, rnd=None, keep_positive=False):
    """(codes of |x| in `table`, exponent bytes); rnd: 16 random bits per element, None: to nearest, ties to even."""
    x = np.asarray(x, np.float32)
    b = exponents(x)
    y = np.abs(x.astype(np.float64)) / _scale(b, x.size)
    y = np.where(np.repeat(b == 255, BLOCK)[:x.size], 0.0, y)
    lo = np.minimum(np.searchsorted(table, y, side="right") - 1, table.size - 2)
    place = np.rint((y - table[lo]) / (table[lo + 1] - table[lo]) * 2.0 ** 20)
    up = place + 16.0 * rnd >= 2.0 ** 20 if rnd is not None else \
        (place > 2.0 ** 19) | ((place == 2.0 ** 19) & (lo % 2 == 1))
    # a place that rounds to the upper neighbour by itself (below the smallest float) is that neighbour
    code = np.where(up, lo + 1, lo)
    if keep_positive:
        code = np.where((y > 0) & (code == 0), 1, code)
    return code.astype(np.uint8), b


def encode_m(m, rnd=None):
    code, b = encode(m, TABLE_M, rnd)
    sign = np.signbit(np.asarray(m, np.float32)) & ~np.repeat(b == 255, BLOCK)[:code.size]
    return code | np.where(sign, 128, 0).astype(np.uint8), b


def encode_v(v, rnd=None):
    return encode(v, TABLE_V, rnd, keep_positive=True)


def decode_m(code, b):
    v = TABLE_M[code & 127] * _scale(b, code.size) * np.where(code & 128, -1.0, 1.0)
    v = np.where(np.repeat(b == 255, BLOCK)[:code.size], np.nan, v)
    return v.astype(np.float32)


def decode_v(code, b):
    v = TABLE_V[code] * _scale(b, code.size)
    v = np.where(np.repeat(b == 255, BLOCK)[:code.size], np.nan, v)
    return v.astype(np.float32)
