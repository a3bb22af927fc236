"""AdamW with moments in 64 bits or as 8-bit codes, restated in NumPy from the formulas (test infrastructure).

`step64` is the update in float64.  `step32` computes the two moments in float32 in the order the product documents — each product and sum rounded by itself — so that
the codes of 8-bit moments can be predicted bit for bit; `encode` / `decode` are the 8-bit format."""
import numpy as np

BLOCK = 128
WORDS = np.array([0x6A09E667, 0xBB67AE85, 0x3C6EF373, 0xA54FF53B, 0x510E527F, 0x9B05688D, 0x1F83D9AB, 0x5BE0CD19], dtype=np.uint64)
M32 = np.uint64(0xFFFFFFFF)


def mix(x):
    x = np.asarray(x, dtype=np.uint64) & M32
    x = (x ^ (x >> np.uint64(16))) * np.uint64(0x7FEB352D) & M32
    x = (x ^ (x >> np.uint64(15))) * np.uint64(0x846CA68B) & M32
    return x ^ (x >> np.uint64(16))


def random_bits(n, seed, step, place, first=0):
    """The 16 bits of the first and of the second moments of elements [first, first + n)."""
    key = mix((seed + step * 0x9E3779B1 + place * 0x85EBCA6B) & 0xFFFFFFFF)
    j = np.arange(first, first + n, dtype=np.uint64)
    r = mix((j >> np.uint64(3)) ^ key) * WORDS[j & np.uint64(7)] & M32
    return r & np.uint64(0xFFFF), r >> np.uint64(16)


def blocks_of(x):
    """(blocks, 128), the last one filled with zeros."""
    nb = -(-x.size // BLOCK)
    out = np.zeros(nb * BLOCK, dtype=x.dtype)
    out[:x.size] = x
    return out.reshape(nb, BLOCK)


def decode(moments, exps, dtype=np.float64):
    c = np.asarray(moments).view(np.uint16).astype(np.int64)
    e = np.repeat(np.asarray(exps).view(np.uint16).astype(np.int64), BLOCK)[:c.size]
    mag, vc = c & 127, c >> 8

    def value(code, base):
        return np.where(code > 0, np.ldexp(1.0 + (code % 8) / 8.0, code // 8 + base - 127), 0.0)
    m = np.where(mag == 127, np.nan, np.where(mag == 0, 0.0, value(mag, e & 255) * np.where(c & 128, -1.0, 1.0)))
    v = np.where(vc == 255, np.inf, value(vc, e >> 8))
    return m.astype(dtype), v.astype(dtype)


def encode(m, v, um, uv):
    """float32 moments -> (codes, exps), uint16."""
    n = m.size
    mb, vb = (blocks_of(np.ascontiguousarray(x, dtype=np.float32)).view(np.uint32).astype(np.int64) for x in (m, v))
    sign, mb, vb = mb >> 31, mb & 0x7FFFFFFF, vb & 0x7FFFFFFF
    um, uv = blocks_of(um.astype(np.int64)), blocks_of(uv.astype(np.int64))
    base = lambda b, below: np.maximum((np.where(b < 0x7F800000, b, 0).max(1, keepdims=True) >> 23) - below, 1)   # noqa: E731
    bm, bv = base(mb, 14), base(vb, 30)
    m_out, v_out = mb >= 0x7F800000, vb >= 0x7F800000
    mb, vb = np.minimum(mb, 0x7F700000), np.minimum(vb, 0x7F700000)      # 1.875 * 2^127, the last finite code of any base: larger ones do not round up to infinity
    a = mb.astype(np.uint32).view(np.float32)
    low = ((bm << 23) + (1 << 20)).astype(np.uint32).view(np.float32)
    rounded = ((mb + (um << 4) + 8) >> 20) - (bm << 3)
    mc = np.where(a < low, (a > (low * np.float32(2.0 ** -16)) * (um.astype(np.float32) + np.float32(0.5))).astype(np.int64), rounded)
    mc = np.where(m_out, 127, mc | sign << 7)                # a zero may carry a sign: it stands for zero all the same
    vc = np.maximum(((vb + (uv << 4) + 8) >> 20) - (bv << 3), 1)
    vc = np.where(vb == 0, 0, np.where(v_out, 255, vc))
    return (mc | vc << 8).reshape(-1)[:n].astype(np.uint16), (bm | bv << 8).reshape(-1).astype(np.uint16)


def gather(moments, exps, width, index, rows):
    """Rows of 8-bit moments by index (outside: zero), re-blocked: each value keeps itself unless it is below the smallest code of its new block."""
    c = np.asarray(moments).view(np.uint16).astype(np.int64).reshape(rows, width)
    e = np.repeat(np.asarray(exps).view(np.uint16).astype(np.int64), BLOCK)[:c.size].reshape(rows, width)
    inside = (index >= 0) & (index < rows)
    take = lambda x: np.where(inside[:, None], x[np.where(inside, index, 0)], 0).reshape(-1)       # noqa: E731
    c, e = take(c), take(e)
    mag, sign, vc = c & 127, c & 128, c >> 8
    out = []
    for code, base, top, below in ((mag, e & 255, 127, 14), (vc, e >> 8, 255, 30)):
        special = code == top
        absolute = np.where((code > 0) & ~special, code + 8 * base, 0)
        new = np.maximum((blocks_of(absolute).max(1) >> 3) - below, 1)
        moved = np.maximum(absolute - 8 * np.repeat(new, BLOCK)[:absolute.size], 0 if top == 127 else 1)
        out.append((np.where(special, top, np.where(absolute > 0, moved, 0)), new))
    (m, bm), (v, bv) = out
    return (m | sign | v << 8).astype(np.uint16), (bm | bv << 8).astype(np.uint16)


def step32(m, v, g, betas, clip=None):
    """The moments of one step in float32, each operation rounded by itself."""
    f = np.float32
    g = np.asarray(g, dtype=f)
    with np.errstate(all="ignore"):
        if clip is not None:
            g = g * f(clip)
        return f(betas[0]) * m.astype(f) + g * f(1.0 - betas[0]), f(betas[1]) * v.astype(f) + (g * f(1.0 - betas[1])) * g


def step64(p, m, v, g, lr, wd, betas, eps, t, clip=1.0):
    """-> (p, m, v) in float64, and a bound for the float32 kernel's error in each: every float32 operation and constant is off by at most u = 2^-24 of its result."""
    p, m, v, g = (np.asarray(x, dtype=np.float64) for x in (p, m, v, g))
    b1, b2 = betas
    u = 2.0 ** -24
    with np.errstate(all="ignore"):
        g = g * clip
        ug = 0.0 if isinstance(clip, float) and clip == 1.0 else 3 * u             # norm, factor, product
        a, b = b1 * m, (1 - b1) * g
        m1 = a + b
        dm = 2 * u * np.abs(a) + (2 * u + ug) * np.abs(b) + u * np.abs(m1)          # constant, product each; sum
        a, b = b2 * v, (1 - b2) * g * g
        v1 = a + b
        dv = 2 * u * a + (3 * u + 2 * ug) * b + u * v1
        den = np.sqrt(v1) / np.sqrt(1 - b2 ** t) + eps
        dden = (np.sqrt(v1) / np.sqrt(1 - b2 ** t)) * (0.5 * np.where(v1 > 0, dv / np.where(v1 > 0, v1, 1), 0) + 3 * u) + u * eps + u * den      # root (2 u), constant; eps; sum
        upd = lr / (1 - b1 ** t) * m1 / den
        # step size (a constant), reciprocal (within one unit of its last place: 2 u), product; the sum of den within the root's 2 u, its constant and the sum itself
        dupd = np.abs(upd) * (4 * u + dden / den) + lr / (1 - b1 ** t) * dm / den
        p1 = p * (1 - lr * wd) - upd
        dp = 2 * u * np.abs(p) + dupd + u * np.abs(p1)
    tiny = 2.0 ** -149
    return (p1, m1, v1), (1.01 * dp + tiny, 1.01 * dm + 3 * tiny, 1.01 * dv + 4 * tiny)
