"""4-bit rows, rotary positions and sampling in numpy, in 64 bits, for the tests
of the entry points that serve a scheduler's passes."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def blocks_of(D):
    return -(-D // 32)


def fp4_rows(x):
    """[..., D] float32 values as codes [..., 32 b] (0 .. 15) and exponents [..., b]: by search, block by block."""
    x = np.asarray(x, np.float32)
    D = x.shape[-1]
    b = blocks_of(D)
    x = np.concatenate([x, np.zeros(x.shape[:-1] + (32 * b - D,), np.float32)], -1).reshape(x.shape[:-1] + (b, 32))
    bad = ~np.isfinite(x).all(-1)
    a = np.where(bad[..., None], 0, np.abs(x)).astype(np.float64)
    top = a.max(-1)
    e = np.full(top.shape, 2)
    for n in range(2, 253):                # the smallest that takes the largest to 7 or less
        e = np.where(top > 7 * 2.0 ** (e - 127), np.minimum(n + 1, 252), e)
    y = np.minimum(a * 2.0 ** (127 - e[..., None]), 6)
    off = np.abs(y[..., None] - LEVELS)
    near = off.min(-1, keepdims=True) == off
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1)) | (np.signbit(x) * 8)
    code = np.where(bad[..., None], 0, code).reshape(x.shape[:-2] + (32 * b,))
    return code.astype(np.uint8), np.where(bad, 255, e).astype(np.uint8)


def fp4_values(code, e, D):
    s = np.where(e == 255, np.nan, 2.0 ** (e.astype(np.float64) - 127))
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    return (v.reshape(e.shape + (32,)) * s[..., None]).reshape(code.shape)[..., :D]


def fp4_held(x):
    return fp4_values(*fp4_rows(x), np.shape(x)[-1])


def fp4_bytes(code):
    return code[..., 0::2] | code[..., 1::2] << 4


def frequencies(turn, base=5e6, factor=1.0, low=0.0, high=0.0, original=0):
    """Radians a position, of each pair, in extended precision."""
    i = np.arange(turn // 2).astype(np.longdouble)
    f = np.longdouble(np.float32(base)) ** (-2 * i / turn)
    g = np.zeros_like(f)
    if low or high:
        t = original * f / (2 * np.pi)
        g = np.clip((t - np.float32(low)) / (np.longdouble(np.float32(high)) - np.float32(low)), 0, 1)
    return f * (g + (1 - g) / np.longdouble(np.float32(factor)))


def turned(x, positions, turn, interleaved, magnitude=1.0, **kw):
    """x [rows][heads][D] (float64) turned, and |a| + |b| of each value's pair (0 past `turn`)."""
    a = np.asarray(positions).astype(np.longdouble)[:, None, None] * frequencies(turn, **kw)
    m = np.longdouble(np.float32(magnitude))
    c, s = np.cos(a) * m, np.sin(a) * m
    first, second = (np.s_[..., :turn:2], np.s_[..., 1:turn:2]) if interleaved else (np.s_[..., :turn // 2], np.s_[..., turn // 2:turn])
    u, w = x[first].astype(np.longdouble), x[second].astype(np.longdouble)
    out, size = x.astype(np.longdouble), np.zeros(x.shape)
    out[first], out[second] = u * c - w * s, u * s + w * c
    size[first] = size[second] = (np.abs(u) + np.abs(w)).astype(np.float64) * float(m)
    return out, size


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, probability) of one row: logits in float64, settings as float32; weights in whole steps of 2^-43."""
    l = np.where(np.isnan(logits), -np.inf, logits)
    order = np.lexsort((np.arange(len(l)), -l))
    order = order[l[order] > -np.inf]
    if not len(order):
        return -1, 0.0
    temperature, top_p, min_p, u = (float(np.float32(v)) for v in (temperature, top_p, min_p, u))
    if not temperature > 0:
        return int(order[0]), 1.0
    l = l[order]
    with np.errstate(all="ignore"):
        w = np.exp(np.where(l == l[0], 0.0, -np.inf if np.isinf(l[0]) else (l - l[0]) / temperature))
    w = np.rint(w * 2.0 ** 43).astype(np.int64)
    upto = np.cumsum(w)
    n = top_k if 0 < top_k < len(l) else len(l)
    mass = int(upto[n - 1])
    kept = mass
    if top_p < 1:
        kept = int(upto[np.searchsorted(upto, max(1.0, np.ceil(top_p * float(mass))))])
    if min_p > 0:
        weighs = np.flatnonzero(w.astype(np.float64) >= min(min_p, 1.0) * 2.0 ** 43)
        kept = min(kept, int(upto[weighs[-1]]))
    i = np.searchsorted(upto, min(int(max(u, 0.0) * float(kept)), kept - 1), side="right")
    return int(order[i]), int(w[i]) / kept
