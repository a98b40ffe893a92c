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
