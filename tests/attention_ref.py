"""Attention, int8 rows and 16-bit types in numpy float64, for the tests of the
prompt and paged attention entry points, and the error bounds they allow."""
import math

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
DTYPE = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


def to_bits(x, t):
    """float values as the type's array (bf16: uint16 bits, rounded to nearest even)."""
    x = np.asarray(x, np.float32)
    if t != "bf16":
        return x.astype(DTYPE[t])
    b = x.view(np.uint32)
    r = (b + 0x7FFF + ((b >> 16) & 1)) >> 16
    return np.where(np.isnan(x), (b >> 16) | 0x40, r).astype(np.uint16)


def from_bits(a, t):
    if t != "bf16":
        return np.asarray(a, np.float64)
    return (np.asarray(a, np.uint32) << 16).view(np.float32).astype(np.float64)


def rand(rng, shape, t, scale=1.0):
    return to_bits((rng.standard_normal(shape) * scale).astype(np.float32), t)


def visible(nq, nk, causal=True, window=0, sink=0):
    """[nq][nk]: which keys a query sees; the queries are the last nq positions."""
    p = np.arange(nk - nq, nk)[:, None]
    j = np.arange(nk)[None]
    see = (j <= p) if causal else np.ones((nq, nk), bool)
    if window:
        see = see & ((j > p - window) | (j < sink))
    return see


def attend(q, k, v, see, scale, t, exact_keys=False):
    """float64 attention of one sequence: q [nq][H][D] over k, v [nk][G][D].
    Returns the output and a bound of the error of a kernel that multiplies
    rows of type t and sums in fp32.

    The bound.  With u half a step of t (rows in), e = 2^-24 and A_i =
    sum_j w_ij |v_j|:
      scores: the products of 16-bit rows are exact in fp32, fp32 rows leave
      out less than 2^-23 of each; D sums and the scaling's two roundings:
      |ds| <= ((D + 2) e + 2^-23) S, S = scale sum_d |q k|, plus 2 e |s| for
      the base-2 form;
      weights: exp2's and the correction factors' relative error, at most
      2^-21 in all for up to 2^5 moves of the maximum; a weight times 2^ds
      has the relative error 2 ds (its own and its sum's);
      P rounded to t: u (fp32: 2^-23 of its products is left out);
      the sums over n keys: (n + 8) e, twice (numerator and denominator);
      the result rounded to t: u |y|.
    exact_keys: int8 rows with their scales' two roundings, 4 e more."""
    nq, H, D = q.shape
    G = k.shape[1]
    nk = k.shape[0]
    out = np.zeros((nq, H, D))
    tol = np.zeros((nq, H, D))
    u, e = HALF_STEP[t], 2.0 ** -24
    for h in range(H):
        kh, vh = k[:, h // (H // G)], v[:, h // (H // G)]
        if nk == 0:
            continue
        with np.errstate(all="ignore"):
            s = (q[:, h] @ kh.T) * scale
            S = (np.abs(q[:, h]) @ np.abs(kh).T) * scale
            s = np.where(see, s, -np.inf)
            m = s.max(1, keepdims=True)
            w = np.exp(s - np.where(np.isfinite(m), m, 0.0))
            w = np.where(see, w, 0.0)
            some = see.any(1)
            w = np.where(some[:, None], w / w.sum(1, keepdims=True), 0.0)
            for i in np.flatnonzero(some):      # masked rows of v may hold anything
                out[i, h] = w[i, see[i]] @ vh[see[i]]
                A = w[i, see[i]] @ np.abs(vh[see[i]])
                ds = ((D + 2) * e + 2.0 ** -23) * S[i, see[i]].max() + 2 * e * np.abs(s[i, see[i]]).max()
                if exact_keys:
                    ds += 4 * e * np.abs(s[i, see[i]]).max()
                n = see[i].sum()
                rel = 2 * ds + 2.0 ** -21 + (u if t != "f32" else 2.0 ** -23) + 2 * (n + 8) * e + 4 * e
                tol[i, h] = A * rel + u * np.abs(out[i, h])
    return out, tol


def quantize_rows(x):
    """KVCache::quantize_row on [..., D] floats: codes and scales in fp32 arithmetic."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        inv = np.where(amax == 0, np.float32(1), np.minimum(np.float32(127) / amax, np.finfo(np.float32).max))
        v = (x * inv.astype(np.float32)).astype(np.float64)
        codes = np.sign(v) * np.floor(np.abs(v) + 0.5)
        scale = np.where(amax == 0, np.float32(1), amax / np.float32(127)).astype(np.float32)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    codes = np.where(bad, 0, codes)
    return codes.astype(np.int8), np.where(bad, np.float32(np.nan), scale)


def default_scale(D):
    return 1.0 / math.sqrt(D)


def check(got, want, tol, what=""):
    got = np.asarray(got, np.float64)
    off = np.abs(got - want)
    ok = (off <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    if not ok.all():
        i = np.unravel_index(np.argmax(np.where(ok, 0, np.nan_to_num(off / np.maximum(tol, 1e-300), nan=np.inf))), ok.shape)
        raise AssertionError(f"{what}: {np.count_nonzero(~ok)} of {ok.size} off, worst at {i}: {got[i]} for {want[i]} +- {tol[i]}")
