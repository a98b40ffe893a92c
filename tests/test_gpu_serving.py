"""Rotary positions, alone and with a pass's store, and sampling of a batch of
rows, against the formulas in 64 bits and more."""
import ctypes as C

import numpy as np
import pytest

import attention_ref as R
import pocketforge_amd as pf
import serving_ref as S
import test_gpu_attention as A

pytestmark = pytest.mark.gpu
dev = A.dev
TYPE = dict(A.TYPE, fp4=pf.TYPE_FP4)
RAMP = dict(base=5e5, factor=8.0, low=1.0, high=32.0, original=8192)


def bound(want, size, t):
    """With e = 2^-24: cosine and sine are off by at most their argument's rounding (e pi / 4), the polynomial's last two
    roundings (2 e) and the magnitude's product (e); the product b s rounds (e), the sum too (e |y|); the result to its
    type, in fp16 no finer than half of 2^-24."""
    w = np.abs(want.astype(np.float64))
    return size * 6 * 2.0 ** -24 + w * (2.0 ** -24 + R.HALF_STEP[t]) + (2.0 ** -25 if t == "f16" else 0.0)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("rows,H,D,turn", [(1, 1, 16, 0), (3, 5, 128, 0), (70, 3, 80, 40), (33, 20, 128, 64), (9, 2, 48, 24),
                                           (200, 12, 64, 0), (2, 7, 112, 8), (1, 40, 96, 96)])
def test_rotary(gpu, t, interleaved, rows, H, D, turn):
    rng = np.random.default_rng(rows * H + D)
    for kw in (dict(), dict(RAMP, magnitude=1.25), dict(factor=4.0, base=1e4)):
        x = R.rand(rng, (rows, H, D), t)
        at = rng.integers(0, 200000, rows).astype(np.int32)
        at[:1] = 0
        rot = pf.Rotary(gpu, D, turn, interleaved, **kw)
        y = R.from_bits(rot.apply(dev(gpu, x), dev(gpu, at)).numpy(), t)
        want, size = S.turned(R.from_bits(x, t), at, turn or D, interleaved, **kw)
        R.check(y, want.astype(np.float64), bound(want, size, t), f"rotary {kw}")
        np.testing.assert_array_equal(y[..., turn or D:], R.from_bits(x, t)[..., turn or D:])
        rot.close()


def test_rotary_far(gpu):
    """Positions up to the largest, and negative ones: angles of 2^31 radians keep their fraction; and the steps
    between neighbours turn back what they turned."""
    at = np.array([0, 1, -1, 2 ** 31 - 1, -2 ** 31, 2 ** 30 + 1, 123456789, 16777217], np.int32)
    rng = np.random.default_rng(3)
    for interleaved in (True, False):
        x = R.rand(rng, (len(at), 2, 64), "f32")
        rot = pf.Rotary(gpu, 64, interleaved=interleaved, base=1e4)
        y = rot.apply(dev(gpu, x), dev(gpu, at))
        want, size = S.turned(x.astype(np.float64), at, 64, interleaved, base=1e4)
        R.check(y.numpy(), want.astype(np.float64), bound(want, size, "f32"))
        np.testing.assert_array_equal(y.numpy()[0], x[0])
        back = rot.apply(y, dev(gpu, np.where(at == -2 ** 31, at, -at))).numpy()
        keep = at != -2 ** 31
        R.check(back[keep], x[keep].astype(np.float64), 3 * bound(want, size, "f32")[keep] + 6 * 2.0 ** -24 * size[keep])
        rot.close()


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_in_place_and_strides(gpu, t, interleaved):
    """q and k of a fused row turned in place in one call; into columns beside them; the rest of the rows stays."""
    n, H, D = 37, 6, 64
    rng = np.random.default_rng(8)
    w = 3 * H * D
    x = R.rand(rng, (n, w), t)
    at = dev(gpu, np.arange(n, dtype=np.int32))
    rot = pf.Rotary(gpu, D, 48, interleaved)
    want, size = S.turned(R.from_bits(x, t)[:, :H * D].reshape(n, H, D), np.arange(n), 48, interleaved)
    L, es = pf.lib(), x.itemsize
    for column in (0, 2 * H * D, H * D):
        b = dev(gpu, x)
        gpu.check(L.pf_rotary_apply(rot.h, TYPE[t], H, C.c_void_p(b.ptr), C.c_void_p(b.ptr + column * es), C.c_void_p(at.ptr), n, w, w), "apply")
        y = b.numpy()
        got = R.from_bits(y[:, column:column + H * D], t).reshape(n, H, D)
        R.check(got, want.astype(np.float64), bound(want, size, t))
        y[:, column:column + H * D] = x[:, column:column + H * D]
        np.testing.assert_array_equal(y, x)
    rot.close()


def test_rotary_not_finite(gpu):
    """An infinity or a NaN reaches its pair and nothing else."""
    x = np.ones((2, 3, 32), np.float32)
    x[0, 1, 5], x[1, 2, 20] = np.inf, np.nan
    for interleaved, first, second in ((True, (4, 5), (20, 20)), (False, (5, 13), (20, 20))):
        rot = pf.Rotary(gpu, 32, 16, interleaved)
        y = rot.apply(dev(gpu, x), dev(gpu, np.array([3, 5], np.int32))).numpy()
        bad = ~np.isfinite(y)
        assert bad[0, 1, list(first)].all() and bad[1, 2, 20] and bad.sum() == 3
        rot.close()


def test_rotary_refusals(gpu):
    L = pf.lib()
    h = pf.vp()

    def make(**kw):
        d = pf.RotaryDesc(**dict(dict(head_dim=64, interleaved=1), **kw))
        rc = L.pf_rotary_create(gpu.h, C.byref(d), C.byref(h))
        if rc == 0:
            L.pf_rotary_destroy(h)
        return rc

    assert make() == 0 and make(turn=8, base=10.0, factor=0.5, magnitude=2.0) == 0 and make(low=0, high=2, original=7) == 0
    assert make(head_dim=0) == -4 and make(head_dim=72) == -4 and make(head_dim=256) == -4
    assert make(turn=12) == -1 and make(turn=72) == -1
    for bad in (-1.0, float("nan"), float("inf")):
        assert make(base=bad) == -1 and make(factor=bad) == -1 and make(magnitude=bad) == -1 and make(high=bad, original=5) == -1
    assert make(base=1.0) == -1 and make(low=2, high=2, original=5) == -1 and make(low=3, high=1, original=5) == -1
    assert make(low=1, high=2) == -1 and make(low=float("nan"), high=1, original=5) == -1
    n, H, D = 8, 2, 64
    rot = pf.Rotary(gpu, D)
    x, y, at = gpu.empty((n, H, D), np.float16), gpu.empty((n, H, D), np.float16), dev(gpu, np.zeros(n, np.int32))

    def call(code, type=pf.TYPE_F16, heads=H, a=x.ptr, b=y.ptr, p=at.ptr, rows=n, xs=0, os=0):
        v = [C.c_void_p(i) if i else None for i in (a, b, p)]
        rc = L.pf_rotary_apply(rot.h, type, heads, *v, rows, xs, os)
        assert rc == code, (rc, L.pf_last_error(gpu.h))

    call(0)
    call(0, b=x.ptr)
    call(0, rows=0, a=None, b=None, p=None)
    call(-1, type=pf.TYPE_I8)
    call(-1, heads=0)
    call(-1, heads=70000)
    call(-1, xs=H * D - 8)
    call(-1, os=H * D + 4)
    call(-1, a=None)
    call(-1, b=None)
    call(-1, p=None)
    call(-1, a=x.ptr + 2)
    call(-1, p=at.ptr + 2)
    call(-1, b=x.ptr + 16)
    call(-1, b=x.ptr, rows=4, os=2 * H * D)       # in place with another stride
    call(-1, b=at.ptr, rows=1)
    for bad in (lambda: rot.apply(x, dev(gpu, np.zeros(n, np.int64))), lambda: rot.apply(x, dev(gpu, np.zeros(n + 1, np.int32))),
                lambda: rot.apply(x, at, out=gpu.empty((n, H, D), np.float32)),
                lambda: rot.apply(gpu.empty((n, H, 32), np.float16), at), lambda: pf.Rotary(gpu, 64, turn=-8)):
        with pytest.raises(pf.PFError):
            bad()
    rot.close()


# ------------------------------------------------ a pass's rows, turned and stored

@pytest.mark.parametrize("ct", ["fp4", "i8", "bf16", "f16"])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("H,G,D,turn", [(4, 4, 64, 0), (16, 2, 128, 64), (6, 3, 80, 40), (5, 5, 48, 24), (1, 1, 16, 8)])
def test_store_rotary(gpu, ct, t, interleaved, H, G, D, turn):
    """Keys in the pages are the turned keys' codes, whole steps alike; values as store() has them; queries turned."""
    if ct == "f16" and t != "f16":
        t = "f32"
    rng = np.random.default_rng(H * D)
    c = pf.PagedCache(gpu, 2, G, D, 40, 4, 300, 16, TYPE[ct])
    rot = pf.Rotary(gpu, D, turn, interleaved, magnitude=1.25, **RAMP)
    c.append([2, 0, 3], [70, 5, 33])
    seqs, rows = [3, 1, 0, 2], [2, 40, 0, 7]
    c.append(seqs, rows)
    n = sum(rows)
    at = np.concatenate([np.arange(b, b + r) for b, r in zip((33, 0, 5, 70), rows)])
    q, k, v = (R.rand(rng, (n, h, D), t) for h in (H, G, G))
    print(f"store rotary {t} into {ct} interleaved {interleaved} H {H} G {G} D {D} turn {turn}", flush=True)
    y = R.from_bits(c.store_rotary(1, rot, dev(gpu, q), dev(gpu, k), dev(gpu, v)).numpy(), t)
    kw = dict(RAMP, magnitude=1.25)
    want, size = S.turned(R.from_bits(q, t), at, turn or D, interleaved, **kw)
    R.check(y, want.astype(np.float64), bound(want, size, t), "queries")
    want, size = S.turned(R.from_bits(k, t), at, turn or D, interleaved, **kw)
    gk, gv = (g.numpy() for g in c.gather(1, seqs))        # (rows of before hold anything)
    new = np.concatenate([np.arange(a + b - r, a + b) for a, b, r in
                          zip(np.cumsum([0] + [c.length(s) for s in seqs]), [c.length(s) for s in seqs], rows)])

    def held(x):
        if ct == "fp4":
            return S.fp4_held(x)
        if ct == "i8":
            codes, scale = R.quantize_rows(x)
            return (codes.astype(np.float32) * scale).astype(np.float64)
        return R.from_bits(R.to_bits(x, ct), ct)

    np.testing.assert_array_equal(gv[new].astype(np.float64), held(R.from_bits(v, t).astype(np.float32)))
    if ct in ("fp4", "i8"):
        np.testing.assert_array_equal(gk[new].astype(np.float64), held(want.astype(np.float32)))
    else:
        R.check(gk[new], want.astype(np.float64), bound(want, size, ct), "keys")
    c.close()
    rot.close()


@pytest.mark.parametrize("t,ct", [("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("H,G,D,turn", [(4, 4, 64, 0), (16, 2, 128, 64), (6, 3, 80, 40), (1, 1, 16, 8)])
def test_store_rotary_of_another_type(gpu, t, ct, interleaved, H, G, D, turn):
    """16-bit rows into pages of the other 16-bit type, with positions (turned in fp32, rounded once) and without."""
    rng = np.random.default_rng(H + D)
    c = pf.PagedCache(gpu, 1, G, D, 12, 2, 90, 16, TYPE[ct])
    rot = pf.Rotary(gpu, D, turn, interleaved, magnitude=1.25, **RAMP)
    c.append([1], [21])
    c.append([0, 1], [40, 7])
    at = np.concatenate([np.arange(40), np.arange(21, 28)])
    q, k, v = (R.rand(rng, (47, h, D), t) for h in (H, G, G))
    print(f"store rotary {t} into {ct} interleaved {interleaved} H {H} G {G} D {D}", flush=True)
    y = R.from_bits(c.store_rotary(0, rot, dev(gpu, q), dev(gpu, k), dev(gpu, v)).numpy(), t)
    kw = dict(RAMP, magnitude=1.25)
    want, size = S.turned(R.from_bits(q, t), at, turn or D, interleaved, **kw)
    R.check(y, want.astype(np.float64), bound(want, size, t), "queries")
    want, size = S.turned(R.from_bits(k, t), at, turn or D, interleaved, **kw)
    new = np.r_[0:40, 61:68]
    gk, gv = (g.numpy()[new] for g in c.gather(0, [0, 1]))
    R.check(gk, want.astype(np.float64), bound(want, size, ct), "keys")
    held = [R.from_bits(R.to_bits(R.from_bits(x, t).astype(np.float32), ct), ct) for x in (k, v)]
    np.testing.assert_array_equal(gv, held[1])
    c.store(0, dev(gpu, k), dev(gpu, v))
    gk, gv = (g.numpy()[new] for g in c.gather(0, [0, 1]))
    np.testing.assert_array_equal(gk, held[0])
    np.testing.assert_array_equal(gv, held[1])
    c.close()
    rot.close()


def test_store_rotary_in_place_and_refusals(gpu):
    """Queries of a fused row turned in place; and the calls that are refused, which change nothing."""
    H, G, D, n = 4, 2, 64, 9
    rng = np.random.default_rng(1)
    c = pf.PagedCache(gpu, 1, G, D, 4, 2, 64, 16, pf.TYPE_FP4)
    rot, other = pf.Rotary(gpu, D), pf.Rotary(gpu, 128)
    w = (H + 2 * G) * D
    x = R.rand(rng, (n, w), "bf16")
    b, L = dev(gpu, x), pf.lib()
    q, k, v = b.ptr, b.ptr + H * D * 2, b.ptr + (H + G) * D * 2

    def call(code, layer=0, r=rot, type=pf.TYPE_BF16, heads=H, q=q, k=k, v=v, out=q, s=(w, w, w, w)):
        p = [C.c_void_p(i) if i else None for i in (q, k, v, out)]
        rc = L.pf_pages_store_rotary(c.h, layer, r.h if r else None, type, heads, *p, *s)
        assert rc == code, (rc, L.pf_last_error(gpu.h))

    call(-5)
    c.append([1], [n])
    call(-1, layer=1)
    call(-1, r=None)
    call(-1, r=other)
    call(-1, type=pf.TYPE_FP4)
    call(-1, heads=0)
    call(-1, q=None)
    call(-1, out=None)
    call(-1, k=k + 2)
    call(-1, s=(w, w, w, H * D))
    call(-1, s=(w, G * D - 8, w, w))
    call(-1, out=k)
    call(-1, out=q + D * 2)                       # its last head would be k's first
    np.testing.assert_array_equal(b.numpy(), x)
    call(0)
    f = R.from_bits(x, "bf16")
    want, size = S.turned(f[:, :H * D].reshape(n, H, D), np.arange(n), D, True)
    y = b.numpy()
    R.check(R.from_bits(y[:, :H * D], "bf16").reshape(n, H, D), want.astype(np.float64), bound(want, size, "bf16"))
    np.testing.assert_array_equal(y[:, H * D:], x[:, H * D:])
    gk, gv = c.gather(0, [1])
    want, _ = S.turned(f[:, H * D:(H + G) * D].reshape(n, G, D), np.arange(n), D, True)
    np.testing.assert_array_equal(gk.numpy(), S.fp4_held(want.astype(np.float32)))
    np.testing.assert_array_equal(gv.numpy(), S.fp4_held(f[:, (H + G) * D:].reshape(n, G, D).astype(np.float32)))
    with pytest.raises(pf.PFError):
        c.store_rotary(0, rot, gpu.empty((n + 1, H, D), np.float32), gpu.empty((n, G, D), np.float32), gpu.empty((n, G, D), np.float32))
    c.append([0], [0])
    call(0, q=None, k=None, v=None, out=None)     # a pass without rows
    c.close()
    rot.close()
    other.close()


# -------------------------------------------------------------------- sampling

SETTINGS = [dict(temperature=0.0), dict(temperature=0.8, top_p=0.95), dict(top_k=50), dict(temperature=0.7, top_k=40, top_p=0.9, min_p=0.05),
            dict(min_p=0.02), dict(temperature=1.3, top_k=200, top_p=0.98), dict(), dict(temperature=2.0, top_p=0.999),
            dict(temperature=3.0, top_k=1500), dict(temperature=1.5, top_k=1100, top_p=0.6, min_p=1e-4), dict(top_k=1), dict(top_p=0.0),
            dict(min_p=1.0), dict(temperature=1e-3), dict(temperature=1e-45), dict(temperature=1e30), dict(temperature=float("inf")), dict(temperature=50.0, top_p=0.5)]
U = [0.0, 0.1, 0.5, 0.9, 0.999, 1 - 2.0 ** -24]


def logits_of(rng, rows, V, t, kind="zipf"):
    if kind == "zipf":
        x = -1.6 * np.log(rng.permuted(np.tile(np.arange(1, V + 1), (rows, 1)), axis=1)) + 0.7 * rng.standard_normal((rows, V)) + 9
    elif kind == "flat":
        x = rng.standard_normal((rows, V))
    else:
        x = np.full((rows, V), 2.5)
    return R.to_bits(x.astype(np.float32), t)


def sample_case(gpu, x, t, u, settings, stride=0):
    """Every row with every setting and u, as rows of one call, with settings of the rows' own."""
    rows, V = x.shape
    print(f"sample {t} {x.shape} stride {stride}", flush=True)
    all_ = [(r, s, v) for r in range(rows) for s in settings for v in u]
    pick = np.array([r for r, _, _ in all_])
    big = np.zeros((len(all_), stride or V), x.dtype)
    big[:, :V] = x[pick]
    full = [dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **s) for _, s, _ in all_]
    cols = {n: dev(gpu, np.array([f[n] for f in full], np.int32 if n == "top_k" else np.float32)) for n in full[0]}
    b, uu = dev(gpu, big), dev(gpu, np.array([v for _, _, v in all_], np.float32))
    n = len(all_)
    tokens, probs = gpu.empty((n,), np.int32), gpu.empty((n,), np.float32)
    d = pf.SampleDesc(TYPE[t], V, stride, 0, 0, 0, 0, *(cols[k].ptr for k in ("temperature", "top_k", "top_p", "min_p")))
    gpu.check(pf.lib().pf_sample_rows(gpu.h, C.byref(d), C.c_void_p(b.ptr), C.c_void_p(uu.ptr), n, C.c_void_p(tokens.ptr),
                                      C.c_void_p(probs.ptr)), "pf_sample_rows")
    tokens, probs = tokens.numpy(), probs.numpy()
    f = R.from_bits(x, t)
    for i, (r, s, v) in enumerate(all_):
        token, prob = S.sample(f[r], v, **s)
        assert tokens[i] == token, (r, s, v, tokens[i], token, probs[i], prob)
        # (a weight is off by half a step of 2^-43 and 2^-47 of itself, the kept sum by as much of each of its own: far
        # below fp32's half step where the token's share is above 2^-20 of the largest's)
        assert abs(probs[i] - prob) <= 2.0 ** -23 * prob + 2.0 ** -44, (r, s, v, probs[i], prob)


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 9, 100, 1000, 5003])
def test_sample(gpu, t, V):
    sample_case(gpu, logits_of(np.random.default_rng(V), 2, V, t), t, U, SETTINGS)


@pytest.mark.parametrize("t,V,kind", [("f32", 16384, "zipf"), ("f32", 16385, "zipf"), ("bf16", 40000, "zipf"), ("f16", 130560, "zipf"),
                                      ("f32", 30011, "flat"), ("bf16", 30011, "flat"), ("f16", 70000, "flat"), ("bf16", 16384, "flat")])
def test_sample_large(gpu, t, V, kind):
    """One row, a slice of the card each; then many rows."""
    x = logits_of(np.random.default_rng(V), 1, V, t, kind)
    for s in SETTINGS:
        sample_case(gpu, x, t, [0.37], [s])
    sample_case(gpu, x, t, U, SETTINGS)


@pytest.mark.parametrize("V", [3, 1000, 3000, 20000])
def test_sample_equal_logits(gpu, V):
    """Every token the same: tokens in order of their numbers, borders on whole counts."""
    u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24]
    sample_case(gpu, logits_of(None, 1, V, "f32", "equal"), "f32", u,
                [dict(), dict(top_p=0.5), dict(top_k=V // 2 + 1), dict(top_k=V // 2 + 1, top_p=0.25), dict(min_p=0.5), dict(temperature=0.0)])


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_sample_few_distinct(gpu, t):
    """More equal logits than a sorted list holds on both sides of the borders, with the first few above them."""
    rng = np.random.default_rng(5)
    V = 18000
    x = rng.choice(np.array([1.0, 1.5, 1.5, 2.0, -3.0]), (1, V))
    x[0, rng.permutation(V)[:5]] = 4.0
    x[0, 77] = -0.0
    x[0, 78] = 0.0
    sample_case(gpu, R.to_bits(x.astype(np.float32), t), t, [0.0, 0.2, 0.4, 0.6, 0.8, 0.97],
                [dict(), dict(top_k=3000), dict(top_k=9000, top_p=0.7), dict(top_p=0.3), dict(min_p=0.05), dict(min_p=0.2, top_p=0.9),
                 dict(top_k=1000), dict(temperature=0.5, top_k=900, top_p=0.8)])


def test_sample_masked(gpu):
    """Masked tokens are never chosen; rows of one token, and of none; infinities and NaN; logits of the largest size."""
    V = 3001
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, V)).astype(np.float32)
    x[0, rng.permutation(V)[:V - 3]] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, V - 1] = -3e38
    x[3, ::2] = np.nan
    x[4, [7, 2000]] = np.inf
    x[5] = np.nan
    x[6] = np.where(np.arange(V) % 2, 3e38, -3e38)
    x[7, 5:] = np.finfo(np.float32).min           # a mask of the type's lowest value
    sample_case(gpu, x, "f32", [0.0, 0.3, 0.7, 1 - 2.0 ** -24], SETTINGS)
    y = np.full((2, 20001), -np.inf, np.float32)
    y[0, 20000] = 1
    sample_case(gpu, y, "f32", [0.5], SETTINGS)
    z = R.to_bits(rng.standard_normal((1, 20001)).astype(np.float32), "f16")
    z[0, 100:] = np.finfo(np.float16).min
    sample_case(gpu, z, "f16", [0.5, 0.99], SETTINGS)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("V,stride", [(1003, 1005), (16390, 16397), (17, 19)])
def test_sample_strides(gpu, t, V, stride):
    """Rows that start anywhere."""
    sample_case(gpu, logits_of(np.random.default_rng(V), 3, V, t), t, [0.0, 0.6, 0.97], SETTINGS[:8], stride)


def test_sample_settings_of_all_rows(gpu):
    """Numbers for every row, rows' own, and both; u outside its range; the same call again."""
    rng = np.random.default_rng(9)
    x = logits_of(rng, 7, 4000, "f32")
    u = np.array([0.3, -1, 2, np.nan, 0.0, 0.99, 0.5], np.float32)
    for kw in (dict(), dict(temperature=0.7, top_k=30, top_p=0.9, min_p=0.01), dict(temperature=0)):
        a, p = gpu.sample_rows(dev(gpu, x), dev(gpu, u), **kw)
        b, _ = gpu.sample_rows(dev(gpu, x), dev(gpu, u), **kw)
        np.testing.assert_array_equal(a.numpy(), b.numpy())
        for i in range(7):
            v = 0.0 if not u[i] > 0 else min(u[i], 1.0)
            token, prob = S.sample(x[i].astype(np.float64), v, **kw)
            assert a.numpy()[i] == token and abs(p.numpy()[i] - prob) <= 2.0 ** -23 * prob + 2.0 ** -44
    k = np.array([1, 0, -5, 4000, 9999, 3, 2000], np.int32)
    a, _ = gpu.sample_rows(dev(gpu, x), dev(gpu, np.full(7, 0.8, np.float32)), temperature=1.1, top_k=dev(gpu, k), out=(gpu.empty((7,), np.int32), None))
    gpu.synchronize()
    assert a.numpy().tolist() == [S.sample(x[i].astype(np.float64), 0.8, temperature=1.1, top_k=max(0, int(k[i])))[0] for i in range(7)]


# temperatures at which log2(e) / T has fp32 pieces far above 1, of either sign
NEARLY_GREEDY = [dict(temperature=t) for t in (1e-6, 8e-8, 4e-8, 1e-8, 1e-9, 1e-10, 2e-10, 1e-12, 1e-15, 1e-20, 1e-30)]
NEARLY_GREEDY += [dict(temperature=1e-10, top_p=0.6), dict(temperature=1e-10, min_p=0.3), dict(temperature=1e-10, top_k=2000)]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [100, 5003, 16384, 32768, 40001, 130560])
def test_sample_nearly_greedy(gpu, t, V):
    """Small temperatures beside masked tokens (-infinity, NaN, the type's lowest value) and what lies past a row's end:
    none of them weighs anything; of equal largest logits each weighs the same."""
    rng = np.random.default_rng(V)
    x = rng.standard_normal((5, V)).astype(np.float32)
    x[:, ::3] = -np.inf
    x[1, 1::5] = np.nan
    x[2, 2::3] = R.from_bits(R.to_bits(np.float32(-3.3e38 if t != "f16" else -65504), t), t)
    for r, n in ((1, 1), (2, 2), (3, 5), (4, 40)):              # this many largest logits, all equal
        x[r, 1 + 3 * rng.permutation(V // 3 - 1)[:min(n, V // 6)]] = 6.5
    sample_case(gpu, R.to_bits(x, t), t, [0.0, 0.3, 0.52, 0.56, 0.8, 1 - 2.0 ** -24], NEARLY_GREEDY)


def masses(l):
    """Float64 logits' tokens in their order and cumulative weights (extended precision, the largest logit's 1) at temperature 1."""
    order = np.lexsort((np.arange(len(l)), -l))
    return order, np.cumsum(np.exp(l[order] - l[order[0]]).astype(np.longdouble))


def kept_within(upto, top_p, off):
    """The least and the largest mass that top_p may keep where the row's is known to `off` of itself."""
    p = np.longdouble(np.float32(top_p))
    at = [np.searchsorted(upto, p * upto[-1] * (1 + s * off)) for s in (-1, 1)]
    return upto[at[0]], upto[min(at[1], len(upto) - 1)]


@pytest.mark.parametrize("V,tail", [(16384, 4.0), (16384, 6.5), (32768, 5.0)])
def test_sample_border_where_the_list_ends(gpu, V, tail):
    """top_p whose border is the last of the listed tokens to fp32's last bit.  A thread of a row of one launch has one of
    64 large logits of its wave, so the 41st of these (the 41 lanes that c = 64 (1 - e^(-1040 / 1024)) + 1 counts) is the
    first listed value's bound in each of the 16 waves; below come the other 23 lanes' and equal ones, whose weights fp32
    rounds alike.  Whatever side rounding puts the border on, what stays is top_p of the row's weight to 2^-19 of it, and
    a token more."""
    off = 2.0 ** -19
    rows, ps, known = [], [], []
    for i in range(64):
        x = np.full((V // 4, 4), -tail - i / 37, np.float32)
        for t in range(1024):
            x[t, (t * 7) % 4] = 2 - (t % 64) / 64
        x = x.reshape(-1)
        order, upto = masses(x.astype(np.float64))
        p = np.float32(upto[41 * 16 - 1] / upto[-1])
        rows += 7 * [x]
        known += 7 * [(order, upto)]
        ps += [np.float32(p + k * np.spacing(p)) for k in range(-3, 4)]
    print(f"sample border V {V} tail {tail}", flush=True)
    b, pp = dev(gpu, np.stack(rows)), dev(gpu, np.array(ps, np.float32))
    for u in (0.0, 0.5, 0.9, 0.99, 1 - 2.0 ** -24):
        tokens, probs = (a.numpy() for a in gpu.sample_rows(b, dev(gpu, np.full(len(rows), u, np.float32)), top_p=pp))
        for i, (order, upto) in enumerate(known):
            least, most = kept_within(upto, ps[i], off)
            at = int(np.flatnonzero(order == tokens[i])[0])
            w = upto[at] - (upto[at - 1] if at else 0)
            # (a probability rounds to fp32; cumulative weights are known to off as well)
            assert w / most * (1 - off - 2.0 ** -24) <= probs[i] <= w / least * (1 + off + 2.0 ** -24), (i, u, tokens[i], probs[i], w / most, w / least)
            assert upto[at] >= u * least * (1 - off) and upto[at] - w <= u * most * (1 + off), (i, u, tokens[i])


@pytest.mark.parametrize("t", ["f32", "f16"])
def test_sample_light_tail(gpu, t):
    """A million tokens of 2^-13 to 2^-33 of the largest's weight, below 16 that a slice lists (four lanes of each of its
    waves, and c = 64 (1 - e^(-1700 / 128 / 256)) + 1 = 4): together a third of the row.  What stays is known to 2^-19."""
    V, E, off = 1 << 20, 4 if t == "f32" else 8, 2.0 ** -19
    rng = np.random.default_rng(31)
    x = (1 - np.log(2) * rng.uniform(13, 33, V)).astype(np.float32)
    x[[E * (64 * w + i) for w in range(4) for i in range(4)]] = 1
    b = R.to_bits(x, t)
    order, upto = masses(R.from_bits(b, t).astype(np.float64))
    total = upto[-1]
    print(f"sample light tail {t} mass {float(total)}", flush=True)
    for settings, kept in ((dict(), (total, total)), (dict(top_p=0.95), kept_within(upto, 0.95, off))):
        least, most = kept
        for u in (0.0, 0.5, 0.8, 0.9, 0.99):
            uu = dev(gpu, np.array([u], np.float32))
            tokens, probs = (a.numpy() for a in gpu.sample_rows(dev(gpu, b[None]), uu, **settings))
            at = int(np.flatnonzero(order == tokens[0])[0])
            w = upto[at] - (upto[at - 1] if at else 0)
            # (and the token's weight to half a step of 2^-43)
            tol = w / total * (off + 2.0 ** -24) + 2.0 ** -44
            assert w / most - tol <= probs[0] <= w / least + tol, (settings, u, tokens[0], probs[0], w / most)
            u = float(np.float32(u))
            assert upto[at] >= u * least * (1 - off) and upto[at] - w <= u * most * (1 + off), (settings, u, tokens[0])


def test_sample_equal_tails_below_lists(gpu):
    """Thousands of equal tokens o = 9 to 13 octaves below the largest, with logits, temperatures and sums that round alike
    for each, below 41 listed ones of each wave (test_sample_border_where_the_list_ends) that lie as little above as 16
    bits tell.  The difference's and the product's rounding are ln 2 2^-24 o each, exp2's 2^-23; of a thread's eight chunks
    of four, whose own sums are exact, the sums of 3, 5, 6 and 7 round, 21 / 8 2^-24, and in 41 threads of 64, whose last
    chunk has three, the last two, (21 4 + 3 + 31) / 31: 3.4 on the average.  What is not in the tail is exact, the
    probability rounds once more."""
    V = 32768
    cases = [(6.903881072998047, 0.5513023138046265, 2.8222405910491943), (3.1673521995544434, 0.5426825881004333, -0.8532230854034424),
             (6.047861099243164, 1.0479786396026611, -1.9790167808532715), (8.076173782348633, 0.5354180932044983, 3.9715540409088135),
             (7.283297538757324, 0.5564096570014954, 3.1821577548980713), (5.566736221313477, 0.5240152478218079, 1.5442888736724854),
             (2.0830864906311035, 1.264405369758606, -6.6693010330200195), (0.5012397766113281, 1.1914342641830444, -7.728212833404541)]
    x = np.zeros((len(cases), V), np.float32)
    for i, (top, T, low) in enumerate(cases):
        u = np.array([low], np.float32).view(np.uint32)
        x[i] = low
        x[i, [4 * (7 * 1024 + t) for t in range(1024) if t % 64 < 41]] = (u + (1 << 16) & 0xFFFF0000 if low > 0 else (u & 0xFFFF0000) - 1).view(np.float32)[0]
        x[i, 0] = top
    T = np.array([c[1] for c in cases], np.float32)
    print("sample tails below lists", flush=True)
    tokens, probs = (a.numpy() for a in gpu.sample_rows(dev(gpu, x), dev(gpu, np.zeros(len(cases), np.float32)), temperature=dev(gpu, T)))
    for i in range(len(cases)):
        l = x[i].astype(np.float64)
        w = np.exp((l - l[0]) / float(T[i])).astype(np.longdouble)
        share = float(w[x[i] == x[i, 1]].sum() / w.sum())
        o = float(l[0] - l[1]) / float(T[i]) / np.log(2)
        tol = (share * (2 * np.log(2) * o + 2 + 3.4) + 1) * 2.0 ** -24
        assert tokens[i] == 0 and abs(probs[i] * w.sum() - 1) <= tol, (cases[i], probs[i], float(probs[i] * w.sum() - 1) * 2 ** 24, tol * 2 ** 24)


@pytest.mark.parametrize("t,V,stride", [("f32", 40000, 40000), ("bf16", 65536, 65536), ("f32", 33001, 33002), ("f16", 50001, 50003),
                                        ("bf16", 20000, 20000), ("bf16", 100000, 100000)])
def test_sample_rows_among_others(gpu, t, V, stride):
    """A row's token and probability are the same, to the last bit, among many rows, among few and alone."""
    rng = np.random.default_rng(V)
    rows = 160
    x = np.zeros((rows, stride), R.to_bits(np.zeros(1, np.float32), t).dtype)
    x[::2, :V], x[1::2, :V] = (logits_of(rng, rows // 2, V, t, kind) for kind in ("zipf", "flat"))
    # and equal tails, whose sums fp32 rounds all alike: 1300 tokens are listed
    for i in range(0, rows, 4):
        y = np.full(V, 1 - 7.5 - i / 97, np.float32)
        y[rng.permutation(V)[:1300]] = -6
        y[rng.integers(V)] = 1
        x[i, :V] = R.to_bits(y, t)
    b, u = dev(gpu, x), dev(gpu, (rng.random(rows) * (np.arange(rows) % 4 > 0)).astype(np.float32))
    p = dev(gpu, rng.choice(np.array([1.0, 0.9, 0.97], np.float32), rows))
    print(f"sample among others {t} {V}", flush=True)

    def call(first, n):
        tokens, probs = gpu.empty((n,), np.int32), gpu.empty((n,), np.float32)
        d = pf.SampleDesc(TYPE[t], V, stride, 0.8, 0, 1.0, 0.0, None, None, p.ptr + 4 * first, None)
        gpu.check(pf.lib().pf_sample_rows(gpu.h, C.byref(d), C.c_void_p(b.ptr + first * stride * x.itemsize), C.c_void_p(u.ptr + 4 * first), n,
                                          C.c_void_p(tokens.ptr), C.c_void_p(probs.ptr)), "pf_sample_rows")
        return tokens.numpy(), probs.numpy()

    tokens, probs = call(0, rows)
    for first, n in [(i, 1) for i in range(rows)] + [(0, 20), (20, 77), (97, 63)]:
        a, q = call(first, n)
        np.testing.assert_array_equal(a, tokens[first:first + n])
        np.testing.assert_array_equal(q.view(np.uint32), probs[first:first + n].view(np.uint32))


def test_sample_many_rows(gpu):
    """More rows than are taken at a time, with settings of their own."""
    rng = np.random.default_rng(12)
    rows, V = 65535, 7
    x = logits_of(rng, rows, V, "f16", "flat")
    u = rng.random(rows).astype(np.float32)
    k = rng.integers(0, 9, rows).astype(np.int32)
    temp = rng.choice(np.array([0, 0.5, 2], np.float32), rows)
    tokens, probs = (a.numpy() for a in gpu.sample_rows(dev(gpu, x), dev(gpu, u), temperature=dev(gpu, temp), top_k=dev(gpu, k)))
    f = R.from_bits(x, "f16")
    for i in list(range(0, rows, 97)) + [rows - 1, 60000, 60001]:
        token, prob = S.sample(f[i], u[i], temp[i], int(k[i]))
        assert tokens[i] == token and abs(probs[i] - prob) <= 2.0 ** -23 * prob + 2.0 ** -44, i


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [63, 64, 65, 513, 2048, 2049, 4096, 8200, 16383])
def test_sample_one_workgroup(gpu, t, V):
    """Rows of one launch, of few threads and of all, and top-k around what they list."""
    ks = [dict(top_k=k, top_p=p) for k in (2, 20, 300, 1024, 1025) for p in (1.0, 0.9)]
    for kind in ("zipf", "flat"):
        sample_case(gpu, logits_of(np.random.default_rng(V), 1, V, t, kind), t, U, SETTINGS[:8] + ks)


@pytest.mark.parametrize("t,V", [("bf16", 130560), ("f32", 130560), ("f16", 90001), ("bf16", 1 << 19)])
def test_sample_flat(gpu, t, V):
    """Borders and tokens among thousands of tokens of one bin, equal ones and different ones."""
    x = logits_of(np.random.default_rng(V + 1), 1, V, t, "flat")
    sample_case(gpu, x, t, [0.05, 0.3, 0.55, 0.8, 0.97, 1 - 2.0 ** -24],
                [dict(), dict(temperature=0.8, top_p=0.95), dict(top_p=0.4), dict(temperature=0.5), dict(min_p=0.03), dict(temperature=4.0, top_p=0.9)])


def test_sample_masked_slices(gpu):
    """Masks, infinities and NaN in rows of several workgroups."""
    V = 20003
    rng = np.random.default_rng(3)
    x = rng.standard_normal((8, V)).astype(np.float32)
    x[0, rng.permutation(V)[:V - 3]] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, V - 1] = -3e38
    x[3, ::2] = np.nan
    x[4, [7, 12000]] = np.inf
    x[5] = np.nan
    x[6] = np.where(np.arange(V) % 2, 3e38, -3e38)
    x[7, 5:] = np.finfo(np.float32).min
    sample_case(gpu, x, "f32", [0.0, 0.3, 0.7, 1 - 2.0 ** -24], SETTINGS)


def test_sample_many_sliced_rows(gpu):
    """More rows of several workgroups than have room for their lists at a time, with settings of their own."""
    rng = np.random.default_rng(13)
    rows, V = 2500, 16401
    x = np.tile(logits_of(rng, 50, V, "f16"), (50, 1))
    u = rng.random(rows).astype(np.float32)
    k = rng.integers(0, 60, rows).astype(np.int32)
    temp = rng.choice(np.array([0, 0.5, 1], np.float32), rows)
    tokens, probs = (a.numpy() for a in gpu.sample_rows(dev(gpu, x), dev(gpu, u), temperature=dev(gpu, temp), top_k=dev(gpu, k)))
    f = R.from_bits(x[:50], "f16")
    for i in list(range(0, rows, 61)) + list(range(rows - 520, rows, 13)):
        token, prob = S.sample(f[i % 50], u[i], temp[i], int(k[i]))
        assert tokens[i] == token and abs(probs[i] - prob) <= 2.0 ** -23 * prob + 2.0 ** -44, i


def test_sample_masked_long_rows(gpu):
    """Masks, infinities and NaN in rows of two launches."""
    V = 40003
    rng = np.random.default_rng(4)
    x = rng.standard_normal((8, V)).astype(np.float32)
    x[0, rng.permutation(V)[:V - 3]] = -np.inf
    x[1] = -np.inf
    x[2] = -np.inf
    x[2, V - 1] = -3e38
    x[3, ::2] = np.nan
    x[4, [7, 32000]] = np.inf
    x[5] = np.nan
    x[6] = np.where(np.arange(V) % 2, 3e38, -3e38)
    x[7, 5:] = np.finfo(np.float32).min
    sample_case(gpu, x, "f32", [0.0, 0.3, 0.7, 1 - 2.0 ** -24], SETTINGS)
    y = rng.choice(np.array([1.0, 1.5, 1.5, 2.0, -3.0], np.float32), (1, V))
    for t in ("f32", "bf16"):
        sample_case(gpu, R.to_bits(y, t), t, [0.0, 0.2, 0.4, 0.6, 0.8, 0.97],
                    [dict(), dict(top_k=3000), dict(top_k=9000, top_p=0.7), dict(top_p=0.3), dict(min_p=0.2, top_p=0.9), dict(top_k=1000)])


def test_sample_many_long_rows(gpu):
    """More rows of two launches than have room for their lists at a time, with settings of their own, rows that start anywhere."""
    rng = np.random.default_rng(14)
    rows, V, stride = 3700, 33001, 33003
    x = logits_of(rng, 20, V, "bf16")
    big = np.zeros((rows, stride), x.dtype)
    big[:, :V] = np.tile(x, (rows // 20, 1))
    u = rng.random(rows).astype(np.float32)
    k = rng.integers(0, 60, rows).astype(np.int32)
    temp = rng.choice(np.array([0, 0.5, 1], np.float32), rows)
    b, tokens, probs = dev(gpu, big), gpu.empty((rows,), np.int32), gpu.empty((rows,), np.float32)
    uu, kk, tt = dev(gpu, u), dev(gpu, k), dev(gpu, temp)
    d = pf.SampleDesc(TYPE["bf16"], V, stride, 1.0, 0, 1.0, 0, tt.ptr, kk.ptr, None, None)
    gpu.check(pf.lib().pf_sample_rows(gpu.h, C.byref(d), C.c_void_p(b.ptr), C.c_void_p(uu.ptr), rows, C.c_void_p(tokens.ptr),
                                      C.c_void_p(probs.ptr)), "pf_sample_rows")
    tokens, probs = tokens.numpy(), probs.numpy()
    f = R.from_bits(x, "bf16")
    for i in list(range(0, rows, 61)) + list(range(rows - 520, rows, 13)):
        token, prob = S.sample(f[i % 20], u[i], temp[i], int(k[i]))
        assert tokens[i] == token and abs(probs[i] - prob) <= 2.0 ** -23 * prob + 2.0 ** -44, i


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V,stride", [(16384, 16384), (16385, 16386), (24001, 24003), (32761, 32763), (32768, 32768), (32769, 32771)])
def test_sample_around_one_workgroup(gpu, t, V, stride):
    """Rows of 16 and of 32 tokens a thread, and the first that take two launches."""
    for kind in ("zipf", "flat"):
        sample_case(gpu, logits_of(np.random.default_rng(V), 2, V, t, kind), t, U, SETTINGS[:10], stride)


def test_sample_equal_tails(gpu):
    """Far below the largest logit a row's weight lies in equal ones, which fp32 rounds alike: a weight 2^-o of the largest's,
    o up to 32, is off by half a step of o, ln 2 2^-20, and by what exp2 is, 2^-23."""
    for t, V, d in (("f32", 16000, 9.7), ("bf16", 16000, 7.3125), ("bf16", 100000, 11.125), ("f32", 1 << 18, 17.3)):
        x = np.full((1, V), 1.0 - d, np.float32)
        x[0, V // 3] = 1.0
        b = R.to_bits(x, t)
        f = R.from_bits(b, t)
        u = np.array([0.0, 2.0 ** -24], np.float32)
        tokens, probs = (a.numpy() for a in gpu.sample_rows(dev(gpu, np.tile(b, (2, 1))), dev(gpu, u)))
        for i in range(2):
            token, prob = S.sample(f[0], u[i])
            assert tokens[i] == token and abs(probs[i] - prob) <= 2.0 ** -19.9 * prob, (t, V, d, probs[i], prob)


@pytest.mark.parametrize("kind", ["zipf", "flat"])
def test_sample_largest_vocabulary(gpu, kind):
    x = logits_of(np.random.default_rng(20), 1, 1 << 20, "f32", kind)
    for s in (dict(temperature=0.0), dict(top_k=50), dict(temperature=0.8, top_p=0.9), dict(), dict(top_k=5000, min_p=1e-3)):
        sample_case(gpu, x, "f32", [0.2, 0.8, 0.9999], [s])


def test_two_contexts_at_once(gpu):
    """Calls of two contexts under way together, each with its own scratch and stream: what each alone gives."""
    rng = np.random.default_rng(15)
    other = pf.Context(0)
    rot = [pf.Rotary(c, 64, interleaved=False) for c in (gpu, other)]
    want, runs = [], []
    for i, c in enumerate((gpu, other)):
        x, u = dev(c, logits_of(rng, 40, 40000, "bf16")), dev(c, rng.random(40).astype(np.float32))
        y, p = dev(c, rng.standard_normal((300, 6, 64)).astype(np.float32)), dev(c, np.arange(300, dtype=np.int32) * 977)
        out = c.empty((40,), np.int32), c.empty((40,), np.float32), c.empty((300, 6, 64), np.float32)
        a, b = c.sample_rows(x, u, temperature=0.9, top_p=0.97)
        want.append((a.numpy(), b.numpy(), rot[i].apply(y, p).numpy()))
        runs.append((c, rot[i], x, u, y, p, out))
    for _ in range(30):
        for c, r, x, u, y, p, out in runs:
            c.sample_rows(x, u, temperature=0.9, top_p=0.97, out=out[:2])
            r.apply(y, p, out=out[2])
    for (c, _, _, _, _, _, out), w in zip(runs, want):
        c.synchronize()
        for a, b in zip(out, w):
            np.testing.assert_array_equal(a.numpy(), b)
    for r in rot:
        r.close()
    other.close()


def test_sample_refusals(gpu):
    L = pf.lib()
    x, u, o, p = gpu.empty((4, 100), np.float32), dev(gpu, np.zeros(4, np.float32)), gpu.empty((4,), np.int32), gpu.empty((4,), np.float32)
    x = dev(gpu, np.zeros((4, 100), np.float32))

    def call(code, type=pf.TYPE_F32, V=100, stride=0, l=x.ptr, uu=u.ptr, rows=4, out=o.ptr, probs=p.ptr, **kw):
        d = pf.SampleDesc(type, V, stride, 1.0, 0, 1.0, 0.0, **kw)
        v = [C.c_void_p(i) if i else None for i in (l, uu, out, probs)]
        rc = L.pf_sample_rows(gpu.h, C.byref(d), v[0], v[1], rows, v[2], v[3])
        assert rc == code, (rc, L.pf_last_error(gpu.h))

    call(0)
    call(0, probs=None)
    call(0, rows=0, l=None, uu=None, out=None, probs=None)
    call(-1, type=pf.TYPE_I8)
    call(-4, V=0)
    call(-4, V=(1 << 20) + 1)
    call(-1, stride=99)
    call(-4, rows=65536)
    call(-1, l=None)
    call(-1, uu=None)
    call(-1, out=None)
    call(-1, l=x.ptr + 2)
    call(-1, uu=u.ptr + 2)
    call(-1, top_k_dev=o.ptr + 1)
    call(-1, out=x.ptr + 16)
    call(-1, probs=u.ptr)
    call(-1, out=p.ptr)
    call(-1, top_p_dev=p.ptr)
    assert L.pf_sample_rows(gpu.h, None, None, None, 1, None, None) == -1
    f = np.float32
    for bad in (lambda: gpu.sample_rows(x, dev(gpu, np.zeros(5, f))), lambda: gpu.sample_rows(x, u, top_k=u), lambda: gpu.sample_rows(x, u, top_k=-1),
                lambda: gpu.sample_rows(x, u, temperature=o), lambda: gpu.sample_rows(dev(gpu, np.zeros((4, 100, 1), f)), u),
                lambda: gpu.sample_rows(x, u, out=(p, o)), lambda: gpu.sample_rows(np.zeros((4, 100), f), u)):
        with pytest.raises(pf.PFError):
            bad()


# --------------------------------------------------------- a serving loop's run

@pytest.mark.parametrize("ct", ["fp4", "i8"])
def test_serving_steps(gpu, ct):
    """Prompts and steps of a small model's one layer: turn and store, attend over the pages, unembed, sample; rejected
    rows truncated; against the same in float64."""
    H, G, D, V = 4, 2, 64, 500
    rng = np.random.default_rng(6)
    wq, wk, wv = (rng.standard_normal((V, h, D)).astype(np.float32) for h in (H, G, G))   # a token's rows
    un = rng.standard_normal((H * D, V)).astype(np.float32) / 8
    c = pf.PagedCache(gpu, 1, G, D, 40, 3, 200, 16, TYPE[ct])
    rot = pf.Rotary(gpu, D, interleaved=False)
    seqs = [0, 1, 2]
    text = [list(rng.integers(0, V, n)) for n in (5, 40, 17)]
    rows = [len(x) for x in text]

    def held(x):
        if ct == "fp4":
            return S.fp4_held(x)
        codes, scale = R.quantize_rows(x)
        return codes.astype(np.float64) * scale

    for step in range(6):
        c.append(seqs, rows)
        new = np.concatenate([x[-r:] for x, r in zip(text, rows)])
        y = c.store_rotary(0, rot, dev(gpu, wq[new]), dev(gpu, wk[new]), dev(gpu, wv[new]))
        o = c.attention(0, y).numpy()
        last = np.cumsum(rows) - 1
        logits = (o[last].reshape(3, -1) @ un).astype(np.float32)
        u = rng.random(3).astype(np.float32)
        tokens, _ = gpu.sample_rows(dev(gpu, logits), dev(gpu, u), temperature=0.9, top_k=100, top_p=0.9)
        for i, x in enumerate(text):
            at = np.arange(len(x))
            q, _ = S.turned(wq[x].astype(np.float64), at, D, False)
            k, _ = S.turned(wk[x].astype(np.float64), at, D, False)
            k, v = held(k.astype(np.float32)), held(wv[x])
            q = q.astype(np.float32).astype(np.float64)
            want, tol = R.attend(q[-rows[i]:], k, v, R.visible(rows[i], len(x)), R.default_scale(D), "f32", ct == "i8")
            # (a turned query is off by up to 6 e of its pair's two values and e of itself, a score by D products of
            # that, a weight by twice a score's)
            more = 2 * D * 13 * 2.0 ** -24 * np.abs(q).max() * np.abs(k).max() * R.default_scale(D) * np.abs(v).max()
            R.check(o[last[i] + 1 - rows[i]:last[i] + 1], want, tol + more, f"step {step} sequence {i}")
            assert tokens.numpy()[i] == S.sample(logits[i].astype(np.float64), u[i], 0.9, 100, 0.9)[0]
        for x, t in zip(text, tokens.numpy()):
            x.append(int(t))
        rows = [1, 1, 1]
        if step == 3:                            # a verify pass whose last row is rejected
            for x in text:
                x.append(int(rng.integers(0, V)))
            rows = [2, 2, 2]
        if step == 4:
            c.truncate(seqs, [len(x) - 2 for x in text])
            for x in text:
                del x[-2:]
                x.append(int(rng.integers(0, V)))
    c.close()
    rot.close()
