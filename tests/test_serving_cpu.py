"""What the entry points of a serving step answer without a GPU: NULL handles,
the Python binding's argument checks, and the tests' own formulas."""
import ctypes as C

import numpy as np
import pytest

import pocketforge_amd as pf
import serving_ref as S


def test_null_handles():
    L = pf.lib()
    assert L.pf_rotary_create(None, None, None) == -1
    L.pf_rotary_destroy(None)
    assert L.pf_rotary_apply(None, pf.TYPE_F32, 1, None, None, None, 0, 0, 0) == -1
    assert L.pf_pages_store_rotary(None, 0, None, pf.TYPE_F32, 1, None, None, None, None, 0, 0, 0, 0) == -1
    assert L.pf_sample_rows(None, None, None, None, 0, None, None) == -1
    assert L.pf_sample_rows(None, C.byref(pf.SampleDesc()), None, None, 0, None, None) == -1


def array(shape, dtype, ctx, ptr=4096):
    a = pf.DeviceArray.__new__(pf.DeviceArray)
    a.ctx, a.ptr, a.shape, a.dtype = ctx, ptr, shape, np.dtype(dtype)
    return a


def context(device=0):
    ctx = pf.Context.__new__(pf.Context)
    ctx.device, ctx.h = device, None
    return ctx


def test_matrices_and_columns():
    ctx = context()
    assert pf._matrix(array((3, 70), np.float32, ctx), "x", ctx) == (3, 70, 70)
    assert pf._column(array((3,), np.int32, ctx), "k", 3, "int32", ctx) == 4096
    for bad in (array((3, 70, 1), np.float32, ctx), array((3,), np.float32, ctx), np.zeros((3, 70)), None,
                array((3, 70), np.float32, context(1)), array((3, 70), np.float32, ctx, None)):
        with pytest.raises(pf.PFError):
            pf._matrix(bad, "x", ctx)
    for bad in (array((4,), np.int32, ctx), array((3, 1), np.int32, ctx), array((3,), np.float32, ctx), array((3,), np.int64, ctx),
                array((3,), np.int32, context(1)), np.zeros(3, np.int32), [1, 2, 3]):
        with pytest.raises(pf.PFError):
            pf._column(bad, "k", 3, "int32", ctx)
    torch = pytest.importorskip("torch")

    class On:
        """A tensor's shape and strides, on a GPU."""

        def __init__(self, t):
            self.t, self.shape, self.dtype = t, t.shape, t.dtype

        def get_device(self):
            return 0

        def is_contiguous(self):
            return self.t.is_contiguous()

        def stride(self, *d):
            return self.t.stride(*d)

        def data_ptr(self):
            return 64

    x = torch.zeros((6, 40))
    assert pf._matrix(On(x), "x", ctx) == (6, 40, 40) and pf._matrix(On(x[::2, :30]), "x", ctx) == (3, 30, 80)
    assert pf._matrix(On(x[:1]), "x", ctx) == (1, 40, 40)
    for bad in (x.t(), x[:, ::2], x[:1].expand(6, 40), x[:1, ::2]):
        with pytest.raises(pf.PFError):
            pf._matrix(On(bad), "x", ctx)
    u = torch.zeros(12)
    assert pf._column(On(u), "u", 12, "float32", ctx) == 64
    for bad in (u[::2], u[:1].expand(6), u[:6].double()):
        with pytest.raises(pf.PFError):
            pf._column(On(bad), "u", 6, "float32", ctx)
    with pytest.raises(pf.PFError):
        pf._column(u, "u", 12, "float32", ctx)


def test_calls_refused_by_the_binding():
    ctx = context()
    x, u = array((2, 50), np.float32, ctx), array((2,), np.float32, ctx)
    o = array((2,), np.int32, ctx), array((2,), np.float32, ctx)
    for kw in (dict(top_k=-1), dict(top_k=1 << 32), dict(top_k=u), dict(temperature=o[0]), dict(top_p=array((3,), np.float32, ctx)),
               dict(min_p=None), dict(out=(u, u)), dict(out=(o[0], o[0]))):
        with pytest.raises(pf.PFError):
            ctx.sample_rows(x, u, **dict(dict(out=o), **kw))
    with pytest.raises(pf.PFError):
        ctx.sample_rows(array((2, 50), np.int32, ctx), u, out=o)
    for kw in (dict(head_dim=-1), dict(head_dim=64, turn=-8), dict(head_dim=64, original=1 << 32)):
        with pytest.raises(pf.PFError):
            pf.Rotary(ctx, **kw)
    rot = pf.Rotary.__new__(pf.Rotary)
    rot.ctx, rot.h, rot.head_dim = ctx, None, 64
    q, at = array((2, 4, 64), np.float16, ctx), array((2,), np.int32, ctx)
    for a in ((q, u, q), (q, array((3,), np.int32, ctx), q), (array((2, 4, 48), np.float16, ctx), at, q), (q, at, array((2, 4, 64), np.float32, ctx)),
              (q, at, array((2, 3, 64), np.float16, ctx)), (np.zeros((2, 4, 64), np.float16), at, q)):
        with pytest.raises(pf.PFError):
            rot.apply(a[0], a[1], out=a[2])
    c = pf.PagedCache.__new__(pf.PagedCache)
    c.ctx, c.h, c.pass_rows, c.n_kv_heads, c.head_dim, c.max_seqs, c.n_layers = ctx, None, 2, 2, 64, 3, 2
    k = array((2, 2, 64), np.float16, ctx)
    for a in ((q, k, q), (q, q, k), (array((3, 4, 64), np.float16, ctx), k, k), (array((2, 4, 64), np.float32, ctx), k, k)):
        with pytest.raises(pf.PFError):
            c.store_rotary(0, rot, *a, out=q)
    for layer in (-1, 1 << 32):
        with pytest.raises(pf.PFError):
            c.store_rotary(layer, rot, q, k, k, out=q)


def test_closed_after_the_context(monkeypatch):
    """A cache or a rotary handle that outlives its context does not reach into it."""
    called = []

    class Lib:
        pf_pages_destroy = pf_rotary_destroy = staticmethod(lambda h: called.append(h))

    monkeypatch.setattr(pf, "lib", Lib)
    for kind in (pf.PagedCache, pf.Rotary):
        for h, calls in ((None, []), (1234, [5678])):
            x = kind.__new__(kind)
            x.ctx, x.h = context(), 5678
            x.ctx.h = h
            del called[:]
            x.close()
            assert called == calls and x.h is None
            x.close()
            assert called == calls


def test_reference_codes():
    """The search against the rule in bits, and ties."""
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((300, 32)) * 2.0 ** rng.integers(-130, 127, (300, 1))).astype(np.float32)
    x[0] = 0
    x[1, 0], x[2, 3] = np.inf, np.nan
    x[3] = [1.75 if i == 0 else 0.1 for i in range(32)]
    x[4] = np.nextafter(np.float32(1.75), np.float32(2))
    code, e = S.fp4_rows(x)
    top = np.abs(x).max(-1)
    want = np.clip(((top.view(np.uint32).astype(np.int64) + 0x1FFFFF) >> 23) - 2, 2, 252)
    want[[1, 2]] = 255
    np.testing.assert_array_equal(e[:, 0], want)
    assert e[3, 0] == 125 and e[4, 0] == 126
    v = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6.9, -0.25, -5.1, 4], np.float32)
    row = np.zeros(32, np.float32)
    row[:11] = v
    assert S.fp4_held(row)[:11].tolist() == [0, 1, 1, 2, 2, 4, 4, 6, -0.0, -6, 4]


def test_reference_turn():
    """Against a complex product, and lengths of pairs."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 2, 12))
    at = [0, 3, 1000, -7]
    for inter in (True, False):
        y, size = S.turned(x, at, 8, inter, base=100.0)
        f = 100.0 ** (-np.arange(4) / 4)
        a = (slice(0, 8, 2), slice(1, 8, 2)) if inter else (slice(0, 4), slice(4, 8))
        z = (x[..., a[0]] + 1j * x[..., a[1]]) * np.exp(1j * np.array(at)[:, None, None] * f)
        np.testing.assert_allclose(y[..., a[0]].astype(float), z.real, atol=1e-12)
        np.testing.assert_allclose(y[..., a[1]].astype(float), z.imag, atol=1e-12)
        np.testing.assert_array_equal(y[..., 8:].astype(float), x[..., 8:])
        assert (size[..., 8:] == 0).all()
    f = S.frequencies(64, 1e4, 8.0, 1.0, 4.0, 4096)
    plain = S.frequencies(64, 1e4)
    assert f[0] == plain[0] and abs(f[-1] / plain[-1] - 0.125) < 1e-12 and (np.diff((f / plain).astype(float)) <= 1e-15).all()


def test_reference_sample():
    """Against a direct walk, one filter after the other."""
    rng = np.random.default_rng(2)
    for trial in range(300):
        n = int(rng.integers(1, 12))
        l = np.round(rng.standard_normal(n) * 3) / 2
        kw = dict(temperature=float(rng.choice([0.5, 1, 2])), top_k=int(rng.integers(0, n + 2)),
                  top_p=float(rng.choice([1, 0.9, 0.5, 0.1])), min_p=float(rng.choice([0, 0.1, 0.6])))
        u = float(np.float32(rng.random()))
        order = sorted(range(n), key=lambda i: (-l[i], i))
        w = [np.exp((l[i] - l[order[0]]) / kw["temperature"]) for i in order]
        m = n if not 0 < kw["top_k"] < n else kw["top_k"]
        order, w = order[:m], w[:m]
        if kw["top_p"] < 1:
            p = float(np.float32(kw["top_p"]))
            m = next(j + 1 for j in range(m) if sum(w[:j + 1]) >= p * sum(w) - 1e-12)
            order, w = order[:m], w[:m]
        keep = [j for j in range(m) if w[j] >= np.float32(kw["min_p"])]
        order, w = [order[j] for j in keep], [w[j] for j in keep]
        at = next(j for j in range(len(w)) if sum(w[:j + 1]) > u * sum(w))
        token, prob = S.sample(l, u, **kw)
        assert token == order[at] and abs(prob - w[at] / sum(w)) < 1e-12
    assert S.sample(np.array([1, 3, 3.0]), 0.9, 0.0) == (1, 1.0) and S.sample(np.array([-np.inf, np.nan]), 0.5) == (-1, 0.0)


def test_reference_bound_of_the_largest():
    """A block's largest value comes out between four fifths (5 powers, a tie, go to 4) and below six fifths of itself (the
    next value above 5 goes to 6), and no value is off by more than the block's power of two."""
    x = np.zeros((3000, 32), np.float32)
    x[:, 0] = np.geomspace(1, 64, 3000)
    x[:3, 0] = 5, np.nextafter(np.float32(5), np.float32(6)), 7
    x[:, 1:] = np.random.default_rng(3).uniform(-1, 1, (3000, 31)) * x[:, :1]
    code, e = S.fp4_rows(x)
    held = S.fp4_values(code, e, 32)
    r = held[:, 0] / x[:, 0].astype(np.float64)
    assert r.min() == r[0] == 0.8 and r.max() == r[1] < 1.2 and r[1] > 1.2 - 1e-6 and r[2] == 6 / 7
    assert (np.abs(held - x) <= 2.0 ** (e.astype(np.float64) - 127)).all()


def pages_plan(t, cache, H, G, D, rows, lens):
    """(waves of a workgroup, whether the keys are cut, workgroups on a compute unit) of a pass over pages of a type."""
    d = pf.AttnDesc(t, H, G, D, 1, 0, 0, 0.0, 0, 0, 0, 0)
    x = [C.c_uint32() for _ in range(4)]
    a, b = ((C.c_uint32 * len(y))(*y) for y in (rows, lens))
    assert pf.lib().pf_test_pages_plan_of(C.byref(d), cache, a, b, len(lens), *map(C.byref, x)) == 0
    return x[0].value, x[1].value < x[2].value, x[3].value


def test_plans_of_4_bit_pages():
    """What 4-bit pages take otherwise than wider ones: a third workgroup on a compute unit from 24 tiles a wave of two on
    (24 4 2 256 = 49152 tiles, 33 of each of 24 heads: 62 contexts are fewer, 63 more), and joins priced twice as high."""
    bf, f32, i8, fp4 = pf.TYPE_BF16, pf.TYPE_F32, pf.TYPE_I8, pf.TYPE_FP4
    for n, held in ((62, 2), (63, 3), (64, 3)):
        assert pages_plan(bf, fp4, 24, 24, 128, [1] * n, [1025] * n) == (4, False, held)
        assert pages_plan(bf, i8, 24, 24, 128, [1] * n, [1025] * n) == (4, False, 2)
    many = [4100 + 187 * i for i in range(64)]
    assert pages_plan(bf, fp4, 16, 4, 128, [1] * 64, many) == (4, True, 3)
    assert pages_plan(bf, i8, 16, 4, 128, [1] * 64, many) == (4, True, 2)
    assert pages_plan(pf.TYPE_F16, fp4, 16, 2, 128, [1, 1], [120000, 64000]) == (4, True, 2)
    # two tiles of 16 rows: two workgroups, however many tiles
    assert pages_plan(bf, fp4, 40, 2, 128, [1] * 64, [16000] * 64)[2] == 2
    assert pages_plan(bf, fp4, 16, 16, 128, [1], [700]) == (8, False, 2) and pages_plan(bf, i8, 16, 16, 128, [1], [700]) == (4, True, 2)
    assert pages_plan(bf, fp4, 16, 16, 128, [1], [4000])[1] and pages_plan(f32, fp4, 16, 16, 128, [5] * 16, [2100] * 16) == (8, False, 2)
