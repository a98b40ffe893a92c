"""Attention over packed prompts and over paged caches, and the pages'
bookkeeping, against float64 on the host: types, head layouts, lengths from
nothing to several tiles, odd sizes, strides, windows with sinks, values that
are not finite in masked places, and the calls that are refused."""
import ctypes as C

import numpy as np
import pytest

import attention_ref as R
import pocketforge_amd as pf

pytestmark = pytest.mark.gpu

TYPE = {"f32": pf.TYPE_F32, "f16": pf.TYPE_F16, "bf16": pf.TYPE_BF16, "i8": pf.TYPE_I8}


def dev(ctx, a):
    return pf.DeviceArray.from_numpy(ctx, a)


def prompt_case(gpu, t, H, G, D, ql, kl, causal=True, window=0, sink=0, scale=0.0, edit=None, seed=0):
    rng = np.random.default_rng(seed)
    q, k, v = (R.rand(rng, (sum(n), h, D), t) for n, h in ((ql, H), (kl, G), (kl, G)))
    if edit:
        edit(q, k, v)
    print(f"prompt {t} H {H} G {G} D {D} q {ql[:6]} k {kl[:6]} causal {causal} window {window} sink {sink}", flush=True)
    y = gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), ql, kl, causal, window, sink, scale).numpy()
    y = R.from_bits(y, t)
    q, k, v = (R.from_bits(x, t) for x in (q, k, v))
    qa = ka = 0
    for s, (a, b) in enumerate(zip(ql, kl)):
        want, tol = R.attend(q[qa:qa + a], k[ka:ka + b], v[ka:ka + b], R.visible(a, b, causal, window, sink),
                             scale or R.default_scale(D), t)
        R.check(y[qa:qa + a], want, tol, f"sequence {s}")
        qa, ka = qa + a, ka + b
    return y


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,G,D,lens", [
    (4, 4, 64, [1]), (2, 1, 128, [31, 32, 33]), (16, 2, 128, [64, 65, 0, 127, 128, 129]), (3, 3, 16, [7, 200]),
    (6, 2, 80, [1, 1, 300]), (5, 1, 112, [0, 257]), (2, 2, 48, [130]),
])
def test_prompt(gpu, t, H, G, D, lens):
    prompt_case(gpu, t, H, G, D, lens, lens)


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("ql,kl,causal,window,sink", [
    ([5, 1, 140], [77, 300, 513], True, 0, 0),            # a cached prefix
    ([40, 3, 9], [10, 0, 9], True, 0, 0),                 # queries before the first key see nothing
    ([40, 3, 0, 2], [10, 0, 70, 130], False, 0, 0),       # every key, or none
    ([300], [300], True, 1, 0), ([300], [300], True, 64, 4), ([300, 200], [700, 900], True, 100, 70),
    ([260], [500], True, 33, 1000), ([100], [400], False, 50, 3), ([200], [200], True, 4000, 4),
])
def test_prompt_masks(gpu, t, ql, kl, causal, window, sink):
    prompt_case(gpu, t, 4, 2, 64, ql, kl, causal, window, sink)


def test_prompt_many_sequences(gpu):
    lens = [(7 * i) % 37 for i in range(150)]
    prompt_case(gpu, "bf16", 2, 1, 64, lens, [n + i % 5 for i, n in enumerate(lens)])


def test_prompt_large_scores(gpu):
    """Scores of hundreds: the weights of all but a few keys vanish."""
    def edit(q, k, v):
        q[:] = R.to_bits(R.from_bits(q, "f16") * 30, "f16")
    prompt_case(gpu, "f16", 2, 2, 64, [150], [150], edit=edit)
    prompt_case(gpu, "bf16", 2, 2, 64, [150], [150], scale=0.001)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_prompt_not_finite(gpu, t):
    """An infinity or a NaN in a key's or value's row stays out of the queries
    that do not see it; those that see the value get what the formula says."""
    rng = np.random.default_rng(3)
    n, H, D, at = 200, 2, 64, 100
    for bad in (np.inf, -np.inf, np.nan):
        q, k, v = (R.rand(rng, (n, H, D), t) for _ in range(3))
        v[at, 0, 5] = R.to_bits(np.float32(bad), t)
        k[at + 20, 1, 7] = R.to_bits(np.float32(np.nan), t)
        y = R.from_bits(gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), [n]).numpy(), t)
        q, k, v = (R.from_bits(x, t) for x in (q, k, v))
        want, tol = R.attend(q, k, v, R.visible(n, n), R.default_scale(D), t)
        R.check(y[:at], want[:at], tol[:at])
        R.check(y[:at + 20, 1], want[:at + 20, 1], tol[:at + 20, 1])
        assert np.isnan(y[at + 20:, 1]).all()
        rest = np.arange(D) != 5
        R.check(y[at:, 0][:, rest], want[at:, 0][:, rest], tol[at:, 0][:, rest])
        assert not np.isfinite(y[at:, 0, 5]).any()
        if t != "f32":
            np.testing.assert_array_equal(y[at:, 0, 5], bad)


def test_prompt_empty_rows_beside_nan(gpu):
    """Queries that see no key get zeros, whatever the keys hold."""
    def edit(q, k, v):
        v[:] = R.to_bits(np.full(v.shape, np.nan, np.float32), "bf16")
    y = prompt_case(gpu, "bf16", 2, 2, 64, [20], [4], edit=edit)
    assert (y[:16] == 0).all() and np.isnan(y[16:]).all()


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_prompt_strides(gpu, t):
    """Rows of a fused q|k|v buffer, and output rows apart: what lies between them stays."""
    rng = np.random.default_rng(5)
    n, H, G, D = 70, 4, 2, 64
    w = (H + 2 * G) * D
    x = R.rand(rng, (n, w), t)
    o = np.full((n, H * D + 32), 7, R.DTYPE[t])
    xd, od = dev(gpu, x), dev(gpu, o)
    es = x.itemsize
    d = pf.AttnDesc(TYPE[t], H, G, D, 1, 0, 0, 0.0, w, w, w, H * D + 32)
    lens = (C.c_uint32 * 1)(n)
    gpu.check(pf.lib().pf_prompt_attention(gpu.h, C.byref(d), C.c_void_p(xd.ptr), C.c_void_p(xd.ptr + H * D * es),
                                           C.c_void_p(xd.ptr + (H + G) * D * es), C.c_void_p(od.ptr), lens, None, 1),
              "pf_prompt_attention")
    y = od.numpy()
    assert (y[:, H * D:] == 7).all()
    x = R.from_bits(x, t)
    want, tol = R.attend(x[:, :H * D].reshape(n, H, D), x[:, H * D:(H + G) * D].reshape(n, G, D),
                         x[:, (H + G) * D:].reshape(n, G, D), R.visible(n, n), R.default_scale(D), t)
    R.check(R.from_bits(y[:, :H * D], t).reshape(n, H, D), want, tol)


def test_prompt_refusals(gpu):
    n, H, D = 8, 4, 64
    b = [gpu.empty((n, H, D), np.float16) for _ in range(4)]
    lens = (C.c_uint32 * 2)(n, 0)

    def call(code, bufs=None, lens=lens, nseq=2, **kw):
        f = dict(type=pf.TYPE_F16, n_heads=H, n_kv_heads=H, head_dim=D, causal=1, window=0, sink=0, scale=0.0,
                 q_stride=0, k_stride=0, v_stride=0, o_stride=0)
        f.update(kw)
        d = pf.AttnDesc(**f)
        p = [C.c_void_p(x) if x else None for x in (bufs or [x.ptr for x in b])]
        rc = pf.lib().pf_prompt_attention(gpu.h, C.byref(d), *p, lens, None, nseq)
        assert rc == code, (rc, pf.lib().pf_last_error(gpu.h))

    call(0)
    call(0, nseq=0)
    call(-1, type=7)
    call(-1, type=pf.TYPE_I8)
    call(-1, n_kv_heads=3)
    call(-1, n_heads=0)
    call(-1, n_kv_heads=0)
    call(-4, head_dim=72)
    call(-4, head_dim=256)
    call(-1, scale=-1.0)
    call(-1, scale=float("nan"))
    call(-1, q_stride=H * D - 8)
    call(-1, k_stride=H * D + 1)
    q, k, v, o = (x.ptr for x in b)
    call(-1, bufs=[q, k, v, None])
    call(-1, bufs=[q + 2, k, v, o])
    call(-1, bufs=[q, k, v, q + 16])
    call(-1, bufs=[q, k, v, v])
    call(-1, lens=None)
    call(-4, lens=(C.c_uint32 * 2)(0xFFFFFFFF, 0))
    lib = pf.lib()
    assert lib.pf_prompt_attention(None, None, None, None, None, None, None, None, 0) == -1
    with pytest.raises(pf.PFError):
        gpu.prompt_attention(b[0], b[1], b[2], [n + 1])
    with pytest.raises(pf.PFError):
        gpu.prompt_attention(b[0], gpu.empty((n, H, D), np.float32), b[2], [n])


# -------------------------------------------------------------- paged cache

class Mirror:
    """A PagedCache beside the rows that each sequence should hold (float64)."""

    def __init__(self, gpu, ct, G, D, page, pages, seqs, context, layers=1, t=None):
        self.gpu, self.ct, self.G, self.D, self.layers = gpu, ct, G, D, layers
        self.t = t or (ct if ct != "i8" else "f32")
        self.c = pf.PagedCache(gpu, layers, G, D, pages, seqs, context, page, TYPE[ct])
        self.rows = [[(np.zeros((0, G, D)), np.zeros((0, G, D))) for _ in range(layers)] for _ in range(seqs)]
        self.rng = np.random.default_rng(17)

    def held(self, x):
        """What the cache holds of rows of type self.t."""
        if self.ct == "i8":
            c, s = R.quantize_rows(R.from_bits(x, self.t))
            return c.astype(np.float64) * s
        return R.from_bits(R.to_bits(R.from_bits(x, self.t), self.ct), self.ct)

    def append(self, seqs, rows, data=None):
        self.c.append(seqs, rows)
        new = []
        for l in range(self.layers):
            k, v = data or (R.rand(self.rng, (sum(rows), self.G, self.D), self.t, 1.5) for _ in range(2))
            self.c.store(l, dev(self.gpu, k), dev(self.gpu, v))
            new.append((self.held(k), self.held(v)))
        at = 0
        for s, n in zip(seqs, rows):
            for l in range(self.layers):
                self.rows[s][l] = tuple(np.concatenate([a, b[at:at + n]]) for a, b in zip(self.rows[s][l], new[l]))
            at += n

    def attention(self, H, seqs, rows, layer=0, t=None, **kw):
        t = t or self.t
        q = R.rand(self.rng, (sum(rows), H, self.D), t)
        y = R.from_bits(self.c.attention(layer, dev(self.gpu, q), **kw).numpy(), t)
        q = R.from_bits(q, t)
        scale = kw.pop("scale", 0.0) or R.default_scale(self.D)
        at = 0
        for s, n in zip(seqs, rows):
            k, v = self.rows[s][layer]
            want, tol = R.attend(q[at:at + n], k, v, R.visible(n, len(k), **kw), scale, t, self.ct == "i8")
            R.check(y[at:at + n], want, tol, f"sequence {s}")
            at += n

    def check(self, seqs):
        for l in range(self.layers):
            got = self.c.gather(l, seqs)
            for g, w in zip(got, (0, 1)):
                want = np.concatenate([self.rows[s][l][w] for s in seqs])
                np.testing.assert_array_equal(g.numpy(), want.astype(np.float32), err_msg=f"layer {l}")


COMBOS = [("bf16", "bf16"), ("f16", "f16"), ("f32", "i8"), ("bf16", "i8"), ("f16", "i8"), ("f32", "bf16")]


@pytest.mark.parametrize("t,ct", COMBOS)
@pytest.mark.parametrize("H,G,D,page,lens,new", [
    (4, 4, 64, 16, [1], 1), (8, 2, 128, 64, [63, 64, 65, 200], 1), (16, 1, 64, 32, [31, 700], 1),
    (6, 3, 80, 16, [5, 130, 33], 5), (16, 2, 128, 128, [900, 8], 5), (32, 1, 112, 256, [300], 3),
    (2, 2, 16, 16, [40, 9], 8), (12, 12, 64, 64, [70], 20),
])
def test_paged_attention(gpu, t, ct, H, G, D, page, lens, new):
    pages = sum(-(-n // page) for n in lens)
    m = Mirror(gpu, ct, G, D, page, pages, len(lens), max(lens), t=t)
    seqs = list(range(len(lens)))
    print(f"paged {t} over {ct} H {H} G {G} D {D} page {page} lens {lens} new {new}", flush=True)
    old = [max(0, n - new) for n in lens]
    for part in (3, 2, 1):       # grown in turn, so that their pages interleave
        m.append(seqs, [n // 3 if part > 1 else n - 2 * (n // 3) for n in old])
    m.append(seqs, [n - o for n, o in zip(lens, old)])
    assert m.c.free_pages == 0
    m.check(seqs)
    m.attention(H, seqs, [n - o for n, o in zip(lens, old)])
    m.c.close()


@pytest.mark.parametrize("t,ct", [("bf16", "bf16"), ("f32", "i8")])
@pytest.mark.parametrize("window,sink,causal", [(1, 0, True), (64, 4, True), (100, 70, True), (33, 500, True),
                                                (0, 0, False), (50, 3, False), (5000, 4, True)])
def test_paged_masks(gpu, t, ct, window, sink, causal):
    lens, new = [1, 40, 333, 700], [1, 6, 6, 0]
    m = Mirror(gpu, ct, 2, 64, 32, 80, 4, 1000, t=t)
    m.append([0, 1, 2, 3], [n - a for n, a in zip(lens, new)])
    m.append([3, 1, 0, 2], [new[i] for i in (3, 1, 0, 2)])
    m.attention(4, [3, 1, 0, 2], [new[i] for i in (3, 1, 0, 2)], causal=causal, window=window, sink=sink)
    m.c.close()


@pytest.mark.parametrize("t,ct", [("bf16", "bf16"), ("f32", "i8")])
def test_paged_split(gpu, t, ct):
    """Contexts long enough to be shared among workgroups, beside short ones; scale given; a second layer."""
    m = Mirror(gpu, ct, 2, 128, 64, 260, 5, 9000, layers=2, t=t)
    lens, new = [9000, 1, 2500, 0, 700], [2, 1, 3, 0, 1]
    m.append(list(range(5)), [a - b for a, b in zip(lens, new)])
    m.append([4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)])
    for layer in (0, 1):
        m.attention(8, [4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)], layer=layer, scale=0.05)
    m.attention(8, [4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)], window=3000, sink=4)
    m.attention(2, [4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)])
    m.c.close()


def test_paged_many_sequences(gpu):
    """More sequences than a wave looks at at once, with rows of different counts and none."""
    n = 300
    m = Mirror(gpu, "bf16", 1, 64, 16, 3000, n, 200)
    lens = [(13 * i) % 90 for i in range(n)]
    m.append(list(range(n)), lens)
    order = [(7 * i) % n for i in range(n)]
    new = [i % 4 for i in range(n)]
    m.append(order, new)
    m.check(order)
    m.attention(2, order, new)
    m.c.close()


@pytest.mark.parametrize("ct", ["bf16", "f16"])
def test_paged_not_finite(gpu, ct):
    """Infinities and NaN in rows of a verify pass's later drafts stay out of the earlier ones, and those that a
    shortened sequence leaves behind in its page out of all."""
    m = Mirror(gpu, ct, 1, 64, 64, 4, 1, 200)
    m.append([0], [30])
    bad = [R.rand(m.rng, (6, 1, 64), ct) for _ in range(2)]
    for b in bad:
        b[3:] = R.to_bits(np.float32(np.nan), ct)
    m.append([0], [6], bad)
    q = R.rand(m.rng, (6, 2, 64), ct)
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), ct)
    k, v = m.rows[0][0]
    want, tol = R.attend(R.from_bits(q, ct), k, v, R.visible(6, 36), R.default_scale(64), ct)
    R.check(y[:3], want[:3], tol[:3])
    assert np.isnan(y[3:]).all()
    m.c.truncate([0], [32])
    m.rows[0][0] = tuple(x[:32] for x in m.rows[0][0])
    m.append([0], [1])
    m.attention(2, [0], [1])
    inf = R.rand(m.rng, (3, 1, 64), ct), R.rand(m.rng, (3, 1, 64), ct)
    inf[1][1, 0, 9] = R.to_bits(np.float32(np.inf), ct)
    m.append([0], [3], inf)
    q = R.rand(m.rng, (3, 2, 64), ct)
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), ct)
    assert np.isfinite(y[0]).all() and np.isfinite(y[1:, :, :9]).all() and (y[1:, :, 9] == np.inf).all()
    m.c.close()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ct", ["i8", "f16", "bf16"])
def test_store_and_gather(gpu, t, ct):
    """Every row type into every cache type and back, bit for bit; rows of zeros, tiny and not finite values."""
    m = Mirror(gpu, ct, 5, 48, 16, 40, 3, 200, t=t)
    k, v = (R.rand(m.rng, (50, 5, 48), t) for _ in range(2))
    k[3] = 0
    v[7, 2] = R.to_bits(np.full(48, 6e-8 if t == "f16" else 1e-38, np.float32), t)
    m.append([2, 0], [33, 17], (k, v))
    m.check([2, 0])
    m.check([0])
    k2 = R.rand(m.rng, (1, 5, 48), t)
    k2[0, 1, 0] = R.to_bits(np.float32(np.inf), t)
    m.c.append([1], [1])
    m.c.store(0, dev(gpu, k2), dev(gpu, k2))
    got = m.c.gather(0, [1])[0].numpy()
    if ct == "i8":
        assert np.isnan(got[0, 1]).all()
    else:
        assert got[0, 1, 0] == np.inf and np.isfinite(got[0, 1, 1:]).all()
    assert np.isfinite(got[0, [0, 2, 3, 4]]).all()
    m.c.close()


def test_store_strides_and_gather_types(gpu):
    """K and V rows of one fused buffer in, rows of both in one buffer out."""
    G, D, n = 2, 64, 21
    rng = np.random.default_rng(4)
    c = pf.PagedCache(gpu, 1, G, D, 4, 1, 64, 16, pf.TYPE_BF16)
    x = R.rand(rng, (n, 3 * G * D), "f32")
    xd = dev(gpu, x)
    c.append([0], [n])
    L = pf.lib()
    gpu.check(L.pf_pages_store(c.h, 0, pf.TYPE_F32, C.c_void_p(xd.ptr + 4 * G * D), C.c_void_p(xd.ptr + 8 * G * D),
                               3 * G * D, 3 * G * D), "store")
    o = dev(gpu, np.zeros((n, 2 * G * D), np.float16))
    s = (C.c_uint32 * 1)(0)
    gpu.check(L.pf_pages_gather(c.h, 0, s, 1, pf.TYPE_F16, C.c_void_p(o.ptr), C.c_void_p(o.ptr + 2 * G * D), 2 * G * D,
                                2 * G * D), "gather")
    held = R.from_bits(R.to_bits(x[:, G * D:], "bf16"), "bf16").astype(np.float16)
    np.testing.assert_array_equal(o.numpy(), held)
    # the same buffer for both is refused
    assert L.pf_pages_gather(c.h, 0, s, 1, pf.TYPE_F16, C.c_void_p(o.ptr), C.c_void_p(o.ptr + 16), 2 * G * D, 2 * G * D) == -1
    c.close()


@pytest.mark.parametrize("ct", ["bf16", "i8"])
def test_pages_against_a_model(gpu, ct):
    """Two hundred random calls: every sequence's rows after each few, the
    number of free pages, and pages handed out lowest first."""
    G, D, page, pages, seqs, most = 2, 32, 16, 40, 9, 150
    m = Mirror(gpu, ct, G, D, page, pages, seqs, most, layers=2)
    rng = np.random.default_rng(23)
    shared = {}                  # page number -> holders, rebuilt from the tables
    for step in range(200):
        op = rng.choice(["append", "append", "append", "fork", "copy", "truncate", "free", "compact"])
        empty = [s for s in range(seqs) if m.c.length(s) == 0]
        some = list(rng.permutation(seqs)[:rng.integers(1, 4)])
        before = m.c.tables(range(seqs)), m.c.free_pages
        try:
            if op == "append":
                m.append(some, [int(rng.integers(0, 40)) for _ in some])
            elif op == "fork" and len(empty) > 1:
                src = int(rng.integers(seqs))
                dst = [s for s in empty if s != src][:2]
                m.c.fork(src, dst)
                for d in dst:
                    m.rows[d] = list(m.rows[src])
            elif op == "copy" and len(empty) > 1:
                src = int(rng.integers(seqs))
                m.c.copy([src], [empty[0]])
                m.rows[empty[0]] = list(m.rows[src])
            elif op == "truncate":
                to = [int(rng.integers(0, m.c.length(s) + 1)) for s in some]
                m.c.truncate(some, to)
                for s, n in zip(some, to):
                    m.rows[s] = [tuple(x[:n] for x in kv) for kv in m.rows[s]]
            elif op == "free" and step % 3 == 0:
                m.c.free(some)
                for s in some:
                    m.rows[s] = [tuple(x[:0] for x in kv) for kv in m.rows[s]]
            elif op == "compact":
                m.c.compact()
                used = np.unique(m.c.tables(range(seqs))[0])
                used = used[used >= 0]
                assert list(used) == list(range(len(used)))
        except pf.PFError as e:
            assert "(-6)" in str(e), e       # too few pages, or a sequence too long: nothing has changed
            (t0, l0), f0 = before
            t1, l1 = m.c.tables(range(seqs))
            np.testing.assert_array_equal(t0, t1)
            np.testing.assert_array_equal(l0, l1)
            assert m.c.free_pages == f0
        tables, lens = m.c.tables(range(seqs))
        assert [len(m.rows[s][0][0]) for s in range(seqs)] == list(lens)
        shared = {p for row in tables for p in row if p >= 0}
        assert m.c.free_pages == pages - len(shared)
        for row, n in zip(tables, lens):
            assert (row >= 0).sum() == -(-n // page) and len(set(row[row >= 0])) == (row >= 0).sum()
        if step % 5 == 4:
            m.check(range(seqs))
    m.check(range(seqs))
    m.c.close()


def test_pages_lowest_first_and_copy_on_write(gpu):
    m = Mirror(gpu, "bf16", 1, 16, 16, 12, 5, 64)
    m.append([0], [40])
    assert m.c.tables([0])[0].tolist() == [[0, 1, 2]]
    m.c.fork(0, [1, 2])
    for d in (1, 2):
        m.rows[d] = list(m.rows[0])
    assert m.c.free_pages == 9
    m.append([2, 1], [1, 1])                 # both copy the shared last page: the first sequence keeps it
    assert m.c.tables([0, 1, 2])[0].tolist() == [[0, 1, 2], [0, 1, 4], [0, 1, 3]]
    m.append([0], [1])                       # alone on page 2 now
    assert m.c.tables([0])[0].tolist() == [[0, 1, 2]] and m.c.free_pages == 7
    m.check([0, 1, 2])
    m.c.free([0])
    assert m.c.free_pages == 8
    m.c.fork(1, [3])
    m.rows[3] = list(m.rows[1])
    m.c.free([1])                            # 3 is alone on page 4
    m.append([3], [1])
    assert m.c.tables([3])[0].tolist() == [[0, 1, 4]]
    m.check([2, 3])
    m.c.copy([3, 3], [0, 4])
    m.rows[0], m.rows[4] = list(m.rows[3]), list(m.rows[3])
    assert m.c.tables([0, 4])[0].tolist() == [[2, 5, 6], [7, 8, 9]]
    m.c.free([0])
    assert m.c.compact() == 3                # used: 0 1 3 4 7 8 9 -> 0 .. 6
    assert m.c.tables([2, 3, 4])[0].tolist() == [[0, 1, 3], [0, 1, 4], [2, 5, 6]]
    m.check([2, 3, 4])
    assert m.c.compact() == 0
    m.c.close()


def test_pages_refusals(gpu):
    L = pf.lib()
    h = pf.vp()

    def create(**kw):
        f = dict(type=pf.TYPE_BF16, n_layers=1, n_kv_heads=2, head_dim=64, page_size=16, n_pages=4, max_seqs=3,
                 max_context=64)
        f.update(kw)
        cfg = pf.PagesConfig(**f)
        return L.pf_pages_create(gpu.h, C.byref(cfg), C.byref(h))

    assert create(type=pf.TYPE_F32) == -1 and create(type=9) == -1
    assert create(head_dim=72) == -4 and create(head_dim=144) == -4 and create(page_size=48) == -4
    assert create(page_size=8) == -4 and create(page_size=512) == -4
    for k in ("n_layers", "n_kv_heads", "n_pages", "max_seqs", "max_context"):
        assert create(**{k: 0}) == -1, k
    assert create(max_context=0x7FFFFFFF) == -4 and create(n_pages=0xFFFFFFFF) == -4
    before = gpu.device_bytes
    assert create(n_pages=0x7FFFFFFF, n_layers=4096) == -2        # more memory than there is
    assert gpu.device_bytes == before and not h
    c = pf.PagedCache(gpu, 1, 2, 64, 4, 3, 64, 16, pf.TYPE_BF16)
    k = gpu.empty((3, 2, 64), np.uint16)

    def refused(f, *a, code):
        with pytest.raises(pf.PFError, match=rf"\({code}\)"):
            f(*a)

    c.pass_rows = 3
    refused(c.store, 0, k, k, code=-5)       # no pass
    refused(c.attention, 0, k, code=-5)
    refused(c.append, [3], [1], code=-1)
    refused(c.append, [1, 1], [1, 1], code=-1)
    refused(c.append, [0], [65], code=-6)
    refused(c.append, [0, 1], [33, 32], code=-6)
    assert c.length(0) == 0 and c.free_pages == 4
    c.append([0, 2], [2, 1])
    c.store(0, k, k)
    refused(c.store, 1, k, k, code=-1)
    refused(c.attention, 1, k, code=-1)
    refused(c.fork, 0, [0], code=-5)
    refused(c.fork, 0, [2], code=-5)
    refused(c.fork, 5, [1], code=-1)
    refused(c.fork, 0, [1, 1], code=-1)
    refused(c.copy, [0], [2], code=-5)
    refused(c.copy, [7], [1], code=-1)
    refused(c.truncate, [0], [3], code=-1)
    refused(c.truncate, [0, 0], [1, 1], code=-1)
    refused(c.free, [0, 0], code=-1)
    c.attention(0, gpu.empty((3, 4, 64), np.uint16))                       # the pass is still open
    refused(c.attention, 0, gpu.empty((3, 2, 64), np.float16), code=-4)    # fp16 rows over bf16 pages
    d = pf.AttnDesc(pf.TYPE_BF16, 4, 4, 64, 1, 0, 0, 0.0, 0, 0, 0, 0)      # another number of kv heads
    o = gpu.empty((3, 4, 64), np.uint16)
    assert L.pf_pages_attention(c.h, C.byref(d), 0, C.c_void_p(o.ptr), C.c_void_p(k.ptr)) == -1
    d.n_kv_heads = 2
    assert L.pf_pages_attention(c.h, C.byref(d), 0, C.c_void_p(o.ptr), C.c_void_p(o.ptr)) == -1   # in place
    assert L.pf_pages_attention(c.h, C.byref(d), 0, C.c_void_p(o.ptr + 8), C.c_void_p(k.ptr)) == -1
    assert L.pf_pages_attention(c.h, C.byref(d), 0, None, C.c_void_p(k.ptr)) == -1
    assert L.pf_pages_store(c.h, 0, pf.TYPE_I8, C.c_void_p(k.ptr), C.c_void_p(k.ptr), 0, 0) == -1
    assert L.pf_pages_store(c.h, 0, pf.TYPE_BF16, C.c_void_p(k.ptr), C.c_void_p(k.ptr), 64, 0) == -1
    s = (C.c_uint32 * 1)(4)
    assert L.pf_pages_gather(c.h, 0, s, 1, pf.TYPE_F32, None, None, 0, 0) == -1
    c.truncate([0], [1])
    c.pass_rows = 3
    refused(c.store, 0, k, k, code=-5)       # the pass has ended
    c.append([], [])
    c.free([])
    assert L.pf_pages_append(None, None, None, 0) == -1 and L.pf_pages_length(None, 0) == 0
    used = gpu.device_bytes
    c.close()
    assert gpu.device_bytes < used


def test_serving_run(gpu):
    """Prompts through prompt attention and into the pages, answers forked
    from one of them, verify passes with rejected drafts, a sequence that ends,
    compaction, and a second prompt over the cached rows."""
    H, G, D = 4, 2, 64
    m = Mirror(gpu, "bf16", G, D, 32, 60, 6, 400)
    lens = [70, 129, 33]
    q, k, v = (R.rand(m.rng, (sum(lens), h, D), "bf16") for h in (H, G, G))
    m.append([0, 1, 2], lens, (k, v))
    y = gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), lens).numpy()
    yp = m.c.attention(0, dev(gpu, q)).numpy()       # the same rows, read from the pages
    at = 0
    for s, n in enumerate(lens):
        want, tol = R.attend(R.from_bits(q[at:at + n], "bf16"), *m.rows[s][0], R.visible(n, n), R.default_scale(D), "bf16")
        R.check(R.from_bits(y[at:at + n], "bf16"), want, tol, f"prompt {s}")
        R.check(R.from_bits(yp[at:at + n], "bf16"), want, tol, f"pages {s}")
        at += n
    m.c.fork(1, [3, 4])
    for d in (3, 4):
        m.rows[d] = list(m.rows[1])
    live = [0, 1, 2, 3, 4]
    for step in range(12):
        rows = [1 + (step + s) % 5 for s in live]
        m.append(live, rows)
        m.attention(H, live, rows)
        keep = [m.c.length(s) - (step * 7 + s) % n for s, n in zip(live, rows)]
        m.c.truncate(live, keep)
        for s, n in zip(live, keep):
            m.rows[s][0] = tuple(x[:n] for x in m.rows[s][0])
        if step == 5:
            m.c.free([1])
            m.rows[1] = [tuple(x[:0] for x in m.rows[1][0])]
            live.remove(1)
            m.c.compact()
    m.check(live)
    # a long pass over a cached prefix: its rows read back, the prompt's behind them
    n = m.c.length(3)
    pk, pv = m.c.gather(0, [3], dtype=np.float16)
    q2, k2, v2 = (R.rand(m.rng, (90, h, D), "f16") for h in (H, G, G))
    kk, vv = (np.concatenate([a.numpy(), b]) for a, b in ((pk, k2), (pv, v2)))
    y = gpu.prompt_attention(dev(gpu, q2), dev(gpu, kk), dev(gpu, vv), [90], [n + 90]).numpy()
    want, tol = R.attend(q2.astype(np.float64), kk.astype(np.float64), vv.astype(np.float64), R.visible(90, n + 90),
                         R.default_scale(D), "f16")
    R.check(y, want, tol)
    m.c.close()


def test_two_caches_and_a_second_pass_between(gpu):
    """Split attention of two caches in turn: they share the context's scratch, not their results."""
    a = Mirror(gpu, "bf16", 1, 64, 64, 80, 2, 4000)
    b = Mirror(gpu, "i8", 1, 128, 16, 400, 2, 3000)
    for m, lens in ((a, [4000, 900]), (b, [2600, 3000])):
        m.append([0, 1], [n - 1 for n in lens])
    a.append([0, 1], [1, 1])
    b.append([1, 0], [1, 1])
    for _ in range(2):
        a.attention(8, [0, 1], [1, 1])
        b.attention(4, [1, 0], [1, 1])
    a.c.close()
    b.c.close()


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("size", [3e-4, 1.2e4])
def test_paged_int8_value_range(gpu, t, size):
    """Values far from one, in int8 pages: their row scales are outside what fp16 weights hold."""
    m = Mirror(gpu, "i8", 2, 64, 32, 20, 1, 600, t=t)
    k = R.rand(m.rng, (500, 2, 64), t)
    v = R.to_bits((m.rng.standard_normal((500, 2, 64)) * size).astype(np.float32), t)
    m.append([0], [500], (k, v))
    m.append([0], [2], (k[:2], v[:2]))
    m.attention(4, [0], [2])
    m.c.close()


def test_prompt_window_before_the_first_key(gpu):
    """Queries before the first key with a window: causal, they see nothing; else every key and the sinks."""
    for causal in (True, False):
        prompt_case(gpu, "bf16", 2, 2, 64, [40, 130, 7], [10, 20, 0], causal, 5, 2)


@pytest.mark.parametrize("H,G", [(40, 40), (48, 24), (80, 40), (32, 8), (12, 6)])
def test_prompt_many_heads(gpu, H, G):
    """Each head's tiles are taken once, whatever the order that the heads and the sequences go in."""
    prompt_case(gpu, "bf16", H, G, 32, [33, 300, 1, 130], [40, 300, 400, 135])


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,G,D,ql,kl,causal,window,sink", [
    (4, 4, 128, [1], [2049], True, 0, 0), (4, 2, 64, [5, 64, 130], [2000, 700, 131], True, 0, 0),
    (3, 1, 48, [70], [1500], False, 0, 0), (2, 2, 112, [33, 2, 0, 9], [900, 1, 70, 0], True, 0, 0),
    (2, 1, 128, [90], [3000], True, 1200, 130), (2, 2, 64, [900, 40], [880, 10], True, 0, 0),
    (1, 1, 16, [1, 1, 65], [1279, 64, 1300], True, 0, 0),
])
def test_prompt_few_rows_many_keys(gpu, t, H, G, D, ql, kl, causal, window, sink):
    """Keys cut over workgroups, whose parts are joined: parts that a row sees nothing of, rows that see nothing."""
    prompt_case(gpu, t, H, G, D, ql, kl, causal, window, sink)


def test_prompt_parts_of_many_sequences(gpu):
    """More sequences than a launch takes, each cut; a smaller call between two of them finds its results whole."""
    lens = [600 + 13 * (i % 40) for i in range(70)]
    ql = [1 + i % 3 for i in range(70)]
    prompt_case(gpu, "bf16", 2, 1, 32, ql, lens)
    prompt_case(gpu, "bf16", 4, 4, 128, [3], [1111])
    prompt_case(gpu, "f32", 2, 1, 32, ql, lens)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n,window,spot", [(50, 0, 10), (50, 0, 0), (64, 12, 45), (300, 20, 40), (200, 0, 63)])
def test_prompt_infinity_in_a_first_tile(gpu, t, n, window, spot):
    """An infinite value in the first tile that a row sees, or in the only half of one, reaches it as that infinity."""
    rng = np.random.default_rng(9)
    q, k, v = (R.rand(rng, (n, 1, 64), t) for _ in range(3))
    v[spot, 0, 3] = R.to_bits(np.float32(np.inf), t)
    y = R.from_bits(gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), [n], window=window).numpy(), t)
    p = np.arange(n)
    see = (p >= spot) & (p < spot + window if window else True)
    assert (y[see, 0, 3] == np.inf).all() and np.isfinite(y[~see]).all() and np.isfinite(y[:, 0, 4:]).all()


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_prompt_parts_not_finite(gpu, t):
    """A NaN in one part's keys reaches the rows that see it and no others; so does one in a value."""
    rng = np.random.default_rng(5)
    nq, nk, H, D = 130, 1500, 1, 64
    for spot in (3, 1400):
        q, k, v = (R.rand(rng, (n, H, D), t) for n in (nq, nk, nk))
        v[spot, 0, 5] = k[1450, 0, 7] = R.to_bits(np.float32(np.nan), t)
        print(f"parts not finite {t} {spot}", flush=True)
        y = R.from_bits(gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), [nq], [nk]).numpy(), t)
        q, k, v = (R.from_bits(x, t) for x in (q, k, v))
        want, tol = R.attend(q, k, v, R.visible(nq, nk), R.default_scale(D), t)
        R.check(y, want, tol)
        p = nk - nq + np.arange(nq)
        assert np.isnan(y[p >= 1450]).all() and np.isfinite(y[p < 1450][:, :, 6:]).all()
        np.testing.assert_array_equal(np.isnan(y[:, 0, 5]), p >= spot)


def test_prompt_too_many_rows(gpu):
    b = gpu.empty((64, 64, 64), np.float16)
    d = pf.AttnDesc(pf.TYPE_F16, 64, 64, 64, 1, 0, 0, 0.0, 0, 0, 0, 0)
    lens = (C.c_uint32 * 1)(1 << 30)
    p = C.c_void_p(b.ptr)
    assert pf.lib().pf_prompt_attention(gpu.h, C.byref(d), p, p, p, p, lens, None, 1) == -4


def test_many_forks_without_a_pass(gpu):
    """Table changes that no pass sends go to the device when there are many."""
    m = Mirror(gpu, "bf16", 1, 16, 16, 2010, 12, 32000)
    m.append([0], [31999])
    for _ in range(6):
        m.c.fork(0, list(range(1, 12)))
        m.c.free(list(range(2, 12)))
        m.c.copy([], [])
        m.c.free([1])
    m.c.fork(0, [5])
    m.rows[5] = list(m.rows[0])
    m.check([5])
    m.append([5], [1])
    m.check([0, 5])
    m.attention(2, [5], [1])
    m.c.close()


def test_copies_in_one_call(gpu):
    """More copies on write than go with a step's message, and a step of more sequences than fit one message."""
    n = 200
    m = Mirror(gpu, "i8", 2, 32, 16, 900, n + 1, 64)
    m.append([0], [23])
    m.c.fork(0, list(range(1, n + 1)))
    for s in range(1, n + 1):
        m.rows[s] = list(m.rows[0])
    m.append(list(range(n, 0, -1)), [1 + s % 3 for s in range(n)])
    m.check(range(n + 1))
    m.attention(2, list(range(n, 0, -1)), [1 + s % 3 for s in range(n)])
    m.c.free(list(range(1, n, 2)))
    for s in range(1, n, 2):
        m.rows[s] = [tuple(x[:0] for x in kv) for kv in m.rows[s]]
    m.c.copy([0] * 100, list(range(1, n, 2)))
    for s in range(1, n, 2):
        m.rows[s] = list(m.rows[0])
    m.check(range(n + 1))
    m.c.free(list(range(2, n + 1, 2)))
    for s in range(2, n + 1, 2):
        m.rows[s] = [tuple(x[:0] for x in kv) for kv in m.rows[s]]
    m.c.compact()
    m.check(range(n + 1))
    m.c.close()


def test_pool_sizes_past_64_bits(gpu):
    """A pool whose bytes do not fit 64 bits is refused: 2^64 bytes came out as none, and were taken."""
    h = pf.vp()
    for ct, layers in ((pf.TYPE_BF16, 1 << 13), (pf.TYPE_BF16, (1 << 13) + 1), (pf.TYPE_I8, 1 << 14), (pf.TYPE_F16, 65535)):
        cfg = pf.PagesConfig(ct, layers, 1 << 15, 128, 256, 1 << 20, 1, 256)
        assert pf.lib().pf_pages_create(gpu.h, C.byref(cfg), C.byref(h)) == -4, (ct, layers)
    assert not h


def beside_a_sink(t, n, low, first):
    """One key that outweighs the n - 1 others by exp(low) each, with a value of zero; theirs are about 100."""
    rng = np.random.default_rng(31)
    k, v = np.zeros((n, 1, 64), np.float32), (100 + 10 * rng.standard_normal((n, 1, 64))).astype(np.float32)
    k[:, :, 0] = -low
    k[0 if first else n - 1, :, 0] = 0
    v[0 if first else n - 1] = 0
    return R.to_bits(k, t), R.to_bits(v, t)


def fp16_step(v):
    """What rounding takes of n weights: they are held against 2^11 times the largest at least, and half a step of
    fp16's smallest values is 2^-25, so 2^-36 of the largest each (fp32 and bf16 reach far below)."""
    return 2.0 ** -36 * np.abs(v).sum(0)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("low", [14, 16, 18, 20])
def test_many_keys_beside_a_sink(gpu, t, first, low):
    """Thousands of keys that weigh 2^-20 to 2^-29 of one: together they are what comes out."""
    n, nq = 8000, 3
    k, v = beside_a_sink(t, n, low, first)
    q = R.to_bits(np.zeros((nq, 2, 64), np.float32), t)
    q[:, :, 0] = R.to_bits(np.float32(1), t)
    kf, vf = R.from_bits(k, t), R.from_bits(v, t)
    want, tol = R.attend(R.from_bits(q, t), kf, vf, R.visible(nq, n, False), 1.0, t)
    if t == "f16":
        tol = tol + fp16_step(vf)
    print(f"beside a sink {t} first {first} low {low}", flush=True)
    y = gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), [nq], [n], causal=False, scale=1.0).numpy()
    R.check(R.from_bits(y, t), want, tol, "prompt")
    c = pf.PagedCache(gpu, 1, 1, 64, 130, 1, n, 64, TYPE[t])
    c.append([0], [n - nq])
    c.store(0, dev(gpu, k[:-nq]), dev(gpu, v[:-nq]))
    c.append([0], [nq])
    c.store(0, dev(gpu, k[-nq:]), dev(gpu, v[-nq:]))
    y = c.attention(0, dev(gpu, q), causal=False, scale=1.0).numpy()
    R.check(R.from_bits(y, t), want, tol, "pages")
    c.close()


LARGE = [("f32", 3e38), ("f32", 1e37), ("bf16", 3e38), ("bf16", 1e36), ("f16", 6e4), ("f32", 1e-30), ("bf16", 1e-30)]


def far_values(rng, t, n, nq, size, G=1):
    """Rows whose scores rise by 7.9 (base 2) after the first keys, less than what moves the running maximum:
    weights of 2^7.9, and values all near `size`."""
    k = np.zeros((n, G, 64), np.float32)
    k[70:, :, 0] = 7.9 * np.log(2)
    v = (size * (1 - 0.02 * rng.random((n, G, 64)))).astype(np.float32)
    v[:, :, 32:] *= np.where(np.arange(n) % 2, 1, -1)[:, None, None].astype(np.float32)
    q = np.zeros((nq, 2 * G, 64), np.float32)
    q[:, :, 0] = 1
    return (R.to_bits(x, t) for x in (q, k, v))


def lost_below(t, n):
    """What sums lose below fp32's normal range: 2^-126 of each product, weights held to 2^-K, K = 10 + log2 n at
    most (six products of each key where rows are fp32, and two pieces else)."""
    return 0.0 if t == "f16" else 6 * n * 2.0 ** (-126 + 10 + np.log2(n))


@pytest.mark.parametrize("t,size", LARGE)
@pytest.mark.parametrize("ql,kl", [([3], [100]), ([2, 1], [3000, 80]), ([5], [700]), ([130], [300])])
def test_prompt_far_values(gpu, t, size, ql, kl):
    """Values near the type's largest, or far below one: sums of them stay in range whatever the number of keys."""
    rng = np.random.default_rng(8)
    q, k, v = (np.concatenate(x) for x in zip(*(list(far_values(rng, t, n, a, size)) for a, n in zip(ql, kl))))
    print(f"far values {t} {size} {ql} {kl}", flush=True)
    y = R.from_bits(gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), ql, kl, scale=1.0).numpy(), t)
    q, k, v = (R.from_bits(x, t) for x in (q, k, v))
    qa = ka = 0
    for a, n in zip(ql, kl):
        want, tol = R.attend(q[qa:qa + a], k[ka:ka + n], v[ka:ka + n], R.visible(a, n), 1.0, t)
        R.check(y[qa:qa + a], want, tol + lost_below(t, max(kl)), f"{n} keys")
        qa, ka = qa + a, ka + n


@pytest.mark.parametrize("t,ct,size", [("f32", "bf16", 3e38), ("f32", "bf16", 1e-30), ("bf16", "bf16", 3e38),
                                       ("bf16", "bf16", 1e-30), ("f32", "i8", 3e38), ("f32", "i8", 1e36),
                                       ("bf16", "i8", 3e38), ("f32", "i8", 1e-25), ("f16", "i8", 6e4), ("f16", "f16", 6e4)])
@pytest.mark.parametrize("n,nq", [(100, 1), (3000, 2), (700, 5)])
def test_paged_far_values(gpu, t, ct, size, n, nq):
    """The same over pages."""
    m = Mirror(gpu, ct, 1, 64, 64, 50, 1, 3200, t=t)
    q, k, v = far_values(m.rng, t, n, nq, size)
    m.append([0], [n - nq], (k[:-nq], v[:-nq]))
    m.append([0], [nq], (k[-nq:], v[-nq:]))
    print(f"far values {t} over {ct} {size} {n}", flush=True)
    y = R.from_bits(m.c.attention(0, dev(gpu, q), scale=1.0).numpy(), t)
    kf, vf = m.rows[0][0]
    want, tol = R.attend(R.from_bits(q, t), kf, vf, R.visible(nq, n), 1.0, t, ct == "i8")
    R.check(y, want, tol + lost_below(t, n))
    m.c.close()


@pytest.mark.parametrize("t,ct", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("n,window", [(36, 0), (700, 0), (700, 300), (5000, 0)])
@pytest.mark.parametrize("D,H", [(64, 2), (128, 20), (48, 2)])
def test_paged_infinity_as_the_context_grows(gpu, t, ct, n, window, D, H):
    """An infinite value reaches the rows that see it as that infinity wherever its key lies; two that differ as a
    NaN; the rest of the row as ever."""
    spot = n - 30
    for bad in (np.inf, -np.inf):
        m = Mirror(gpu, ct, 1, D, 32, 160, 1, 5100, t=t)
        k, v = (R.rand(m.rng, (n, 1, D), t) for _ in range(2))
        v[spot, 0, 5] = v[spot - 1, 0, 5] = v[spot - 3, 0, 6] = R.to_bits(np.float32(bad), t)
        v[spot - 4, 0, 6] = R.to_bits(np.float32(-bad), t)
        m.append([0], [n - 2], (k[:-2], v[:-2]))
        m.append([0], [2], (k[-2:], v[-2:]))
        print(f"infinity {t} over {ct} n {n} window {window} D {D} {bad}", flush=True)
        for grown in (0, 1, 64):             # the key moves into tiles that every row sees whole
            if grown:
                new = [R.rand(m.rng, (grown, 1, D), t) for _ in range(2)]
                m.append([0], [grown], new)
            rows = grown or 2
            q = R.rand(m.rng, (rows, H, D), t)
            y = R.from_bits(m.c.attention(0, dev(gpu, q), window=window).numpy(), t)
            assert (y[:, :, 5] == bad).all() and np.isnan(y[:, :, 6]).all()
            assert np.isfinite(y[:, :, :5]).all() and np.isfinite(y[:, :, 7:]).all()
        m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 112, 128])
def test_minus_infinity_in_a_key(gpu, t, D):
    """A key of minus infinity where the queries are positive has a score of minus infinity: it weighs nothing."""
    rng = np.random.default_rng(6)
    n, at = 150, 20
    q, k, v = (R.rand(rng, (n, 2, D), t) for _ in range(3))
    q[:, :, D - 2] = R.to_bits(np.float32(0.5), t)
    k[at, :, D - 2] = R.to_bits(np.float32(-np.inf), t)
    print(f"minus infinity {t} {D}", flush=True)
    qf, kf, vf = (R.from_bits(x, t) for x in (q, k, v))
    want, tol = R.attend(qf, np.where(np.isinf(kf), 0, kf), vf, R.visible(n, n) & (np.arange(n) != at)[None],
                         R.default_scale(D), t)
    y = R.from_bits(gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), [n]).numpy(), t)
    R.check(y, want, tol, "prompt")
    c = pf.PagedCache(gpu, 1, 2, D, 10, 1, 160, 16, TYPE[t])
    c.append([0], [n])
    c.store(0, dev(gpu, k), dev(gpu, v))
    R.check(R.from_bits(c.attention(0, dev(gpu, q)).numpy(), t), want, tol, "pages")
    c.close()


def test_scale_out_of_range(gpu):
    """A scale that is not finite in base 2 would make a NaN of scores of zero: it is refused."""
    q, k, v, o = (gpu.empty((4, 2, 64), np.float16) for _ in range(4))
    c = pf.PagedCache(gpu, 1, 2, 64, 1, 1, 16, 16, pf.TYPE_F16)
    c.append([0], [4])
    c.store(0, k, v)
    for scale in (2.4e38, 3e38, float("inf")):
        with pytest.raises(pf.PFError, match=r"\(-1\)"):
            gpu.prompt_attention(q, k, v, [4], scale=scale, out=o)
        with pytest.raises(pf.PFError, match=r"\(-1\)"):
            c.attention(0, q, scale=scale, out=o)
    z = dev(gpu, np.zeros((4, 2, 64), np.float16))
    x = np.arange(512, dtype=np.float16).reshape(4, 2, 64)
    y = gpu.prompt_attention(z, z, dev(gpu, x), [4], causal=False, scale=1.6e38).numpy()
    np.testing.assert_array_equal(y, np.broadcast_to(x.astype(np.float64).mean(0).astype(np.float16), y.shape))
    c.close()


def test_calls_that_change_nothing_end_the_pass(gpu):
    """fork, copy, truncate, free and compact end the pass, whatever there is for them to do."""
    c = pf.PagedCache(gpu, 1, 2, 64, 4, 3, 64, 16, pf.TYPE_BF16)
    k = gpu.empty((2, 2, 64), np.uint16)
    for f in (lambda: c.fork(1, [2]), lambda: c.fork(0, []), lambda: c.copy([], []), lambda: c.truncate([], []),
              lambda: c.free([]), c.compact):
        c.free([0])
        c.append([0], [2])
        c.store(0, k, k)
        f()
        with pytest.raises(pf.PFError, match=r"\(-5\)"):
            c.store(0, k, k)
        assert c.length(0) == 2 and c.length(2) == 0 and c.free_pages == 3
    c.close()


# ------------------------------------------- each kernel of the dispatch rules

def prompt_plan(t, H, G, D, ql, kl):
    """(query rows of a workgroup, parts of the keys) that a call takes."""
    d = pf.AttnDesc(TYPE[t], H, G, D, 1, 0, 0, 0.0, 0, 0, 0, 0)
    rows, parts = C.c_uint32(), C.c_uint32()
    a, b = ((C.c_uint32 * len(x))(*x) for x in (ql, kl))
    assert pf.lib().pf_test_prompt_plan(C.byref(d), a, b, len(ql), C.byref(rows), C.byref(parts)) == 0
    return rows.value, parts.value


def pages_plan(t, H, G, D, rows, lens, window=0, sink=0):
    """(waves of a workgroup, whether the keys are cut) of a pass."""
    d = pf.AttnDesc(TYPE[t], H, G, D, 1, window, sink, 0.0, 0, 0, 0, 0)
    x = [C.c_uint32() for _ in range(3)]
    a, b = ((C.c_uint32 * len(y))(*y) for y in (rows, lens))
    assert pf.lib().pf_test_pages_plan(C.byref(d), a, b, len(lens), *map(C.byref, x)) == 0
    return x[0].value, x[1].value < x[2].value


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [48, 64, 80, 128])
@pytest.mark.parametrize("ql,prefix,causal,window,sink", [
    ([1, 130, 2, 0, 3, 129, 1, 9], 0, True, 0, 0), ([64, 129, 5, 33, 1, 2, 7], 300, True, 0, 0),
    ([64, 129, 5, 33, 1, 2, 7], 200, True, 70, 5), ([1, 200, 2, 0, 3, 129, 1, 9], 20, False, 0, 0),
    ([140, 129, 40, 1, 5, 2], -40, True, 30, 2),
])
def test_prompt_tiles_of_128_rows(gpu, t, D, ql, prefix, causal, window, sink):
    """Enough heads and sequences that a workgroup takes 128 query rows, a wave 32 of them over whole key tiles."""
    kl = [max(0, n + prefix) for n in ql]
    assert prompt_plan(t, 64, 16, D, ql, kl) == (128, 1)
    prompt_case(gpu, t, 64, 16, D, ql, kl, causal, window, sink)


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [64, 112])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_prompt_tiles_of_128_rows_not_finite(gpu, t, D, bad):
    """An infinity or a NaN in a value reaches the rows that see it and no others, over whole tiles and others."""
    rng = np.random.default_rng(12)
    n, H, spots = 150, 64, (3, 70, 149)
    lens = [n] * 4
    assert prompt_plan(t, H, H, D, lens, lens) == (128, 1)
    q, k, v = (R.rand(rng, (4 * n, H, D), t) for _ in range(3))
    for s, at in enumerate(spots):
        v[s * n + at, :, 9] = R.to_bits(np.float32(bad), t)
    print(f"128 rows not finite {t} {D} {bad}", flush=True)
    y = R.from_bits(gpu.prompt_attention(dev(gpu, q), dev(gpu, k), dev(gpu, v), lens).numpy(), t)
    for s, at in enumerate(spots + (n,)):
        got = y[s * n:(s + 1) * n]
        assert np.isfinite(got[:at]).all() and np.isfinite(got[:, :, :9]).all() and np.isfinite(got[:, :, 10:]).all()
        if t == "f32" or np.isnan(bad):
            assert not np.isfinite(got[at:, :, 9]).any()
        else:
            assert (got[at:, :, 9] == bad).all()


@pytest.mark.parametrize("t,ct", COMBOS)
@pytest.mark.parametrize("D", [48, 64, 112, 128])
@pytest.mark.parametrize("H,G,lens,new,window,sink,causal", [
    (4, 2, [500, 405, 9, 430], 1, 0, 0, True), (16, 2, [402, 33, 512], 1, 0, 0, True),
    (8, 2, [390, 461], 5, 0, 0, True), (6, 1, [480, 7], 7, 0, 0, True), (4, 2, [900, 500, 30], 3, 420, 5, True),
    (8, 1, [700, 460], 4, 410, 0, True), (6, 2, [449, 403], 6, 0, 0, False),
])
def test_paged_workgroups_of_8_waves(gpu, t, ct, D, H, G, lens, new, window, sink, causal):
    """Contexts that workgroups of 8 waves take uncut (fp32 rows of over 64 dims and 16 score columns: 4 waves)."""
    waves, _ = pages_plan(t, H, G, D, [new] * len(lens), lens, window, sink)
    assert waves == (4 if t == "f32" and D > 64 and new * H // G > 16 else 8)
    m = Mirror(gpu, ct, G, D, 32, sum(-(-n // 32) for n in lens), len(lens), max(lens), t=t)
    seqs = list(range(len(lens)))
    print(f"8 waves {t} over {ct} D {D} H {H} G {G} lens {lens} new {new} window {window}", flush=True)
    m.append(seqs, [n - new for n in lens])
    m.append(seqs, [new] * len(lens))
    m.attention(H, seqs, [new] * len(lens), causal=causal, window=window, sink=sink)
    m.c.close()


@pytest.mark.parametrize("t,ct", [("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("D,H", [(48, 2), (64, 10), (128, 2)])
def test_paged_workgroups_of_8_waves_not_finite(gpu, t, ct, D, H):
    """Infinities and NaN in values reach the rows that see them as themselves, and no others."""
    n, new = 450, 4
    assert pages_plan(t, H, 1, D, [new], [n])[0] == 8
    m = Mirror(gpu, ct, 1, D, 16, 29, 1, n, t=t)
    k, v = (R.rand(m.rng, (n, 1, D), t) for _ in range(2))
    for at, d, bad in ((7, 1, np.inf), (300, 2, -np.inf), (n - 2, 3, np.inf), (n - 1, 4, np.nan)):
        v[at, 0, d] = R.to_bits(np.float32(bad), t)
    m.append([0], [n - new], (k[:-new], v[:-new]))
    m.append([0], [new], (k[-new:], v[-new:]))
    q = R.rand(m.rng, (new, H, D), t)
    print(f"8 waves not finite {t} over {ct} D {D} H {H}", flush=True)
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), t)
    kf, vf = m.rows[0][0]
    want, tol = R.attend(R.from_bits(q, t), kf, vf, R.visible(new, n), R.default_scale(D), t)
    with np.errstate(invalid="ignore"):
        R.check(y, want, tol)
    assert (y[:, :, 1] == np.inf).all() and (y[:, :, 2] == -np.inf).all() and np.isfinite(y[:2, :, 3:]).all()
    assert (y[2:, :, 3] == np.inf).all() and np.isfinite(y[2, :, 4:]).all() and np.isnan(y[3, :, 4]).all()
    m.c.close()


@pytest.mark.parametrize("t,ct", [("bf16", "bf16"), ("f32", "i8")])
def test_pool_past_32_bits(gpu, t, ct):
    """A sequence whose pages lie more than 2^32 bytes (and values) into a layer, in the second layer."""
    G, D, page, pages = 8, 128, 256, 17000
    m = Mirror(gpu, ct, G, D, page, pages, 4, 16996 * page, layers=2, t=t)
    assert pages * G * page * D > 1 << 32
    m.c.append([0], [16995 * page])              # (its rows are never read)
    m.append([1], [300])
    assert m.c.tables([1])[0].tolist() == [[16995, 16996]]
    m.c.copy([1], [2])
    m.c.fork(1, [3])
    m.rows[2], m.rows[3] = list(m.rows[1]), list(m.rows[1])
    assert m.c.free_pages == 1
    m.c.truncate([2], [256])
    m.rows[2] = [tuple(x[:256] for x in kv) for kv in m.rows[2]]
    m.append([3, 1], [2, 1])                     # 3 copies the last page
    print(f"past 32 bits {t} over {ct}", flush=True)
    for layer in (0, 1):
        m.attention(16, [3, 1], [2, 1], layer=layer)
    m.check([1, 2, 3])
    m.c.free([0])
    m.c.compact()
    m.check([1, 2, 3])
    m.append([2], [1])
    m.attention(16, [2], [1], layer=1)
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_prompt_rows_past_32_bits(gpu, t):
    """Key and value rows so far apart that a tile of them spans more than 2^32 bytes."""
    H, G, D, n, nq = 4, 2, 64, 70, 3
    es = np.dtype(R.DTYPE[t]).itemsize
    stride = (1 << 27) // es                     # 2^27 bytes: 64 rows are 2^33
    rng = np.random.default_rng(2)
    q, k, v = R.rand(rng, (nq, H, D), t), R.rand(rng, (n, G, D), t), R.rand(rng, (n, G, D), t)
    buf = gpu.empty(((n - 1) * (stride * es) + 2 * G * D * es,), np.uint8)
    L = pf.lib()
    for i in range(n):
        row = np.concatenate([k[i].ravel(), v[i].ravel()])
        gpu.check(L.pf_memcpy(gpu.h, C.c_void_p(buf.ptr + i * stride * es), row.ctypes.data_as(pf.vp), row.nbytes, 0), "row")
    qd, o = dev(gpu, q), gpu.empty((nq, H, D), R.DTYPE[t])
    d = pf.AttnDesc(TYPE[t], H, G, D, 1, 0, 0, 0.0, 0, stride, stride, 0)
    a, b = (C.c_uint32 * 1)(nq), (C.c_uint32 * 1)(n)
    print(f"rows past 32 bits {t}", flush=True)
    gpu.check(L.pf_prompt_attention(gpu.h, C.byref(d), C.c_void_p(qd.ptr), C.c_void_p(buf.ptr),
                                    C.c_void_p(buf.ptr + G * D * es), C.c_void_p(o.ptr), a, b, 1), "prompt")
    y = R.from_bits(o.numpy(), t)
    want, tol = R.attend(*(R.from_bits(x, t) for x in (q, k, v)), R.visible(nq, n), R.default_scale(D), t)
    R.check(y, want, tol)
    buf.free()
