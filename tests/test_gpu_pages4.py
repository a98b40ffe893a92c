"""Paged caches of 4-bit floats against float64 on the host: what the pages hold
of rows, rows read back, attention over them, and the pages' moves."""
import numpy as np
import pytest

import attention_ref as R
import pocketforge_amd as pf
import serving_ref as S
import test_gpu_attention as A
from test_serving_cpu import pages_plan

pytestmark = pytest.mark.gpu

A.TYPE["fp4"] = pf.TYPE_FP4
dev = A.dev


class Mirror(A.Mirror):
    def __init__(self, gpu, G, D, page, pages, seqs, context, layers=1, t="f32"):
        super().__init__(gpu, "fp4", G, D, page, pages, seqs, context, layers, t)

    def held(self, x):
        return S.fp4_held(R.from_bits(x, self.t))


def plane(gpu, p, n):
    out = np.empty(n, np.uint8)
    at = p.__cuda_array_interface__["data"][0]
    gpu.check(pf.lib().pf_memcpy(gpu.h, out.ctypes.data_as(pf.vp), pf.C.c_void_p(at), n, 1), "pf_memcpy")
    return out


def test_codes(gpu):
    """Every step's borders and their neighbours, with a block's largest value on both sides of 7 steps; small and
    large blocks; rows of zeros; the bytes of the pages themselves."""
    D, G, page = 128, 2, 16
    borders = np.array([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5, 7], np.float32)
    some = np.concatenate([borders, np.nextafter(borders, np.float32(9)), np.nextafter(borders, np.float32(-9))])
    rng = np.random.default_rng(1)
    x = np.zeros((40, G, D), np.float32)
    for i in range(40):
        for g in range(G):
            for b in range(4):
                v = rng.choice(some, 32) * rng.choice(np.array([-1, 1], np.float32), 32)
                v[rng.integers(32)] = rng.choice(np.array([3.5, np.nextafter(np.float32(3.5), np.float32(4)), 7, 6, 4, 8], np.float32))
                scale = rng.choice(np.array([-127, -126, -125, -124, -60, -1, 0, 1, 50, 122, 123, 124, 125], np.float64))
                with np.errstate(over="ignore"):
                    v = (v.astype(np.float64) * 2.0 ** scale).astype(np.float32)
                x[i, g, 32 * b:32 * b + 32] = np.where(np.isfinite(v), v, 3e38)
    x[5] = 0
    x[6, 1] = -0.0
    c = pf.PagedCache(gpu, 1, G, D, 3, 1, 48, page, pf.TYPE_FP4)
    c.append([0], [40])
    c.store(0, dev(gpu, x), dev(gpu, -x))
    code, e = S.fp4_rows(x)
    k, v, ks, vs = c.planes(0)
    got = plane(gpu, k, 3 * G * page * 64).reshape(3, G, page, 64).transpose(0, 2, 1, 3).reshape(48, G, 64)[:40]
    np.testing.assert_array_equal(got & 0x77, S.fp4_bytes(code) & 0x77)
    got = plane(gpu, ks, 3 * G * page * 4).reshape(3, G, page, 4).transpose(0, 2, 1, 3).reshape(48, G, 4)[:40]
    np.testing.assert_array_equal(got, e)
    gk, gv = c.gather(0, [0])
    np.testing.assert_array_equal(gk.numpy(), S.fp4_values(code, e, D))
    np.testing.assert_array_equal(gv.numpy(), S.fp4_held(-x))
    assert c.memory_usage() == 2 * 3 * G * page * (64 + 4) + 3 * 4
    c.close()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("G,D", [(5, 48), (1, 16), (2, 80), (4, 64), (3, 112), (2, 128)])
def test_store_and_gather(gpu, t, G, D):
    m = Mirror(gpu, G, D, 16, 40, 3, 200, t=t)
    k, v = (R.rand(m.rng, (50, G, D), t) for _ in range(2))
    k[3] = 0
    m.append([2, 0], [33, 17], (k, v))
    m.append([0, 2], [5, 1])
    m.check([2, 0])
    m.check([0])
    for dt in (np.float16, np.uint16):
        got = m.c.gather(0, [2], dtype=dt)[0].numpy()
        name = "f16" if dt == np.float16 else "bf16"
        np.testing.assert_array_equal(R.from_bits(got, name), R.from_bits(R.to_bits(m.rows[2][0][0], name), name))
    # a block with an infinity or a NaN reads back as NaN, the others stay
    for bad in (np.inf, np.nan):
        x = R.rand(m.rng, (1, G, D), t)
        x[0, G - 1, D - 1] = R.to_bits(np.float32(bad), t)
        m.c.free([1])
        m.c.append([1], [1])
        m.c.store(0, dev(gpu, x), dev(gpu, x))
        got = m.c.gather(0, [1])[0].numpy()
        first = (D - 1) // 32 * 32
        assert np.isnan(got[0, G - 1, first:]).all()
        got[0, G - 1, first:] = 0
        want = S.fp4_held(R.from_bits(x, t))
        want[0, G - 1, first:] = 0
        np.testing.assert_array_equal(got, want)
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("H,G,D,page,lens,new", [
    (4, 4, 64, 16, [1], 1), (8, 2, 128, 64, [63, 64, 65, 200], 1), (16, 1, 64, 32, [31, 700], 1),
    (6, 3, 80, 16, [5, 130, 33], 5), (16, 2, 128, 128, [900, 8], 5), (32, 1, 112, 256, [300], 3),
    (2, 2, 16, 16, [40, 9], 8), (12, 12, 64, 64, [70], 20), (4, 2, 48, 16, [77, 32], 2), (3, 3, 96, 32, [257], 1),
])
def test_attention(gpu, t, H, G, D, page, lens, new):
    m = Mirror(gpu, G, D, page, sum(-(-n // page) for n in lens), len(lens), max(lens), t=t)
    seqs = list(range(len(lens)))
    print(f"4 bits {t} H {H} G {G} D {D} page {page} lens {lens} new {new}", flush=True)
    old = [max(0, n - new) for n in lens]
    for part in (3, 2, 1):       # grown in turn, so that their pages interleave
        m.append(seqs, [n // 3 if part > 1 else n - 2 * (n // 3) for n in old])
    m.append(seqs, [n - o for n, o in zip(lens, old)])
    assert m.c.free_pages == 0
    m.check(seqs)
    m.attention(H, seqs, [n - o for n, o in zip(lens, old)])
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("window,sink,causal", [(1, 0, True), (64, 4, True), (100, 70, True), (33, 500, True),
                                                (0, 0, False), (50, 3, False), (5000, 4, True)])
def test_masks(gpu, t, window, sink, causal):
    lens, new = [1, 40, 333, 700], [1, 6, 6, 0]
    m = Mirror(gpu, 2, 64, 32, 80, 4, 1000, t=t)
    m.append([0, 1, 2, 3], [n - a for n, a in zip(lens, new)])
    m.append([3, 1, 0, 2], [new[i] for i in (3, 1, 0, 2)])
    m.attention(4, [3, 1, 0, 2], [new[i] for i in (3, 1, 0, 2)], causal=causal, window=window, sink=sink)
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
def test_split(gpu, t):
    """Contexts long enough to be shared among workgroups, beside short ones; scale given; a second layer."""
    m = Mirror(gpu, 2, 128, 64, 260, 5, 9000, layers=2, t=t)
    lens, new = [9000, 1, 2500, 0, 700], [2, 1, 3, 0, 1]
    m.append(list(range(5)), [a - b for a, b in zip(lens, new)])
    m.append([4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)])
    for layer in (0, 1):
        m.attention(8, [4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)], layer=layer, scale=0.05)
    m.attention(8, [4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)], window=3000, sink=4)
    m.attention(2, [4, 0, 3, 2, 1], [new[i] for i in (4, 0, 3, 2, 1)])
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [48, 64, 112, 128])
def test_not_finite(gpu, t, D):
    """NaN blocks in keys and values of a verify pass's later drafts stay out of the earlier ones, what a shortened
    sequence leaves behind in its page out of all; a NaN block of a value reaches its own dims alone."""
    m = Mirror(gpu, 1, D, 64, 4, 1, 200, t=t)
    m.append([0], [30])
    bad = [R.rand(m.rng, (6, 1, D), t) for _ in range(2)]
    bad[0][4:] = R.to_bits(np.float32(np.nan), t)
    bad[1][3, 0, 5] = R.to_bits(np.float32(np.inf), t)
    m.append([0], [6], bad)
    q = R.rand(m.rng, (6, 2, D), t)
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), t)
    k, v = m.rows[0][0]
    want, tol = R.attend(R.from_bits(q, t), k, v, R.visible(6, 36), R.default_scale(D), t)
    R.check(y[:4, :, 32:], want[:4, :, 32:], tol[:4, :, 32:])
    R.check(y[:3], want[:3], tol[:3])
    assert np.isnan(y[3, :, :32]).all() and np.isnan(y[4:]).all()
    m.c.truncate([0], [33])
    m.rows[0][0] = tuple(x[:33] for x in m.rows[0][0])
    m.append([0], [1])
    m.attention(2, [0], [1])
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D,H", [(48, 2), (64, 10), (128, 2)])
def test_not_finite_in_whole_tiles(gpu, t, D, H):
    n, new = 450, 4
    m = Mirror(gpu, 1, D, 16, 29, 1, n, t=t)
    k, v = (R.rand(m.rng, (n, 1, D), t) for _ in range(2))
    v[7, 0, 1] = R.to_bits(np.float32(np.nan), t)
    m.append([0], [n - new], (k[:-new], v[:-new]))
    m.append([0], [new], (k[-new:], v[-new:]))
    q = R.rand(m.rng, (new, H, D), t)
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), t)
    want, tol = R.attend(R.from_bits(q, t), *m.rows[0][0], R.visible(new, n), R.default_scale(D), t)
    assert np.isnan(y[:, :, :32]).all()
    R.check(y[:, :, 32:], want[:, :, 32:], tol[:, :, 32:])
    m.c.close()


@pytest.mark.parametrize("t,size", [("f32", 2e38), ("bf16", 2e38), ("f32", 1e-30), ("bf16", 1e-30), ("f16", 6e4)])
@pytest.mark.parametrize("n,nq", [(100, 1), (3000, 2), (700, 5)])
def test_far_values(gpu, t, size, n, nq):
    """Values near the largest that the codes hold, and small ones.  6e4 is 3.66 * 2^14 and goes to 4 * 2^14 = 65536, as
    any value above 3.5 * 2^14 = 57344 does: more than fp16's largest, 65504, so an fp16 result of it is an infinity."""
    m = Mirror(gpu, 1, 64, 64, 50, 1, 3200, t=t)
    q, k, v = A.far_values(m.rng, t, n, nq, size)
    m.append([0], [n - nq], (k[:-nq], v[:-nq]))
    m.append([0], [nq], (k[-nq:], v[-nq:]))
    y = R.from_bits(m.c.attention(0, dev(gpu, q), scale=1.0).numpy(), t)
    want, tol = R.attend(R.from_bits(q, t), *m.rows[0][0], R.visible(nq, n), 1.0, t)
    if t == "f16":
        # 65520 and more round to infinity: results whose bounds reach there may be that
        inf = (np.abs(want) + tol >= 65520) & (y == np.copysign(np.inf, want))
        y, want, tol = y[~inf], want[~inf], tol[~inf]
    R.check(y, want, tol + A.lost_below(t, n))
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("D", [48, 64, 112, 128])
@pytest.mark.parametrize("H,G,lens,new,window,sink,causal", [
    (4, 2, [500, 405, 9, 430], 1, 0, 0, True), (16, 2, [402, 33, 512], 1, 0, 0, True),
    (8, 2, [390, 461], 5, 0, 0, True), (4, 2, [900, 500, 30], 3, 420, 5, True), (6, 2, [449, 403], 6, 0, 0, False),
])
def test_contexts_of_hundreds(gpu, t, D, H, G, lens, new, window, sink, causal):
    m = Mirror(gpu, G, D, 32, sum(-(-n // 32) for n in lens), len(lens), max(lens), t=t)
    seqs = list(range(len(lens)))
    print(f"4 bits {t} D {D} H {H} G {G} lens {lens} new {new} window {window}", flush=True)
    m.append(seqs, [n - new for n in lens])
    m.append(seqs, [new] * len(lens))
    m.attention(H, seqs, [new] * len(lens), causal=causal, window=window, sink=sink)
    m.c.close()


def test_many_tiles_a_wave(gpu):
    """Forks of one context, enough of them for a third workgroup on each compute unit (49152 tiles of 32 keys and a head)."""
    G, n = 24, 64
    m = Mirror(gpu, G, 128, 256, 4 + n, n, 1100, t="bf16")
    m.append([0], [1024])
    m.c.fork(0, list(range(1, n)))
    for s in range(1, n):
        m.rows[s] = list(m.rows[0])
    seqs = list(range(n))
    m.append(seqs, [1] * n)
    q = R.rand(m.rng, (n, G, 128), "bf16")
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), "bf16")
    for s in range(0, n, 9):
        want, tol = R.attend(R.from_bits(q[s:s + 1], "bf16"), *m.rows[s][0], R.visible(1, 1025), R.default_scale(128), "bf16")
        R.check(y[s:s + 1], want, tol, f"sequence {s}")
    m.c.close()


@pytest.mark.parametrize("t", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,held", [(62, 2), (63, 3)])
def test_around_many_tiles(gpu, t, n, held):
    """The last pass with two workgroups on a compute unit and the first with three (49152 tiles), its rule's choice asserted."""
    G = 24
    assert pages_plan(A.TYPE[t], pf.TYPE_FP4, G, G, 128, [1] * n, [1025] * n)[2] == held
    m = Mirror(gpu, G, 128, 256, 4 + n, n, 1100, t=t)
    m.append([0], [1024])
    m.c.fork(0, list(range(1, n)))
    for s in range(1, n):
        m.rows[s] = list(m.rows[0])
    m.append(list(range(n)), [1] * n)
    q = R.rand(m.rng, (n, G, 128), t)
    print(f"4 bits {t} {n} contexts of 1025", flush=True)
    y = R.from_bits(m.c.attention(0, dev(gpu, q)).numpy(), t)
    for s in range(0, n, 15):
        want, tol = R.attend(R.from_bits(q[s:s + 1], t), *m.rows[s][0], R.visible(1, 1025), R.default_scale(128), t)
        R.check(y[s:s + 1], want, tol, f"sequence {s}")
    m.c.close()


def test_many_sequences(gpu):
    n = 300
    m = Mirror(gpu, 1, 64, 16, 3000, n, 200, t="bf16")
    lens = [(13 * i) % 90 for i in range(n)]
    m.append(list(range(n)), lens)
    order = [(7 * i) % n for i in range(n)]
    new = [i % 4 for i in range(n)]
    m.append(order, new)
    m.check(order)
    m.attention(2, order, new)
    m.c.close()


@pytest.mark.parametrize("D", [32, 80])
def test_pages_moved(gpu, D):
    """Forks that grow into a shared page (odd counts of rows), copies, truncation and compaction keep rows and exponents."""
    m = Mirror(gpu, 3, D, 16, 40, 8, 150, layers=2)
    m.append([0, 1], [37, 21])
    m.c.fork(0, [2, 3])
    m.c.copy([1, 0], [4, 5])
    for s, src in ((2, 0), (3, 0), (4, 1), (5, 0)):
        m.rows[s] = list(m.rows[src])
    m.append([3, 0, 2, 4], [1, 2, 3, 30])
    m.check(range(6))
    m.c.truncate([5, 3], [33, 1])
    for s, n in ((5, 33), (3, 1)):
        m.rows[s] = [tuple(x[:n] for x in kv) for kv in m.rows[s]]
    m.c.free([1, 0])
    for s in (0, 1):
        m.rows[s] = [tuple(x[:0] for x in kv) for kv in m.rows[s]]
    assert m.c.compact() > 0
    m.check(range(6))
    m.append([3, 5, 2], [2, 1, 40])
    m.check(range(6))
    for layer in (0, 1):
        m.attention(6, [3, 5, 2], [2, 1, 40], layer=layer)
    m.c.close()


def test_pool_past_32_bits(gpu):
    """A sequence whose pages lie more than 2^32 bytes into a layer, in the second layer."""
    G, D, page, pages = 8, 128, 256, 34000
    m = Mirror(gpu, G, D, page, pages, 4, 33996 * page, layers=2, t="bf16")
    assert pages * G * page * D // 2 > 1 << 32
    m.c.append([0], [33995 * page])              # (its rows are never read)
    m.append([1], [300])
    assert m.c.tables([1])[0].tolist() == [[33995, 33996]]
    m.c.copy([1], [2])
    m.c.fork(1, [3])
    m.rows[2], m.rows[3] = list(m.rows[1]), list(m.rows[1])
    m.append([3, 1], [2, 1])                     # 3 copies the last page
    for layer in (0, 1):
        m.attention(16, [3, 1], [2, 1], layer=layer)
    m.check([1, 2, 3])
    m.c.free([0])
    m.c.compact()
    m.check([1, 2, 3])
    m.c.close()
