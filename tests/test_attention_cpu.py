"""What the attention and paged-cache entry points answer without a GPU: NULL
handles, the Python binding's argument checks, and the tests' own float64
attention against a direct sum."""
import numpy as np
import pytest

import attention_ref as R
import pocketforge_amd as pf


def test_null_handles():
    L = pf.lib()
    assert L.pf_prompt_attention(None, None, None, None, None, None, None, None, 0) == -1
    assert L.pf_pages_create(None, None, None) == -1
    L.pf_pages_destroy(None)
    assert L.pf_pages_memory_usage(None) == 0 and L.pf_pages_free_count(None) == 0 and L.pf_pages_length(None, 0) == 0
    assert L.pf_pages_tables(None, None, 0, None, 0, None) == -1
    assert L.pf_pages_planes(None, None, None, None, None) == -1
    assert L.pf_pages_append(None, None, None, 0) == -1
    assert L.pf_pages_store(None, 0, pf.TYPE_F32, None, None, 0, 0) == -1
    assert L.pf_pages_attention(None, None, 0, None, None) == -1
    assert L.pf_pages_gather(None, 0, None, 0, pf.TYPE_F32, None, None, 0, 0) == -1
    assert L.pf_pages_fork(None, 0, None, 0) == -1 and L.pf_pages_copy(None, None, None, 0) == -1
    assert L.pf_pages_truncate(None, None, None, 0) == -1 and L.pf_pages_free(None, None, 0) == -1
    assert L.pf_pages_compact(None, None) == -1


def test_lists():
    for a in ([], [1, 2], (3,), range(4), np.arange(3), np.arange(3, dtype=np.uint32), [np.int64(7)]):
        assert list(pf._u32(a, "a")) == [int(x) for x in a]
    for a in ([-1], [1.5], [1 << 32], "ab", 5, None, np.array([0.5]), [[1]]):
        with pytest.raises(pf.PFError):
            pf._u32(a, "a")


class Rows:
    """What the binding looks at in a device array."""

    def __init__(self, shape, stride, dtype):
        self.shape, self._stride, self.dtype = shape, stride, dtype

    def stride(self):
        return self._stride


def test_rows():
    assert pf._rows(Rows((5, 4, 64), (256, 64, 1), "torch.float16"), "q") == (5, 4, 64, 256)
    assert pf._rows(Rows((5, 4, 64), (768, 64, 1), "torch.float16"), "q") == (5, 4, 64, 768)
    assert pf._rows(Rows((1, 4, 64), (1, 64, 1), "torch.float16"), "q") == (1, 4, 64, 256)
    for shape, stride in (((5, 256), (256, 1)), ((5, 4, 64), (256, 1, 4)), ((5, 4, 64), (64, 320, 1))):
        with pytest.raises(pf.PFError):
            pf._rows(Rows(shape, stride, "torch.float16"), "q")


def test_types():
    for name, t in (("float32", pf.TYPE_F32), ("float16", pf.TYPE_F16), ("torch.bfloat16", pf.TYPE_BF16),
                    (np.dtype(np.uint16), pf.TYPE_BF16)):
        assert pf._type(Rows((), (), name)) == t
    with pytest.raises(pf.PFError):
        pf._type(Rows((), (), "torch.int8"))


@pytest.mark.parametrize("causal,window,sink", [(True, 0, 0), (False, 0, 0), (True, 3, 1), (False, 2, 0), (True, 1, 9)])
def test_reference_attention(causal, window, sink):
    rng = np.random.default_rng(1)
    nq, nk, H, G, D = 5, 9, 4, 2, 8
    q, k, v = (rng.standard_normal(s) for s in ((nq, H, D), (nk, G, D), (nk, G, D)))
    got, tol = R.attend(q, k, v, R.visible(nq, nk, causal, window, sink), 0.3, "f32")
    for i in range(nq):
        p = nk - nq + i
        for h in range(H):
            num, den = np.zeros(D), 0.0
            for j in range(nk):
                if causal and j > p:
                    continue
                if window and not (j > p - window or j < sink):
                    continue
                w = np.exp(0.3 * float(q[i, h] @ k[j, h // 2]))
                num += w * v[j, h // 2]
                den += w
            np.testing.assert_allclose(got[i, h], num / den, rtol=1e-12, atol=1e-14)
    assert (tol > 0).all() and (tol < 1e-4).all()


def test_reference_empty_rows_and_masked_nan():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((4, 1, 8)), rng.standard_normal((2, 1, 8)), rng.standard_normal((2, 1, 8))
    v[1] = np.nan
    got, _ = R.attend(q, k, v, R.visible(4, 2), 1.0, "f32")
    assert (got[:2] == 0).all() and np.isfinite(got[2]).all() and np.isnan(got[3]).all()


def test_reference_types():
    x = np.array([1.0, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, -0.0, np.inf, np.nan, 3e38], np.float32)
    b = R.from_bits(R.to_bits(x, "bf16"), "bf16")
    assert b[0] == 1 and b[1] == 1 and b[2] == 1 + 2.0 ** -6 and b[4] == np.inf and np.isnan(b[5])
    c, s = R.quantize_rows(np.array([[0.0, 0.0], [1.0, -2.0], [np.inf, 1.0]], np.float32))
    assert c.tolist() == [[0, 0], [64, -127], [0, 0]] and s[0, 0] == 1 and s[1, 0] == np.float32(2) / np.float32(127)
    assert np.isnan(s[2, 0])


@pytest.mark.parametrize("stride", [0, 64, 255])
def test_rows_that_overlap(stride):
    """Rows that share memory (x.expand(n, heads, head_dim) has a stride of 0, which the C calls read as packed)."""
    assert pf._rows(Rows((1, 4, 64), (stride, 64, 1), "torch.float16"), "q") == (1, 4, 64, 256)
    with pytest.raises(pf.PFError):
        pf._rows(Rows((5, 4, 64), (stride, 64, 1), "torch.float16"), "q")
    torch = pytest.importorskip("torch")
    with pytest.raises(pf.PFError):
        pf._rows(torch.zeros((1, 4, 64)).expand(5, 4, 64), "k")


class Placed:
    """A tensor of one GPU, as the binding asks for it."""

    def __init__(self, device):
        self.device = device

    def get_device(self):
        return self.device


def test_rows_elsewhere():
    """Rows in host memory or on another GPU than the context's are refused before their address goes anywhere."""
    ctx = pf.Context.__new__(pf.Context)
    ctx.device, ctx.h = 1, None
    own = pf.DeviceArray.__new__(pf.DeviceArray)
    own.ctx, own.ptr = ctx, 256
    pf._here(ctx, own, "q")
    pf._here(ctx, Placed(1), "k")
    other = pf.Context.__new__(pf.Context)
    other.device, other.h = 0, None
    far = pf.DeviceArray.__new__(pf.DeviceArray)
    far.ctx, far.ptr = other, 256
    freed = pf.DeviceArray.__new__(pf.DeviceArray)
    freed.ctx, freed.ptr = ctx, None
    for x in (far, freed, Placed(0), Placed(-1), np.zeros((2, 4, 64), np.float16), [1.0], None):
        with pytest.raises(pf.PFError, match="k "):
            pf._here(ctx, x, "k")
    torch = pytest.importorskip("torch")
    with pytest.raises(pf.PFError, match="out "):
        pf._here(ctx, torch.zeros((2, 4, 64)), "out")
    x = np.zeros((2, 4, 64), np.float16)
    host = torch.zeros((2, 4, 64), dtype=torch.float16)
    cache = pf.PagedCache.__new__(pf.PagedCache)
    cache.ctx, cache.h, cache.pass_rows, cache.n_kv_heads, cache.head_dim = ctx, None, 2, 4, 64
    for a, ctx.device in ((x, 1), (host, 1), (x, 0), (host, 0)):
        with pytest.raises(pf.PFError, match="GPU"):
            ctx.prompt_attention(a, a, a, [2], out=a)
        with pytest.raises(pf.PFError, match="GPU"):
            cache.store(0, a, a)
        with pytest.raises(pf.PFError, match="GPU"):
            cache.attention(0, a, out=a)


def test_numbers():
    """Numbers that do not fit 32 bits are refused, not taken modulo 2^32."""
    assert [pf._num(x, "n") for x in (0, 7, np.int64(9), 0xFFFFFFFF)] == [0, 7, 9, 0xFFFFFFFF]
    for x in (-1, 1 << 32, 1.5, "1", None, [1]):
        with pytest.raises(pf.PFError, match="n is"):
            pf._num(x, "n")
    ctx = pf.Context.__new__(pf.Context)
    ctx.device, ctx.h = 0, None
    x = pf.DeviceArray.__new__(pf.DeviceArray)
    x.ctx, x.ptr, x.shape, x.dtype = ctx, 256, (2, 4, 64), np.dtype(np.float16)
    y = pf.DeviceArray.__new__(pf.DeviceArray)
    y.ctx, y.ptr, y.shape, y.dtype = ctx, 4096, (2, 4, 64), np.dtype(np.float16)
    c = pf.PagedCache.__new__(pf.PagedCache)
    c.ctx, c.h, c.pass_rows, c.n_kv_heads, c.head_dim, c.max_seqs, c.n_layers = ctx, None, 2, 4, 64, 3, 2
    for bad in (-1, 1 << 32):
        for kw in (dict(window=bad), dict(sink=bad)):
            with pytest.raises(pf.PFError, match=next(iter(kw))):
                ctx.prompt_attention(x, x, x, [2], out=y, **kw)
            with pytest.raises(pf.PFError, match=next(iter(kw))):
                c.attention(0, x, out=y, **kw)
        for f in (lambda: c.attention(bad, x, out=y), lambda: c.store(bad, x, x), lambda: c.gather(bad, []),
                  lambda: c.planes(bad)):
            with pytest.raises(pf.PFError, match="layer"):
                f()
        with pytest.raises(pf.PFError, match="src"):
            c.fork(bad, [1])
        with pytest.raises(pf.PFError, match="seq"):
            c.length(bad)
        for name in ("n_layers", "n_kv_heads", "head_dim", "n_pages", "max_seqs", "max_context", "page_size"):
            f = dict(n_layers=1, n_kv_heads=1, head_dim=64, n_pages=1, max_seqs=1, max_context=64, page_size=64)
            f[name] = bad
            with pytest.raises(pf.PFError, match=name):
                pf.PagedCache(ctx, **f)
    with pytest.raises(pf.PFError, match="layer"):
        c.planes(2)
    with pytest.raises(pf.PFError, match="stride"):
        pf._rows(Rows((2, 4, 64), ((1 << 32) + 256, 64, 1), "torch.float16"), "q")
