"""Operators of a serving step around the paged cache, as cases.

  decode   attention of each sequence's newest rows over pages of 4-bit floats
  store    new key / value rows quantised into such pages, and rows read back
  rotary   rows of heads turned by their positions
  turned   a pass's queries turned, its keys turned and stored, its values stored
  sample   tokens chosen from rows of logits with temperature, top-k, top-p and
           min-p, from given random numbers

Head counts, head sizes, verify rows, the base of the positions, vocabularies
and sampling settings are those of the repository's models and defaults (4 x 64, 12 x 64,
16 x 128; five verify rows; base 5e6; 16384 and 130560 tokens; 0.8 and top-p
0.95), and of the same models with grouped key / value heads.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
BLOCK = 32          # dims that share a power of two in 4-bit pages
GROW = 4            # appends that bring a sequence to its length, in turn with the others

_ctx = []


def _context():
    """One context per process, as the library's programs keep it."""
    if not _ctx:
        import pocketforge_amd as pf
        _ctx.append(pf.Context(0))
    return _ctx[0]


# ------------------------------------------------------------------ cases

# positions of a model stretched to eight times the context it was trained on
LONG = dict(base=5e6, factor=8.0, low=1.0, high=32.0, original=8192, magnitude=1.2079441541679836)
PLAIN = dict(base=5e6, factor=1.0, low=0.0, high=0.0, original=0, magnitude=1.0)


def listed():
    return [
        # one user, a short context: a decode step's latency
        dict(name="decode_single", kind="decode", type="bf16", heads=16, kv=16, dim=128, seqs=1, context=700, rows=1,
             page=64, window=0, sink=0),
        # a serving batch of ragged contexts, grouped heads
        dict(name="decode_batch", kind="decode", type="bf16", heads=16, kv=4, dim=128, seqs=64, context=16000, rows=1,
             page=64, window=0, sink=0),
        # two long documents: the work has to be split over the context
        dict(name="decode_long", kind="decode", type="f16", heads=16, kv=2, dim=128, seqs=2, context=120000, rows=1,
             page=128, window=0, sink=0),
        # verify passes of four drafts: fp32 rows, every head with its own keys
        dict(name="verify", kind="decode", type="f32", heads=16, kv=16, dim=128, seqs=16, context=2100, rows=5,
             page=64, window=0, sink=0),
        # one decode step's rows of a batch, and the batch read back
        dict(name="store_step", kind="store", type="bf16", kv=4, dim=128, seqs=64, context=90, rows=1, page=64),
        # a prompt's fp32 rows into the pages, and read back for the next prompt pass
        dict(name="store_prompt", kind="store", type="f32", kv=16, dim=128, seqs=3, context=64, rows=2000, page=64),
        # queries and keys of a decode batch (16 + 4 heads) at far positions
        dict(name="rotary_step", kind="rotary", type="bf16", heads=20, dim=128, turn=128, pairs=False, rows=64,
             far=100000, **LONG),
        # a long document's queries
        dict(name="rotary_long", kind="rotary", type="bf16", heads=16, dim=128, turn=128, pairs=True, rows=8192,
             far=0, **PLAIN),
        # a decode step of a batch over 16-bit pages
        dict(name="turned_step", kind="turned", type="bf16", cache="bf16", heads=16, kv=4, dim=128, turn=128,
             pairs=True, seqs=64, context=500, rows=1, page=64, **PLAIN),
        # packed prompts into 4-bit pages, half of each head turned, stretched positions
        dict(name="turned_prompt", kind="turned", type="bf16", cache="fp4", heads=16, kv=4, dim=128, turn=64,
             pairs=False, seqs=24, context=1, rows=700, page=64, **LONG),
        # the rows of one verify pass, as the engine's models have them
        dict(name="sample_verify", kind="sample", type="f32", rows=5, vocab=16384, sets="p"),
        # a serving batch of requests with settings of their own, some under a grammar's mask
        dict(name="sample_batch", kind="sample", type="bf16", rows=64, vocab=130560, sets="mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _positions(rng):
    s = dict(rng.choice([LONG, PLAIN, PLAIN]))
    if rng.random() < 0.3:      # every frequency divided alike
        s = dict(PLAIN, factor=float(rng.choice([2, 4])))
    return dict(s, base=float(rng.choice([1e4, 5e5, 5e6])))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "store", "rotary", "turned", "sample", "sample"])
    dim = rng.choice([64, 128, 128, 16 * rng.randint(2, 8)])
    kv, group = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4, 8])
    if kv * group > 64:
        group = 1
    turn = rng.choice([dim, dim, dim // 2 & ~7])
    if kind == "decode":
        c = dict(kind=kind, type=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=kv * group, kv=kv, dim=dim,
                 seqs=_log(rng, 1, 128), context=_log(rng, 1, 120000), rows=rng.choice([1, 1, 1, 5, rng.randint(2, 8)]),
                 page=rng.choice([16, 32, 64, 64, 128]), window=rng.choice([0, 0, 0, _log(rng, 16, 4000)]),
                 sink=rng.choice([0, 4]))
        c["context"] = max(c["context"], c["rows"])
        while c["seqs"] * c["context"] * c["kv"] * c["dim"] > 5e8 or c["seqs"] * c["context"] * c["heads"] * c["rows"] > 1e8:
            c["context"] = max(c["rows"], c["context"] * 2 // 3)
            c["seqs"] = max(1, c["seqs"] * 2 // 3)
        return c
    if kind == "store":
        c = dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), kv=kv, dim=dim, seqs=_log(rng, 1, 128),
                 context=_log(rng, 1, 2000), rows=rng.choice([1, 5, _log(rng, 1, 4000)]),
                 page=rng.choice([16, 32, 64, 128]))
        while c["seqs"] * (c["rows"] + c["context"]) * c["kv"] * c["dim"] > 4e7:
            c["rows"], c["context"] = max(1, c["rows"] * 2 // 3), max(1, c["context"] * 2 // 3)
            c["seqs"] = max(1, c["seqs"] * 3 // 4)
        return c
    if kind == "rotary":
        c = dict(kind=kind, type=rng.choice(["bf16", "f16", "f32"]), heads=kv * group + kv, dim=dim, turn=turn,
                 pairs=rng.random() < 0.5, rows=_log(rng, 1, 20000), far=rng.choice([0, 0, _log(rng, 1000, 1000000)]),
                 **_positions(rng))
        while c["rows"] * c["heads"] * c["dim"] > 1.6e7:
            c["rows"] = c["rows"] * 2 // 3
        return c
    if kind == "turned":
        c = dict(kind=kind, type=rng.choice(["bf16", "f16", "f32"]), cache=rng.choice(["fp4", "fp4", "i8", "bf16"]),
                 heads=kv * group, kv=kv, dim=dim, turn=turn, pairs=rng.random() < 0.5, seqs=_log(rng, 1, 128),
                 context=_log(rng, 1, 2000), rows=rng.choice([1, 5, _log(rng, 1, 3000)]),
                 page=rng.choice([16, 32, 64, 128]), **_positions(rng))
        while c["seqs"] * (c["rows"] + c["context"]) * (c["kv"] + c["heads"]) * c["dim"] > 4e7:
            c["rows"], c["context"] = max(1, c["rows"] * 2 // 3), max(1, c["context"] * 2 // 3)
            c["seqs"] = max(1, c["seqs"] * 3 // 4)
        return c
    c = dict(kind=kind, type=rng.choice(["bf16", "f16", "f32"]), rows=_log(rng, 1, 300),
             vocab=_log(rng, 1000, 200000), sets=rng.choice(["mixed", "mixed", "p", "k", "all"]))
    while c["rows"] * c["vocab"] > 8.2e6:
        c["rows"] = max(1, c["rows"] * 2 // 3)
    return c


def _ragged(n, longest, least=1):
    """n lengths between a quarter of the longest and the longest itself."""
    return [max(least, int(longest * (1.0 - 0.75 * (0.618034 * i % 1.0)))) for i in range(n)]


def _visible(q_len, k_len, window, sink):
    """Pairs of a query and a key that it sees (the queries are the last q_len positions), and keys seen by any."""
    pairs, first = 0, max(0, k_len - q_len)
    lo = max(0, first - window + 1) if window else 0
    for p in range(first, k_len):
        w = max(0, p - window + 1) if window else 0
        pairs += p + 1 - w + min(sink, w)
    return pairs, k_len - lo + min(sink, lo)


def _blocks(dim):
    return -(-dim // BLOCK)


def _row_bytes(cache, kv, dim):
    if cache == "fp4":
        return kv * _blocks(dim) * (BLOCK // 2 + 1)
    return kv * (dim * SIZE[cache] + (4 if cache == "i8" else 0))


def work(case):
    kind = case["kind"]
    if kind == "sample":
        # per logit: its difference, the product, 2^x by a polynomial, two sums, comparisons
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * SIZE[case["type"]] + 32 * case["rows"], flops=25.0 * n)
    dim, size = case["dim"], SIZE[case["type"]]
    if kind == "rotary":
        n = case["rows"] * case["heads"] * dim
        return dict(bytes=2 * n * size + 4 * case["rows"], flops=3.0 * n)
    kv, row = case["kv"], _row_bytes(case.get("cache", "fp4"), case["kv"], dim)
    if kind == "decode":
        k = _ragged(case["seqs"], case["context"], case["rows"])
        seen = [_visible(case["rows"], n, case["window"], case["sink"]) for n in k]
        q = 2 * case["heads"] * case["seqs"] * case["rows"] * dim * size
        return dict(bytes=2 * row * sum(k for _, k in seen) + q,
                    flops=4.0 * dim * case["heads"] * sum(p for p, _ in seen))
    new = sum(_new_rows(case))
    got = 2 * new * kv * dim * size + 2 * row * new
    back = 0
    if case.get("cache", "fp4") != "bf16":
        old = sum(_ragged(case["seqs"], case["context"]))
        back = 2 * (old + new) * (row + kv * dim * size)
    turned = 2 * new * case["heads"] * dim * size if kind == "turned" else 0
    return dict(bytes=got + back + turned, flops=3.0 * new * dim * (kv + case["heads"]) if turned else 0.0)


# ---------------------------------------------------------------- inputs

def _rand(seed, shape, type):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(TYPES[type])


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _new_rows(case):
    return [case["rows"]] * case["seqs"] if case["kind"] == "decode" else _ragged(case["seqs"], case["rows"])


def _lens(case):
    if case["kind"] == "decode":
        return _ragged(case["seqs"], case["context"], case["rows"])
    return [a + b for a, b in zip(_ragged(case["seqs"], case["context"]), _new_rows(case))]


def _rows(case, seed):
    """Key and value rows of every sequence, one after another; a row in sixteen and a dim in fifty stand out, as
    caches have them."""
    shape = (sum(_lens(case)), case["kv"], case["dim"])
    k, v = _rand(seed + 1, shape, "f32"), _rand(seed + 2, shape, "f32")
    k[::16] *= 2.0
    v[::16] *= 4.0
    k[..., ::50] *= 3.0
    return k.to(TYPES[case["type"]]), v.to(TYPES[case["type"]])


def _last_rows(lens, new):
    return torch.cat([torch.arange(a + n - c, a + n) for a, n, c in zip(_starts(lens), lens, new)]).cuda()


def _far(case, seed):
    rng = random.Random(seed)
    return [rng.randint(0, case["far"]) for _ in range(case["rows"])]


def _settings(case, seed):
    """Each row's temperature, top-k, top-p and min-p: one setting for all ("p", "k", "all"), or requests' own."""
    rng, out = random.Random(seed), []
    fixed = {"p": (0.8, 0, 0.95, 0.0), "k": (1.0, 50, 1.0, 0.0), "all": (1.0, 0, 1.0, 0.0)}
    for _ in range(case["rows"]):
        out.append(fixed.get(case["sets"]) or rng.choice([
            (0.0, 0, 1.0, 0.0), (0.8, 0, 0.95, 0.0), (1.0, 50, 1.0, 0.0), (0.7, 40, 0.9, 0.05), (1.0, 0, 1.0, 0.02),
            (1.3, 200, 0.98, 0.0), (1.0, 0, 1.0, 0.0)]))
    return [torch.tensor(x, device="cuda", dtype=t) for x, t in
            zip(zip(*out), (torch.float32, torch.int32, torch.float32, torch.float32))]


def _logits(case, seed):
    """Logits that fall with the logarithm of a token's rank, in an order of each row's own, with noise; every
    fifth row of mixed settings has two thirds of its tokens masked."""
    n, v = case["rows"], case["vocab"]
    rank = torch.rand((n, v), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * v + 1.0
    x = -1.6 * rank.log() + 0.7 * _rand(seed + 1, (n, v), "f32") + 9.0
    if case["sets"] == "mixed":
        x[::5, torch.arange(v, device="cuda") % 3 > 0] = -math.inf
    return x.to(TYPES[case["type"]])


def _place(case, lens, old):
    """For the plain form: the pages that the cache gives the sequences (lowest first, by the growth of _fill, then
    by the last rows), the place of each row, and the number of pages."""
    ps, table, at = case["page"], [[] for _ in lens], 0
    for r in range(GROW + 1):
        for i, n in enumerate(lens):
            have = old[i] * (r + 1) // GROW if r < GROW else n
            while len(table[i]) * ps < have:
                table[i].append(at)
                at += 1
    place = torch.cat([(torch.tensor(t)[:, None] * ps + torch.arange(ps)).flatten()[:n] for t, n in zip(table, lens)])
    most = max(map(len, table))
    return torch.tensor([t + [0] * (most - len(t)) for t in table], device="cuda"), place.cuda(), at


def _cache(case, lens):
    import pocketforge_amd as pf
    kinds = {"i8": pf.TYPE_I8, "bf16": pf.TYPE_BF16, "fp4": pf.TYPE_FP4}
    ps = case["page"]
    return pf.PagedCache(_context(), n_layers=1, n_kv_heads=case["kv"], head_dim=case["dim"], page_size=ps,
                         n_pages=sum(-(-n // ps) for n in lens), max_seqs=len(lens), max_context=max(lens),
                         type=kinds[case.get("cache", "fp4")])


def _fill(cache, k, v, lens, counts):
    """Grows every sequence by its count, a part at a time and in turn, so that their pages interleave."""
    at, done, seqs = _starts(lens), [0] * len(lens), list(range(len(lens)))
    for r in range(GROW):
        part = [c * (r + 1) // GROW - c * r // GROW for c in counts]
        if not sum(part):
            continue
        rows = torch.cat([torch.arange(a + d, a + d + p) for a, d, p in zip(at, done, part)]).cuda()
        kr, vr = k[rows], v[rows]
        torch.cuda.synchronize()
        cache.append(seqs, part)
        cache.store(0, kr, vr)
        cache.ctx.synchronize()
        done = [d + p for d, p in zip(done, part)]


def _rotary(case):
    import pocketforge_amd as pf
    return pf.Rotary(_context(), case["dim"], turn=case["turn"], interleaved=case["pairs"], base=case["base"],
                     factor=case["factor"], low=case["low"], high=case["high"], original=case["original"],
                     magnitude=case["magnitude"])


def prepare(case, seed):
    state, kind = dict(case), case["kind"]
    if kind == "rotary":
        n = case["rows"]
        state["x"] = _rand(seed, (n, case["heads"], case["dim"]), case["type"])
        state["out"] = torch.zeros_like(state["x"])
        at = torch.arange(n, dtype=torch.int32)
        if case["far"]:
            at = torch.tensor(_far(case, seed), dtype=torch.int32)
        state["at"] = at.cuda()
        if own:
            state["rotary"] = _rotary(case)
    elif kind == "sample":
        state["logits"] = _logits(case, seed)
        state["u"] = torch.rand(case["rows"], generator=torch.Generator(device="cuda").manual_seed(seed + 2),
                                device="cuda")
        state["temperature"], state["top_k"], state["top_p"], state["min_p"] = _settings(case, seed)
        if own:
            state["ctx"] = _context()
            state["tokens"] = torch.zeros(case["rows"], dtype=torch.int32, device="cuda")
            state["probs"] = torch.zeros(case["rows"], device="cuda")
    else:
        lens, new = _lens(case), _new_rows(case)
        old = [n - c for n, c in zip(lens, new)]
        k, v = _rows(case, seed)
        last = _last_rows(lens, new)
        state.update(lens=lens, old=old, new=new, seq_ids=list(range(len(lens))))
        state["k"], state["v"] = k[last].contiguous(), v[last].contiguous()
        if kind != "store":
            state["q"] = _rand(seed, (sum(new), case["heads"], case["dim"]), case["type"])
            state["out"] = torch.zeros_like(state["q"])
        cache = case.get("cache", "fp4")
        if own:
            handle = state["handle"] = _cache(case, lens)
            if kind != "decode":
                # pages that no row has been written to hold zeros
                planes = handle.planes(0)
                torch.cuda.synchronize()
                for p in planes:
                    torch.as_tensor(p, device="cuda").zero_()
                torch.cuda.synchronize()
            _fill(handle, k, v, lens, old)
            torch.cuda.synchronize()
            handle.append(state["seq_ids"], new)
            if kind == "decode":
                handle.store(0, state["k"], state["v"])
            handle.ctx.synchronize()
            if kind == "turned":
                state["rotary"] = _rotary(case)
            if cache != "bf16" and kind != "decode":
                state["back"] = [torch.zeros_like(k) for _ in range(2)]
            elif kind == "turned":
                state["pool"] = [torch.as_tensor(p, device="cuda").view(torch.bfloat16) for p in handle.planes(0)]
        else:
            state["table"], place, pages = _place(case, lens, old)
            state["place"], state["last"] = place, place[last]
            keep = torch.ones(len(k), dtype=torch.bool, device="cuda")
            if kind != "decode":
                keep[last] = False
            state["pool"] = []
            for x in (k, v):
                for part in _held(x, cache):
                    pool = torch.zeros((pages, case["kv"], case["page"]) + part.shape[2:], dtype=part.dtype,
                                       device="cuda")
                    pool[place[keep] // case["page"], :, place[keep] % case["page"]] = part[keep]
                    state["pool"].append(pool)
            state["k_lens"] = torch.tensor(lens, device="cuda")
            state["q_pos"] = torch.tensor([list(range(n - c, n)) for n, c in zip(lens, new)], device="cuda") \
                if kind == "decode" else None
            state["at"] = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, new)]).cuda()
    torch.cuda.synchronize()
    return state


# ------------------------------------------------------------ plain forms

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _codes4(x):
    """4-bit codes, two to a byte (the even dim's low), and the exponent of each block of 32 dims: the smallest power
    of two that takes the block's largest value to 7 or less; ties to even codes."""
    x = torch.nn.functional.pad(x.float(), (0, _blocks(x.shape[-1]) * BLOCK - x.shape[-1]))
    x = x.unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1, keepdim=True)
    e = (((top.view(torch.int32) + 0x1FFFFF) >> 23) - 2).clamp(2, 252)
    a = x.abs().double() * torch.exp2((127 - e).double())
    c = (a > 0.25).int()
    for border, up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= border if up else a > border).int()
    c = (c | ((x < 0).int() << 3)).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), e[..., 0].to(torch.uint8)


def _values4(codes, e, dim):
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    table = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=codes.device)
    x = table[both].unflatten(-1, (-1, BLOCK)) * torch.exp2(e.float() - 127.0)[..., None]
    return x.flatten(-2)[..., :dim]


def _codes8(x):
    """The cache's int8 rows: codes round(x * (127 / max|x|)), scale max|x| / 127."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    full = torch.full_like(amax, 127.0)   # tensors: a division by or of a number may be a product
    one = torch.ones_like(amax)
    v = (x * torch.where(amax == 0, one, full / amax)).double()
    codes = torch.sign(v) * torch.floor(v.abs() + 0.5)
    return codes.to(torch.int8), torch.where(amax == 0, one, amax / full)


def _held(x, cache):
    """What the pages hold of rows."""
    return _codes4(x) if cache == "fp4" else _codes8(x) if cache == "i8" else (x.to(TYPES[cache]),)


def _read(parts, cache, dim):
    if cache == "fp4":
        return _values4(*parts, dim)
    return parts[0].float() * parts[1] if cache == "i8" else parts[0].float()


def _attend(q, k, v, q_pos, k_lens, window, sink):
    """q [n, rows, heads, dim] at positions q_pos [n, rows] over k, v
    [n, keys, kv heads, dim] of k_lens keys, in 32 bits."""
    n, rows, heads, dim = q.shape
    kv = k.shape[2]
    q = q.permute(0, 2, 1, 3).reshape(n, kv, heads // kv * rows, dim)
    k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()
    s = torch.matmul(q, k).view(n, heads, rows, -1)
    s *= 1.0 / math.sqrt(dim)
    j = torch.arange(k.shape[-1], device=q.device)
    p = q_pos[:, :, None]
    seen = (j <= p) & (j < k_lens[:, None, None])
    if window:
        seen &= (j > p - window) | (j < sink)
    s.masked_fill_(~seen[:, None], -math.inf)
    s -= s.amax(-1, keepdim=True)
    s.exp_()
    s /= s.sum(-1, keepdim=True)
    return torch.matmul(s.view(n, kv, heads // kv * rows, -1), v).view(n, heads, rows, dim).transpose(1, 2)


def _plain_decode(s):
    k, v = (_values4(c[s["table"]], e[s["table"]], s["dim"]) for c, e in (s["pool"][:2], s["pool"][2:]))
    k, v = (t.transpose(2, 3).reshape(s["seqs"], -1, s["kv"], s["dim"]) for t in (k, v))
    # pages past a sequence's end hold other sequences' rows: their weight is zero
    q = s["q"].float().view(s["seqs"], s["rows"], s["heads"], s["dim"])
    o = _attend(q, k, v, s["q_pos"], s["k_lens"], s["window"], s["sink"])
    return o.reshape(-1, s["heads"], s["dim"]).to(s["q"].dtype)


def _angles(s, at):
    """[rows, turn / 2] in 64 bits."""
    i = torch.arange(s["turn"] // 2, device=at.device, dtype=torch.float64)
    f = torch.exp2(i * (-2.0 / s["turn"] * math.log2(s["base"])))
    if s["high"] > s["low"]:
        keep = ((f * (s["original"] / (2 * math.pi)) - s["low"]) / (s["high"] - s["low"])).clamp(0, 1)
        f = f * (keep + (1 - keep) / s["factor"])
    else:
        f = f / s["factor"]
    return at.double()[:, None] * f


def _turn(s, x, at, dtype):
    """x [rows, heads, dim] turned, with products of dtype, as 32 bits."""
    a = _angles(s, at)
    c, d = ((t * s["magnitude"]).to(dtype)[:, None] for t in (torch.cos(a), torch.sin(a)))
    x, out, r = x.to(dtype), x.float().clone(), s["turn"]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if s["pairs"] else (slice(0, r // 2), slice(r // 2, r))
    u, w = x[..., first], x[..., second]
    out[..., first] = (u * c - w * d).float()
    out[..., second] = (u * d + w * c).float()
    return out


def _write(s, k, v):
    """Rows into the pages; what the pages hold after that."""
    ps, to, cache = s["page"], s["last"], s.get("cache", "fp4")
    parts = [p for x in (k, v) for p in _held(x, cache)]
    for pool, x in zip(s["pool"], parts):
        pool[to // ps, :, to % ps] = x
    if cache == "bf16":
        return dict(k=s["pool"][0], v=s["pool"][1])
    at = s["place"]
    rows = [p[at // ps, :, at % ps] for p in s["pool"]]
    k, v = (_read(r, cache, s["dim"]).to(TYPES[s["type"]]) for r in (rows[:2], rows[2:]))
    return dict(k=k, v=v)


def _plain_turned(s):
    # (64 bits where a rounding decides on a code)
    wide = torch.float32 if s["cache"] == "bf16" else torch.float64
    q = _turn(s, s["q"], s["at"], torch.float32).to(s["q"].dtype)
    return dict(_write(s, _turn(s, s["k"], s["at"], wide), s["v"]), q=q)


def _plain_sample(s):
    x = s["logits"].double()
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    hot = s["temperature"][:, None].double()
    n = torch.arange(x.shape[1], device=x.device)
    w = torch.where(hot > 0, torch.exp((x - x[:, :1]) / torch.where(hot > 0, hot, 1.0)), (n == 0).double())
    total = w.cumsum(-1)
    k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1]).clamp(max=x.shape[1]).long()[:, None]
    kept = n < k
    mass = total.gather(1, k - 1)
    p = s["top_p"][:, None].double()
    kept &= (total - w < p * mass) | (p >= 1)
    kept &= w >= s["min_p"][:, None].double()
    mass = (w * kept).sum(-1, keepdim=True)
    pick = (total <= s["u"][:, None].double() * mass).sum(-1, keepdim=True)
    return dict(tokens=order.gather(1, pick)[:, 0].int(), probs=(w.gather(1, pick) / mass)[:, 0].float())


def run(s):
    kind = s["kind"]
    if not own:
        if kind == "rotary":
            return _turn(s, s["x"], s["at"], torch.float32).to(s["x"].dtype)
        if kind == "store":
            return _write(s, s["k"], s["v"])
        return {"decode": _plain_decode, "turned": _plain_turned, "sample": _plain_sample}[kind](s)
    if kind == "rotary":
        return s["rotary"].apply(s["x"], s["at"], out=s["out"])
    if kind == "sample":
        tokens, probs = s["ctx"].sample_rows(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                                             top_p=s["top_p"], min_p=s["min_p"], out=(s["tokens"], s["probs"]))
        return dict(tokens=tokens, probs=probs)
    cache = s["handle"]
    if kind == "decode":
        return cache.attention(0, s["q"], causal=True, window=s["window"], sink=s["sink"], out=s["out"])
    cache.truncate(s["seq_ids"], s["old"])
    cache.append(s["seq_ids"], s["new"])
    got = {}
    if kind == "store":
        cache.store(0, s["k"], s["v"])
    else:
        got["q"] = cache.store_rotary(0, s["rotary"], s["q"], s["k"], s["v"], out=s["out"])
    if "pool" in s:
        return dict(got, k=s["pool"][0], v=s["pool"][1])
    k, v = cache.gather(0, s["seq_ids"], out=s["back"])
    return dict(got, k=k, v=v)


# ----------------------------------------------------- values in 64 bits

def _stands4(x):
    """What 4-bit codes of 32-bit rows stand for."""
    dim = x.shape[-1]
    out = torch.empty_like(x, dtype=torch.float64)
    for d in range(0, dim, BLOCK):
        b = x[..., d:d + BLOCK].double()
        top = b.abs().max(-1, keepdim=True).values
        scale = torch.exp2(torch.ceil(torch.log2(top / 7)).clamp(-125, 125))
        scale = torch.where(top > 7 * scale, 2 * scale, scale)      # (log2 next to a power of two)
        scale = torch.where((top <= 3.5 * scale) & (scale > 2.0 ** -125), scale / 2, scale)
        y = (b / scale).abs()
        step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0).double())
        out[..., d:d + BLOCK] = torch.copysign((torch.round(y / step) * step).clamp(max=6.0) * scale, b)
    return out


def _stands8(x):
    """What int8 codes of the rows stand for; the codes are defined by products of 32 bits."""
    x = x.float()
    top = x.abs().max(-1, keepdim=True).values
    top = torch.where(top == 0, torch.full_like(top, 127.0), top)
    v = x * (torch.full_like(top, 127.0) / top)
    return torch.trunc(v.double() + torch.copysign(torch.full_like(v, 0.5), v).double()) * (top.double() / 127.0)


def _exact_attention(q, k, v, q_lens, k_lens, window, sink):
    out, qa, ka = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0, 0
    group = q.shape[1] // k.shape[1]
    for ql, kl in zip(q_lens, k_lens):
        pos = torch.arange(kl - ql, kl, device="cuda")[:, None]
        key = torch.arange(kl, device="cuda")[None]
        hidden = key > pos
        if window:
            hidden |= (key <= pos - window) & (key >= sink)
        for h in range(q.shape[1]):
            kh, vh = k[ka:ka + kl, h // group].double(), v[ka:ka + kl, h // group].double()
            s = (q[qa:qa + ql, h].double() @ kh.T) / math.sqrt(q.shape[2])
            out[qa:qa + ql, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ vh
        qa, ka = qa + ql, ka + kl
    return out


def _exact_turn(case, x, at):
    """Rows as complex numbers, times e^(i angle)."""
    r, at = case["turn"], at.double()
    f = torch.tensor([case["base"] ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
    slow = f / case["factor"]
    if case["high"] > case["low"]:
        turns = case["original"] * f / (2 * math.pi)
        g = torch.clamp((turns - case["low"]) / (case["high"] - case["low"]), min=0.0, max=1.0)
        slow = torch.lerp(slow, f, g)
    by = torch.polar(torch.full_like(f, case["magnitude"]).expand(len(at), -1).contiguous(), at[:, None] * slow)
    out = x.double().clone()
    pair = out[..., :r].unflatten(-1, (-1, 2)) if case["pairs"] else out[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * by[:, None])
    out[..., :r] = (z if case["pairs"] else z.transpose(-1, -2)).flatten(-2)
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "rotary":
        n = case["rows"]
        x = _rand(seed, (n, case["heads"], case["dim"]), case["type"])
        at = _far(case, seed) if case["far"] else list(range(n))
        return _exact_turn(case, x, torch.tensor(at, device="cuda"))
    if kind == "sample":
        # whole numbers have no value in 64 bits other than their own
        x = _logits(case, seed).double()
        u = torch.rand(case["rows"], generator=torch.Generator(device="cuda").manual_seed(seed + 2), device="cuda")
        probs = torch.ones(case["rows"], dtype=torch.float64, device="cuda")
        for i, (hot, k, p, least) in enumerate(zip(*(t.tolist() for t in _settings(case, seed)))):
            if hot <= 0:
                continue
            w, _ = torch.sort(torch.softmax(x[i] / hot, 0), descending=True)
            w = w[:k] if k > 0 else w
            if p < 1:
                upto = torch.cumsum(w / w.sum(), 0)
                w = w[:int((upto < p).sum()) + 1]
            w = w[w >= least * w[0]]
            w = w / w.sum()
            probs[i] = w[torch.searchsorted(torch.cumsum(w, 0), u[i:i + 1].double(), right=True).clamp(max=len(w) - 1)]
        return dict(tokens=None, probs=probs)
    lens, new = _lens(case), _new_rows(case)
    k, v = _rows(case, seed)
    if kind == "decode":
        q = _rand(seed, (sum(new), case["heads"], case["dim"]), case["type"])
        return _exact_attention(q, _stands4(k.float()), _stands4(v.float()), new, lens, case["window"], case["sink"])
    out, last = {}, _last_rows(lens, new)
    k, v = k.double(), v.double()
    if kind == "turned":
        at = torch.tensor([p for n, c in zip(lens, new) for p in range(n - c, n)], device="cuda")
        q = _rand(seed, (sum(new), case["heads"], case["dim"]), case["type"])
        out["q"] = _exact_turn(case, q, at)
        k[last] = _exact_turn(case, k[last], at)
    cache = case.get("cache", "fp4")
    if cache != "bf16":     # rows are quantised as values of 32 bits
        stands = _stands4 if cache == "fp4" else _stands8
        return dict(out, k=stands(k.float()), v=stands(v.float()))
    ps = case["page"]
    table, _, pages = _place(case, lens, [n - c for n, c in zip(lens, new)])
    for name, x in (("k", k), ("v", v)):
        pool = torch.zeros((pages, case["kv"], ps, case["dim"]), dtype=torch.float64, device="cuda")
        for t, a, n in zip(table.tolist(), _starts(lens), lens):
            for j in range(-(-n // ps)):
                part = x[a + j * ps:a + min(n, (j + 1) * ps)]
                pool[t[j], :, :len(part)] = part.transpose(0, 1)
        out[name] = pool
    return out
