"""The attention operators over prompts and paged key-value caches, as cases.

  prompt  causal attention over whole prompts: packed sequences of different
          lengths, grouped heads, a cached prefix before the queries, a
          sliding window with sink tokens
  decode  attention of each sequence's newest rows (one, or a verify pass's
          few) over the pages of its cache
  pages   what a scheduler does with the pages: fork and grow (the shared
          last page is copied), copy, free, compact
  store   new key / value rows written into the pages, and rows read back

Head counts, head sizes, draft rows, sink rows and cached formats are those of
the repository's models (4 x 64, 12 x 64, 16 x 128; five verify rows; four
sinks; int8 codes with a scale per row) and of the same models with grouped
key / value heads.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GROW = 4            # appends that bring a sequence to its length, in turn with the others

_ctx = []


def _context():
    """One context per process, as the library's programs keep it."""
    if not _ctx:
        import pocketforge_amd as pf
        _ctx.append(pf.Context(0))
    return _ctx[0]


# ------------------------------------------------------------------ cases

def listed():
    return [
        # a short question to the smallest model: one call's latency
        dict(name="prompt_short", kind="prompt", type="bf16", heads=4, kv=4, dim=64, seqs=1, rows=19, prefix=0,
             window=0, sink=0),
        # requests of different lengths that arrive together, packed into one pass, grouped heads
        dict(name="prompt_packed", kind="prompt", type="bf16", heads=16, kv=4, dim=128, seqs=24, rows=700, prefix=0,
             window=0, sink=0),
        # one long document
        dict(name="prompt_long", kind="prompt", type="bf16", heads=16, kv=16, dim=128, seqs=1, rows=8192, prefix=0,
             window=0, sink=0),
        # fp32 rows, as the engine's passes hold them: new turns after a cached prefix, sinks and a window
        dict(name="prompt_f32_window", kind="prompt", type="f32", heads=12, kv=12, dim=64, seqs=3, rows=1100,
             prefix=333, window=1024, sink=4),
        # one user, a short context: a decode step's latency
        dict(name="decode_single", kind="decode", type="bf16", cache="bf16", heads=16, kv=16, dim=128, seqs=1,
             context=700, rows=1, page=64, window=0, sink=0),
        # a serving batch of ragged contexts, grouped heads
        dict(name="decode_batch", kind="decode", type="bf16", cache="bf16", heads=16, kv=4, dim=128, seqs=64,
             context=8000, rows=1, page=64, window=0, sink=0),
        # two long documents: the work has to be split over the context
        dict(name="decode_long", kind="decode", type="f16", cache="f16", heads=16, kv=2, dim=128, seqs=2,
             context=60000, rows=1, page=128, window=0, sink=0),
        # verify passes of four drafts: fp32 rows over int8 codes, every head with its own keys
        dict(name="verify_int8", kind="decode", type="f32", cache="i8", heads=16, kv=16, dim=128, seqs=16,
             context=2100, rows=5, page=64, window=0, sink=0),
        # eight answers sampled from one prompt: fork, and each answer's first token
        dict(name="fork_answers", kind="pages", do="fork", layers=12, kv=12, dim=64, context=1000, copies=8, page=64),
        # sequences copied, half of them ended, the rest moved together
        dict(name="copy_compact", kind="pages", do="compact", layers=24, kv=4, dim=128, context=1500, copies=12,
             page=64),
        # one decode step's rows of a batch: the step's bookkeeping and one layer's store
        dict(name="store_step", kind="store", type="bf16", cache="bf16", kv=4, dim=128, seqs=64, context=500, rows=1,
             page=64),
        # a prompt's fp32 rows into int8 pages, and read back for the next prompt pass
        dict(name="store_prompt_int8", kind="store", type="f32", cache="i8", kv=16, dim=128, seqs=3, context=64,
             rows=2000, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "decode", "decode", "decode", "pages", "store"])
    dim = rng.choice([64, 128, 128, 16 * rng.randint(2, 8)])
    kv, group = rng.choice([1, 2, 4, 8, 12, 16]), rng.choice([1, 1, 2, 4, 8])
    if kv * group > 64:
        group = 1
    if kind == "prompt":
        type = rng.choice(["bf16", "bf16", "f16", "f32"])
        c = dict(kind=kind, type=type, heads=kv * group, kv=kv, dim=dim, seqs=_log(rng, 1, 40),
                 rows=_log(rng, 1, 2500 if type == "f32" else 8000), prefix=rng.choice([0, 0, _log(rng, 1, 2000)]),
                 window=rng.choice([0, 0, 0, _log(rng, 16, 2000)]), sink=rng.choice([0, 4]))
        while work(c)["flops"] > (6e10 if type == "f32" else 2.5e11) or c["seqs"] * c["heads"] * c["rows"] * (c["rows"] + c["prefix"]) > 1.1e9:
            c["rows"] = max(1, c["rows"] * 3 // 4)
            c["seqs"] = max(1, c["seqs"] * 3 // 4)
        return c
    if kind == "decode":
        type, cache = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "i8"), ("bf16", "i8"),
                                  ("f16", "i8"), ("f32", "bf16")])
        c = dict(kind=kind, type=type, cache=cache, heads=kv * group, kv=kv, dim=dim, seqs=_log(rng, 1, 128),
                 context=_log(rng, 1, 60000), rows=rng.choice([1, 1, 1, 5, rng.randint(2, 8)]),
                 page=rng.choice([16, 32, 64, 64, 128]), window=rng.choice([0, 0, 0, _log(rng, 16, 4000)]),
                 sink=rng.choice([0, 4]))
        c["context"] = max(c["context"], c["rows"])
        while c["seqs"] * c["context"] * c["kv"] * c["dim"] > 2.6e8 or c["seqs"] * c["context"] * c["heads"] * c["rows"] > 1e8:
            c["context"] = max(c["rows"], c["context"] * 2 // 3)
            c["seqs"] = max(1, c["seqs"] * 2 // 3)
        return c
    if kind == "pages":
        c = dict(kind=kind, do=rng.choice(["fork", "compact"]), layers=rng.choice([2, 12, 24]), kv=kv, dim=dim,
                 context=2 * _log(rng, 1, 4000) + 1, copies=_log(rng, 2, 48), page=rng.choice([16, 32, 64, 128]))
        while c["layers"] * c["kv"] * c["dim"] * c["copies"] * c["context"] > 2.2e8:
            c["context"] = c["context"] // 3 | 1
            c["copies"] = max(2, c["copies"] * 2 // 3)
        return c
    c = dict(kind=kind, type=rng.choice(["f32", "f16", "bf16"]), cache=rng.choice(["i8", "bf16", "f16"]), kv=kv,
             dim=dim, seqs=_log(rng, 1, 128), context=_log(rng, 1, 2000), rows=rng.choice([1, 5, _log(rng, 1, 4000)]),
             page=rng.choice([16, 32, 64, 128]))
    while c["seqs"] * (c["rows"] + c["context"]) * c["kv"] * c["dim"] > 4e7:
        c["rows"], c["context"] = max(1, c["rows"] * 2 // 3), max(1, c["context"] * 2 // 3)
        c["seqs"] = max(1, c["seqs"] * 3 // 4)
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


def work(case):
    kind, dim, kv = case["kind"], case["dim"], case["kv"]
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
    if kind == "prompt":
        q = _ragged(case["seqs"], case["rows"])
        seen = [_visible(n, n + case["prefix"], case["window"], case["sink"]) for n in q]
        rows = 2 * case["heads"] * sum(q) + 2 * kv * sum(k for _, k in seen)
        return dict(bytes=rows * dim * size[case["type"]], flops=4.0 * dim * case["heads"] * sum(p for p, _ in seen))
    row = kv * (dim * size[case.get("cache", "bf16")] + (4 if case.get("cache") == "i8" else 0))
    if kind == "decode":
        k = _ragged(case["seqs"], case["context"], case["rows"])
        seen = [_visible(case["rows"], n, case["window"], case["sink"]) for n in k]
        q = 2 * case["heads"] * case["seqs"] * case["rows"] * dim * size[case["type"]]
        return dict(bytes=2 * row * sum(k for _, k in seen) + q,
                    flops=4.0 * dim * case["heads"] * sum(p for p, _ in seen))
    if kind == "pages":
        n, row = case["context"], 2 * row * case["layers"]
        if case["do"] == "fork":      # the shared page's rows once, and each copy's
            return dict(bytes=row * (n % case["page"]) * (1 + case["copies"]), flops=0.0)
        # the sequence's pages read once, each copy written, each moved page read and written
        pages = _pages_of(case) * (1 + case["copies"]) + 2 * len(_moves(case)[0])
        return dict(bytes=row * case["page"] * pages, flops=0.0)
    new = sum(_ragged(case["seqs"], case["rows"]))
    got = 2 * new * kv * dim * size[case["type"]]
    back = 0
    if case["cache"] == "i8":
        old = sum(_ragged(case["seqs"], case["context"]))
        back = 2 * row * (old + new) + 2 * (old + new) * kv * dim * 4
    return dict(bytes=got + 2 * row * new + back, flops=0.0)


# ------------------------------------------------------------ page numbers

def _pages_of(case):
    return -(-case["context"] // case["page"])


def _moves(case):
    """Pages that a compaction moves, (from, to), once every second of the
    copies behind the first sequence has ended: used pages from the number of
    used pages on, in order, to the free ones before it, in order."""
    m = _pages_of(case)
    pages = {m * (1 + i) + j for i in range(1, case["copies"], 2) for j in range(m)}
    used = m + len(pages)
    src = sorted(p for p in pages if p >= used)
    return src, [p for p in range(m, used) if p not in pages][:len(src)]


# ---------------------------------------------------------------- inputs

def _rand(seed, shape, type):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(TYPES[type])


def _codes(x):
    """The cache's int8 rows: codes round(x * (127 / max|x|)), scale max|x| / 127."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    full = torch.full_like(amax, 127.0)   # tensors: a division by or of a number may be a product
    one = torch.ones_like(amax)
    v = (x * torch.where(amax == 0, one, full / amax)).double()
    codes = torch.sign(v) * torch.floor(v.abs() + 0.5)
    return codes.to(torch.int8), torch.where(amax == 0, one, amax / full)


def _starts(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return at


def _rows(case, seed):
    """Key and value rows of every sequence, one after another; a row in sixteen stands out, as caches have them."""
    lens = _lens(case)
    shape = (sum(lens), case["kv"], case["dim"])
    k, v = _rand(seed + 1, shape, "f32"), _rand(seed + 2, shape, "f32")
    k[::16] *= 2.0
    v[::16] *= 4.0
    type = case["type"] if case["kind"] == "store" or case["cache"] == "i8" else case["cache"]
    return lens, k.to(TYPES[type]), v.to(TYPES[type])


def _lens(case):
    if case["kind"] == "decode":
        return _ragged(case["seqs"], case["context"], case["rows"])
    return [a + b for a, b in zip(_ragged(case["seqs"], case["context"]), _ragged(case["seqs"], case["rows"]))]


def _new_rows(case):
    return [case["rows"]] * case["seqs"] if case["kind"] == "decode" else _ragged(case["seqs"], case["rows"])


def _place(case, lens, seed):
    """For the plain form: a page table in shuffled order, and the place of each row."""
    ps, rng = case["page"], random.Random(seed)
    counts = [-(-n // ps) for n in lens]
    free = list(range(sum(counts)))
    rng.shuffle(free)
    most, table, place = max(counts), [], []
    for n, c in zip(lens, counts):
        pages = [free.pop() for _ in range(c)]
        table.append(pages + [0] * (most - c))
        place.append((torch.tensor(pages)[:, None] * ps + torch.arange(ps)).flatten()[:n])
    return torch.tensor(table, device="cuda"), torch.cat(place).cuda(), sum(counts)


def _cache(case, lens):
    import pocketforge_amd as pf
    kinds = {"i8": pf.TYPE_I8, "bf16": pf.TYPE_BF16, "f16": pf.TYPE_F16}
    ps = case["page"]
    return pf.PagedCache(_context(), n_layers=1, n_kv_heads=case["kv"], head_dim=case["dim"], page_size=ps,
                         n_pages=sum(-(-n // ps) for n in lens), max_seqs=len(lens), max_context=max(lens),
                         type=kinds[case["cache"]])


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


def prepare(case, seed):
    state = dict(case)
    kind = case["kind"]
    if kind == "prompt":
        q = _ragged(case["seqs"], case["rows"])
        k = [n + case["prefix"] for n in q]
        state.update(q_lens=q, k_lens=k, q=_rand(seed, (sum(q), case["heads"], case["dim"]), case["type"]),
                     k=_rand(seed + 1, (sum(k), case["kv"], case["dim"]), case["type"]),
                     v=_rand(seed + 2, (sum(k), case["kv"], case["dim"]), case["type"]))
        state["out"] = torch.zeros_like(state["q"])
        if own:
            state["ctx"] = _context()
        else:
            state["at"] = _padded_rows(q), _padded_rows(k)
    elif kind in ("decode", "store"):
        lens, k, v = _rows(case, seed)
        new = _new_rows(case)
        old = [n - c for n, c in zip(lens, new)]
        last = torch.cat([torch.arange(a + o, a + o + c) for a, o, c in zip(_starts(lens), old, new)]).cuda()
        state.update(lens=lens, old=old, new=new, seq_ids=list(range(len(lens))))
        if kind == "decode":
            state["q"] = _rand(seed, (sum(new), case["heads"], case["dim"]), case["type"])
            state["out"] = torch.zeros_like(state["q"])
        state["k"], state["v"] = k[last].contiguous(), v[last].contiguous()
        if own:
            cache = state["handle"] = _cache(case, lens)
            if kind == "store":
                # the rows from before; pages that no row has been written to hold zeros
                planes = cache.planes(0)
                torch.cuda.synchronize()
                for p in planes:
                    torch.as_tensor(p, device="cuda").zero_()
                torch.cuda.synchronize()
            _fill(cache, k, v, lens, old)
            torch.cuda.synchronize()
            cache.append(state["seq_ids"], new)
            if kind == "decode":
                cache.store(0, state["k"], state["v"])
            cache.ctx.synchronize()
            if kind == "store":
                if case["cache"] == "i8":
                    shape = (sum(lens), case["kv"], case["dim"])
                    state["back"] = [torch.zeros(shape, device="cuda") for _ in range(2)]
                else:
                    state["pool"] = [torch.as_tensor(p, device="cuda").view(TYPES[case["cache"]])
                                     for p in cache.planes(0)]
        else:
            ps = case["page"]
            if kind == "decode":
                state["table"], place, pages = _place(case, lens, seed)
            else:
                table, pages = _table(case, lens, old)
                state["table"] = torch.tensor([t + [0] * (max(map(len, table)) - len(t)) for t in table], device="cuda")
                place = torch.cat([(torch.tensor(t)[:, None] * ps + torch.arange(ps)).flatten()[:n]
                                   for t, n in zip(table, lens)]).cuda()
            state["place"], state["last"] = place, place[last]
            i8 = case["cache"] == "i8"
            state["pool"] = []
            for x in (k, v):
                x, scale = _codes(x) if i8 else (x.to(TYPES[case["cache"]]), None)
                pool = torch.zeros((pages, case["kv"], ps, case["dim"]), dtype=x.dtype, device="cuda")
                keep = torch.ones(len(x), dtype=torch.bool, device="cuda")
                if kind == "store":
                    keep[last] = False
                pool[place[keep] // ps, :, place[keep] % ps] = x[keep]
                state["pool"].append(pool)
                if i8:
                    s = torch.zeros((pages, case["kv"], ps, 1), device="cuda")
                    s[place[keep] // ps, :, place[keep] % ps] = scale[keep]
                    state["pool"].append(s)
            state["k_lens"] = torch.tensor(lens, device="cuda")
            state["q_pos"] = torch.tensor([list(range(n - c, n)) for n, c in zip(lens, new)], device="cuda") \
                if kind == "decode" else None
    else:
        m, n, ps = _pages_of(case), case["copies"], case["page"]
        total = m + n * (m if case["do"] == "compact" else 1)
        rows = [_rand(seed + s, (case["layers"], m, case["kv"], ps, case["dim"]), "bf16") for s in (1, 2)]
        state.update(total=total)
        if own:
            import pocketforge_amd as pf
            cache = state["handle"] = pf.PagedCache(
                _context(), n_layers=case["layers"], n_kv_heads=case["kv"], head_dim=case["dim"], page_size=ps,
                n_pages=total, max_seqs=1 + n, max_context=m * ps, type=pf.TYPE_BF16)
            cache.append([0], [case["context"]])
            cache.ctx.synchronize()
            state["pool"] = [torch.as_tensor(p, device="cuda").view(torch.bfloat16) for p in cache.planes()]
        else:
            state["pool"] = [torch.zeros((case["layers"], total, case["kv"], ps, case["dim"]), dtype=torch.bfloat16,
                                         device="cuda") for _ in range(2)]
        for pool, x in zip(state["pool"], rows):
            pool.zero_()
            pool[:, :m] = x
        if not own:
            state["moves"] = _moves(case) if case["do"] == "compact" else None
    torch.cuda.synchronize()
    return state


def _table(case, lens, old):
    """The pages that the cache gives the sequences, lowest first: by the growth of _fill, then by the last rows."""
    ps, table, at = case["page"], [[] for _ in lens], 0
    for r in range(GROW + 1):
        for i, n in enumerate(lens):
            have = old[i] * (r + 1) // GROW if r < GROW else n
            while len(table[i]) * ps < have:
                table[i].append(at)
                at += 1
    return table, at


def _padded_rows(lens):
    """[sequence, row] -> row of the packed tensor (the last sequence's rows repeat), and which of them are real."""
    r = torch.arange(max(lens))
    n = torch.tensor(lens)
    at = torch.tensor(_starts(lens)[:-1])
    return (at[:, None] + torch.minimum(r, n[:, None] - 1)).cuda(), (r < n[:, None]).cuda()


# ------------------------------------------------------------ plain forms

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


def _plain_prompt(s):
    (q_at, q_real), (k_at, _) = s["at"]
    k_lens = torch.tensor(s["k_lens"], device="cuda")
    first = k_lens - torch.tensor(s["q_lens"], device="cuda")
    q_pos = first[:, None] + torch.arange(q_at.shape[1], device="cuda")
    o = _attend(s["q"][q_at].float(), s["k"][k_at].float(), s["v"][k_at].float(), q_pos, k_lens, s["window"], s["sink"])
    return o[q_real].to(s["q"].dtype)


def _plain_decode(s):
    n, table = s["seqs"], s["table"]
    if s["cache"] == "i8":
        k, ks, v, vs = (p[table] for p in s["pool"])
        k, v = k.float() * ks, v.float() * vs
    else:
        k, v = (p[table].float() for p in s["pool"])
    k, v = (t.transpose(2, 3).reshape(n, -1, s["kv"], s["dim"]) for t in (k, v))
    # pages past a sequence's end hold other sequences' rows: their weight is zero
    q = s["q"].float().view(n, s["rows"], s["heads"], s["dim"])
    o = _attend(q, k, v, s["q_pos"], s["k_lens"], s["window"], s["sink"])
    return o.reshape(-1, s["heads"], s["dim"]).to(s["q"].dtype)


def _plain_pages(s):
    m, n, ps, ctx, pool = _pages_of(s), s["copies"], s["page"], s["context"], s["pool"]
    first = list(range(m))
    if s["do"] == "fork":
        # the full pages are shared, the last one's rows go to a page of each copy's own
        used = ctx % ps
        for p in pool:
            p[:, m:m + n, :, :used] = p[:, m - 1:m, :, :used]
        tables = [first] + [first[:-1] + [m + i] for i in range(n)]
        lens = [ctx] + [ctx + 1] * n
    else:
        src, dst = s["moves"]
        for p in pool:
            p[:, m:].unflatten(1, (n, m)).copy_(p[:, None, :m])
            p[:, dst] = p[:, src]
        page = dict(zip(src, dst))
        tables = [first] + [[page.get(p, p) for p in range(m * (1 + i), m * (2 + i))] if i % 2 else [] for i in range(n)]
        lens = [ctx] + [ctx if i % 2 else 0 for i in range(n)]
    return dict(k=pool[0], v=pool[1], tables=torch.tensor([t + [-1] * (m - len(t)) for t in tables]),
                lens=torch.tensor(lens))


def _plain_store(s):
    ps, to = s["page"], s["last"]
    if s["cache"] != "i8":
        for p, x in zip(s["pool"], (s["k"], s["v"])):
            p[to // ps, :, to % ps] = x.to(p.dtype)
        return dict(k=s["pool"][0], v=s["pool"][1])
    for i, x in enumerate((s["k"], s["v"])):
        codes, scale = _codes(x)
        s["pool"][2 * i][to // ps, :, to % ps] = codes
        s["pool"][2 * i + 1][to // ps, :, to % ps] = scale
    at = s["place"]
    k, ks, v, vs = (p[at // ps, :, at % ps] for p in s["pool"])
    return dict(k=k.float() * ks, v=v.float() * vs)


def run(s):
    kind = s["kind"]
    if not own:
        return {"prompt": _plain_prompt, "decode": _plain_decode, "pages": _plain_pages, "store": _plain_store}[kind](s)
    if kind == "prompt":
        return s["ctx"].prompt_attention(s["q"], s["k"], s["v"], s["q_lens"], s["k_lens"], causal=True,
                                         window=s["window"], sink=s["sink"], out=s["out"])
    cache = s["handle"]
    if kind == "decode":
        return cache.attention(0, s["q"], causal=True, window=s["window"], sink=s["sink"], out=s["out"])
    if kind == "store":
        cache.truncate(s["seq_ids"], s["old"])
        cache.append(s["seq_ids"], s["new"])
        cache.store(0, s["k"], s["v"])
        if s["cache"] == "i8":
            k, v = cache.gather(0, s["seq_ids"], out=s["back"])
            return dict(k=k, v=v)
        return dict(k=s["pool"][0], v=s["pool"][1])
    n = s["copies"]
    children = list(range(1, n + 1))
    cache.free(children)
    if s["do"] == "fork":
        cache.fork(0, children)
        cache.append(children, [1] * n)
    else:
        cache.copy([0] * n, children)
        cache.free(children[::2])
        cache.compact()
    tables, lens = cache.tables([0] + children)
    return dict(k=s["pool"][0], v=s["pool"][1], tables=tables, lens=lens)


# ----------------------------------------------------- values in 64 bits

def _exact_attention(q, k, v, q_lens, k_lens, window, sink):
    out, qa, ka = torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0, 0
    group = q.shape[1] // k.shape[1]
    for ql, kl in zip(q_lens, k_lens):
        for h in range(q.shape[1]):
            kh, vh = k[ka:ka + kl, h // group].double(), v[ka:ka + kl, h // group].double()
            for r in range(0, ql, 2048):
                rows = torch.arange(r, min(ql, r + 2048), device="cuda")
                s = (q[qa + rows, h].double() @ kh.T) / math.sqrt(q.shape[2])
                pos = (rows + kl - ql)[:, None]
                key = torch.arange(kl, device="cuda")[None]
                hidden = key > pos
                if window:
                    hidden |= (key <= pos - window) & (key >= sink)
                w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                out[qa + rows, h] = w @ vh
        qa, ka = qa + ql, ka + kl
    return out


def _held(x):
    """What int8 codes of the rows stand for; the codes are defined by products of 32 bits."""
    x = x.float()
    top = x.abs().max(-1, keepdim=True).values
    top = torch.where(top == 0, torch.full_like(top, 127.0), top)
    v = x * (torch.full_like(top, 127.0) / top)
    return torch.trunc(v.double() + torch.copysign(torch.full_like(v, 0.5), v).double()) * (top.double() / 127.0)


def exact(case, seed):
    kind = case["kind"]
    if kind == "prompt":
        q = _ragged(case["seqs"], case["rows"])
        k = [n + case["prefix"] for n in q]
        shapes = [(sum(q), case["heads"], case["dim"])] + 2 * [(sum(k), case["kv"], case["dim"])]
        x = [_rand(seed + i, s, case["type"]) for i, s in enumerate(shapes)]
        return _exact_attention(*x, q, k, case["window"], case["sink"])
    if kind in ("decode", "store"):
        lens, k, v = _rows(case, seed)
        if case["cache"] == "i8":
            k, v = _held(k), _held(v)
        if kind == "decode":
            new = _new_rows(case)
            q = _rand(seed, (sum(new), case["heads"], case["dim"]), case["type"])
            return _exact_attention(q, k, v, new, lens, case["window"], case["sink"])
        if case["cache"] == "i8":
            return dict(k=k, v=v)
        ps = case["page"]
        table, pages = _table(case, lens, [n - c for n, c in zip(lens, _new_rows(case))])
        out = {}
        for name, x in (("k", k), ("v", v)):
            pool = torch.zeros((pages, case["kv"], ps, case["dim"]), dtype=torch.float64, device="cuda")
            for t, a, n in zip(table, _starts(lens), lens):
                for j, p in enumerate(t):
                    part = x[a + j * ps:a + min(n, (j + 1) * ps)].double()
                    pool[p, :, :len(part)] = part.transpose(0, 1)
            out[name] = pool
        return out
    m, n, ps, ctx = _pages_of(case), case["copies"], case["page"], case["context"]
    out = {}
    for name, s in (("k", 1), ("v", 2)):
        base = _rand(seed + s, (case["layers"], m, case["kv"], ps, case["dim"]), "bf16").double()
        each = m if case["do"] == "compact" else 1
        pool = torch.zeros((case["layers"], m + n * each) + base.shape[2:], dtype=torch.float64, device="cuda")
        pool[:, :m] = base
        if case["do"] == "fork":
            tail = ctx - (m - 1) * ps
            for i in range(n):
                pool[:, m + i, :, :tail] = base[:, -1, :, :tail]
        else:
            for i in range(n):
                pool[:, m * (1 + i):m * (2 + i)] = base
            owner = {m * (1 + i) + j for i in range(1, n, 2) for j in range(m)}
            holes = [p for p in range(m, m + len(owner)) if p not in owner]
            for p, h in zip(sorted(p for p in owner if p >= m + len(owner)), holes):
                pool[:, h] = pool[:, p]
        out[name] = pool
    # whole numbers have no value in 64 bits other than their own
    return dict(out, tables=None, lens=None)
