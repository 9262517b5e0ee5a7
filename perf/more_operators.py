"""The operators around a paged key/value cache with grouped-query attention (GQA) whose speed is measured, over the range of
shapes and types they serve.

Kinds of work (``case["kind"]``):

* ``append``   what a layer does with the projections of new tokens: RMSNorm of each head's query and key, their rotation (the
               whole head or a part of it), keys and values written to the paged cache
* ``decode``   attention of single query tokens over the paged cache
* ``chunk``    attention of each sequence's newest tokens (a prompt, its next chunk, drafted tokens) over the paged cache
* ``fork``     sequences that go on from another's tokens: they share its full pages, the last one is copied, in all layers
* ``compact``  the pages in use moved to the front of the pools of all layers, and the block tables rewritten

Attention sees the tokens up to the query's own or, with a window, the newest ``window`` of them and the first ``sinks``.
``run`` computes a pass in plain torch operations, or, where ``own`` is true, through vib3_amd.gqa and vib3_amd.pages.
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6


# ------------------------------------------------------------------------------- the cases

# the attention of a Mixtral-shaped layer (hidden 4096), and others
_MIXTRAL = dict(heads=32, kv_heads=8, dim=128)
_SMALL = dict(heads=64, kv_heads=8, dim=64)
_WIDE = dict(heads=16, kv_heads=2, dim=256)


def listed():
    return [
        # one decode step of one conversation: a single token, the call's fixed cost
        dict(name="append_token", kind="append", **_MIXTRAL, dt="bf16", src="bf16", page=64, rot=128, norm=False, halves=True,
             seqs=1, tokens=1, start=4000, pad=0),
        # prompts of several conversations taken in at once, padded: norms, a rotation of part of the head, f32 projections
        dict(name="append_prompts", kind="append", heads=40, kv_heads=8, dim=128, dt="f16", src="f32", page=16, rot=64, norm=True,
             halves=False, seqs=5, tokens=6007, start=70000, pad=9),
        # the next token of one conversation of ordinary length: latency
        dict(name="decode_one", kind="decode", **_MIXTRAL, dt="bf16", page=64, seqs=1, shortest=901, longest=901, window=0, sinks=0),
        # a serving batch of short conversations and long documents
        dict(name="decode_batch", kind="decode", **_MIXTRAL, dt="bf16", page=64, seqs=61, shortest=300, longest=50000, window=0,
             sinks=0),
        # a layer with a sliding window, old and new conversations, f16, small pages
        dict(name="decode_window", kind="decode", **_SMALL, dt="f16", page=16, seqs=97, shortest=1, longest=30000, window=4096,
             sinks=4),
        # drafted tokens to check: four queries a sequence
        dict(name="chunk_draft", kind="chunk", **_WIDE, dt="bf16", page=48, q=",".join(["4"] * 16),
             k=",".join(str(317 + 355 * i) for i in range(16)), window=0, sinks=0),
        # one long prompt
        dict(name="chunk_prompt", kind="chunk", **_MIXTRAL, dt="bf16", page=64, q="12288", k="12288", window=0, sinks=0),
        # a layer with a sliding window: next chunks of long documents beside single tokens, f16, small pages
        dict(name="chunk_window", kind="chunk", **_SMALL, dt="f16", page=16, q="2048,1,611,1,37,1500", k="20000,4500,8611,17,937,1500",
             window=4096, sinks=4),
        # one prompt, four answers to it, one layer
        dict(name="fork_one", kind="fork", **_MIXTRAL, dt="bf16", page=64, layers=1, parents=1, children=4, shortest=777, longest=777),
        # several prompts with many answers each, all layers at once
        dict(name="fork_samples", kind="fork", **_MIXTRAL, dt="bf16", page=64, layers=8, parents=3, children=32, shortest=200,
             longest=700),
        # a small pool after one of its conversations ended
        dict(name="compact_small", kind="compact", **_SMALL, dt="f16", page=16, layers=1, pages=64, seqs=6, live=40),
        # a pool half empty, made smaller: half of what is live has to move
        dict(name="compact_pool", kind="compact", **_MIXTRAL, dt="bf16", page=64, layers=4, pages=407, seqs=37, live=207),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dims = dict(rng.choice([_MIXTRAL, _MIXTRAL, _SMALL, _WIDE]))
    if rng.random() < 0.5:
        dims["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
        dims["heads"] = dims["kv_heads"] * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
    dims["dt"], dims["page"] = rng.choice(["bf16", "f16"]), rng.choice([16, 32, 48, 64, 128])
    kind = rng.choice(["append", "decode", "decode", "chunk", "chunk", "fork", "compact"])
    if kind == "append":
        seqs = _log(rng, 1, 128)
        rot = rng.choice([dims["dim"], dims["dim"], dims["dim"] // 2, dims["dim"] // 4])
        return dict(kind=kind, **dims, src=rng.choice([dims["dt"], dims["dt"], "f32"]), rot=rot, norm=rng.random() < 0.5,
                    halves=rng.random() < 0.5, seqs=seqs, tokens=max(seqs, _log(rng, 1, 5000)),
                    start=rng.choice([0, _log(rng, 1, 130000)]), pad=rng.choice([0, rng.randint(1, 16)]))
    window, sinks = rng.choice([(0, 0), (0, 0), (_log(rng, 64, 8192), 0), (_log(rng, 64, 8192), rng.randint(1, 16))])
    if kind == "decode":
        while True:
            longest = _log(rng, 1, 130000)
            case = dict(kind=kind, **dims, seqs=_log(rng, 1, 128), shortest=_log(rng, 1, longest), longest=longest, window=window,
                        sinks=sinks)
            if case["seqs"] * longest < 2000000 and work(case)["bytes"] < 2e9:
                return case
    if kind == "chunk":
        while True:
            n = _log(rng, 1, 16)
            most = _log(rng, 1, 8000)
            q = [_log(rng, 1, most) for _ in range(n)]
            k = [a + rng.choice([0, 0, _log(rng, 1, 20000)]) for a in q]
            case = dict(kind=kind, **dims, q=",".join(map(str, q)), k=",".join(map(str, k)), window=window, sinks=sinks)
            if sum(a * b for a, b in zip(q, k)) * dims["heads"] * dims["dim"] < 2.5e11 and work(case)["bytes"] < 1e9:
                return case
    layers = _log(rng, 1, 8)
    if kind == "fork":
        parents = _log(rng, 1, 4)
        longest = _log(rng, 1, 1500)
        return dict(kind=kind, **dims, layers=layers, parents=parents, children=max(parents, _log(rng, 1, 32)),
                    shortest=_log(rng, 1, longest), longest=longest)
    while True:
        pages = _log(rng, 4, 2000)
        live = rng.randint(1, pages)
        case = dict(kind=kind, **dims, layers=layers, pages=pages, seqs=min(live, _log(rng, 1, 64)), live=live)
        if pages * _page_bytes(case) * layers < 4.2e8:
            return case


def _page_bytes(case):
    """Bytes of a page of one layer: its keys and values."""
    return 4 * case["page"] * case["kv_heads"] * case["dim"]


def _spread(n, lo, hi):
    """n lengths, spread evenly over the logarithm, in a mixed order."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    out = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    return [out[i * step % n] for i in range(n)]


def _counts(case):
    """New tokens of each sequence of an append."""
    n, t = case["seqs"], case["tokens"]
    return [t // n + (i < t % n) for i in range(n)]


def _spans(case):
    """New tokens and cached tokens (these among them) of each sequence."""
    if case["kind"] == "decode":
        k = _spread(case["seqs"], case["shortest"], case["longest"])
        return [1] * len(k), k
    return [[int(a) for a in case[n].split(",")] for n in ("q", "k")]


# ------------------------------------------------------------------------------- what a program holds before the call


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(lengths):
    return _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def _pages(g, needed, max_pages):
    """Block table [len(needed)][max_pages] whose entries needed[i] (a list of page indices) are pages of a pool in a random
    order; the other entries are never used. Returns the table and the number of pages in the pool."""
    total = sum(len(n) for n in needed)
    ids = torch.randperm(total + 3, generator=g, device=DEV)[:total].tolist()
    table = torch.full((len(needed), max_pages), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(needed):
        table[i, n] = torch.tensor(ids[at:at + len(n)], dtype=torch.int32)
        at += len(n)
    return table.to(DEV), total + 3


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, ps = _DT[case["dt"]], case["page"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    def cache(pages):
        return normal(pages, ps, kv_heads, dim), normal(pages, ps, kv_heads, dim)

    st = dict(case=case, scale=dim ** -0.5)
    if case["kind"] == "append":
        counts = _counts(case)
        starts = [case["start"] * (i + 1) // len(counts) for i in range(len(counts))]
        used = [list(range(s // ps, (s + n - 1) // ps + 1)) for s, n in zip(starts, counts)]
        st["table"], pages = _pages(g, used, max(u[-1] for u in used) + 1)
        st["keys"], st["values"] = cache(pages)
        st["seqs"] = _ints([i for i, n in enumerate(counts) for _ in range(n)] + [-1] * case["pad"])
        st["positions"] = _ints([s + j for s, n in zip(starts, counts) for j in range(n)] + [0] * case["pad"])
        rows = case["tokens"] + case["pad"]
        qkv = normal(rows, heads + 2 * kv_heads, dim, scale=1.5, dtype=_DT[case["src"]])  # one projection's output
        st["q"], st["k"], st["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        st["inv_freq"] = (1e6 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])).float()
        st["q_norm"] = st["k_norm"] = None
        if case["norm"]:
            st["q_norm"], st["k_norm"] = (1.0 + normal(dim, scale=0.2, dtype=torch.float32) for _ in range(2))
        st["q_out"] = torch.zeros(rows, heads, dim, dtype=dt, device=DEV)
        if own:
            from vib3_amd import gqa
            st["cache"] = gqa.GqaCache(st["keys"], st["values"])
    elif case["kind"] in ("decode", "chunk"):
        nq, nk = _spans(case)
        used = [list(range((n + ps - 1) // ps)) for n in nk]
        st["table"], pages = _pages(g, used, max(len(u) for u in used))
        st["keys"], st["values"] = cache(pages)
        st["lens"], st["q"] = _ints(nk), normal(sum(nq), heads, dim, scale=2.0)
        if case["kind"] == "chunk":
            st["cu_q"] = _offsets(nq)
        if own:
            from vib3_amd import gqa
            c = gqa.GqaCache(st["keys"], st["values"])
            st["op"] = gqa.GqaDecode(c, heads, max_rows=len(nq)) if case["kind"] == "decode" else \
                gqa.GqaChunk(c, heads, max_tokens=sum(nq), max_seqs=len(nq))
    elif case["kind"] == "fork":
        # the parents' rows of the table come first, the children's (of earlier use) behind them
        np_, nc = case["parents"], case["children"]
        lens = _spread(np_, case["shortest"], case["longest"])
        width = max(lens) // ps + 2
        need = [(n + ps - 1) // ps for n in lens]
        pages = sum(need) + nc + 3
        ids = torch.randperm(pages, generator=g, device=DEV).tolist()
        table = torch.full((np_ + nc, width), -1, dtype=torch.int32)
        for i, n in enumerate(need):
            table[i, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
        table[np_:, 0] = 0
        st["table"], st["lens"] = table.to(DEV), _ints(lens + [0] * nc)
        st["parents"], st["children"] = _ints([i % np_ for i in range(nc)]), _ints([np_ + i for i in range(nc)])
        st["new_pages"] = _ints([ids.pop() for _ in range(nc)])
        st["pools"] = [cache(pages) for _ in range(case["layers"])]
    else:
        # live pages of sequences of mixed lengths, anywhere in the pool; the last sequence shares the first one's first page,
        # and every row holds, behind its tokens' pages, one that it no longer uses
        n, pages, live = case["seqs"], case["pages"], case["live"]
        ids = torch.randperm(pages, generator=g, device=DEV).tolist()
        weight = _spread(n, 1, 8)
        count = [1 + (live - n) * w // sum(weight) for w in weight]
        count[0] += live - sum(count)
        table = torch.full((n, max(count) + 2), -1, dtype=torch.int32)
        at = 0
        for i, c in enumerate(count):
            table[i, :c] = torch.tensor(ids[at:at + c], dtype=torch.int32)
            table[i, c] = ids[(at * 7 + i) % pages]
            at += c
        if n > 1:
            table[n - 1, 0] = table[0, 0]
        st["table"] = table.to(DEV)
        st["lens"] = _ints([c * ps - (5 * i) % ps for i, c in enumerate(count)])
        st["out_table"] = torch.empty_like(st["table"])
        st["pools"] = [cache(pages) for _ in range(case["layers"])]
    if own and case["kind"] in ("fork", "compact"):
        from vib3_amd import gqa, pages
        st["caches"] = [gqa.GqaCache(k, v) for k, v in st["pools"]]
        if case["kind"] == "compact":
            st["op"] = pages.PageCompaction(st["caches"])
    return st


# ------------------------------------------------------------------------------- one pass


def run(st):
    return {"append": _append, "decode": _decode, "chunk": _chunk, "fork": _fork, "compact": _compact}[st["case"]["kind"]](st)


def _append(st):
    case = st["case"]
    if own:
        from vib3_amd import gqa
        gqa.gqa_append(st["cache"], st["table"], st["seqs"], st["positions"], st["q"], st["k"], st["v"], st["inv_freq"], st["q_out"],
                       q_norm=st["q_norm"], k_norm=st["k_norm"], eps=_EPS, interleaved=not case["halves"])
        return st["keys"], st["values"], st["q_out"]
    n, rot, halves = case["tokens"], case["rot"], case["halves"]  # the rows behind are padding
    dt = st["keys"].dtype
    seqs, pos = st["seqs"][:n].long(), st["positions"][:n].long()
    angle = (pos.double()[:, None] * st["inv_freq"].double())[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turned(x, weight):
        x = x[:n].float()
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight
        r = x[..., :rot]
        a, b = r.chunk(2, -1) if halves else (r[..., 0::2], r[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([r, x[..., rot:]], -1).to(dt)

    page, row = st["table"][seqs, pos // case["page"]].long(), pos % case["page"]
    st["keys"][page, row] = turned(st["k"], st["k_norm"])
    st["values"][page, row] = st["v"][:n].to(dt)
    st["q_out"][:n] = turned(st["q"], st["q_norm"])
    return st["keys"], st["values"], st["q_out"]


def _decode(st):
    case = st["case"]
    if own:
        return st["op"].launch(st["q"], st["table"], st["lens"], st["scale"], window=case["window"], sinks=case["sinks"])
    return _attention(st)


def _chunk(st):
    case = st["case"]
    if own:
        return st["op"].launch(st["q"], st["table"], st["cu_q"], st["lens"], st["scale"], window=case["window"], sinks=case["sinks"])
    return _attention(st)


def _attention(st):
    case = st["case"]
    ps, window, group = case["page"], case["window"], case["heads"] // case["kv_heads"]
    out = torch.empty_like(st["q"])
    q0 = 0
    for i, (nq, nk) in enumerate(zip(*_spans(case))):
        used = st["table"][i, :(nk + ps - 1) // ps].long()
        for h in range(case["kv_heads"]):
            k, v = (st[n][used, :, h].flatten(0, 1)[:nk].float() for n in ("keys", "values"))
            step = max(1, 2 ** 28 // (nk * group))  # queries at a time: their scores fill a GB
            for a in range(0, nq, step):
                b = min(nq, a + step)
                # these queries' keys: from the first one's window on, and the first tokens
                first = max(0, nk - nq + a - window + 1) if window else 0
                j = torch.arange(first, nk - nq + b, device=DEV)
                if window and first > 0:
                    j = torch.cat([torch.arange(min(first, case["sinks"]), device=DEV), j])
                at = torch.arange(nk - nq + a, nk - nq + b, device=DEV)[:, None]
                hidden = j > at
                if window:
                    hidden |= (j <= at - window) & (j >= case["sinks"])
                q = st["q"][q0 + a:q0 + b, h * group:(h + 1) * group].float()
                s = (q.flatten(0, 1) @ k[j].t()).view(b - a, group, -1).mul_(st["scale"]).masked_fill_(hidden[:, None], -math.inf)
                p = s.sub_(s.amax(-1, keepdim=True)).exp_()
                o = (p.flatten(0, 1) @ v[j]).view(b - a, group, -1) / p.sum(-1, keepdim=True)
                out[q0 + a:q0 + b, h * group:(h + 1) * group] = o.to(out.dtype)
        q0 += nq
    return out


def _fork(st):
    case, table = st["case"], st["table"]
    if own:
        from vib3_amd import pages
        pages.fork_pages(st["caches"], table, st["lens"], st["parents"], st["children"], st["new_pages"])
        return [table] + [t for kv in st["pools"] for t in kv]
    ps, parents, children = case["page"], st["parents"].long(), st["children"].long()
    lens = st["lens"][parents].long()
    full = lens // ps
    column = torch.arange(table.shape[1], device=DEV)
    rows = torch.where(column < full[:, None], table[parents], torch.full_like(table[parents], -1))
    rows.scatter_(1, full[:, None], st["new_pages"][:, None])
    table[children] = rows
    src = table[parents, full].long()
    i, j = (torch.arange(ps, device=DEV) < (lens % ps)[:, None]).nonzero(as_tuple=True)  # the tokens to copy
    for kv in st["pools"]:
        for t in kv:
            t[st["new_pages"].long()[i], j] = t[src[i], j]
    return [table] + [t for kv in st["pools"] for t in kv]


def _compact(st):
    case, table = st["case"], st["table"]
    if own:
        live = st["op"].launch(table, st["lens"], out_table=st["out_table"])
        return [live, st["out_table"]] + [t for kv in st["pools"] for t in kv]
    pages, ps = case["pages"], case["page"]
    used = torch.arange(table.shape[1], device=DEV) < ((st["lens"] + ps - 1) // ps)[:, None]
    mark = torch.zeros(pages, dtype=torch.bool, device=DEV)
    mark[table[used].long()] = True
    live = mark.sum()
    at = torch.arange(pages, device=DEV)
    src = (mark & (at >= live)).nonzero()[:, 0]
    dst = (~mark & (at < live)).nonzero()[:, 0]
    for kv in st["pools"]:
        for t in kv:
            t[dst] = t[src]
    place = at.clone()
    place[src] = dst
    st["out_table"].copy_(torch.where(used, place[table.clamp_min(0).long()], torch.full_like(place[:1], -1)))
    return [live[None].int(), st["out_table"]] + [t for kv in st["pools"] for t in kv]


# ------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    ps, heads, kv_heads = case["page"], case["heads"], case["kv_heads"]
    if case["kind"] == "append":
        keys, values, q_out = (st[n].double() for n in ("keys", "values", "q_out"))
        live = (st["seqs"] >= 0).nonzero()[:, 0]
        pos, rot = st["positions"][live], case["rot"]
        half = rot // 2
        turn = torch.polar(torch.ones(len(live), half, device=DEV, dtype=torch.float64),
                           torch.outer(pos.double(), st["inv_freq"].double()))[:, None]
        i = torch.arange(half, device=DEV)
        first, second = (i, i + half) if case["halves"] else (2 * i, 2 * i + 1)

        def turned(x, weight):  # a pair as a complex number times e^(i angle)
            x = x[live].double()
            if weight is not None:
                x = x / (x.square().sum(-1, keepdim=True) / case["dim"] + _EPS).sqrt() * weight.double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            out = x.clone()
            out[..., first], out[..., second] = z.real, z.imag
            return out

        at = st["table"][st["seqs"][live].long(), pos.long() // ps].long() * ps + pos.long() % ps
        keys.flatten(0, 1)[at] = turned(st["k"], st["k_norm"])
        values.flatten(0, 1)[at] = st["v"][live].double()
        q_out[live] = turned(st["q"], st["q_norm"])
        return keys, values, q_out
    if case["kind"] in ("decode", "chunk"):
        out = torch.zeros(st["q"].shape, device=DEV, dtype=torch.float64)
        group, end = heads // kv_heads, 0
        window = case["window"] or 1 << 30
        for i, (nq, nk) in enumerate(zip(*_spans(case))):
            end += nq
            j = torch.arange(nk, device=DEV)
            slot = st["table"][i].long()[j // ps] * ps + j % ps
            for h in range(heads):
                k, v = (st[n].flatten(0, 1)[:, h // group][slot].double() for n in ("keys", "values"))
                k = k.t().contiguous()
                for a in range(0, nq, 2048):  # positions nk - nq + a and on
                    b = min(nq, a + 2048)
                    p = torch.arange(nk - nq + a, nk - nq + b, device=DEV)[:, None]
                    x = st["q"][end - nq + a:end - nq + b, h].double() @ k * st["scale"]
                    x[~((j <= p) & ((p - j < window) | (j < case["sinks"])))] = -math.inf
                    out[end - nq + a:end - nq + b, h] = torch.softmax(x, -1) @ v
        return out
    table, lens = st["table"].tolist(), st["lens"].tolist()
    pools = [t for kv in st["pools"] for t in kv]
    if case["kind"] == "fork":
        before = [row[:] for row in table]
        for p, c, new in zip(st["parents"].tolist(), st["children"].tolist(), st["new_pages"].tolist()):
            full, rest = divmod(lens[p], ps)
            table[c] = before[p][:full] + [new] + [-1] * (len(table[c]) - full - 1)
            for t in pools if rest else []:
                t[new, :rest] = t[before[p][full], :rest].clone()
        return [_ints(table)] + [t.double() for t in pools]
    held = [row[:-(-n // ps)] for row, n in zip(table, lens)]
    live = sorted({p for row in held for p in row})
    holes = sorted(set(range(len(live))) - set(live))
    to = dict(zip([p for p in live if p >= len(live)], holes))
    for t in pools:
        for a, b in to.items():
            t[b] = t[a]
    width = len(table[0])
    return [_ints([len(live)]), _ints([[to.get(p, p) for p in row] + [-1] * (width - len(row)) for row in held])] + \
        [t.double() for t in pools]


# ------------------------------------------------------------------------------- what a pass cannot do without


def _visible(p, window, sinks):
    """Tokens that a query at position p sees."""
    if not window or p < window:
        return p + 1
    return window + min(sinks, p - window + 1)


def work(case):
    heads, kv_heads, dim, ps = (case[n] for n in ("heads", "kv_heads", "dim", "page"))
    if case["kind"] == "append":
        n, size = case["tokens"], 4 if case["src"] == "f32" else 2
        turned = n * (heads + kv_heads)
        # the projections read, the queries and the cached rows written
        return {"bytes": n * (heads + 2 * kv_heads) * dim * (size + 2) + n * 12,
                "flops": turned * (3 * case["rot"] + (4 * dim if case["norm"] else 0))}
    if case["kind"] in ("decode", "chunk"):
        window, sinks = case["window"], case["sinks"]
        seen = read = 0
        for nq, nk in zip(*_spans(case)):
            seen += sum(_visible(p, window, sinks) for p in range(nk - nq, nk))
            first = max(0, nk - nq - window + 1) if window else 0  # the oldest token that a query's window reaches
            read += nk - first + min(first, sinks)
        return {"bytes": read * kv_heads * dim * 4 + sum(_spans(case)[0]) * heads * dim * 4, "flops": 4 * seen * heads * dim}
    if case["kind"] == "fork":
        lens = _spread(case["parents"], case["shortest"], case["longest"])
        of = [lens[i % len(lens)] for i in range(case["children"])]
        entries = sum(n // ps for n in of)
        return {"bytes": 2 * sum(n % ps for n in of) * _page_bytes(case) // ps * case["layers"] + 8 * entries, "flops": 0}
    # on average a page lies behind the live ones with the share of the free ones
    moved = case["live"] * (case["pages"] - case["live"]) // case["pages"]
    return {"bytes": 2 * moved * _page_bytes(case) * case["layers"] + 8 * case["live"], "flops": 0}
