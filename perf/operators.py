"""The latent-attention (MLA) operators whose speed is measured, over the range of shapes and types they serve.

Kinds of work (``case["kind"]``):

* ``append``   what a layer does with the projections of new tokens: RMSNorm of the latent, rotation of the shared
               key, both written to the paged latent cache, and the rotation of the queries' rotary part
* ``decode``   attention of single query tokens over the paged latent cache, absorbed form: the queries go into the
               latent space by W_uk, the result comes back by W_uv
* ``prefill``  causal attention of whole prompts (or the next chunk of them), expanded form: a key and a value a head

``run`` computes a pass in plain torch operations, or, where ``own`` is true, through vib3_amd.mla.
"""
import math

import torch

own = False

DEV = "cuda"
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6


# ------------------------------------------------------------------------------- the cases

# the widths of Kimi-K2.5's attention (a latent of 512 and a shared rotary key of 64 a token), and a small model's
_WIDE = dict(rank=512, rope=64, nope=128, v=128)
_NARROW = dict(rank=256, rope=32, nope=64, v=64)


def listed():
    return [
        # one decode step of one conversation: a single token, the call's fixed cost
        dict(name="append_token", kind="append", **_WIDE, heads=64, dt="bf16", kv="bf16", page=64, halves=False,
             seqs=1, tokens=1, start=4000, pad=0),
        # one decode step of a padded batch, f16 cache, f32 projections, half-split rotation
        dict(name="append_batch", kind="append", **_WIDE, heads=64, dt="f16", kv="f32", page=16, halves=True,
             seqs=57, tokens=57, start=90000, pad=7),
        # three prompts taken in at once
        dict(name="append_prompts", kind="append", **_WIDE, heads=64, dt="bf16", kv="bf16", page=64, halves=False,
             seqs=3, tokens=6201, start=0, pad=0),
        # the next token of one conversation of ordinary length: latency
        dict(name="decode_one", kind="decode", **_WIDE, heads=64, dt="bf16", page=64, seqs=1, new=1, shortest=777,
             longest=777),
        # the next token over a long document: one row, all of the card on it
        dict(name="decode_one_long", kind="decode", **_WIDE, heads=64, dt="bf16", page=64, seqs=1, new=1,
             shortest=131072, longest=131072),
        # a batch of new and old conversations, f16, small pages
        dict(name="decode_ragged", kind="decode", **_WIDE, heads=64, dt="f16", page=16, seqs=41, new=1, shortest=1,
             longest=4100),
        # a full serving batch
        dict(name="decode_batch", kind="decode", **_WIDE, heads=64, dt="bf16", page=64, seqs=96, new=1, shortest=2048,
             longest=12288),
        # a small model with a head count that is no power of two, three drafted tokens a sequence to check
        dict(name="decode_draft", kind="decode", **_NARROW, heads=40, dt="bf16", page=48, seqs=16, new=3, shortest=300,
             longest=5000),
        # one short prompt
        dict(name="prefill_short", kind="prefill", **_WIDE, heads=64, dt="bf16", q="173", k="173"),
        # prompts of several conversations at once, some of them the next chunk after earlier tokens
        dict(name="prefill_ragged", kind="prefill", **_WIDE, heads=64, dt="f16", q="1500,37,1,2048,611",
             k="1500,937,4000,2048,2611"),
        # one long document
        dict(name="prefill_long", kind="prefill", **_WIDE, heads=64, dt="bf16", q="12288", k="12288"),
        # a small model's prompts
        dict(name="prefill_narrow", kind="prefill", **_NARROW, heads=40, dt="bf16", q="1000,2300,515",
             k="1000,2300,515"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dims = rng.choice([_WIDE, _WIDE, _NARROW])
    heads = rng.choice([64, 64, 128, 40, 16, 8, rng.randint(1, 128)])
    dt = rng.choice(["bf16", "f16"])
    kind = rng.choice(["append", "decode", "decode", "prefill"])
    page = rng.choice([16, 32, 48, 64, 128])
    if kind == "append":
        seqs = _log(rng, 1, 128)
        return dict(kind=kind, **dims, heads=min(heads, 64), dt=dt, kv=rng.choice([dt, dt, "f32"]), page=page,
                    halves=rng.random() < 0.5, seqs=seqs, tokens=max(seqs, _log(rng, 1, 6000)),
                    start=rng.choice([0, _log(rng, 1, 130000)]), pad=rng.choice([0, rng.randint(1, 16)]))
    if kind == "decode":
        while True:
            longest = _log(rng, 1, 130000)
            case = dict(kind=kind, **dims, heads=heads, dt=dt, page=page, seqs=_log(rng, 1, 128),
                        new=rng.choice([1, 1, 2, 4]), shortest=_log(rng, 1, longest), longest=longest)
            w = work(case)
            if w["bytes"] < 6e8 and w["flops"] < 7e10:
                return case
    while True:
        n = _log(rng, 1, 12)
        q = [_log(rng, 1, 8000) for _ in range(n)]
        k = [a + rng.choice([0, 0, _log(rng, 1, 4000)]) for a in q]
        case = dict(kind=kind, **dims, heads=heads, dt=dt, q=",".join(map(str, q)), k=",".join(map(str, k)))
        w = work(case)
        if w["bytes"] < 9e8 and w["flops"] < 2e12:
            return case


def _lens(case):
    """Cached tokens of each sequence: spread evenly over the logarithm, in a mixed order."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
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
    q, k = ([int(a) for a in case[n].split(",")] for n in ("q", "k"))
    return q, k


# ------------------------------------------------------------------------------- what a program holds before the call


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _offsets(lengths):
    return _ints([sum(lengths[:i]) for i in range(len(lengths) + 1)])


def _pages(g, needed, max_pages):
    """Block table [len(needed)][max_pages] whose first needed[i] entries (a list of page indices) are pages of a pool in a
    random order; the other entries are never used. Returns the table and the number of pages in the pool."""
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
    dt = _DT[case["dt"]]
    rank, rope, nope, v, heads = (case[n] for n in ("rank", "rope", "nope", "v", "heads"))

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    if case["kind"] == "append":
        ps, counts = case["page"], _counts(case)
        starts = [case["start"] * (i + 1) // len(counts) for i in range(len(counts))]
        used = [list(range(s // ps, (s + n - 1) // ps + 1)) for s, n in zip(starts, counts)]
        table, pages = _pages(g, used, max(u[-1] for u in used) + 1)
        st = dict(pool=normal(pages, ps, rank + rope), table=table)
        rows = case["tokens"] + case["pad"]
        st["seqs"] = _ints([i for i, n in enumerate(counts) for _ in range(n)] + [-1] * case["pad"])
        st["positions"] = _ints([s + j for s, n in zip(starts, counts) for j in range(n)] + [0] * case["pad"])
        st["kv"] = normal(rows, rank + rope, scale=1.5, dtype=_DT[case["kv"]])
        st["q"] = normal(rows, heads, nope + rope)
        st["weight"] = (1.0 + 0.2 * torch.randn(rank, generator=g, device=DEV)).to(torch.float16)
        st["inv_freq"] = (50000.0 ** (-torch.arange(0, rope, 2, device=DEV, dtype=torch.float64) / rope)).float()
        st["q_out"] = torch.zeros(rows, heads, rope, dtype=dt, device=DEV)
        st["kv_out"] = torch.zeros(rows, rank + rope, dtype=dt, device=DEV)
        if own:
            from vib3_amd import mla
            st["cache"] = mla.MlaCache(st["pool"], rank)
    elif case["kind"] == "decode":
        ps, lens, new = case["page"], _lens(case), case["new"]
        used = [list(range((n + ps - 1) // ps)) for n in lens]
        table, pages = _pages(g, used, max(len(u) for u in used))
        st = dict(pool=normal(pages, ps, rank + rope), table=table)
        # the rows of a sequence are its newest tokens: row j sees everything up to itself
        st["seqs"] = _ints([i for i in range(len(lens)) for _ in range(new)])
        st["lens"] = _ints([max(0, n - new + 1 + j) for n in lens for j in range(new)])
        st["q"] = normal(len(lens) * new, heads, nope + rope, scale=2.0)
        st["kv_b"] = normal(heads, nope + v, rank, scale=rank ** -0.5)
        if own:
            from vib3_amd import mla
            st["op"] = mla.MlaDecode(mla.MlaCache(st["pool"], rank), heads, nope, v, max_rows=len(lens) * new)
    else:
        nq, nk = _spans(case)
        st = dict(cu_q=_offsets(nq), cu_k=_offsets(nk))
        st["q"] = normal(sum(nq), heads, nope + rope, scale=2.0)
        st["kv"] = normal(sum(nk), heads, nope + v)
        st["rows"] = normal(sum(nk), rank + rope)  # the latent and the rotated key of each token, as appended
        st["out"] = torch.empty(sum(nq), heads, v, dtype=dt, device=DEV)
    st["case"], st["scale"] = case, (nope + rope) ** -0.5
    return st


# ------------------------------------------------------------------------------- one pass


def run(st):
    return {"append": _append, "decode": _decode, "prefill": _prefill}[st["case"]["kind"]](st)


def _append(st):
    case = st["case"]
    rank, nope, halves = case["rank"], case["nope"], case["halves"]
    q_rope = st["q"][..., nope:]
    if own:
        from vib3_amd import mla
        mla.mla_append(st["cache"], st["table"], st["seqs"], st["positions"], st["kv"], st["inv_freq"], norm_weight=st["weight"],
                       eps=_EPS, interleaved=not halves, q_rope=q_rope, q_out=st["q_out"], kv_out=st["kv_out"])
        return st["pool"], st["q_out"], st["kv_out"]
    pool, n = st["pool"], case["tokens"]  # the rows behind are padding
    seqs, pos = st["seqs"][:n].long(), st["positions"][:n].long()
    angle = pos.double()[:, None] * st["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()

    def rotate(x, cos, sin):
        a, b = x.chunk(2, -1) if halves else (x[..., 0::2], x[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([a, b], -1) if halves else torch.stack([a, b], -1).flatten(-2)

    kv = st["kv"][:n].float()
    c = kv[:, :rank]
    c = c * torch.rsqrt((c * c).mean(-1, keepdim=True) + _EPS) * st["weight"].float()
    row = torch.cat([c, rotate(kv[:, rank:], cos, sin)], -1).to(pool.dtype)
    page = st["table"][seqs, pos // case["page"]].long()
    pool[page, pos % case["page"]] = row
    st["kv_out"][:n] = row
    st["q_out"][:n] = rotate(q_rope[:n].float(), cos[:, None], sin[:, None]).to(pool.dtype)
    return pool, st["q_out"], st["kv_out"]


def _decode(st):
    case = st["case"]
    rank, nope, new = case["rank"], case["nope"], case["new"]
    q_nope, q_rope = st["q"][..., :nope], st["q"][..., nope:]
    if own:
        return st["op"].launch(q_nope, q_rope, st["kv_b"], st["table"], st["lens"], seqs=st["seqs"], scale=st["scale"])
    w_uk, w_uv = st["kv_b"][:, :nope].float(), st["kv_b"][:, nope:].float()
    ql = torch.bmm(q_nope.float().transpose(0, 1).contiguous(), w_uk).transpose(0, 1)  # [rows, heads, rank]
    ql = torch.cat([ql, q_rope.float()], -1)
    out = torch.empty(ql.shape[0], case["heads"], rank, device=DEV)
    for i, n in enumerate(_lens(case)):
        rows = slice(i * new, (i + 1) * new)
        used = st["table"][i, :(n + case["page"] - 1) // case["page"]].long()
        c = st["pool"][used].flatten(0, 1)[:n].float()
        s = (ql[rows].flatten(0, 1) @ c.t()).view(new, -1, n) * st["scale"]
        seen = torch.arange(n, device=DEV) < st["lens"][rows, None]
        s = s.masked_fill(~seen[:, None], -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-3e38))
        out[rows] = (p @ c[:, :rank]) / p.sum(-1, keepdim=True).clamp_min(1e-38)
    out = torch.bmm(out.transpose(0, 1).contiguous(), w_uv.transpose(1, 2).contiguous())
    return out.transpose(0, 1).contiguous().to(st["q"].dtype)


def _prefill(st):
    case = st["case"]
    rank, nope, heads = case["rank"], case["nope"], case["heads"]
    k_rope = st["rows"][:, rank:]
    if own:
        from vib3_amd import mla
        return mla.mla_prefill(st["q"][..., :nope], st["q"][..., nope:], st["kv"], k_rope, st["cu_q"], st["cu_k"],
                               scale=st["scale"], out=st["out"])
    q0 = k0 = 0
    for nq, nk in zip(*_spans(case)):
        hidden = torch.arange(nk, device=DEV) > torch.arange(nq, device=DEV)[:, None] + (nk - nq)
        kr = k_rope[k0:k0 + nk].float()
        for h in range(heads):
            q = st["q"][q0:q0 + nq, h].float()
            k = torch.cat([st["kv"][k0:k0 + nk, h, :nope].float(), kr], -1)
            s = (q @ k.t()).mul_(st["scale"]).masked_fill_(hidden, -math.inf)
            p = s.sub_(s.amax(-1, keepdim=True)).exp_()
            o = (p @ st["kv"][k0:k0 + nk, h, nope:].float()) / p.sum(-1, keepdim=True)
            st["out"][q0:q0 + nq, h] = o.to(st["out"].dtype)
        q0, k0 = q0 + nq, k0 + nk
    return st["out"]


# ------------------------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    rank, nope, heads, scale = case["rank"], case["nope"], case["heads"], st["scale"]
    if case["kind"] == "append":
        pool, half = st["pool"].double(), case["rope"] // 2
        q_out, kv_out = st["q_out"].double(), st["kv_out"].double()
        live = (st["seqs"] >= 0).nonzero()[:, 0]
        pos = st["positions"][live].double()
        turn = torch.polar(torch.ones(len(live), half, device=DEV, dtype=torch.float64), torch.outer(pos, st["inv_freq"].double()))
        i = torch.arange(half, device=DEV)
        first, second = (i, i + half) if case["halves"] else (2 * i, 2 * i + 1)

        def turned(x, turn):  # a pair as a complex number times e^(i angle)
            z = torch.complex(x[..., first], x[..., second]) * turn
            out = torch.empty_like(x)
            out[..., first], out[..., second] = z.real, z.imag
            return out

        kv = st["kv"][live].double()
        norm = (kv[:, :rank].square().sum(-1) / rank + _EPS).sqrt()
        kv_out[live, :rank] = kv[:, :rank] / norm[:, None] * st["weight"].double()
        kv_out[live, rank:] = turned(kv[:, rank:], turn)
        q_out[live] = turned(st["q"][live][..., nope:].double(), turn[:, None])
        at = st["positions"][live].long()
        pool[st["table"][st["seqs"][live].long(), at // case["page"]].long(), at % case["page"]] = kv_out[live]
        return pool, q_out, kv_out
    if case["kind"] == "decode":
        rows = len(st["lens"])
        out = torch.zeros(rows, heads, case["v"], device=DEV, dtype=torch.float64)
        lens, seqs = st["lens"].tolist(), st["seqs"].tolist()
        kv_b = st["kv_b"].double()
        flat = st["pool"].flatten(0, 1)
        for s, n in enumerate(_lens(case)):
            j = torch.arange(n, device=DEV)
            c = flat[st["table"][s].long()[j // case["page"]] * case["page"] + j % case["page"]].double()
            mine = [r for r in range(rows) if seqs[r] == s]
            for h0 in range(0, heads, max(1, min(heads, 400000 // n))):  # some heads at a time: keys and values of each
                hs = slice(h0, min(heads, h0 + max(1, min(heads, 400000 // n))))
                kv = torch.matmul(kv_b[hs].flatten(0, 1), c[:, :rank].t().contiguous()).view(-1, nope + case["v"], n)
                for r in mine:
                    if lens[r] == 0:
                        continue
                    q = st["q"][r, hs].double()
                    x = torch.bmm(q[:, None, :nope].contiguous(), kv[:, :nope].contiguous())[:, 0] + q[:, nope:] @ c[:, rank:].t()
                    p = torch.softmax(x[:, :lens[r]] * scale, -1)
                    out[r, hs] = (kv[:, nope:, :lens[r]] * p[:, None]).sum(-1)
        return out
    out = torch.zeros(st["out"].shape, device=DEV, dtype=torch.float64)
    q0 = k0 = 0
    for nq, nk in zip(*_spans(case)):
        kr = st["rows"][k0:k0 + nk, rank:].double()
        for h in range(heads):
            kv = st["kv"][k0:k0 + nk, h].double()
            k = torch.cat([kv[:, :nope], kr], 1).t().contiguous()
            for a in range(0, nq, 4096):
                b = min(nq, a + 4096)
                see = nk - nq + b  # keys that the last of these queries sees
                x = st["q"][q0 + a:q0 + b, h].double() @ k[:, :see] * scale
                x += torch.full_like(x, -math.inf).triu_(nk - nq + a + 1)
                out[q0 + a:q0 + b, h] = torch.softmax(x, -1) @ kv[:see, nope:]
        q0, k0 = q0 + nq, k0 + nk
    return out


# ------------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    rank, rope, nope, v, heads = (case[n] for n in ("rank", "rope", "nope", "v", "heads"))
    if case["kind"] == "append":
        n, kvb = case["tokens"], 4 if case["kv"] == "f32" else 2
        # the new rows read, written to the cache and to kv_out; the rotary part of the queries read and written
        bytes_ = n * (rank + rope) * (kvb + 2 + 2) + n * heads * rope * 4 + rank * 2 + n * 12
        return {"bytes": bytes_, "flops": n * (4 * rank + 3 * rope) + n * heads * rope * 3}
    if case["kind"] == "decode":
        lens, new = _lens(case), case["new"]
        rows = len(lens) * new
        seen = sum(max(0, n - new + 1 + j) for n in lens for j in range(new))
        bytes_ = sum(lens) * (rank + rope) * 2 + heads * (nope + v) * rank * 2 + rows * heads * (nope + rope + v) * 2
        return {"bytes": bytes_, "flops": 2 * rows * heads * rank * (nope + v) + 2 * seen * heads * (2 * rank + rope)}
    nq, nk = _spans(case)
    pairs = sum(q * (k - q) + q * (q + 1) // 2 for q, k in zip(nq, nk))
    bytes_ = (sum(nq) * heads * (nope + rope + v) + sum(nk) * (heads * (nope + v) + rope)) * 2
    return {"bytes": bytes_, "flops": 2 * pairs * heads * (nope + rope + v)}
