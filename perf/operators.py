"""Serving from a paged key/value cache: the operators' measured cases, their plain forms and their results in 64 bits.

The cache is kp / vp [pages, Hkv, page, D] fp16; position p of sequence b lies on page table[b][p // page], row
p % page. A case is a dict of plain values; `op` selects the operator:

  append   hi.rope_cache_paged: rotates the q and k heads of M projected rows, writes k and v to their pages
  attn     hi.attn_paged: `seqs` sequences, one row each (rows_hi 0: a decode step) or a ragged run of rows_lo to
           rows_hi rows each, causal, after ctx_lo to ctx_hi cached positions
  shared   hi.attn_shared: a decode step of `seqs` sequences that have their first `shared` positions in common and
           ctx_lo to ctx_hi positions of their own

Queries, keys and values are N(0, 1) in fp16, as normalised projections are; pages are handed out in random order and
table entries behind a sequence's last page hold -1, as an allocator leaves them.
"""
import math

import torch

own = False

# q heads, kv heads, head dim of the models the framework's tests and benchmark name
HEADS = {"tinyllama": (32, 4, 64), "qwen25_1p5b": (12, 2, 128), "llama31_8b": (32, 8, 128)}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the cache write of one token of one conversation: a launch's latency is all there is
        {"name": "append_b1", "op": "append", "model": "llama31_8b", "page": 16, "seqs": 1, "rows": 1, "ctx": 4000,
         "rot": 128, "interleaved": False, "wide_table": False},
        # a full prefill chunk put together from three prompts
        {"name": "append_t2048", "op": "append", "model": "llama31_8b", "page": 16, "seqs": 3, "rows": 2048, "ctx": 1000,
         "rot": 128, "interleaved": False, "wide_table": False},
        # an odd number of rows far into long contexts, half of each head rotated in interleaved pairs, fp32 angles
        {"name": "append_partial_t333", "op": "append", "model": "qwen25_1p5b", "page": 64, "seqs": 5, "rows": 333,
         "ctx": 30000, "rot": 64, "interleaved": True, "wide_table": True},
        # one conversation of 4000 tokens, the smallest decode step there is
        {"name": "decode_b1_4k", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 1, "rows_lo": 0, "rows_hi": 0,
         "ctx_lo": 4000, "ctx_hi": 4000},
        # continuous batching: 48 conversations of 100 to 2000 tokens
        {"name": "decode_b48", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 48, "rows_lo": 0, "rows_hi": 0,
         "ctx_lo": 100, "ctx_hi": 2000},
        # many short conversations of a small model on large pages
        {"name": "decode_tiny_b120", "op": "attn", "model": "tinyllama", "page": 64, "seqs": 120, "rows_lo": 0,
         "rows_hi": 0, "ctx_lo": 1, "ctx_hi": 700},
        # four drafted tokens to verify in each of 8 conversations
        {"name": "verify_b8", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 8, "rows_lo": 5, "rows_hi": 5,
         "ctx_lo": 700, "ctx_hi": 4000},
        # prompt chunks of unequal lengths in one batch, some of a single row
        {"name": "ragged_qwen_b7", "op": "attn", "model": "qwen25_1p5b", "page": 32, "seqs": 7, "rows_lo": 1,
         "rows_hi": 411, "ctx_lo": 0, "ctx_hi": 1500},
        # a full chunk far into a long prompt: the largest matrix products
        {"name": "chunk_t2048_p4096", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 1, "rows_lo": 2048,
         "rows_hi": 2048, "ctx_lo": 4096, "ctx_hi": 4096},
        # a few conversations over a short system prompt
        {"name": "shared_b5_p512", "op": "shared", "model": "tinyllama", "page": 16, "seqs": 5, "shared": 512,
         "ctx_lo": 1, "ctx_hi": 300},
        # questions about one long document
        {"name": "shared_b32_p8192", "op": "shared", "model": "llama31_8b", "page": 16, "seqs": 32, "shared": 8192,
         "ctx_lo": 30, "ctx_hi": 700},
        # sampling many answers to one very long prompt
        {"name": "shared_b64_p32768", "op": "shared", "model": "llama31_8b", "page": 64, "seqs": 64, "shared": 32768,
         "ctx_lo": 1, "ctx_hi": 400},
    ]


def _log(rng, lo, hi, multiple=1):
    """A whole number spread over the logarithm of [lo, hi]."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v) // multiple * multiple))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "ragged", "ragged", "shared"])
    c = {"op": op if op in ("append", "shared") else "attn", "model": rng.choice(sorted(HEADS)),
         "page": rng.choice([8, 16, 16, 32, 64, 128])}
    D = HEADS[c["model"]][2]
    if op == "append":
        rows = _log(rng, 1, 2048)
        return {**c, "seqs": min(rows, rng.randint(1, 64)), "rows": rows, "ctx": _log(rng, 1, 30000),
                "rot": rng.choice([D, D, D // 2, D // 4]), "interleaved": rng.random() < 0.3,
                "wide_table": rng.random() < 0.5}
    if op == "decode":
        seqs = rng.choice([1, rng.randint(2, 8), rng.randint(9, 64), rng.randint(65, 128)])
        top = _log(rng, 16, 32000 if seqs == 1 else 6000 if seqs <= 8 else 2000)
        return {**c, "seqs": seqs, "rows_lo": 0, "rows_hi": 0, "ctx_lo": rng.randint(0, top), "ctx_hi": top}
    if op == "ragged":
        seqs = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 24)])
        rows = _log(rng, 1, 2048 // seqs)
        ctx = _log(rng, 1, 4096)
        return {**c, "seqs": seqs, "rows_lo": rng.randint(1, rows), "rows_hi": rows, "ctx_lo": rng.randint(0, ctx),
                "ctx_hi": ctx}
    top = _log(rng, 1, 700)
    return {**c, "seqs": _log(rng, 2, 64), "shared": _log(rng, 128, 32768, 128), "ctx_lo": rng.randint(1, top),
            "ctx_hi": top}


def _spread(lo, hi, n, turn=0):
    """n whole numbers spread evenly over [lo, hi], both ends among them, in a mixed order."""
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((step * b + turn) % n) // max(1, n - 1) if n > 1 else hi for b in range(n)]


def _plan(c):
    """Rows and cached positions before them, of each sequence (shared: before its last position)."""
    if c["op"] == "append":
        n = [c["rows"] // c["seqs"] + (b < c["rows"] % c["seqs"]) for b in range(c["seqs"])]
        return n, _spread(0, c["ctx"], c["seqs"])
    ctx = _spread(c["ctx_lo"], c["ctx_hi"], c["seqs"])
    if c["op"] == "shared":
        return [1] * c["seqs"], [c["shared"] + x - 1 for x in ctx]
    return [max(1, r) for r in _spread(c["rows_lo"], c["rows_hi"], c["seqs"], 1)], ctx


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    Hq, Hkv, D = HEADS[case["model"]]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, before = _plan(case)
    B, M, page = len(rows), sum(rows), case["page"]
    ends = [p + r for p, r in zip(before, rows)]
    W = max(-(-e // page) for e in ends)
    common = case.get("shared", 0) // page  # pages that every sequence has
    need = [max(0, -(-e // page) - common) for e in ends]
    pages = common + sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    at = common
    for b, n in enumerate(need):
        table[b, :common] = order[:common]
        table[b, common:common + n] = order[at:at + n]
        at += n

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float16)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device="cuda")

    s = {"c": case, "kp": normal(pages, Hkv, page, D), "vp": normal(pages, Hkv, page, D), "table": table}
    if case["op"] == "append":
        s["qkv"] = normal(M, (Hq + 2 * Hkv) * D)
        s["seq"] = ints([b for b, n in enumerate(rows) for _ in range(n)])
        s["pos"] = ints([p + t for p, n in zip(before, rows) for t in range(n)])
        angle = torch.arange(max(ends), device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"]))
        s["cs"] = torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32 if case["wide_table"] else torch.float16)
        s["q_out"] = torch.empty(M, Hq * D, dtype=torch.float16, device="cuda")
        return s
    s["q"] = normal(M, Hq * D)
    s["out"] = torch.empty_like(s["q"])
    s["pos"] = ints(before)
    if case["op"] == "attn" and case["rows_hi"]:
        first = [sum(rows[:b]) for b in range(B + 1)]
        s["start"] = ints(first)
        s["lse"] = torch.empty(Hq, M, dtype=torch.float32, device="cuda")
        s["longest"] = max(ends), max(rows)
        s["row_seq"] = ints([b for b, n in enumerate(rows) for _ in range(n)]).long()
        s["row_at"] = ints([t for n in rows for t in range(n)]).long()
    else:
        s["longest"] = max(ends), 1
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    Hq, Hkv, D = HEADS[c["model"]]
    if own:
        from hipinfer_amd import hipinfer as hi
        if c["op"] == "append":
            hi.rope_cache_paged(s["qkv"], Hq, Hkv, s["cs"], s["kp"], s["vp"], s["table"], s["pos"], seq=s["seq"],
                                interleaved=c["interleaved"], q_out=s["q_out"])
            return s["q_out"], s["kp"], s["vp"]
        if c["op"] == "shared":
            if "work" not in s:  # a serving loop keeps it
                s["work"] = hi.attn_shared_work(s["pos"].shape[0], Hq, Hkv, D)
            return hi.attn_shared(s["q"], s["kp"], s["vp"], s["table"], s["pos"], c["shared"], Hq, Hkv, out=s["out"],
                                  work=s["work"])
        if "work" not in s:
            s["work"] = hi.attn_paged_work(s["q"].shape[0], s["pos"].shape[0], Hq, Hkv, D, ragged="start" in s)
        hi.attn_paged(s["q"], s["kp"], s["vp"], s["table"], s["pos"], Hq, Hkv, start=s.get("start"), out=s["out"],
                      lse=s.get("lse"), work=s["work"])
        return (s["out"], s["lse"]) if "start" in s else s["out"]
    if c["op"] == "append":
        return _append_plain(s, c, Hq, Hkv, D)
    if c["op"] == "shared":
        return _shared_plain(s, c, Hq, Hkv, D)
    return _attn_plain(s, c, Hq, Hkv, D)


def _append_plain(s, c, Hq, Hkv, D):
    qkv, page, pos = s["qkv"], c["page"], s["pos"].long()
    M = qkv.shape[0]
    heads = qkv.view(M, Hq + 2 * Hkv, D)
    x = heads[:, :Hq + Hkv].float()
    cs = s["cs"][pos].float()[:, None]  # [M, 1, rot / 2, 2]
    cos, sin = cs[..., 0], cs[..., 1]
    rot = 2 * cos.shape[-1]
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    y = torch.cat([turned, x[..., rot:]], -1).half()
    pg = s["table"][s["seq"].long(), pos // page].long()
    s["kp"][pg, :, pos % page] = y[:, Hq:]
    s["vp"][pg, :, pos % page] = heads[:, Hq + Hkv:]
    s["q_out"].copy_(y[:, :Hq].reshape(M, Hq * D))
    return s["q_out"], s["kp"], s["vp"]


def _gather(cache, table, first, last, page):
    """Positions first .. last - 1 of each row of table, [B, n, Hkv, D] in 32 bits (page 0 where there is none)."""
    p = torch.arange(first, last, device=table.device)
    pg = table[:, p // page].clamp(min=0).long()
    return cache[pg, :, (p % page).expand_as(pg)].float()


def _attn_plain(s, c, Hq, Hkv, D):
    B, (L, R), G, page = s["pos"].shape[0], s["longest"], Hq // Hkv, c["page"]
    q = s["q"].float()
    if "start" in s:  # each sequence's rows, padded to the longest run
        padded = torch.zeros(B, R, Hq * D, device=q.device)
        padded[s["row_seq"], s["row_at"]] = q
        q = padded
    q = q.view(B, R, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, R * G, D)
    K, V = (_gather(s[n], s["table"], 0, L, page).permute(0, 2, 1, 3).contiguous() for n in ("kp", "vp"))
    x = torch.matmul(q, K.transpose(2, 3).contiguous()).div_(math.sqrt(D)).view(B, Hkv, R, G, L)
    last = s["pos"].long()[:, None] + torch.arange(R, device=q.device)
    hidden = torch.arange(L, device=q.device) > last[:, :, None]
    x.masked_fill_(hidden[:, None, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hkv, R * G, L), V).view(B, Hkv, R, G, D) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(B, R, Hq * D)
    if "start" not in s:
        return o[:, 0].half()
    lse = ((m + total.log()) / math.log(2.0)).permute(0, 2, 1, 3, 4).reshape(B, R, Hq)
    return o[s["row_seq"], s["row_at"]].half(), lse[s["row_seq"], s["row_at"]].t().contiguous()


def _shared_plain(s, c, Hq, Hkv, D):
    B, (L, _), G, page, P = s["pos"].shape[0], s["longest"], Hq // Hkv, c["page"], c["shared"]
    q = s["q"].float().view(B, Hkv, G, D)
    # the common keys once for all rows, then each sequence's own
    Kp, Vp = (_gather(s[n], s["table"][:1], 0, P, page)[0].transpose(0, 1).contiguous() for n in ("kp", "vp"))
    Ks, Vs = (_gather(s[n], s["table"], P, L, page).transpose(1, 2).contiguous() for n in ("kp", "vp"))
    every = q.transpose(0, 1).reshape(Hkv, B * G, D)
    xp = torch.matmul(every, Kp.transpose(1, 2).contiguous()).view(Hkv, B, G, P).transpose(0, 1)
    xs = torch.matmul(q, Ks.transpose(2, 3).contiguous())
    x = torch.cat([xp, xs], -1).div_(math.sqrt(D))
    hidden = torch.arange(L, device=q.device) > s["pos"].long()[:, None]
    x.masked_fill_(hidden[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    op = torch.matmul(p[..., :P].transpose(0, 1).reshape(Hkv, B * G, P), Vp).view(Hkv, B, G, D).transpose(0, 1)
    o = (op + torch.matmul(p[..., P:], Vs)) / p.sum(-1, keepdim=True)
    return o.reshape(B, Hq * D).half()


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    Hq, Hkv, D = HEADS[case["model"]]
    rows, before = _plan(case)
    B, M = len(rows), sum(rows)
    if case["op"] == "append":
        cs = M * case["rot"] * (4 if case["wide_table"] else 2)
        return {"bytes": 2 * M * (Hq + 2 * Hkv) * D * 2 + cs + 12 * M, "flops": 3 * M * (Hq + Hkv) * case["rot"]}
    visible = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, before))
    keys = sum(p + r for p, r in zip(before, rows))
    if case["op"] == "shared":
        keys -= (B - 1) * case["shared"]
    return {"bytes": keys * (2 * Hkv * D * 2 + 4 / case["page"]) + 2 * M * Hq * D * 2 + (4 * M * Hq if case.get("rows_hi") else 0),
            "flops": 4 * D * Hq * visible}


# ------------------------------------------------------------------ the results in 64 bits
def exact(case, seed):
    Hq, Hkv, D = HEADS[case["model"]]
    s = prepare(case, seed)
    rows, before = _plan(case)
    page = case["page"]
    if case["op"] == "append":
        x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
        half = case["rot"] // 2
        j = torch.arange(half, device=x.device)
        lo, hi_ = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
        z = torch.view_as_complex(s["cs"].double().contiguous())[s["pos"].long()][:, None]
        z = z * torch.complex(x[:, :Hq + Hkv, lo], x[:, :Hq + Hkv, hi_])
        x[:, :Hq + Hkv, lo], x[:, :Hq + Hkv, hi_] = z.real, z.imag
        kp, vp = s["kp"].double(), s["vp"].double()
        m = 0
        for b, (n, p) in enumerate(zip(rows, before)):
            for at in range(p, p + n):
                pg = int(s["table"][b, at // page]) if at % page == 0 or at == p else pg
                kp[pg, :, at % page] = x[m, Hq:Hq + Hkv]
                vp[pg, :, at % page] = x[m, Hq + Hkv:]
                m += 1
        return x[:, :Hq].reshape(-1, Hq * D), kp, vp
    out = torch.empty(sum(rows), Hq * D, dtype=torch.float64, device="cuda")
    lse = torch.empty(Hq, sum(rows), dtype=torch.float64, device="cuda")
    m = 0
    for b, (n, p) in enumerate(zip(rows, before)):
        ids = s["table"][b, :-(-(p + n) // page)].long()
        K, V = (s[name][ids].double().transpose(0, 1).reshape(Hkv, -1, D)[:, :p + n] for name in ("kp", "vp"))
        unseen = torch.ones(n, p + n, dtype=torch.bool, device="cuda").triu(p + 1)
        for h in range(Hq):
            x = s["q"][m:m + n, h * D:(h + 1) * D].double() @ K[h * Hkv // Hq].T.contiguous() / math.sqrt(D)
            x[unseen] = -math.inf
            total = torch.logsumexp(x, -1)
            out[m:m + n, h * D:(h + 1) * D] = torch.exp(x - total[:, None]) @ V[h * Hkv // Hq]
            lse[h, m:m + n] = total / math.log(2.0)
        m += n
    return (out, lse) if case.get("rows_hi") else out
