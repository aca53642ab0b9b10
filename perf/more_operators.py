"""Beam search and long contexts on a paged cache held in 8 bits: the operators' measured cases, their plain forms and their
results in 64 bits.

The 8-bit cache is kp / vp [pages, Hkv, page, D] float8_e4m3fn with kexp / vexp [pages, Hkv] int8: position p of sequence b lies on
page table[b][p // page], row p % page, and holds code * 2^exponent of its page and head. The exponent of a page is the least k
(-32 to 8) with max |x| <= 448 * 2^k over the values written to it. `op` selects the operator:

  append   hi.rope_cache_paged8: rotates the q and k heads of projected rows, rounds k and v to 8 bits on their pages; a page whose
           exponent grows has its earlier positions rounded to the new one
  attn     hi.attn_paged8: `seqs` sequences, one row each (rows_hi 0: a decode step) or a ragged run of rows_lo to rows_hi
           rows each, causal, after ctx_lo to ctx_hi cached positions
  beam     hi.beam_select: the n best continuations of each of `seqs` sequences over `beams` beams and the vocabulary
  fork     hi.cache_fork: every row of a page table becomes a continuation of its parent's row: whole pages are shared, a
           part-filled one is copied unless the row inherits it, the next positions' pages are taken from the free ones
  compact  hi.cache_compact: pages in use move to the front of the pool

Queries, keys and values are normal, keys and values with a magnitude of their own per head; pages are handed out in random order
and table entries behind a sequence's last page hold -1, as an allocator leaves them.
"""
import math

import torch

own = False

# q heads, kv heads, head dim, layers, vocabulary of the models the framework's tests and benchmark name
MODELS = {"tinyllama": (32, 4, 64, 22, 32000), "qwen25_1p5b": (12, 2, 128, 28, 151936), "llama31_8b": (32, 8, 128, 32, 128256)}
F8 = torch.float8_e4m3fn


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the cache write of one decode step of 48 conversations: a launch's latency is most of it
        {"name": "append8_b48", "op": "append", "model": "llama31_8b", "page": 16, "seqs": 48, "rows": 48, "ctx": 2000,
         "rot": 128, "interleaved": False, "wide_table": False},
        # a full prefill chunk put together from three prompts, their first rows behind earlier chunks on large pages
        {"name": "append8_t2048", "op": "append", "model": "llama31_8b", "page": 64, "seqs": 3, "rows": 2048, "ctx": 1000,
         "rot": 64, "interleaved": True, "wide_table": True},
        # one conversation of 4000 tokens, the smallest decode step there is
        {"name": "decode8_b1_4k", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 1, "rows_lo": 0, "rows_hi": 0,
         "ctx_lo": 4000, "ctx_hi": 4000},
        # continuous batching: 48 conversations of 100 to 8000 tokens, what 8 bits are there for
        {"name": "decode8_b48", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 48, "rows_lo": 0, "rows_hi": 0,
         "ctx_lo": 100, "ctx_hi": 8000},
        # prompt chunks of unequal lengths in one batch, some of a single row
        {"name": "ragged8_qwen_b7", "op": "attn", "model": "qwen25_1p5b", "page": 32, "seqs": 7, "rows_lo": 1,
         "rows_hi": 411, "ctx_lo": 0, "ctx_hi": 1500},
        # a full chunk far into a long prompt: the largest matrix products
        {"name": "chunk8_t2048_p4096", "op": "attn", "model": "llama31_8b", "page": 16, "seqs": 1, "rows_lo": 2048,
         "rows_hi": 2048, "ctx_lo": 4096, "ctx_hi": 4096},
        # one request's four beams, twice as many continuations as some may have ended
        {"name": "beam_b1_k4", "op": "beam", "model": "qwen25_1p5b", "seqs": 1, "beams": 4, "n": 8},
        # a batch of requests with eight beams each
        {"name": "beam_b32_k8", "op": "beam", "model": "llama31_8b", "seqs": 32, "beams": 8, "n": 16},
        # one request's beams behind a long prompt, the 8-bit caches of some layers
        {"name": "fork_b1_k4", "op": "fork", "model": "llama31_8b", "page": 16, "seqs": 1, "beams": 4, "ctx": 4000, "made": 37,
         "layers": 4, "bits": 8},
        # a batch of requests with eight beams, the fp16 caches of all layers
        {"name": "fork_b32_k8", "op": "fork", "model": "qwen25_1p5b", "page": 16, "seqs": 32, "beams": 8, "ctx": 1500, "made": 73,
         "layers": 28, "bits": 16},
        # a small pool after most of its conversations have ended
        {"name": "compact_p500", "op": "compact", "model": "tinyllama", "page": 16, "pages": 500, "fill": 0.3, "seqs": 6,
         "layers": 22, "bits": 8},
        # a large pool, a good half of it in use
        {"name": "compact_p6000", "op": "compact", "model": "qwen25_1p5b", "page": 16, "pages": 6000, "fill": 0.55, "seqs": 40,
         "layers": 28, "bits": 8},
    ]


def _log(rng, lo, hi, multiple=1):
    """A whole number spread over the logarithm of [lo, hi]."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))
    return max(lo, min(hi, int(v) // multiple * multiple))


def draw(rng):
    op = rng.choice(["append", "append", "decode", "decode", "ragged", "ragged", "beam", "beam", "fork", "compact"])
    c = {"op": "attn" if op in ("decode", "ragged") else op, "model": rng.choice(sorted(MODELS))}
    D = MODELS[c["model"]][2]
    if op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        return {**c, "seqs": _log(rng, 1, 256 // beams), "beams": beams, "n": rng.randint(1, 2 * beams)}
    c["page"] = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "append":
        rows = _log(rng, 1, 2048)
        return {**c, "seqs": rng.choice([rows, rng.randint(1, rows)]) if rows <= 128 else rng.randint(1, 64), "rows": rows,
                "ctx": _log(rng, 1, 8000), "rot": rng.choice([D, D, D // 2, D // 4]), "interleaved": rng.random() < 0.3,
                "wide_table": rng.random() < 0.5}
    if op == "decode":
        seqs = rng.choice([1, rng.randint(2, 8), rng.randint(9, 64), rng.randint(65, 128)])
        top = _log(rng, 16, 32000 if seqs == 1 else 8000 if seqs <= 48 else 2500)
        return {**c, "seqs": seqs, "rows_lo": 0, "rows_hi": 0, "ctx_lo": rng.randint(0, top), "ctx_hi": top}
    if op == "ragged":
        seqs = rng.choice([1, 1, rng.randint(2, 8), rng.randint(9, 24)])
        rows = _log(rng, 1, 2048 // seqs)
        ctx = _log(rng, 1, 4096)
        return {**c, "seqs": seqs, "rows_lo": rng.randint(1, rows), "rows_hi": rows, "ctx_lo": rng.randint(0, ctx),
                "ctx_hi": ctx}
    c |= {"layers": rng.randint(1, 8), "bits": rng.choice([8, 16])}
    if op == "fork":
        beams = rng.choice([2, 3, 4, 5, 8])
        return {**c, "seqs": _log(rng, 1, 24), "beams": beams, "ctx": _log(rng, 1, 1500), "made": rng.randint(0, 100)}
    pages = _log(rng, 40, 12000 // c["page"])
    return {**c, "pages": pages, "fill": round(rng.uniform(0.1, 0.9), 2), "seqs": rng.randint(1, min(40, max(1, pages // 20)))}


def _spread(lo, hi, n, turn=0):
    """n whole numbers spread evenly over [lo, hi], both ends among them, in a mixed order."""
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((step * b + turn) % n) // max(1, n - 1) if n > 1 else hi for b in range(n)]


def _rows(c):
    """Rows and cached positions before them, of each sequence."""
    if c["op"] == "append":
        n = [c["rows"] // c["seqs"] + (b < c["rows"] % c["seqs"]) for b in range(c["seqs"])]
        return n, _spread(0, c["ctx"], c["seqs"])
    return [max(1, r) for r in _spread(c["rows_lo"], c["rows_hi"], c["seqs"], 1)], _spread(c["ctx_lo"], c["ctx_hi"], c["seqs"])


def _held(c):
    """Pages that each of compact's sequences holds."""
    used = max(1, int(c["pages"] * c["fill"]))
    return [used // c["seqs"] + (b < used % c["seqs"]) for b in range(c["seqs"])]


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"append": _prepare_rows, "attn": _prepare_rows, "beam": _prepare_beam, "fork": _prepare_fork,
            "compact": _prepare_compact}[case["op"]](case, g)


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float16)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cache8(g, pages, Hkv, page, D):
    """Codes and exponents of normal values whose magnitude is 1/2, 1 or 2 by page and head."""
    size = torch.randint(-1, 2, (pages, Hkv), device="cuda", generator=g)
    exp = size - 6  # the largest of some thousand normal values lies between 3.5 and 7, 448 / 128 and 448 / 64
    codes = (torch.randn(pages, Hkv, page, D, device="cuda", generator=g) * 64).clamp_(-448, 448).to(F8)
    return codes, exp.to(torch.int8)


def _prepare_rows(case, g):
    Hq, Hkv, D = MODELS[case["model"]][:3]
    rows, before = _rows(case)
    B, M, page = len(rows), sum(rows), case["page"]
    ends = [p + r for p, r in zip(before, rows)]
    W = max(-(-e // page) for e in ends)
    # append: the pages that the rows lie on, and the entries before them that other calls have filled
    first = [p // page if case["op"] == "append" else 0 for p in before]
    need = [-(-e // page) - f for e, f in zip(ends, first)]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, first[b]:first[b] + n] = order[at:at + n]
        at += n
    s = {"c": case, "table": table, "pos": _ints(before)}
    s["kp"], s["kexp"] = _cache8(g, pages, Hkv, page, D)
    s["vp"], s["vexp"] = _cache8(g, pages, Hkv, page, D)
    s["row_seq"] = _ints([b for b, n in enumerate(rows) for _ in range(n)]).long()
    s["row_at"] = _ints([t for n in rows for t in range(n)]).long()
    if M > B or case.get("rows_hi"):
        s["start"] = _ints([sum(rows[:b]) for b in range(B + 1)])
    if case["op"] == "append":
        s["qkv"] = _normal(g, M, (Hq + 2 * Hkv) * D)
        angle = torch.arange(max(ends), device="cuda", dtype=torch.float64)[:, None] * (
            500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"]))
        s["cs"] = torch.stack([angle.cos(), angle.sin()], -1).to(torch.float32 if case["wide_table"] else torch.float16)
        s["q_out"] = torch.empty(M, Hq * D, dtype=torch.float16, device="cuda")
        return s
    s["q"] = _normal(g, M, Hq * D)
    s["out"] = torch.empty_like(s["q"])
    s["longest"] = max(ends), max(rows)
    if "start" in s:
        s["lse"] = torch.empty(Hq, M, dtype=torch.float32, device="cuda")
    return s


def _prepare_beam(case, g):
    V, R = MODELS[case["model"]][4], case["seqs"] * case["beams"]
    s = {"c": case}
    # logits of a language model: most far below a few; cumulative scores of beams that have run for some tokens
    s["logits"] = _normal(g, R, V) * 2.5
    s["scores"] = -10 * torch.rand(R, device="cuda", generator=g) - 5
    s["best"] = torch.empty(case["seqs"], case["n"], device="cuda")
    s["parent"], s["token"] = (torch.empty(case["seqs"], case["n"], dtype=torch.int32, device="cuda") for _ in range(2))
    return s


def _pool(case, g, pages):
    """The layers' caches as [layers, pages, ...] pools, and each layer's as the calls take them."""
    _, Hkv, D = MODELS[case["model"]][:3]
    L, page = case["layers"], case["page"]
    if case["bits"] == 16:
        pools = [_normal(g, L, pages, Hkv, page, D) for _ in range(2)]
    else:
        pools = [x.view(L, pages, *x.shape[1:]) for _ in range(2) for x in _cache8(g, L * pages, Hkv, page, D)]
    return pools, [p[l] for l in range(L) for p in pools]


def _prepare_fork(case, g):
    K, page = case["beams"], case["page"]
    ctx = _spread(max(1, case["ctx"] // 4), case["ctx"], case["seqs"])
    S, common = case["seqs"] * K, [p // page for p in ctx]  # the prompt's whole pages belong to all of its beams
    held = [-(-(p + case["made"]) // page) for p in ctx]
    W = max(held) + 2
    used = sum(n + K * (h - n) for n, h in zip(common, held))
    pages = used + 2 * S + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((S, W), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for b, (n, h) in enumerate(zip(common, held)):
        table[b * K:(b + 1) * K, :n] = order[at:at + n]
        refs[order[at:at + n].long()] = K
        at += n
        table[b * K:(b + 1) * K, n:h] = order[at:at + K * (h - n)].view(K, h - n)
        refs[order[at:at + K * (h - n)].long()] = 1
        at += K * (h - n)
    # of each request's beams a half goes on, the better ones more than once
    d = max(1, K // 2)
    parent = torch.cat([torch.arange(d, device="cuda").expand(case["seqs"], d),
                        torch.randint(0, d, (case["seqs"], K - d), device="cuda", generator=g)], 1)
    turn = torch.rand(case["seqs"], K, device="cuda", generator=g)
    parent = turn.argsort(1).gather(1, parent.gather(1, torch.rand(case["seqs"], K, device="cuda", generator=g).argsort(1)))
    parent = (parent + K * torch.arange(case["seqs"], device="cuda")[:, None]).flatten().to(torch.int32)
    s = {"c": case, "table": table, "refs": refs, "parent": parent,
         "lens": _ints([p + case["made"] for p in ctx for _ in range(K)])}
    s["pools"], s["caches"] = _pool(case, g, pages)
    s["table_out"], s["lens_out"], s["refs_out"] = (torch.empty_like(s[n]) for n in ("table", "lens", "refs"))
    s["missing"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


def _prepare_compact(case, g):
    held = _held(case)
    pages, W = case["pages"], max(held) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["seqs"], W), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        refs[order[at:at + n].long()] = 1
        at += n
    s = {"c": case, "table": table, "refs": refs}
    s["pools"], s["caches"] = _pool(case, g, pages)
    s["table_out"], s["refs_out"] = torch.empty_like(table), torch.empty_like(refs)
    s["moved"], s["used"] = torch.empty_like(refs), torch.zeros(1, dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    c = s["c"]
    Hq, Hkv, D = MODELS[c["model"]][:3]
    if own:
        from hipinfer_amd import hipinfer as hi
        if c["op"] == "append":
            hi.rope_cache_paged8(s["qkv"], Hq, Hkv, s["cs"], s["kp"], s["vp"], s["kexp"], s["vexp"], s["table"], s["pos"],
                                 start=s.get("start"), interleaved=c["interleaved"], q_out=s["q_out"])
            return s["q_out"], s["kp"], s["vp"], s["kexp"], s["vexp"]
        if c["op"] == "attn":
            if "work" not in s:  # a serving loop keeps it
                s["work"] = hi.attn_paged_work(s["q"].shape[0], s["pos"].shape[0], Hq, Hkv, D, ragged="start" in s)
            hi.attn_paged8(s["q"], s["kp"], s["vp"], s["kexp"], s["vexp"], s["table"], s["pos"], Hq, Hkv, start=s.get("start"),
                           out=s["out"], lse=s.get("lse"), work=s["work"])
            return (s["out"], s["lse"]) if "start" in s else s["out"]
        if c["op"] == "beam":
            if "work" not in s:
                s["work"] = hi.beam_select_work(c["seqs"], c["beams"], s["logits"].shape[1], c["n"])
            hi.beam_select(s["logits"], s["scores"], c["beams"], c["n"], out=(s["best"], s["parent"], s["token"]), work=s["work"])
            return s["best"], s["parent"], s["token"]
        if c["op"] == "fork":
            if "work" not in s:
                s["set"] = hi.cache_set(s["caches"], c["page"])
                s["work"] = hi.cache_work(s["table"].shape[0], s["parent"].shape[0], s["refs"].shape[0])
            hi.cache_fork(s["set"], s["table"], s["lens"], s["parent"], s["refs"], grow=1, table_out=s["table_out"],
                          lens_out=s["lens_out"], refs_out=s["refs_out"], missing=s["missing"], work=s["work"])
            return s["table_out"], s["lens_out"], s["refs_out"], s["missing"], s["pools"]
        if "work" not in s:
            s["set"] = hi.cache_set(s["caches"], c["page"])
            s["work"] = hi.cache_work(s["table"].shape[0], 0, s["refs"].shape[0])
        hi.cache_compact(s["set"], s["table"], s["refs"], table_out=s["table_out"], refs_out=s["refs_out"], moved=s["moved"],
                         used=s["used"], work=s["work"])
        return s["table_out"], s["refs_out"], s["moved"], s["used"], s["pools"]
    return {"append": _append_plain, "attn": _attn_plain, "beam": _beam_plain, "fork": _fork_plain,
            "compact": _compact_plain}[c["op"]](s, c)


def _exponent(most):
    """The least k of -32 to 8 with most <= 448 * 2^k."""
    m, e = torch.frexp(most)
    return torch.where(most > 0, e - 9 + (m > 0.875), -32).clamp(-32, 8)


def _append_plain(s, c):
    Hq, Hkv, D = MODELS[c["model"]][:3]
    page, seq, M = c["page"], s["row_seq"], s["qkv"].shape[0]
    pos = s["pos"].long()[seq] + s["row_at"]
    heads = s["qkv"].view(M, Hq + 2 * Hkv, D).float()
    x = heads[:, :Hq + Hkv]
    cs = s["cs"][pos].float()[:, None]
    cos, sin = cs[..., 0], cs[..., 1]
    rot = 2 * cos.shape[-1]
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    y = torch.cat([turned, x[..., rot:]], -1)
    s["q_out"].copy_(y[:, :Hq].reshape(M, Hq * D))
    pg, off = s["table"][seq, pos // page].long(), pos % page
    # each sequence's first page holds earlier positions
    pg0, n0 = s["table"].gather(1, (s["pos"].long() // page)[:, None])[:, 0].long(), s["pos"].long() % page
    for t, codes, exps in ((y[:, Hq:], s["kp"], s["kexp"]), (heads[:, Hq + Hkv:], s["vp"], s["vexp"])):
        t = t.clamp(-61440, 61440)
        most = torch.zeros(exps.shape, device=t.device).scatter_reduce_(0, pg[:, None].expand(M, Hkv), t.abs().amax(-1), "amax")
        grown = _exponent(most)
        new = grown[pg0]
        new = torch.where(n0[:, None] > 0, torch.maximum(new, exps[pg0].int()), new)
        grown[pg0] = new
        change = torch.ldexp(torch.ones((), device=t.device), exps[pg0].int() - new)[:, :, None, None]
        earlier = codes.view(torch.uint8)[pg0].view(F8)
        again = (earlier.float() * change).to(F8)
        kept = (torch.arange(page, device=t.device) < n0[:, None])[:, None, :, None]
        codes.view(torch.uint8)[pg0] = torch.where(kept, again.view(torch.uint8), earlier.view(torch.uint8))
        exps[pg] = grown[pg].to(torch.int8)
        codes.view(torch.uint8)[pg, :, off] = torch.ldexp(t, -grown[pg][..., None]).to(F8).view(torch.uint8)
    return s["q_out"], s["kp"], s["vp"], s["kexp"], s["vexp"]


def _gather8(codes, exps, table, last, page):
    """Positions 0 .. last - 1 of each row of table, [B, Hkv, last, D] in 32 bits (page 0 where there is none)."""
    pg = table[:, :-(-last // page)].clamp(min=0).long()
    x = torch.ldexp(codes.view(torch.uint8)[pg].view(F8).float(), exps[pg].int()[..., None, None])
    return x.transpose(1, 2).flatten(2, 3)[:, :, :last].contiguous()


def _attn_plain(s, c):
    Hq, Hkv, D = MODELS[c["model"]][:3]
    B, (L, R), G, page = s["pos"].shape[0], s["longest"], Hq // Hkv, c["page"]
    q = s["q"].float()
    if "start" in s:  # each sequence's rows, padded to the longest run
        padded = torch.zeros(B, R, Hq * D, device=q.device)
        padded[s["row_seq"], s["row_at"]] = q
        q = padded
    q = q.view(B, R, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, R * G, D)
    K, V = _gather8(s["kp"], s["kexp"], s["table"], L, page), _gather8(s["vp"], s["vexp"], s["table"], L, page)
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


def _beam_plain(s, c):
    # in 64 bits: two candidates a rounding apart must not change places
    V, K = s["logits"].shape[1], c["beams"]
    x = s["logits"].double()
    m = x.amax(1, keepdim=True)
    x = x - m
    x = x - x.exp().sum(1, keepdim=True).log() + s["scores"].double()[:, None]
    best, at = x.view(c["seqs"], K * V).sort(dim=1, descending=True, stable=True)
    at = at[:, :c["n"]]
    first = K * torch.arange(c["seqs"], device=x.device)[:, None]
    return best[:, :c["n"]].float(), (first + at // V).int(), (at % V).int()


def _fork_plain(s, c):
    table, lens, refs, page, grow = s["table"], s["lens"].long(), s["refs"], c["page"], 1
    (S, W), N, pages = table.shape, s["parent"].shape[0], refs.shape[0]
    dev = table.device
    p = s["parent"].long()
    ok = (p >= 0) & (p < S)
    p = torch.where(ok, p, 0)
    n = torch.where(ok, lens[p], 0)
    full, need = (n // page)[:, None], (((n + grow + page - 1) // page).clamp(max=W) * ok)[:, None]
    row, j = torch.arange(N, device=dev), torch.arange(W, device=dev)
    first = torch.full((S + 1,), N, device=dev).scatter_reduce(0, torch.where(ok, p, S), row, "amin")
    ent = torch.where(ok[:, None], table[p], -1)
    there = (ent >= 0) & (ent < pages)
    e = ent.clamp(0, pages - 1).long()
    keep = (first[p] == row)[:, None] & there & (j >= full) & (j < need) & (refs[e] == 1)
    fresh = (j >= full) & (j < need) & ~keep
    rank = (fresh.flatten().cumsum(0) - 1).view(N, W)
    empty = refs == 0
    order, free = torch.sort((~empty).int(), stable=True).indices, empty.sum()
    got = fresh & (rank < free)
    page_of = order[rank.clamp(0, pages - 1)]
    out = torch.where((there & (j < full)) | keep, e, torch.where(got, page_of, -1))
    # references: what the rows held before, what they hold now
    held = (table >= 0) & (table < pages)
    count = refs.long().scatter_add(0, table.clamp(0, pages - 1).long().flatten(), -held.flatten().long())
    count = count.scatter_add(0, out.clamp(min=0).flatten(), (out >= 0).flatten().long())
    # the positions of a part-filled page are copied (onto themselves where nothing is to be copied)
    at = full.clamp(max=W - 1)
    src = e.gather(1, at)[:, 0]
    copied = (got & there).gather(1, at)[:, 0] & (n % page > 0)
    dst = torch.where(copied, page_of.gather(1, at)[:, 0], src)
    held = (torch.arange(page, device=dev) < (n % page)[:, None])[:, None, :, None]
    for pool in s["pools"]:
        raw = pool.view(torch.uint8)
        raw[:, dst] = raw[:, src] if pool.dim() == 3 else torch.where(held, raw[:, src], raw[:, dst])
    return out.int(), n.int(), count.int(), (fresh.sum() - got.sum()).view(1).int(), s["pools"]


def _compact_plain(s, c):
    table, refs = s["table"], s["refs"]
    pages = refs.shape[0]
    idx, used = torch.arange(pages, device=refs.device), refs > 0
    n = used.sum()
    moving, hole = used & (idx >= n), ~used & (idx < n)
    holes = torch.sort((~hole).int(), stable=True).indices
    moved = torch.where(moving, holes[(moving.cumsum(0) - 1).clamp(min=0)], torch.where(used, idx, -1))
    there = (table >= 0) & (table < pages)
    out = torch.where(there, moved[table.clamp(0, pages - 1).long()], -1)
    count = torch.zeros(pages + 1, dtype=torch.int32, device=refs.device).scatter_(0, torch.where(used, moved, pages), refs)[:pages]
    src = moving.nonzero()[:, 0]
    for pool in s["pools"]:
        raw = pool.view(torch.uint8)
        raw[:, moved[src]] = raw[:, src]
    return out.int(), count, moved.int(), n.view(1).int(), s["pools"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    Hq, Hkv, D, _, V = MODELS[case["model"]]
    if case["op"] == "beam":
        R = case["seqs"] * case["beams"]
        return {"bytes": 2 * R * V + 4 * R + 12 * case["seqs"] * case["n"], "flops": 4 * R * V}
    page = case["page"]
    if case["op"] in ("fork", "compact"):
        position = 2 * Hkv * D * case["bits"] // 8 * case["layers"]  # bytes of one position in all layers
        if case["op"] == "fork":
            K, S = case["beams"], case["seqs"] * case["beams"]
            ctx = _spread(max(1, case["ctx"] // 4), case["ctx"], case["seqs"])
            tail = sum((p + case["made"]) % page for p in ctx) * (K - max(1, K // 2))
            W = max(-(-(p + case["made"]) // page) for p in ctx)
            return {"bytes": 2 * tail * position + 8 * S * W, "flops": 0}
        used = sum(_held(case))
        moves = used * (case["pages"] - used) / case["pages"]  # expected, for pages handed out at random
        return {"bytes": int(2 * moves * page * position) + 12 * case["pages"] + 8 * used, "flops": 0}
    rows, before = _rows(case)
    M = sum(rows)
    if case["op"] == "append":
        cs = M * case["rot"] * (4 if case["wide_table"] else 2)
        return {"bytes": M * ((Hq + 2 * Hkv) * D * 2 + Hq * D * 2 + 2 * Hkv * D) + cs, "flops": 3 * M * (Hq + Hkv) * case["rot"]}
    visible = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, before))
    keys = sum(p + r for p, r in zip(before, rows))
    return {"bytes": int(keys * (2 * Hkv * D + (4 + 2 * Hkv) / page)) + 2 * M * Hq * D * 2 + (4 * M * Hq if case["rows_hi"] else 0),
            "flops": 4 * D * Hq * visible}


# ------------------------------------------------------------------ the results in 64 bits
def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers, and copies
    s = prepare(case, seed)
    Hq, Hkv, D = MODELS[case["model"]][:3]
    if case["op"] == "beam":
        lp = s["scores"].double()[:, None] + torch.log_softmax(s["logits"].double(), 1)
        return lp.view(case["seqs"], -1).topk(case["n"]).values, None, None
    rows, before = _rows(case)
    page = case["page"]
    if case["op"] == "append":
        return _append_exact(case, s, rows, before, Hq, Hkv, D)
    out = torch.empty(sum(rows), Hq * D, dtype=torch.float64, device="cuda")
    lse = torch.empty(Hq, sum(rows), dtype=torch.float64, device="cuda")
    m = 0
    for b, (n, p) in enumerate(zip(rows, before)):
        ids = s["table"][b, :-(-(p + n) // page)].long()
        K, V = ((s[t + "p"].view(torch.uint8)[ids].view(F8).double() * 2.0 ** s[t + "exp"][ids].double()[..., None, None])
                .transpose(0, 1).reshape(Hkv, -1, D)[:, :p + n] for t in "kv")
        unseen = torch.ones(n, p + n, dtype=torch.bool, device="cuda").triu(p + 1)
        for h in range(Hq):
            x = s["q"][m:m + n, h * D:(h + 1) * D].double() @ K[h * Hkv // Hq].T.contiguous() / math.sqrt(D)
            x[unseen] = -math.inf
            total = torch.logsumexp(x, -1)
            out[m:m + n, h * D:(h + 1) * D] = torch.exp(x - total[:, None]) @ V[h * Hkv // Hq]
            lse[h, m:m + n] = total / math.log(2.0)
        m += n
    return (out, lse) if case["rows_hi"] else out


def _append_exact(case, s, rows, before, Hq, Hkv, D):
    page = case["page"]
    x = s["qkv"].double().view(-1, Hq + 2 * Hkv, D)
    half = case["rot"] // 2
    j = torch.arange(half, device=x.device)
    lo, hi_ = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + half)
    at = s["pos"].long()[s["row_seq"]] + s["row_at"]
    z = torch.view_as_complex(s["cs"].double().contiguous())[at][:, None]
    z = z * torch.complex(x[:, :Hq + Hkv, lo], x[:, :Hq + Hkv, hi_])
    x[:, :Hq + Hkv, lo], x[:, :Hq + Hkv, hi_] = z.real, z.imag
    table = s["table"].tolist()
    result = [x[:, :Hq].reshape(-1, Hq * D)]
    for name, first in (("k", Hq), ("v", Hq + Hkv)):
        codes, exps = s[name + "p"].double(), s[name + "exp"].double()
        m = 0
        for b, (n, p) in enumerate(zip(rows, before)):
            while n > 0:
                pg, o = table[b][p // page], p % page
                take = min(n, page - o)
                t = x[m:m + take, first:first + Hkv].transpose(0, 1)
                k = torch.ceil(torch.log2(t.abs().amax((1, 2)) / 448))
                k = torch.maximum(k, exps[pg]) if o else k
                codes[pg, :, :o] *= 2.0 ** (exps[pg] - k)[:, None, None]
                codes[pg, :, o:o + take] = t * 2.0 ** -k[:, None, None]
                exps[pg] = k
                m, p, n = m + take, p + take, n - take
        result += [codes]
    return (*result, None, None)
