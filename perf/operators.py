"""The operators of a serving step over a paged KV cache: their cases, inputs, plain forms, least work and 64-bit results.

kind "tables"  block tables and slot maps of a step from the requests' lengths and new tokens: pages from a free stack
kind "write"   per-head q/k norm (optional), rotary embedding, keys and values into their pages
kind "attn"    causal attention of every request's new tokens over its pages (one token, a few, or a chunk of a prompt)
kind "logits"  penalties for repeated tokens, biases, grammar masks, and the arg-max of what is left

A batch is `chunks` requests with about `new` new tokens each (from half of that to all of it) and `singles` with one; before
them `context` tokens (again from half to all) are in the cache.  The lengths follow from the case, the contents from the seed.
"""
import torch

own = False

NEG = float("-inf")


def listed():
    return [
        # the tables of a decode step of forty sequences (the size of a lock-step batch): launch and latency
        {"name": "tables 40 singles", "kind": "tables", "chunks": 0, "new": 0, "singles": 40, "context": 300, "page": 16, "pad": 24},
        # a large server's step: chunks of prompts beside decoding requests, padded to the captured row count
        {"name": "tables 16k rows", "kind": "tables", "chunks": 12, "new": 1800, "singles": 500, "context": 4000, "page": 64, "pad": 333},
        # 16 / 8 heads of 128 (the 1B-class decoder): the rows of a decode step
        {"name": "write 40 rows", "kind": "write", "chunks": 0, "new": 0, "singles": 40, "context": 300, "page": 16, "hq": 16, "hkv": 8,
         "d": 128, "rot": 128, "norm": False},
        # 24 / 4 heads of 256 with q/k norms and a rotary part of 64 (the hybrid decoder's attention): chunks of prompts
        {"name": "write 8k rows norm", "kind": "write", "chunks": 5, "new": 2048, "singles": 17, "context": 1000, "page": 64, "hq": 24,
         "hkv": 4, "d": 256, "rot": 64, "norm": True},
        # one sequence of the 1B-class decoder behind a prompt of about a thousand tokens: latency
        {"name": "attn single 1100", "kind": "attn", "chunks": 0, "new": 0, "singles": 1, "context": 1100, "page": 16, "hq": 16, "hkv": 8,
         "d": 128, "pad": 0},
        # a batch of decoding requests of different lengths: bound by the cache's bytes
        {"name": "attn 64 singles", "kind": "attn", "chunks": 0, "new": 0, "singles": 64, "context": 6000, "page": 64, "hq": 16, "hkv": 8,
         "d": 128, "pad": 0},
        # drafts of a few tokens under verification, 24 / 4 heads of 256
        {"name": "attn 16 drafts d256", "kind": "attn", "chunks": 16, "new": 5, "singles": 0, "context": 2500, "page": 32, "hq": 24, "hkv": 4,
         "d": 256, "pad": 7},
        # a step that mixes chunks of prompts with decoding requests, heads of 64, rows and pages that end inside tiles
        {"name": "attn mixed d64", "kind": "attn", "chunks": 3, "new": 333, "singles": 29, "context": 2000, "page": 16, "hq": 32, "hkv": 8,
         "d": 64, "pad": 40},
        # a chunk of a long prompt of the 1B-class decoder (a pass takes 2048 rows): bound by the tensor core
        {"name": "attn chunk 2048", "kind": "attn", "chunks": 1, "new": 2048, "singles": 0, "context": 12000, "page": 64, "hq": 16, "hkv": 8,
         "d": 128, "pad": 0},
        # the 1B-class decoder's vocabulary, one sequence, logits as the head's product leaves them
        {"name": "logits 1 bf16", "kind": "logits", "rows": 1, "vocab": 73448, "history": 1100, "bias": 0, "masks": 0, "f32": False},
        # an odd batch of fp32 logits, some requests under a grammar
        {"name": "logits 17 f32", "kind": "logits", "rows": 17, "vocab": 73448, "history": 500, "bias": 40, "masks": 5, "f32": True},
        # the hybrid decoder's vocabulary, a large batch with long histories
        {"name": "logits 64 bf16", "kind": "logits", "rows": 64, "vocab": 151936, "history": 4000, "bias": 300, "masks": 64, "f32": False},
    ]


def _log(rng, lo, hi):
    """a whole number spread evenly over the logarithm of [lo, hi]"""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["tables", "write", "attn", "attn", "attn", "logits"])
    if kind == "logits":
        rows = _log(rng, 1, 64)
        return {"kind": kind, "rows": rows, "vocab": _log(rng, 8000, 151936), "history": _log(rng, 1, 4000), "bias": rng.choice([0, _log(rng, 1, 300)]),
                "masks": rng.choice([0, rng.randint(1, rows)]), "f32": rng.random() < 0.3}
    style = rng.choice(["singles", "drafts", "chunks", "mixed"])
    c = {"kind": kind, "chunks": {"singles": 0, "drafts": rng.randint(1, 24), "chunks": rng.randint(1, 2), "mixed": rng.randint(1, 4)}[style],
         "new": {"singles": 0, "drafts": rng.randint(2, 16), "chunks": _log(rng, 17, 1000), "mixed": _log(rng, 17, 500)}[style],
         "singles": {"singles": _log(rng, 1, 64), "drafts": 0, "chunks": 0, "mixed": rng.randint(1, 32)}[style],
         "context": _log(rng, 1, 5000 if style != "mixed" else 2000), "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "tables":
        return {**c, "pad": rng.choice([0, rng.randint(1, 64)])}
    c["d"] = rng.choice([64, 128, 128, 256])
    c["hkv"] = rng.choice([1, 2, 4, 8] if c["d"] < 256 else [1, 2, 4])
    c["hq"] = c["hkv"] * rng.choice([g for g in (1, 2, 3, 4, 6, 8) if g * c["hkv"] <= 24])
    if kind == "attn":
        return {**c, "pad": rng.choice([0, rng.randint(1, 64)])}
    norm = rng.random() < 0.5
    return {**c, "rot": rng.choice([c["d"], 64]), "norm": norm}


# ------------------------------------------------------------------------------------------------ lengths of a batch
def _lengths(case):
    """(new tokens, tokens before them) of every request; chunks lie among the singles"""
    n = case["chunks"] + case["singles"]
    new = [case["new"] - (i * (case["new"] // 2)) // max(1, case["chunks"] - 1) for i in range(case["chunks"])] + [1] * case["singles"]
    order = sorted(range(n), key=lambda i: (i * 7919 + 13) % 10007)
    ctx = [case["context"] - (i * 5 % n * (case["context"] // 2)) // max(1, n - 1) for i in range(n)]
    return [new[i] for i in order], ctx


def _pages_of(case):
    new, ctx = _lengths(case)
    p = case["page"]
    return [-(-(a + b) // p) for a, b in zip(new, ctx)]


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "logits":
        return _prepare_logits(case, gen)
    rnd = lambda *shape: torch.randn(*shape, generator=gen, device="cuda").bfloat16()  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    new, ctx = _lengths(case)
    page, rows = case["page"], sum(new)
    need = _pages_of(case)
    n_pages, width = sum(need) + 7, max(need) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    s = {"case": case, "page": page, "rows": rows + case.get("pad", 0), "max_q": max(new)}
    if case["kind"] == "tables":
        have = [-(-c // page) for c in ctx]
        s.update(q_len=i32(new), length=i32(ctx), table=_table(order, have, width), n_free=i32([n_pages - sum(have)]))
        s["free"] = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        s["free"][:n_pages - sum(have)] = order[sum(have):]
        if own:
            from ixrun_b200 import paged

            s["out"] = paged.PageStep.empty(len(new), s["rows"], "cuda")
        return s
    table = _table(order, need, width)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    s.update(hq=hq, hkv=hkv, d=d)
    if case["kind"] == "write":
        req = torch.repeat_interleave(torch.arange(len(new), device="cuda"), i32(new).long())
        start = i32(new).long().cumsum(0) - i32(new)
        pos = (torch.arange(rows, device="cuda") - start[req] + i32(ctx)[req])
        slot = table[req, pos // page].long() * page + pos % page
        half = case["rot"] // 2
        ang = torch.arange(max(a + b for a, b in zip(new, ctx)), dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
        qkv = rnd(rows, (hq + 2 * hkv) * d)                        # a fused projection: q, k and v are column slices of it
        s.update(pos=pos.int(), slot=slot.int(), cos=ang.cos().float().cuda(), sin=ang.sin().float().cuda(), q=qkv[:, :hq * d],
                 k=qkv[:, hq * d:(hq + hkv) * d], v=qkv[:, (hq + hkv) * d:], k_pages=rnd(n_pages, page, hkv, d), v_pages=rnd(n_pages, page, hkv, d),
                 q_norm=None, k_norm=None, out=torch.zeros(rows, hq * d, dtype=torch.bfloat16, device="cuda"))
        if case["norm"]:
            s.update(q_norm=(1 + 0.1 * rnd(d).float()).bfloat16(), k_norm=(1 + 0.1 * rnd(d).float()).bfloat16())
        return s
    # keys with a part that all of a head's keys share, and some that fit a query better than others: scores of a few units
    s.update(q=rnd(s["rows"], hq * d) * 1.5, k_pages=rnd(n_pages, page, hkv, d), v_pages=rnd(n_pages, page, hkv, d), table=table,
             length=i32([a + b for a, b in zip(new, ctx)]), cu_rows=i32([sum(new[:i]) for i in range(len(new) + 1)]),
             out=torch.zeros(s["rows"], hq * d, dtype=torch.bfloat16, device="cuda"))
    s["k_pages"] += 0.5 * rnd(1, 1, hkv, d)
    if own:
        from ixrun_b200 import paged

        s["attn"] = paged.AttnPaged(hq, hkv, d, "cuda")
    return s


def _table(order, need, width):
    """[requests, width] page numbers: request r has the first need[r] entries of its row, the rest are -1"""
    t = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    held = torch.tensor(need, device="cuda")[:, None] > torch.arange(width, device="cuda")
    t[held] = order[:sum(need)]
    return t


def _prepare_logits(case, gen):
    b, v, n = case["rows"], case["vocab"], case["history"]
    s = {"case": case}
    x = torch.randn(b, v, generator=gen, device="cuda") * 2
    # text repeats itself: tokens by a skewed distribution, from half of the history's length to all of it, a third of it prompt
    s["history"] = (v * torch.rand(b, n, generator=gen, device="cuda") ** 6).to(torch.int32).clamp_(max=v - 1)
    total = (n * (0.5 + 0.5 * torch.rand(b, generator=gen, device="cuda"))).int().clamp_(min=1)
    s["n_tokens"], s["n_prompt"] = total, total // 3
    x.scatter_add_(1, s["history"][:, :64].long(), torch.full((b, min(64, n)), 4.0, device="cuda"))     # what was said is likely again
    s["logits"] = x if case["f32"] else x.bfloat16()
    u = torch.rand(3, b, generator=gen, device="cuda")
    s["repetition"], s["presence"], s["frequency"] = 1 + 0.5 * u[0], u[1] * 1.5 - 0.25, u[2] * 0.8
    s["bias_ids"] = s["bias_values"] = s["mask"] = s["mask_row"] = None
    if case["bias"]:
        ids = torch.randint(-1, v, (b, case["bias"]), generator=gen, device="cuda", dtype=torch.int32)     # -1: no entry
        ids[:, -1] = ids[:, 0]                                       # a token named twice: the later entry counts
        s["bias_ids"], s["bias_values"] = ids, torch.randn(b, case["bias"], generator=gen, device="cuda") * 3
    if case["masks"]:
        words = -(-v // 32)
        bits = torch.randint(-2**31, 2**31 - 1, (4, case["masks"], words), generator=gen, device="cuda", dtype=torch.int32)
        s["mask"] = bits[0] & bits[1] & bits[2] & bits[3]            # a grammar allows few tokens
        s["mask_row"] = torch.where(torch.arange(b, device="cuda") < case["masks"], torch.arange(b, device="cuda"), -1).int()
        s["mask_row"] = s["mask_row"][torch.randperm(b, generator=gen, device="cuda")].contiguous()
    s["out"], s["token"] = torch.empty(b, v, device="cuda"), torch.empty(b, dtype=torch.long, device="cuda")
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    kind = s["case"]["kind"]
    if own:
        from ixrun_b200 import logits, paged

        if kind == "tables":
            st = paged.page_step(s["q_len"], s["length"], s["table"], s["free"], s["n_free"], s["page"], s["rows"], out=s["out"])
            return {"table": s["table"], "cu_rows": st.cu_rows, "length": st.length, "n_free": st.n_free, "slot": st.slot, "pos": st.pos,
                    "owner": st.owner, "status": st.status}
        if kind == "write":
            paged.rope_kv_paged(s["q"], s["k"], s["v"], s["pos"], s["slot"], s["k_pages"], s["v_pages"], s["cos"], s["sin"], s["hq"],
                                s["hkv"], s["d"], rot_dim=s["case"]["rot"], q_norm=s["q_norm"], k_norm=s["k_norm"], out=s["out"])
            return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if kind == "attn":
            return s["attn"](s["q"], s["k_pages"], s["v_pages"], s["table"], s["length"], s["cu_rows"], max_q=s["max_q"], out=s["out"])
        logits.apply_rules(s["logits"], s["history"], s["n_tokens"], s["n_prompt"], repetition=s["repetition"], presence=s["presence"],
                           frequency=s["frequency"], bias_ids=s["bias_ids"], bias_values=s["bias_values"], mask=s["mask"],
                           mask_row=s["mask_row"], out=s["out"], token=s["token"])
        return {"logits": s["out"], "token": s["token"]}
    return {"tables": _plain_tables, "write": _plain_write, "attn": _plain_attn, "logits": _plain_logits}[kind](s)


def _plain_tables(s):
    page, rows, q, n, table = s["page"], s["rows"], s["q_len"].long(), s["length"].long(), s["table"]
    have, total = (n + page - 1) // page, n + q
    need = (total + page - 1) // page
    cu = torch.nn.functional.pad(q.cumsum(0), (1, 0))
    first = (need - have).cumsum(0) - (need - have)                  # pages taken by the requests before
    b = torch.arange(table.shape[1], device="cuda")
    fits = ((need - have).sum() <= s["n_free"]) & (cu[-1] <= rows) & (need.max() <= table.shape[1])
    fresh = (b >= have[:, None]) & (b < need[:, None]) & fits
    at = (s["n_free"] - 1 - first[:, None] - (b - have[:, None])).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(fresh, s["free"][at], table))
    t = torch.arange(rows, device="cuda")
    live = (t < cu[-1]) & fits
    r = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=q.numel() - 1)
    pos = n[r] + t - cu[r]
    slot = table[r, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    status = torch.cat([(~fits).long(), (need - have).sum().view(1)])
    return {"table": table, "cu_rows": (cu * fits).int(), "length": torch.where(fits, total, n).int(),
            "n_free": (s["n_free"] - (need - have).sum() * fits).int(), "slot": torch.where(live, slot, -1).int(),
            "pos": torch.where(live, pos, 0).int(), "owner": torch.where(live, r, -1).int(), "status": status.int()}


def _plain_write(s):
    hq, hkv, d, rot = s["hq"], s["hkv"], s["d"], s["case"]["rot"]
    c, sn = s["cos"][s["pos"].long()][:, None], s["sin"][s["pos"].long()][:, None]

    def turned(x, heads, w):
        x = x.float().view(x.shape[0], heads, d)
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        return torch.cat([a * c - b * sn, b * c + a * sn, x[..., rot:]], -1).bfloat16()

    at = s["slot"].long()
    s["k_pages"].view(-1, hkv, d)[at] = turned(s["k"], hkv, s["k_norm"])
    s["v_pages"].view(-1, hkv, d)[at] = s["v"].reshape(-1, hkv, d)
    return {"q": turned(s["q"], hq, s["q_norm"]).view(-1, hq * d), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_attn(s):
    """every request padded to the longest: scores [requests, kv heads, group * new, keys]"""
    hq, hkv, d, page = s["hq"], s["hkv"], s["d"], s["page"]
    g, r, new, n = hq // hkv, s["length"].numel(), s["max_q"], s["length"].long()
    cu = s["cu_rows"].long()
    q_len = cu[1:] - cu[:-1]
    j = torch.arange(new, device="cuda")
    row = (cu[:-1, None] + j).clamp(max=s["rows"] - 1)               # [requests, new]
    live = j < q_len[:, None]
    width = min(s["table"].shape[1], max(_pages_of(s["case"])))
    pages = s["table"][:, :width].long().clamp(min=0)
    k = s["k_pages"][pages].view(r, width * page, hkv, d).permute(0, 2, 3, 1).float()
    v = s["v_pages"][pages].view(r, width * page, hkv, d).permute(0, 2, 1, 3).float()
    q = s["q"][row].view(r, new, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(r, hkv, new * g, d).float()
    score = (q @ k).mul_(d ** -0.5).view(r, hkv, new, g, width * page)
    seen = torch.arange(width * page, device="cuda") <= (n - q_len)[:, None, None] + j[:, None]
    score.masked_fill_(~seen[:, None, :, None], NEG)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    score = score.div_(score.sum(-1, keepdim=True)).view(r, hkv, new * g, width * page)
    o = (score @ v).view(r, hkv, new, g, d).permute(0, 2, 1, 3, 4).reshape(r, new, hq * d).bfloat16()
    s["out"][row[live]] = o[live]
    return s["out"]


def _plain_logits(s):
    x = s["logits"].float()
    b, v = x.shape
    h, t = s["history"].long(), torch.arange(s["history"].shape[1], device="cuda")
    made = (t >= s["n_prompt"][:, None]) & (t < s["n_tokens"][:, None])
    count = torch.zeros(b, v, device="cuda").scatter_add_(1, h, made.float())
    seen = torch.zeros(b, v, device="cuda").scatter_add_(1, h, (t < s["n_tokens"][:, None]).float()) > 0
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if s["bias_ids"] is not None:
        ids, e = s["bias_ids"].long(), torch.arange(s["bias_ids"].shape[1], device="cuda")
        last = torch.full((b, v + 1), -1, dtype=torch.long, device="cuda")
        last.scatter_reduce_(1, torch.where(ids < 0, v, ids), e.expand_as(ids), "amax")
        last = last[:, :v]
        x = torch.where(last >= 0, x + s["bias_values"].gather(1, last.clamp(min=0)), x)
    if s["mask"] is not None:
        bit = torch.arange(v, device="cuda")
        allowed = (s["mask"][s["mask_row"].long().clamp(min=0)][:, bit // 32] >> (bit % 32)) & 1
        x = torch.where((allowed == 0) & (s["mask_row"] >= 0)[:, None], NEG, x)
    return {"logits": x, "token": torch.where(x == x.amax(-1, keepdim=True), torch.arange(v, device="cuda"), v).amin(-1)}


# ------------------------------------------------------------------------------------------------ least work
def work(case):
    if case["kind"] == "logits":
        b, v = case["rows"], case["vocab"]
        return {"bytes": b * v * ((4 if case["f32"] else 2) + 4) + case["masks"] * -(-v // 32) * 4 + b * case["history"] * 3 + b * case["bias"] * 8,
                "flops": b * v}
    new, ctx = _lengths(case)
    rows, n = sum(new), len(new)
    if case["kind"] == "tables":
        fresh = sum(_pages_of(case)) - sum(-(-c // case["page"]) for c in ctx)
        return {"bytes": 12 * (rows + case["pad"]) + 16 * n + 8 * fresh, "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "write":
        return {"bytes": rows * ((hq + 2 * hkv) * d * 4 + case["rot"] * 4 + 8), "flops": rows * (hq + hkv) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}
    keys = sum(a + b for a, b in zip(new, ctx))
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, ctx))
    return {"bytes": keys * hkv * d * 4 + rows * hq * d * 4, "flops": 4 * d * hq * pairs}


# ------------------------------------------------------------------------------------------------ 64-bit results
def exact(case, seed):
    if case["kind"] == "tables":
        return None                                                 # whole numbers only
    s = prepare(case, seed)
    if case["kind"] == "logits":
        return _exact_logits(s)
    hq, hkv, d = s["hq"], s["hkv"], s["d"]
    if case["kind"] == "write":
        half = case["rot"] // 2
        z = torch.complex(s["cos"].double(), s["sin"].double())[s["pos"].long()].unsqueeze(1)

        def turned(x, w):
            x = x.double().reshape(x.shape[0], -1, d)
            if w is not None:
                x = x / (x.square().sum(-1, keepdim=True) / d + 1e-6).sqrt() * w.double()
            y = torch.complex(x[..., :half], x[..., half:2 * half]) * z
            return torch.cat([y.real, y.imag, x[..., 2 * half:]], -1)

        k, v = s["k_pages"].double().flatten(0, 1), s["v_pages"].double().flatten(0, 1)
        k.index_copy_(0, s["slot"].long(), turned(s["k"], s["k_norm"]))
        v.index_copy_(0, s["slot"].long(), s["v"].double().reshape(-1, hkv, d))
        return {"q": turned(s["q"], s["q_norm"]).flatten(1), "k_pages": k.view(s["k_pages"].shape), "v_pages": v.view(s["v_pages"].shape)}
    out = torch.zeros(s["rows"], hkv, hq // hkv, d, dtype=torch.float64, device="cuda")
    cu, length = s["cu_rows"].tolist(), s["length"].tolist()
    for r, n in enumerate(length):                                  # one request and KV head after the other
        a, b = cu[r], cu[r + 1]
        pages = s["table"][r, :-(-n // s["page"])].long()
        for h in range(hkv):
            k, v = (t[pages, :, h].flatten(0, 1)[:n].double() for t in (s["k_pages"], s["v_pages"]))
            for g in range(hq // hkv):
                q = s["q"][a:b].view(b - a, hkv, hq // hkv, d)[:, h, g].double()
                sc = torch.tril(torch.ones(b - a, n, dtype=torch.bool, device="cuda"), diagonal=n - (b - a))
                p = torch.softmax((q @ k.T / d ** 0.5).masked_fill(~sc, NEG), -1)
                out[a:b, h, g] = p @ v
    return out.flatten(1)


def _exact_logits(s):
    x = s["logits"].double()
    b, v = x.shape
    for i in range(b):
        h, n, p = s["history"][i].long(), int(s["n_tokens"][i]), int(s["n_prompt"][i])
        said, made = h[:n].unique(), torch.bincount(h[p:n], minlength=v)
        rho = float(s["repetition"][i])
        y = x[i, said]
        x[i, said] = torch.maximum(y, torch.zeros_like(y)) / rho + torch.minimum(y, torch.zeros_like(y)) * rho
        x[i] -= float(s["frequency"][i]) * made + float(s["presence"][i]) * (made > 0)
        if s["bias_ids"] is not None:
            wanted = {t: w for t, w in zip(s["bias_ids"][i].tolist(), s["bias_values"][i].tolist()) if t >= 0}
            x[i, torch.tensor(list(wanted), device="cuda")] += torch.tensor(list(wanted.values()), dtype=torch.float64, device="cuda")
        if s["mask"] is not None and int(s["mask_row"][i]) >= 0:
            w = s["mask"][int(s["mask_row"][i])].long() & 0xFFFFFFFF
            x[i][((w[:, None] >> torch.arange(32, device="cuda")) & 1).flatten()[:v] == 0] = NEG
    return {"logits": x, "token": None}                             # (the arg-max of the rounded logits: no 64-bit value of its own)
