"""What is measured of the serving operators: page planning, the 8-bit paged KV cache's write and read-back, attention
over that cache, and token sampling.

A serving step of many requests runs, once, ``plan_step`` (pages, slots and positions of the step's new tokens from the
request lengths), then per layer ``cache_write`` (RoPE, the new K/V into 8-bit pages with one scale per page and KV
head) and ``attn_paged``, and at the end ``sample_tokens``.  ``run`` is one pass through one of them: with ``own``
through the framework's entry points, otherwise through plain torch operations.

Cases are dicts with an ``op`` of "plan", "write", "attend" or "sample".  Request lengths follow from the case alone
(so that ``work`` knows them); the seed permutes them and makes every value.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one decode step of 64 requests of a chat server: every request adds one token
        dict(name="plan decode 64", op="plan", requests=64, page=64, lo=1, hi=2047, new_lo=1, new_hi=1, idle=0),
        # a mixed step: most requests decode or wait, some bring prompts of up to 2048 tokens; small pages
        dict(name="plan mixed 256", op="plan", requests=256, page=16, lo=1, hi=8191, new_lo=1, new_hi=2048, idle=19),
        # the new token of 64 decoding requests in one layer of a 28/4-head model, RoPE included
        dict(name="write decode 64", op="write", dtype="bf16", requests=64, q_heads=28, kv_heads=4, head_dim=128,
             page=64, lo=1, hi=2047, new_lo=1, new_hi=1, rope=True),
        # a prefill's keys and values (already rotated by the model) go into the cache: about 16k tokens
        dict(name="write prefill 16k", op="write", dtype="bf16", requests=8, q_heads=24, kv_heads=8, head_dim=128,
             page=64, lo=0, hi=0, new_lo=1021, new_hi=3081, rope=False),
        # a few short requests of a small model continue at odd places in 16-token pages
        dict(name="write ragged 5 f16", op="write", dtype="f16", requests=5, q_heads=4, kv_heads=2, head_dim=64,
             page=16, lo=3, hi=90, new_lo=1, new_hi=37, rope=True),
        # the smallest call: one request of a small model, latency only
        dict(name="attend one f16", op="attend", dtype="f16", requests=1, q_heads=4, kv_heads=2, head_dim=64, page=16,
             lo=513, hi=513, new_lo=1, new_hi=1),
        # a decode step of 64 requests of very different lengths, 7 query heads per KV head
        dict(name="attend decode 64", op="attend", dtype="bf16", requests=64, q_heads=28, kv_heads=4, head_dim=128,
             page=64, lo=61, hi=4096, new_lo=1, new_hi=1),
        # two requests over long documents
        dict(name="attend long 2", op="attend", dtype="bf16", requests=2, q_heads=24, kv_heads=8, head_dim=128,
             page=128, lo=98303, hi=131071, new_lo=1, new_hi=1),
        # drafted tokens are verified: up to four new tokens per request, 5 query heads per KV head
        dict(name="attend drafts 16", op="attend", dtype="bf16", requests=16, q_heads=40, kv_heads=8, head_dim=128,
             page=32, lo=509, hi=8190, new_lo=1, new_hi=4),
        # one request of a small model, odd vocabulary (rows off the 16-byte grid)
        dict(name="sample one f16", op="sample", dtype="f16", rows=1, vocab=32003, temperature=0.7, top_k=50,
             top_p=0.9, min_p=0.0, masked=0.0),
        # 16 requests with the plain temperature: the whole vocabulary stays in
        dict(name="sample 16", op="sample", dtype="bf16", rows=16, vocab=128256, temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.0, masked=0.0),
        # a large batch with every filter on and a grammar that masks half of the vocabulary
        dict(name="sample 192 masked", op="sample", dtype="bf16", rows=192, vocab=152064, temperature=0.9, top_k=2000,
             top_p=0.95, min_p=0.01, masked=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("plan", "write", "attend", "attend", "sample"))
    dtype = rng.choice(("bf16", "f16"))
    page = rng.choice((16, 32, 64, 128))
    if op == "plan":
        most = _log_int(rng, 1, 2048)
        return dict(op=op, requests=_log_int(rng, 1, 256), page=page, lo=_log_int(rng, 1, 500),
                    hi=_log_int(rng, 500, 8191), new_lo=1, new_hi=most, idle=rng.choice((0, 0, 3, 11)))
    if op == "sample":
        return dict(op=op, dtype=dtype, rows=_log_int(rng, 1, 192), vocab=_log_int(rng, 1000, 152064),
                    temperature=rng.choice((0.5, 0.8, 1.0, 1.3)), top_k=rng.choice((0, 1, 20, 400)),
                    top_p=rng.choice((1.0, 0.95, 0.6)), min_p=rng.choice((0.0, 0.02)),
                    masked=rng.choice((0.0, 0.0, 0.3, 0.9)))
    head_dim = rng.choice((64, 128))
    kv_heads = rng.choice((1, 2, 4, 8))
    q_heads = kv_heads * rng.choice((1, 3, 4, 5, 7, 8))
    requests = _log_int(rng, 1, 64)
    if op == "write":
        most = max(1, min(3000, 16384 // requests))
        return dict(op=op, dtype=dtype, requests=requests, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                    page=page, lo=rng.choice((0, 5, 77)), hi=_log_int(rng, 100, 2000), new_lo=1,
                    new_hi=_log_int(rng, 1, most), rope=rng.random() < 0.5)
    most = rng.choice((1, 1, 2, 4))
    hi = _log_int(rng, 40, max(41, (196608 if most == 1 else 49152) // requests))
    return dict(op=op, dtype=dtype, requests=requests, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
                lo=max(4, int(hi * rng.uniform(0.1, 1.0))), hi=max(4, hi), new_lo=1, new_hi=most)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spaced."""
    return [lo + (hi - lo) * i // (n - 1) for i in range(n)] if n > 1 else [hi]


def _lengths(case):
    """(tokens cached before the step, new tokens of the step) of each request, before the seed permutes them.  An
    attention case's ``lo``/``hi`` count the step's own tokens too."""
    n = case["requests"]
    before = _spread(case["lo"], case["hi"], n)
    new = _spread(case["new_lo"], case["new_hi"], n)
    new = new[n // 2:] + new[:n // 2]  # long and short requests bring few and many tokens alike
    if case["op"] == "plan":
        if case["idle"]:  # every so many requests wait or are empty slots; most of the others decode
            new = [0 if i % case["idle"] == 1 else (v if i % 4 == 0 else 1) for i, v in enumerate(new)]
    if case["op"] == "attend":
        before = [b - w for b, w in zip(before, new)]
    return before, new


def work(case):
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        return {"bytes": rows * (2 * vocab + 4 + 8 + 4 + 16), "flops": 4 * rows * vocab}
    before, new = _lengths(case)
    page, total = case["page"], sum(new)
    if case["op"] == "plan":
        fresh = sum(-(-(b + w) // page) - -(-b // page) for b, w in zip(before, new))
        return {"bytes": case["requests"] * 16 + total * 16 + fresh * 8, "flops": 0}
    hq, hk, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "write":
        # new rows in and their codes out; the touched pages' codes in and values out (the read-back); q and angles
        pages = sum((b + w - 1) // page - b // page + 1 for b, w in zip(before, new) if w)
        rot = (2 * hq * d * 2 + 2 * d * 2) * total if case["rope"] else 0
        return {"bytes": 2 * total * hk * d * 3 + 2 * pages * hk * (page * d * 3 + 8) + rot, "flops": 8 * total * hk * d}
    keys = sum(b + w for b, w in zip(before, new))
    pairs = sum(w * b + w * (w + 1) // 2 for b, w in zip(before, new))
    pages = sum(-(-(b + w) // page) for b, w in zip(before, new))
    return {"bytes": 2 * keys * hk * d + pages * (8 * hk + 4) + 2 * total * hq * d * 2, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------------------------------------ inputs
def _pages(case, gen, dev):
    """The pool's state before the step: lengths, block table and the stack of free pages."""
    before, new = _lengths(case)
    order = torch.randperm(len(before), generator=gen, device=dev)
    before = torch.tensor(before, device=dev)[order]
    new = torch.tensor(new, device=dev)[order]
    page = case["page"]
    used = (before + page - 1) // page
    need = (before + new + page - 1) // page
    spare = 3
    total = int(need.sum()) + spare
    width = int(need.max()) + 1
    ids = torch.randperm(total, generator=gen, device=dev)
    table = torch.full((len(before), width), -1, dtype=torch.int64, device=dev)
    col = torch.arange(width, device=dev)
    held = col < used[:, None]
    owned = int(used.sum())
    table[held] = ids[:owned]
    free = torch.cat([ids[owned:], torch.zeros(owned, dtype=torch.int64, device=dev)])
    return dict(before=before, new=new, table=table.int(), free=free.int(), free_count=total - owned, pages=total,
                width=width)


def _touched(st, page):
    """Of the step: slot of every new token, the touched pages in request order, the page index of every new token and
    how many tokens each touched page held before."""
    before, new, dev = st["before"], st["new"], st["before"].device
    req = torch.repeat_interleave(torch.arange(len(new), device=dev), new)
    cu = torch.cumsum(new, 0) - new
    pos = before[req] + torch.arange(len(req), device=dev) - cu[req]
    # the table after the step: fresh pages are popped from the top of the stack, in request order
    need = (before + new + page - 1) // page
    used = (before + page - 1) // page
    col = torch.arange(st["width"], device=dev)
    fresh = (col >= used[:, None]) & (col < need[:, None])
    table = st["table"].long()
    count = int(fresh.sum())
    table[fresh] = st["free"].long()[st["free_count"] - 1 - torch.arange(count, device=dev)]
    slots = table[req, pos // page] * page + pos % page
    touched = (col >= (before // page)[:, None]) & (col < need[:, None]) & (new > 0)[:, None]
    key = req * st["width"] + pos // page
    keys, tok_item = torch.unique(key, sorted=True, return_inverse=True)
    exist = (before[keys // st["width"]] - (keys % st["width"]) * page).clamp(min=0)
    return dict(slots=slots, positions=pos, req=req, table_after=table, touched=table[touched], tok_item=tok_item,
                exist=exist)


def _own_plan(case, st, tokens):
    import tilequant_b200 as tq

    pool = tq.PagePool(st["pages"], len(st["new"]), st["width"] * case["page"], page_size=case["page"],
                       device=st["before"].device)
    pool.lengths.copy_(st["before"])
    pool.block_table.copy_(st["table"])
    pool.free_pages.copy_(st["free"])
    pool.free_count.fill_(st["free_count"])
    plan = tq.StepPlan(pool, tokens, q_heads=case.get("q_heads", 8), kv_heads=case.get("kv_heads", 8),
                       head_dim=case.get("head_dim", 128), max_new=case["new_hi"])
    return pool, plan


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a model's logits: a broad body, a few strong candidates per row, everything in 16 bits (so many are equal)
        logits = normal(rows, vocab) * 2.0 - 1.0
        best = torch.randint(vocab, (rows, 24), generator=gen, device=dev)
        logits.scatter_add_(1, best, normal(rows, 24).abs() * 5)
        if case["masked"]:
            off = torch.rand(rows, vocab, generator=gen, device=dev) < case["masked"]
            logits = logits.masked_fill(off, -math.inf)
        full = torch.full((rows,), 1.0, device=dev)
        return dict(op="sample", logits=logits.to(DTYPES[case["dtype"]]),
                    uniform=torch.rand(rows, generator=gen, device=dev), temperature=full * case["temperature"],
                    top_k=torch.full((rows,), case["top_k"], dtype=torch.int32, device=dev),
                    top_p=full * case["top_p"], min_p=full * case["min_p"],
                    ids=torch.empty(rows, dtype=torch.int64, device=dev), logprobs=torch.empty(rows, device=dev))

    st = _pages(case, gen, dev)
    page = case["page"]
    if case["op"] == "plan":
        # captured steps have a fixed number of token rows: some rows behind the last token stay unused
        tokens = sum(_lengths(case)[1]) + 5
        st = dict(st, op="plan", page=page, tokens=tokens, new32=st["new"].int(), before32=st["before"].int())
        if own:
            pool, plan = _own_plan(case, st, tokens)
            st.update(pool=pool, plan=plan, lengths_out=torch.empty_like(pool.lengths),
                      count_out=torch.empty_like(pool.free_count))
        return st

    st.update(_touched(st, page))
    hq, hk, d, dtype = case["q_heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]]
    tokens = int(st["new"].sum())
    shape = (st["pages"], hk, page, d)
    # what the cache holds: codes of roughly normal keys and values; pages and places not in use hold leavings
    codes = [(normal(*shape) * 40).round_().clamp_(-127, 127).to(torch.int8) for _ in range(2)]
    scales = [0.02 * torch.exp(0.5 * normal(st["pages"], hk)) for _ in range(2)]
    st.update(op=case["op"], page=page, q_heads=hq, kv_heads=hk, head_dim=d, k_codes=codes[0], v_codes=codes[1],
              k_scale=scales[0], v_scale=scales[1])
    # the projections' stacked output, of which q, k and v are column ranges
    width = torch.exp(0.4 * normal(d))  # some channels are larger than others
    qkv = (normal(tokens, hq + 2 * hk, d) * width).to(dtype).reshape(tokens, -1)
    st.update(q=qkv[:, :hq * d], k=qkv[:, hq * d:(hq + hk) * d], v=qkv[:, (hq + hk) * d:], dtype=dtype,
              rope=bool(case.get("rope")))
    if st["rope"]:
        freq = 10000.0 ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        angle = st["positions"].double()[:, None] * freq
        angle = torch.cat([angle, angle], 1)
        st.update(cos=angle.cos().to(dtype), sin=angle.sin().to(dtype))
    st.update(page_ids=st["touched"].int(), most_new=int(st["new"].max()))
    if own:
        import tilequant_b200 as tq

        pool, plan = _own_plan(case, st, tokens)
        tq.plan_step(st["new"].int(), pool, plan)
        kv = tq.KVPages(st["pages"], hk, page, d, device=dev)
        kv.k.copy_(st["k_codes"])
        kv.v.copy_(st["v_codes"])
        kv.k_scale.copy_(st["k_scale"])
        kv.v_scale.copy_(st["v_scale"])
        st.update(pool=pool, plan=plan, kv=kv, k_codes=None, v_codes=None)
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"plan": _plan, "write": _write, "attend": _attend, "sample": _sample}[state["op"]](state)


def _plan(st):
    if own:
        import tilequant_b200 as tq

        pool, plan = st["pool"], st["plan"]
        tq.plan_step(st["new32"], pool, plan, lengths_out=st["lengths_out"], free_count_out=st["count_out"])
        return dict(table=pool.block_table, lengths=st["lengths_out"], free_count=st["count_out"], cu_new=plan.cu_new,
                    slots=plan.slots, positions=plan.positions)
    page, tokens = st["page"], st["tokens"]
    before, new, dev = st["before32"].long(), st["new32"].long(), st["table"].device
    after = before + new
    ends = torch.cumsum(new, 0)
    used, need = (before + page - 1) // page, (after + page - 1) // page
    first = torch.cumsum(need - used, 0) - (need - used)
    col = torch.arange(st["width"], device=dev)
    fresh = (col >= used[:, None]) & (col < need[:, None])
    nth = (first[:, None] + col - used[:, None]).clamp(0, st["pages"] - 1)
    taken = st["free"][(st["free_count"] - 1 - nth).clamp(min=0)]
    st["table"].copy_(torch.where(fresh, taken, st["table"]))
    row = torch.arange(tokens, device=dev)
    req = (row[:, None] >= ends).sum(1).clamp(max=len(new) - 1)
    pos = before[req] + row - (ends - new)[req]
    slots = st["table"][req, (pos // page).clamp(max=st["width"] - 1)].long() * page + pos % page
    there = row < ends[-1]
    cu = torch.cat([torch.zeros_like(ends[:1]), ends]).int()
    return dict(table=st["table"], lengths=after.int(), free_count=(st["free_count"] - (need - used).sum()).int()[None],
                cu_new=cu, slots=torch.where(there, slots, -1), positions=torch.where(there, pos, -1))


def _rotate(x, cos, sin):
    """The decoder's rotary embedding of [tokens, heads, D]: each product and the sum rounded to the 16-bit type."""
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    a = (x.float() * cos.float()[:, None]).to(x.dtype)
    b = (turned.float() * sin.float()[:, None]).to(x.dtype)
    return (a.float() + b.float()).to(x.dtype)


def _write_side(x, codes, scale, st):
    """New rows x [tokens, heads, D] into the touched pages of one side; those pages' values."""
    at, exist, page = st["touched"], st["exist"], st["page"]
    x = x.float()
    most = torch.zeros(len(at), x.shape[1], device=x.device)
    most.scatter_reduce_(0, st["tok_item"][:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
    old = torch.where(exist[:, None] > 0, scale[at], 0.0)
    s = torch.maximum(old, most / 127.0)
    ratio = torch.where(s > 0, old / s, 0.0)
    held = codes[at].float()
    keep = torch.arange(page, device=x.device) < exist[:, None]
    held = torch.where(keep[:, None, :, None], torch.round(held * ratio[:, :, None, None]), held)
    s_tok = s[st["tok_item"]][..., None]
    q = torch.where(s_tok > 0, torch.round(x / s_tok).clamp(-127, 127), 0.0)
    held[st["tok_item"], :, st["slots"] % page] = q
    codes[at] = held.to(torch.int8)
    scale[at] = s
    return (held * s[:, :, None, None]).to(st["dtype"])


def _write(st):
    hq, hk, d = st["q_heads"], st["kv_heads"], st["head_dim"]
    if own:
        import tilequant_b200 as tq

        if st["rope"]:
            q = tq.cache_write(st["k"], st["v"], st["kv"], st["plan"], q=st["q"], cos=st["cos"], sin=st["sin"])
        else:
            q = tq.cache_write(st["k"], st["v"], st["kv"], st["plan"])
        k, v = tq.read_pages(st["kv"], st["page_ids"], st["dtype"])
        return dict(q=q, k=k, v=v)
    k, q = st["k"].view(-1, hk, d), None
    if st["rope"]:
        k = _rotate(k, st["cos"], st["sin"])
        q = _rotate(st["q"].view(-1, hq, d), st["cos"], st["sin"]).view(-1, hq * d)
    return dict(q=q, k=_write_side(k, st["k_codes"], st["k_scale"], st),
                v=_write_side(st["v"].view(-1, hk, d), st["v_codes"], st["v_scale"], st))


def _attend(st):
    scale = st["head_dim"] ** -0.5
    if own:
        import tilequant_b200 as tq

        return tq.attn_paged(st["q"], st["kv"], st["plan"], scale)
    hq, hk, d, page, dev = st["q_heads"], st["kv_heads"], st["head_dim"], st["page"], st["q"].device
    before, new, table = st["before"], st["new"], st["table_after"].clamp(min=0)
    n, most, width = len(new), st["most_new"], table.shape[1]
    # queries as [request, KV head, new token and query head of the group, D], short requests padded
    row = (torch.cumsum(new, 0) - new)[:, None] + torch.arange(most, device=dev)
    there = torch.arange(most, device=dev) < new[:, None]
    q = st["q"].view(-1, hk, hq // hk, d)[row.clamp(max=st["q"].shape[0] - 1)].float()
    q = q.permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    # the pages' values as [request, KV head, key, D]
    k = (st["k_codes"][table].float() * st["k_scale"][table][..., None, None]).transpose(1, 2).reshape(n, hk, -1, d)
    s = q @ k.transpose(-1, -2) * scale
    del k
    key = torch.arange(width * page, device=dev)
    seen = key <= (before[:, None] + torch.arange(most, device=dev))[..., None]
    seen = seen[:, None, :, None].expand(-1, hk, -1, hq // hk, -1).reshape(n, hk, -1, width * page)
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = (st["v_codes"][table].float() * st["v_scale"][table][..., None, None]).transpose(1, 2).reshape(n, hk, -1, d)
    o = (p @ v).view(n, hk, most, hq // hk, d).transpose(1, 2)
    return o[there].reshape(-1, hq * d).to(st["dtype"])


def _sample(st):
    if own:
        import tilequant_b200 as tq

        return tq.sample_tokens(st["logits"], st["uniform"], temperature=st["temperature"], top_k=st["top_k"],
                                top_p=st["top_p"], min_p=st["min_p"], out=st["ids"], logprobs=st["logprobs"])
    # tokens in falling order, equal ones by index; every filter keeps a head of that order
    x, index = torch.sort(st["logits"].double(), dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / st["temperature"].double()[:, None])
    nth = torch.arange(x.shape[1], device=x.device)
    k = torch.where(st["top_k"] > 0, st["top_k"], x.shape[1])[:, None]
    w = torch.where(nth < k, w, 0.0)
    upto = torch.cumsum(w, 1)
    w = torch.where(upto - w < st["top_p"].double()[:, None] * upto[:, -1:], w, 0.0)
    w = torch.where(w >= st["min_p"].double()[:, None], w, 0.0)
    upto = torch.cumsum(w, 1)
    target = st["uniform"].double()[:, None] * upto[:, -1:]
    at = ((upto <= target) & (w > 0)).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    return index.gather(1, at)[:, 0], torch.log(w.gather(1, at) / upto[:, -1:])[:, 0].float()


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"plan": _exact_plan, "write": _exact_write, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](st)


def _exact_plan(st):
    """Request by request, page by page."""
    page, tokens = st["page"], st["tokens"]
    table, stack = st["table"].tolist(), st["free"].tolist()[:st["free_count"]]
    before, new = st["before"].tolist(), st["new"].tolist()
    slots, positions, cu, after = [], [], [0], []
    for row, b, w in zip(table, before, new):
        for p in range(b, b + w):
            if p % page == 0:
                row[p // page] = stack.pop()
            slots.append(row[p // page] * page + p % page)
            positions.append(p)
        cu.append(cu[-1] + w)
        after.append(b + w)
    pad = [-1] * (tokens - len(slots))
    i32 = torch.int32
    return dict(table=torch.tensor(table, dtype=i32), lengths=torch.tensor(after, dtype=i32),
                free_count=torch.tensor([len(stack)], dtype=i32), cu_new=torch.tensor(cu, dtype=i32),
                slots=torch.tensor(slots + pad), positions=torch.tensor(positions + pad))


def _exact_turn(x, cos, sin, dtype):
    """x [tokens, heads, D] turned by its angles; the 16-bit roundings of the decoder's operators are part of the
    definition."""
    x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
    h = x.shape[-1] // 2
    near, far = x[..., :h], x[..., h:]

    def r(t):
        return t.float().to(dtype).double()

    return torch.cat([r(r(near * cos[..., :h]) + r(-far * sin[..., :h])),
                      r(r(far * cos[..., h:]) + r(near * sin[..., h:]))], -1)


def _exact_write(st):
    """Page by page.  The scale of a page and the quotients that are rounded to codes are held in 32 bits by
    definition (a quotient of two 32-bit numbers taken in 64 bits and rounded to 32 is the 32-bit quotient)."""
    hk, d, page = st["kv_heads"], st["head_dim"], st["page"]
    k, v = st["k"].view(-1, hk, d).double(), st["v"].view(-1, hk, d).double()
    q = None
    if st["rope"]:
        k = _exact_turn(k, st["cos"], st["sin"], st["dtype"])
        q = _exact_turn(st["q"].view(-1, st["q_heads"], d), st["cos"], st["sin"], st["dtype"]).reshape(len(k), -1)
    items = len(st["touched"])
    counts = torch.bincount(st["tok_item"], minlength=items).tolist()
    pages, exist = st["touched"].tolist(), st["exist"].tolist()
    out = []
    for x, codes, scale in ((k, st["k_codes"], st["k_scale"]), (v, st["v_codes"], st["v_scale"])):
        values, t = [], 0
        for i in range(items):
            rows = x[t:t + counts[i]].transpose(0, 1)  # heads, tokens, D
            t += counts[i]
            here = codes[pages[i]].double()
            old = scale[pages[i]].double() if exist[i] else torch.zeros(hk, device=x.device, dtype=torch.float64)
            s = torch.maximum(old, (rows.abs().amax((1, 2)) / 127).float().double())
            if exist[i]:
                here[:, :exist[i]] = torch.round((here[:, :exist[i]] * (old / s).float().double()[:, None, None]).float()
                                                 .double())
            here[:, exist[i]:exist[i] + counts[i]] = torch.round((rows / s[:, None, None]).float().double())
            values.append(here * s[:, None, None])
        out.append(torch.stack(values))
    return dict(q=q, k=out[0], v=out[1])


def _exact_attend(st):
    """Request by request, one KV head at a time."""
    hq, hk, d, page = st["q_heads"], st["kv_heads"], st["head_dim"], st["page"]
    group, t, rows = hq // hk, 0, []
    for b, w, table in zip(st["before"].tolist(), st["new"].tolist(), st["table_after"]):
        n = b + w
        at = table[:-(-n // page)]
        q = st["q"][t:t + w].view(w, hk, group, d).double()
        t += w
        heads = []
        for h in range(hk):
            k = (st["k_codes"][at, h].double() * st["k_scale"][at, h].double()[:, None, None]).reshape(-1, d)[:n]
            v = (st["v_codes"][at, h].double() * st["v_scale"][at, h].double()[:, None, None]).reshape(-1, d)[:n]
            s = torch.einsum("wgd,nd->wgn", q[:, h], k) / math.sqrt(d)
            late = torch.arange(n, device=s.device) > b + torch.arange(w, device=s.device)[:, None]
            s = s.masked_fill(late[:, None], -math.inf)
            heads.append(torch.einsum("wgn,nd->wgd", torch.softmax(s, -1), v))
        rows.append(torch.stack(heads, 1).reshape(w, hq * d))
    return torch.cat(rows)


def _exact_sample(st):
    """Row by row on the host: the order by (logit falling, index rising), and sums from the smallest weight up where
    only a total is wanted."""
    import numpy as np

    ids, logs = [], []
    rows = st["logits"].double().cpu().numpy()
    for r, x in enumerate(rows):
        t, top_p, min_p, u = (float(st[n][r].double()) for n in ("temperature", "top_p", "min_p", "uniform"))
        order = np.lexsort((np.arange(len(x)), -x))
        order = order[np.isfinite(x[order])]
        w = np.exp((x[order] - x[order[0]]) / t).astype(np.longdouble)
        k = int(st["top_k"][r])
        if k > 0:
            w = w[:k]
        upto = np.cumsum(w)
        w = w[:int(np.searchsorted(upto, top_p * w[::-1].sum(), side="left")) + 1]
        w = w[w >= min_p]
        total = w[::-1].sum()
        at = min(int(np.searchsorted(np.cumsum(w), u * total, side="right")), len(w) - 1)
        ids.append(int(order[at]))
        logs.append(float(np.log(w[at] / total)))
    return torch.tensor(ids), torch.tensor(logs, dtype=torch.float64)
