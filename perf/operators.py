"""What the operators of paged serving are measured on: inputs, a plain form of each operator, and the calls a user makes.

Four operators that one scheduling step of a server runs one after another: the step's page tables and slot maps are
built from the requests' lengths (`plan`), the new keys and values join the pages (`append`), the new tokens read their
requests' pages (`attend`), and drafted tokens are held against the target's probabilities (`verify`).  With `own` false
`run` computes them from elementary torch operations, in 32 bits (64 where a sum decides between two tokens) and rounded
once; with `own` true it calls ava_b200.serving.
"""
import math
import random

import torch

own = False

DEV = "cuda"
FLOAT = {"f32": torch.float32, "bf16": torch.bfloat16}
NO_PAGES, NO_TABLE, BAD_LENGTH, NO_TOKENS = 1, 2, 4, 8


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 256 sequences: a page is crossed by one request in sixteen (latency: a few kilobytes of lists)
        dict(name="plan_decode_256", op="plan", rows=256, fresh=1, ctx=2048, page=16, trim=False),
        # a step that admits prompts: many new tokens, finished requests give their pages back
        dict(name="plan_prompts_1000", op="plan", rows=1000, fresh=500, ctx=3000, page=64, trim=True),
        # the keys and values of one decode step of 256 sequences: 12 heads of 64, f32 rows, a bf16 store (latency)
        dict(name="append_decode_256", op="append", tokens=256, kv_heads=12, hs=64, q="f32", kv="bf16", page=64, packed=True),
        # a chunk of prompts, 8 key heads of 128, out of one packed q|k|v row, some slots of a padded batch empty
        dict(name="append_chunk_16000", op="append", tokens=16000, kv_heads=8, hs=128, q="bf16", kv="bf16", page=16, packed=True),
        # the smallest read: three requests, the reference's head size and its f32 store, a cap on the store, pages of 24
        dict(name="attend_small_f32", op="attend", rows=3, fresh=7, ctx=200, heads=24, kv_heads=24, hs=32, q="f32", kv="f32", page=24, window=64, first=True),
        # decode at the benchmark's shape: 256 sequences around a context of 1536, 12 heads of 64, bf16 store
        dict(name="attend_decode_256", op="attend", rows=256, fresh=1, ctx=2048, heads=12, kv_heads=12, hs=64, q="f32", kv="bf16", page=64, window=0, first=False),
        # one token of one long sequence: the store's length has to be split over the GPU
        dict(name="attend_long_131072", op="attend", rows=1, fresh=1, ctx=131072, heads=12, kv_heads=12, hs=64, q="f32", kv="bf16", page=256, window=0, first=False),
        # a drafted run of five tokens for 64 requests, query heads sharing key heads
        dict(name="attend_drafts_64", op="attend", rows=64, fresh=5, ctx=8192, heads=32, kv_heads=8, hs=128, q="bf16", kv="bf16", page=16, window=0, first=False),
        # prompt chunks of the benchmark's shape behind what is already stored, ragged, with left padding
        dict(name="attend_chunk_16x1024", op="attend", rows=16, fresh=1024, ctx=2048, heads=12, kv_heads=12, hs=64, q="f32", kv="bf16", page=64, window=0, first=True),
        # long prompt chunks with shared key heads: the largest
        dict(name="attend_chunk_4x2048", op="attend", rows=4, fresh=2048, ctx=8192, heads=32, kv_heads=8, hs=128, q="bf16", kv="bf16", page=128, window=0, first=False),
        # one request's four drafted tokens (latency)
        dict(name="verify_1", op="verify", rows=1, drafts=4, vocab=16384, mode="draft"),
        # a batch's drafted tokens, ragged, at the larger vocabulary
        dict(name="verify_256", op="verify", rows=256, drafts=8, vocab=32768, mode="draft"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend", "verify"])
    if op == "plan":
        rows = _log(rng, 1, 2000)
        return dict(op=op, rows=rows, fresh=min(_log(rng, 1, 2000), 500000 // rows), ctx=_log(rng, 16, 20000), page=rng.choice([8, 16, 24, 32, 64, 100, 128, 256]),
                    trim=rng.random() < 0.5)
    if op == "append":
        q, kv = rng.choice([("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16")])
        return dict(op=op, tokens=_log(rng, 1, 8000), kv_heads=rng.choice([1, 2, 5, 8, 12]), hs=rng.choice([32, 64, 128]), q=q, kv=kv,
                    page=rng.choice([8, 16, 24, 64, 100, 256]), packed=rng.random() < 0.5)
    if op == "attend":
        q, kv = rng.choice([("f32", "bf16"), ("f32", "f32"), ("bf16", "bf16"), ("bf16", "bf16")])
        heads, kv_heads = rng.choice([(12, 12), (24, 24), (8, 2), (32, 8), (7, 1), (16, 16), (40, 8)])
        hs, ctx, fresh = rng.choice([32, 64, 128]), _log(rng, 1, 20000), rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 1500)])
        ctx = max(ctx, fresh)
        work = 250_000_000 if kv == "f32" else 1_000_000_000   # rows x heads x new tokens x keys, of which the largest listed case has more
        most = max(1, min(256, work // (heads * fresh * ctx), 200_000_000 // (ctx * kv_heads * hs)))
        if heads * fresh * ctx > work:
            fresh = max(1, work // (heads * ctx))
        return dict(op=op, rows=_log(rng, 1, most), fresh=fresh, ctx=ctx, heads=heads, kv_heads=kv_heads, hs=hs, q=q, kv=kv,
                    page=rng.choice([8, 16, 24, 32, 64, 100, 128, 256]), window=rng.choice([0, 0, 0, _log(rng, 1, 4000)]), first=rng.random() < 0.4)
    return dict(op=op, rows=_log(rng, 1, 200), drafts=rng.randint(0, 8), vocab=_log(rng, 2, 33000), mode=rng.choice(["draft", "draft", "point", "greedy"]))


def _lengths(case):
    """(tokens stored, new tokens) per request: a property of the case."""
    r = random.Random("%s %s %s" % (case["rows"], case["fresh"], case["ctx"]))
    cached, fresh = [], []
    for i in range(case["rows"]):
        n = case["fresh"] if i == 0 or case["fresh"] == 1 else r.randint((case["fresh"] + 1) // 2, case["fresh"])
        total = max(n, case["ctx"]) if i == 0 else r.randint(max(n, case["ctx"] // 2), max(n, case["ctx"]))
        if case["rows"] > 8 and i % 16 == 9:     # a finished request, or a row that pads the batch
            n, total = 0, 0 if case["op"] == "plan" else total
        cached.append(total - n)
        fresh.append(n)
    return cached, fresh


def _drafted(case):
    r = random.Random("%s %s" % (case["rows"], case["drafts"]))
    return [case["drafts"] if i == 0 else r.randint((case["drafts"] + 1) // 2, case["drafts"]) for i in range(case["rows"])]


def _starts(counts):
    s = [0]
    for n in counts:
        s.append(s[-1] + n)
    return s


def _seen(case, c, i, first):
    """How many keys new token i of a request with c stored tokens sees."""
    lo = max(first, c + i + 1 - case["window"] if case["window"] else 0, 0)
    return max(0, c + i + 1 - lo)


def _first(case, cached):
    """The first key that counts, per request: left padding of a quarter of what is stored; one request sees nothing of its own."""
    if not case["first"]:
        return [0] * len(cached)
    return [c // 4 if i != 1 else c + 2 for i, c in enumerate(cached)]


# ------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    rand = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    empty = lambda n, t=torch.int32: torch.full((n,), -7, dtype=t, device=DEV)  # noqa: E731
    op = case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        page = case["page"]
        total = sum(fresh)
        need = [-(-(c + f) // page) for c, f in zip(cached, fresh)]
        # pages held now: what the stored tokens fill, one more where a rejected draft left it, a finished request's old ones
        have = [-(-c // page) + (1 if i % 5 == 2 else 0) if c + f else 1 + i % 7 for i, (c, f) in enumerate(zip(cached, fresh))]
        n_pages = sum(max(a, b) for a, b in zip(need, have)) + 100
        ids = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        width = max(max(need), max(have)) + 3
        table = torch.full((len(cached), width), -1, dtype=torch.int32, device=DEV)
        owned = i32(have)
        mask = torch.arange(width, device=DEV)[None] < owned[:, None]
        table[mask] = ids[: sum(have)]
        free = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
        n_free = n_pages - sum(have)
        free[:n_free] = ids[sum(have):]
        cap = total + 37
        return dict(op=op, cached=i32(cached), fresh=i32(fresh), table=table, owned=owned, free=free, free_count=i32([n_free]), page=page, trim=case["trim"],
                    owned_out=empty(len(cached)), free_count_out=empty(1), q_start=empty(len(cached) + 1), slot=empty(cap, torch.int64), pos=empty(cap),
                    row=empty(cap), status=empty(1))
    if op == "append":
        n, h, hs, page = case["tokens"], case["kv_heads"], case["hs"], case["page"]
        pages = -(-n // page) + 3
        if case["packed"]:
            qkv = rand(n, 3, h, hs).to(FLOAT[case["q"]])
            k, v = qkv[:, 1], qkv[:, 2]
        else:
            k, v = rand(n, h, hs).to(FLOAT[case["q"]]), rand(n, h, hs).to(FLOAT[case["q"]])
        slot = torch.randperm(pages * page, generator=g, device=DEV)[:n]
        if n > 20:
            slot[torch.randint(0, n, (n // 20,), generator=g, device=DEV)] = -1
        kp, vp = (rand(pages, h, page, hs).to(FLOAT[case["kv"]]) for _ in range(2))
        return dict(op=op, k=k, v=v, slot=slot, k_pages=kp, v_pages=vp)
    if op == "attend":
        cached, fresh = _lengths(case)
        page, h, hs = case["page"], case["kv_heads"], case["hs"]
        need = [-(-(c + f) // page) for c, f in zip(cached, fresh)]
        n_pages = sum(need) + 5
        width = max(need) + 1
        table = torch.full((len(cached), width), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV)[None] < i32(need)[:, None]] = torch.randperm(n_pages, generator=g, device=DEV)[: sum(need)].to(torch.int32)
        kp, vp = (torch.randn(n_pages, h, page, hs, generator=g, device=DEV, dtype=FLOAT[case["kv"]]) for _ in range(2))
        q = (1.5 * rand(sum(fresh), case["heads"], hs)).to(FLOAT[case["q"]])
        return dict(op=op, q=q, k_pages=kp, v_pages=vp, table=table, cached=i32(cached), q_start=i32(_starts(fresh)), max_fresh=max(fresh), max_keys=case["ctx"],
                    window=case["window"], first=i32(_first(case, cached)) if case["first"] else None, out=torch.empty_like(q),
                    lse=torch.empty(q.shape[:2], device=DEV), room=torch.empty(64 << 20, dtype=torch.uint8, device=DEV), scale=1 / math.sqrt(hs))
    n = _drafted(case)
    starts, vocab = _starts([x + 1 for x in n]), case["vocab"]
    z = 3 * rand(starts[-1], vocab)
    p = torch.softmax(z, -1)
    q = torch.softmax(0.9 * z + 0.5 * rand(starts[-1], vocab), -1)
    noise = -torch.log(-torch.log(torch.rand(q.shape, generator=g, device=DEV).clamp_(1e-10, 1 - 1e-7)))
    drawn = (torch.log(q) + noise).argmax(-1)
    if case["mode"] == "point":
        drawn = p.argmax(-1)
    elif case["mode"] == "greedy":
        drawn = torch.where(torch.rand(drawn.shape, generator=g, device=DEV) < 0.9, p.argmax(-1), drawn)
    tok = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), drawn[:-1]]).to(torch.int32)   # row i proposed the token fed at i + 1
    uniform = torch.rand(starts[-1], generator=g, device=DEV, dtype=torch.float64)
    return dict(op="verify", p=p, q=q if case["mode"] == "draft" else None, tok=tok, q_start=i32(starts), uniform=None if case["mode"] == "greedy" else uniform,
                out=empty(case["rows"] * (case["drafts"] + 1)).view(case["rows"], -1), n_out=empty(case["rows"]))


# --------------------------------------------------------------------------------------------------- the operators
def run(state):
    return {"plan": _plan, "append": _append, "attend": _attend, "verify": _verify}[state["op"]](state)


def _plan(s):
    if own:
        from ava_b200 import serving
        serving.plan(s["cached"], s["fresh"], s["table"], s["owned"], s["free"], s["free_count"], s["page"], s["q_start"], s["slot"], pos=s["pos"], row=s["row"],
                     status=s["status"], trim=s["trim"], owned_out=s["owned_out"], free_count_out=s["free_count_out"])
    else:
        _plain_plan(s)
    return {k: s[k] for k in ("table", "owned_out", "free", "free_count_out", "q_start", "slot", "pos", "row", "status")}


def _plain_plan(s):
    cached, fresh, owned, table, free, page = s["cached"].long(), s["fresh"].long(), s["owned"].long(), s["table"], s["free"], s["page"]
    rows, width = table.shape
    need = (cached + fresh + page - 1) // page
    give = (owned - need).clamp(min=0) if s["trim"] else torch.zeros_like(owned)
    take = (need - owned).clamp(min=0)
    have = s["free_count"].long() + give.sum()
    bad = ((cached < 0) | (fresh < 0)).any() * BAD_LENGTH + (need > width).any() * NO_TABLE + (fresh.sum() > s["slot"].numel()) * NO_TOKENS
    bad = bad + (take.sum() > have) * NO_PAGES
    fine = bad == 0
    j = torch.arange(width, device=DEV)[None]
    # pages given back go on the stack of free pages in order of request and place ...
    at = s["free_count"].long() + (give.cumsum(0) - give)[:, None] + (j - need[:, None])
    back = (j >= need[:, None]) & (j < owned[:, None]) & (give[:, None] > 0) & fine
    free.copy_(torch.cat([free, free[:1]]).scatter(0, torch.where(back, at, free.numel()).view(-1), table.view(-1))[:-1])
    # ... and new ones come off its top
    at = have - 1 - ((take.cumsum(0) - take)[:, None] + (j - owned[:, None]))
    new = (j >= owned[:, None]) & (j < need[:, None]) & fine
    table.copy_(torch.where(new, free[at.clamp(0, free.numel() - 1)], table))
    s["owned_out"].copy_(torch.where(fine, owned - give + take, owned))
    s["free_count_out"].copy_(torch.where(fine, have - take.sum(), s["free_count"]))
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), fresh.cumsum(0)]) * fine
    s["q_start"].copy_(starts)
    t = torch.arange(s["slot"].numel(), device=DEV)
    r = torch.searchsorted(starts[1:].contiguous(), t, right=True).clamp(max=rows - 1)
    pos = cached[r] + t - starts[r]
    held = t < starts[-1]
    s["slot"].copy_(torch.where(held, table[r, (pos // page).clamp(0, width - 1)].long() * page + pos % page, -1))
    s["pos"].copy_(torch.where(held, pos, -1))
    s["row"].copy_(torch.where(held, r, -1))
    s["status"].copy_(bad)


def _append(s):
    if own:
        from ava_b200 import serving
        serving.append(s["k"], s["v"], s["slot"], s["k_pages"], s["v_pages"])
    else:
        kept = s["slot"] >= 0
        slot, page = s["slot"][kept], s["k_pages"].shape[2]
        s["k_pages"][slot // page, :, slot % page] = s["k"][kept].to(s["k_pages"].dtype)
        s["v_pages"][slot // page, :, slot % page] = s["v"][kept].to(s["v_pages"].dtype)
    return s["k_pages"], s["v_pages"]


def _attend(s):
    if own:
        from ava_b200 import serving
        serving.attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["cached"], s["q_start"], s["out"], max_fresh=s["max_fresh"], workspace=s["room"], scale=s["scale"],
                       window=s["window"], first=s["first"], lse=s["lse"])
        return s["out"], s["lse"]
    q, table, cached, starts = s["q"].float(), s["table"], s["cached"].long(), s["q_start"].long()
    page, (rows, width) = s["k_pages"].shape[2], table.shape
    heads, kv_heads, hs = q.shape[1], s["k_pages"].shape[1], q.shape[2]
    key, i = torch.arange(s["max_keys"], device=DEV), torch.arange(s["max_fresh"], device=DEV)
    pages = table[:, (key // page).clamp(max=width - 1)].long().clamp(min=0)                        # [rows, keys]
    k, v = (x[pages, :, (key % page)[None]].float().transpose(1, 2) for x in (s["k_pages"], s["v_pages"]))   # [rows, kv heads, keys, hs]
    token = (starts[:-1, None] + i).clamp(max=max(0, q.shape[0] - 1))                               # [rows, new tokens]
    qr = q[token].view(rows, -1, kv_heads, heads // kv_heads, hs).permute(0, 2, 3, 1, 4).reshape(rows, kv_heads, -1, hs)
    x = torch.matmul(qr, k.transpose(-1, -2)).mul_(s["scale"]).view(rows, kv_heads, heads // kv_heads, len(i), len(key))
    at = (cached[:, None] + i)[:, :, None]
    seen = (key <= at) & (at < (cached + starts[1:] - starts[:-1])[:, None, None])
    if s["window"]:
        seen = seen & (key > at - s["window"])
    if s["first"] is not None:
        seen = seen & (key >= s["first"][:, None, None])
    x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(rows, kv_heads, -1, len(key)), v).view(*x.shape[:-1], hs) / total.clamp(min=1e-30)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    held = i < (starts[1:] - starts[:-1])[:, None]                                                  # tokens in packed order
    o = o.permute(0, 3, 1, 2, 4).reshape(rows, len(i), heads, hs)[held]
    return o.to(s["q"].dtype), lse.permute(0, 3, 1, 2).reshape(rows, len(i), heads)[held].contiguous()


def _verify(s):
    if own:
        from ava_b200 import serving
        serving.verify_drafts(s["p"], s["tok"], s["q_start"], s["out"], s["n_out"], q=s["q"], uniform=s["uniform"])
        return s["out"], s["n_out"]
    p, q, tok, u = s["p"], s["q"], s["tok"].long(), s["uniform"]
    starts = s["q_start"].long()
    n = starts[1:] - starts[:-1] - 1
    i = torch.arange(s["out"].shape[1], device=DEV)
    at = (starts[:-1, None] + i).clamp(max=p.shape[0] - 1)                        # the row of p behind place i
    draft = tok[(at + 1).clamp(max=p.shape[0] - 1)]
    if u is None:
        best = p.argmax(-1)
        taken = best[at] == draft
    else:
        pd = p[at, draft].double()
        taken = u[at] * (q[at, draft].double() if q is not None else 1.0) < pd
    taken = taken & (i < n[:, None])
    kept = taken.long().cumprod(1).sum(1)                                         # drafts before the first refused one
    last = starts[:-1] + kept
    if u is None:
        final = best[last]
    else:
        w = p[last].double()
        refused = (kept < n)[:, None]
        if q is not None:
            w = torch.where(refused, w - q[last].double(), w)
        else:
            w = torch.where(refused & (torch.arange(p.shape[1], device=DEV) == draft.gather(1, kept[:, None].clamp(max=len(i) - 1))), 0.0, w)
        w = w.clamp(min=0)
        w = torch.where(w.sum(1, keepdim=True) > 0, w, p[last].double())          # nothing left over: the target's own
        c = w.cumsum(1)
        final = (c <= (u[starts[1:] - 1] * c[:, -1])[:, None]).sum(1).clamp(max=p.shape[1] - 1)
    s["out"].copy_(torch.where(i < kept[:, None], draft, torch.where(i == kept[:, None], final[:, None], -1)))
    s["n_out"].copy_(kept + 1)
    return s["out"], s["n_out"]


# ------------------------------------------------------------------------------------------------- what they cost
def work(case):
    size = {"f32": 4, "bf16": 2}
    op = case["op"]
    if op == "plan":
        cached, fresh = _lengths(case)
        # lengths, page counts, first tokens; a table entry and a list entry per page that changes hands; 16 bytes a token
        moved = sum(-(-f // case["page"]) for f in fresh)
        return {"bytes": 20 * case["rows"] + 8 * moved + 16 * sum(fresh), "flops": 0}
    if op == "append":
        n = case["tokens"] * case["kv_heads"] * case["hs"] * 2
        return {"bytes": n * (size[case["q"]] + size[case["kv"]]) + 8 * case["tokens"], "flops": 0}
    if op == "attend":
        cached, fresh = _lengths(case)
        first = _first(case, cached)
        keys = pairs = 0
        for c, n, f in zip(cached, fresh, first):
            if n:
                lo = max(f, c + 1 - case["window"] if case["window"] else 0, 0)
                keys += max(0, c + n - lo)
                w = case["window"] or c + n
                base = max(0, f)
                # sum over the new tokens of what each sees
                pairs += sum(max(0, c + i + 1 - max(base, c + i + 1 - w)) for i in range(n))
        tokens = sum(fresh)
        moved = keys * case["kv_heads"] * case["hs"] * 2 * size[case["kv"]] + tokens * case["heads"] * (case["hs"] * 2 * size[case["q"]] + 4)
        return {"bytes": moved + 4 * case["rows"], "flops": 4 * pairs * case["heads"] * case["hs"]}
    n = _drafted(case)
    if case["mode"] == "greedy":   # rows of probabilities up to the first draft that is not the most likely token
        return {"bytes": sum(sum(0.9 ** i for i in range(x + 1)) for x in n) * case["vocab"] * 4 + 8 * case["rows"], "flops": 0}
    # one row of the target's and, where a draft was refused, one of the draft's probabilities
    rows = case["rows"] * (2 if case["mode"] == "draft" and case["drafts"] else 1)
    return {"bytes": rows * case["vocab"] * 4 + sum(n) * 24 + 8 * case["rows"], "flops": 0}


# ------------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        page = case["page"]
        for t, at in enumerate(s["slot"].tolist()):
            if at >= 0:
                k[at // page, :, at % page], v[at // page, :, at % page] = s["k"][t].double(), s["v"][t].double()
        return k, v
    if op == "attend":
        cached, starts, group = s["cached"].tolist(), s["q_start"].tolist(), case["heads"] // case["kv_heads"]
        first = s["first"].tolist() if s["first"] is not None else [0] * case["rows"]
        o, lse = [], []
        for r, c in enumerate(cached):
            n = starts[r + 1] - starts[r]
            total = c + n
            ids = s["table"][r, : -(-total // case["page"])].long()
            k, v = (x[ids].double().transpose(0, 1).reshape(case["kv_heads"], -1, case["hs"])[:, :total] for x in (s["k_pages"], s["v_pages"]))
            row, column = torch.arange(c, total, device=DEV)[:, None], torch.arange(total, device=DEV)[None]
            hidden = (column > row) | (column < first[r])
            if case["window"]:
                hidden |= row - column >= case["window"]
            for h in range(case["heads"] if n else 0):
                x = (s["q"][starts[r]: starts[r + 1], h].double() @ k[h // group].T) * s["scale"]
                total_log = torch.logsumexp(x.masked_fill(hidden, -math.inf), -1)
                weight = torch.where(hidden, 0.0, torch.exp(x - torch.where(total_log.isinf(), 0.0, total_log)[:, None]))
                o.append(weight @ v[h // group])
                lse.append(total_log)
        if not o:
            return s["q"].double(), s["lse"].double()
        counts = [starts[r + 1] - starts[r] for r in range(case["rows"])]
        o, lse = iter(o), iter(lse)
        whole = [(torch.stack([next(o) for _ in range(case["heads"])], 1), torch.stack([next(lse) for _ in range(case["heads"])], 1)) for n in counts if n]
        return torch.cat([a for a, _ in whole]), torch.cat([b for _, b in whole])
    return None   # whole numbers
