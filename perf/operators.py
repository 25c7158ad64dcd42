"""Measured cases of the paged-cache operators: one serving step over a paged
KV cache, from the step's block tables to its attention.

  plan     block tables, slots and positions of a step from request lengths
  append   per-head query/key norm, rotation and the append to the cache
  means    mean key of every page the step completed
  attend   attention of a ragged batch whose requests share a prefix
  sparse   attention over the pages that each query scores highest

`own` selects what run() computes with: False, elementary torch operations;
True, the framework's operators.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # One decode step of 64 concurrent sessions: latency is all there is.
        dict(name="plan decode 64", op="plan", n=64, held=8192, chunks=0, chunk=0, page=32),
        # A busy server's step: 1,000 decoding requests and 24 prefill chunks of up to 512 tokens.
        dict(name="plan mixed 1024", op="plan", n=1024, held=4096, chunks=24, chunk=512, page=32),
        # One token of a small grouped-query model: the smallest call.
        dict(name="append one token", op="append", T=1, H=8, KVH=4, hd=64, q="f16", kv="f16", norm="none", pairs=32, adjacent=True, page=32, strided=False),
        # The 3B model's heads, a 64-branch step in the framework's own types: float32 rows, binary16 cache, 25 % rotary.
        dict(name="append 3B step 64", op="append", T=64, H=32, KVH=32, hd=80, q="f32", kv="f16", norm="layer", pairs=10, adjacent=False, page=32, strided=True),
        # Eight prefill chunks of 512 tokens, grouped-query heads, every feature rotated.
        dict(name="append prefill 4096", op="append", T=4096, H=32, KVH=8, hd=128, q="bf16", kv="bf16", norm="rms", pairs=64, adjacent=False, page=32, strided=False),
        # A decode step of 256 requests, of which about one in 32 completes a page.
        dict(name="means decode 256", op="means", T=256, n=256, KVH=8, hd=128, kv="bf16", page=32),
        # A long prompt's pages, the 3B model's heads.
        dict(name="means prefill 16384", op="means", T=16384, n=4, KVH=32, hd=80, kv="f16", page=32),
        # 64 branches with suffixes of 1 to 96 tokens over a 4,043-token prompt (126 whole pages of it shared).
        dict(name="attend 3B branches 64", op="attend", n=64, H=32, KVH=32, hd=80, q="f16", kv="f16", prefix=126, own=107, fresh=1, page=32),
        # 256 requests over one 32,768-token document: the largest.
        dict(name="attend document 256", op="attend", n=256, H=32, KVH=8, hd=128, q="bf16", kv="bf16", prefix=1024, own=1024, fresh=1, page=32),
        # Eight short float32 requests of up to four tokens each (drafted tokens being verified).
        dict(name="attend drafts f32", op="attend", n=8, H=8, KVH=4, hd=64, q="f32", kv="f32", prefix=16, own=80, fresh=4, page=32),
        # 64 long chats decoding at once, 66 pages of up to 1,024 read for each.
        dict(name="sparse decode 64", op="sparse", n=64, H=32, KVH=8, hd=128, q="bf16", kv="bf16", length=32768, fresh=1, first=1, last=1, top=64, page=32),
        # One reader of a 131,072-token book, ungrouped heads.
        dict(name="sparse book 1", op="sparse", n=1, H=32, KVH=32, hd=80, q="f16", kv="f16", length=131072, fresh=1, first=1, last=4, top=59, page=32),
    ]


def spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["plan", "append", "means", "attend", "sparse"])
    page = rng.choice([16, 32, 32, 64])
    if op == "plan":
        n = spread(rng, 1, 2048)
        chunks = rng.choice([0, rng.randint(0, max(1, n // 16))])
        return dict(op=op, n=n, held=spread(rng, 16, 32768), chunks=chunks, chunk=spread(rng, 2, 512) if chunks else 0, page=page)
    KVH = rng.choice([1, 2, 4, 8, 8, 16, 32])
    H = KVH * rng.choice([1, 2, 4, 4, 8] if KVH <= 8 else [1, 2] if KVH == 16 else [1])
    hd = rng.choice([64, 80, 128, 128])
    q, kv = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f16", "f16"), ("f32", "f32"), ("f32", "f16")])
    if op == "append":
        pairs = rng.choice([0, hd // 8, hd // 2])
        T = spread(rng, 1, 8192 * 4096 // ((H + 2 * KVH) * hd * (2 if q == "f32" else 1)) // 2 + 1)
        return dict(op=op, T=T, H=H, KVH=KVH, hd=hd, q=q, kv=kv, norm=rng.choice(["none", "rms", "layer"]), pairs=pairs,
                    adjacent=rng.random() < 0.3, page=page, strided=rng.random() < 0.3)
    if op == "means":
        T = spread(rng, 32, 1 + 16384 * 32 * 80 // (KVH * hd * (2 if kv == "f32" else 1)))
        return dict(op=op, T=T, n=min(T, spread(rng, 1, 256)), KVH=KVH, hd=hd, kv=kv, page=page)
    while True:
        fresh = rng.choice([1, 1, 1, 1, spread(rng, 2, 64)])
        n = spread(rng, 1, 256)
        if op == "attend":
            c = dict(op=op, n=n, H=H, KVH=KVH, hd=hd, q=q, kv=kv, prefix=rng.choice([0, spread(rng, 1, 32768 // page)]),
                     own=fresh + spread(rng, 1, 2048), fresh=fresh, page=page)
            most = n * fresh * H * (c["prefix"] * page + c["own"] + page)  # scores of the plain form
            held = n * KVH * hd * (c["own"] + page)
            if most > 256 * 32 * 33792 or held > 256 * 8 * 128 * 1056:
                continue
        else:
            length = fresh + spread(rng, 64, 131072)
            top = spread(rng, 1, 128)
            first, last = rng.choice([0, 1, 2]), rng.choice([1, 2, 4])
            c = dict(op=op, n=n, H=H, KVH=KVH, hd=hd, q=q, kv=kv, length=length, fresh=fresh, first=first, last=last, top=top, page=page)
            most = n * fresh * KVH * hd * page * (first + last + top)
            pages = n * fresh * KVH * hd * -(-length // page)  # means, in 64 bits
            if most > 64 * 8 * 128 * 32 * 66 or pages > 64 * 8 * 128 * 1024 or n * length * KVH * hd > 64 * 32768 * 8 * 128:
                continue
        big, cost = work(LARGEST), work(c)
        if cost["flops"] <= big["flops"] and cost["bytes"] <= big["bytes"]:
            return c


def lengths_of(case, seed):
    """Host-side lengths of the step, from the seed: positions held before it and tokens of it, for each request."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    n = case["n"]
    if case["op"] == "plan":
        held = torch.randint(0, case["held"] + 1, (n,), generator=g)
        fresh = torch.ones(n, dtype=torch.long)
        at = torch.randperm(n, generator=g)[: case["chunks"]]
        if len(at):
            fresh[at] = torch.randint(1, case["chunk"] + 1, (len(at),), generator=g)
        return held, fresh
    # The same counts for every seed, in another order.
    fresh = (torch.arange(n) * 7 % case["fresh"] + 1)[torch.randperm(n, generator=g)]
    at = int(fresh.argmax())
    fresh[[0, at]] = fresh[[at, 0]]  # the first request has the most
    if case["op"] == "attend":
        grown = torch.randint(0, case["own"] - case["fresh"] + 1, (n,), generator=g)
        return case["prefix"] * case["page"] + grown, fresh
    least = (case["length"] - case["fresh"]) // 4
    held = torch.randint(least, case["length"] - case["fresh"] + 1, (n,), generator=g)
    held[0] = case["length"] - case["fresh"]
    return held, fresh


def normal(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32) * scale).to(dtype)


def cache_of(case, num_pages, gen):
    """Keys and values of the pool [pages][KV heads][positions][features]: keys of a page have a direction in common, as neighbouring text has."""
    t = TYPES[case["kv"]]
    KVH, P, hd = case["KVH"], case["page"], case["hd"]
    k = normal((num_pages, KVH, P, hd), gen, t)
    k += normal((num_pages, KVH, 1, hd), gen, t, 0.8)
    v = normal((num_pages, KVH, P, hd), gen, t)
    return k, v


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case=dict(case), op=case["op"])
    P = case["page"]
    if case["op"] == "plan":
        held, fresh = lengths_of(case, seed)
        width = (case["held"] + max(1, case["chunk"]) + P - 1) // P
        total = int(((held + fresh + P - 1) // P).sum())
        need = total - int(((held + P - 1) // P).sum())
        ids = torch.randperm(total + 16, generator=gen, device=DEVICE).to(torch.int32)
        s["free"] = ids[: need + 16].clone()
        have = (held + P - 1) // P
        j = torch.arange(width)
        tables = torch.full((case["n"], width), -1, dtype=torch.int32)
        mask = j[None] < have[:, None]
        tables[mask] = ids[need + 16:][: int(have.sum())].cpu()
        s["tables"] = tables.to(DEVICE)
        s["held"], s["fresh"] = held.to(DEVICE, torch.int32), fresh.to(DEVICE, torch.int32)
        s["capacity"] = case["n"] + case["chunks"] * case["chunk"]  # what the step's buffers hold
        if own:
            from tinyoai_b200 import paged
            s["plan"] = paged.StepPlan(case["n"], s["capacity"], P, device=s["held"].device)
        return s
    KVH, hd = case["KVH"], case["hd"]
    kt = TYPES[case["kv"]]
    if case["op"] == "append":
        T, H, qt = case["T"], case["H"], TYPES[case["q"]]
        width = (H + 2 * KVH) * hd
        rows = normal((T, width + (hd if case["strided"] else 0)), gen, qt)
        s["qkv"] = rows[:, :width]
        pages = T // P + 9
        s["k"], s["v"] = (torch.zeros(pages, KVH, P, hd, dtype=kt, device=DEVICE) for _ in range(2))
        s["slots"] = torch.randperm(pages * P, generator=gen, device=DEVICE)[:T].clone()
        most = 8192
        s["positions"] = torch.randint(0, most, (T,), generator=gen, device=DEVICE).to(torch.int32)
        pairs = case["pairs"]
        rate = 10000.0 ** (-torch.arange(max(pairs, 1), device=DEVICE, dtype=torch.float64) / max(pairs, 1))
        angle = torch.arange(most, device=DEVICE, dtype=torch.float64)[:, None] * rate
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float()[:, :pairs].contiguous()
        per_head = case["norm"] == "layer"  # a layer norm has weights for every head, a root-mean-square one shares them
        s["qw"] = 1 + normal((H if per_head else 1, hd), gen, torch.float32, 0.1)
        s["kw"] = 1 + normal((KVH if per_head else 1, hd), gen, torch.float32, 0.1)
        s["eps"] = 1e-5
        if own:
            from tinyoai_b200 import paged
            s["cache"] = paged.Cache(s["k"], s["v"])
            s["rotary"] = paged.Rotary(s["table"], adjacent=case["adjacent"]) if pairs else None
            s["norm"] = None if case["norm"] == "none" else paged.HeadNorm(case["norm"], s["qw"], s["kw"], s["eps"])
        return s
    if case["op"] == "means":
        T, n = case["T"], case["n"]
        # Request i appends T // n tokens (the first one T % n more) from an offset within its first page.
        count = torch.full((n,), T // n, device=DEVICE)
        count[0] += T % n
        begin = torch.randint(0, P, (n,), generator=gen, device=DEVICE)
        need = (begin + count + P - 1) // P
        base = torch.cumsum(need, 0) - need
        pages = T // P + 2 * n + 3
        s["k"], s["v"] = cache_of(case, pages, gen)
        s["means"] = torch.zeros(pages, KVH, hd, dtype=kt, device=DEVICE)
        order = torch.randperm(pages, generator=gen, device=DEVICE)
        r = torch.repeat_interleave(torch.arange(n, device=DEVICE), count)
        pos = begin[r] + torch.arange(T, device=DEVICE) - (torch.cumsum(count, 0) - count)[r]
        s["slots"] = order[base[r] + pos // P] * P + pos % P
        if own:
            from tinyoai_b200 import paged
            s["cache"] = paged.Cache(s["k"], s["v"])
        return s
    held, fresh = lengths_of(case, seed)
    n, H, qt = case["n"], case["H"], TYPES[case["q"]]
    length = held + fresh
    have = (length + P - 1) // P
    width = int(have.max())
    shared = case.get("prefix", 0)
    total = shared + int((have - shared).clamp(min=0).sum())
    order = torch.randperm(total + 5, generator=gen, device=DEVICE).to(torch.int32)
    tables = torch.full((n, width), -1, dtype=torch.int32, device=DEVICE)
    j = torch.arange(width, device=DEVICE)
    tables[:, :shared] = order[:shared]
    tables[(j[None] >= shared) & (j[None] < have.to(DEVICE)[:, None])] = order[shared:total]
    s["tables"] = tables
    s["prefix"] = order[:shared].clone()
    s["k"], s["v"] = cache_of(case, total + 5, gen)
    s["starts"] = torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(fresh, 0)]).to(DEVICE, torch.int32)
    s["lengths"] = length.to(DEVICE, torch.int32)
    s["most"] = int(length.max())
    s["q"] = normal((int(fresh.sum()), H, hd), gen, qt, 1.5)
    s["scale"] = 1 / math.sqrt(hd)
    if case["op"] == "sparse":
        s["means"] = s["k"].float().mean(2).to(kt)
    if own:
        from tinyoai_b200 import paged
        s["cache"] = paged.Cache(s["k"], s["v"])
    return s


def run(s):
    return RUN[s["op"]](s)


def run_plan(s):
    held, fresh, tables, free = s["held"], s["fresh"], s["tables"], s["free"]
    P, capacity = s["case"]["page"], s["capacity"]
    if own:
        p = s["plan"].build(held, fresh, tables, free)
        return dict(tables=tables, starts=p.starts, lengths=p.lengths, positions=p.positions, slots=p.slots, counts=p.counts)
    n, width = tables.shape
    have = (held + P - 1) // P
    need = (held + fresh + P - 1) // P - have
    fits = (torch.cumsum(fresh, 0) <= capacity) & (torch.cumsum(need, 0) <= free.numel()) & (have + need <= width)
    planned = torch.cumprod(fits.int(), 0).int()
    fresh, need = fresh * planned, need * planned
    starts = torch.zeros(n + 1, dtype=torch.int32, device=held.device)
    starts[1:] = torch.cumsum(fresh, 0)
    taken = torch.cumsum(need, 0)
    j = torch.arange(width, device=held.device)[None] - have[:, None]
    new = (j >= 0) & (j < need[:, None])
    at = ((taken - need)[:, None] + j).clamp(0, max(free.numel() - 1, 0))
    tables.copy_(torch.where(new, free[at], tables))
    t = torch.arange(capacity, dtype=torch.int32, device=held.device)
    r = torch.searchsorted(starts[1:], t, right=True).clamp(max=n - 1)
    used = t < starts[-1]
    pos = torch.where(used, held[r] + t - starts[r], -1)
    at = pos.clamp(min=0)
    slots = torch.where(used, tables[r, at // P].long() * P + at % P, -1)
    counts = torch.stack([planned.sum(), starts[-1].long(), taken[-1]]).int()
    return dict(tables=tables, starts=starts, lengths=held + fresh, positions=pos.int(), slots=slots, counts=counts)


def normed(x, kind, w, eps):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w


def rotated(x, table, adjacent):
    pairs = table.shape[1]
    c, s = table[:, None, :, 0], table[:, None, :, 1]
    out = x.clone()
    at_a = slice(0, 2 * pairs, 2) if adjacent else slice(0, pairs)
    at_b = slice(1, 2 * pairs, 2) if adjacent else slice(pairs, 2 * pairs)
    a, b = x[..., at_a], x[..., at_b]
    out[..., at_a] = a * c - b * s
    out[..., at_b] = b * c + a * s
    return out


def run_append(s):
    c, k, v = s["case"], s["k"], s["v"]
    if own:
        q = s["cache"].append(s["qkv"], c["H"], s["positions"], s["slots"], rotary=s["rotary"], norm=s["norm"])
        return dict(q=q, k=k, v=v)
    T, H, KVH, hd, P = c["T"], c["H"], c["KVH"], c["hd"], c["page"]
    x = s["qkv"].float().reshape(T, H + 2 * KVH, hd)
    table = s["table"][s["positions"].long()]
    q = rotated(normed(x[:, :H], c["norm"], s["qw"], s["eps"]), table, c["adjacent"])
    key = rotated(normed(x[:, H:H + KVH], c["norm"], s["kw"], s["eps"]), table, c["adjacent"])
    page, at = s["slots"] // P, s["slots"] % P
    k[page, :, at] = key.to(k.dtype)
    v[page, :, at] = x[:, H + KVH:].to(v.dtype)
    return dict(q=q.to(s["qkv"].dtype), k=k, v=v)


def run_means(s):
    k, means, slots, P = s["k"], s["means"], s["slots"], s["case"]["page"]
    if own:
        return s["cache"].page_means(slots, means)
    done = slots[(slots >= 0) & (slots % P == P - 1)] // P
    means[done] = k[done].float().mean(2).to(means.dtype)
    return means


def softmax_parts(score):
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    return p, p.sum(-1, keepdim=True)


def query_grid(s):
    """Queries as [request][token of it]: the token's row and its position; unused places have the row behind the last one and the position -1."""
    starts, F = s["starts"].long(), s["case"]["fresh"]
    fresh = starts[1:] - starts[:-1]
    j = torch.arange(F, device=starts.device)
    used = j[None] < fresh[:, None]
    token = torch.where(used, starts[:-1, None] + j, len(s["q"]))
    pos = torch.where(used, (s["lengths"].long() - fresh)[:, None] + j, -1)
    return token, pos


def rows_of(grid, token, rows, dtype):
    """The rows [T, ...] of a grid [request][token of it, ...]."""
    out = torch.empty((rows + 1, *grid.shape[2:]), dtype=dtype, device=grid.device)
    out[token] = grid.to(dtype)
    return out[:rows]


def run_attend(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    if own:
        return s["cache"].attend(q, s["tables"], s["starts"], s["lengths"], c["fresh"], prefix=s["prefix"], scale=s["scale"], max_length=s["most"])
    n, H, KVH, hd, P, F = c["n"], c["H"], c["KVH"], c["hd"], c["page"], c["fresh"]
    G, shared = H // KVH, c["prefix"]
    token, pos = query_grid(s)
    x = q.float()[token.clamp(max=len(q) - 1)].reshape(n, F, KVH, G, hd) * s["scale"]
    pk = k[s["prefix"].long()].float().transpose(0, 1).reshape(KVH, shared * P, hd)
    pv = v[s["prefix"].long()].float().transpose(0, 1).reshape(KVH, shared * P, hd)
    tables = s["tables"][:, shared:].long().clamp(min=0)
    W = tables.shape[1]
    ok = k[tables].float().transpose(1, 2).reshape(n, KVH, W * P, hd)
    ov = v[tables].float().transpose(1, 2).reshape(n, KVH, W * P, hd)
    score = torch.cat([torch.einsum("nfkgd,ksd->nfkgs", x, pk), torch.einsum("nfkgd,nksd->nfkgs", x, ok)], -1)
    t = torch.arange(score.shape[-1], device=q.device)
    score.masked_fill_((t > pos[..., None])[:, :, None, None], -math.inf)
    p, total = softmax_parts(score)
    o = torch.einsum("nfkgs,ksd->nfkgd", p[..., : shared * P], pv) + torch.einsum("nfkgs,nksd->nfkgd", p[..., shared * P:], ov)
    return rows_of((o / total).reshape(n, F, H, hd), token, len(q), q.dtype)


def chosen_pages(s, score, pos):
    """Pages [..., budget] that each query reads, ascending, from its scores of every page."""
    c = s["case"]
    w = torch.arange(score.shape[-1], device=score.device)
    npages = (pos // c["page"] + 1)[..., None, None]
    candidate = (w >= c["first"]) & (w < npages - c["last"])
    score = torch.where(candidate, score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., : c["top"]]
    best = torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True) & candidate
    always = (w < npages) & ((w < c["first"]) | (w >= npages - c["last"]))
    past = score.shape[-1]
    pages = torch.where(best | always, w, past).sort(-1).values[..., : c["first"] + c["last"] + c["top"]]
    pages = torch.nn.functional.pad(pages, (0, c["first"] + c["last"] + c["top"] - pages.shape[-1]), value=past)
    return torch.where(pages < past, pages, -1)


def run_sparse(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    if own:
        out, pages = s["cache"].attend_sparse(q, s["means"], s["tables"], s["starts"], s["lengths"], c["fresh"], top=c["top"], first=c["first"],
                                              last=c["last"], scale=s["scale"])
        return dict(out=out, pages=pages)
    n, H, KVH, hd, P, F = c["n"], c["H"], c["KVH"], c["hd"], c["page"], c["fresh"]
    G = H // KVH
    token, pos = query_grid(s)
    tables = s["tables"].long().clamp(min=0)
    x = q[token.clamp(max=len(q) - 1)].reshape(n, F, KVH, G, hd)
    # The choice of pages is a matter of order: scores in 64 bits.
    score = torch.einsum("nfkgd,nwkd->nfkgw", x.double(), s["means"][tables].double()).amax(3)
    pages = chosen_pages(s, score, pos)
    request = torch.arange(n, device=q.device)[:, None, None, None]
    head = torch.arange(KVH, device=q.device)[None, None, :, None]
    at = tables[request, pages.clamp(min=0)]
    B = pages.shape[-1]
    t = pages[..., None] * P + torch.arange(P, device=q.device)
    seen = ((pages[..., None] >= 0) & (t <= pos[:, :, None, None, None])).reshape(n, F, KVH, 1, B * P)
    gk = k[at, head].float().reshape(n, F, KVH, B * P, hd)
    gv = v[at, head].float().reshape(n, F, KVH, B * P, hd)
    score = torch.einsum("nfkgd,nfksd->nfkgs", x.float() * s["scale"], gk)
    p, total = softmax_parts(torch.where(seen, score, -math.inf))
    o = torch.einsum("nfkgs,nfksd->nfkgd", p, gv) / total
    return dict(out=rows_of(o.reshape(n, F, H, hd), token, len(q), q.dtype), pages=rows_of(pages, token, len(q), torch.int32))


RUN = dict(plan=run_plan, append=run_append, means=run_means, attend=run_attend, sparse=run_sparse)


def mean_lengths(c):
    """Expected positions of a request and tokens of a step, for the counts of work()."""
    fresh = (c["fresh"] + 1) / 2
    if c["op"] == "attend":
        return c["prefix"] * c["page"] + (c["own"] - c["fresh"]) / 2 + fresh, fresh
    return (c["length"] - c["fresh"]) * 0.625 + fresh, fresh


def work(c):
    P = c["page"]
    if c["op"] == "plan":
        tokens = c["n"] + c["chunks"] * (c["chunk"] + 1) / 2
        pages = tokens / P
        return dict(bytes=8 * c["n"] + 8 * pages + 8 * c["n"] + 4 + 12 * (c["n"] + c["chunks"] * c["chunk"]), flops=0)
    KVH, hd = c["KVH"], c["hd"]
    es = SIZE[c["kv"]]
    if c["op"] == "append":
        qs, H = SIZE[c["q"]], c["H"]
        values = (H + 2 * KVH) * hd
        return dict(bytes=c["T"] * (values * qs + H * hd * qs + 2 * KVH * hd * es + 8 * c["pairs"] + 12), flops=c["T"] * values * 8)
    if c["op"] == "means":
        pages = c["T"] / P
        return dict(bytes=pages * (P + 1) * KVH * hd * es + 8 * c["T"], flops=pages * P * KVH * hd)
    length, fresh = mean_lengths(c)
    T, H, qs = c["n"] * fresh, c["H"], SIZE[c["q"]]
    outside = 2 * T * H * hd * qs + 4 * c["n"] * length / P
    if c["op"] == "attend":
        shared = c["prefix"] * P
        positions = shared + c["n"] * (length - shared)
        return dict(bytes=outside + 2 * positions * KVH * hd * es, flops=4 * T * H * hd * (length - fresh / 2))
    pages = length / P
    read = min(c["first"] + c["last"] + c["top"], pages)
    kv_pages = T * KVH * read if fresh == 1 else min(T * KVH * read, c["n"] * KVH * pages)
    return dict(bytes=outside + c["n"] * pages * KVH * hd * es + 2 * kv_pages * P * hd * es + 4 * T * KVH * read,
                flops=T * H * hd * (2 * pages + 4 * read * P))


def exact(case, seed):
    s = prepare(case, seed)
    return EXACT[case["op"]](s, case)


def exact_append(s, c):
    T, H, KVH, hd, P, pairs = (c[x] for x in ("T", "H", "KVH", "hd", "page", "pairs"))
    x = s["qkv"].double().reshape(T, -1, hd)
    parts = []
    for lo, hi, w in ((0, H, s["qw"]), (H, H + KVH, s["kw"])):
        y = x[:, lo:hi]
        if c["norm"] != "none":
            var, mean = torch.var_mean(y, -1, correction=0, keepdim=True)
            y = (y - mean) / (var + s["eps"]).sqrt() if c["norm"] == "layer" else y / (var + mean ** 2 + s["eps"]).sqrt()
            y = y * w.double()
        if pairs:
            # As complex numbers: each pair times e^(i angle).
            turn = torch.view_as_complex(s["table"].double()[s["positions"].long()].contiguous())[:, None]
            head = y[..., : 2 * pairs]
            z = head.reshape(T, -1, pairs, 2) if c["adjacent"] else head.reshape(T, -1, 2, pairs).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = z if c["adjacent"] else z.transpose(-1, -2)
            y = torch.cat([z.reshape(T, -1, 2 * pairs), y[..., 2 * pairs:]], -1)
        parts.append(y)
    k, v = (torch.zeros(s["k"].shape[0] * P, KVH, hd, dtype=torch.float64, device=DEVICE) for _ in range(2))
    k[s["slots"]], v[s["slots"]] = parts[1], x[:, H + KVH:]
    k, v = (y.reshape(-1, P, KVH, hd).transpose(1, 2).contiguous() for y in (k, v))
    return dict(q=parts[0], k=k, v=v)


def exact_means(s, c):
    P = c["page"]
    out = torch.zeros(s["means"].shape, dtype=torch.float64, device=DEVICE)
    pages = sorted(int(x) // P for x in s["slots"].tolist() if x >= 0 and x % P == P - 1)
    at = torch.tensor(pages, dtype=torch.long, device=DEVICE)
    for part in at.split(1024):
        out[part] = s["k"][part].double().sum(2) / P
    return out


def exact_rows(q, keys, values, scale, visible):
    """softmax(scale q keys^T) values in 64 bits: q [f, KVH, G, hd], keys and values [KVH, t, hd], visible [f or 1, t]."""
    score = torch.matmul(q.permute(1, 0, 2, 3).flatten(1, 2) * scale, keys.transpose(1, 2))
    KVH, f, G = q.shape[1], q.shape[0], q.shape[2]
    score = score.reshape(KVH, f, G, -1).masked_fill(~visible[None, :, None], -math.inf)
    w = torch.softmax(score, -1).reshape(KVH, f * G, -1)
    return torch.matmul(w, values).reshape(KVH, f, G, -1).permute(1, 0, 2, 3)


def exact_attend(s, c):
    H, KVH, hd, P = c["H"], c["KVH"], c["hd"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    prefix = s["prefix"].long()
    pk, pv = (x[prefix].double().transpose(0, 1).reshape(KVH, -1, hd) for x in (s["k"], s["v"]))
    for i in range(c["n"]):
        a, b, L = starts[i], starts[i + 1], lengths[i]
        own_pages = s["tables"][i, c["prefix"]: -(-L // P)].long()
        keys, values = (torch.cat([y, x[own_pages].double().transpose(0, 1).reshape(KVH, -1, hd)], 1)[:, :L] for x, y in ((s["k"], pk), (s["v"], pv)))
        pos = L - (b - a) + torch.arange(b - a, device=DEVICE)
        visible = torch.arange(keys.shape[1], device=DEVICE)[None] <= pos[:, None]
        q = s["q"][a:b].double().reshape(b - a, KVH, H // KVH, hd)
        out[a:b] = exact_rows(q, keys, values, s["scale"], visible).reshape(b - a, H, hd)
    return out


def exact_sparse(s, c):
    H, KVH, hd, P = c["H"], c["KVH"], c["hd"], c["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEVICE)
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    if len(s["q"]) * KVH > 4096:
        return None  # a loop over queries and heads
    for i in range(c["n"]):
        table = s["tables"][i].long()
        for t in range(starts[i], starts[i + 1]):
            pos = lengths[i] - (starts[i + 1] - t)
            count = pos // P + 1
            q = s["q"][t].double().reshape(KVH, H // KVH, hd)
            score = torch.matmul(q, s["means"][table[:count]].double().permute(1, 2, 0)).amax(1)
            lo, hi = min(c["first"], count), max(count - c["last"], 0)
            for g in range(KVH):
                picks = set(range(lo)) | set(range(max(hi, 0), count))
                if hi > lo:
                    row = score[g, lo:hi]
                    best = torch.topk(row, min(c["top"], hi - lo)).indices
                    picks |= {lo + int(x) for x in best.tolist()}
                at = torch.tensor(sorted(picks), device=DEVICE)
                keys, values = (x[table[at], g].double().reshape(1, -1, hd) for x in (s["k"], s["v"]))
                when = (at[:, None] * P + torch.arange(P, device=DEVICE)).reshape(1, -1)
                part = exact_rows(q[None, g:g + 1], keys, values, s["scale"], when <= pos)
                out[t, g * (H // KVH):(g + 1) * (H // KVH)] = part.reshape(-1, hd)
    return dict(out=out, pages=None)


EXACT = dict(plan=lambda s, c: None, append=exact_append, means=exact_means, attend=exact_attend, sparse=exact_sparse)

#: draw() costs no more than this listed case.
LARGEST = next(c for c in listed() if c["name"] == "attend document 256")
