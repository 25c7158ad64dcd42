"""Operators over a paged KV cache (tinyoai_b200.paged) against plain float64
computations.

Tolerances. u = eps / 2 of a type is the largest relative rounding error of a
store (float32 2^-24, binary16 2^-11, bfloat16 2^-8).
 - plan: whole numbers, equal.
 - append: a value passes a mean and a sum of squares (under 20 additions in
   any lane order), a reciprocal root (2 steps), three products and two
   operations of the rotation; each is within 2^-24 or two of them of the
   largest value it combines, under 64 * 2^-24 of the head's largest value in
   all, plus u of the value for its store.
 - means: P additions and a division: (P + 1) * 2^-24 * mean |k| + u |mean|.
 - attention: a score's float32 sum over hd products errs by at most
   (hd + 8) * 2^-23 * scale * sum |q k| (2^-23: the tensor core's additions
   may truncate), which changes a weight by that factor; the base-2
   exponential adds 2^-20 at most, the weight's own rounding u_w where the
   cache has 16 bits (float32 queries over a binary16 cache keep pairs of
   binary16 values: 2^-21), the sums over the positions n * 2^-23 at most
   (bounded here by 2^-13, for n <= 1,024 in one chain). All are relative to
   sum_t w_t |v_t|; the output's store adds u |o|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tinyoai_b200 import BackendError, _lib  # noqa: E402

if torch.cuda.is_available():
    from tinyoai_b200 import paged

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
PAIRS = [("f32", "f32"), ("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]
DEV = "cuda:0"


def unit(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# The plan


def plan_ref(held, fresh, tables, free, P, capacity):
    n, width = len(held), len(tables[0]) if tables else 0
    tables = [list(r) for r in tables]
    starts, lengths, pos, slots = [0], list(held), [-1] * capacity, [-1] * capacity
    tok = pg = planned = 0
    for i in range(n):
        have, pages = -(-held[i] // P), -(-(held[i] + fresh[i]) // P)
        if held[i] < 0 or fresh[i] < 0 or pages > width or tok + fresh[i] > capacity or pg + pages - have > len(free):
            break
        for j in range(have, pages):
            tables[i][j] = free[pg]
            pg += 1
        for t in range(fresh[i]):
            p = held[i] + t
            pos[tok + t] = p
            slots[tok + t] = tables[i][p // P] * P + p % P if tables[i][p // P] >= 0 else -1
        tok += fresh[i]
        lengths[i] = held[i] + fresh[i]
        starts.append(tok)
        planned += 1
    starts += [tok] * (n + 1 - len(starts))
    return tables, starts, lengths, pos, slots, [planned, tok, pg]


def plan_case(n, P, most, chunk, width, free, capacity, seed):
    import random
    r = random.Random(seed)
    held = [r.choice([0, P, r.randint(0, most)]) for _ in range(n)]
    fresh = [r.choice([0, 1, 1, r.randint(1, chunk)]) for _ in range(n)]
    ids = list(range(100000))
    r.shuffle(ids)
    tables = [[ids[(i * 131 + j) % 60000] if j < -(-held[i] // P) else -7 for j in range(width)] for i in range(n)]
    return held, fresh, tables, ids[60000:60000 + free], P, capacity


@pytest.mark.parametrize("n, P, most, chunk, width, free, capacity", [
    (1, 32, 100, 1, 8, 4, 4),
    (7, 16, 60, 40, 16, 64, 300),
    (64, 32, 500, 1, 20, 64, 64),
    (255, 1, 30, 9, 64, 4000, 3000),
    (256, 7, 90, 20, 32, 4000, 6000),
    (300, 32, 500, 200, 40, 4000, 40000),   # several tiles of requests and of tokens
    (700, 24, 300, 3, 30, 2000, 1500),
    (64, 16, 100, 60, 20, 40, 4000),        # the pool runs out
    (64, 16, 100, 60, 20, 4000, 500),       # the step's token capacity runs out
    (40, 16, 400, 200, 20, 4000, 9000),     # a table is too narrow
    (5, 16, 100, 10, 20, 0, 100),           # no free page at all
    (3, 70, 100, 10, 4, 9, 0),              # no token capacity
])
def test_plan(n, P, most, chunk, width, free, capacity):
    case = plan_case(n, P, most, chunk, width, free, capacity, seed=n + P)
    held, fresh, tables, pages, P, capacity = case
    plan = paged.StepPlan(n + 3, capacity, P, DEV)
    t = i32(tables)
    plan.build(i32(held), i32(fresh), t, i32(pages))
    want = plan_ref(*case)
    got = [t.tolist(), plan.starts.tolist(), plan.lengths.tolist(), plan.positions.tolist(), plan.slots.tolist(), plan.counts.tolist()]
    assert got == [list(x) for x in want]


def test_plan_edges():
    plan = paged.StepPlan(4, 6, 4, DEV)
    # No requests: only padding.
    plan.build(i32([]), i32([]), torch.zeros((0, 3), dtype=torch.int32, device=DEV), i32([1, 2]))
    assert plan.starts.tolist() == [0] and plan.counts.tolist() == [0, 0, 0] and plan.slots.tolist() == [-1] * 6
    # A negative count stops the plan; a missing page in the held part gives slot -1.
    t = i32([[5, -1, -1], [-1, -1, -1], [8, 9, 9]])
    plan.build(i32([2, 3, -1]), i32([1, 2, 1]), t, i32([20, 21]))
    assert plan.counts.tolist() == [2, 3, 1]
    assert plan.positions.tolist() == [2, 3, 4, -1, -1, -1]
    assert plan.slots.tolist() == [22, -1, 80, -1, -1, -1]
    assert plan.lengths.tolist() == [3, 5, -1] and t.tolist() == [[5, -1, -1], [-1, 20, -1], [8, 9, 9]]
    # Counts whose sum passes 2^31 are one that does not fit.
    plan.build(i32([2**31 - 1]), i32([2]), i32([[1, 2, 3]]), i32([]))
    assert plan.counts.tolist() == [0, 0, 0] and plan.lengths.tolist() == [2**31 - 1]
    # Slots past 32 bits.
    plan = paged.StepPlan(1, 1, 65536, DEV)
    plan.build(i32([65537]), i32([1]), i32([[3, 100000]]), i32([]))
    assert plan.slots.tolist() == [100000 * 65536 + 1]
    # Tables that are columns of a wider array.
    wide = torch.full((2, 9), -3, dtype=torch.int32, device=DEV)
    plan = paged.StepPlan(2, 4, 2, DEV)
    plan.build(i32([0, 0]), i32([3, 1]), wide[:, 2:6], i32([7, 8, 9]))
    assert wide.tolist() == [[-3, -3, 7, 8, -3, -3, -3, -3, -3], [-3, -3, 9, -3, -3, -3, -3, -3, -3]]


# ---------------------------------------------------------------------------
# Caches


def make_cache(pages, KVH, P, hd, dtype, g, order="heads", fill=None):
    """A cache in one of three orders of its first dimensions: its own
    [pages][heads][positions], [pages][positions][heads], or keys and values
    of a page side by side."""
    if order == "heads":
        k, v = (normal((pages, KVH, P, hd), g, dtype) for _ in range(2))
    elif order == "positions":
        k, v = (normal((pages, P, KVH, hd), g, dtype).transpose(1, 2) for _ in range(2))
    else:
        both = normal((pages, 2, KVH, P, hd), g, dtype)
        k, v = both[:, 0], both[:, 1]
    if fill is not None:
        k.fill_(fill)
        v.fill_(fill)
    return k, v


def append_ref(x, H, KVH, norm, eps, qw, kw, table, pos, adjacent):
    """Queries, keys and values in float64 of rows x [T, heads, hd]."""
    x = x.double()
    out = []
    for lo, hi, w in ((0, H, qw), (H, H + KVH, kw)):
        y = x[:, lo:hi]
        if norm == "rms":
            y = y / ((y * y).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        elif norm == "layer":
            y = y - y.mean(-1, keepdim=True)
            y = y / ((y * y).mean(-1, keepdim=True) + eps).sqrt() * w.double()
        if table is not None:
            c, s = table.double()[pos][:, None, :, 0], table.double()[pos][:, None, :, 1]
            n = c.shape[-1]
            z = y.clone()
            ia = torch.arange(n, device=DEV) * 2 if adjacent else torch.arange(n, device=DEV)
            ib = ia + 1 if adjacent else ia + n
            z[..., ia] = y[..., ia] * c - y[..., ib] * s
            z[..., ib] = y[..., ib] * c + y[..., ia] * s
            y = z
        out.append(y)
    return out[0], out[1], x[:, H + KVH:]


def near(got, want, tol):
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), (float((d - tol).max()), float(d.max()))


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("T, H, KVH, hd, P, norm, pairs, adjacent, order", [
    (1, 8, 4, 8, 32, "none", 4, True, "heads"),
    (5, 4, 4, 80, 32, "layer", 10, False, "heads"),
    (33, 8, 2, 128, 16, "rms", 64, False, "positions"),
    (64, 6, 1, 64, 7, "rms", 0, False, "both"),
    (17, 2, 2, 256, 5, "layer", 128, False, "heads"),
    (9, 4, 2, 200, 64, "rms", 33, True, "positions"),
    (130, 3, 3, 24, 1, "none", 12, False, "heads"),
    (257, 5, 5, 40, 33, "layer", 1, True, "both"),
])
def test_append(qt, kt, T, H, KVH, hd, P, norm, pairs, adjacent, order):
    g = gen(T + hd)
    qt, kt = TYPES[qt], TYPES[kt]
    pages = T // P + 3
    k, v = make_cache(pages, KVH, P, hd, kt, g, order)
    k0, v0 = k.clone(), v.clone()
    width = (H + 2 * KVH) * hd
    qkv = normal((T, width + 16), g, qt, 2.0)[:, 8:width + 8] if T % 2 else normal((T, width), g, qt, 2.0)
    if qkv.data_ptr() % 16:
        qkv = normal((T, width), g, qt, 2.0)
    slots = torch.randperm(pages * P, generator=g, device=DEV)[:T].clone()
    pos = torch.randint(0, 500, (T,), generator=g, device=DEV).to(torch.int32)
    skipped = []
    if T > 8:  # a padding row, a slot and a position outside
        slots[3], slots[5], skipped = -1, pages * P, [3, 5]
        if pairs:
            pos[7], skipped = 500, [3, 5, 7]
    table = torch.rand((500, pairs, 2), generator=g, device=DEV) * 2 - 1 if pairs else None
    heads = (H, KVH) if norm == "layer" else (1, 1)
    qw, kw = (normal((n, hd), g) for n in heads)
    eps = 1e-5
    out = torch.full((T, H, hd), 7.0, dtype=qt, device=DEV)
    paged.Cache(k, v).append(qkv, H, pos, slots, rotary=paged.Rotary(table, adjacent) if pairs else None,
                             norm=None if norm == "none" else paged.HeadNorm(norm, qw, kw, eps), out=out)
    live = torch.ones(T, dtype=torch.bool, device=DEV)
    live[skipped] = False
    x = qkv.reshape(T, H + 2 * KVH, hd)[live]
    q_want, k_want, v_want = append_ref(x, H, KVH, norm, eps, qw, kw, table, pos[live].long(), adjacent)
    for got, want, t in ((out[live], q_want, qt), (k[slots[live] // P, :, slots[live] % P], k_want, kt)):
        tol = 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + unit(t) * want.abs()
        if t == torch.float16:
            tol = tol + 2.0 ** -25  # half a step of the subnormal values
        near(got, want, tol)
    near(v[slots[live] // P, :, slots[live] % P], v_want, unit(kt) * v_want.abs() + (2.0 ** -25 if kt == torch.float16 else 0))
    assert bool((out[~live] == 7).all())
    untouched = torch.ones(pages * P, dtype=torch.bool, device=DEV)
    untouched[slots[live]] = False
    at = untouched.nonzero()[:, 0]
    assert torch.equal(k[at // P, :, at % P], k0[at // P, :, at % P]) and torch.equal(v[at // P, :, at % P], v0[at // P, :, at % P])


def test_norm_weights_of_a_single_key_head():
    """Weights per head where one of the two kinds has a single head."""
    g = gen(8)
    for H, KVH in ((4, 1), (1, 1)):
        k, v = make_cache(2, KVH, 8, 64, torch.bfloat16, g)
        qw, kw = normal((H, 64), g), normal((KVH, 64), g)
        x = normal((5, (H + 2 * KVH) * 64), g, torch.bfloat16)
        slots = torch.arange(5, device=DEV) + 3
        c = paged.Cache(k, v)
        q = c.append(x, H, i32([0] * 5), slots, norm=paged.HeadNorm("layer", qw, kw, 1e-5))
        qr, kr, _ = append_ref(x.reshape(5, -1, 64), H, KVH, "layer", 1e-5, qw, kw, None, None, False)
        for got, want in ((q, qr), (k[slots // 8, :, slots % 8], kr)):
            near(got, want, 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + 2.0 ** -8 * want.abs())
    with pytest.raises(BackendError):  # one row for several heads beside rows per head
        k, v = make_cache(2, 2, 8, 64, torch.bfloat16, g)
        paged.Cache(k, v).append(normal((5, 8 * 64), g, torch.bfloat16), 4, i32([0] * 5), slots,
                                 norm=paged.HeadNorm("layer", normal((1, 64), g), normal((2, 64), g), 1e-5))


def test_append_keeps_values_it_only_moves():
    """Without norm and rotation keys, values and queries are copies: infinities, NaN and the type's extremes among them."""
    g = gen(5)
    for t in TYPES.values():
        x = normal((3, 4 * 16), g, t)
        top = torch.finfo(t).max
        x[1, :6] = torch.tensor([math.inf, -math.inf, math.nan, top, -top, -0.0], dtype=t, device=DEV)
        k, v = make_cache(2, 1, 4, 16, t, g)
        q = paged.Cache(k, v).append(x, 2, i32([0, 1, 2]), torch.tensor([0, 5, 7], device=DEV))
        assert torch.equal(q.reshape(3, 32).nan_to_num(3), x[:, :32].nan_to_num(3))
        assert torch.equal(k[1, 0, 1], x[1, 32:48]) and torch.equal(v[1, 0, 3], x[2, 48:])


# ---------------------------------------------------------------------------
# Page means


@pytest.mark.parametrize("kt", list(TYPES))
@pytest.mark.parametrize("T, KVH, hd, P, order", [(1, 1, 8, 1, "heads"), (40, 4, 80, 32, "heads"), (100, 3, 128, 7, "positions"), (300, 2, 256, 64, "both"),
                                                   (64, 8, 136, 16, "heads")])
def test_page_means(kt, T, KVH, hd, P, order):
    g = gen(T)
    dt = TYPES[kt]
    pages = T // P + 4
    k, v = make_cache(pages, KVH, P, hd, dt, g, order)
    means = torch.full((pages, KVH, hd), 9.0, dtype=dt, device=DEV)
    slots = torch.randperm(pages * P, generator=g, device=DEV)[:T].clone()
    slots[0] = 2 * P - 1
    if T > 4:
        slots[1], slots[2] = -1, pages * P + P - 1  # outside the pool: nothing
    paged.Cache(k, v).page_means(slots, means)
    done = {int(s) // P for s in slots.tolist() if 0 <= s < pages * P and s % P == P - 1}
    for p in range(pages):
        if p not in done:
            assert bool((means[p] == 9).all())
            continue
        x = k[p].double()
        want = x.mean(1)
        near(means[p], want, (P + 1) * 2.0 ** -24 * x.abs().mean(1) + unit(dt) * want.abs() + (2.0 ** -25 if kt == "f16" else 0))


# ---------------------------------------------------------------------------
# Attention


def attention_ref(q, k, v, scale, visible):
    """q [rows, heads, hd], k and v [t, heads, hd], visible [rows, t]: outputs, sum of w |v| and largest score sum, float64."""
    q, k, v = q.double(), k.double(), v.double()
    s = torch.einsum("rhd,thd->rht", q, k) * scale
    size = torch.einsum("rhd,thd->rht", q.abs(), k.abs()) * abs(scale)
    mask = visible[:, None].expand_as(s)
    s = s.masked_fill(~mask, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    l = w.sum(-1, keepdim=True)
    w = torch.where(l == 0, 0.0, w / l)
    return torch.einsum("rht,thd->rhd", w, v), torch.einsum("rht,thd->rhd", w, v.abs()), size.masked_fill(~mask, 0).amax(-1)


def attention_tol(o, wv, size, hd, qt, kt):
    u_w = 2.0 ** -21 if qt == torch.float32 else unit(kt)
    rel = 2 * (hd + 8) * 2.0 ** -23 * size[..., None] + 2.0 ** -20 + 2.0 ** -13 + u_w
    return rel * wv + unit(qt) * o.abs() + (2.0 ** -25 if qt == torch.float16 else 0)


def attention_state(lens, fresh, H, KVH, hd, P, qt, kt, seed, prefix=0, order="heads", fill=math.nan, q_order="rows"):
    """Requests of lens positions (the step's fresh ones included) over shuffled pages; everything unused is `fill`."""
    g = gen(seed)
    n = len(lens)
    width = max([-(-x // P) for x in lens] + [prefix, 1])
    count = prefix + sum(max(0, -(-x // P) - prefix) for x in lens)
    pages = count + 3
    ids = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    k, v = make_cache(pages, KVH, P, hd, kt, g, order, fill)
    table = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
    at = prefix
    for i, x in enumerate(lens):
        have = -(-x // P)
        table[i, :min(prefix, have)] = ids[:min(prefix, have)]
        own = max(0, have - prefix)
        table[i, prefix:prefix + own] = ids[at:at + own]
        at += own
    lim = max(lens + [prefix * P])
    for i, x in enumerate(lens):
        t = torch.arange(x, device=DEV)
        pg = table[i][t // P].long()
        k[pg, :, t % P] = normal((x, KVH, hd), g, kt)
        v[pg, :, t % P] = normal((x, KVH, hd), g, kt)
    if prefix:  # the prefix is whole, whatever the requests hold
        t = torch.arange(prefix * P, device=DEV)
        pg = ids[:prefix][t // P].long()
        k[pg, :, t % P] = normal((prefix * P, KVH, hd), g, kt)
        v[pg, :, t % P] = normal((prefix * P, KVH, hd), g, kt)
    T = sum(fresh)
    if q_order == "rows":
        q = normal((T + 2, H, hd), g, qt)
    else:
        q = normal((H, T + 2, hd), g, qt).transpose(0, 1)
    starts = [0]
    for f in fresh:
        starts.append(starts[-1] + f)
    return dict(k=k, v=v, table=table, prefix=ids[:prefix].clone(), starts=i32(starts), lengths=i32(lens), q=q, T=T, lim=lim)


def expected(s, lens, fresh, H, KVH, hd, P, scale, prefix, chosen=None):
    """Reference outputs and tolerances of every used row."""
    outs, tols = [], []
    G = H // KVH
    qt, kt = s["q"].dtype, s["k"].dtype
    row = 0
    for i, (x, f) in enumerate(zip(lens, fresh)):
        for j in range(f):
            pos = x - f + j
            q = s["q"][row:row + 1]
            parts = []
            for g in range(KVH):
                t = torch.arange(max(pos + 1, 0), device=DEV)
                if chosen is not None:
                    t = t[torch.isin(t // P, torch.tensor(sorted(chosen[row][g]), device=DEV, dtype=torch.long))]
                page = torch.where(t // P < prefix, s["prefix"][(t // P).clamp(max=max(prefix - 1, 0))] if prefix else 0, s["table"][i][t // P]).long()
                ok = (page >= 0) & (page < len(s["k"]))  # before any of it is used as an index
                t, page = t[ok], page[ok]
                kk, vv = s["k"][page, g, t % P][:, None].expand(-1, G, -1), s["v"][page, g, t % P][:, None].expand(-1, G, -1)
                if len(t) == 0:
                    parts.append((torch.zeros((1, G, hd), dtype=torch.float64, device=DEV),) * 2 + (torch.zeros((1, G), dtype=torch.float64, device=DEV),))
                else:
                    parts.append(attention_ref(q[:, g * G:(g + 1) * G], kk, vv, scale, torch.ones((1, len(t)), dtype=torch.bool, device=DEV)))
            o, wv, size = (torch.cat([p[c] for p in parts], 1) for c in range(3))
            outs.append(o)
            tols.append(attention_tol(o, wv, size, hd, qt, kt))
            row += 1
    return torch.cat(outs), torch.cat(tols)


ATTEND = [
    # lens, fresh, H, KVH, hd, P, prefix pages, order
    ([1], [1], 8, 4, 8, 32, 0, "heads"),
    ([1, 2, 31, 32, 33, 500], [1] * 6, 4, 4, 80, 32, 0, "heads"),
    ([0, 7, 0, 130], [1, 1, 1, 1], 8, 2, 64, 16, 0, "positions"),           # rows that see nothing
    ([5, 64, 200], [5, 3, 9], 8, 1, 128, 16, 0, "heads"),                    # several tokens each
    ([40, 41, 70, 300], [1, 1, 1, 1], 4, 4, 80, 16, 2, "heads"),            # a shared prefix of two pages
    ([33, 64, 65, 200], [1, 0, 2, 4], 8, 2, 64, 32, 1, "both"),             # and ragged tokens, one request without any
    ([3, 90, 17, 300], [3, 2, 1, 6], 8, 8, 40, 24, 3, "heads"),             # requests shorter than the prefix
    ([700, 900, 650], [1, 1, 1], 32, 2, 128, 32, 20, "heads"),              # groups of 16
    ([300, 257], [2, 1], 64, 1, 64, 32, 4, "positions"),                    # a group of 64
    ([130, 77, 259], [1, 1, 1], 6, 2, 256, 13, 3, "heads"),                 # pages of 13, three heads a group
    ([100, 90], [1, 1], 5, 5, 200, 1, 7, "heads"),                          # pages of one position
    ([600, 513, 512, 511], [64, 33, 1, 17], 8, 2, 96, 64, 4, "heads"),      # chunks of a prefill
    ([2100, 1300], [1, 1], 4, 2, 64, 128, 10, "heads"),                     # pages of 128
    ([90, 200], [1, 7], 4, 2, 72, 512, 0, "heads"),                         # one page holds everything
]


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("case", range(len(ATTEND)))
def test_attend(qt, kt, case):
    lens, fresh, H, KVH, hd, P, prefix, order = ATTEND[case]
    qt, kt = TYPES[qt], TYPES[kt]
    s = attention_state(lens, fresh, H, KVH, hd, P, qt, kt, seed=case, prefix=prefix, order=order, q_order="rows" if case % 2 else "heads")
    scale = 1.3 / math.sqrt(hd)
    out = torch.full((s["T"] + 2, H, hd), 5.0, dtype=qt, device=DEV)
    paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], max(fresh), prefix=s["prefix"] if prefix else None, scale=scale,
                                       max_length=s["lim"] if case % 3 else 0, out=out)
    want, tol = expected(s, lens, fresh, H, KVH, hd, P, scale, prefix)
    near(out[:s["T"]], want, tol)
    assert bool((out[s["T"]:] == 5).all())  # rows behind the last request


LONG = [
    # lens, fresh, H, KVH, hd, P, prefix pages: kernels and joins that only many or long requests reach
    ([2048 + 17 + i % 5 for i in range(64)], [1] * 64, 2, 2, 64, 16, 128),   # a prefix of its own kernel for every type
    ([2048 + 60 + i % 9 for i in range(40)], [1 + i % 3 for i in range(40)], 6, 2, 128, 32, 64),
    ([9000], [1], 4, 2, 128, 32, 0),                                          # more parts than a cluster joins
    ([5000, 4200], [3, 1], 8, 2, 256, 16, 40),
    ([3000, 900], [1, 1], 4, 4, 80, 7, 0),                                    # eight parts, pages of 7
    ([1200, 1300, 0, 40], [1, 2, 1, 1], 20, 1, 64, 16, 0),                    # clusters with parts that have nothing
]


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("case", range(len(LONG)))
def test_attend_long(qt, kt, case):
    lens, fresh, H, KVH, hd, P, prefix = LONG[case]
    qt, kt = TYPES[qt], TYPES[kt]
    s = attention_state(lens, fresh, H, KVH, hd, P, qt, kt, seed=40 + case, prefix=prefix)
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], max(fresh), prefix=s["prefix"] if prefix else None,
                                             max_length=s["lim"])
    want, tol = expected(s, lens, fresh, H, KVH, hd, P, 1 / math.sqrt(hd), prefix)
    # Sums over up to 9,000 positions, 2,304 in one chain of a lane at most.
    near(out[:s["T"]], want, 2 * tol)


def test_out_may_be_q():
    """The queries' own buffer as the output: each row is read before it is written."""
    for n, prefix, lens in ((3, 0, [700, 90, 33]), (48, 40, [1280 + i for i in range(48)]), (1, 0, [9000])):
        s = attention_state(lens, [1] * n, 8, 2, 64, 32, torch.bfloat16, torch.bfloat16, seed=n, prefix=prefix)
        c = paged.Cache(s["k"], s["v"])
        args = (s["table"], s["starts"], s["lengths"], 1)
        want = c.attend(s["q"], *args, prefix=s["prefix"] if prefix else None)
        q = s["q"].clone()
        c.attend(q, *args, prefix=s["prefix"] if prefix else None, out=q)
        assert torch.equal(q[:n], want[:n])


def test_a_max_length_that_cuts():
    """Positions from max_length on are not attended."""
    s = attention_state([100, 40], [1, 1], 4, 2, 64, 16, torch.float32, torch.float32, seed=2)
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1, max_length=64)
    want, tol = expected(s, [64, 40], [1, 1], 4, 2, 64, 16, 1 / 8, 0)
    near(out[:2], want, tol)


FIRST_CALL = """
import torch
from tinyoai_b200 import paged
n = 40
k = torch.randn(64 + n, 2, 16, 64, device="cuda").bfloat16(); v = torch.randn_like(k)
c = paged.Cache(k, v)
held = torch.full((n,), 1030, dtype=torch.int32, device="cuda"); fresh = torch.ones_like(held)
tables = torch.arange(65, device="cuda").int().repeat(n, 1)
tables[:, 64] += torch.arange(n, device="cuda").int()  # a page of its own behind the shared ones
plan = paged.StepPlan(n, n, 16)
qkv = torch.randn(n, 8 * 64, device="cuda").bfloat16()
free = tables[0].clone(); prefix = tables[0, :64].clone()
means = torch.zeros(64 + n, 2, 64, dtype=torch.bfloat16, device="cuda")
def step():
    plan.build(held, fresh, tables, free)
    q = c.append(qkv, 4, plan.positions, plan.slots)
    c.page_means(plan.slots, means)
    return c.attend(q, tables, plan.starts, plan.lengths, 1, prefix=prefix), *c.attend_sparse(q, means, tables, plan.starts, plan.lengths, 1, top=3)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = step()
g.replay()
torch.cuda.synchronize()
got = [x.clone() for x in got]
want = step()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print("same")
"""


def test_first_calls_inside_a_capture():
    """A process whose first calls of all are captured ones."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_calls_from_two_threads():
    """One cache, two threads, different shapes, each on a stream of its own."""
    import threading
    s = attention_state([900, 700, 333, 64], [1] * 4, 16, 4, 128, 32, torch.bfloat16, torch.bfloat16, seed=6)
    c = paged.Cache(s["k"], s["v"])
    whole = (s["q"], s["table"], s["starts"], s["lengths"])
    part = (s["q"][:2].clone(), s["table"][:2], s["starts"][:3], s["lengths"][:2])
    want = [c.attend(*a, 1).clone() for a in (whole, part)]
    torch.cuda.synchronize()
    bad = []

    def work(args, w, rows):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            for _ in range(50):
                if not torch.equal(c.attend(*args, 1)[:rows], w[:rows]):
                    bad.append(rows)

    threads = [threading.Thread(target=work, args=a) for a in ((whole, want[0], 4), (part, want[1], 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


SHARED = [
    # requests, fresh, H, KVH, hd, P, prefix pages, own positions, order: row tiles of the tensor cores
    (40, 1, 4, 4, 80, 32, 17, 40, "heads"),          # one tile, the streams take alternate blocks, a part block at the end
    (33, 1, 2, 1, 64, 8, 64, 9, "positions"),        # pages of 8, one 64-feature operand
    (128, 1, 8, 8, 128, 16, 40, 33, "heads"),        # a full tile
    (129, 1, 4, 4, 128, 64, 9, 70, "both"),          # two tiles, the second almost empty
    (70, 3, 16, 2, 128, 32, 33, 5, "heads"),         # three tokens each, groups of 8
    (100, 1, 28, 4, 112, 128, 5, 20, "heads"),       # groups of 7, pages of 128
    (20, 2, 64, 1, 96, 256, 3, 300, "positions"),    # a group of 64, pages of 256
    (300, 1, 4, 2, 72, 32, 24, 64, "heads"),         # 72 features
    (64, 1, 2, 2, 64, 32, 150, 0, "heads"),          # nothing but the prefix
]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(SHARED)))
def test_attend_shared_prefix_tiles(t, case):
    n, fresh, H, KVH, hd, P, prefix, own, order = SHARED[case]
    dt = TYPES[t]
    lens = [prefix * P + (own * (i * 7 % 11)) // 10 for i in range(n)]
    f = [1 + i % fresh for i in range(n)]
    if case % 2:
        lens[3], lens[5] = prefix * P // 2, 0  # shorter than the prefix, and empty
        f[4] = 0
    s = attention_state(lens, f, H, KVH, hd, P, dt, dt, seed=70 + case, prefix=prefix, order=order)
    for scale in (1 / math.sqrt(hd), -0.7 / math.sqrt(hd), 0.0)[: 3 if case < 2 else 1]:
        out = torch.full((s["T"] + 2, H, hd), 5.0, dtype=dt, device=DEV)
        paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], max(f), prefix=s["prefix"], scale=scale,
                                           max_length=s["lim"], out=out)
        want, tol = expected(s, lens, f, H, KVH, hd, P, scale, prefix)
        near(out[:s["T"]], want, tol)
        assert bool((out[s["T"]:] == 5).all())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("n", [48, 200])
def test_attend_prefix_with_missing_pages(t, n):
    """Ids outside the pool among the prefix's pages; a growing score, so that rows move their reference again and again."""
    dt, P, prefix, hd = TYPES[t], 32, 40, 64
    lens = [prefix * P + 1 + i % 40 for i in range(n)]
    s = attention_state(lens, [1] * n, 2, 2, hd, P, dt, dt, seed=5, prefix=prefix)
    for j in range(prefix):
        s["k"][s["prefix"][j].long()] *= 0.2 + j / 4
    s["prefix"][3], s["prefix"][4], s["prefix"][17], s["prefix"][39] = -1, 10 ** 6, -7, len(s["k"])
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"])
    want, tol = expected(s, lens, [1] * n, 2, 2, hd, P, 1 / math.sqrt(hd), prefix)
    near(out[:n], want, tol)


@pytest.mark.parametrize("qt, kt", PAIRS)
def test_attend_ignores_missing_pages_and_stale_values(qt, kt):
    """Page ids outside the pool are no pages; the values behind a request's
    length (infinities and NaN here) and in other pages never show."""
    qt, kt = TYPES[qt], TYPES[kt]
    lens, fresh = [100, 64, 33], [1, 1, 1]
    for fill in (math.inf, math.nan, -math.inf):
        s = attention_state(lens, fresh, 4, 2, 64, 16, qt, kt, seed=9, fill=fill)
        s["table"][0, 2] = -1
        s["table"][1, 1] = 10 ** 6
        s["table"][2, :] = -5  # nothing at all: a row of zeros
        out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1)
        want, tol = expected(s, lens, fresh, 4, 2, 64, 16, 1 / math.sqrt(64), 0)
        near(out[:3], want, tol)
        assert bool((out[2] == 0).all())


UNSEEN = [
    # lens, fresh, H, KVH, hd, P, prefix pages, (request, position) of the values that are no numbers
    ([70, 300], [8, 5], 8, 2, 64, 16, 0, (0, 66)),                                # later tokens of a chunk
    ([70, 300], [8, 5], 8, 2, 64, 16, 0, (1, 299)),                               # the last of all
    ([3000], [40], 2, 1, 80, 7, 0, (0, 2965)),                                    # parts joined in a cluster, pages of 7
    ([9000], [3], 4, 2, 256, 32, 0, (0, 8998)),                                   # and in a join of their own
    ([40, 300, 33], [2, 4, 1], 4, 2, 128, 32, 4, (1, 100)),                       # requests shorter than a short prefix
    ([2100] * 26 + [700, 1, 0, 1999], [1] * 30, 2, 2, 128, 16, 128, (0, 1200)),   # a prefix of its own kernel
    ([2100] * 41 + [700, 1, 0, 1200, 1201], [1] * 46, 2, 2, 128, 16, 128, (0, 1200)),   # of tensor-core tiles: one tile
    ([2100] * 41 + [700, 1, 0, 1200, 1201], [1] * 46, 8, 2, 80, 32, 64, (0, 2047)),     # two, the prefix's last position
    ([700] * 40 + [1201] * 2, [1] * 42, 4, 2, 64, 8, 256, (40, 1200)),            # most see little of it
]


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("case", range(len(UNSEEN)))
def test_attend_values_of_unseen_positions(qt, kt, case):
    """Infinities and NaN at a position that later rows of the step, or longer
    requests, attend to stay out of the rows that do not."""
    lens, fresh, H, KVH, hd, P, prefix, (i, x) = UNSEEN[case]
    qt, kt = TYPES[qt], TYPES[kt]
    for fill in (math.inf, math.nan):
        s = attention_state(lens, fresh, H, KVH, hd, P, qt, kt, seed=50 + case, prefix=prefix)
        page = (s["prefix"] if x // P < prefix else s["table"][i])[x // P].long()
        s["v"][page, :, x % P, ::3] = fill
        if fill != fill:
            s["k"][page, 0, x % P, 1] = fill
        out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], max(fresh), prefix=s["prefix"] if prefix else None,
                                                 max_length=s["lim"])[:s["T"]]
        want, tol = expected(s, lens, fresh, H, KVH, hd, P, 1 / math.sqrt(hd), prefix)
        there = want.isfinite()
        rows = there.all(-1).all(-1)
        assert bool(rows.any()) and not bool(rows.all())
        assert torch.equal(out.isfinite(), there)
        near(out[there], want[there], (2 if max(lens) > 2000 else 1) * tol[there])  # long sums as above


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("prefix", [0, 2, 300])
def test_rows_before_the_first_position(qt, kt, prefix):
    """Requests shorter than their tokens of the step: rows at -1, -2, -9 are zero, in every attention."""
    lens, fresh, H, KVH, hd, P = [1, 0, 5, 40], [9, 6, 5, 3], 4, 2, 64, 16
    if prefix == 300:
        lens, fresh = [1, 0, 5] + [4840] * 30, [9, 6, 5] + [1] * 30
    qt, kt = TYPES[qt], TYPES[kt]
    s = attention_state(lens, fresh, H, KVH, hd, P, qt, kt, seed=31, prefix=prefix)
    before = torch.cat([torch.arange(f, device=DEV) < f - x for x, f in zip(lens, fresh)])
    c = paged.Cache(s["k"], s["v"])
    out = torch.full((s["T"] + 2, H, hd), 5.0, dtype=qt, device=DEV)
    c.attend(s["q"], s["table"], s["starts"], s["lengths"], max(fresh), prefix=s["prefix"] if prefix else None, out=out)
    want, tol = expected(s, lens, fresh, H, KVH, hd, P, 1 / math.sqrt(hd), prefix)
    near(out[:s["T"]], want, (2 if prefix == 300 else 1) * tol)
    assert bool((out[:s["T"]][before] == 0).all()) and bool((out[s["T"]:] == 5).all())
    if prefix == 0:
        means = torch.zeros((len(s["k"]), KVH, hd), dtype=kt, device=DEV)
        out.fill_(5.0)
        got, pages = c.attend_sparse(s["q"], means, s["table"], s["starts"], s["lengths"], max(fresh), first=1, last=1, top=1, out=out)
        assert bool((out[:s["T"]][before] == 0).all()) and bool((pages[:s["T"]][before] == -1).all())
        near(out[:s["T"]], want, tol)  # three pages hold every request


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strides_of_dimensions_of_one(t):
    """One row, one head, one page, one position: what torch keeps as that dimension's stride is no stride."""
    dt, hd = TYPES[t], 64
    for lens, fresh, H, P in (([5], [1], 1, 8), ([1], [1], 1, 1), ([9], [3], 1, 16), ([40], [1], 2, 8)):
        s = attention_state(lens, fresh, H, 1, hd, P, dt, dt, seed=len(lens) + P)
        args = (s["table"], s["starts"], s["lengths"], max(fresh))
        want, tol = expected(s, lens, fresh, H, 1, hd, P, 1 / math.sqrt(hd), 0)
        near(paged.Cache(s["k"], s["v"]).attend(s["q"], *args)[:s["T"]], want, tol)

        def odd(x):  # dimensions of one get a stride of 3
            return x.as_strided(x.shape, [st if n > 1 else 3 for n, st in zip(x.shape[:-1], x.stride())] + [1])
        k, v, q = (odd(x) for x in (s["k"], s["v"], s["q"][:s["T"]].clone()))
        out = odd(torch.zeros_like(q))
        paged.Cache(k, s["v"]).attend(q, *args, out=out)
        near(out, want, tol)
        near(paged.Cache(k, v).attend(q, *args), want, tol)


@pytest.mark.parametrize("qt, kt", PAIRS)
def test_attend_extreme_scores(qt, kt):
    """Scores far apart and scores at the type's lowest value: one position
    takes all the weight, or all weights are equal."""
    qt, kt = TYPES[qt], TYPES[kt]
    lens = [200]
    s = attention_state(lens, [1], 2, 1, 64, 16, qt, kt, seed=4, fill=0.0)
    t = torch.arange(200, device=DEV)
    page = s["table"][0][t // 16].long()
    s["q"].fill_(1.0)
    s["k"].fill_(-200.0)
    s["k"][page[77], 0, 77 % 16] = 200.0
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1, scale=1.0)
    near(out[0, 0], s["v"][page[77], 0, 77 % 16].double(), 2 * unit(qt) * s["v"][page[77], 0, 77 % 16].double().abs())
    s["k"].fill_(torch.finfo(kt).min if kt == torch.float16 else -1e30)
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1, scale=1.0)
    v = s["v"][page, 0, t % 16].double()
    near(out[0, 0], v.mean(0), (2.0 ** -13 + unit(kt)) * v.abs().mean(0) + unit(qt) * v.mean(0).abs())


# ---------------------------------------------------------------------------
# Sparse attention


def choose_ref(q, means, table, pos, P, first, last, top, pages_in_pool):
    """Pages of one query, for each KV head: q [KVH, G, hd], means [pages, KVH, hd]."""
    npages = pos // P + 1 if pos >= 0 else 0
    got = []
    for g in range(means.shape[1]):
        lo, hi = min(first, npages), max(min(first, npages), npages - last)
        scored = []
        for b in range(lo, hi):
            p = int(table[b])
            if not 0 <= p < pages_in_pool:
                scored.append((2, 0.0, b))
                continue
            s = float((q[g].double() @ means[p, g].double()).amax())
            scored.append((1, 0.0, b) if math.isnan(s) else (0, -s, b))
        best = {b for _, _, b in sorted(scored)[:top]}
        got.append(sorted(best | set(range(lo)) | set(range(hi, npages))))
    return got


SPARSE = [
    # lens, fresh, H, KVH, hd, P, first, last, top, order
    ([1], [1], 8, 4, 8, 32, 1, 1, 2, "heads"),
    ([500, 129, 33, 16, 0], [1] * 5, 8, 2, 64, 16, 1, 1, 4, "heads"),
    ([700, 640], [1, 1], 4, 4, 80, 32, 0, 2, 3, "positions"),
    ([1500, 900], [3, 2], 8, 1, 128, 16, 2, 1, 9, "heads"),
    ([2000], [1], 16, 2, 64, 7, 0, 1, 0, "heads"),                 # only the last page
    ([300, 280], [1, 1], 6, 2, 256, 13, 3, 4, 5, "both"),
    ([9000], [2], 4, 2, 64, 16, 1, 3, 100, "heads"),               # several tiles of pages
    ([64, 65], [1, 1], 32, 1, 40, 1, 0, 1, 20, "heads"),
    ([400], [1], 4, 2, 64, 16, 1, 1, 64, "heads"),                 # more room than pages: everything
    ([9000, 8000], [1, 1], 4, 2, 64, 16, 1, 1, 300, "heads"),      # more parts than a cluster joins
    ([20011], [1], 2, 1, 64, 2, 1, 2, 700, "heads"),               # ten thousand pages: scores that do not all stay in shared memory
    ([2200], [1], 2, 2, 64, 1, 0, 1, 1500, "positions"),           # over a thousand pages of one position
]


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("case", range(len(SPARSE)))
def test_attend_sparse(qt, kt, case):
    lens, fresh, H, KVH, hd, P, first, last, top, order = SPARSE[case]
    qt, kt = TYPES[qt], TYPES[kt]
    s = attention_state(lens, fresh, H, KVH, hd, P, qt, kt, seed=20 + case, order=order)
    means = torch.nan_to_num(s["k"].float(), nan=0.0).mean(2).to(kt)
    if case in (1, 3):  # equal scores: ties go to the lower page
        means[:] = means[0]
    if case == 6:  # a NaN mean ranks last, infinite ones where they belong
        means[s["table"][0, 5].long()] = math.nan
        means[s["table"][0, 9].long(), :, 0] = math.inf
    out = torch.full((s["T"] + 2, H, hd), 5.0, dtype=qt, device=DEV)
    pages = torch.full((s["T"] + 2, KVH, first + last + top), -9, dtype=torch.int32, device=DEV)
    paged.Cache(s["k"], s["v"]).attend_sparse(s["q"], means, s["table"], s["starts"], s["lengths"], max(fresh), top=top, first=first, last=last, out=out,
                                              pages=pages)
    chosen, row = [], 0
    for i, (x, f) in enumerate(zip(lens, fresh)):
        for j in range(f):
            pos = x - f + j
            want = choose_ref(s["q"][row].reshape(KVH, H // KVH, hd), means, s["table"][i], pos, P, first, last, top, len(s["k"]))
            assert pages[row].tolist() == [w + [-1] * (first + last + top - len(w)) for w in want], (row, pos)
            chosen.append(want)
            row += 1
    want, tol = expected(s, lens, fresh, H, KVH, hd, P, 1 / math.sqrt(hd), 0, chosen)
    near(out[:s["T"]], want, tol)
    assert bool((out[s["T"]:] == 5).all()) and bool((pages[s["T"]:] == -9).all())


def test_sparse_over_everything_is_attend():
    s = attention_state([300, 77], [2, 1], 8, 2, 64, 16, torch.float32, torch.float32, seed=3)
    c = paged.Cache(s["k"], s["v"])
    means = torch.nan_to_num(s["k"], nan=0.0).mean(2)
    dense = c.attend(s["q"], s["table"], s["starts"], s["lengths"], 2)[:3]
    sparse, _ = c.attend_sparse(s["q"], means, s["table"], s["starts"], s["lengths"], 2, top=40)
    near(sparse[:3], dense.double(), 2.0 ** -18 * dense.abs().amax())


# ---------------------------------------------------------------------------
# Large offsets, streams, graphs


def test_offsets_past_32_bits():
    """A pool of 2.4e9 values: pages at its end."""
    g = gen(1)
    P, KVH, hd = 32, 8, 128
    pages = 73400
    k = torch.empty((pages, KVH, P, hd), dtype=torch.float16, device=DEV)
    v = torch.empty((pages, KVH, P, hd), dtype=torch.float16, device=DEV)
    assert k.numel() > 2 ** 31
    c = paged.Cache(k, v)
    H, n = 16, 3
    tables = i32([[pages - 1, 0], [pages - 2, pages - 4], [1, pages - 3]])
    qkv = normal((n, (H + 2 * KVH) * hd), g, torch.float16)
    hist = normal((n, 40, 2, KVH, hd), g, torch.float16)
    for i in range(n):
        for t in range(40):
            k[int(tables[i, t // P]), :, t % P], v[int(tables[i, t // P]), :, t % P] = hist[i, t, 0], hist[i, t, 1]
    plan = paged.StepPlan(n, n, P, DEV)
    plan.build(i32([39, 31, 32]), i32([1, 1, 1]), tables, i32([pages - 3]))  # the third request begins a page
    assert plan.slots.tolist() == [0 * P + 7, (pages - 2) * P + 31, (pages - 3) * P]
    q = c.append(qkv, H, plan.positions, plan.slots)
    means = torch.zeros((pages, KVH, hd), dtype=torch.float16, device=DEV)
    c.page_means(plan.slots, means)
    near(means[pages - 2], k[pages - 2].double().mean(1), 2.0 ** -11 * 4)
    out = c.attend(q, tables, plan.starts, plan.lengths, 1)
    out2, _ = c.attend_sparse(q, means, tables, plan.starts, plan.lengths, 1, top=1)
    s = dict(k=k, v=v, table=tables, q=q, prefix=i32([]))
    want, tol = expected(s, [40, 32, 33], [1, 1, 1], H, KVH, hd, P, 1 / math.sqrt(hd), 0)
    near(out, want, tol)
    near(out2, want, tol)


def step_state(seed, qt, kt, n=6, H=8, KVH=2, hd=64, P=16, pages=64, width=8):
    g = gen(seed)
    k, v = make_cache(pages, KVH, P, hd, kt, g, fill=math.nan)
    return dict(c=paged.Cache(k, v), plan=paged.StepPlan(n, 64, P, DEV), tables=torch.full((n, width), -1, dtype=torch.int32, device=DEV),
                means=torch.zeros((pages, KVH, hd), dtype=kt, device=DEV), table=torch.rand((256, 16, 2), generator=g, device=DEV),
                norm=paged.HeadNorm("rms", 1 + normal((1, hd), g, scale=0.1), 1 + normal((1, hd), g, scale=0.1), 1e-6), H=H, KVH=KVH, hd=hd, P=P, n=n,
                qkv=normal((64, (H + 2 * KVH) * hd), g, qt), free=torch.randperm(pages, generator=g, device=DEV).to(torch.int32))


def whole_step(s, held, fresh, free, most):
    s["plan"].build(held, fresh, s["tables"], free)
    p = s["plan"]
    q = s["c"].append(s["qkv"], s["H"], p.positions, p.slots, rotary=paged.Rotary(s["table"]), norm=s["norm"])
    s["c"].page_means(p.slots, s["means"])
    dense = s["c"].attend(q, s["tables"], p.starts, p.lengths, most)
    sparse, pages = s["c"].attend_sparse(q, s["means"], s["tables"], p.starts, p.lengths, most, top=2, first=1, last=1)
    return q, dense, sparse, pages


@pytest.mark.parametrize("qt, kt", PAIRS)
def test_steps_together(qt, kt):
    """A prefill of ragged prompts, then decode steps, each a plan, an append,
    page means and both attentions, against float64 attention over the history
    that the cache holds; the history itself against the rows appended."""
    qt, kt = TYPES[qt], TYPES[kt]
    s = step_state(2, qt, kt)
    n, H, KVH, hd, P = s["n"], s["H"], s["KVH"], s["hd"], s["P"]
    held, taken = [0] * n, 0
    history = [[] for _ in range(n)]
    for step, fresh in enumerate([[5, 16, 1, 17, 0, 9], [1, 1, 1, 1, 3, 1], [1, 1, 1, 1, 1, 1], [1, 0, 1, 15, 1, 1], [1] * n]):
        s["qkv"].copy_(normal(s["qkv"].shape, gen(50 + step), qt))
        q, dense, sparse, pages = whole_step(s, i32(held), i32(fresh), s["free"][taken:], max(fresh))
        counts = s["plan"].counts.tolist()
        assert counts[:2] == [n, sum(fresh)]
        taken += counts[2]
        x = s["qkv"].reshape(64, H + 2 * KVH, hd)[:sum(fresh)]
        pos = s["plan"].positions[:sum(fresh)].long()
        qr, kr, vr = append_ref(x, H, KVH, "rms", 1e-6, s["norm"].q_weight, s["norm"].k_weight, s["table"], pos, False)
        row = 0
        for i, f in enumerate(fresh):
            for j in range(f):
                history[i].append((kr[row + j], vr[row + j]))
            row += f
            held[i] += f
        # The cache holds the history.
        for i in range(n):
            if not held[i]:
                continue
            t = torch.arange(held[i], device=DEV)
            page = s["tables"][i][t // P].long()
            for got, want in ((s["c"].k, torch.stack([h[0] for h in history[i]])), (s["c"].v, torch.stack([h[1] for h in history[i]]))):
                near(got[page, :, t % P], want, 64 * 2.0 ** -24 * want.abs().amax(-1, keepdim=True) + unit(kt) * want.abs() + 2.0 ** -25)
        near(q[:sum(fresh)], qr, 64 * 2.0 ** -24 * qr.abs().amax(-1, keepdim=True) + unit(qt) * qr.abs() + 2.0 ** -25)
        ref = dict(k=s["c"].k, v=s["c"].v, table=s["tables"], q=q, prefix=i32([]))
        want, tol = expected(ref, held, fresh, H, KVH, hd, P, 1 / math.sqrt(hd), 0)
        near(dense[:sum(fresh)], want, tol)
        chosen, row = [], 0
        for i, f in enumerate(fresh):
            for j in range(f):
                w = choose_ref(q[row].reshape(KVH, H // KVH, hd), s["means"], s["tables"][i], held[i] - f + j, P, 1, 1, 2, s["c"].num_pages)
                assert [[b for b in r if b >= 0] for r in pages[row].tolist()] == w
                chosen.append(w)
                row += 1
        want, tol = expected(ref, held, fresh, H, KVH, hd, P, 1 / math.sqrt(hd), 0, chosen)
        near(sparse[:sum(fresh)], want, tol)


@pytest.mark.parametrize("qt, kt", [("bf16", "bf16"), ("f32", "f16")])
def test_captured_steps(qt, kt):
    """A whole step captured into a CUDA graph, replayed for other lengths and
    rows, equals the same calls made eagerly, with the same bits; two graphs of
    one cache do not share a workspace."""
    qt, kt = TYPES[qt], TYPES[kt]
    a, b = step_state(7, qt, kt), step_state(7, qt, kt)
    fresh = [[5, 3, 1, 2, 0, 9], [1] * 6, [1, 1, 0, 1, 1, 1]]
    held = torch.zeros(6, dtype=torch.int32, device=DEV)
    free = torch.zeros(40, dtype=torch.int32, device=DEV)
    new = torch.zeros(6, dtype=torch.int32, device=DEV)
    whole_step(a, held, new, free, 9)  # first use outside the capture
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = whole_step(a, held, new, free, 9)
        graphs.append((gr, res))
    taken, at = 0, [0] * 6
    for step, f in enumerate(fresh):
        rows = normal(a["qkv"].shape, gen(90 + step), qt)
        a["qkv"].copy_(rows)
        b["qkv"].copy_(rows)
        held.copy_(i32(at))
        new.copy_(i32(f))
        free.copy_(a["free"][taken:taken + 40] if taken + 40 <= 64 else a["free"][24:])
        gr, res = graphs[step % 2]
        gr.replay()
        want = whole_step(b, i32(at), i32(f), free.clone(), 9)
        n = sum(f)
        for x, y in zip(res, want):
            assert torch.equal(x[:n], y[:n])
        assert torch.equal(a["plan"].slots, b["plan"].slots) and torch.equal(a["tables"], b["tables"])
        assert torch.equal(a["c"].k.nan_to_num(5), b["c"].k.nan_to_num(5))
        taken += a["plan"].counts.tolist()[2]
        at = [x + y for x, y in zip(at, f)]
    del graphs


def test_two_streams_at_once():
    """Attention on two streams over one cache, many times, with the same bits as alone."""
    s = attention_state([900, 700, 333, 64], [1] * 4, 16, 4, 128, 32, torch.bfloat16, torch.bfloat16, seed=6, prefix=2)
    c = paged.Cache(s["k"], s["v"])
    q2 = s["q"].flip(0).contiguous()
    want1 = c.attend(s["q"], s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"]).clone()
    want2 = c.attend(q2, s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"]).clone()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    outs = [(c.attend(s["q"], s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"], stream=one), torch.empty_like(want2)) for _ in range(20)]
    for x, y in outs:
        with torch.cuda.stream(two):
            c.attend(q2, s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"], out=y)
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x[:4], want1[:4]) and torch.equal(y[:4], want2[:4])


def test_refusals():
    g = gen(1)
    k, v = make_cache(4, 2, 16, 64, torch.float16, g)
    c = paged.Cache(k, v)
    t = torch.zeros((1, 4), dtype=torch.int32, device=DEV)
    q = normal((1, 4, 64), g, torch.float16)
    st, le = i32([0, 1]), i32([5])

    def bad(f, text, code=_lib.TCU_EINVAL):
        with pytest.raises(BackendError) as e:
            f()
        assert e.value.code == code and text in str(e.value), str(e.value)

    bad(lambda: paged.Cache(k.cpu(), v.cpu()), "on a GPU")
    bad(lambda: paged.Cache(k, v[:2]), "one shape")
    bad(lambda: paged.Cache(k.transpose(2, 3), v.transpose(2, 3)), "contiguous last")
    bad(lambda: paged.Cache(k.double(), v.double()), "float64", _lib.TCU_EUNSUP)
    bad(lambda: c.attend(q.cpu(), t, st, le, 1), "q must be")
    bad(lambda: c.attend(q[..., :32], t, st, le, 1), "q must be")
    bad(lambda: c.attend(q.bfloat16(), t, st, le, 1), "cache's type", _lib.TCU_EUNSUP)
    bad(lambda: c.attend(q, t.long(), st, le, 1), "tables must be")
    bad(lambda: c.attend(q, t, st, i32([5, 6]), 1), "2 lengths")
    bad(lambda: c.attend(q, t, st, le, 0), "max_fresh")
    bad(lambda: c.attend(q, t, st, le, 1, prefix=st.cpu()), "prefix must be")
    bad(lambda: c.attend(q, t, st, le, 1, out=q.float()), "out must be")
    bad(lambda: c.attend(normal((1, 4, 72), g, torch.float16)[..., 4:68], t, st, le, 1), "16-byte aligned")
    bad(lambda: c.attend_sparse(q, k[:, :, 0].float(), t, st, le, 1, top=1), "means must be")
    bad(lambda: c.attend_sparse(q, k[:, :, 0].contiguous(), t, st, le, 1, top=-1), "must not be negative")
    bad(lambda: c.append(normal((1, 8 * 64 + 8), g, torch.float16), 4, i32([0]), torch.zeros(1, dtype=torch.int64, device=DEV)), "qkv must be")
    bad(lambda: c.append(normal((1, 8 * 64), g, torch.float16), 4, i32([0]), i32([0])), "slots must be")
    bad(lambda: paged.HeadNorm("max", q[0].float(), q[0].float(), 0.0), "unknown norm")
    bad(lambda: paged.StepPlan(1, 1, 16, "cpu"), "lives on a GPU")
    bad(lambda: paged.StepPlan(1, 1, 16, DEV).build(i32([1, 2]), i32([1, 2]), t, i32([])), "room for 1")
    # A workspace that is too small or not aligned, and host memory, at the C entry.
    wide = torch.zeros((1, 4096), dtype=torch.int32, device=DEV)
    out, qs = c._queries(q, wide, st, le, 1, None, None, None)
    L = _lib.lib()
    w = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    assert L.tcu_paged_attend(0, None, c._ref, qs, None, 0, 0, w.data_ptr(), 16) == _lib.TCU_EINVAL
    assert b"workspace of 16 bytes" in L.tcu_last_error()
    assert L.tcu_paged_attend(0, None, c._ref, qs, None, 0, 0, w.data_ptr() + 16, 1 << 19) == _lib.TCU_EINVAL
    assert b"256-byte aligned" in L.tcu_last_error()
    host = torch.zeros(1 << 20, dtype=torch.uint8)
    assert L.tcu_paged_attend(0, None, c._ref, qs, None, 0, 0, (host.data_ptr() + 255) // 256 * 256, 1 << 19) == _lib.TCU_EINVAL
    assert b"device memory" in L.tcu_last_error()
    assert L.tcu_paged_attend(7, None, c._ref, qs, None, 0, 0, w.data_ptr(), 1 << 20) == _lib.TCU_ENODEV
    # Nothing to do is not an error.
    none = torch.zeros((0, 4, 64), dtype=torch.float16, device=DEV)
    assert c.attend(none, t[:0], i32([0]), i32([]), 1).shape == (0, 4, 64)
    assert c.append(normal((0, 8 * 64), g, torch.float16), 4, i32([]), torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# The batch step of the library's own sessions


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads, kv_heads, hidden", [(4, 4, 320), (8, 2, 512)])
def test_batch_of_forks_shares_its_prefix(kv, heads, kv_heads, hidden):
    """Forks of one session advance together with share_prefix on; every row
    equals the same step with it off (the tolerance of a batch row against a
    session of its own), and so does the cache: the steps after it go on
    unshared. Sessions of other prefixes in the batch turn it off by themselves."""
    import numpy as np

    from tinyoai_b200 import Model
    from tinyoai_b200.synth import prompt_ids, synth_stablelm

    cfg, tensors = synth_stablelm(dict(model_type="stablelm", vocab_size=2048, hidden_size=hidden, intermediate_size=864, num_hidden_layers=3,
                                       num_attention_heads=heads, num_key_value_heads=kv_heads, max_position_embeddings=1024, layer_norm_eps=1e-5,
                                       rope_theta=10000.0, partial_rotary_factor=0.25, use_parallel_residual=True, use_qkv_bias=False,
                                       qk_layernorm=False, tie_word_embeddings=False, hidden_act="silu", bos_token_id=0, eos_token_id=0), "Q8_0", seed=7)
    m = Model.load_stablelm(cfg, tensors)
    opened = []
    try:
        parent = m.session(kv)
        opened.append(parent)
        parent.forward(0, prompt_ids(300, cfg["vocab_size"], seed=1), want_logits=False)
        groups = []
        for _ in range(2):  # the same forks twice: shared and not
            forks = [parent.fork() for _ in range(7)]
            opened.extend(forks)
            for i, f in enumerate(forks):  # ragged continuations of 0 to 40 tokens
                if i:
                    f.forward(300, prompt_ids(i * 7 - 2, cfg["vocab_size"], seed=20 + i), want_logits=False)
            groups.append(forks)
        shared, plain = m.batch(8), m.batch(8)
        opened.extend([shared, plain])
        shared.share_prefix(256)
        toks = prompt_ids(7, cfg["vocab_size"], seed=9)
        for step in range(5):
            if step == 3:
                shared.share_prefix(0)
            rows, ids = shared.forward(groups[0], toks)
            want, want_ids = plain.forward(groups[1], toks)
            for i in range(7):
                span = float(np.max(want[i]) - np.min(want[i]))
                assert float(np.max(np.abs(rows[i] - want[i]))) <= 1e-4 * span, (step, i)
            toks = want_ids.astype(np.int32)
        shared.share_prefix(256)
        other = m.session(kv)
        opened.append(other)
        other.forward(0, prompt_ids(40, cfg["vocab_size"], seed=3), want_logits=False)
        rows, _ = shared.forward([groups[0][0], other], toks[:2])  # nothing in common
        want = other.forward(40, [int(toks[1])])  # the batch step's own position once more
        assert float(np.max(np.abs(rows[1] - want))) <= 1e-4 * float(np.max(want) - np.min(want))
        with pytest.raises(BackendError):
            shared.share_prefix(-1)
    finally:
        for x in reversed(opened):
            x.close()
        m.close()
