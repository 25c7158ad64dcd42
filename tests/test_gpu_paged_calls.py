"""Calls of the operators over a paged KV cache that users make beside the
plain ones: arrays that are inputs and outputs at once, overlapping outputs,
inputs that want gradients, launches that overlap on two streams, bounds inside a
prefix, pages named twice."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from test_gpu_paged import DEV, PAIRS, TYPES, attention_state, expected, gen, i32, near, normal, plan_case, plan_ref  # noqa: E402
from tinyoai_b200 import BackendError, _lib  # noqa: E402

if torch.cuda.is_available():
    from tinyoai_b200 import paged


@pytest.mark.parametrize("n, capacity", [(5, 300), (256, 6000), (1000, 13312)])
@pytest.mark.parametrize("own", ["lengths", "fresh", "starts"])
def test_plan_in_place(n, capacity, own):
    """Lengths that are the next step's held, and lengths or starts over fresh,
    with more tokens than one CTA fills elsewhere: step after step as with arrays apart."""
    P, width = 16, 40
    held, fresh, tables, pages, _, _ = plan_case(n, P, 200, 1, width, 40000, capacity, seed=n)
    plan = paged.StepPlan(n, capacity, P, DEV)
    t = i32(tables)
    starts, lengths, positions, counts = (torch.full((x,), -9, dtype=torch.int32, device=DEV) for x in (n + 1, n, capacity, 3))
    slots = torch.full((capacity,), -9, dtype=torch.int64, device=DEV)
    g = torch.Generator().manual_seed(n)
    h = lengths if own == "lengths" else i32(held)
    for step in range(4):
        fresh = torch.randint(0, 2 * capacity // n + 1 if step % 2 else 2, (n,), generator=g).tolist()
        want = plan_ref(held, fresh, tables, pages, P, capacity)
        free = i32(pages)
        f = i32(fresh)
        if own == "lengths":
            lengths.copy_(i32(held))  # the first step's held
        elif own == "fresh":
            lengths = f
        else:
            starts = torch.cat([f, i32([77])])
            f = starts[:n]
        if own != "lengths":
            h = i32(held)
        rc = _lib.lib().tcu_plan_step(0, torch.cuda.current_stream().cuda_stream, n, h.data_ptr(), f.data_ptr(), P, t.data_ptr(), width, width,
                                      free.data_ptr(), len(pages), capacity, starts.data_ptr(), lengths.data_ptr(), positions.data_ptr(),
                                      slots.data_ptr(), counts.data_ptr())
        assert rc == _lib.TCU_OK, _lib.lib().tcu_last_error()
        got = [x.tolist() for x in (t, starts, lengths, positions, slots, counts)]
        assert got == [list(x) for x in want]
        tables, held, pages = want[0], want[2], pages[want[5][2]:]
    if own == "lengths":  # the plan's own arrays, as the Python class is used
        t2 = t.clone()
        plan.build(i32(held), i32([1] * n), t, i32(pages))
        first = plan.counts.tolist()
        plan.build(plan.lengths, i32([1] * n), t, i32(pages[first[2]:]))
        a = plan_ref(held, [1] * n, t2.tolist(), pages, P, capacity)
        b = plan_ref(a[2], [1] * n, a[0], pages[a[5][2]:], P, capacity)
        assert [t.tolist(), plan.lengths.tolist(), plan.slots.tolist()] == [b[0], b[2], b[4]]


def test_plan_refuses_overlapping_arrays():
    n, cap, width = 8, 32, 4
    buf = torch.zeros(4096, dtype=torch.int32, device=DEV)
    base = buf.data_ptr()
    apart = dict(held=0, fresh=64, tables=128, free=256, starts=384, lengths=512, positions=640, slots=768, counts=1024)

    def call(stride=width, **over):
        at = {k: base + 4 * x for k, x in {**apart, **over}.items()}
        return _lib.lib().tcu_plan_step(0, None, n, at["held"], at["fresh"], 4, at["tables"], width, stride, at["free"], 16, cap, at["starts"], at["lengths"],
                                        at["positions"], at["slots"], at["counts"])

    assert call() == _lib.TCU_OK
    for over in (dict(lengths=0), dict(lengths=64), dict(starts=64), dict(stride=16, held=128 + 4), dict(stride=40, tables=2048, positions=2048 + 4)):
        assert call(**over) == _lib.TCU_OK, over
    for over in (dict(lengths=1), dict(lengths=7), dict(starts=0), dict(starts=60), dict(positions=384), dict(slots=640), dict(counts=8 + 512 - 1),
                 dict(positions=250), dict(tables=0), dict(held=128 + 31), dict(free=128), dict(stride=16, held=128 + 3), dict(stride=16, held=128 + 12),
                 dict(stride=16, positions=128 + 4), dict(starts=64, lengths=64)):
        assert call(**over) == _lib.TCU_EINVAL and b"overlap" in _lib.lib().tcu_last_error(), over


def test_inputs_that_want_gradients():
    """The operators record no gradients: with autograd on such inputs are
    refused, each in its turn; without it they are values like others."""
    H, KVH, hd, P = 4, 2, 64, 16
    g = gen(3)
    k, v = (normal((6, KVH, P, hd), g) for _ in range(2))
    c = paged.Cache(k, v)
    x, table = normal((3, (H + 2 * KVH) * hd), g), torch.rand((64, 8, 2), generator=g, device=DEV)
    qw, kw, means, q = normal((1, hd), g), normal((1, hd), g), normal((6, KVH, hd), g), normal((3, H, hd), g)
    pos, slots, tables, starts, lengths = i32([0, 1, 2]), torch.tensor([0, 1, 2], device=DEV), i32([[0, 1]]), i32([0, 3]), i32([20])
    calls = {
        "append": lambda: c.append(x, H, pos, slots, rotary=paged.Rotary(table), norm=paged.HeadNorm("rms", qw, kw, 1e-5)),
        "page_means": lambda: c.page_means(slots, means),
        "attend": lambda: c.attend(q, tables, starts, lengths, 3),
        "attend_sparse": lambda: c.attend_sparse(q, means, tables, starts, lengths, 3, top=1)[0],
    }
    uses = {"append": (x, k, v, table, qw, kw), "page_means": (k, means), "attend": (q, k, v), "attend_sparse": (q, k, v, means)}
    for name, call in calls.items():
        for t in uses[name]:
            t.requires_grad_(True)
            before = k.detach().clone()
            with pytest.raises(BackendError, match="no gradients") as e:
                call()
            assert e.value.code == _lib.TCU_EUNSUP and torch.equal(k.detach(), before)
            with torch.no_grad():
                out = call()
            t.requires_grad_(False)
            assert torch.equal(out, call())


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("n", [40, 150])
def test_overlapping_launches_on_two_streams(t, n):
    """The shared prefix's kernel with the requests' own positions beside it, on
    two streams at once, eagerly and as captured graphs: the same bits as alone."""
    H, KVH, hd, P, prefix = 4, 2, 128, 32, 40
    lens = [prefix * P + 1 + (i * 37) % 400 for i in range(n)]
    s = attention_state(lens, [1] * n, H, KVH, hd, P, TYPES[t], TYPES[t], seed=n, prefix=prefix)
    c = paged.Cache(s["k"], s["v"])
    qs = [s["q"], s["q"].flip(0).contiguous()]
    call = [lambda out=None, stream=None, q=q: c.attend(q, s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"], out=out, stream=stream) for q in qs]
    want = [f()[:n].clone() for f in call]
    assert all(bool(w.isfinite().all()) for w in want)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[f(stream=st) for _ in range(30)] for f, st in zip(call, streams)]
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(x[:n], w) for x in o)
    graphs = []
    for f in call:
        out = torch.zeros_like(s["q"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(4):  # one call's kernels behind another's
                f(out=out)
        graphs.append((g, out))
    for _ in range(10):
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert torch.equal(out[:n], w)


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("n, most", [(3, 700), (48, 700), (48, 1), (48, 1280), (200, 1100)])
def test_a_max_length_within_the_prefix(qt, kt, n, most):
    """No position from max_length on is attended, also where that ends inside the shared prefix."""
    qt, kt = TYPES[qt], TYPES[kt]
    H, KVH, hd, P, prefix = 4, 2, 64, 32, 40
    lens = [prefix * P + 1 + i % 90 for i in range(n)]
    s = attention_state(lens, [1] * n, H, KVH, hd, P, qt, kt, seed=n, prefix=prefix)
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"], max_length=most)
    cut = [min(x, most) for x in lens]
    want, tol = expected(s, cut, [1] * n, H, KVH, hd, P, 1 / math.sqrt(hd), prefix)
    near(out[:n], want, tol)


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("n", [2, 48])
def test_one_page_in_many_places(qt, kt, n):
    """A page that a prefix and a table name again and again: its positions count each time."""
    qt, kt = TYPES[qt], TYPES[kt]
    H, KVH, hd, P, prefix = 4, 2, 64, 32, 24
    lens = [prefix * P + 70 + i % 20 for i in range(n)]
    s = attention_state(lens, [1] * n, H, KVH, hd, P, qt, kt, seed=n, prefix=prefix)
    s["prefix"][1::2] = s["prefix"][0]
    s["table"][:, prefix:prefix + 2] = s["prefix"][2]
    out = paged.Cache(s["k"], s["v"]).attend(s["q"], s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"])
    want, tol = expected(s, lens, [1] * n, H, KVH, hd, P, 1 / math.sqrt(hd), prefix)
    near(out[:n], want, tol)


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("pairs, norm", [(0, "none"), (6, "rms"), (16, "layer"), (32, "rms")])
def test_append_in_place(qt, kt, pairs, norm):
    """Queries written where they were read from, beside queries in a tensor of their own."""
    qt, kt = TYPES[qt], TYPES[kt]
    H, KVH, hd, P, T = 8, 2, 64, 16, 900
    g = gen(pairs)
    x = normal((T, (H + 2 * KVH) * hd), g, qt)
    table = torch.rand((1000, max(pairs, 1), 2), generator=g, device=DEV)
    rot = paged.Rotary(table) if pairs else None
    nrm = None if norm == "none" else paged.HeadNorm(norm, normal((1, hd), g), normal((1, hd), g), 1e-5)
    pos, slots = torch.arange(T, dtype=torch.int32, device=DEV), torch.randperm(T, generator=g, device=DEV)
    ks = [torch.zeros((2, T // P + 1, KVH, P, hd), dtype=kt, device=DEV) for _ in range(2)]
    want = paged.Cache(*ks[0]).append(x, H, pos, slots, rotary=rot, norm=nrm)
    y = x.clone()
    got = paged.Cache(*ks[1]).append(y, H, pos, slots, rotary=rot, norm=nrm, out=y[:, :H * hd].view(T, H, hd))
    assert got.data_ptr() == y.data_ptr() and torch.equal(got, want) and torch.equal(ks[0], ks[1])
    assert torch.equal(y[:, H * hd:], x[:, H * hd:])


def test_outputs_that_overlap_their_inputs():
    """Views of one buffer: apart they are taken, on top of each other refused."""
    H, KVH, hd, T = 4, 2, 64, 6
    g = gen(1)
    k, v = (normal((3, KVH, 8, hd), g) for _ in range(2))
    c = paged.Cache(k, v)
    args = (i32([[0, 1, 2]]), i32([0, T]), i32([20]), T)
    means = normal((3, KVH, hd), g)

    def attend(q, out):
        want = c.attend(q.clone(), *args)
        assert torch.equal(c.attend(q, *args, out=out), want)
        c.attend_sparse(q, means, *args, top=1, out=out)

    buf = normal((T, 2, H, hd), g)
    attend(buf[:, 0], buf[:, 1])                                  # queries and outputs side by side
    buf = normal((2, H, T, hd), g)
    attend(buf[0].transpose(0, 1), buf[1].transpose(0, 1))        # one behind the other
    buf = normal((T, H, 2, hd), g)
    attend(buf[:, :, 1], buf[:, :, 0])                            # head beside head
    long = normal((T + 2, H, hd), g)
    wide = normal((T, H + 1, hd), g)
    shifted = normal((T * H * hd + 256,), g)
    for q, out in ((long[:T], long[1:T + 1]), (long[2:], long[:T]), (wide[:, :H], wide[:, 1:]), (wide[:, 1:], wide[:, :H]),
                   (shifted[:T * H * hd].view(T, H, hd), shifted[32:32 + T * H * hd].view(T, H, hd))):
        for call in (lambda: c.attend(q, *args, out=out), lambda: c.attend_sparse(q, means, *args, top=1, out=out)):
            with pytest.raises(BackendError, match="out overlaps q"):
                call()
    width = (H + 2 * KVH) * hd
    rows = normal((T, width + H * hd), g)
    pos, slots = torch.arange(T, dtype=torch.int32, device=DEV), torch.arange(T, device=DEV)
    c.append(rows[:, :width], H, pos, slots, out=rows[:, width:].view(T, H, hd))
    for at in (64, width - 64, KVH * hd):
        with pytest.raises(BackendError, match="q_out overlaps qkv"):
            c.append(rows[:, :width], H, pos, slots, out=rows[:, at:at + H * hd].view(T, H, hd))
