"""Numbers that the operators over a paged KV cache have to keep: weights far
below a row's largest one, scores at the end of float32, the rotation's roundings.

Tolerances. u = eps / 2 of a type, as in test_gpu_paged.py.
 - Heavy positions before a light tail: every score is a product of one
   feature, so scores are exact and a weight errs by the exponential (2^-22,
   twice where states are joined) and by its own rounding: u where it is stored
   in 16 bits, 2^-22 where it is a pair of binary16 values, nothing in float32.
   Binary16 values stop shrinking at a step of 2^-24: weights are kept times
   2^11 (binary16 rows) or 2^14 (float32 rows) of the row's largest, which
   leaves each an absolute error of 2^-36 or 2^-39 of it (2^4 more on the
   tensor cores of a shared prefix, whose reference may lag that far). The
   sums' chains add up to n / 32 terms a lane of equal sign: n * 2^-29 of the
   result at most; an instruction's sixteen truncated additions, the joins and
   the exponentials 2^-18.
 - Scores so large that float32 has no halves, or no ones, there: equal keys
   have equal weights, and a larger score takes all. The sums, weights and the
   store as in test_gpu_paged.py, 2^-13 + u and u.
 - Append without a norm: the stored numbers themselves, products and sum of the
   rotation each rounded to float32, then to the stored type.
"""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

import paged_rows as R  # noqa: E402
from test_gpu_paged import DEV, PAIRS, TYPES, attention_state, choose_ref, gen, i32, near, normal, unit  # noqa: E402

if torch.cuda.is_available():
    from tinyoai_b200 import paged


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("rows, heads, n, shared", [(1, 1, 32768, False), (64, 8, 2048, False), (48, 8, 8192, True), (200, 16, 4096, True)])
@pytest.mark.parametrize("below", [13.0, 20.0, 24.0, 25.125, 26.5, 30.0])
def test_light_tail_behind_heavy_positions(qt, kt, rows, heads, n, shared, below):
    """Runs of 256 positions with value 0 before tails of 1,792 whose weights
    are 2^-below of theirs and whose values are 1,024: the output is the tail's
    share. Histories of the requests' own, and one that they share."""
    qt, kt = TYPES[qt], TYPES[kt]
    hd, P = 64, 32
    pages = n // P
    ids = torch.randperm(pages, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).to(torch.int32)
    k, v = (torch.zeros((pages, heads, P, hd), dtype=kt, device=DEV) for _ in range(2))
    t = torch.arange(n, device=DEV)
    heavy = t % 2048 < 256
    page = ids[t // P].long()
    k[page[heavy], :, t[heavy] % P, 0] = below  # exact in every type
    v[page[~heavy], :, t[~heavy] % P] = 1024.0
    q = torch.zeros((rows, heads, hd), dtype=qt, device=DEV)
    q[:, :, 0] = 1.0
    starts, lengths = torch.arange(rows + 1, dtype=torch.int32, device=DEV), torch.full((rows,), n, dtype=torch.int32, device=DEV)
    table = ids[None].expand(rows, -1).contiguous()
    out = paged.Cache(k, v).attend(q, table, starts, lengths, 1, prefix=ids if shared else None, scale=math.log(2.0))
    w, ht, lt = 2.0 ** -below, int(heavy.sum()), int((~heavy).sum())
    want = 1024 * lt * w / (ht + lt * w)
    if qt == torch.float32:
        weight, floor = (2.0 ** -22, 2.0 ** -39) if kt == torch.float16 else (0.0, 0.0)
    else:
        weight, floor = unit(kt), (2.0 ** -36 * (2 ** 4 if shared else 1) if kt == torch.float16 else 0.0)
    # The scale is ln 2 in float32, and so is its product with log2 e: 2^-24 of the exponent each.
    rel = 2 * below * 2.0 ** -24 + weight + n * 2.0 ** -29 + 2.0 ** -18 + unit(qt)
    tol = rel * want + 1024 * lt * floor / ht + (2.0 ** -25 if qt == torch.float16 else 0.0)
    near(out, torch.full_like(out, want, dtype=torch.float64), tol)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [4, 48, 200])
@pytest.mark.parametrize("power", [17, 22, 27, 30, 35, 100])
def test_scores_past_float32_steps(t, rows, power):
    """Scores of -0.7 * 1.75 * 2^power at every position, then one of the other sign
    among them: in a shared prefix, joined with the requests' own positions."""
    dt, P, prefix, hd = TYPES[t], 32, 20, 64
    if power > 35 and dt == torch.float16:
        power = 34  # binary16 rows have no such scores
    lens = [prefix * P + 1 + i % 40 for i in range(rows)]
    s = attention_state(lens, [1] * rows, 2, 2, hd, P, dt, dt, seed=8, prefix=prefix, fill=0.0)
    c = paged.Cache(s["k"], s["v"])
    a, b = 1.75 * 2.0 ** ((power - 6) // 2), 2.0 ** (power - 6 - (power - 6) // 2)  # 64 products of three bits: exact sums
    s["q"].fill_(a)

    def check(at):
        out = c.attend(s["q"], s["table"], s["starts"], s["lengths"], 1, prefix=s["prefix"], scale=0.7)
        for i in range(0, rows, 7):
            x = torch.arange(lens[i], device=DEV)
            page = torch.where(x // P < prefix, s["prefix"][(x // P).clamp(max=prefix - 1)], s["table"][i][x // P]).long()
            v = s["v"][page, :, x % P].double()
            v = v if at is None else v[at:at + 1]
            near(out[i], v.mean(0), (2.0 ** -13 + unit(dt)) * v.abs().mean(0) + unit(dt) * v.mean(0).abs())

    s["k"].fill_(-b)
    check(None)
    s["k"][s["prefix"][9].long(), :, 3] = b
    check(9 * P + 3)


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("pairs, adjacent", [(16, False), (32, False), (6, False), (20, True), (32, True)])
def test_rotation_rounds_each_operation(qt, kt, pairs, adjacent):
    """Queries and keys of an append equal, bit for bit, a rotation whose
    products and sums are rounded one by one."""
    qt, kt = TYPES[qt], TYPES[kt]
    H, KVH, hd, P, T = 4, 2, 64, 16, 96
    g = gen(pairs + adjacent)
    k, v = (torch.zeros((T // P, KVH, P, hd), dtype=kt, device=DEV) for _ in range(2))
    angle = torch.rand((512, pairs), generator=g, device=DEV, dtype=torch.float64) * 6.3
    table = torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()
    pos = torch.randint(0, 512, (T,), generator=g, device=DEV)
    slots = torch.randperm(T, generator=g, device=DEV)
    x = normal((T, (H + 2 * KVH) * hd), g, qt)
    q = paged.Cache(k, v).append(x, H, pos.to(torch.int32), slots, rotary=paged.Rotary(table, adjacent))
    y = x.float().reshape(T, -1, hd)[:, :H + KVH].clone()
    ia = torch.arange(pairs, device=DEV) * (2 if adjacent else 1)
    ib = ia + (1 if adjacent else pairs)
    a, b, c, s = y[..., ia].clone(), y[..., ib].clone(), table[pos][:, None, :, 0], table[pos][:, None, :, 1]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    assert torch.equal(q, y[:, :H].to(qt))
    assert torch.equal(k[slots // P, :, slots % P], y[:, H:].to(kt))
    assert torch.equal(v[slots // P, :, slots % P], x.reshape(T, -1, hd)[:, H + KVH:].to(kt))


@pytest.mark.parametrize("kv", ["f32", "f16"])
@pytest.mark.parametrize("heads, kv_heads, hidden", [(4, 4, 320), (8, 2, 512)])
def test_a_shared_step_stores_what_an_unshared_one_does(kv, heads, kv_heads, hidden, tmp_path):
    """First-layer keys and values do not depend on attention: with share_prefix
    on, the cache of a one-layer model holds the same bytes as without."""
    from tinyoai_b200 import Model
    from tinyoai_b200.synth import prompt_ids, synth_stablelm

    cfg, tensors = synth_stablelm(dict(model_type="stablelm", vocab_size=2048, hidden_size=hidden, intermediate_size=864, num_hidden_layers=1,
                                       num_attention_heads=heads, num_key_value_heads=kv_heads, max_position_embeddings=512, layer_norm_eps=1e-5,
                                       rope_theta=10000.0, partial_rotary_factor=0.25, use_parallel_residual=True, use_qkv_bias=False,
                                       qk_layernorm=False, tie_word_embeddings=False, hidden_act="silu", bos_token_id=0, eos_token_id=0), "Q8_0", seed=11)
    m = Model.load_stablelm(cfg, tensors)
    opened = []
    try:
        parent = m.session(kv)
        opened.append(parent)
        ids = list(prompt_ids(200, cfg["vocab_size"], seed=1))
        parent.forward(0, ids, want_logits=False)
        files = []
        for share in (128, 0):
            forks = [parent.fork() for _ in range(5)]
            batch = m.batch(5)
            opened.extend([*forks, batch])
            batch.share_prefix(share)
            added = [prompt_ids(5, cfg["vocab_size"], seed=30 + step) for step in range(4)]
            for toks in added:
                batch.forward(forks, toks)
            for i, f in enumerate(forks):
                f.save_cache(tmp_path / f"{share}-{i}", bytes(32), ids + [int(t[i]) for t in added])
            files.append([(tmp_path / f"{share}-{i}").read_bytes() for i in range(5)])
        assert files[0] == files[1]
    finally:
        for x in reversed(opened):
            x.close()
        m.close()


@pytest.mark.parametrize("kt", ["f32", "f16"])
@pytest.mark.parametrize("case", R.SHORT + R.LONG)
def test_float32_rows_keep_their_bits(kt, case):
    """Float32 rows within a bound that a lost piece of a query or a weight passes (test_paged_rows.py)."""
    kt = TYPES[kt]
    lens, H, KVH, hd, P, prefix = case
    q, ks, vs = R.inputs(case, kt, seed=2)
    width = max(-(-n // P) for n in lens)
    pages = prefix + sum(-(-n // P) - prefix for n in lens) + 2
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    k, v = (torch.full((pages, KVH, P, hd), math.nan, dtype=kt) for _ in range(2))
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = prefix
    for i, n in enumerate(lens):
        have = -(-n // P)
        table[i, :have] = torch.cat([ids[:prefix], ids[at:at + have - prefix]])
        at += have - prefix
        t = torch.arange(n)
        k[table[i][t // P].long(), :, t % P], v[table[i][t // P].long(), :, t % P] = ks[i], vs[i]
    starts = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV)
    out = paged.Cache(k.to(DEV), v.to(DEV)).attend(q.to(DEV), table.to(DEV), starts, i32(lens), 1, prefix=ids[:prefix].to(DEV) if prefix else None)
    o, wv, size = R.attend(case, q, ks, vs)
    near(out.cpu(), o, R.bound(case, kt, o, wv, size))


@pytest.mark.parametrize("qt, kt", PAIRS)
@pytest.mark.parametrize("kind", ["small beside large", "subnormal", "tiny"])
@pytest.mark.parametrize("hd", [64, 136])
def test_page_choice_where_float32_scores_fail(qt, kt, kind, hd):
    """The order of pages is float64's: values of a query far below its largest
    one, which meets means of zero, and products that float32 does not hold."""
    qt, kt = TYPES[qt], TYPES[kt]
    H, KVH, P, n = 8, 2, 4, 1200
    small, of_means = {"small beside large": (1e-12, 1.0), "subnormal": (3e-23, 1e-22), "tiny": (1e-24, 1e-24)}[kind]
    if kt == torch.float16 and kind != "small beside large":  # the least values of the types
        small, of_means = (1e-37 if kind == "subnormal" else 1e-43) if qt == torch.float32 else 6e-8, 1e-7
    s = attention_state([n], [1], H, KVH, hd, P, qt, kt, seed=hd, fill=0.0)
    g = gen(7)
    means = (normal((len(s["k"]), KVH, hd), g) * of_means).to(kt)
    q = normal((1, H, hd), g) * small
    if kind == "small beside large":
        if qt == torch.float16:
            q = q * (1e-7 / small)  # of the type's least values
        q[..., 0] = 1.0
        means[..., 0] = 0.0
    q = q.to(qt)
    _, pages = paged.Cache(s["k"], s["v"]).attend_sparse(q, means, s["table"], s["starts"], s["lengths"], 1, top=100, first=1, last=1)
    want = choose_ref(q.reshape(KVH, H // KVH, hd), means, s["table"][0], n - 1, P, 1, 1, 100, len(s["k"]))
    assert pages[0].tolist() == want
