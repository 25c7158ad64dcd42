"""Float32 rows over float32 and binary16 caches: inputs, float64 attention and
a bound on the kernels' error, shared by the test of the kernels and by the
test that the bound would show a lost piece.

The bound, in units of 2^-24 (half a step of float32). n positions, c tiles of
them in a lane's longest chain, size = scale * sum |q k| of a row's largest.
 - A score, relative to size: the queries' and the scale's roundings 3; float32
   caches: hd / 8 multiply-adds and 3 additions; binary16 caches: an instruction
   sums 16 products with truncated additions, 2 units each and 17 of them, then
   hd / 8 additions, 4 for what the second piece of a query leaves out and 2 for
   the powers of two around it.
 - A weight's relative error: the score's; two subtractions of numbers up to 2
   size and the bias (14 ln 2 = 10) 4 size + 10; the exponential 2^-22 = 4; each of
   the factors that move it to another reference (c of them, and 3 joins of
   groups, warps and parts) 2 size + 4; a pair of binary16 values 4.
 - A sum, relative to the sum of its terms' sizes: float32 caches: three
   operations a tile of a chain; binary16: two instructions as above, 68, and one
   addition a tile; joins of 16 groups or 4 warps and 8 parts, 26.
Numerator and denominator have both, and the result its own rounding.
"""
import math

import torch

# requests' positions, heads, KV heads, head size, page, shared pages
SHORT = [
    ([2 + i % 3 for i in range(48)], 8, 8, 8, 16, 0),
    ([2 + i % 8 for i in range(64)], 8, 2, 64, 4, 0),
    ([3, 5, 2, 9] * 8, 16, 4, 40, 32, 0),
    ([2 + i % 5 for i in range(32)], 4, 4, 128, 8, 0),
]
LONG = [
    ([40 + 5 * i for i in range(12)], 8, 2, 64, 16, 0),
    ([333, 200], 4, 2, 80, 24, 0),                       # parts that a cluster joins
    ([2048 + 3 + i % 30 for i in range(64)], 8, 4, 64, 32, 64),  # a shared prefix with a kernel of its own
    ([6000, 9000], 4, 2, 64, 32, 0),                     # more parts than a cluster joins
]


def inputs(case, kt, seed):
    """Queries [rows, heads, hd], and keys and values [rows][n, KV heads, hd] on the CPU; shared positions are the same tensors."""
    lens, H, KVH, hd, P, prefix = case
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((len(lens), H, hd), generator=g)
    head = [torch.randn((prefix * P, KVH, hd), generator=g).to(kt) for _ in range(2)]
    own = [[torch.cat([x, torch.randn((n - prefix * P, KVH, hd), generator=g).to(kt)]) for x in head] for n in lens]
    return q, [o[0] for o in own], [o[1] for o in own]


def kept(x, bits):
    """x with `bits` bits of mantissa."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(torch.ldexp(m, torch.tensor(bits))), e - bits)


def attend(case, q, ks, vs, query_bits=None, weight_bits=None):
    """Float64 outputs [rows, heads, hd], sums of w |v|, and size [rows, heads]; with queries or weights cut to so many bits."""
    lens, H, KVH, hd, P, prefix = case
    outs, wvs, sizes = [], [], []
    q = q.double()
    if query_bits:
        q = kept(q, query_bits)
    scale = 1 / math.sqrt(hd)
    for i in range(len(lens)):
        k, v = (x[i].double().repeat_interleave(H // KVH, 1) for x in (ks, vs))
        s = torch.einsum("hd,thd->ht", q[i], k) * scale
        sizes.append((torch.einsum("hd,thd->ht", q[i].abs(), k.abs()) * scale).amax(-1))
        p = torch.exp(s - s.amax(-1, keepdim=True))
        l = p.sum(-1, keepdim=True)
        if weight_bits:
            p = kept(p, weight_bits)
        outs.append(torch.einsum("ht,thd->hd", p / l, v))
        wvs.append(torch.einsum("ht,thd->hd", p / l, v.abs()))
    return torch.stack(outs), torch.stack(wvs), torch.stack(sizes)


def bound(case, kt, o, wv, size):
    lens, H, KVH, hd, P, prefix = case
    half = kt == torch.float16
    # Positions of a part: no part of these cases is longer; 32 or 64 of them a step of a chain.
    part = max(lens) if max(lens) <= 512 else 2048
    c = -(-part // (64 if half else 32))
    score = 3 + (34 + hd / 8 + 6 if half else hd / 8 + 3)
    weight = (score + 4 + 2 * (c + 3)) * size[..., None] + 10 + 4 + 4 * (c + 3) + (4 if half else 0)
    total = 68 + c + 26 if half else 3 * c + 26
    return 2.0 ** -24 * (2 * (weight + total) * wv + o.abs())
