"""The error bound of float32 attention rows (paged_rows.py) is below what a
kernel would show that kept queries or weights to too few bits: 11, one
binary16 piece where two are kept, and 13 over float32 caches."""
import pytest
import torch

import paged_rows as R


@pytest.mark.parametrize("kt, bits", [(torch.float16, 11), (torch.float32, 13)])
@pytest.mark.parametrize("case", R.SHORT)
def test_a_lost_piece_shows(case, kt, bits):
    q, ks, vs = R.inputs(case, kt, seed=1)
    o, wv, size = R.attend(case, q, ks, vs)
    tol = R.bound(case, kt, o, wv, size)
    for cut in (dict(query_bits=bits), dict(weight_bits=bits)):
        worst = ((R.attend(case, q, ks, vs, **cut)[0] - o).abs() / tol).max()
        assert worst > 1.5, (cut, float(worst))


@pytest.mark.parametrize("kt", [torch.float16, torch.float32])
@pytest.mark.parametrize("case", range(2))
def test_a_lossy_join_shows(case, kt):
    """One part in ten thousand of the sums."""
    case = R.LONG[case]
    q, ks, vs = R.inputs(case, kt, seed=1)
    o, wv, size = R.attend(case, q, ks, vs)
    assert bool((1e-4 * wv > R.bound(case, kt, o, wv, size)).any())
