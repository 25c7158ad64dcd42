"""Refusals of the paged-cache operators that protect outputs: rows that share
memory, which several CTAs would write at once. No GPU: arguments are checked
before any device is looked at, and the pointers are never read."""
import pytest

from test_paged_abi import append, attend, kv, queries, refused, sparse
from tinyoai_b200 import _lib


@pytest.mark.parametrize("over", [
    dict(rows=2, out_token_stride=0),                              # an expanded output
    dict(rows=2, out_token_stride=32),
    dict(heads=4, out_head_stride=0),
    dict(rows=2, heads=4, out_token_stride=64, out_head_stride=64),   # (0, 1) is (1, 0)
    dict(rows=9, heads=4, out_token_stride=128, out_head_stride=192),  # (3, 0) is (0, 2)
    dict(rows=9, heads=4, out_token_stride=128, out_head_stride=320),  # half of a row in another
])
def test_outputs_that_overlap(over):
    refused(attend(kv(), queries(requests=2, **over)), _lib.TCU_EINVAL, "output rows overlap")
    refused(sparse(kv(), queries(requests=2, **over)), _lib.TCU_EINVAL, "output rows overlap")


@pytest.mark.parametrize("over", [
    dict(rows=1, out_token_stride=0),                              # a dimension of one
    dict(rows=3, heads=4, out_token_stride=64, out_head_stride=192),   # heads first
    dict(rows=2, heads=4, out_token_stride=512, out_head_stride=128),  # gaps
    dict(rows=2, heads=4, out_token_stride=192, out_head_stride=128),  # rows between each other, none in another
    dict(rows=9, heads=4, q_token_stride=0, q_head_stride=0),          # queries may be one row for all
])
def test_outputs_that_do_not(over):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the fake addresses would be looked up")
    for rc in (attend(kv(), queries(requests=2, **over)), sparse(kv(), queries(requests=2, **over))):
        assert rc in (_lib.TCU_ENODEV, _lib.TCU_ECUDA), _lib.lib().tcu_last_error()


@pytest.mark.parametrize("over", [
    dict(head_stride=0),                           # one head that stands for several: to be read, not written
    dict(page_stride=0),
    dict(token_stride=32),
    dict(page_stride=16 * 64),                     # a page's second head is the next page's first
    dict(head_stride=8 * 64, page_stride=4 * 16 * 64),  # a head's last positions are the next one's first
])
def test_caches_that_overlap(over):
    refused(append(c=kv(**over)), _lib.TCU_EINVAL, "rows overlap")
    import torch
    if not torch.cuda.is_available():  # attention only reads them
        assert attend(kv(**over), queries()) in (_lib.TCU_ENODEV, _lib.TCU_ECUDA)


@pytest.mark.parametrize("over", [dict(head_stride=64, token_stride=128), dict(num_pages=1, page_stride=0), dict(kv_heads=1, head_stride=0),
                                  dict(page_stride=4 * 16 * 64, head_stride=16 * 64), dict(page_tokens=1, token_stride=0, head_stride=64, page_stride=128)])
def test_caches_that_do_not(over):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the fake addresses would be looked up")
    assert append(c=kv(**over)) in (_lib.TCU_ENODEV, _lib.TCU_ECUDA), _lib.lib().tcu_last_error()
