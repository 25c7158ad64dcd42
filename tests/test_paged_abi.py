"""Refusals of the paged-cache operators. Arguments are checked before any
device is looked at, so these run without a GPU; the pointers are never read."""
import ctypes as C

import pytest

from tinyoai_b200 import _lib

FAKE = 1 << 20  # stands for a device address


def kv(**over):
    d = dict(k=FAKE, v=FAKE, dtype=_lib.F16, num_pages=4, page_tokens=16, kv_heads=2, head_dim=64, page_stride=2 * 16 * 64, head_stride=16 * 64,
             token_stride=64)
    return _lib.PagedKV(**{**d, **over})


def queries(**over):
    d = dict(dtype=_lib.F16, requests=1, rows=1, heads=4, max_fresh=1, table_width=2, q=FAKE, q_token_stride=256, q_head_stride=64, out=FAKE,
             out_token_stride=256, out_head_stride=64, starts=FAKE, lengths=FAKE, tables=FAKE, table_stride=2, scale=0.125)
    return _lib.PagedQueries(**{**d, **over})


def refused(rc, want, text):
    assert rc == want, (rc, _lib.lib().tcu_last_error())
    assert text in _lib.lib().tcu_last_error().decode()


def attend(c, q, pages=0, prefix=FAKE, most=0):
    return _lib.lib().tcu_paged_attend(0, None, C.byref(c), C.byref(q), prefix, pages, most, FAKE, 1 << 40)


def sparse(c, q, first=1, last=1, top=4):
    return _lib.lib().tcu_paged_attend_sparse(0, None, C.byref(c), C.byref(q), FAKE, first, last, top, FAKE, FAKE, 1 << 40)


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=_lib.Q8_0), _lib.TCU_EUNSUP, "float32, binary16 and bfloat16"),
    (dict(num_pages=0), _lib.TCU_EINVAL, "no pages"),
    (dict(page_tokens=0), _lib.TCU_EINVAL, "no pages"),
    (dict(page_tokens=65537), _lib.TCU_EINVAL, "positions a page"),
    (dict(head_dim=60), _lib.TCU_EUNSUP, "multiple of 8"),
    (dict(head_dim=264), _lib.TCU_EUNSUP, "multiple of 8"),
    (dict(token_stride=68), _lib.TCU_EINVAL, "multiples of 16 bytes"),
    (dict(page_stride=-2048), _lib.TCU_EINVAL, "negative cache stride"),
])
def test_caches(over, code, text):
    refused(attend(kv(**over), queries()), code, text)
    refused(sparse(kv(**over), queries()), code, text)
    L = _lib.lib()
    refused(L.tcu_paged_means(0, None, C.byref(kv(**over)), 1, FAKE, FAKE), code, text)
    refused(L.tcu_paged_append(0, None, C.byref(kv(**over)), _lib.F16, 1, 4, FAKE, 512, FAKE, FAKE, None, None, FAKE, 256), code, text)


@pytest.mark.parametrize("over, code, text", [
    (dict(dtype=_lib.BF16), _lib.TCU_EUNSUP, "cache's type"),
    (dict(heads=3), _lib.TCU_EINVAL, "3 query heads over 2"),
    (dict(heads=130), _lib.TCU_EUNSUP, "query heads a KV head"),
    (dict(heads=0), _lib.TCU_EINVAL, "0 query heads"),
    (dict(max_fresh=0), _lib.TCU_EINVAL, "max_fresh"),
    (dict(requests=-1), _lib.TCU_EINVAL, "negative count"),
    (dict(rows=-1), _lib.TCU_EINVAL, "negative count"),
    (dict(table_stride=1), _lib.TCU_EINVAL, "table stride"),
    (dict(table_width=1 << 27, table_stride=1 << 27), _lib.TCU_EINVAL, "pass 2^30"),
    (dict(requests=1 << 20, max_fresh=1 << 12), _lib.TCU_EINVAL, "too many rows"),
    (dict(q_token_stride=260), _lib.TCU_EINVAL, "multiples of 16 bytes"),
    (dict(out_head_stride=-64), _lib.TCU_EINVAL, "negative query stride"),
    (dict(scale=float("nan")), _lib.TCU_EINVAL, "scale"),
])
def test_queries(over, code, text):
    refused(attend(kv(), queries(**over)), code, text)
    refused(sparse(kv(), queries(**over)), code, text)


def test_other_arguments():
    L = _lib.lib()
    refused(attend(kv(), queries(), pages=-1), _lib.TCU_EINVAL, "prefix of -1")
    refused(attend(kv(), queries(), pages=1, prefix=None), _lib.TCU_EINVAL, "prefix is null")
    refused(attend(kv(), queries(), most=-1), _lib.TCU_EINVAL, "max_length")
    refused(sparse(kv(), queries(), last=0), _lib.TCU_EINVAL, "at least 1")
    refused(sparse(kv(), queries(), first=-1), _lib.TCU_EINVAL, "must not be negative")
    refused(sparse(kv(), queries(), top=65536), _lib.TCU_EINVAL, "pages a query")
    refused(sparse(kv(page_tokens=65536, token_stride=64, head_stride=1 << 22, page_stride=1 << 23), queries(), top=30000), _lib.TCU_EINVAL, "pass 2^30")
    refused(attend(kv(), queries(), pages=1 << 27), _lib.TCU_EINVAL, "prefix of")
    refused(L.tcu_paged_attend_workspace(None, None, 0, 0, C.byref(C.c_uint64())), _lib.TCU_EINVAL, "null cache")
    refused(L.tcu_paged_attend_workspace(C.byref(kv()), None, 0, 0, C.byref(C.c_uint64())), _lib.TCU_EINVAL, "null queries")
    refused(L.tcu_paged_attend_workspace(C.byref(kv()), C.byref(queries()), 0, 0, None), _lib.TCU_EINVAL, "null argument")


def append(c=None, dtype=_lib.F16, rows=1, heads=4, qkv=FAKE, stride=512, rotary=None, norm=None, q_stride=256):
    c = c or kv()
    return _lib.lib().tcu_paged_append(0, None, C.byref(c), dtype, rows, heads, qkv, stride, FAKE, FAKE, rotary and C.byref(rotary), norm and C.byref(norm),
                                       FAKE, q_stride)


def test_append():
    refused(append(dtype=_lib.F32, c=kv(dtype=_lib.BF16)), _lib.TCU_EUNSUP, "cache's type")
    refused(append(rows=-1), _lib.TCU_EINVAL, "-1 rows")
    refused(append(stride=504), _lib.TCU_EINVAL, "below its width")
    refused(append(stride=516), _lib.TCU_EINVAL, "16 bytes")
    refused(append(q_stride=248), _lib.TCU_EINVAL, "below its width")
    refused(append(qkv=None), _lib.TCU_EINVAL, "null argument")
    refused(append(rotary=_lib.Rotary(FAKE, 16, 33, 0)), _lib.TCU_EINVAL, "33 rotary pairs")
    refused(append(rotary=_lib.Rotary(FAKE, 0, 8, 0)), _lib.TCU_EINVAL, "empty rotary table")
    refused(append(rotary=_lib.Rotary(FAKE, 16, -1, 0)), _lib.TCU_EINVAL, "-1 rotary pairs")
    refused(append(norm=_lib.HeadNorm(7, 1e-5, FAKE, FAKE, 0)), _lib.TCU_EINVAL, "unknown norm")
    refused(append(norm=_lib.HeadNorm(1, -1.0, FAKE, FAKE, 0)), _lib.TCU_EINVAL, "epsilon")
    refused(append(norm=_lib.HeadNorm(1, 1e-5, FAKE, FAKE, 32)), _lib.TCU_EINVAL, "shared (stride 0)")


def plan(n=1, page=16, width=4, stride=4, n_free=1, capacity=8, held=FAKE):
    return _lib.lib().tcu_plan_step(0, None, n, held, FAKE, page, FAKE, width, stride, FAKE, n_free, capacity, FAKE, FAKE, FAKE, FAKE, FAKE)


def test_plan():
    refused(plan(n=-1), _lib.TCU_EINVAL, "negative count")
    refused(plan(capacity=-1), _lib.TCU_EINVAL, "negative count")
    refused(plan(page=0), _lib.TCU_EINVAL, "positions a page")
    refused(plan(stride=3), _lib.TCU_EINVAL, "table stride")
    refused(plan(held=None), _lib.TCU_EINVAL, "null argument")


def test_workspace_sizes_need_no_gpu():
    n = C.c_uint64()
    assert _lib.lib().tcu_paged_attend_workspace(C.byref(kv()), C.byref(queries()), 0, 0, C.byref(n)) == _lib.TCU_OK
    small = n.value
    assert small == 0  # one part: the output is written at once
    # Parts of one row that no cluster joins.
    long = dict(table_width=4096, table_stride=4096)
    assert _lib.lib().tcu_paged_attend_workspace(C.byref(kv()), C.byref(queries(**long)), 0, 0, C.byref(n)) == _lib.TCU_OK
    assert n.value > small
    assert _lib.lib().tcu_paged_attend_sparse_workspace(C.byref(kv()), C.byref(queries()), 1, 1, 4, C.byref(n)) == _lib.TCU_OK


def test_share_prefix_needs_a_batch():
    refused(_lib.lib().tcu_batch_share_prefix(None, 64), _lib.TCU_EINVAL, "null argument")


def test_valid_calls_reach_the_device_check():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible: the fake addresses would be looked up")
    for rc in (plan(), append(), attend(kv(), queries()), sparse(kv(), queries())):
        assert rc in (_lib.TCU_ENODEV, _lib.TCU_ECUDA)
