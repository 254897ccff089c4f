"""The checks of the 8-bit cache's and the page tables' entry points (they come before any GPU call, so they run without one): every
bad argument is refused with a text, calls with nothing to do succeed."""
import ctypes

import pytest
from test_attention_api import P, batch, ref

from lazyweights_amd.attention import BF16, F16, F32, _Cache8
from lazyweights_amd.pages import _Pages


def cache(**kw):
    c = dict(k=P, v=P, k_exp=P + 1, v_exp=P + 3, pages=10, page_stride=2 * 16 * 128, head_stride=16 * 128, row_stride=128,
             exp_page_stride=2, exp_head_stride=1, page_size=16, kv_heads=2, head_dim=128, reserved=0)
    c.update(kw)
    return _Cache8(*[c[f] for f, _ in _Cache8._fields_])


def attend(lib, which, c, b, heads=8, q=P, q_type=F16, ldq=1024, out=P, out_type=F16, ldo=1024, scale=0.1, window=0):
    return getattr(lib, "lw_attn8_" + which)(ref(c), ref(b), heads, q, q_type, ldq, out, out_type, ldo, scale, window, None)


def append(lib, c, b, heads=8, q=P, k=P, v=P, x_type=F32, ldq=1024, ldk=256, ldv=256, cos=P, sin=P, rot=128, rows=50,
           neighbours=0, q_out=P, q_type=F16, ldo=1024):
    return lib.lw_kv8_append(ref(c), ref(b), heads, q, k, v, x_type, ldq, ldk, ldv, cos, sin, rot, rows, neighbours, q_out,
                             q_type, ldo, None)


SHARED = [
    (dict(head_dim=80), {}), (dict(head_dim=256), {}), (dict(page_size=8), {}), (dict(page_size=1), {}), (dict(page_size=48), {}),
    (dict(page_size=1 << 17), {}), (dict(kv_heads=0), {}), (dict(kv_heads=3), {}), (dict(k=None), {}), (dict(v=P + 8), {}),
    (dict(k_exp=None), {}), (dict(v_exp=None), {}), (dict(row_stride=136), {}), (dict(head_stride=-128), {}),
    (dict(page_stride=4104), {}), (dict(exp_page_stride=-1), {}), (dict(exp_head_stride=-1), {}), (dict(pages=-1), {}),
    (dict(reserved=1), {}), ({}, dict(seqs=-1)), ({}, dict(seqs=1 << 17)), ({}, dict(tokens=-1)), ({}, dict(max_kv=65)),
    ({}, dict(q_start=None)), ({}, dict(page_table=None)), ({}, dict(table_stride=3)), ({}, dict(reserved=1)),
]


@pytest.mark.parametrize("bad", SHARED, ids=str)
def test_cache_and_batch_are_checked(lib, bad):
    from lazyweights_amd import last_error
    c, b = cache(**bad[0]), batch(**bad[1])
    for call in (lambda: attend(lib, "decode", c, b), lambda: attend(lib, "prompt", c, b), lambda: append(lib, c, b),
                 lambda: lib.lw_attn8_workspace(ref(c), ref(b), 8)):
        assert call() == -1
        assert last_error()


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=7), dict(q=None), dict(out=None), dict(q=P + 2), dict(out=P + 8),
                                 dict(ldq=1023), dict(ldq=1016), dict(ldo=512), dict(out_type=3), dict(q_type=F32), dict(q_type=3),
                                 dict(scale=float("inf")), dict(scale=float("nan")), dict(window=-1)], ids=str)
def test_attention_arguments_are_checked(lib, bad):
    from lazyweights_amd import last_error
    for which in ("decode", "prompt"):
        assert attend(lib, which, cache(), batch(), **bad) == -1
        assert last_error().startswith("lw_attn8_" + which)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(q_out=None), dict(x_type=3), dict(q_type=F32), dict(ldk=255),
                                 dict(ldk=128), dict(ldq=512), dict(k=P + 4), dict(cos=None), dict(sin=P + 4), dict(rot=130),
                                 dict(rot=12), dict(rot=-8), dict(rows=49), dict(neighbours=2)], ids=str)
def test_append_arguments_are_checked(lib, bad):
    from lazyweights_amd import last_error
    assert append(lib, cache(), batch(), **bad) == -1
    assert last_error().startswith("lw_kv8_append")


def test_decode_limits_and_workspace(lib):
    from lazyweights_amd import last_error
    assert attend(lib, "decode", cache(), batch(max_new=17)) == -1 and "lw_attn8_prompt" in last_error()
    assert lib.lw_attn8_workspace(ref(cache()), ref(batch()), 8) > 0
    for c, b in ((None, batch()), (cache(), None)):
        assert attend(lib, "decode", c, b) == -1 and attend(lib, "prompt", c, b) == -1 and append(lib, c, b) == -1


def test_more_items_than_a_launch_takes(lib):
    from lazyweights_amd import last_error
    c = cache(kv_heads=1024, head_stride=0)
    b = batch(seqs=65535, tokens=1024, max_kv=16, workspace_bytes=1 << 50)
    assert attend(lib, "decode", c, b, heads=1024, ldq=1024 * 128, ldo=1024 * 128) == -1 and "more sequences" in last_error()


def test_nothing_to_do(lib):
    for b in (batch(seqs=0), batch(tokens=0)):
        assert attend(lib, "decode", cache(), b) == 0 and attend(lib, "prompt", cache(), b, q_type=BF16) == 0
        assert append(lib, cache(), b) == 0
    assert attend(lib, "decode", cache(), batch(max_new=0)) == 0
    assert lib.lw_attn8_workspace(ref(cache()), ref(batch(seqs=0)), 8) == 0


@pytest.mark.parametrize("bad", [dict(seqs=-1), dict(seqs=8193), dict(page_size=0), dict(page_size=24), dict(page_size=1 << 17),
                                 dict(pages=-1), dict(pages=1 << 30), dict(rows=-1), dict(rows=1 << 30), dict(table_pages=-1),
                                 dict(table_stride=3), dict(table_pages=1 << 26, table_stride=1 << 26), dict(table=None),
                                 dict(free=None), dict(kv_len=None), dict(left=None), dict(workspace=None), dict(new=None),
                                 dict(kv_len_out=None), dict(left_out=None), dict(q_start=None), dict(whole=None)], ids=str)
def test_page_arguments_are_checked(lib, bad):
    from lazyweights_amd import last_error
    p = dict(table=P, table_stride=4, table_pages=4, seqs=2, page_size=16, pages=10, free=P, kv_len=P, left=P, workspace=P)
    a = dict(new=P, keep=None, rows=5, kv_len_out=P, left_out=P, q_start=P, position=None, slot=None, stream=None)
    for d in (p, a):
        d.update({k: x for k, x in bad.items() if k in d})
    pages = _Pages(*[p[f] for f, _ in _Pages._fields_])
    assert lib.lw_pages_advance(None if "whole" in bad else ctypes.addressof(pages), *a.values()) == -1
    assert last_error().startswith("lw_pages_advance")
