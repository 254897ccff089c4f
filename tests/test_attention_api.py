"""The attention entry points' checks (they come before any GPU call, so they run without one): every bad argument is
refused with a text, calls with nothing to do succeed."""
import ctypes

import pytest

from lazyweights_amd.attention import BF16, F16, F32, _Batch, _Cache

P = 1 << 20  # an address that is never read: aligned, not null


def cache(**kw):
    c = dict(k=P, v=P, pages=10, page_stride=2 * 16 * 128, head_stride=16 * 128, row_stride=128, page_size=16, kv_heads=2,
             head_dim=128, type=F16)
    c.update(kw)
    return _Cache(*[c[f] for f, _ in _Cache._fields_])


def batch(**kw):
    b = dict(seqs=2, tokens=2, max_new=1, max_kv=50, q_start=P, kv_len=P, page_table=P, table_stride=8, table_pages=4,
             reserved=0, workspace=P, workspace_bytes=1 << 40)
    b.update(kw)
    return _Batch(*[b[f] for f, _ in _Batch._fields_])


def ref(x):
    return None if x is None else ctypes.addressof(x)


def attend(lib, which, c, b, heads=8, q=P, ldq=1024, out=P, out_type=F16, ldo=1024, scale=0.1, window=0):
    return getattr(lib, "lw_attn_" + which)(ref(c), ref(b), heads, q, ldq, out, out_type, ldo, scale, window, None)


def append(lib, c, b, heads=8, q=P, k=P, v=P, x_type=F32, ldq=1024, ldk=256, ldv=256, cos=P, sin=P, rot=128, rows=50,
           neighbours=0, q_out=P, ldo=1024):
    return lib.lw_kv_append(ref(c), ref(b), heads, q, k, v, x_type, ldq, ldk, ldv, cos, sin, rot, rows, neighbours, q_out,
                            ldo, None)


def workspace(lib, c, b, heads=8):
    return lib.lw_attn_workspace(ref(c), ref(b), heads)


SHARED = [
    (dict(type=F32), {}), (dict(type=7), {}), (dict(head_dim=80), {}), (dict(head_dim=256), {}), (dict(page_size=0), {}),
    (dict(page_size=24), {}), (dict(page_size=1 << 17), {}), (dict(kv_heads=0), {}), (dict(kv_heads=3), {}),
    (dict(k=None), {}), (dict(v=P + 8), {}), (dict(row_stride=132), {}), (dict(head_stride=-128), {}), (dict(pages=-1), {}),
    ({}, dict(seqs=-1)), ({}, dict(seqs=1 << 17)), ({}, dict(tokens=-1)), ({}, dict(max_kv=-1)), ({}, dict(max_kv=65)),
    ({}, dict(q_start=None)), ({}, dict(kv_len=None)), ({}, dict(page_table=None)), ({}, dict(table_stride=3)),
    ({}, dict(reserved=1)), ({}, dict(tokens=1 << 28)), ({}, dict(table_pages=1 << 27, table_stride=1 << 27)),
]


@pytest.mark.parametrize("bad", SHARED, ids=str)
def test_cache_and_batch_are_checked(lib, bad):
    from lazyweights_amd import last_error
    c, b = cache(**bad[0]), batch(**bad[1])
    for call in (lambda: attend(lib, "decode", c, b), lambda: attend(lib, "prompt", c, b), lambda: append(lib, c, b),
                 lambda: workspace(lib, c, b)):
        assert call() == -1
        assert last_error()


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=7), dict(q=None), dict(out=None), dict(q=P + 2), dict(out=P + 8),
                                 dict(ldq=1023), dict(ldq=1016), dict(ldo=512), dict(out_type=3), dict(scale=float("inf")),
                                 dict(scale=float("nan")), dict(window=-1)], ids=str)
def test_attention_arguments_are_checked(lib, bad):
    from lazyweights_amd import last_error
    for which in ("decode", "prompt"):
        assert attend(lib, which, cache(), batch(), **bad) == -1
        assert last_error().startswith("lw_attn_" + which)


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(q_out=None), dict(x_type=3), dict(ldk=255), dict(ldk=128),
                                 dict(ldq=512), dict(k=P + 4), dict(cos=None), dict(sin=P + 4), dict(rot=130), dict(rot=12),
                                 dict(rot=-8), dict(rows=49), dict(neighbours=2)], ids=str)
def test_append_arguments_are_checked(lib, bad):
    from lazyweights_amd import last_error
    assert append(lib, cache(), batch(), **bad) == -1
    assert last_error().startswith("lw_kv_append")


def test_null_structures(lib):
    for c, b in ((None, batch()), (cache(), None)):
        assert attend(lib, "decode", c, b) == -1 and attend(lib, "prompt", c, b) == -1 and append(lib, c, b) == -1


def test_decode_limits_and_workspace(lib):
    from lazyweights_amd import last_error
    assert attend(lib, "decode", cache(), batch(max_new=17)) == -1 and "lw_attn_prompt" in last_error()
    need = workspace(lib, cache(), batch())
    assert need > 0
    for ws in (dict(workspace_bytes=need - 1), dict(workspace=None), dict(workspace=P + 8)):
        assert attend(lib, "decode", cache(), batch(**ws)) == -1 and "workspace" in last_error()


def test_nothing_to_do(lib):
    for b in (batch(seqs=0), batch(tokens=0)):
        assert attend(lib, "decode", cache(), b) == 0 and attend(lib, "prompt", cache(), b) == 0
        assert append(lib, cache(type=BF16), b) == 0
    assert attend(lib, "decode", cache(), batch(max_new=0)) == 0
    assert workspace(lib, cache(), batch(seqs=0)) == 0
