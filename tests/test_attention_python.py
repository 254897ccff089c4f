"""What the Python classes check before a library call, and how they make it; caches over CPU tensors here, with a library that
only notes its calls, so that nothing of this needs a GPU."""
import ctypes

import pytest
import torch

from lazyweights_amd.attention import Batch, KvCache, _Cache


class Calls:
    """The library: lw_attn_workspace of the built one, the launches noted."""

    def __init__(self, lib):
        self.lw_attn_workspace, self.made = lib.lw_attn_workspace, []

    def note(self, *args):
        self.made.append(args)
        return 0

    lw_kv_append = lw_attn_decode = lw_attn_prompt = note


def cache(lib, kv_heads=8, head_dim=64, pages=4, page=16):
    c = object.__new__(KvCache)  # (its __init__ wants GPU tensors)
    c.lib, c.k, c.v = lib, *(torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.float16) for _ in range(2))
    c.kv_heads, c.head_dim, c.index = kv_heads, head_dim, c.k.get_device()
    c.types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    c._current, c._device = lambda index: 0, lambda: c.index
    c.c = _Cache(c.k.data_ptr(), c.v.data_ptr(), pages, c.k.stride(0), c.k.stride(1), c.k.stride(2), page, kv_heads, head_dim, 1)
    c.ptr = ctypes.addressof(c.c)
    return c


def batch(c, heads=32, seqs=64, max_new=1, max_kv=64):
    return Batch(c, heads, torch.arange(seqs + 1, dtype=torch.int32), torch.full((seqs,), 9, dtype=torch.int32),
                 torch.zeros((seqs, 4), dtype=torch.int32), max_new, max_kv)


def q_of(c, heads=32, rows=64):
    return torch.zeros((rows, heads, c.head_dim), dtype=torch.float16)


def test_a_batch_and_caches_of_other_heads(lib):
    """The counters of 64 sequences take 2048 bytes for 8 key-value heads and 512 for 2: the sums of a call with the smaller cache
    would lie on the larger one's counters, and its next call would leave rows unwritten."""
    calls = Calls(lib)
    big, small, other_dim = cache(calls), cache(calls, kv_heads=2), cache(calls, head_dim=128)
    b = batch(big, max_new=2)
    for attend in (small.attend_decode, small.attend_prompt):
        with pytest.raises(ValueError, match="key-value heads"):
            attend(b, q_of(small))
    assert not calls.made
    big.attend_decode(b, q_of(big))
    other_dim.attend_decode(b, q_of(other_dim))
    k = torch.zeros((64, 2, 64))
    small.append(b, None, k, k)  # (needs no workspace)
    small.attend_prompt(batch(big, max_new=17), q_of(small))  # (no counters)
    assert len(calls.made) == 4


def test_a_batch_of_another_device(lib):
    calls = Calls(lib)
    c = cache(calls)
    b = batch(c)
    b.index = c.index + 1
    k = torch.zeros((64, 8, 64))
    for call in (lambda: c.attend_decode(b, q_of(c)), lambda: c.attend_prompt(b, q_of(c)), lambda: c.append(b, None, k, k)):
        with pytest.raises(ValueError, match="device"):
            call()
    assert not calls.made


def test_calls_are_made_with_the_caches_device_current(lib, monkeypatch):
    """Default streams of all devices have the same handle: the launch goes to the current device, which must be the cache's."""
    device = [3]
    calls = Calls(lib)

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, device[0] = device[0], self.index

        def __exit__(self, *exc):
            device[0] = self.before

    monkeypatch.setattr(torch.cuda, "device", Device)
    seen = []
    calls.lw_kv_append = calls.lw_attn_decode = calls.lw_attn_prompt = lambda *args: seen.append(device[0]) or 0
    c = cache(calls)
    c._device = lambda: device[0]
    b = batch(c)
    k = torch.zeros((64, 8, 64))
    for device[0] in (3, c.index):
        outside = device[0]
        c.append(b, None, k, k)
        c.attend_decode(b, q_of(c))
        c.attend_prompt(b, q_of(c))
        assert device[0] == outside
    assert seen == 6 * [c.index]


@pytest.mark.parametrize("big", [dict(heads=2 ** 32 + 32), dict(max_new=2 ** 32 + 1), dict(max_kv=2 ** 32 + 64),
                                 dict(max_kv=-2 ** 32 + 64), dict(max_new=2 ** 31)], ids=str)
def test_sizes_past_32_bits_are_refused(lib, big):
    """They would be cut to their low 32 bits, which the library could find fine."""
    with pytest.raises(ValueError):
        batch(cache(Calls(lib)), **big)


def test_windows_past_32_bits(lib):
    """A window that no sequence can fill hides nothing; a negative one stays one, which the library refuses."""
    calls = Calls(lib)
    c = cache(calls)
    b = batch(c)
    for window in (5, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, -1, -2 ** 32 + 5):
        c.attend_decode(b, q_of(c), window=window)
    assert [args[-2] for args in calls.made] == [5, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1, -1, -1]
