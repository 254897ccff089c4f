"""A cache in 8 bits in the layouts at the documented limits (large pages, rows far apart, keys and values in one tensor), sequences that share
full pages, and prompts and decode in turn on one batch's workspace."""
import pytest
from test_gpu_attention import make
from test_gpu_attention8 import Made, check, held, reference, values

pytestmark = pytest.mark.gpu


def append_and_attend(torch, m, seed):
    """The new rows of m's batch appended, and all of its rows attended over what the cache then holds."""
    rows = m.q.shape[0]
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = 3 * torch.randn((rows, m.k.shape[1], m.k.shape[3]), generator=g, device="cuda")
    m.cache.append(m.batch, None, x, 2 * x)
    row = 0
    for s, (new, old) in enumerate(m.lengths):
        at = torch.arange(old, old + new, device="cuda")
        pg = m.table[s][at // m.page].long()
        for codes, exps, want in ((m.k, m.k_exp, x[row:row + new].double()), (m.v, m.v_exp, 2 * x[row:row + new].double())):
            step = torch.exp2(exps[pg, :, at % m.page // 16].double())[..., None]
            got = codes.view(torch.uint8)[pg, :, at % m.page].view(torch.float8_e4m3fn).double() * step
            assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * step).all()
        row += new
    ref = reference(m)
    for call, prompt in ((m.cache.attend_decode, False), (m.cache.attend_prompt, True)):
        check(torch, call(m.batch, m.q, out=m.empty(torch.float32)), ref, prompt)


@pytest.mark.parametrize("page", (2048, 65536))
@pytest.mark.parametrize("layout", ((4, 2, 64), (4, 1, 128)), ids=str)
def test_large_pages(gpu, lib, layout, page):
    import torch
    m = Made(torch, layout, page, "float16", [(3, page - 2), (5, 100), (1, 0)] if page == 2048 else [(3, 65534), (2, 40)], 81)
    append_and_attend(torch, m, 82)


@pytest.mark.parametrize("dim", (64, 96, 128))
def test_rows_far_apart(gpu, lib, dim):
    """Rows nearly 2^26 bytes apart."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    m = Made(torch, (4, 1, dim), 16, "float16", [(3, 18)], 83)
    row, pages = (1 << 26) - 16, m.k.shape[0]
    big = [torch.empty(pages * 16 * row + dim, dtype=torch.uint8, device="cuda") for _ in range(2)]
    k, v = (b.as_strided((pages, 1, 16, dim), (16 * row, 16 * row, row, 1)) for b in big)
    k.copy_(m.k.view(torch.uint8))
    v.copy_(m.v.view(torch.uint8))
    m.k, m.v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
    m.cache = KvCache8(m.k, m.v, m.k_exp, m.v_exp)
    m.batch = Batch(m.cache, 4, m.q_start, m.kv_len, m.table, 3, 21)
    append_and_attend(torch, m, 84)


def test_keys_and_values_in_one_tensor(gpu, lib):
    import torch
    from lazyweights_amd import Batch, KvCache8
    m = Made(torch, (8, 2, 96), 32, "bfloat16", [(3, 77), (4, 130)], 85)
    both = torch.stack((m.k.view(torch.uint8), m.v.view(torch.uint8)), 1).view(torch.float8_e4m3fn)
    exps = torch.stack((m.k_exp, m.v_exp), 2)
    m.k, m.v, m.k_exp, m.v_exp = both[:, 0], both[:, 1], exps[:, :, 0], exps[:, :, 1]
    m.cache = KvCache8(m.k, m.v, m.k_exp, m.v_exp)
    m.batch = Batch(m.cache, 8, m.q_start, m.kv_len, m.table, 4, 134)
    append_and_attend(torch, m, 86)


def test_sequences_that_share_full_pages(gpu, lib):
    """A prefix of full pages in several sequences' tables: read by all, and written by nobody who appends behind it."""
    import torch
    m = Made(torch, (8, 2, 128), 32, "float16", [(3, 64), (5, 70), (1, 64), (9, 128)], 87)
    for s in range(1, 4):
        m.table[s, :2] = m.table[0, :2]
    shared = m.table[0, :2].long()
    before = [t[shared].view(torch.uint8).clone() for t in (m.k, m.v, m.k_exp, m.v_exp)]
    append_and_attend(torch, m, 88)
    for now, was in zip((m.k, m.v, m.k_exp, m.v_exp), before):
        assert torch.equal(now[shared].view(torch.uint8), was)


@pytest.mark.parametrize("layout, lengths", [((8, 2, 128), [(16, 6000), (1, 300)]), ((4, 4, 64), [(9, 4000)]),
                                             ((16, 2, 96), [(5, 9000), (16, 20), (0, 7)])], ids=str)
@pytest.mark.parametrize("eight", (False, True))
def test_prompts_and_decode_in_turn(gpu, lib, eight, layout, lengths):
    """A batch of few new tokens over long keys: prompt attention lays its shares of the keys behind the counters of decode's."""
    import torch
    from lazyweights_amd import Batch, KvCache
    most, longest = max(n for n, _ in lengths), max(n + o for n, o in lengths)
    if eight:
        m = Made(torch, layout, 16, "float16", lengths, 89)
        cache, batch, q, ref = m.cache, m.batch, m.q, reference(m)
    else:
        from test_gpu_attention import check as check16, reference as reference16
        k, v, table, starts, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 89)
        cache = KvCache(k, v)
        batch = Batch(cache, layout[0], starts, kv_len, table, most, longest)
        ref = reference16(torch, k, v, table, lengths, q, 0, layout[2] ** -0.5)
    first = {}
    for turn in range(6):
        name = "attend_prompt" if turn % 2 else "attend_decode"
        y = getattr(cache, name)(batch, q, out=torch.full(q.shape, float("nan"), device="cuda"))
        if eight:
            check(torch, y, ref, turn % 2 == 1)
        else:
            check16(torch, y, ref, torch.float16, turn % 2 == 1)
        assert torch.equal(first.setdefault(name, y), y)
