"""Appending to and attention over a paged cache held in 8 bits (lw_kv8_append, lw_attn8_decode, lw_attn8_prompt) against plain
forms in 64 bits of what the cache holds: head layouts, types, lengths from none on, page sizes, windows, exponents, pages that
are not there, NaN in places a row does not see, layouts, long caches, streams and captured calls.

Bounds of attention, elementwise, from the types and the kernels' arithmetic (A = sum p |v| / sum p of the row, n its keys):
  the output's rounding          u |out|, u = 2^-24, 2^-11, 2^-8 for fp32, fp16, bf16 (and 2^-25 for small fp16 outputs)
  the weights' rounding          u_p A: 2^-11 where they are one 16-bit part (prompt, 16-bit out), else 2^-21
  small weights                  n 2^-41 (decode) or 2^-37 (prompt) of 448 max_j p_j 2^e_j / sum p: half of fp16's least step, 2^-24,
                                 where the largest product of a weight and its value's 2^e is lifted to 2^15, or 2^11 at least
  scores, sums, the exponential  A (2 2^-21 max_j scale sum |q k_j| + 2^-20): products exact, a score's sum in a few steps
"""
import pytest
from test_gpu_attention import make

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def held(torch, x, spare):
    """x [pages, kv, page, dim] in 8 bits, blocks' exponents up to `spare` above the least (NaN stay NaN): numbers, exponents."""
    blocks = x.unflatten(2, (-1, 16))
    most = torch.nan_to_num(blocks, 0.0).abs().amax((-2, -1)).double().clamp(min=1e-30)
    e = torch.ceil(torch.log2(most / 448)).int()
    g = torch.Generator(device="cuda").manual_seed(7)
    e = (e + torch.randint(0, spare + 1, e.shape, generator=g, device="cuda")).clamp(-48, 48).int()
    codes = torch.ldexp(blocks, -e[..., None, None]).flatten(2, 3).to(torch.float8_e4m3fn)
    return codes, e.to(torch.int8)


def values(torch, codes, exps):
    """What a cache holds, in 64 bits."""
    e = exps.double().clamp(-48, 48)
    return (codes.double().unflatten(2, (-1, 16)) * torch.exp2(e)[..., None, None]).flatten(2, 3)


class Made:
    def __init__(self, torch, layout, page, q_type, lengths, seed, max_new=None, max_kv=None, spread=4, rows_first=False, **kw):
        from lazyweights_amd import Batch, KvCache8
        k, v, self.table, self.q_start, self.kv_len, q = make(torch, layout, page, torch.float32, lengths, seed, **kw)
        g = torch.Generator(device="cuda").manual_seed(seed + 1000)
        shape = (v.shape[0], v.shape[1], page // 16, 1, 1)
        power = torch.exp2(torch.randint(-spread, spread + 1, shape, generator=g, device="cuda").float())
        v = (v.unflatten(2, (-1, 16)) * power).flatten(2, 3)
        (self.k, self.k_exp), (self.v, self.v_exp) = held(torch, k, 2), held(torch, v, 1)
        if rows_first:
            self.k, self.v = (t.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn)
                              for t in (self.k, self.v))
        self.q, self.lengths, self.page, self.heads = q.to(getattr(torch, q_type)), lengths, page, layout[0]
        self.max_new = max_new or max(n for n, _ in lengths)
        self.max_kv = max_kv or max(n + o for n, o in lengths)
        self.cache = KvCache8(self.k, self.v, self.k_exp, self.v_exp)
        self.batch = Batch(self.cache, layout[0], self.q_start, self.kv_len, self.table, self.max_new, self.max_kv)
        self.torch = torch

    def put(self, where, s, pos, code, head=slice(None), dim=slice(None)):
        where.view(self.torch.uint8)[int(self.table[s, pos // self.page]), head, pos % self.page, dim] = code

    def empty(self, kind):
        return self.torch.full(self.q.shape, float("nan"), dtype=kind, device="cuda")


def reference(m, window=0, scale=None):
    """(out, A, max scale sum |q k|, n, 448 max p 2^e / sum p) per row and head over the seen keys, in 64 bits."""
    torch = m.torch
    k, v = values(torch, m.k, m.k_exp), values(torch, m.v, m.v_exp)
    pages, kv, page, dim = k.shape
    heads = m.heads
    group, scale = heads // kv, dim ** -0.5 if scale is None else scale
    out = torch.zeros(m.q.shape, dtype=torch.float64, device="cuda")
    a, most = torch.zeros_like(out), torch.zeros(m.q.shape[:2] + (1,), dtype=torch.float64, device="cuda")
    n_keys, top = torch.zeros_like(most), torch.zeros_like(most)
    row, tab = 0, m.table.cpu()
    for s, (new, old) in enumerate(m.lengths):
        j = torch.arange(old + new)
        pg = tab[s][j // page].long()
        ok = (pg >= 0) & (pg < pages)
        j, pg = j[ok], pg[ok].cuda()
        off = (j % page).cuda()
        kk, vv = k[pg, :, off], v[pg, :, off]  # [keys, kv, dim]
        power = torch.exp2(m.v_exp[pg, :, off // 16].double().clamp(-48, 48))
        j = j.cuda()
        for i in range(old, old + new):
            see = (j <= i) & (j > i - window if window else j >= 0)
            if int(see.sum()):
                qq = m.q[row].double().view(kv, group, dim)
                x, y = kk[see], vv[see]
                p = torch.softmax(torch.einsum("hgd,jhd->hgj", qq, x) * scale, -1)
                out[row] = torch.einsum("hgj,jhd->hgd", p, y).reshape(heads, dim)
                a[row] = torch.einsum("hgj,jhd->hgd", p, y.abs()).reshape(heads, dim)
                most[row] = (torch.einsum("hgd,jhd->hgj", qq.abs(), x.abs()) * abs(scale)).amax(-1).reshape(heads, 1)
                n_keys[row] = x.shape[0]
                top[row] = 448 * (p * power[see].T[:, None]).amax(-1).reshape(heads, 1)
            row += 1
    return out, a, most, n_keys, top


def check(torch, y, ref, prompt):
    out, a, most, n, top = ref
    kind = str(y.dtype).split(".")[1]
    part = 2.0 ** -11 if prompt and kind != "float32" else 2.0 ** -21
    bound = (U[kind] * out.abs() + a * (part + 2 * 2.0 ** -21 * most + 2.0 ** -20) + n * top * 2.0 ** (-37 if prompt else -41) +
             (2.0 ** -25 if kind == "float16" else 0))
    err = (y.double() - out).abs()
    worst = (err / (bound + 1e-30)).max().item() if err.numel() else 0.0
    print("worst error / bound %.3f" % worst, flush=True)
    assert (err <= bound).all(), worst


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 500, 1025]

DECODE = [
    # layout (heads, kv heads, dim), page, type of q, out, new per sequence, window
    ((8, 8, 64), 16, "float16", "float16", [1], 0),
    ((8, 2, 128), 16, "float16", "float32", [1], 0),
    ((7, 1, 96), 32, "bfloat16", "bfloat16", [1, 0, 1], 0),
    ((8, 1, 128), 64, "bfloat16", "float32", [5, 1, 0, 3], 0),
    ((32, 2, 64), 16, "float16", "float32", [1, 2], 0),
    ((12, 4, 96), 128, "float16", "bfloat16", [16, 7, 11], 0),
    ((8, 2, 128), 32, "float16", "float32", [1], 1),
    ((8, 2, 128), 16, "bfloat16", "float32", [4, 1], 33),
    ((16, 1, 64), 1024, "float16", "float16", [3], 100),
    ((64, 1, 128), 16, "float16", "float32", [2, 9], 0),
    ((4, 4, 96), 16, "float16", "float32", [16], 40),
]


@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode(gpu, lib, case):
    import torch
    layout, page, q_type, out, news, window = case
    m = Made(torch, layout, page, q_type, [(news[i % len(news)], n) for i, n in enumerate(LENGTHS)], 11, max(news), 1025 + max(news))
    y, ref = m.empty(getattr(torch, out)), reference(m, window)
    for _ in range(3):  # the later calls find the workspace as the first left it
        y.fill_(float("nan"))
        assert m.cache.attend_decode(m.batch, m.q, out=y, window=window) is y
        check(torch, y, ref, False)


@pytest.mark.parametrize("bounds", [(1, 3001), (16, 16000), (1, 100), (3, 1)], ids=str)
def test_decode_bounds_other_than_the_lengths(gpu, lib, bounds):
    """max_kv and max_new far above what the arrays hold, and lengths above max_kv, give the same values."""
    import torch
    m = Made(torch, (8, 2, 128), 16, "float16", [(1, 40), (1, 3000), (1, 700)], 12, *bounds, width=1000)
    check(torch, m.cache.attend_decode(m.batch, m.q, out=m.empty(torch.float32)), reference(m), False)


BATCHES = [
    # layout, sequences, longest, bound on the length, new tokens
    ((2, 1, 64), 301, 40, 5000, 2),
    ((8, 8, 96), 70, 700, 700, 1),
    ((16, 8, 128), 130, 600, 600, 1),
    ((4, 2, 128), 3, 250, 250, 4),
    ((64, 2, 96), 5, 2000, 2000, 1),
    ((8, 4, 64), 1000, 3, 9000, 1),
    ((32, 1, 128), 9, 4100, 16000, 3),
    # many items with long bounds: equal runs of the list, of up to 64 sequences and of more
    ((32, 8, 128), 60, 900, 6000, 2),
    ((8, 4, 128), 300, 200, 4500, 1),
    ((16, 8, 128), 33, 5000, 5000, 1),
    ((16, 8, 128), 20, 2500, 2500, 1),
    ((32, 8, 128), 9, 900, 17000, 1),
    # parts of a size
    ((8, 8, 64), 28, 700, 9000, 1),
    # two row tiles in a block per item, in parts
    ((32, 4, 128), 130, 300, 600, 3),
    ((24, 4, 64), 300, 60, 2000, 5),
    ((20, 2, 96), 70, 700, 9000, 4),
]


@pytest.mark.parametrize("case", BATCHES, ids=str)
def test_decode_batches(gpu, lib, case):
    import random

    import torch
    layout, seqs, longest, bound, most = case
    rng = random.Random(seqs)
    lengths = [(rng.randrange(0 if seqs > 60 else 1, most + 1), rng.choice((0, 1, 31, 32, 33, longest - 5, rng.randrange(longest))))
               for _ in range(seqs)]
    lengths = [(n, max(0, min(o, longest - n))) for n, o in lengths]
    m = Made(torch, layout, 16, "float16", lengths, 28, most, bound, width=-(-bound // 16))
    ref = reference(m)
    first = None
    for _ in range(2):
        y = m.cache.attend_decode(m.batch, m.q, out=m.empty(torch.float32))
        check(torch, y, ref, False)
        first = y if first is None else first
        assert torch.equal(y, first)


PROMPT = [
    ((8, 8, 64), 16, "float16", "float16", [(1, 0), (2, 0), (33, 0), (0, 0), (64, 0), (129, 0)], 0),
    ((8, 2, 128), 16, "float16", "float32", [(31, 0), (32, 0), (200, 0), (1, 0)], 0),
    ((7, 1, 96), 32, "bfloat16", "bfloat16", [(300, 0), (1, 64), (17, 0)], 0),
    ((4, 2, 128), 64, "bfloat16", "float32", [(65, 190), (127, 1), (3, 700)], 0),
    ((6, 2, 96), 16, "float16", "float32", [(90, 30), (5, 5)], 0),
    ((4, 1, 64), 32, "float16", "bfloat16", [(257, 0), (100, 333)], 0),
    ((8, 2, 128), 16, "float16", "float32", [(250, 0), (70, 100), (1, 9)], 1),
    ((8, 2, 128), 256, "bfloat16", "float32", [(250, 0), (70, 100)], 65),
    ((4, 4, 96), 16, "float16", "float16", [(400, 20), (300, 0)], 100),
    ((3, 3, 64), 16, "bfloat16", "float32", [(0, 50), (513, 0)], 0),
    # few rows over many keys
    ((4, 2, 128), 16, "float16", "float32", [(20, 3000), (1, 5000), (130, 700), (0, 9), (33, 0)], 0),
    ((8, 1, 96), 64, "bfloat16", "bfloat16", [(40, 6001), (17, 300)], 0),
    ((4, 4, 64), 16, "float16", "float16", [(300, 4000), (5, 100)], 3500),
    # many rows
    ((512, 512, 64), 16, "float16", "float16", [(300, 0), (0, 5), (150, 200), (1, 0), (61, 64)], 0),
    ((512, 512, 128), 64, "bfloat16", "float32", [(300, 0), (0, 5), (150, 200), (1, 0), (61, 64)], 70),
    ((512, 512, 96), 32, "float16", "bfloat16", [(300, 0), (0, 5), (150, 200), (1, 0), (61, 64)], 0),
]


@pytest.mark.parametrize("case", PROMPT, ids=str)
def test_prompt(gpu, lib, case):
    import torch
    layout, page, q_type, out, lengths, window = case
    m = Made(torch, layout, page, q_type, lengths, 13)
    ref = reference(m, window)
    for workspace in (True, False):
        if not workspace:
            m.batch.c.workspace, m.batch.c.workspace_bytes = None, 0
        y = m.empty(getattr(torch, out))
        m.cache.attend_prompt(m.batch, m.q, out=y, window=window)
        check(torch, y, ref, True)


def test_many_sequences(gpu, lib):
    """More sequences than lanes, empty ones among them: rows find theirs."""
    import torch
    m = Made(torch, (2, 1, 64), 16, "float16", [((i * 7) % 5 % 3, (i * 11) % 40) for i in range(301)], 14, 2, 42)
    ref = reference(m)
    for call, prompt in ((m.cache.attend_decode, False), (m.cache.attend_prompt, True)):
        check(torch, call(m.batch, m.q, out=m.empty(torch.float32)), ref, prompt)


@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_pages_that_are_not_there(gpu, lib, call):
    import torch
    m = Made(torch, (4, 2, 96), 16, "float16", [(5, 200), (3, 13), (2, 0), (4, 60)], 15, unmapped=[(0, 1), (0, 4), (0, 12), (1, 0), (2, 0), (3, 3)])
    y = getattr(m.cache, call)(m.batch, m.q, out=m.empty(torch.float32))
    assert (y[8:10] == 0).all()  # nothing to see: zeros
    check(torch, y, reference(m), call == "attend_prompt")


@pytest.mark.parametrize("dim", (64, 96, 128))
@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_what_a_row_does_not_see_never_reaches_it(gpu, lib, call, dim):
    """NaN in keys and values at positions after a row's, or before its window."""
    import torch
    window = 90
    m = Made(torch, (4, 2, dim), 16, "float16", [(9, 100), (16, 0), (7, 300)], 16)
    ref = reference(m, window)
    for where in (m.k, m.v):
        m.put(where, 0, 105, 0x7F)  # rows 0..4 of sequence 0 do not see it
        m.put(where, 1, 8, 0xFF)    # rows 0..7 of sequence 1
        m.put(where, 1, 15, 0x7F)
        m.put(where, 2, 210, 0x7F)  # before every window of sequence 2 (first row: 211 .. 300)
        m.put(where, 2, 304, 0xFF)
    y = getattr(m.cache, call)(m.batch, m.q, out=m.empty(torch.float32), window=window)
    clean = [0, 1, 2, 3, 4] + [9 + i for i in range(8)] + [25 + i for i in range(4)]
    check(torch, y[clean], [t[clean] for t in ref], call == "attend_prompt")
    assert torch.isnan(y[5:9]).all() and torch.isnan(y[17:25]).all() and torch.isnan(y[29:]).all()


@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_a_value_that_is_nan_is_so_in_its_element_alone(gpu, lib, call):
    import torch
    m = Made(torch, (4, 2, 64), 16, "bfloat16", [(6, 70)], 17)
    ref = reference(m)
    m.put(m.v, 0, 35, 0x7F, 1, 20)
    m.put(m.v, 0, 73, 0xFF, 0, 7)
    y = getattr(m.cache, call)(m.batch, m.q, out=m.empty(torch.float32))
    assert torch.isnan(y[:, 2:, 20]).all() and torch.isnan(y[3:, :2, 7]).all()
    there = torch.isfinite(y)
    assert int((~there).sum()) == 6 * 2 + 3 * 2
    check(torch, torch.where(there, y, 0), [torch.where(there, ref[0], 0)] + list(ref[1:]), call == "attend_prompt")


@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
@pytest.mark.parametrize("k_exp, v_exp", [(-48, 48), (48, -48), (-120, 127), (0, 100)], ids=str)
def test_exponents_far_apart(gpu, lib, call, k_exp, v_exp):
    """The smallest and largest exponents beside ordinary ones, and what is past them (taken as the nearer): scores of 2^48 and more
    among the keys, values of 2^48 among ones of 2^-48."""
    import torch
    m = Made(torch, (4, 2, 128), 32, "float16", [(3, 200), (2, 40)], 18)
    at = [(int(m.table[0, 2]), 0), (int(m.table[0, 4]), 1), (int(m.table[1, 0]), 1)]
    for p, b in at:
        m.v_exp[p, :, b] = v_exp
        if k_exp < 0:
            m.k_exp[p, :, b] = k_exp
    if k_exp > 0:  # (two keys alone in a block: their scores are 2^48 times the others', one with each sign)
        p, b = at[0]
        m.k_exp[p, :, b] = k_exp
        m.k.view(torch.uint8)[p, :, 16 * b:16 * b + 16] = 0
        m.k.view(torch.uint8)[p, :, 16 * b, 0] = 0x38
        m.q[..., 0] = -1
    y = getattr(m.cache, call)(m.batch, m.q, out=m.empty(torch.float32))
    assert torch.isfinite(y).all()
    check(torch, y, reference(m), call == "attend_prompt")


def test_scores_far_apart(gpu, lib):
    """Scores of hundreds, first rising and then falling, all alike, and the smallest product first."""
    import torch
    m = Made(torch, (2, 1, 64), 16, "float16", [(1, 500), (1, 500)], 19)
    m.q.fill_(1.0)
    for s, sign in ((0, 1.0), (1, -1.0)):
        for p in range(501):
            page, off = int(m.table[s, p // 16]), p % 16
            m.k_exp[page, :, off // 16] = 0
            m.k[page, :, off] = torch.tensor(sign * (p - 250) / 8).to(torch.float8_e4m3fn).item()
    for scale in (0.125, 0.0, -0.05):
        ref = reference(m, 0, scale)
        for call, prompt in ((m.cache.attend_decode, False), (m.cache.attend_prompt, True)):
            check(torch, call(m.batch, m.q, out=m.empty(torch.float32), scale=scale), ref, prompt)


def test_layouts_and_strides(gpu, lib):
    """A cache with rows before heads, exponents apart, q and out as parts of wider rows: the same bits."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    ys = []
    for rows_first in (False, True):
        m = Made(torch, (8, 2, 96), 32, "bfloat16", [(3, 77), (4, 130)], 20, rows_first=rows_first)
        if rows_first:
            wide = [torch.full((t.shape[0], 3, 5), 9, dtype=torch.int8, device="cuda") for t in (m.k_exp, m.v_exp)]
            for w, t in zip(wide, (m.k_exp, m.v_exp)):
                w[:, 1:, 2:4] = t
            m.cache = KvCache8(m.k, m.v, *(w[:, 1:, 2:4] for w in wide))
            m.batch = Batch(m.cache, 8, m.q_start, m.kv_len, m.table, 4, 134)
        wide = torch.full((7, 3 * 8 * 96), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, 768:1536] = m.q.view(7, -1)
        for call in (m.cache.attend_decode, m.cache.attend_prompt):
            out = torch.full((7, 2 * 768), float("nan"), device="cuda")
            call(m.batch, wide[:, 768:1536], out=out[:, 768:])
            assert torch.isnan(out[:, :768]).all()
            ys += [out[:, 768:].clone(), call(m.batch, m.q, out=m.empty(torch.float32)).view(7, -1)]
    for i in (1, 4, 5):
        assert torch.equal(ys[0], ys[i]) and torch.equal(ys[2], ys[i + 2])


def test_offsets_past_32_bits(gpu, lib):
    """Pages 4 GB and more into the cache."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    m = Made(torch, (4, 2, 64), 64, "float16", [(2, 100)], 21)
    stride = 3 << 30  # bytes from a page to the next
    big = [torch.empty(3 * stride + 2 * 64 * 64, dtype=torch.uint8, device="cuda") for _ in range(2)]
    k, v = (b.as_strided((4, 2, 64, 64), (stride, 64 * 64, 64, 1)) for b in big)
    k.copy_(m.k.view(torch.uint8))
    v.copy_(m.v.view(torch.uint8))
    cache = KvCache8(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), m.k_exp.clone(), m.v_exp.clone())
    batch = Batch(cache, 4, m.q_start, m.kv_len, m.table, 2, 102)
    for call in ("attend_decode", "attend_prompt"):
        assert torch.equal(getattr(cache, call)(batch, m.q), getattr(m.cache, call)(m.batch, m.q))
    x = 9 * torch.randn((2, 2, 64), device="cuda")
    cache.append(batch, None, x, 2 * x)
    m.cache.append(m.batch, None, x, 2 * x)
    for a, b in ((k, m.k), (v, m.v)):
        assert torch.equal(a, b.view(torch.uint8))


def test_long_cache_same_bits_every_call(gpu, lib):
    import torch
    from lazyweights_amd import Batch, KvCache8
    g = torch.Generator(device="cuda").manual_seed(22)
    pages = 70001 // 128 + 3
    (k, k_exp), (v, v_exp) = (held(torch, torch.randn((pages, 1, 128, 128), generator=g, device="cuda"), 1) for _ in range(2))
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.stack((table, table.flip(0))).contiguous()
    q_start = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([70001, 11], dtype=torch.int32, device="cuda")
    q = torch.randn((3, 8, 128), generator=g, device="cuda").half()
    cache = KvCache8(k, v, k_exp, v_exp)
    batch = Batch(cache, 8, q_start, kv_len, table, 2, 70001)
    first = cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32))
    for _ in range(20):
        assert torch.equal(cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32)), first)
    kk, vv = (values(torch, *t)[table[0].long(), 0].reshape(-1, 128)[:70001] for t in ((k, k_exp), (v, v_exp)))
    ref = torch.softmax(q[0].double() @ kk.T.contiguous() * 128 ** -0.5, -1) @ vv
    assert ((first[0].double() - ref).norm() / ref.norm()).item() < 1e-5


@pytest.mark.parametrize("window", (0, 100000))
def test_long_parts(gpu, lib, window):
    """One long sequence, whose parts are of blocks with 8 waves: some rows against 64 bits, NaN that only the last row sees."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    g = torch.Generator(device="cuda").manual_seed(32)
    keys, kv, heads, page = 140003, 4, 16, 64
    pages = -(-keys // page)
    (k, k_exp), (v, v_exp) = (held(torch, torch.randn((pages, kv, page, 128), generator=g, device="cuda"), 1) for _ in range(2))
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None].contiguous()
    cache = KvCache8(k, v, k_exp, v_exp)
    batch = Batch(cache, heads, torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
                  torch.tensor([keys], dtype=torch.int32, device="cuda"), table, 3, keys)
    q = torch.randn((3, heads, 128), generator=g, device="cuda").half()
    v.view(torch.uint8)[int(table[0, (keys - 1) // page]), 1, (keys - 1) % page, 9] = 0x7F
    y = cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32), window=window)
    assert torch.isnan(y[2, 4:8, 9]).all() and int(torch.isnan(y).sum()) == 4
    for row in range(2):
        at = torch.arange(max(0, keys - 2 + row - window) if window else 0, keys - 2 + row, device="cuda")
        kk, vv = (values(torch, *t)[table[0, at // page].long(), :, at % page] for t in ((k, k_exp), (v, v_exp)))
        p = torch.softmax(torch.einsum("hgd,jhd->hgj", q[row].double().view(kv, 4, 128), kk) * 128 ** -0.5, -1)
        ref = torch.einsum("hgj,jhd->hgd", p, vv).reshape(heads, 128)
        assert ((y[row].double() - ref).norm() / ref.norm()).item() < 1e-5


def test_streams_and_captured_calls(gpu, lib):
    """On another stream, and captured: replays read the lengths, pages and rows of their time."""
    import torch
    m = Made(torch, (8, 2, 128), 16, "float16", [(1, 300), (1, 20)], 23, 1, 600, width=40)
    x, kx, vx = (torch.randn((2, h, 128), device="cuda") for h in (8, 2, 2))
    turn = torch.arange(600, device="cuda")[:, None] * 0.01 ** (torch.arange(64, device="cuda") / 64)
    cos, sin = turn.cos().contiguous(), turn.sin().contiguous()
    q16, y, z = torch.empty_like(x, dtype=torch.float16), torch.empty_like(x), torch.empty_like(x)

    def step():
        m.cache.append(m.batch, x, kx, vx, cos, sin, q_out=q16)
        m.cache.attend_decode(m.batch, q16, out=y)
        m.cache.attend_prompt(m.batch, q16, out=z)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    on_side = (q16.clone(), y.clone(), z.clone())
    step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(on_side, (q16, y, z)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    state = (m.k, m.v, m.k_exp, m.v_exp)
    for grow in range(4):
        m.kv_len += 1 + grow
        for t in (x, kx, vx):
            t.normal_(std=1 + grow)
        before = [t.view(torch.uint8).clone() for t in state]
        graph.replay()
        torch.cuda.synchronize()
        got = [t.view(torch.uint8).clone() for t in (q16, y, z) + state]
        for t, b in zip(state, before):
            t.view(torch.uint8).copy_(b)
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(got, (q16, y, z) + state)), grow


@pytest.mark.parametrize("which", ("decode", "prompt", "append"))
def test_calls_on_another_stream(gpu, lib, which):
    """Outputs are of the given stream's memory, and inputs last until it has read them."""
    import torch
    m = Made(torch, (8, 2, 128), 16, "float16", [(5, 300), (16, 64)], 24)
    g = torch.Generator(device="cuda").manual_seed(25)
    new = [torch.randn((21, h, 128), generator=g, device="cuda").half() for h in (8, 2, 2)] if which == "append" else [m.q]
    call = {"decode": lambda t, s: m.cache.attend_decode(m.batch, t[0], stream=s),
            "prompt": lambda t, s: m.cache.attend_prompt(m.batch, t[0], stream=s),
            "append": lambda t, s: m.cache.append(m.batch, *t, stream=s)}[which]
    want = call(new, None).clone()
    side = torch.cuda.Stream()
    tensors = [t.clone() for t in new]
    like, places = [torch.empty_like(t, device="meta") for t in tensors], {t.data_ptr() for t in tensors}
    torch.cuda.synchronize()
    block = torch.empty_like(want)
    at = block.data_ptr()
    torch.cuda._sleep(20_000_000)
    block.fill_(float("nan"))
    del block  # free for the current stream, which has yet to write it
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    y = call(tensors, side.cuda_stream)
    assert y.data_ptr() != at
    del tensors
    for t in like:
        assert torch.full(t.shape, float("nan"), dtype=t.dtype, device="cuda").data_ptr() not in places
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("news, old, max_kv, layout, window", [
    ([1], 40, 200, (8, 2, 128), 0), ([1, 3, 0], 5000, 8192, (8, 2, 128), 0), ([16] * 3, 70000, 70016, (32, 2, 64), 100),
    ([1] * 70, 900, 2000, (4, 1, 96), 0), ([40], 0, 40, (8, 8, 64), 0), ([64], 20000, 20064, (8, 2, 128), 0),
    ([9000], 100, 10000, (32, 4, 64), 50)], ids=str)
def test_no_pages(gpu, lib, news, old, max_kv, layout, window):
    """A cache without pages: nothing is appended, q is rotated all the same, rows see nothing."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    heads, kv, dim = layout
    cache = KvCache8.empty(0, kv, 16, dim)
    starts = torch.tensor([0] + news, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    batch = Batch(cache, heads, starts, torch.tensor([n + old for n in news], dtype=torch.int32, device="cuda"),
                  torch.zeros((len(news), -(-max_kv // 16)), dtype=torch.int32, device="cuda"), max(news), max_kv)
    q, k = (torch.randn((sum(news), h, dim), device="cuda") for h in (heads, kv))
    q16 = cache.append(batch, q, k, k)
    assert torch.equal(q16, q.half())
    for attend in ([cache.attend_decode] if max(news) <= 16 else []) + [cache.attend_prompt]:
        y = attend(batch, q16, out=torch.full(q.shape, float("nan"), device="cuda"), window=window)
        torch.cuda.synchronize()
        assert not y.any()


# ── append ──────────────────────────────────────────────────────────────────────────────────────────────────────────

APPEND = [
    # layout, page, type of q_out, x type, rot, neighbours, size of new rows, (new, old) per sequence
    ((8, 2, 128), 16, "float16", "float32", 128, False, 1, [(1, 0)]),
    ((8, 8, 64), 16, "bfloat16", "float32", 64, False, 40, [(1, 5), (1, 31), (1, 32)]),
    ((7, 1, 96), 16, "float16", "float16", 96, True, 3, [(5, 0), (0, 3), (13, 4), (1, 70)]),
    ((4, 2, 128), 64, "bfloat16", "bfloat16", 64, False, 0.01, [(100, 3), (1, 0)]),
    ((4, 4, 64), 32, "float16", "bfloat16", 32, True, 100, [(17, 2), (3, 9), (30, 1)]),
    ((6, 3, 96), 128, "bfloat16", "float16", 8, False, 30, [(33, 100), (15, 1), (16, 16)]),
    ((4, 2, 128), 16, "float16", "float32", 0, False, 1e-3, [(40, 1), (0, 0), (2, 2)]),
    ((20, 1, 128), 16, "float16", "float32", 128, False, 5, [(i % 3, 7 * i % 40) for i in range(200)]),
    ((1, 1, 64), 16, "float16", "float32", 64, False, 5, [(1, i) for i in range(90)]),
    # (a wave with heads for some of its lanes only, and sequences to search)
    ((3, 1, 64), 16, "float16", "float32", 64, False, 5, [(i % 3, 7 * i % 40) for i in range(200)]),
    ((21, 7, 96), 16, "bfloat16", "float16", 96, True, 5, [(3 * i % 7, 5 * i % 90) for i in range(70)]),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, lib, case):
    import torch
    layout, page, q_type, x_type, rot, neighbours, size, lengths = case
    heads, kv, dim = layout
    q_type, x_type = getattr(torch, q_type), getattr(torch, x_type)
    m = Made(torch, layout, page, "float16", lengths, 26)
    rows, most = int(m.q_start[-1]), m.max_kv
    g = torch.Generator(device="cuda").manual_seed(27)
    # one joined projection with a row that belongs to no sequence
    joined = (size * torch.randn((rows + 1, (heads + 2 * kv) * dim), generator=g, device="cuda")).to(x_type)
    q, kx, vx = joined.split((heads * dim, kv * dim, kv * dim), 1)
    turn = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(max(rot // 2, 1), dtype=torch.float64, device="cuda") / max(rot // 2, 1))
    cos, sin = turn.cos().float(), turn.sin().float()
    before = [t.clone() for t in (m.k, m.v, m.k_exp, m.v_exp)]
    out = torch.full((rows + 1, heads, dim), float("nan"), dtype=q_type, device="cuda")
    got = m.cache.append(m.batch, q, kx, vx, *((cos, sin) if rot else (None, None)), q_out=out, neighbours=neighbours)
    assert got is out and torch.isnan(out[rows:]).all()

    def turned(x, i):
        x = x.double().clone()
        if rot:
            c, n = cos[i].double()[:, None], sin[i].double()[:, None]
            a, b = (slice(0, rot, 2), slice(1, rot, 2)) if neighbours else (slice(0, rot // 2), slice(rot // 2, rot))
            p, r = x[..., a].clone(), x[..., b].clone()
            x[..., a], x[..., b] = p * c - r * n, r * c + p * n
        return x

    untouched = torch.ones((m.k.shape[0], kv, page), dtype=torch.bool, device="cuda")
    same_exp = torch.ones_like(m.k_exp, dtype=torch.bool)
    row = 0
    for s, (new, old) in enumerate(lengths):
        at = torch.arange(old, old + new, device="cuda")
        mine = slice(row, row + new)
        row += new
        if not new:
            continue
        x = q[mine].reshape(new, heads, dim)
        ref = turned(x, at)
        width = x.double().abs().amax(-1, keepdim=True)  # the rounding, and that of three fp32 operations
        assert ((out[mine].double() - ref).abs() <= U[str(q_type).split(".")[1]] * ref.abs() + 2.0 ** -22 * width + 2.0 ** -25).all()
        for x, codes, exps, was, was_exp, rotated in ((kx, m.k, m.k_exp, before[0], before[2], True),
                                                      (vx, m.v, m.v_exp, before[1], before[3], False)):
            x = x[mine].reshape(new, kv, dim)
            ref = turned(x, at) if rotated else x.double()
            slack = (2.0 ** -22 if rotated and rot else 0) * x.double().abs().amax(-1, keepdim=True)
            for block in range(old // 16, (old + new + 15) // 16):
                pg, b = int(m.table[s, 16 * block // page]), 16 * block % page // 16
                here = (at // 16 == block)
                e, e_was = exps[pg, :, b].double(), was_exp[pg, :, b].double()
                large = ref[here].abs().amax((0, 2))
                room = slack[here].amax((0, 2))
                # the least exponent that holds the new rows, or what it was
                had = old > 16 * block
                forced = (e == e_was) & torch.tensor(had, device="cuda") | (e == -48)
                assert (large <= 448 * torch.exp2(e) + room).all()
                assert (forced | (large + room > 224 * torch.exp2(e))).all()
                assert not had or (e >= e_was).all()
                same_exp[pg, :, b] = False
                step = torch.exp2(e)[None, :, None]
                y = codes.view(torch.uint8)[pg, :, at[here] % page].view(torch.float8_e4m3fn).double().transpose(0, 1) * step
                assert ((y - ref[here]).abs() <= 2.0 ** -4 * ref[here].abs() + 2.0 ** -10 * step + slack[here] * (1 + 2.0 ** -4)).all()
                if had:  # older rows, rounded to the new exponent
                    n = slice(16 * block % page, 16 * block % page + old - 16 * block)
                    again = torch.ldexp(was[pg, :, n].float(), (e_was - e)[:, None, None]).to(torch.float8_e4m3fn)
                    assert torch.equal(codes.view(torch.uint8)[pg, :, n], again.view(torch.uint8))
                    if rotated:
                        untouched[pg, :, n] = False
            untouched[m.table[s][at // page].long(), :, at % page] = False
    for now, then in zip((m.k, m.v), before):
        assert torch.equal(now.view(torch.uint8)[untouched], then.view(torch.uint8)[untouched])
    for now, then in zip((m.k_exp, m.v_exp), before[2:]):
        assert torch.equal(now[same_exp], then[same_exp])


def test_append_step_by_step(gpu, lib):
    """Tokens one by one, each larger than the one before, then smaller ones: the block's exponent follows the largest, and what was
    rounded at a smaller exponent is rounded again; the same tokens appended again (as a draft taken back is) change nothing."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    cache = KvCache8.empty(2, 1, 16, 64)
    kv_len = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = Batch(cache, 1, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), kv_len,
                  torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), 1, 32)
    g = torch.Generator(device="cuda").manual_seed(28)
    want, e_now = torch.zeros((20, 64), dtype=torch.float64), None
    for i in range(20):
        x = (2.0 ** (3 * i if i < 8 else -2 * i) * torch.randn((1, 1, 64), generator=g, device="cuda"))
        for _ in range(2):
            kv_len.fill_(i + 1)
            cache.append(batch, None, x, -x)
        e = int(torch.ceil(torch.log2(x.double().abs().max() / 448)))
        if i % 16:
            e = max(e, e_now)
            for j in range(i // 16 * 16, i):
                want[j] = torch.ldexp(torch.ldexp(want[j].float(), torch.tensor(-e)).to(torch.float8_e4m3fn).float(), torch.tensor(e)).double()
        want[i] = torch.ldexp(torch.ldexp(x[0, 0].cpu(), torch.tensor(-e)).to(torch.float8_e4m3fn).float(), torch.tensor(e)).double()
        e_now = e
        k, v = values(torch, cache.k, cache.k_exp).cpu(), values(torch, cache.v, cache.v_exp).cpu()
        for j in range(i + 1):
            assert torch.equal(k[1 - j // 16, 0, j % 16], want[j]) and torch.equal(v[1 - j // 16, 0, j % 16], -want[j]), (i, j)


def test_append_values_at_the_borders(gpu, lib):
    """448 and just above, zeros, values too large and too small for any exponent, infinities and NaN."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    inf, nan = float("inf"), float("nan")
    blocks = [([448.0, 1.0], 0), ([448.0001, 1.0], 1), ([0.0, -0.0], -48), ([3e38, 1.0], 48), ([1e-30, -1e-20], -48),
              ([inf, 2.0], -7), ([nan, -inf], -48), ([464.0, 449.0], 1), ([1.75 * 2 ** -20, 2.0 ** -33], -28)]
    cache = KvCache8.empty(len(blocks), 1, 16, 64)
    n = len(blocks)
    batch = Batch(cache, 1, torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.ones(n, dtype=torch.int32, device="cuda"),
                  torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous(), 1, 16)
    x = torch.zeros((n, 1, 64), device="cuda")
    for i, (values_, _) in enumerate(blocks):
        x[i, 0, 5], x[i, 0, 63] = values_[0], values_[1]
    cache.append(batch, None, x, x)
    assert cache.k_exp[:, 0, 0].tolist() == [e for _, e in blocks] == cache.v_exp[:, 0, 0].tolist()
    scaled = torch.ldexp(x[:, 0], -cache.k_exp[:, 0].int())
    want = torch.where(torch.isfinite(scaled), scaled.clamp(-448, 448), torch.full_like(scaled, nan)).to(torch.float8_e4m3fn).float()
    got = cache.k[:, 0, 0].float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(1), want.nan_to_num(1))


def test_append_skips_pages_that_are_not_there(gpu, lib):
    import torch
    m = Made(torch, (4, 2, 64), 16, "float16", [(40, 5)], 29, unmapped=[(0, 1)])
    before = [t.view(torch.uint8).clone() for t in (m.k, m.v, m.k_exp, m.v_exp)]
    x, q = torch.randn((40, 2, 64), device="cuda"), torch.randn((40, 4, 64), device="cuda")
    assert torch.equal(m.cache.append(m.batch, q, x, x), q.half())
    mapped = {int(m.table[0, 0]), int(m.table[0, 2])}
    for now, was in zip((m.k, m.v, m.k_exp, m.v_exp), before):
        for p in range(m.k.shape[0]):
            same = torch.equal(now[p].view(torch.uint8), was[p])
            assert p in mapped or same
            assert p not in mapped or not same or now.dtype == torch.int8  # (an exponent may be the one that was there)


def test_append_then_attend(gpu, lib):
    """Prompts, single tokens and drafts one after the other through append, decode and prompt, as a layer uses them, with pages from
    Pages: outputs are those of what the cache holds, and that is within a block's rounding of what was appended."""
    import torch
    from lazyweights_amd import Batch, KvCache8, Pages
    heads, kv, dim, page = 8, 2, 128, 32
    cache = KvCache8.empty(40, kv, page, dim)
    pages = Pages.empty(40, page, 3, 12)
    g = torch.Generator(device="cuda").manual_seed(30)
    history = [torch.zeros((0, 2, kv, dim), dtype=torch.float64, device="cuda") for _ in range(3)]
    for step, (new, keep) in enumerate([([70, 5, 33], None), ([1, 1, 1], None), ([4, 4, 4], None), ([1, 1, 1], [73, 7, 36]),
                                        ([100, 0, 2], [0, 8, 38]), ([1, 1, 1], None)]):
        tensor = torch.tensor(new, dtype=torch.int32, device="cuda")
        kept = None if keep is None else torch.tensor(keep, dtype=torch.int32, device="cuda")
        q_start, position, slot = pages.advance(tensor, keep=kept, rows=sum(new))
        batch = Batch(cache, heads, q_start, pages.kv_len, pages.table, max(new), 384)
        q, k, v = (torch.randn((sum(new), h, dim), generator=g, device="cuda") for h in (heads, kv, kv))
        q16 = cache.append(batch, q, k, v)
        attend = cache.attend_decode if max(new) <= 16 else cache.attend_prompt
        y = attend(batch, q16, out=torch.empty_like(q))
        row, held_k, held_v = 0, values(torch, cache.k, cache.k_exp), values(torch, cache.v, cache.v_exp)
        for s, n in enumerate(new):
            if keep is not None:
                history[s] = history[s][:keep[s]]
            history[s] = torch.cat((history[s], torch.stack((k, v), 1)[row:row + n].double()))
            at = torch.arange(history[s].shape[0], device="cuda")
            pg = pages.table[s][at // page].long()
            assert position[row:row + n].tolist() == at[len(at) - n:].tolist()
            assert slot[row:row + n].tolist() == (pg * page + at % page)[len(at) - n:].tolist()
            now = torch.stack((held_k[pg, :, at % page], held_v[pg, :, at % page]), 1)
            # rounded at 2^-4, at most twice, and half a step of the block's least, 2^-10 of 2^e <= 2 max / 448
            off = (now - history[s]).abs()
            assert (off <= 2 * 2.0 ** -4 * 1.07 * history[s].abs() + 2 * 2.0 ** -10 * 2 * 6 / 448).all()
            for i in range(n):
                upto = len(at) - n + i + 1
                qq = q16[row + i].double().view(kv, heads // kv, dim)
                p = torch.softmax(torch.einsum("hgd,jhd->hgj", qq, now[:upto, 0]) * dim ** -0.5, -1)
                ref = torch.einsum("hgj,jhd->hgd", p, now[:upto, 1]).reshape(heads, dim)
                assert ((y[row + i].double() - ref).norm() / ref.norm()).item() < 1e-5, (step, s, i)
            row += n


def test_python_refusals(gpu, lib):
    import torch
    from lazyweights_amd import Batch, KvCache, KvCache8
    m = Made(torch, (8, 2, 64), 16, "float16", [(1, 20)], 31)
    k, v, ke, ve = m.k, m.v, m.k_exp, m.v_exp
    for args in ((k, v.half(), ke, ve), (k.half(), v.half(), ke, ve), (k.cpu(), v.cpu(), ke, ve), (k[0], v[0], ke, ve),
                 (k, v, ke.int(), ve), (k, v, ke[:, :1], ve), (k, v, ke.cpu(), ve.cpu()), (k[..., :48], v[..., :48], ke, ve),
                 (k[:, :, :8], v[:, :, :8], ke[..., :0], ve[..., :0]), (k, v, ke, ve, torch.float32)):
        with pytest.raises((ValueError, RuntimeError)):
            Batch(KvCache8(*args), 8, m.q_start, m.kv_len, m.table, 1, 21)
    x = torch.zeros((1, 2, 64), device="cuda")
    q = m.q
    for call in (lambda: m.cache.attend_decode(m.batch, q.float()), lambda: m.cache.attend_decode(m.batch, q[:, :4]),
                 lambda: m.cache.attend_decode(m.batch, q, out=torch.empty_like(q, dtype=torch.int16)),
                 lambda: m.cache.attend_prompt(m.batch, q.cpu()), lambda: m.cache.attend_prompt(m.batch, q, window=-1),
                 lambda: m.cache.append(m.batch, q, x, x), lambda: m.cache.append(m.batch, None, x, x[:, :1]),
                 lambda: m.cache.append(m.batch, q, x.half(), x.half(), q_out=q.float())):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    wide = KvCache(k.half(), v.half())
    other = Batch(wide, 8, m.q_start, m.kv_len, m.table, 1, 21)
    for call in (lambda: m.cache.attend_decode(other, q), lambda: wide.attend_decode(m.batch, q),
                 lambda: m.cache.attend_prompt(other, q), lambda: wide.attend_prompt(m.batch, q)):
        with pytest.raises(ValueError, match="bits"):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_rows_of_no_sequence_and_before_the_first_position(gpu, lib, call):
    """Rows behind the last sequence's are left as they were; of a sequence with more rows than its length the first ones are before
    its first position: nothing is appended for them, and they see nothing."""
    import torch
    m = Made(torch, (8, 2, 128), 16, "float16", [(3, 40), (5, 30)], 33)
    m.kv_len[1] = 2  # of the second's 5 rows, 3 come before position 0
    m.lengths = [(3, 40), (2, 0)]
    before = [t.view(torch.uint8).clone() for t in (m.k, m.v, m.k_exp, m.v_exp)]
    g = torch.Generator(device="cuda").manual_seed(34)
    x = torch.randn((11, 2, 128), generator=g, device="cuda")
    q = torch.randn((11, 8, 128), generator=g, device="cuda")
    q16 = m.cache.append(m.batch, q, x, 2 * x, q_out=torch.full((11, 8, 128), float("nan"), dtype=torch.float16, device="cuda"))
    real = torch.tensor([0, 1, 2, 6, 7], device="cuda")
    assert torch.equal(q16[real], q[real].half()) and torch.isnan(q16[3:6]).all() and torch.isnan(q16[8:]).all()
    first = int(m.table[1, 0])
    for now, was in zip((m.k, m.v), before):
        assert torch.equal(now.view(torch.uint8)[first, :, 2:], was[first, :, 2:])
    e = m.k_exp[first, :, 0].double()
    got = m.k.view(torch.uint8)[first, :, :2].view(torch.float8_e4m3fn).double() * torch.exp2(e)[:, None, None]
    want = x[6:8].transpose(0, 1).double()
    assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10 * torch.exp2(e)[:, None, None]).all()
    q16[torch.isnan(q16)] = 1
    m.q = q16[real]
    ref = reference(m)
    y = getattr(m.cache, call)(m.batch, q16, out=torch.full((11, 8, 128), float("nan"), device="cuda"))
    check(torch, y[real], ref, call == "attend_prompt")
    assert not y[3:6].any() and torch.isnan(y[8:]).all()


def test_two_batches_at_once(gpu, lib):
    """Calls of two batches over one cache that overlap on two streams, eager and as captured graphs, give each its own result."""
    import torch
    from lazyweights_amd import Batch
    m = Made(torch, (8, 2, 128), 16, "float16", [(1, 3000), (2, 4100), (1, 60)], 35)
    other = Batch(m.cache, 8, m.q_start, m.kv_len, m.table, m.max_new, m.max_kv)
    want = m.cache.attend_decode(m.batch, m.q, out=m.empty(torch.float32)).clone()
    sides = [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], [torch.empty_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for batch, out in zip((m.batch, other), outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                m.cache.attend_decode(batch, m.q, out=out)
        graphs.append(graph)
    for step in range(4):
        for out in outs:
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for side, graph, batch, out in zip(sides, graphs, (m.batch, other), outs):
            with torch.cuda.stream(side):
                if step % 2:
                    graph.replay()
                else:
                    for _ in range(20):
                        m.cache.attend_decode(batch, m.q, out=out)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want), step
