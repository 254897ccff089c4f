"""Attention over a cache in 8 bits in the forms that only larger calls take, each with all that the small calls are tested with: blocks of
8 waves of prompts, long runs of keys with fp32 outputs, decode in equal runs of all items' tiles and in two row tiles; both types of q, windows,
exponents, pages that are not there, NaN in places a row does not see and in single elements.

Bounds as in test_gpu_attention8.py, where they are not derived beside the test. That a call takes the form it is meant for is asked of the library's own
rules (decode) or follows from the sizes by the rule that the tests state (prompts)."""
import ctypes
import math
import random

import pytest
from test_gpu_attention8 import Made, check, held, reference, values

pytestmark = pytest.mark.gpu


class Plan(ctypes.Structure):
    """DecodePlan of csrc/lw_attention.h."""
    _fields_ = [("row_tiles", ctypes.c_int), ("row_blocks", ctypes.c_int), ("blocks", ctypes.c_int), ("blocks_log2", ctypes.c_int),
                ("most_keys", ctypes.c_int), ("whole", ctypes.c_bool), ("runs", ctypes.c_bool), ("spare", ctypes.c_int),
                ("waves", ctypes.c_int), ("count_bytes", ctypes.c_size_t), ("part_bytes", ctypes.c_size_t)]


def plan(lib, m):
    call = lib._ZN2lw12decode8_planEiiiiii
    call.restype, call.argtypes = Plan, [ctypes.c_int] * 6
    heads, kv = m.heads, m.k.shape[1]
    p = call(len(m.lengths), kv, heads // kv, m.k.shape[3], m.max_new, m.max_kv)
    assert p.count_bytes + p.part_bytes == m.batch.c.workspace_bytes  # (the fields are where they are taken to be)
    return p


def waves(m):
    """Waves of a prompt's blocks: 8 where blocks of 256 rows are 160 and more."""
    kv = m.k.shape[1]
    return 8 if m.q.shape[0] * (m.heads // kv) // 256 * kv >= 160 else 4


def where_nan(m, places, window):
    """Which rows see one of the places (sequence, position)."""
    rows = []
    for s, (new, old) in enumerate(m.lengths):
        for i in range(old, old + new):
            rows.append(any(t == s and j <= i and (not window or j > i - window) for t, j in places))
    return m.torch.tensor(rows, device="cuda")


def check_nan_apart(m, call, prompt, places, window, kind):
    """NaN in keys and values at the places: rows that see one are NaN, others as without."""
    torch = m.torch
    ref = reference(m, window)
    for s, j in places:
        m.put(m.k, s, j, 0x7F)
        m.put(m.v, s, j, 0xFF)
    bad = where_nan(m, places, window)
    y = call(m.batch, m.q, out=m.empty(kind), window=window)
    assert torch.isnan(y[bad]).all()
    check(torch, y[~bad], [t[~bad] for t in ref], prompt)
    assert torch.equal(call(m.batch, m.q, out=m.empty(kind), window=window)[~bad], y[~bad])


def check_nan_elements(m, call, prompt, places, kind):
    """NaN in single elements (sequence, position, head, dim) of the values."""
    torch = m.torch
    ref, group = reference(m), m.heads // m.k.shape[1]
    bad = torch.zeros(m.q.shape, dtype=torch.bool, device="cuda")
    for s, j, h, d in places:
        m.put(m.v, s, j, 0x7F, h, d)
        bad[where_nan(m, [(s, j)], 0), h * group:(h + 1) * group, d] = True
    y = call(m.batch, m.q, out=m.empty(kind))
    assert torch.equal(torch.isnan(y), bad)
    check(torch, torch.where(bad, 0, y), [torch.where(bad, 0, ref[0])] + list(ref[1:]), prompt)


def spread_exponents(m, seed):
    """The least and largest exponents of values, and the least of keys, in some blocks."""
    rng = random.Random(seed)
    for n in range(8):
        p, b = rng.randrange(m.k.shape[0]), rng.randrange(m.page // 16)
        m.v_exp[p, :, b] = rng.choice((-48, 48, -120, 127, 20))
        if n % 2:
            m.k_exp[p, :, b] = rng.choice((-48, -100, -20))


# ── prompts in blocks of 8 waves ────────────────────────────────────────────────────────────────────────────────────────────────────────────

EIGHT = [((160, 160, 64), 16, "float16", "float32"), ((160, 160, 64), 64, "bfloat16", "bfloat16"), ((160, 160, 96), 32, "bfloat16", "float32"),
         ((160, 160, 96), 16, "float16", "float16"), ((160, 80, 128), 16, "float16", "float32"), ((160, 160, 128), 16, "bfloat16", "float32"),
         ((160, 160, 128), 32, "float16", "float16")]


@pytest.mark.parametrize("case", EIGHT, ids=str)
def test_pages_that_are_not_there_8_waves(gpu, lib, case):
    import torch
    layout, page, q_type, out = case
    m = Made(torch, layout, page, q_type, [(270, 200), (3, 13), (2, 0), (40, 60)], 61,
             unmapped=[(s, j // page) for s, j in ((0, 20), (0, 70), (0, 200), (1, 0), (2, 0), (3, 20))])
    assert waves(m) == 8
    y = m.cache.attend_prompt(m.batch, m.q, out=m.empty(getattr(torch, out)))
    assert (y[273:275] == 0).all()  # nothing to see: zeros
    check(torch, y, reference(m), True)


@pytest.mark.parametrize("window", (0, 90))
@pytest.mark.parametrize("case", EIGHT, ids=str)
def test_unseen_nan_8_waves(gpu, lib, case, window):
    import torch
    layout, page, q_type, out = case
    m = Made(torch, layout, page, q_type, [(9, 100), (230, 0), (30, 300)], 62)
    assert waves(m) == 8
    check_nan_apart(m, m.cache.attend_prompt, True, [(0, 105), (1, 8 if window else 100), (1, 190), (2, 210 if window else 310), (2, 320)], window,
                    getattr(torch, out))


@pytest.mark.parametrize("case", EIGHT, ids=str)
def test_nan_in_single_elements_8_waves(gpu, lib, case):
    import torch
    layout, page, q_type, out = case
    m = Made(torch, layout, page, q_type, [(200, 70), (90, 0)], 63)
    assert waves(m) == 8
    check_nan_elements(m, m.cache.attend_prompt, True, [(0, 35, 1, 20), (0, 150, 70, 7), (1, 40, 0, 63)], getattr(torch, out))


@pytest.mark.parametrize("case", EIGHT, ids=str)
def test_exponents_far_apart_8_waves(gpu, lib, case):
    import torch
    layout, page, q_type, _ = case
    m = Made(torch, layout, page, q_type, [(200, 170), (90, 0)], 64)
    spread_exponents(m, 65)
    assert waves(m) == 8
    y = m.cache.attend_prompt(m.batch, m.q, out=m.empty(torch.float32))
    assert torch.isfinite(y).all()
    check(torch, y, reference(m), True)


# ── prompts over long runs of keys ──────────────────────────────────────────────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("q_type", ("float16", "bfloat16"))
@pytest.mark.parametrize("keys", (40000, 131000))
@pytest.mark.parametrize("dim", (64, 96, 128))
def test_prompt_sums_of_like_weights(gpu, lib, dim, keys, q_type):
    """Without a workspace a block goes through all keys of its rows; weights are alike, so that each addition to a sum loses the same.
    The scores are exact (q has one element, the first key scores 0 and every other one -1), the values positive and of blocks with
    different exponents, e = -3 to 3.

    Bound, of a positive fp32 output: its own rounding 2^-24, the weights' 2^-21, scores, the exponential and the sum of weights
    (2 2^-21 + 2^-20), the rounding of the n / 16 steps of a product's sum, four standard deviations of a random walk, 4 sqrt(n / 16)
    2^-24; and what is lost of a weight in fp16's least step, 2^-37 of the largest product of a weight and its 2^e for each of n keys, times
    the largest number, 448: n 2^-37 448 2^3 / (n / e) absolute (the row's first key has no more than e times the others' weight)."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    heads, rows, page = 4, 40, 64
    pages = -(-keys // page)
    g = torch.Generator(device="cuda").manual_seed(66)
    k = torch.zeros((pages, 1, page, dim), device="cuda")
    k[..., 0] = -1
    k[0, 0, 0, 0] = 0
    v_exp = torch.randint(-3, 4, (pages, 1, page // 16), generator=g, device="cuda").to(torch.int8)
    v = (0.5 + torch.rand((pages, 1, page, dim), generator=g, device="cuda")).to(torch.float8_e4m3fn)
    q = torch.zeros((rows, heads, dim), dtype=getattr(torch, q_type), device="cuda")
    q[..., 0] = 1
    cache = KvCache8(k.to(torch.float8_e4m3fn), v, torch.zeros_like(v_exp), v_exp)
    batch = Batch(cache, heads, torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                  torch.tensor([keys], dtype=torch.int32, device="cuda"),
                  torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous(), rows, keys)
    batch.c.workspace, batch.c.workspace_bytes = None, 0
    y = cache.attend_prompt(batch, q, out=torch.empty(q.shape, device="cuda"), scale=1.0)
    at, v64 = torch.arange(keys - rows, keys, device="cuda"), values(torch, v, v_exp).view(-1, 1, dim)
    w = math.exp(-1)
    want = (v64[:1] + w * (v64.cumsum(0)[at] - v64[:1])) / (1 + w * at.double())[:, None, None]
    bound = want * (2.0 ** -24 + 2.0 ** -21 + 2 * 2.0 ** -21 + 2.0 ** -20 + 4 * math.sqrt(keys / 16) * 2.0 ** -24) + 2.0 ** -37 * 448 * 8 * math.e
    worst = ((y.double() - want).abs() / bound).max().item()
    print("worst error / bound %.3f" % worst, flush=True)
    assert worst <= 1


@pytest.mark.parametrize("q_type", ("float16", "bfloat16"))
@pytest.mark.parametrize("layout, new, old, window", [
    ((32, 8, 128), 8200, 9000, 0), ((32, 32, 96), 8200, 9000, 0), ((32, 8, 64), 8200, 9000, 0),  # blocks of 8 waves
    ((32, 8, 128), 900, 20000, 0), ((8, 2, 96), 900, 20000, 0), ((7, 1, 64), 2000, 18000, 0),  # of 4
    ((32, 8, 128), 8200, 12000, 17000), ((8, 2, 96), 900, 20000, 17001)], ids=str)
def test_long_runs(gpu, lib, layout, new, old, window, q_type):
    """More than 16384 keys in a block's run and fp32 outputs, exponents that differ from block to block, the last key's value NaN: some rows
    against 64 bits, and the last, which alone sees that."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    heads, kv, dim = layout
    page, keys = 64, new + old
    pages, group = -(-keys // page), heads // kv
    assert min(keys, window or keys) > 16384
    g = torch.Generator(device="cuda").manual_seed(67)
    k, v = (torch.randn((pages, kv, page, dim), generator=g, device="cuda") for _ in range(2))
    power = torch.exp2(torch.randint(-4, 5, (pages, kv, page // 16, 1, 1), generator=g, device="cuda").float())
    (k, k_exp), (v, v_exp) = held(torch, k, 2), held(torch, ((v + 0.25).unflatten(2, (-1, 16)) * power).flatten(2, 3), 1)
    q = (1.5 * torch.randn((new, heads, dim), generator=g, device="cuda")).to(getattr(torch, q_type))
    v.view(torch.uint8)[-1, :, (keys - 1) % page] = 0x7F
    cache = KvCache8(k, v, k_exp, v_exp)
    batch = Batch(cache, heads, torch.tensor([0, new], dtype=torch.int32, device="cuda"),
                  torch.tensor([keys], dtype=torch.int32, device="cuda"),
                  torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous(), new, keys)
    batch.c.workspace, batch.c.workspace_bytes = None, 0
    y = cache.attend_prompt(batch, q, out=torch.full(q.shape, float("nan"), device="cuda"), window=window)
    assert torch.isnan(y[-1]).all() and torch.isfinite(y[:-1]).all()
    kk, vv = (values(torch, *t).transpose(1, 2).reshape(-1, kv, dim) for t in ((k, k_exp), (v, v_exp)))
    powers = torch.exp2(v_exp.double()).transpose(1, 2).reshape(-1, kv).repeat_interleave(16, 0)
    worst = 0.0
    for row in [0, 1, 31, 32, 255, 256, new // 2, new - 300, new - 33, new - 2]:
        see = slice(max(0, old + row + 1 - window) if window else 0, old + row + 1)
        n = see.stop - see.start
        for h in range(kv):
            qq, x, z = q[row, h * group:(h + 1) * group].double(), kk[see, h].contiguous(), vv[see, h].contiguous()
            p = torch.softmax(qq @ x.T.contiguous() * dim ** -0.5, -1)
            want, a = p @ z, p @ z.abs()
            most = (qq.abs() @ x.abs().T.contiguous() * dim ** -0.5).amax(-1, keepdim=True)
            top = 448 * (p * powers[see, h]).amax(-1, keepdim=True)
            bound = 2.0 ** -24 * want.abs() + a * (2.0 ** -21 + 2 * 2.0 ** -21 * most + 2.0 ** -20) + n * top * 2.0 ** -37
            err = (y[row, h * group:(h + 1) * group].double() - want).abs()
            worst = max(worst, (err / bound).max().item())
    print("worst error / bound %.3f" % worst, flush=True)
    assert worst <= 1


# ── decode in equal runs, and in two row tiles ──────────────────────────────────────────────────────────────────────────────────────────────

def batch_lengths(seqs, longest, most, seed):
    rng = random.Random(seed)
    lengths = [(rng.randrange(0 if seqs > 60 else 1, most + 1), rng.choice((0, 1, 31, 32, 33, longest - 5, rng.randrange(longest))))
               for _ in range(seqs)]
    return [(n, max(0, min(o, longest - n))) for n, o in lengths]


BATCHES = [
    # layout, sequences, longest, bound on the length, new tokens, type of q, out, window
    ((16, 8, 128), 33, 5000, 5000, 1, "bfloat16", "bfloat16", 0),
    ((16, 8, 128), 33, 5000, 5000, 1, "float16", "float16", 700),
    ((8, 4, 128), 70, 900, 6000, 2, "bfloat16", "float32", 33),
    ((32, 8, 128), 20, 3100, 3200, 3, "float16", "float32", 1),
    ((32, 8, 128), 9, 3900, 17000, 1, "bfloat16", "float32", 1000),
    ((8, 8, 128), 130, 120, 9000, 1, "bfloat16", "float32", 0),
    # two row tiles
    ((32, 4, 128), 130, 300, 600, 3, "bfloat16", "float32", 0),
    ((32, 4, 128), 130, 300, 900, 3, "bfloat16", "bfloat16", 100),
    ((24, 4, 64), 300, 60, 2000, 5, "bfloat16", "float16", 20),
    ((20, 2, 96), 70, 700, 9000, 4, "bfloat16", "float32", 0),
    ((20, 2, 96), 70, 700, 9000, 4, "float16", "float32", 333),
]


def form(p):
    return "two" if p.row_tiles == 2 else "runs" if p.runs else "other"


@pytest.mark.parametrize("case", BATCHES, ids=str)
def test_decode_batches(gpu, lib, case):
    import torch
    layout, seqs, longest, bound, most, q_type, out, window = case
    m = Made(torch, layout, 16, q_type, batch_lengths(seqs, longest, most, seqs), 71, most, bound, width=-(-bound // 16))
    assert form(plan(lib, m)) == ("two" if layout[0] // layout[1] * most > 16 else "runs")
    ref = reference(m, window)
    first = None
    for _ in range(2):
        y = m.cache.attend_decode(m.batch, m.q, out=m.empty(getattr(torch, out)), window=window)
        check(torch, y, ref, False)
        first = y if first is None else first
        assert torch.equal(y, first)


# (short sequences under a long bound: a run's block has several items, of one wave's tile each, one gone over again beside others)
MIXED = [((16, 8, 128), "float16", 1, 5000), ((8, 8, 128), "bfloat16", 2, 9000), ((32, 4, 128), "bfloat16", 4, 1000),
         ((12, 4, 64), "float16", 8, 2000), ((12, 4, 96), "bfloat16", 8, 2000)]


def mixed(torch, lib, case, **kw):
    layout, q_type, most, bound = case
    lengths = [(1 + i % most, (37 * i) % 131) for i in range(70)] + [(1, 850), (most, 0)]
    m = Made(torch, layout, 16, q_type, lengths, 72, most, bound, width=-(-bound // 16), **kw)
    assert form(plan(lib, m)) == ("two" if layout[0] // layout[1] * most > 16 else "runs")
    return m


@pytest.mark.parametrize("window", (0, 50))
@pytest.mark.parametrize("case", MIXED, ids=str)
def test_unseen_nan_decode(gpu, lib, case, window):
    import torch
    m = mixed(torch, lib, case)
    places = []
    for s in range(0, 72, 3):  # the last position, which only a sequence's last row sees, or one before every window
        new, old = m.lengths[s]
        if s % 2 or new + old < 60:
            places.append((s, new + old - 1))
        elif window:
            places.append((s, old - window - 1 if old > window + 1 else 0))
    check_nan_apart(m, m.cache.attend_decode, False, places, window, torch.float32)


@pytest.mark.parametrize("case", MIXED, ids=str)
def test_nan_in_single_elements_decode(gpu, lib, case):
    import torch
    m = mixed(torch, lib, case)
    places = [(s, (m.lengths[s][0] + m.lengths[s][1] - 1) // (1 + s % 2), s % 4, 5 * s % 64) for s in range(0, 72, 5)]
    check_nan_elements(m, m.cache.attend_decode, False, places, torch.float32)


@pytest.mark.parametrize("case", MIXED, ids=str)
def test_pages_that_are_not_there_decode(gpu, lib, case):
    import torch
    unmapped = [(s, j) for s in range(0, 71, 2) for j in range((37 * s % 131) // 16 + 1) if (s + j) % 3 == 0] + [(70, 20), (70, 53), (71, 0)]
    m = mixed(torch, lib, case, unmapped=unmapped)
    check(torch, m.cache.attend_decode(m.batch, m.q, out=m.empty(torch.float32)), reference(m), False)


@pytest.mark.parametrize("case", MIXED, ids=str)
def test_exponents_far_apart_decode(gpu, lib, case):
    import torch
    m = mixed(torch, lib, case)
    for seed in range(12):
        spread_exponents(m, seed)
    y = m.cache.attend_decode(m.batch, m.q, out=m.empty(torch.float32))
    assert torch.isfinite(y).all()
    check(torch, y, reference(m), False)
