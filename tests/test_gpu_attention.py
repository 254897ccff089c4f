"""Attention over a paged cache (lw_kv_append, lw_attn_decode, lw_attn_prompt) against plain forms in 64 bits: head layouts,
types, lengths from none on, page sizes, windows, pages that are not there, values that are not finite in places a row does
not see, layouts, long caches, streams and captured calls.

Bounds, elementwise, from the types and the kernels' arithmetic (A = sum p |v| / sum p of the row, n its keys):
  the output's rounding          u |out|, u = 2^-24, 2^-11, 2^-8 for fp32, fp16, bf16
  the weights' rounding          u_p A: 2^-11 or 2^-8 where they are one 16-bit part (prompt, 16-bit out), else 2^-21
  small fp16 weights             n 2^-25 max |v| (subnormal below 2^-14 of the row's largest)
  scores, sums, the exponential  A (2 2^-21 max_j scale sum |q k_j| + 2^-20): products exact, a score's sum in a few steps
"""
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def unit(dtype):
    return U[str(dtype).split(".")[1]]


def make(torch, layout, page, dtype, lengths, seed, unmapped=(), width=None, layout_rows_first=False):
    """Cache pages (NaN wherever nothing was written), table, q_start, kv_len, q for (new, old) per sequence."""
    heads, kv, dim = layout
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-(n + o) // page) for n, o in lengths]
    width = max([1] + need) + 1 if width is None else width
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((len(lengths), width), -7, dtype=torch.int32)  # entries past a sequence's pages: anything
    table[:, 1::2] = 1 << 30
    at = 0
    shape = (pages, page, kv, dim) if layout_rows_first else (pages, kv, page, dim)
    k, v = (torch.full(shape, float("nan"), dtype=dtype, device="cuda") for _ in range(2))
    if layout_rows_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    for s, (n, o) in enumerate(lengths):
        table[s, :need[s]] = order[at:at + need[s]]
        at += need[s]
        pos = torch.arange(n + o)
        pg, off = table[s][pos // page].long().cuda(), (pos % page).cuda()
        k[pg, :, off] = torch.randn((n + o, kv, dim), generator=g, device="cuda").to(dtype)
        v[pg, :, off] = (torch.randn((n + o, kv, dim), generator=g, device="cuda") + 0.25).to(dtype)
    for s, p in unmapped:
        table[s, p] = pages + 5 if p % 2 else -1
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    q = (1.5 * torch.randn((starts[-1], heads, dim), generator=g, device="cuda")).to(dtype)
    return (k, v, table.cuda(), torch.tensor(starts, dtype=torch.int32, device="cuda"),
            torch.tensor([n + o for n, o in lengths], dtype=torch.int32, device="cuda"), q)


def reference(torch, k, v, table, lengths, q, window, scale):
    """(out, bound terms A, S = max scale sum |q k|, n, max |v|) per row and head, in 64 bits over the seen keys only."""
    pages, kv, page, dim = k.shape
    heads = q.shape[1]
    group = heads // kv
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    a, most = torch.zeros_like(out), torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device="cuda")
    n_keys, v_max = torch.zeros_like(most), torch.zeros_like(most)
    row = 0
    tab = table.cpu()
    for s, (new, old) in enumerate(lengths):
        for i in range(old, old + new):
            j = torch.arange(max(0, i - window + 1) if window else 0, i + 1)
            pg = tab[s][j // page].long()
            ok = (pg >= 0) & (pg < pages)
            j, pg = j[ok], pg[ok].cuda()
            if len(j):
                off = (j % page).cuda()
                kk, vv = k[pg, :, off].double(), v[pg, :, off].double()  # [keys, kv, dim]
                qq = q[row].double().view(kv, group, dim)
                sc = torch.einsum("hgd,jhd->hgj", qq, kk) * scale
                p = torch.softmax(sc, -1)
                out[row] = torch.einsum("hgj,jhd->hgd", p, vv).reshape(heads, dim)
                a[row] = torch.einsum("hgj,jhd->hgd", p, vv.abs()).reshape(heads, dim)
                most[row] = (torch.einsum("hgd,jhd->hgj", qq.abs(), kk.abs()) * abs(scale)).amax(-1).reshape(heads, 1)
                n_keys[row], v_max[row] = len(j), vv.abs().max()
            row += 1
    return out, a, most, n_keys, v_max


def check(torch, y, ref, dtype, prompt):
    out, a, most, n, v_max = ref
    one_part = prompt and y.dtype != torch.float32
    bound = unit(y.dtype) * out.abs() + a * ((unit(dtype) if one_part else 2.0 ** -21) + 2 * 2.0 ** -21 * most + 2.0 ** -20)
    if one_part and dtype == torch.float16:
        bound = bound + n * 2.0 ** -25 * v_max
    err = (y.double() - out).abs()
    worst = (err / (bound + 1e-30)).max().item() if err.numel() else 0.0
    print("worst error / bound %.3f" % worst, flush=True)
    assert (err <= bound).all(), worst


def build(torch, layout, k, v, table, q_start, kv_len, max_new, max_kv):
    from lazyweights_amd import Batch, KvCache
    cache = KvCache(k, v)
    return cache, Batch(cache, layout[0], q_start, kv_len, table, max_new, max_kv)


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 500, 1025]

DECODE = [
    # layout (heads, kv heads, dim), page, type, out, new per sequence, window
    ((8, 8, 64), 16, "float16", "float16", [1], 0),
    ((8, 2, 128), 16, "float16", "float32", [1], 0),
    ((7, 1, 96), 8, "bfloat16", "bfloat16", [1, 0, 1], 0),
    ((8, 1, 128), 64, "bfloat16", "float32", [5, 1, 0, 3], 0),
    ((32, 2, 64), 1, "float16", "float32", [1, 2], 0),
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
    layout, page, dtype, out, news, window = case
    dtype, out = getattr(torch, dtype), getattr(torch, out)
    lengths = [(news[i % len(news)], n) for i, n in enumerate(LENGTHS)]
    k, v, table, q_start, kv_len, q = make(torch, layout, page, dtype, lengths, 11)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, max(news), 1025 + max(news))
    y = torch.full(q.shape, float("nan"), dtype=out, device="cuda")
    for _ in range(3):  # the later calls find the workspace as the first left it
        y.fill_(float("nan"))
        assert cache.attend_decode(batch, q, out=y, window=window) is y
    check(torch, y, reference(torch, k, v, table, lengths, q, window, layout[2] ** -0.5), dtype, False)


def test_decode_bounds_larger_than_the_lengths(gpu, lib):
    """max_kv and max_new far above what the arrays hold, and lengths above max_kv, give the same values."""
    import torch
    layout, lengths = (8, 2, 128), [(1, 40), (1, 3000), (1, 700)]
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 12, width=1000)
    ref = reference(torch, k, v, table, lengths, q, 0, 128 ** -0.5)
    for max_new, max_kv in ((1, 3001), (16, 16000), (1, 100), (3, 1)):
        cache, batch = build(torch, layout, k, v, table, q_start, kv_len, max_new, max_kv)
        check(torch, cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32)), ref, torch.float16, False)


PROMPT = [
    ((8, 8, 64), 16, "float16", "float16", [(1, 0), (2, 0), (33, 0), (0, 0), (64, 0), (129, 0)], 0),
    ((8, 2, 128), 16, "float16", "float32", [(31, 0), (32, 0), (200, 0), (1, 0)], 0),
    ((7, 1, 96), 8, "bfloat16", "bfloat16", [(300, 0), (1, 64), (17, 0)], 0),
    ((4, 2, 128), 64, "bfloat16", "float32", [(65, 190), (127, 1), (3, 700)], 0),
    ((6, 2, 96), 1, "float16", "float32", [(90, 30), (5, 5)], 0),
    ((4, 1, 64), 32, "float16", "bfloat16", [(257, 0), (100, 333)], 0),
    ((8, 2, 128), 16, "float16", "float32", [(250, 0), (70, 100), (1, 9)], 1),
    ((8, 2, 128), 256, "bfloat16", "float32", [(250, 0), (70, 100)], 65),
    ((4, 4, 96), 16, "float16", "float16", [(400, 20), (300, 0)], 100),
    ((3, 3, 64), 16, "bfloat16", "float32", [(0, 50), (513, 0)], 0),
]


@pytest.mark.parametrize("case", PROMPT, ids=str)
def test_prompt(gpu, lib, case):
    import torch
    layout, page, dtype, out, lengths, window = case
    dtype, out = getattr(torch, dtype), getattr(torch, out)
    k, v, table, q_start, kv_len, q = make(torch, layout, page, dtype, lengths, 13)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, max(n for n, _ in lengths),
                         max(n + o for n, o in lengths))
    y = torch.full(q.shape, float("nan"), dtype=out, device="cuda")
    cache.attend_prompt(batch, q, out=y, window=window)
    check(torch, y, reference(torch, k, v, table, lengths, q, window, layout[2] ** -0.5), dtype, True)


def test_many_sequences(gpu, lib):
    """More sequences than lanes, empty ones among them: rows find theirs."""
    import torch
    layout = (2, 1, 64)
    lengths = [((i * 7) % 5 % 3, (i * 11) % 40) for i in range(301)]
    k, v, table, q_start, kv_len, q = make(torch, layout, 8, torch.float16, lengths, 14)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 2, 42)
    ref = reference(torch, k, v, table, lengths, q, 0, 64 ** -0.5)
    for call, prompt in ((cache.attend_decode, False), (cache.attend_prompt, True)):
        check(torch, call(batch, q, out=torch.empty_like(q, dtype=torch.float32)), ref, torch.float16, prompt)


@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_pages_that_are_not_there(gpu, lib, call):
    import torch
    layout, lengths = (4, 2, 96), [(5, 200), (3, 13), (2, 0), (4, 60)]
    unmapped = [(0, 1), (0, 4), (0, 12), (1, 0), (2, 0), (3, 3)]
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 15, unmapped=unmapped)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 5, 205)
    y = getattr(cache, call)(batch, q, out=torch.full(q.shape, float("nan"), device="cuda"))
    assert (y[8:10] == 0).all()  # nothing to see: zeros
    check(torch, y, reference(torch, k, v, table, lengths, q, 0, 96 ** -0.5), torch.float16, call == "attend_prompt")


@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf"), 65504.0))
@pytest.mark.parametrize("dim", (64, 96, 128))
@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_what_a_row_does_not_see_never_reaches_it(gpu, lib, call, dim, bad):
    """Keys and values that are not finite at positions after a row's, or before its window, change none of its bits."""
    import torch
    layout, lengths, window = (4, 2, dim), [(9, 100), (16, 0), (7, 300)], 90
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 16)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 16, 307)
    ref = reference(torch, k, v, table, lengths, q, window, dim ** -0.5)

    def put(s, pos, where):
        where[int(table[s, pos // 16]), :, pos % 16] = bad

    for where in (k, v):
        put(0, 105, where)   # rows 0..4 of sequence 0 do not see it
        put(1, 8, where)     # rows 0..7 of sequence 1
        put(1, 15, where)
        put(2, 210, where)   # before every window of sequence 2 (first row: 211 .. 300)
        put(2, 304, where)
    y = getattr(cache, call)(batch, q, out=torch.empty_like(q, dtype=torch.float32), window=window)
    clean = [0, 1, 2, 3, 4] + [9 + i for i in range(8)] + [25 + i for i in range(4)]
    check(torch, y[clean], [t[clean] for t in ref], torch.float16, call == "attend_prompt")
    if bad != bad:
        assert torch.isnan(y[5:9]).all() and torch.isnan(y[24]).all() and torch.isnan(y[29:]).all()


@pytest.mark.parametrize("call", ("attend_decode", "attend_prompt"))
def test_infinite_values_that_are_seen(gpu, lib, call):
    """An infinite value that a row sees is infinite in its output, in that element only."""
    import torch
    layout, lengths = (4, 2, 64), [(6, 70)]
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 17)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 6, 76)
    ref = reference(torch, k, v, table, lengths, q, 0, 0.125)
    v[int(table[0, 2]), 1, 3, 20] = float("inf")
    v[int(table[0, 73 // 16]), 0, 73 % 16, 7] = -float("inf")
    y = getattr(cache, call)(batch, q, out=torch.empty_like(q, dtype=torch.float32))
    assert (y[:, 2:, 20] == float("inf")).all() and (y[3:, :2, 7] == -float("inf")).all()
    there = torch.isfinite(y)
    assert int((~there).sum()) == 6 * 2 + 3 * 2
    check(torch, torch.where(there, y, 0), [torch.where(there, ref[0], 0)] + list(ref[1:]), torch.float16,
          call == "attend_prompt")


def test_scores_far_apart(gpu, lib):
    """Scores of hundreds, first rising and then falling: no weight overflows and the largest wins."""
    import torch
    layout, lengths = (2, 1, 64), [(1, 500), (1, 500)]
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 18)
    q.fill_(1.0)
    for s, sign in ((0, 1.0), (1, -1.0)):
        for p in range(501):
            k[int(table[s, p // 16]), :, p % 16] = sign * (p - 250) / 8
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 1, 501)
    ref = reference(torch, k, v, table, lengths, q, 0, 0.125)
    for call, prompt in ((cache.attend_decode, False), (cache.attend_prompt, True)):
        check(torch, call(batch, q, out=torch.empty_like(q, dtype=torch.float32)), ref, torch.float16, prompt)
    for scale in (0.0, -0.05):  # all weights alike; the smallest product wins
        ref = reference(torch, k, v, table, lengths, q, 0, scale)
        for call, prompt in ((cache.attend_decode, False), (cache.attend_prompt, True)):
            check(torch, call(batch, q, out=torch.empty_like(q, dtype=torch.float32), scale=scale), ref, torch.float16, prompt)


def test_layouts_and_strides(gpu, lib):
    """A cache with rows before heads, q and out as parts of wider rows: the same bits."""
    import torch
    layout, lengths = (8, 2, 96), [(3, 77), (4, 130)]
    ys = []
    for rows_first in (False, True):
        k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.bfloat16, lengths, 19, layout_rows_first=rows_first)
        cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 4, 134)
        wide = torch.full((7, 3 * 8 * 96), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, 768:1536] = q.view(7, -1)
        for call in (cache.attend_decode, cache.attend_prompt):
            out = torch.full((7, 2 * 768), float("nan"), device="cuda")
            call(batch, wide[:, 768:1536], out=out[:, 768:])
            assert torch.isnan(out[:, :768]).all()
            ys.append(out[:, 768:].clone())
            ys.append(call(batch, q, out=torch.empty_like(q, dtype=torch.float32)).view(7, -1))
    assert torch.equal(ys[0], ys[1]) and torch.equal(ys[0], ys[4]) and torch.equal(ys[0], ys[5])
    assert torch.equal(ys[2], ys[3]) and torch.equal(ys[2], ys[6]) and torch.equal(ys[2], ys[7])


def test_offsets_past_32_bits(gpu, lib):
    """Pages 5 GB and more into the cache, in elements past 2^31 and in bytes past 2^32."""
    import torch
    layout, page, far = (4, 2, 64), 64, 3 << 30  # elements from the first page to the third
    k0, v0, table, q_start, kv_len, q = make(torch, layout, page, torch.float16, [(2, 100)], 20)
    small = build(torch, layout, k0, v0, table, q_start, kv_len, 2, 102)
    stride = far // 2
    big = [torch.empty(3 * stride + 2 * page * 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    k, v = (b.as_strided((4, 2, page, 64), (stride, page * 64, 64, 1)) for b in big)
    k.copy_(k0)
    v.copy_(v0)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 2, 102)
    for call in ("attend_decode", "attend_prompt"):
        assert torch.equal(getattr(cache, call)(batch, q), getattr(small[0], call)(small[1], q))
    x = torch.randn((2, 2, 64), device="cuda")
    cache.append(batch, None, x, 2 * x)
    small[0].append(small[1], None, x, 2 * x)
    pg, pos = table[0, 1].long(), torch.tensor([100 % 64, 101 % 64])
    for a, b in ((k, k0), (v, v0)):
        assert torch.equal(a[pg, :, pos], b[pg, :, pos]) and not torch.isnan(a[pg, :, pos]).any()


def test_long_cache_same_bits_every_call(gpu, lib):
    import torch
    layout, lengths = (8, 1, 128), [(1, 70000), (2, 9)]
    g = torch.Generator(device="cuda").manual_seed(21)
    pages = 70001 // 128 + 3
    k, v = (torch.randn((pages, 1, 128, 128), generator=g, device="cuda").half() for _ in range(2))
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.stack((table, table.flip(0))).contiguous()
    q_start = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    kv_len = torch.tensor([70001, 11], dtype=torch.int32, device="cuda")
    q = torch.randn((3, 8, 128), generator=g, device="cuda").half()
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 2, 70001)
    first = cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32))
    for _ in range(20):
        assert torch.equal(cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32)), first)
    kk, vv = (t[table[0].long(), 0].reshape(-1, 128)[:70001].double() for t in (k, v))
    ref = torch.softmax(q[0].double() @ kk.T.contiguous() * 128 ** -0.5, -1) @ vv
    assert ((first[0].double() - ref).norm() / ref.norm()).item() < 1e-5


def test_streams_and_captured_calls(gpu, lib):
    """On another stream, and captured: replays read the lengths, pages and rows of their time."""
    import torch
    layout, page = (8, 2, 128), 16
    lengths = [(1, 300), (1, 20)]
    k, v, table, q_start, kv_len, q = make(torch, layout, page, torch.float16, lengths, 22, width=40)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 1, 600)
    x, kx, vx = (torch.randn((2, h, 128), device="cuda") for h in (8, 2, 2))
    turn = torch.arange(600, device="cuda")[:, None] * 0.01 ** (torch.arange(64, device="cuda") / 64)
    cos, sin = turn.cos().contiguous(), turn.sin().contiguous()
    q16, y = torch.empty_like(x, dtype=torch.float16), torch.empty_like(x)

    def step():
        cache.append(batch, x, kx, vx, cos, sin, q_out=q16)
        cache.attend_decode(batch, q16, out=y)
        cache.attend_prompt(batch, q16, out=z)

    z = torch.empty_like(x)
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
    free = [p for p in range(k.shape[0]) if p not in set(table.flatten().tolist())]
    for grow in range(3):
        kv_len += 1 + grow
        for t in (x, kx, vx):
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        got = (q16.clone(), y.clone(), z.clone(), k.clone(), v.clone())
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int16), b.view(torch.int16))
                   for a, b in zip(got, (q16, y, z, k, v))), (grow, free)


# ── append ──────────────────────────────────────────────────────────────────────────────────────────────────────────

APPEND = [
    # layout, page, cache type, x type, rot, neighbours, (new, old) per sequence
    ((8, 2, 128), 16, "float16", "float32", 128, False, [(1, 0)]),
    ((8, 8, 64), 16, "bfloat16", "float32", 64, False, [(1, 5), (1, 31), (1, 32)]),
    ((7, 1, 96), 8, "float16", "float16", 96, True, [(5, 0), (0, 3), (13, 4), (1, 70)]),
    ((4, 2, 128), 64, "bfloat16", "bfloat16", 64, False, [(100, 3), (1, 0)]),
    ((4, 4, 64), 1, "float16", "bfloat16", 32, True, [(17, 2), (3, 9)]),
    ((6, 3, 96), 128, "bfloat16", "float16", 8, False, [(33, 100)]),
    ((4, 2, 128), 16, "float16", "float32", 0, False, [(40, 1), (0, 0), (2, 2)]),
]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(gpu, lib, case):
    import torch
    layout, page, dtype, x_type, rot, neighbours, lengths = case
    heads, kv, dim = layout
    dtype, x_type = getattr(torch, dtype), getattr(torch, x_type)
    k, v, table, q_start, kv_len, _ = make(torch, layout, page, dtype, lengths, 23)
    most = max(n + o for n, o in lengths)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, max(n for n, _ in lengths), most)
    rows = int(q_start[-1])
    # one joined projection with a row that belongs to no sequence
    joined = torch.randn((rows + 1, (heads + 2 * kv) * dim), device="cuda").to(x_type)
    q, kx, vx = joined.split((heads * dim, kv * dim, kv * dim), 1)
    turn = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(max(rot // 2, 1), dtype=torch.float64, device="cuda") / max(rot // 2, 1))
    cos, sin = turn.cos().float(), turn.sin().float()
    before = (k.clone(), v.clone())
    out = torch.full((rows + 1, heads, dim), float("nan"), dtype=dtype, device="cuda")
    got = cache.append(batch, q, kx, vx, *((cos, sin) if rot else (None, None)), q_out=out, neighbours=neighbours)
    assert got is out and torch.isnan(out[rows:]).all()
    written = torch.zeros(k.shape[0], page, dtype=torch.bool)
    row = 0
    for s, (new, old) in enumerate(lengths):
        for i in range(old, old + new):
            pg, off = int(table[s, i // page]), i % page
            written[pg, off] = True
            c, n = cos[i].double(), sin[i].double()

            def turned(x):
                x = x.double().clone()
                if rot:
                    a, b = ((slice(0, rot, 2), slice(1, rot, 2)) if neighbours
                            else (slice(0, rot // 2), slice(rot // 2, rot)))
                    p, r = x[..., a].clone(), x[..., b].clone()
                    x[..., a], x[..., b] = p * c - r * n, r * c + p * n
                return x

            # the result's rounding, and that of three fp32 operations on values up to the pair's
            for y, x, h in ((out[row], q[row], heads), (k[pg, :, off], kx[row], kv)):
                ref = turned(x.view(h, dim))
                size = x.view(h, dim).double().abs().amax(-1, keepdim=True)
                assert ((y.double() - ref).abs() <= unit(dtype) * ref.abs() + 2.0 ** -22 * size + 2.0 ** -25).all()
            assert torch.equal(v[pg, :, off], vx[row].view(kv, dim).to(dtype))
            row += 1
    for now, was in ((k, before[0]), (v, before[1])):  # nothing else was touched
        keep = ~written.cuda()[:, None, :].expand(-1, kv, -1)
        assert torch.equal(now[keep].view(torch.int16), was[keep].view(torch.int16))


def test_append_skips_pages_that_are_not_there(gpu, lib):
    import torch
    layout, lengths = (4, 2, 64), [(40, 5)]
    k, v, table, q_start, kv_len, _ = make(torch, layout, 16, torch.float16, lengths, 24, unmapped=[(0, 1)])
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 40, 45)
    before = (k.clone(), v.clone())
    x = torch.randn((40, 2, 64), device="cuda")
    q = torch.randn((40, 4, 64), device="cuda")
    assert torch.equal(cache.append(batch, q, x, x), q.half())
    for p in range(3):
        for now, was in ((k, before[0]), (v, before[1])):
            for i in range(max(5, 16 * p), min(45, 16 * p + 16)):
                if p != 1:
                    assert torch.equal(now[int(table[0, p]), :, i % 16], x[i - 5].half())
            if p == 2:
                assert torch.equal(now[int(table[0, p]), :, 45 % 16:].view(torch.int16),
                                   was[int(table[0, p]), :, 45 % 16:].view(torch.int16))
    mapped = {int(table[0, 0]), int(table[0, 2])}
    for p in range(k.shape[0]):
        if p not in mapped:
            assert torch.equal(k[p].view(torch.int16), before[0][p].view(torch.int16))


def test_append_non_finite_and_large_values(gpu, lib):
    """Values past the type's range become infinite, NaN stay NaN, neighbours unharmed; many tokens across pages."""
    import torch
    layout = (2, 2, 64)
    k, v, table, q_start, kv_len, _ = make(torch, layout, 16, torch.float16, [(3, 0)], 25)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 3, 3)
    x = torch.ones((3, 2, 64), device="cuda")
    x[0, 0, 5], x[1, 1, 7], x[2, 0, 9] = 1e6, float("nan"), -float("inf")
    q = cache.append(batch, x, x, x)
    assert q[0, 0, 5] == float("inf") and torch.isnan(q[1, 1, 7]) and q[2, 0, 9] == -float("inf")
    assert int((q == 1).sum()) == 3 * 128 - 3
    assert torch.equal(v[int(table[0, 0]), :, 0], q[0])


def test_python_refusals(gpu, lib):
    import torch
    from lazyweights_amd import Batch, KvCache
    k, v, table, q_start, kv_len, q = make(torch, (8, 2, 64), 16, torch.float16, [(1, 20)], 26)
    cache, batch = build(torch, (8, 2, 64), k, v, table, q_start, kv_len, 1, 21)
    for args in ((k, v.bfloat16()), (k.float(), v.float()), (k[..., :48], v[..., :48]), (k.cpu(), v.cpu()), (k[0], v[0]),
                 (k, v.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises((ValueError, RuntimeError)):
            Batch(KvCache(*args), 8, q_start, kv_len, table, 1, 21)
    for args in ((8, q_start.long(), kv_len, table), (8, q_start[:1], kv_len, table), (8, q_start, kv_len, table[0]),
                 (7, q_start, kv_len, table), (8, q_start, kv_len.cpu(), table)):
        with pytest.raises(ValueError):
            Batch(cache, *args, 1, 21)
    with pytest.raises(ValueError):
        Batch(cache, 8, q_start, kv_len, table, 1, 16 * table.shape[1] + 1)
    x = torch.zeros((1, 2, 64), device="cuda")
    for call in (lambda: cache.attend_decode(batch, q.float()), lambda: cache.attend_decode(batch, q[:, :4]),
                 lambda: cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.int16)),
                 lambda: cache.attend_prompt(batch, q.cpu()), lambda: cache.attend_prompt(batch, q, window=-1),
                 lambda: cache.attend_decode(batch, q, scale=float("nan")),
                 lambda: cache.append(batch, q, x, x), lambda: cache.append(batch, None, x, x[:, :1]),
                 lambda: cache.append(batch, None, x, x, torch.zeros(5, 32, device="cuda"), torch.zeros(5, 32, device="cuda")),
                 lambda: cache.append(batch, None, x, x, torch.zeros(21, 31, device="cuda"), torch.zeros(21, 31, device="cuda")),
                 lambda: cache.append(batch, None, x, x, torch.zeros(21, 32, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    many = Batch(cache, 8, q_start, kv_len, table, 17, 21)
    with pytest.raises(RuntimeError, match="attn_prompt"):
        cache.attend_decode(many, q)
    cache.attend_prompt(many, q)
    torch.cuda.synchronize()


MANY = [
    # dim, page, type, out, window: 512 rows of 512 heads, enough blocks for the form with 8 waves
    (64, 16, "float16", "float16", 0),
    (96, 8, "bfloat16", "float32", 0),
    (128, 64, "float16", "float32", 70),
    (128, 16, "bfloat16", "bfloat16", 0),
    (64, 32, "bfloat16", "float32", 33),
    (96, 16, "float16", "float16", 200),
]


@pytest.mark.parametrize("case", MANY, ids=str)
def test_prompt_of_many_rows(gpu, lib, case):
    """Rows that see 1 to 6 key tiles in blocks of 256, a hidden NaN among the values, a part of the rows of a block."""
    import torch
    dim, page, dtype, out, window = case
    dtype, out = getattr(torch, dtype), getattr(torch, out)
    layout, lengths = (512, 512, dim), [(300, 0), (0, 5), (150, 200), (1, 0), (61, 64)]
    k, v, table, q_start, kv_len, q = make(torch, layout, page, dtype, lengths, 27)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 300, 350)
    ref = reference(torch, k, v, table, lengths, q, window, dim ** -0.5)
    y = cache.attend_prompt(batch, q, out=torch.full(q.shape, float("nan"), dtype=out, device="cuda"), window=window)
    check(torch, y, ref, dtype, True)
    v[int(table[0, 250 // page]), :, 250 % page] = float("nan")  # rows 250 .. 299 of the first sequence see it
    y = cache.attend_prompt(batch, q, out=torch.empty_like(q, dtype=out), window=window)
    seen = torch.zeros(512, dtype=torch.bool, device="cuda")
    seen[250:min(300, 250 + window) if window else 300] = True
    assert torch.isnan(y[seen]).all()
    check(torch, y[~seen], [t[~seen] for t in ref], dtype, True)


BATCHES = [
    # layout, sequences, longest, bound on the length, new tokens: forms of the launch by items (sequences x kv heads), bound
    ((2, 1, 64), 301, 40, 5000, 2),    # 301 items, runs over more sequences than lanes
    ((8, 8, 96), 70, 700, 700, 1),     # 560 items, more blocks than CUs
    ((16, 8, 128), 130, 600, 600, 1),  # 1040 items, one block each
    ((4, 2, 128), 3, 250, 250, 4),     # short: one block each
    ((64, 2, 96), 5, 2000, 2000, 1),   # two row tiles
    ((8, 4, 64), 1000, 3, 9000, 1),    # most sequences empty or of a token, runs of a few tiles
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
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 28, width=-(-bound // 16))
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, most, bound)
    ref = reference(torch, k, v, table, lengths, q, 0, layout[2] ** -0.5)
    y = torch.full(q.shape, float("nan"), device="cuda")
    for _ in range(2):
        check(torch, cache.attend_decode(batch, q, out=y.fill_(float("nan"))), ref, torch.float16, False)


SHARED_KEYS = [
    # layout, page, type, out, (new, old) per sequence, window: few rows, so that blocks share a row tile's keys
    ((4, 2, 128), 16, "float16", "float32", [(20, 3000), (1, 5000), (130, 700), (0, 9), (33, 0)], 0),
    ((8, 1, 96), 64, "bfloat16", "bfloat16", [(40, 6001), (17, 300)], 0),
    ((4, 4, 64), 8, "float16", "float16", [(300, 4000), (5, 100)], 3500),
    ((2, 2, 128), 32, "bfloat16", "float32", [(129, 4000)], 300),
    ((3, 1, 64), 16, "float16", "float32", [(18, 511), (2, 20000)], 0),
]


@pytest.mark.parametrize("case", SHARED_KEYS, ids=str)
def test_prompt_of_few_rows_and_many_keys(gpu, lib, case):
    import torch
    layout, page, dtype, out, lengths, window = case
    dtype, out = getattr(torch, dtype), getattr(torch, out)
    unmapped = [(0, 300 // page)]
    k, v, table, q_start, kv_len, q = make(torch, layout, page, dtype, lengths, 29, unmapped=unmapped)
    most = max(n + o for n, o in lengths)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, max(n for n, _ in lengths), most)
    assert batch.workspace.numel() > 0
    ref = reference(torch, k, v, table, lengths, q, window, layout[2] ** -0.5)
    y = torch.full(q.shape, float("nan"), dtype=out, device="cuda")
    for _ in range(3):
        check(torch, cache.attend_prompt(batch, q, out=y.fill_(float("nan")), window=window), ref, dtype, True)
    # the same without a workspace, in one block per row tile
    batch.c.workspace, batch.c.workspace_bytes = None, 0
    check(torch, cache.attend_prompt(batch, q, out=y.fill_(float("nan")), window=window), ref, dtype, True)


def test_prompt_and_decode_share_a_workspace(gpu, lib):
    """Few new tokens go through either call, one after the other, with the batch's workspace."""
    import torch
    layout, lengths = (8, 2, 128), [(3, 4000), (1, 900)]
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 30)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 3, 4003)
    ref = reference(torch, k, v, table, lengths, q, 0, 128 ** -0.5)
    for _ in range(3):
        for call, prompt in ((cache.attend_decode, False), (cache.attend_prompt, True)):
            check(torch, call(batch, q, out=torch.full(q.shape, float("nan"), device="cuda")), ref, torch.float16, prompt)
    v[int(table[0, 250]), 1, 4, 9] = float("nan")  # the last position but two of the first sequence: hidden from one row
    bad = [i for i in range(3) if 4000 + i >= 250 * 16 + 4]
    assert not bad
    v[int(table[0, 4001 // 16]), 1, 4001 % 16, 9] = float("nan")
    for call, prompt in ((cache.attend_decode, False), (cache.attend_prompt, True)):
        y = call(batch, q, out=torch.empty_like(q, dtype=torch.float32))
        clean = [0, 3]
        check(torch, y[clean], [t[clean] for t in ref], torch.float16, prompt)
        assert torch.isnan(y[1:3, 4:, 9]).all() and not torch.isnan(y[1:3, :4]).any()


MANY_ROWS = [
    # layout, page, type, out, new tokens per sequence, window; more than 16 rows (token, head) per key-value head and bounds
    # of 2^17 positions of all heads, from which on an item has two row tiles
    ((8, 2, 128), 16, "float16", "float32", [5, 16, 8, 0, 1], 0),
    ((8, 1, 128), 64, "bfloat16", "float32", [3, 0, 4], 0),
    ((64, 2, 96), 16, "float16", "float16", [1], 0),
    ((12, 4, 96), 128, "bfloat16", "bfloat16", [16, 7, 11], 0),
    ((40, 1, 64), 1, "float16", "float32", [2, 1], 0),
    ((4, 4, 64), 16, "float16", "float32", [16, 9], 40),  # (16 rows: one)
    ((17, 1, 128), 32, "float16", "float32", [1], 300),
    ((6, 2, 96), 8, "float16", "float32", [11, 12], 33),
]


@pytest.mark.parametrize("case", MANY_ROWS, ids=str)
def test_decode_of_many_rows(gpu, lib, case):
    import torch
    layout, page, dtype, out, news, window = case
    dtype, out = getattr(torch, dtype), getattr(torch, out)
    lengths = [(news[i % len(news)], n) for i, n in enumerate(LENGTHS + [1500, 4001])]
    bound = -(-(1 << 17) // len(lengths) // layout[1])
    bound = max(bound, 4001 + max(news))
    k, v, table, q_start, kv_len, q = make(torch, layout, page, dtype, lengths, 31, unmapped=[(18, 700 // page)],
                                           width=-(-bound // page) + 1)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, max(news), bound)
    ref = reference(torch, k, v, table, lengths, q, window, layout[2] ** -0.5)
    y = torch.full(q.shape, float("nan"), dtype=out, device="cuda")
    first = None
    for _ in range(3):
        check(torch, cache.attend_decode(batch, q, out=y.fill_(float("nan")), window=window), ref, dtype, False)
        first = y.clone() if first is None else first
        assert torch.equal(first, y)
    # what no row of a sequence sees, and what only its last row sees
    if window == 0 and max(news) > 1:
        s = max(i for i, (n, o) in enumerate(lengths) if n > 1)
        n, o = lengths[s]
        last = o + n - 1
        v[int(table[s, last // page]), :, last % page] = float("inf")
        y = cache.attend_decode(batch, q, out=torch.empty_like(q, dtype=torch.float32))
        row = int(q_start[s + 1]) - 1
        keep = [r for r in range(q.shape[0]) if r != row]
        check(torch, y[keep], [t[keep] for t in ref], dtype, False)
        assert not torch.isfinite(y[row]).any()
