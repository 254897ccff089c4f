"""Batches whose rows do not begin at row 0 of a call's tensors (another batch's rows come first, as where prompts and single tokens of
one step are packed together), and starts in no order: appending to caches of 8 and of 16 bits, and attention over them, touch their own rows and
pages alone."""
import pytest
from test_gpu_attention import make
from test_gpu_attention8 import Made, check, held, reference

pytestmark = pytest.mark.gpu

LENGTHS = [
    [(1, 16)],  # a short cache: items before the sequence's would have blocks before its first
    [(1, 300), (1, 5)],  # a long one: its older, full blocks
    [(20, 33), (0, 40), (3, 0), (16, 250)],
    [(1, 7 * i % 90) for i in range(70)],
]


def guarded(torch, table, pages):
    """The table as a view with numbers of the cache's pages before and behind it."""
    around = torch.arange(128 + table.numel(), dtype=torch.int32, device="cuda") % pages
    view = around[64:64 + table.numel()].view(table.shape)
    view.copy_(table)
    return view


def raw(tensors, torch):
    return [t.view(torch.uint8).clone() for t in tensors]


@pytest.mark.parametrize("first", (1, 15, 16, 17, 64, 200))
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: str(x[:4]))
def test_rows_behind_others(gpu, lib, lengths, first):
    """8 bits: the same cache as of rows from 0 on, other blocks' exponents (out of range, so that they would change if they were written
    again) as they were, and the rows before left alone."""
    import torch
    from lazyweights_amd import Batch
    m, other = (Made(torch, (8, 2, 128), 16, "float16", lengths, 51) for _ in range(2))
    rows = int(m.q_start[-1])
    g = torch.Generator(device="cuda").manual_seed(52)
    q, k, v = (torch.randn((first + rows + 3, h, 128), generator=g, device="cuda") for h in (8, 2, 2))
    mine = torch.zeros(m.k_exp.shape, dtype=torch.bool, device="cuda")
    for s, (new, old) in enumerate(lengths):
        for block in range(old // 16, (old + new + 15) // 16 if new else 0):
            mine[int(m.table[s, block]), :, 0] = True
    for x in (m, other):
        for e in (x.k_exp, x.v_exp):
            e[~mine] = torch.where(torch.arange(int((~mine).sum()), device="cuda") % 2 == 0, 100, -100).to(torch.int8)
    tensors, others = ((x.k, x.v, x.k_exp, x.v_exp) for x in (m, other))
    before = raw(tensors, torch)
    batch = Batch(m.cache, 8, m.q_start + first, m.kv_len, guarded(torch, m.table, m.k.shape[0]), m.max_new, m.max_kv)
    out = m.cache.append(batch, q, k, v, q_out=torch.full(q.shape, float("nan"), dtype=torch.float16, device="cuda"))
    other.cache.append(other.batch, None, k[first:first + rows], v[first:first + rows])
    assert torch.isnan(out[:first]).all() and torch.isnan(out[first + rows:]).all()
    assert torch.equal(out[first:first + rows], q[first:first + rows].half())
    for now, want in zip(raw(tensors, torch), raw(others, torch)):
        assert torch.equal(now, want)
    for now, was in zip((m.k_exp, m.v_exp), before[2:]):
        assert torch.equal(now.view(torch.uint8)[~mine], was[~mine])
    untouched = ~mine[..., 0]
    for now, was in zip((m.k, m.v), before):
        assert torch.equal(now.view(torch.uint8)[untouched], was[untouched])
    for x in (m, other):  # (2^48 beside ordinary values would hide everything else)
        for e in (x.k_exp, x.v_exp):
            e[~mine] = 0
    m.q = out[first:first + rows]
    ref = reference(m)
    for call, prompt in ([(m.cache.attend_decode, False)] if m.max_new <= 16 else []) + [(m.cache.attend_prompt, True)]:
        y = call(batch, torch.where(torch.isnan(out), 1, out), out=torch.full(q.shape, float("nan"), device="cuda"))
        assert torch.isnan(y[:first]).all() and torch.isnan(y[first + rows:]).all()
        check(torch, y[first:first + rows], ref, prompt)


@pytest.mark.parametrize("first", (16, 64))
@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda x: str(x[:4]))
def test_rows_behind_others_16_bits(gpu, lib, lengths, first):
    """The same calls over a 16-bit cache: bits as of rows from 0 on."""
    import torch
    from lazyweights_amd import Batch, KvCache
    made = [make(torch, (8, 2, 128), 16, torch.float16, lengths, 53) for _ in range(2)]
    rows, most, longest = int(made[0][3][-1]), max(n for n, _ in lengths), max(n + o for n, o in lengths)
    g = torch.Generator(device="cuda").manual_seed(54)
    q, k, v = (torch.randn((first + rows + 3, h, 128), generator=g, device="cuda") for h in (8, 2, 2))
    results = []
    for shift, (kc, vc, table, starts, kv_len, _) in zip((first, 0), made):
        cache = KvCache(kc, vc)
        batch = Batch(cache, 8, starts + shift, kv_len, guarded(torch, table, kc.shape[0]), most, longest)
        part = slice(0, None) if shift else slice(first, first + rows)
        q16 = cache.append(batch, q[part].contiguous(), k[part].contiguous(), v[part].contiguous(),
                           q_out=torch.zeros_like(q[part], dtype=torch.float16))
        y = cache.attend_decode(batch, q16, out=torch.zeros_like(q[part])) if most <= 16 else q16.float()
        assert not q16[:shift].any() and not y[:shift].any() and not q16[shift + rows:].any() and not y[shift + rows:].any()
        results.append(raw((kc, vc, q16[shift:shift + rows], y[shift:shift + rows]), torch))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize("starts", ([50, 3, 40], [70, 80, 16], [90, 17, 60, 0, 33], [-5, 200, 1 << 30], [64, 64, 64]), ids=str)
def test_starts_in_no_order(gpu, lib, starts):
    """Nothing but the sequences' own pages is written, and nothing at all for sequences without rows."""
    import torch
    from lazyweights_amd import Batch, KvCache8
    seqs, page, tokens = len(starts) - 1, 16, 96
    pages = 3 * seqs + 6
    g = torch.Generator(device="cuda").manual_seed(55)
    (k, k_exp), (v, v_exp) = (held(torch, torch.randn((pages, 2, page, 64), generator=g, device="cuda"), 1) for _ in range(2))
    k_exp.fill_(100)
    v_exp.fill_(-100)
    table = guarded(torch, torch.arange(3 * seqs, dtype=torch.int32, device="cuda").view(seqs, 3), pages)
    cache = KvCache8(k, v, k_exp, v_exp)
    batch = Batch(cache, 4, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                  torch.full((seqs,), 48, dtype=torch.int32, device="cuda"), table, 16, 48)
    before = raw((k, v, k_exp, v_exp), torch)
    q, x = (torch.randn((tokens, h, 64), generator=g, device="cuda") for h in (4, 2))
    q16 = cache.append(batch, q, x, x, q_out=torch.zeros(q.shape, dtype=torch.float16, device="cuda"))
    torch.cuda.synchronize()
    inside = [min(max(n, 0), tokens) for n in starts]
    for s in range(seqs + 1):  # (the last: pages of no sequence)
        if s == seqs or inside[s + 1] <= inside[s]:
            own = slice(3 * s, 3 * s + 3 if s < seqs else None)
            for now, was in zip(raw((k, v, k_exp, v_exp), torch), before):
                assert torch.equal(now[own], was[own]), s
    for call in (cache.attend_decode, cache.attend_prompt):
        call(batch, q16, out=torch.empty_like(q))
    torch.cuda.synchronize()
