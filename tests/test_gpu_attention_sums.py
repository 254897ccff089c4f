"""The sum of a row's weights over many keys that one wave goes through, against the formula in 64 bits: where the weights are
alike every addition to a sum in 32 bits is rounded the same way, so n additions in a row would be off by up to n 2^-25 of it.

The scores are exact (q has one element, the first key scores 0 and every other one -1), the values differ, so that the
products' sums are rounded one way and the other.

Bound, elementwise, of an fp32 output (A = sum p |v| / sum p of the row): its own rounding 2^-24 |out|, the weights' 2^-21 A,
scores, the exponential and the sum of weights (2 2^-21 + 2^-20) A, and the rounding of the n / 16 steps of a product's sum,
four standard deviations of a random walk, 4 sqrt(n / 16) 2^-24 A."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("keys", (40000, 131000))
def test_prompt_sums_of_like_weights(gpu, lib, keys, dtype):
    """Without a workspace a block goes through all keys of its rows."""
    import torch
    from lazyweights_amd import Batch, KvCache
    heads, dim, rows, page = 4, 96, 40, 64
    kind, pages = getattr(torch, dtype), -(-keys // page)
    g = torch.Generator(device="cuda").manual_seed(41)
    k = torch.zeros((pages * page, 1, dim), dtype=kind, device="cuda")
    k[1:, :, 0] = -1
    v = (0.5 + torch.rand((pages * page, 1, dim), generator=g, device="cuda")).to(kind)
    q = torch.zeros((rows, heads, dim), dtype=kind, device="cuda")
    q[..., 0] = 1
    cache = KvCache(*(x.view(pages, page, 1, dim).transpose(1, 2).contiguous() for x in (k, v)))
    batch = Batch(cache, heads, torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                  torch.tensor([keys], dtype=torch.int32, device="cuda"),
                  torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous(), rows, keys)
    batch.c.workspace, batch.c.workspace_bytes = None, 0
    y = cache.attend_prompt(batch, q, out=torch.empty(q.shape, device="cuda"), scale=1.0)
    at = torch.arange(keys - rows, keys, device="cuda")
    w, v64 = math.exp(-1), v.double()
    want = (v64[:1] + w * (v64.cumsum(0)[at] - v64[:1])) / (1 + w * at.double())[:, None, None]  # (values are positive: A too)
    err = ((y.double() - want).abs() / want).max().item()
    bound = 2.0 ** -24 + 2.0 ** -21 + 2 * 2.0 ** -21 + 2.0 ** -20 + 4 * math.sqrt(keys / 16) * 2.0 ** -24
    print("worst relative error %.2g, bound %.2g" % (err, bound), flush=True)
    assert err <= bound


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
@pytest.mark.parametrize("layout, new, old", [((32, 8, 128), 8200, 9000), ((32, 32, 96), 8200, 9000), ((32, 4, 64), 8200, 9000),
                                              ((32, 8, 128), 900, 20000), ((7, 1, 64), 2000, 18000)], ids=str)
def test_long_runs(gpu, lib, layout, new, old, dtype):
    """Blocks of 8 and of 4 waves over more than 16384 keys, fp32 outputs, the last key's value not finite: some rows against 64 bits,
    and the last, which alone sees that value. Bound as in the tests of any length: 2^-24 |out| + A (2^-21 + 2 2^-21 max_j scale
    sum |q k_j| + 2^-20)."""
    import torch
    from lazyweights_amd import Batch, KvCache
    heads, kv, dim = layout
    kind, page, keys = getattr(torch, dtype), 64, new + old
    pages, group = -(-keys // page), heads // kv
    g = torch.Generator(device="cuda").manual_seed(42)
    k = torch.randn((pages * page, kv, dim), generator=g, device="cuda").to(kind)
    v = (torch.randn((pages * page, kv, dim), generator=g, device="cuda") + 0.25).to(kind)
    q = (1.5 * torch.randn((new, heads, dim), generator=g, device="cuda")).to(kind)
    v[keys - 1] = float("inf")
    cache = KvCache(*(x.view(pages, page, kv, dim).transpose(1, 2).contiguous() for x in (k, v)))
    batch = Batch(cache, heads, torch.tensor([0, new], dtype=torch.int32, device="cuda"),
                  torch.tensor([keys], dtype=torch.int32, device="cuda"),
                  torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous(), new, keys)
    batch.c.workspace, batch.c.workspace_bytes = None, 0
    y = cache.attend_prompt(batch, q, out=torch.full(q.shape, float("nan"), device="cuda"))
    assert torch.isinf(y[-1]).all() and torch.isfinite(y[:-1]).all()
    worst = 0.0
    for row in [0, 1, 31, 32, 255, 256, new // 2, new - 300, new - 33, new - 2]:
        n = old + row + 1
        qq, kk, vv = q[row].double().view(kv, group, dim).cpu(), k[:n].double().cpu(), v[:n].double().cpu()
        s = torch.einsum("hgd,jhd->hgj", qq, kk) * dim ** -0.5
        p = torch.softmax(s, -1)
        want, a = (torch.einsum("hgj,jhd->hgd", p, x).reshape(heads, dim) for x in (vv, vv.abs()))
        most = (torch.einsum("hgd,jhd->hgj", qq.abs(), kk.abs()) * dim ** -0.5).amax(-1).reshape(heads, 1)
        bound = 2.0 ** -24 * want.abs() + a * (2.0 ** -21 + 2 * 2.0 ** -21 * most + 2.0 ** -20)
        worst = max(worst, ((y[row].double().cpu() - want).abs() / bound).max().item())
    print("worst error / bound %.3f" % worst, flush=True)
    assert worst <= 1
