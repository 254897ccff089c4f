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
