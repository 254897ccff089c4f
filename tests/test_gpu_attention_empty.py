"""A cache without pages, whose memory may be no memory at all: every page is one that is not there, so nothing is appended, queries
are rotated all the same and rows of attention see nothing."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ("float16", "float32"))
@pytest.mark.parametrize("news, old, max_kv, layout, window", [
    ([1], 40, 200, (8, 2, 128), 0), ([1, 3, 0], 5000, 8192, (8, 2, 128), 0), ([16] * 3, 70000, 70016, (32, 2, 64), 100),
    ([1] * 70, 900, 2000, (4, 1, 96), 0), ([40], 0, 40, (8, 8, 64), 0), ([64], 20000, 20064, (8, 2, 128), 0),
    ([9000], 100, 10000, (32, 4, 64), 50)], ids=str)
def test_no_pages(gpu, lib, news, old, max_kv, layout, window, out):
    """A block per item, runs, two row tiles, many sequences, short prompts, shared row tiles, blocks of 8 waves."""
    import torch
    from lazyweights_amd import Batch, KvCache
    heads, kv, dim = layout
    page, rows = 16, sum(news)
    cache = KvCache.empty(0, kv, page, dim)
    assert cache.k.data_ptr() == 0
    starts = torch.tensor([0] + news, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    table = torch.zeros((len(news), -(-max_kv // page)), dtype=torch.int32, device="cuda")
    batch = Batch(cache, heads, starts, torch.tensor([n + old for n in news], dtype=torch.int32, device="cuda"), table,
                  max(news), max_kv)
    g = torch.Generator(device="cuda").manual_seed(61)
    q, k = (torch.randn((rows, h, dim), generator=g, device="cuda") for h in (heads, kv))
    q16 = cache.append(batch, q, k, k)
    assert torch.equal(q16, q.half())
    for attend in ([cache.attend_decode] if max(news) <= 16 else []) + [cache.attend_prompt]:
        y = torch.full(q.shape, float("nan"), dtype=getattr(torch, out), device="cuda")
        attend(batch, q16, out=y, window=window)
        torch.cuda.synchronize()
        assert not y.any()
