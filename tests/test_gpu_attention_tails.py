"""Attention where one key outweighs all the others by far (a first token that every row attends to), against the formula in
64 bits: the small weights of a long tail count in full, as many bits of them as the outputs show.

The scores are exact: q has one element, the dominant key scores 0 and every other one -below, so the row at position i is
(sink + w (v_1 + .. + v_i)) / (1 + w i), w = exp(-below). Like weights are the worst case, since what rounding takes from one
it takes from all.

Bounds, elementwise (A = sum p |v| / sum p of the row, l = 1 + w i the sum of its weights against the largest):
  the output's rounding          u |out|, u = 2^-24, 2^-11, 2^-8 for fp32, fp16, bf16, and 2^-25 for small fp16 outputs
  the weights' rounding          u_p A: 2^-11 where they are one fp16 part (prompt, 16-bit out), 2^-8 of bf16, else 2^-21
  small fp16 weights             (i + 1) max |v| / l times 2^-25 of the unit that the largest is 2^15 of (decode: 2^-40), or at
                                 least 2^11 (prompt: 2^-36)
  scores, sums, the exponential  A (2 2^-21 below + 2^-20)
"""
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def run(torch, layout, dtype, out, rows, keys, below, sink, prompt, seed, workspace=True):
    from lazyweights_amd import Batch, KvCache
    heads, kv, dim = layout
    page = 64
    pages = -(-keys // page)
    kind = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(seed)
    k = torch.zeros((pages * page, kv, dim), dtype=kind, device="cuda")
    k[1:, :, 0] = -below
    v = (0.5 + torch.rand((pages * page, kv, dim), generator=g, device="cuda")).to(kind)
    v[0] = sink
    q = torch.zeros((rows, heads, dim), dtype=kind, device="cuda")
    q[..., 0] = 1
    k_pages, v_pages = (x.view(pages, page, kv, dim).transpose(1, 2).contiguous() for x in (k, v))
    cache = KvCache(k_pages, v_pages)
    tab = torch.arange(pages, dtype=torch.int32, device="cuda")[None].contiguous()
    batch = Batch(cache, heads, torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                  torch.tensor([keys], dtype=torch.int32, device="cuda"), tab, rows, keys)
    if not workspace:
        batch.c.workspace, batch.c.workspace_bytes = None, 0
    y = torch.full(q.shape, float("nan"), dtype=getattr(torch, out), device="cuda")
    (cache.attend_prompt if prompt else cache.attend_decode)(batch, q, out=y, scale=1.0)
    w = torch.exp(torch.tensor(-float(k[-1, 0, 0].abs()), dtype=torch.float64))
    sums = v.double().cumsum(0) - v[:1].double()  # v_1 + .. + v_i
    at = torch.arange(keys - rows, keys, device="cuda")
    total = (1 + w.item() * at.double())[:, None, None]
    tail = w.item() * sums[at]
    want = ((v[:1].double() + tail) / total).repeat_interleave(heads // kv, 1)
    a = ((v[:1].double().abs() + tail) / total).repeat_interleave(heads // kv, 1)
    one_part = prompt and out != "float32"
    bound = U[out] * want.abs() + a * ((U[dtype] if one_part else 2.0 ** -21) + 2 * 2.0 ** -21 * below + 2.0 ** -20)
    if out == "float16":
        bound = bound + 2.0 ** -25
    if dtype == "float16":
        bound = bound + (at.double()[:, None, None] + 1) * v.double().max() / total * 2.0 ** (-36 if prompt else -40)
    err = (y.double() - want).abs()
    print("worst error %.2g of the output, error / bound %.3f" % (
        (err / want.abs().clamp(min=1e-30)).max().item(), (err / bound).max().item()), flush=True)
    assert (err <= bound).all()


BELOW = (12, 14, 16, 17, 18)


@pytest.mark.parametrize("sink", (0, 1))
@pytest.mark.parametrize("below", BELOW)
@pytest.mark.parametrize("keys, rows, layout, out", [
    (2999, 1, (8, 2, 128), "float32"), (131071, 1, (8, 2, 128), "float32"), (131071, 5, (8, 1, 64), "float16"),
    (201, 3, (4, 4, 96), "float32")], ids=str)
def test_decode_counts_the_tail(gpu, lib, keys, rows, layout, out, below, sink):
    """A block per item, runs of tiles joined in memory, two row tiles."""
    import torch
    run(torch, layout, "float16", out, rows, keys, below, sink, False, 31)


@pytest.mark.parametrize("sink", (0, 1))
@pytest.mark.parametrize("below", BELOW)
@pytest.mark.parametrize("out", ("float32", "float16", "bfloat16"))
@pytest.mark.parametrize("keys, rows, layout, workspace", [
    (2999, 40, (8, 2, 128), True), (40000, 40, (8, 2, 64), True), (40000, 40, (4, 1, 96), False),
    (8200, 8200, (32, 4, 64), True)], ids=str)
def test_prompt_counts_the_tail(gpu, lib, keys, rows, layout, workspace, out, below, sink):
    """A row tile per block, its keys shared out over blocks, blocks of 8 waves."""
    import torch
    run(torch, layout, "float16", out, rows, keys, below, sink, True, 32, workspace)


@pytest.mark.parametrize("prompt", (False, True))
def test_bfloat16_counts_the_tail(gpu, lib, prompt):
    import torch
    for below in (12, 18, 40):
        run(torch, (8, 2, 128), "bfloat16", "float32", 3, 20000, below, 0, prompt, 33)
