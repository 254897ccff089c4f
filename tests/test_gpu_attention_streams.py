"""Calls on a stream that is not torch's current one: memory that the current stream still writes is not handed out as an output, and
the memory of inputs is not handed out again while the call has yet to read it."""
import pytest
from test_gpu_attention import build, make

pytestmark = pytest.mark.gpu

LAYOUT = (8, 2, 128)


def setup(torch):
    k, v, table, q_start, kv_len, q = make(torch, LAYOUT, 16, torch.float16, [(5, 300), (16, 64)], 71)
    cache, batch = build(torch, LAYOUT, k, v, table, q_start, kv_len, 16, 305)
    g = torch.Generator(device="cuda").manual_seed(72)
    new = [torch.randn((21, h, 128), generator=g, device="cuda").half() for h in (8, 2, 2)]
    return cache, batch, q, new


def calls(torch, cache, batch):
    """A call of (tensors, stream) by name."""
    return {"decode": lambda t, s: cache.attend_decode(batch, t[0], stream=s),
            "prompt": lambda t, s: cache.attend_prompt(batch, t[0], stream=s),
            "append": lambda t, s: cache.append(batch, t[0], t[1], t[2], stream=s)}


@pytest.mark.parametrize("which", ("decode", "prompt", "append"))
def test_outputs_are_of_the_given_stream(gpu, lib, which):
    import torch
    cache, batch, q, new = setup(torch)
    tensors, call = new if which == "append" else [q], calls(torch, cache, batch)[which]
    want = call(tensors, None).clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    block = torch.empty_like(want)
    at = block.data_ptr()
    torch.cuda._sleep(20_000_000)
    block.fill_(float("nan"))
    del block  # free for the current stream, which has yet to write it
    y = call(tensors, side.cuda_stream)
    assert y.data_ptr() != at
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("which", ("decode", "prompt", "append"))
def test_inputs_last_until_the_given_stream_has_read_them(gpu, lib, which):
    import torch
    cache, batch, q, new = setup(torch)
    call = calls(torch, cache, batch)[which]
    want = call(new if which == "append" else [q], None).clone()
    side = torch.cuda.Stream()
    tensors = [t.clone() for t in (new if which == "append" else [q])]
    like, places = [torch.empty_like(t, device="meta") for t in tensors], {t.data_ptr() for t in tensors}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
    y = call(tensors, side.cuda_stream)
    del tensors
    for t in like:
        z = torch.full(t.shape, float("nan"), dtype=t.dtype, device="cuda")
        assert z.data_ptr() not in places
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_the_default_and_the_current_stream_by_handle(gpu, lib):
    import torch
    cache, batch, q, _ = setup(torch)
    want = cache.attend_decode(batch, q).clone()
    torch.cuda.synchronize()
    current = torch.cuda.current_stream().cuda_stream
    assert torch.equal(cache.attend_decode(batch, q, stream=current), want)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = cache.attend_decode(batch, q, stream=0)
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    assert cache.attend_decode(batch, q, out=out, stream=side.cuda_stream) is out
    torch.cuda.synchronize()
    assert torch.equal(out, want)
