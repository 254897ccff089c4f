"""The decoder layer of examples/decoder_layer.py over a cache in 8 bits: prompts, single tokens and drafts, a captured step, and
its program."""
import os
import subprocess
import sys

import pytest
from test_gpu_layer import ROOT, example  # noqa: F401

pytestmark = pytest.mark.gpu


def test_captured_decode_step(gpu, lib, example, tmp_path):  # noqa: F811
    """A decode step captured once and replayed while the sequences grow gives the steps' own results."""
    import torch
    from lazyweights_amd import Runtime
    example.write_layer(str(tmp_path), example.SMALL)
    with Runtime(tmp_path) as rt:
        layers = [example.Layer(rt, example.SMALL, 8, 2, pages=40, eight=True) for _ in range(2)]
        seqs = [example.Sequences(layer, 2, most=160) for layer in layers]
        g = torch.Generator(device="cuda").manual_seed(8)
        for news in ([30, 20], [4, 4], [1, 1]):  # (the last: scratch grown before the capture)
            x = torch.randn((sum(news), 512), generator=g, device="cuda")
            first, second = (layer(x, s.batch(news)) for layer, s in zip(layers, seqs))
            assert torch.isfinite(first).all() and torch.equal(first, second)
        torch.cuda.synchronize()
        graph, batch = torch.cuda.CUDAGraph(), seqs[0].steady[(1, 1)]
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            layers[0].mul("q", x)
        side.synchronize()
        with torch.cuda.graph(graph):
            y = layers[0](x, batch)
        for step in range(20):
            x.copy_(torch.randn((2, 512), generator=g, device="cuda"))
            seqs[0].grow([1, 1])
            graph.replay()
            torch.cuda.synchronize()
            want = layers[1](x, seqs[1].batch([1, 1]))
            torch.cuda.synchronize()
            assert torch.equal(y, want), step


def test_no_pages_left(gpu, lib, example, tmp_path):  # noqa: F811
    from lazyweights_amd import Runtime
    example.write_layer(str(tmp_path), example.SMALL)
    with Runtime(tmp_path) as rt:
        seqs = example.Sequences(example.Layer(rt, example.SMALL, 8, 2, pages=5, eight=True), 2, most=64)
        seqs.batch([40, 30])
        with pytest.raises(RuntimeError, match="pages"):
            seqs.batch([10, 10])


@pytest.mark.parametrize("args", ([], ["--cache8"]), ids=str)
def test_program(gpu, lib, args):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "decoder_layer.py"), "--small", "--steps", "4"] + args,
                         stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert out.returncode == 0, out.stderr[-2000:]
    assert "draft of 4 tokens" in out.stdout
