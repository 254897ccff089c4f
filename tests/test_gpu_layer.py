"""A decoder layer of coded matrices with its attention (examples/decoder_layer.py) against the same layer in 64 bits from the
dequantized weights: packed prompts, single tokens and drafts one after the other, and a captured decode step."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# q, k and v rounded to fp16 once each (2^-11 of values whose products enter scores of a few units), attention's weights and
# the outputs' sums beyond that: a few 2^-11 of the hidden states' size
TOL = 4 * 2.0 ** -11


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("decoder_layer", os.path.join(ROOT, "examples", "decoder_layer.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


class Exact:
    """The layer over whole histories, in 64 bits."""

    def __init__(self, torch, orc, bundle, shapes, layer):
        self.torch, self.layer = torch, layer
        self.w = {}
        for i, (n, rows, cols) in enumerate(shapes):
            codes, side = bundle.synth_matrix(1, rows, cols, 2.3, 2000 + i)
            self.w[n] = torch.from_numpy(np.asarray(orc.dequant(1, codes, side), np.float64)) * (layer.scale[n] / 16)

    def norm(self, x):
        return x * self.torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)

    def __call__(self, x):
        torch, layer = self.torch, self.layer
        n, heads, kv, dim = x.shape[0], layer.heads, layer.kv_heads, layer.dim
        h = self.norm(x)
        cos, sin = layer.cos[:n].double().cpu()[:, None], layer.sin[:n].double().cpu()[:, None]

        def turned(y, count):
            a, b = y.view(n, count, dim).split(dim // 2, -1)
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        q, k = turned(h @ self.w["q"].T, heads), turned(h @ self.w["k"].T, kv)
        v = (h @ self.w["v"].T).view(n, kv, dim)
        k, v = (t.repeat_interleave(heads // kv, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * dim ** -0.5
        s = s.masked_fill(torch.ones(n, n).triu(1).bool(), -float("inf"))
        y = torch.einsum("hij,jhd->ihd", s.softmax(-1), v).reshape(n, heads * dim)
        x = x + y @ self.w["o"].T
        h = self.norm(x)
        g = h @ self.w["gate"].T
        return x + (g * torch.sigmoid(g) * (h @ self.w["up"].T)) @ self.w["down"].T


def test_layer_against_64_bits(gpu, lib, orc, example, tmp_path):
    import torch
    from lazyweights_amd import Runtime, bundle
    example.write_layer(str(tmp_path), example.SMALL)
    with Runtime(tmp_path) as rt:
        layer = example.Layer(rt, example.SMALL, 8, 2, pages=40, page_size=16)
        exact = Exact(torch, orc, bundle, example.SMALL, layer)
        seqs = example.Sequences(layer, 3, most=160)
        g = torch.Generator().manual_seed(5)
        history = [torch.zeros((0, 512), dtype=torch.float64) for _ in range(3)]
        for news in ([70, 5, 33], [1, 1, 1], [1, 1, 1], [4, 4, 4], [1, 1, 1], [20, 1, 2], [5, 5, 5]):
            x = torch.randn((sum(news), 512), generator=g)
            y = layer(x.cuda(), seqs.batch(news)).double().cpu()
            at = 0
            for s, n in enumerate(news):
                history[s] = torch.cat((history[s], x[at:at + n].double()))
                ref = exact(history[s])[-n:]
                err = ((y[at:at + n] - ref).abs().max() / ref.abs().max()).item()
                print(news, s, "err %.2g" % err, flush=True)
                assert err < TOL
                at += n


def test_captured_decode_step(gpu, lib, example, tmp_path):
    """A decode step captured once and replayed while the sequences grow gives the steps' own results."""
    import torch
    from lazyweights_amd import Runtime
    example.write_layer(str(tmp_path), example.SMALL)
    with Runtime(tmp_path) as rt:
        layers = [example.Layer(rt, example.SMALL, 8, 2, pages=40) for _ in range(2)]
        seqs = [example.Sequences(layer, 2, most=160) for layer in layers]
        g = torch.Generator(device="cuda").manual_seed(6)
        prompt = torch.randn((50, 512), generator=g, device="cuda")
        for layer, s in zip(layers, seqs):
            layer(prompt, s.batch([30, 20]))
        x = torch.randn((2, 512), generator=g, device="cuda")
        for layer, s in zip(layers, seqs):  # scratch grown before the capture
            layer(x, s.batch([1, 1]))
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
