"""A decoder layer of coded matrices with its attention, as a serving loop would run it: prompts of several sequences at once,
then one token per sequence and step, then a draft of a few tokens per sequence in one pass.

    python examples/decoder_layer.py            # a Mistral-7B-shaped layer, synthetic weights
    python examples/decoder_layer.py --small    # 512 wide

The matrices (q, k, v, o, gate, up, down) are multiplied from their coded form (Runtime.matmul_dev); between q, k, v and o the
keys and values go into a paged cache, rotated on the way, and the new tokens attend over it (KvCache, Batch). Norms and the
gate are plain torch. Pages are handed out from a pool as sequences grow; the batch of a decode step and its tensors are kept
over the steps, so that the loop only writes lengths and page numbers on the GPU.
"""
import argparse
import os
import sys
import tempfile
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from lazyweights_amd import Batch, KvCache, Runtime, bundle  # noqa: E402
from lazyweights_amd.configs import MISTRAL, Q4_K  # noqa: E402

SMALL = [("q", 512, 512), ("k", 128, 512), ("v", 128, 512), ("o", 512, 512), ("gate", 1024, 512), ("up", 1024, 512),
         ("down", 512, 1024)]


def write_layer(path, shapes, seed=2000):
    """A bundle of one layer: its matrices with synthetic Q4_K weights."""
    return bundle.write_synthetic_bundle(path, [(n, Q4_K, rows, cols, 2.3, seed + i) for i, (n, rows, cols) in enumerate(shapes)])


class Layer:
    """One decoder layer over a bundle, with a cache of `pages` pages that its sequences share."""

    def __init__(self, rt, shapes, heads, kv_heads, pages, page_size=16, positions=8192, window=0):
        self.rt, self.heads, self.kv_heads, self.window = rt, heads, kv_heads, window
        self.size = {n: (rows, cols) for n, rows, cols in shapes}
        self.hidden, self.dim = self.size["q"][1], self.size["q"][0] // heads
        self.cache = KvCache.empty(pages, kv_heads, page_size, self.dim)
        turn = torch.arange(positions, dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(0, self.dim, 2, dtype=torch.float64) / self.dim)
        self.cos, self.sin = turn.cos().float().cuda(), turn.sin().float().cuda()
        self.scale = {n: (rows * cols) ** -0.25 for n, rows, cols in shapes}  # synthetic weights are not normalised

    def mul(self, name, x):
        """x [tokens, K] through a coded matrix: fp16 activations for up to 16 tokens, fp32 beyond (fp32 out)."""
        y = torch.empty((x.shape[0], self.size[name][0]), device="cuda")
        few = x.shape[0] <= 16
        self.rt.matmul_dev(name, x.half() if few else x.float(), y, x_f16=few,
                           stream=torch.cuda.current_stream().cuda_stream)
        return y * (self.scale[name] / 16)

    def norm(self, x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)

    def __call__(self, x, batch):
        """Hidden states [tokens, hidden] (fp32) of the batch's new tokens through the layer."""
        h = self.norm(x)
        q, k, v = self.mul("q", h), self.mul("k", h), self.mul("v", h)
        q16 = self.cache.append(batch, q, k, v, self.cos, self.sin)
        attend = self.cache.attend_decode if batch.max_new <= 16 else self.cache.attend_prompt
        y = attend(batch, q16, out=torch.empty((x.shape[0], self.heads, self.dim), device="cuda"), window=self.window)
        x = x + self.mul("o", y.view(x.shape[0], -1))
        h = self.norm(x)
        return x + self.mul("down", torch.nn.functional.silu(self.mul("gate", h)) * self.mul("up", h))


class Sequences:
    """Lengths and pages of the sequences in a layer's cache."""

    KEPT = 8  # batches

    def __init__(self, layer, count, most):
        page = layer.cache.k.shape[2]
        self.layer, self.page, self.most = layer, page, most
        self.table = torch.full((count, -(-most // page)), -1, dtype=torch.int32, device="cuda")
        self.kv_len = torch.zeros(count, dtype=torch.int32, device="cuda")
        self.lengths, self.free = [0] * count, list(range(layer.cache.k.shape[0]))
        self.pages = [[] for _ in range(count)]
        self.steady = {}

    def grow(self, news):
        """Room for news[s] more tokens of every sequence, in the tensors that the batches read."""
        for s, n in enumerate(news):
            self.lengths[s] += n
            while len(self.pages[s]) * self.page < self.lengths[s]:
                self.table[s, len(self.pages[s])] = self.free[0]
                self.pages[s].append(self.free.pop(0))
        self.kv_len.copy_(torch.tensor(self.lengths, dtype=torch.int32))

    def batch(self, news):
        """The batch in which every sequence has news[s] new tokens; the last KEPT kinds of them are kept, each with its workspace
        (steps of single tokens and drafts come again and again, prompts hardly ever in the same lengths; who captures a call keeps
        its batch)."""
        self.grow(news)
        key = tuple(news)
        batch = self.steady.pop(key, None)
        if batch is None:
            starts = torch.tensor([0] + news, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
            batch = Batch(self.layer.cache, self.layer.heads, starts, self.kv_len, self.table, max(news), self.most)
        self.steady[key] = batch  # (the last one used at the end)
        while len(self.steady) > self.KEPT:
            del self.steady[next(iter(self.steady))]
        return batch


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--small", action="store_true")
    ap.add_argument("--steps", type=int, default=32)
    a = ap.parse_args()
    shapes, heads, kv_heads = (SMALL, 8, 2) if a.small else (MISTRAL, 32, 8)
    prompts = [700, 33, 1500, 4]
    with tempfile.TemporaryDirectory() as d:
        write_layer(d, shapes)
        with Runtime(d) as rt:
            layer = Layer(rt, shapes, heads, kv_heads, pages=512)
            seqs = Sequences(layer, len(prompts), most=2000)
            torch.manual_seed(0)

            def run(news, steps=1):
                torch.cuda.synchronize()
                t = time.perf_counter()
                for _ in range(steps):
                    y = layer(torch.randn((sum(news), layer.hidden), device="cuda"), seqs.batch(news))
                torch.cuda.synchronize()
                if not torch.isfinite(y).all():
                    raise RuntimeError("hidden states are not finite")
                return (time.perf_counter() - t) / steps * 1e6

            print("prompts of %s tokens, the process's first calls: %.0f us" % (prompts, run(prompts)), flush=True)
            print("a token per sequence, %d steps: %.0f us a step" % (a.steps, run([1] * len(prompts), a.steps)), flush=True)
            print("a draft of 4 tokens per sequence: %.0f us" % run([4] * len(prompts)), flush=True)


if __name__ == "__main__":
    main()
