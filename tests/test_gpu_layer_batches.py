"""The batches that examples/decoder_layer.py keeps: those of the steps that come again, and not one for every prompt there ever was."""
import pytest
from test_gpu_layer import example  # noqa: F401

pytestmark = pytest.mark.gpu


def test_batches_kept(gpu, lib, example):  # noqa: F811
    import torch
    from lazyweights_amd import KvCache

    class Layer:
        cache, heads = KvCache.empty(64, 2, 16, 64), 8

    seqs = example.Sequences(Layer, 1, most=1000)
    torch.cuda.synchronize()
    step = seqs.batch([1])
    for n in range(2, 22):
        seqs.batch([n])
        assert seqs.batch([1]) is step
    assert len(seqs.steady) <= 8
    assert seqs.lengths == [1 + sum(range(2, 22)) + 20] == [int(seqs.kv_len)]
