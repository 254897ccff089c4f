"""The sequences of examples/decoder_layer.py after a step for which there are no pages, or no room: as they were, so that smaller steps
go on."""
import pytest
from test_gpu_layer import example  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eight", (False, True))
def test_after_a_refused_step(gpu, lib, example, eight):  # noqa: F811
    import torch
    from lazyweights_amd import KvCache, KvCache8

    class Layer:
        cache, heads = (KvCache8 if eight else KvCache).empty(5, 2, 16, 64), 8

    seqs = example.Sequences(Layer, 2, most=64)

    def agree(lengths):
        torch.cuda.synchronize()
        assert seqs.lengths == lengths == seqs.kv_len.tolist()
        assert seqs.pages.left.tolist() == [5 - sum(-(-n // 16) for n in lengths), 0]

    seqs.batch([30, 20])
    step = seqs.batch([1, 1])
    agree([31, 21])
    seqs.batch([1, 10])
    agree([32, 31])
    for news in ([1, 2], [20, 20], [40, 0]):  # one page is left: too many pages, and more than 64 tokens
        for _ in range(2):
            with pytest.raises(RuntimeError, match="pages"):
                seqs.batch(news)
            agree([32, 31])
    with pytest.raises(ValueError):  # (counts of another number of sequences)
        seqs.batch([1])
    agree([32, 31])
    assert seqs.batch([1, 1]) is step  # the last page, and the batch kept before the refusals
    agree([33, 32])
    with pytest.raises(RuntimeError, match="pages"):
        seqs.batch([0, 1])
    assert seqs.batch([15, 0]).tensors[0].tolist() == [0, 15, 15]
    agree([48, 32])
    with pytest.raises(RuntimeError, match="pages"):
        seqs.batch([1, 1])
    assert seqs.steady[(1, 1)] is step
