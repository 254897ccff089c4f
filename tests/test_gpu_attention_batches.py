"""Decode of batches whose sequences a block holds 64 at a time, in the form that cuts the list of key tiles into equal runs (more
keys than a block per item takes, fewer items), against 64 bits: one to four times 64, so that some, all or none of a block's
waves have a part in the count."""
import pytest
from test_gpu_attention import build, check, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [64, 65, 128, 129, 150, 192, 193, 256, 300])
@pytest.mark.parametrize("layout", [(4, 1, 64), (8, 2, 128)], ids=str)
def test_many_sequences_in_runs(gpu, lib, seqs, layout):
    import torch
    lengths = [((1, 2, 0, 1)[s % 4], (s * 37) % 300) for s in range(seqs)]
    lengths[seqs // 2], lengths[-1] = (1, 1100), (2, 700)
    k, v, table, q_start, kv_len, q = make(torch, layout, 16, torch.float16, lengths, 51)
    cache, batch = build(torch, layout, k, v, table, q_start, kv_len, 2, 1102)
    y = torch.full(q.shape, float("nan"), device="cuda")
    for _ in range(2):
        y.fill_(float("nan"))
        cache.attend_decode(batch, q, out=y)
    check(torch, y, reference(torch, k, v, table, lengths, q, 0, layout[2] ** -0.5), torch.float16, False)
