"""Decoder(attn_split=n) with whole caches: n workgroups for each (sequence, head)."""
import pytest
import torch

from test_fork_of_written_positions import decoder
from test_gpu_dense_decoder import dec, logits64, model


def test_workgroups_of_all_queries():
    assert decoder(attn_split=1).scratch.dense == (4, None)
    for n, want in ((2, 4 * 2 * 6), (5, 4 * 5 * 6), (64, 4 * 64 * 6), (2048, 8192)):      # 3 sequences, 2 heads
        ns, ws = decoder(attn_split=n).scratch.dense
        assert ns == want and ws is not None and not ws.any()


@pytest.mark.gpu
@pytest.mark.parametrize('split', [1, 2, 7, 100, 4000])
def test_logits_do_not_depend_on_it(split):
    """Float32 sums in another order: 1e-4 of the logits' size, where they are off by some 1e-6."""
    m, cfg = model()
    idx = torch.randint(0, 97, (3, 150), generator=torch.Generator().manual_seed(1)).cuda()
    want = logits64(m, cfg, idx)
    d = dec(m, cfg, batch=3, attn_split=split)
    d.prefill(idx[:, :140])
    for t in range(140, 150):
        lg, _ = d.step(idx[:, t], t)
        assert float((lg.double() - want[:, t]).abs().max()) <= 1e-4 * float(want.abs().max())
