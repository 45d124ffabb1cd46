"""Sequences forked between the replays of a captured step, at positions that the replays have written and at others
(engine.Decoder.fork).  GPU only."""
import pytest
import torch

from test_gpu_dense_decoder import BF16, DEV, dec, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('mode,dkw', [('dense', {}), ('seg', {}), ('seg', dict(cache='e4m3'))])
def test_a_fork_takes_what_replays_have_written(mode, dkw):
    m, cfg = model(BF16, n_head=2, dh=64, neighbors=False)
    idx = torch.randint(0, 97, (3, 20), generator=torch.Generator().manual_seed(1)).to(DEV)
    d = dec(m, cfg, mode, batch=3, reserve_ahead=150, **dkw)
    d.capture(d.prefill(idx).argmax(-1), 20)
    leaf = d.pool.leaf
    for n in range(20, 20 + 2 * leaf):
        for t in (n + 1, n + leaf, 150):
            with pytest.raises(ValueError, match='holds no'):
                d.fork(0, 1, t)
        d.replay()
    at = 20 + 2 * leaf
    d.fork(0, 1, at)
    d.g_t[1] = at
    n_shared = d.pool.n_shared
    assert n_shared == at // leaf * d.H
    # sequence 2 goes back to position 9 and is forked at a later one: its replays leave the fork alone
    d.g_t[2] = 9
    d.fork(2, 0, at - 3)
    d.g_t[0] = at - 3
    whole = (at - 3) // leaf * leaf if dkw else at - 3   # (an 8-bit cache reads its last block unrounded until it goes on)
    keep = [x.clone() for st in d.states for b, n in ((0, whole), (1, at // leaf * leaf)) for x in st.dense_kv(b, n)]
    for _ in range(leaf + 3):
        d.replay()
    torch.cuda.synchronize()
    for x, y in zip(keep, [x for st in d.states for b, n in ((0, whole), (1, at // leaf * leaf)) for x in st.dense_kv(b, n)]):
        assert torch.equal(x, y)
    assert d.g_t.tolist() == [at + leaf, at + leaf + 3, 12 + leaf]
