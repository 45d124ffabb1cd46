"""SegState.fill of a view of some sequences (SegState.rows) takes pages of their own, not of the sequences of the same number.
CPU: the tree's kernel has a stand-in, the rows go through the page table."""
import torch

from test_page_pool_fork import sound
from treeattn_amd import selection as SEL
from treeattn_amd.config import Config
from treeattn_amd.engine import PagePool, SegState


def test_fill_leaves_shared_pages_alone(monkeypatch):
    monkeypatch.setattr(SEL, 'build_pyramid', lambda k, shape, t_end=None, out=None: out)
    cfg = Config(vocab_size=11, seq_len=32, n_layer=1, n_head=2, n_embd=8, attn='seg', leaf=4, neighbors=False)
    pool = PagePool(3, 2, 4, 4, 32, 60, 1, torch.float32, 'cpu')
    st = SegState(cfg, 32, 2, 4, 'cpu', batch=3, pages=pool)
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(3, 2, 12, 4, generator=g), torch.randn(3, 2, 12, 4, generator=g)
    st.fill(k, v)
    assert pool.tokens == [12] * 3
    pool.fork(1, 2, 12)
    view = st.rows(1, 3).rows(1, 2)                         # sequence 2
    new = [torch.randn(1, 2, 9, 4, generator=g) for _ in range(2)]
    view.fill(*new)
    sound(pool)
    for b in (0, 1):                                        # as they were
        got = st.dense_kv(b, 12)
        assert torch.equal(got[0][0], k[b]) and torch.equal(got[1][0], v[b])
    got = st.dense_kv(2, 9)
    assert torch.equal(got[0], new[0]) and torch.equal(got[1], new[1])
    assert pool.tokens == [12, 12, 12] and pool.nblk == [3, 3, 3]
