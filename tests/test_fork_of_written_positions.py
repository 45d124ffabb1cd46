"""A fork takes positions that have been written, not those whose pages were handed out ahead, and shares no block that a
captured step of its source is still to write.  CPU (the pool, and a dense decoder's bookkeeping: no kernel runs)."""
import pytest
import torch

from test_page_pool_fork import new, rows, sound, write
from treeattn_amd.config import Config
from treeattn_amd.engine import Decoder


def test_pages_handed_out_ahead_are_not_positions():
    pool = new()
    pool.ensure(12, seqs=[0])                # pages for 12 positions, of which 5 are written
    for t in range(5):
        write(pool, 0, t, t)
    pool.wrote(5, [0])
    for t in (6, 8, 12):
        with pytest.raises(ValueError, match='holds no'):
            pool.fork(0, 1, t)
        sound(pool)
    pool.fork(0, 1, 5)
    sound(pool)
    with pytest.raises(ValueError, match='holds no'):
        pool.fork(1, 2, 6)                   # nor does the fork hold more than it took
    for t in range(5, 12):
        write(pool, 0, t, t)                 # (asserts that the page is its own)
    assert torch.equal(rows(pool, 1, 5)[0, 0], torch.arange(5.))
    pool.wrote(12, [0])
    pool.fork(0, 1, 12)
    pool.wrote(3, [0])                       # (written again: the others still hold what they held)
    pool.fork(0, 2, 11)
    sound(pool)
    pool.release(0)
    pool.ensure(8, seqs=[0])
    pool.fork(0, 2, 8)                       # nobody said what is written: what has pages
    sound(pool)


def test_blocks_that_the_source_is_still_to_write_are_copied():
    pool = new()
    pool.ensure(14, seqs=[0])
    for t in range(14):
        write(pool, 0, t, t)
    pool.wrote(14, [0])
    before = rows(pool, 0, 14)
    pool.fork(0, 1, 13, ahead=6)             # it goes on from 6: block 0 shared, 1 to 3 copied
    sound(pool)
    assert pool.n_shared == 2
    for t in range(6, 14):
        write(pool, 0, t, -t)
    assert torch.equal(rows(pool, 1, 13), before[..., :13])
    pool.fork(1, 2, 13, ahead=13)            # the part of a block alone
    sound(pool)
    assert pool.n_shared == 6
    pool = new(pages=12)
    pool.ensure(12, seqs=[0])
    pool.wrote(12, [0])
    pool.ensure(8, seqs=[2])
    with pytest.raises(RuntimeError, match='out of pages'):
        pool.fork(0, 1, 12, ahead=4)
    sound(pool)
    assert pool.nblk[1] == 0


def decoder(**kw):
    cfg = Config(vocab_size=11, seq_len=256, n_layer=2, n_head=2, n_embd=32, attn='seg')
    W = dict(wte=torch.zeros(11, 32), wpe=torch.zeros(256, 32), ln_f=torch.ones(32),
             layers=[dict(ln1=torch.ones(32), ln2=torch.ones(32), c_attn=torch.zeros(96, 32), c_proj=torch.zeros(32, 32),
                          c_fc=torch.zeros(128, 32), c_mlp=torch.zeros(32, 128)) for _ in range(2)])
    return Decoder(W, 2, 2, 32, 256, 'dense', cfg, 'cpu', batch=3, paged=True, **kw)


def captured(d, at):
    """As after Decoder.capture and replays up to positions `at`."""
    d.graph, d.graphs, d.g_t = object(), [], torch.tensor(at)
    d._t_host = max(at)
    d._reserved = d._t_host + 1 + d.reserve_ahead
    d.pool.ensure(d._reserved)


def test_a_decoder_forks_what_its_steps_wrote():
    d = decoder(reserve_ahead=100)
    d.pool.ensure(50)
    d.pool.wrote(10)
    captured(d, [40, 25, 12])
    for bad in ((1, 0, 26), (0, 1, 41), (2, 0, 64)):
        with pytest.raises(ValueError, match='holds no'):
            d.fork(*bad)
        sound(d.pool)
    d.fork(1, 2, 12)
    assert d.g_t.tolist() == [40, 25, 12]     # (the caller's)
    d.fork(0, 1, 20)
    with pytest.raises(ValueError, match='holds no'):
        d.fork(1, 2, 21)                      # g_t still says 25, which sequence 1 had before
    sound(d.pool)
    d.g_t[1] = 20
    d.g_t += 100                              # replays
    d.fork(0, 1, 140)
    d.g_t[1] = 140
    assert d.pool.n_shared == 140 // 64 * 2
    d.fork(0, 2, 125)
    d.g_t[2] = 125
    d.g_t[0] = 70                             # sequence 0 goes back: its next replays write blocks 1 and 2
    d.pool.own(0, 70)
    with pytest.raises(ValueError, match='holds no'):
        d.fork(2, 0, 126)
    d.fork(0, 2, 130)
    sound(d.pool)
    for j in (1, 2):
        assert all(d.pool.refs[int(p)] == 1 for p in d.pool.host[0, :, j])
    d.resize(d.pool.P + 1)                    # (no captured step any more: what its replays wrote stays known)
    assert d.graph is None and d.pool.tokens[:2] == [140, 140]


def test_a_fork_forgets_the_tail_of_its_target():
    """The unrounded rows of an 8-bit cache's last block belong to what the target held before."""
    pool = new(cache='e4m3')
    held = [torch.tensor([[2, 2], [1, 1], [0, 0]], dtype=torch.int32) for _ in range(2)]
    pool.held += held
    pool.ensure(12)
    pool.fork(0, 1, 8)
    assert all(x.tolist() == [[2, 2], [-1, -1], [0, 0]] for x in held)
    with pytest.raises(ValueError):
        pool.fork(0, 2, 13)
    assert all(x.tolist() == [[2, 2], [-1, -1], [0, 0]] for x in held)
