"""Forks, replays and captures that find too few pages leave a decoder as it was.  CPU: bookkeeping, no kernel runs."""
import pytest
import torch

from test_fork_of_written_positions import captured, decoder
from test_page_pool_fork import new, sound


def snapshot(d):
    p = d.pool
    return (p.host.tolist(), p.table.tolist(), list(p.free), list(p.refs), list(p.nblk), list(p.tokens), d.g_t.tolist(), d._t_host,
            d._reserved, [x.tolist() for x in p.pools])


def test_a_fork_with_the_pages_of_replays_to_come():
    d = decoder(reserve_ahead=60)
    captured(d, [130, 70, 20])                # pages for 191 positions: 3 blocks x 2 heads each
    d.resize(18)                              # as many as are in use
    captured(d, [130, 70, 20])
    d._reserved = 200                         # a fourth block for the replays to come
    d._replayed()
    was = snapshot(d)
    with pytest.raises(RuntimeError, match='out of pages'):
        d.fork(0, 1, 5)                       # nothing shared, 4 blocks of its own: 8 pages, 6 come back
    assert snapshot(d) == was
    sound(d.pool)
    d.fork(0, 1, 130)                         # 2 blocks shared, 2 of its own
    sound(d.pool)
    assert d.pool.nblk == [3, 4, 3] and d.pool.tokens == [130, 130, 20]


def test_pool_forks_are_whole_or_nothing():
    pool = new(pages=14)                      # B 3, H 2, leaf 4
    pool.ensure(12, seqs=[0])
    pool.ensure(8, seqs=[1])
    pool.ensure(8, seqs=[2])
    state = lambda: (pool.host.tolist(), pool.table.tolist(), list(pool.free), list(pool.refs), list(pool.nblk), list(pool.tokens))
    was = state()
    with pytest.raises(RuntimeError, match='out of pages'):
        pool.fork(0, 1, 10, t_end=24)         # 2 blocks shared, 4 of its own: 8 pages, 4 come back
    assert state() == was
    pool.fork(0, 1, 10, t_end=16)             # 2 of its own
    sound(pool)
    assert pool.nblk[1] == 4
    pool.fork(0, 1, 10, t_end=3)              # not past t: the block that t lies in
    sound(pool)
    assert pool.nblk[1] == 3


def test_replays_ask_again(monkeypatch):
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: None)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    d = decoder(reserve_ahead=4)
    captured(d, [62, 62, 62])
    d.resize(12)
    captured(d, [62, 62, 62])                 # 2 blocks each: full
    for _ in range(61):
        d.replay()
        d.g_t += 1
    d.pool.resize(12)
    for _ in range(3):
        d.replay()
        d.g_t += 1
    assert d._t_host == 126
    was = snapshot(d)
    for _ in range(3):
        with pytest.raises(RuntimeError, match='out of pages'):
            d.replay()
        assert snapshot(d) == was
    d.pool.resize(40)
    d.replay()
    assert d._t_host == 127 and d._reserved > 128


def test_a_capture_that_finds_too_few_pages(monkeypatch):
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    d = decoder(reserve_ahead=4)
    d.pool.resize(12)
    captured(d, [62, 62, 62])
    d._replayed()
    d.g_tok = torch.tensor([1, 2, 3])
    was, tok, graph = snapshot(d), d.g_tok, d.graph
    with pytest.raises(RuntimeError, match='out of pages'):
        d.capture(torch.tensor([4, 5, 6]), 140)
    assert snapshot(d) == was and d.g_tok is tok and d.graph is graph
