"""A step makes its own the one block of each sequence that it writes: no copies of blocks between a sequence's position and the
longest one's, no pages wanted for them.  CPU: bookkeeping, the step's kernels have stand-ins."""
import time

import pytest
import torch

from test_fork_of_written_positions import decoder
from test_page_pool_fork import new, sound


def test_only_what_is_written_is_owned():
    pool = new(B=3, Tcap=32, pages=22)           # H 2, leaf 4
    pool.ensure(32, seqs=[0])
    pool.wrote(32)
    pool.fork(0, 1, 28)
    pool.fork(0, 2, 28)
    pool.ensure(29, [1], start=[5], stop=[6])    # 2 of the 6 pages left for block 1, 2 for the block of position 28
    sound(pool)
    assert pool.n_shared == 14 and pool.nblk[1] == 8 and len(pool.free) == 2
    pool.ensure(29, [1], start=[9], stop=[9])    # nothing to write
    pool.ensure(7, [1], start=[-3], stop=[1])
    sound(pool)
    assert len(pool.free) == 0
    with pytest.raises(RuntimeError, match='out of pages'):
        pool.ensure(29, [1], start=[8])
    sound(pool)


def test_a_step_of_ragged_sequences(monkeypatch):
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    d = decoder()
    monkeypatch.setattr(type(d), '_forward_step', lambda self, tok, tpos: torch.zeros(self.B, 11))
    monkeypatch.setattr(type(d), 'keys_read', lambda self: torch.zeros(self.B))
    d.step(torch.zeros(3, dtype=torch.long), 200)
    d.fork(0, 1, 200)
    d.fork(0, 2, 130)
    d.resize(sum(r > 0 for r in d.pool.refs) + 4)   # for the block that 1 writes, and 2's up to the longest
    d.step(torch.zeros(3, dtype=torch.long), torch.tensor([200, 70, 130]))
    sound(d.pool)
    assert d.pool.n_shared == 6                     # blocks 0 to 2 by 2 heads (1 is 0's and 2's)
    assert len(d.pool.free) == 0 and d.pool.tokens == [201, 200, 131]


def test_the_host_looks_at_the_block_alone():
    """Eight sequences, one far behind, nothing of it shared: what a step asks for takes some microseconds a sequence (25 ms and
    more when every block between was looked at)."""
    pool = new(B=8, H=12, leaf=64, Tcap=32768, pages=8 * 12 * 512, layers=1)
    pool.ensure(32768)
    pool.fork(0, 1, 64)
    pool.ensure(32768)
    at = [100] + [32767] * 7
    best = 1.0
    for _ in range(5):
        t0 = time.perf_counter()
        pool.ensure(32768, start=at, stop=[t + 1 for t in at])
        best = min(best, time.perf_counter() - t0)
    assert best < 3e-3, best
