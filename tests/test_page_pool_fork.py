"""Shared, copied and moved pages of the decoder's page pool, and what the new C entry points refuse (CPU tensors: no kernel
runs)."""
import ctypes
import random

import pytest
import torch

from treeattn_amd.engine import PagePool


def new(B=3, H=2, leaf=4, Tcap=32, pages=40, layers=2, cache=None):
    return PagePool(B, H, 4, leaf, Tcap, pages, layers, torch.float32, 'cpu', cache)


def write(pool, b, t, value):
    """What a step writes: row t of every layer and head, through the device's table."""
    for i, x in enumerate(pool.pools):
        for h in range(pool.H):
            p = int(pool.table[b, h, t // pool.leaf])
            assert p >= 0 and pool.refs[p] == 1, 'a step writes into a page of its own'
            x[p, :, t % pool.leaf] = value + 100 * i + 1000 * h


def rows(pool, b, n):
    """Positions 0 .. n-1 as they are read."""
    out = []
    for x in pool.pools:
        pg = pool.table[b, :, :(n + pool.leaf - 1) // pool.leaf].long()
        out.append(x[pg][:, :, 0, :, 0].reshape(pool.H, -1)[:, :n].clone())
    return torch.stack(out)


def sound(pool):
    """Counts, free list and tables agree."""
    seen = [0] * pool.P
    for b in range(pool.B):
        assert torch.equal(pool.table[b], pool.host[b])
        assert bool((pool.host[b, :, pool.nblk[b]:] == -1).all())
        for p in pool.host[b, :, :pool.nblk[b]].reshape(-1).tolist():
            seen[p] += 1
    assert seen == pool.refs
    assert sorted(pool.free) == [p for p in range(pool.P) if seen[p] == 0]
    assert pool.n_shared == sum(c > 1 for c in seen)


def test_fork_shares_whole_blocks_and_copies_the_rest():
    pool = new()
    pool.ensure(11, seqs=[0])
    for t in range(11):
        write(pool, 0, t, t)
    before = rows(pool, 0, 11)
    pool.fork(0, 1, 10)                      # blocks 0 and 1 shared, rows 8 and 9 of block 2 copied
    sound(pool)
    assert torch.equal(pool.table[1, :, :2], pool.table[0, :, :2]) and not torch.equal(pool.table[1, :, 2], pool.table[0, :, 2])
    assert torch.equal(rows(pool, 1, 10), before[..., :10])
    write(pool, 1, 10, -5)                   # both go on
    write(pool, 0, 11, 70)
    assert torch.equal(rows(pool, 0, 11), before)
    pool.fork(1, 2, 8)                       # ends with a block: nothing copied
    sound(pool)
    assert len([p for p in pool.refs if p == 3]) == 4
    pool.release(0)
    sound(pool)
    assert torch.equal(rows(pool, 2, 8), before[..., :8]) and torch.equal(rows(pool, 1, 10), before[..., :10])
    pool.fork(1, 2, 0)                       # nothing taken: an empty sequence
    sound(pool)
    assert pool.nblk[2] == 0
    pool.release(1)
    sound(pool)
    assert len(pool.free) == pool.P


def test_going_back_takes_a_page_of_ones_own():
    pool = new()
    pool.ensure(12, seqs=[0])
    for t in range(12):
        write(pool, 0, t, t)
    before = rows(pool, 0, 12)
    pool.fork(0, 1, 12)
    pool.ensure(6, seqs=[1], start=[5])      # goes back to position 5, in a shared block
    sound(pool)
    write(pool, 1, 5, 55)
    assert torch.equal(rows(pool, 0, 12), before)
    got = rows(pool, 1, 12)
    assert torch.equal(got[..., 6:], before[..., 6:]) and torch.equal(got[..., :5], before[..., :5])
    assert not torch.equal(got[..., 5], before[..., 5])
    pool.own(0, 0)                           # the rest of what is shared
    sound(pool)
    assert pool.n_shared == 0 and torch.equal(rows(pool, 0, 12), before)


def test_resize_moves_what_is_in_use():
    for cache in (None, 'e4m3'):
        pool = new(pages=30, cache=cache)
        pool.ensure(9, seqs=[0])
        pool.ensure(4, seqs=[2])
        if cache is None:
            for t in range(9):
                write(pool, 0, t, t)
            for t in range(4):
                write(pool, 2, t, 40 + t)
        else:
            for i, s in enumerate(pool.scales):
                s.copy_(torch.arange(60.).view(30, 2) + 100 * i)
        pool.fork(0, 1, 8)
        table = pool.table
        want = [rows(pool, b, n) for b, n in ((0, 9), (1, 8), (2, 4))] if cache is None else \
            [[s[pool.table[b, :, :2].long().clamp(min=0)].clone() for s in pool.scales] for b in range(3)]
        for P in (8, 50, 9):
            pool.resize(P)
            sound(pool)
            assert pool.table is table and all(x.shape[0] == P for x in pool._tensors())
            got = [rows(pool, b, n) for b, n in ((0, 9), (1, 8), (2, 4))] if cache is None else \
                [[s[pool.table[b, :, :2].long().clamp(min=0)].clone() for s in pool.scales] for b in range(3)]
            for b in range(3):
                n = pool.nblk[b]
                for x, y in zip(got[b], want[b]):
                    assert torch.equal(x, y) if cache is None else torch.equal(x[:, :min(n, 2)], y[:, :min(n, 2)])
        used = sorted(p for p in range(pool.P) if pool.refs[p])
        assert used == list(range(8))
        with pytest.raises(RuntimeError, match='8 pages are in use'):
            pool.resize(7)
        sound(pool)


def test_refusals_change_nothing():
    pool = new(pages=14)
    pool.ensure(10, seqs=[0])                # 3 blocks x 2 heads
    pool.ensure(8, seqs=[1])                 # 2 x 2
    pool.ensure(8, seqs=[2])
    sound(pool)
    for bad in ((0, 0, 4), (0, 3, 4), (-1, 1, 4), (0, 1, 13), (0, 1, -1), (1, 0, 9)):
        with pytest.raises(ValueError):
            pool.fork(*bad)
    sound(pool)
    pool.fork(0, 1, 9)                       # 1's own pages come back first: enough
    sound(pool)
    pool = new(pages=6)
    pool.ensure(10, seqs=[0])
    with pytest.raises(RuntimeError, match='out of pages'):
        pool.fork(0, 1, 10)
    sound(pool)
    pool.fork(0, 1, 8)                       # shared only: no page needed
    sound(pool)
    with pytest.raises(RuntimeError, match='out of pages'):
        pool.own(1, 0)
    sound(pool)


def test_any_order_of_calls():
    """Random forks, steps, steps back, releases and sizes against plain lists of what each sequence holds."""
    rng = random.Random(7)
    pool = new(B=4, leaf=4, Tcap=40, pages=120)
    held = [[] for _ in range(4)]
    for i in range(600):
        b = rng.randrange(4)
        what = rng.choice(['step', 'step', 'step', 'step', 'back', 'fork', 'release', 'resize'])
        if what == 'step' and len(held[b]) < 40:
            pool.ensure(len(held[b]) + 1, seqs=[b], start=[len(held[b])])
            write(pool, b, len(held[b]), i)
            held[b].append(i)
        elif what == 'back' and held[b]:
            t = rng.randrange(len(held[b]))
            pool.ensure(t + 1, seqs=[b], start=[t])
            write(pool, b, t, i)
            held[b][t] = i
        elif what == 'fork':
            d = (b + rng.randint(1, 3)) % 4
            t = rng.randint(0, len(held[b]))
            pool.fork(b, d, t)
            held[d] = held[b][:t]
        elif what == 'release':
            pool.release(b)
            held[b] = []
        elif what == 'resize' and rng.random() < 0.3:
            pool.resize(rng.randint(80, 140))
        sound(pool)
        for k in range(4):
            if held[k]:
                assert rows(pool, k, len(held[k]))[1, 1].tolist() == [x + 1100 for x in held[k]]


def test_entry_points_refuse_on_the_host():
    """Bad sizes, strides and pointers come back as an error before anything is launched."""
    from treeattn_amd import _lib
    L = _lib.lib()
    one = ctypes.c_void_p(4096)              # never dereferenced
    i64 = lambda *v: (ctypes.c_int64 * len(v))(*v)
    ptrs = lambda *v: (ctypes.c_void_p * len(v))(*v)

    def attn(q=one, k=one, v=one, dt=2, strides=None, B=1, Hq=4, H=2, Nq=1, D=64, Tk=100, tq=one, out=one, nsplit=1, ws=None,
             ws_bytes=0, pages=None):
        st = strides or [256, 64, 64] + [12800, 6400, 64] * 2
        return L.ta_dense_attn_fwd(q, k, v, dt, *st, B, Hq, H, Nq, D, Tk, tq, 1, 0.1, out, 256, 64, 64, None, nsplit, ws,
                                   ws_bytes, pages, None)
    bad = [(dict(dt=3), b'dtype'), (dict(D=48), b'head dim'), (dict(Hq=3), b'multiple'), (dict(Tk=0), b'bad sizes'),
           (dict(H=0), b'bad sizes'), (dict(Nq=-1), b'bad sizes'), (dict(nsplit=3), b'nsplit'), (dict(nsplit=8196), b'nsplit'),
           (dict(nsplit=0), b'nsplit'), (dict(q=None), b'missing'), (dict(tq=None), b'missing'), (dict(out=None), b'missing'),
           (dict(q=ctypes.c_void_p(4098)), b'aligned'), (dict(strides=[256, 64, 64, 12800, 6400, 60, 12800, 6400, 64]), b'aligned'),
           (dict(nsplit=8), b'workspace'), (dict(nsplit=8, ws=one, ws_bytes=1), b'workspace'),
           (dict(nsplit=8, ws=ctypes.c_void_p(4100), ws_bytes=1 << 30), b'workspace'),
           (dict(strides=[256, 64, 64, 1 << 40, 1 << 39, 1 << 25, 12800, 6400, 64]), b'row strides'),
           (dict(pages=ctypes.byref(_lib.KvPages(None, 1, 1, 8192, 4, 6))), b'page'),
           (dict(pages=ctypes.byref(_lib.KvPages(4096, 1, 1, 8192, 0, 6))), b'page'),
           (dict(pages=ctypes.byref(_lib.KvPages(4096, 1, 1, 8192, 4, 0))), b'page')]
    for kw, word in bad:
        assert attn(**kw) != 0, kw
        assert word in L.ta_last_error(), (kw, L.ta_last_error())
    assert attn(B=0) == 0 and attn(Nq=0) == 0
    size = L.ta_dense_attn_workspace_size
    assert size(2, 4, 2, 1, 64, 1) == size(2, 4, 2, 1, 64, 4) == 0
    assert size(2, 4, 2, 1, 64, 8) >= 4 * 4 + (4 + 2) * 16 * 66 * 4
    assert size(2, 4, 2, 40, 64, 64) >= 2 * 2 * 3 * 4 + (2 * 2 * 3 + 16) * 32 * 66 * 4

    def rope(x=one, dt=2, D=64, rot=64, turns=one, pos=one, H=2):
        return L.ta_rope(x, dt, 128, 64, 128, one, 128, 64, 128, 1, H, 5, D, rot, turns, 0, 1.0, 0, pos, 0, None)
    for kw in (dict(dt=7), dict(rot=63), dict(rot=66), dict(rot=-2), dict(turns=None), dict(turns=ctypes.c_void_p(4100)),
               dict(pos=None), dict(x=None), dict(D=0, rot=0), dict(H=-1)):
        assert rope(**kw) != 0, kw
        assert b'ta_rope' in L.ta_last_error()
    assert rope(H=0) == 0

    def store(k=one, Hq=0, q=None, q_out=None, Tcap=64, rot=0, turns=None, pages=None, H=2):
        return L.ta_kv_store(k, one, 2, 1, 1, 1, 1, 1, 1, q, 1, 1, 1, q_out, 1, 1, 1, Hq, one, one, 1, 1, 64, 1, H, 1, 64, Tcap,
                             one, 0, rot, turns, 0, 1.0, pages, None)
    for kw in (dict(k=None), dict(Hq=2), dict(Hq=2, q=one), dict(Tcap=0), dict(rot=2), dict(H=0),
               dict(pages=ctypes.byref(_lib.KvPages(4096, 1, 1, 64, 4, 6))), dict(pages=ctypes.byref(_lib.KvPages(None, 1, 1, 8192, 4, 6)))):
        assert store(**kw) != 0, kw
        assert b'ta_kv_store' in L.ta_last_error()

    def copy(n=1, fr=ptrs(4096), to=ptrs(8192), size=i64(64), a=i64(4), b=i64(4), src=one, dst=one, pairs=1):
        return L.ta_copy_rows(n, fr, to, size, a, b, src, dst, pairs, None)
    for kw in (dict(n=-1), dict(pairs=-1), dict(src=None), dict(dst=None), dict(fr=None), dict(size=None), dict(size=i64(-1)),
               dict(a=i64(-1)), dict(fr=ptrs(None)), dict(to=ptrs(None))):
        assert copy(**kw) != 0, kw
        assert b'ta_copy_rows' in L.ta_last_error()
    assert copy(pairs=0) == 0 and copy(n=0, fr=None, to=None, size=None, a=None, b=None) == 0
