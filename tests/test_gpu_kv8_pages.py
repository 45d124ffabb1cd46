"""Positions of an 8-bit cache without a page: nothing is stored or formed for them, the gate's log sums and gated vectors
among it.  GPU only."""
import pytest
import torch

from treeattn_amd import kernels as K
from treeattn_amd.config import Config
from treeattn_amd.engine import PagePool, SegState

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def rnd(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def state(cfg, B, H, dh, Tcap, t_end, dtype=torch.bfloat16, cache='e4m3'):
    pool = PagePool(B, H, dh, cfg.leaf, Tcap, B * H * (Tcap // cfg.leaf), 1, dtype, DEV, cache=cache)
    pool.ensure(t_end)
    return SegState(cfg, Tcap, H, dh, DEV, B, dtype, pages=pool)


def node_arrays(st):
    return [t for t in st.levels + st.lg + st.gl if t is not None]


@pytest.mark.parametrize('dtype,dh,leaf', [(torch.bfloat16, 64, 8), (torch.float32, 128, 4), (torch.float16, 16, 16)])
@pytest.mark.parametrize('part', [False, True])
def test_gate_forms_nothing_without_a_page(dtype, dh, leaf, part):
    """Tokens past the pages leave every node array as it was, as the pages in the model's type do; with pages for one of the
    sequences the other goes on."""
    cfg = Config(leaf=leaf, wmax=4, beam=4, neighbors=False, gate=True)
    B, H, Tcap, have = 2, 2, 8 * leaf, 3 * leaf
    sts = [state(cfg, B, H, dh, Tcap, have, dtype, cache) for cache in ('e4m3', None)]
    for st in sts:
        if part:
            st.pages.ensure(Tcap, [1])
        for t in range(have):
            st.add(t, rnd(B, H, dh, seed=t, dtype=dtype), rnd(B, H, dh, seed=100 + t, dtype=dtype))
    before = [[t.clone() for t in node_arrays(st)] for st in sts]
    pool = sts[0].cache8.pool.view(torch.uint8).clone()
    for st in sts:
        for t in range(have, Tcap):
            st.add(t, rnd(B, H, dh, seed=t, dtype=dtype), rnd(B, H, dh, seed=100 + t, dtype=dtype))
    now = [node_arrays(st) for st in sts]
    for a, b in zip(now[0], before[0]):
        assert torch.equal(a[0], b[0])
        if not part:
            assert torch.equal(a, b)
    assert torch.equal(sts[0].cache8.pool.view(torch.uint8), pool) == (not part)
    for a, b in zip(*now):
        assert torch.equal(a, b)


def test_gate_over_views_and_positions_of_their_own():
    """Part of the sequences, each at its own position, some outside the cache: the nodes of the whole state's sequences."""
    cfg = Config(leaf=4, wmax=4, beam=4, neighbors=False, gate=True, arity=4)
    B, H, dh, Tcap = 4, 3, 32, 64
    a, b = state(cfg, B, H, dh, Tcap, Tcap), state(cfg, B, H, dh, Tcap, Tcap)
    view = b.rows(1, 3)
    for i in range(40):
        k, v = rnd(B, H, dh, seed=i), rnd(B, H, dh, seed=100 + i)
        t = torch.tensor([-1, i, i + 3 if i >= 24 else i, 70], dtype=torch.int32, device=DEV)
        a.append(k, v, t)
        a.gate_append(t)
        view.append(k[1:3], v[1:3], t[1:3].contiguous())
        view.gate_append(t[1:3].contiguous())
    for x, y in zip(node_arrays(a), node_arrays(b)):
        assert torch.equal(x, y)
    assert any(x[1].any() for x in a.gl if x is not None) and not any(x[[0, 3]].any() for x in node_arrays(a))


def test_gate_refusals():
    cfg = Config(leaf=8, wmax=4, beam=4, neighbors=False, gate=True)
    st = state(cfg, 1, 1, 32, 64, 64)
    t = torch.zeros(1, dtype=torch.int32, device=DEV)
    args = [st.levels, st.lg, st.gl, st.shape.blevels, st.shape.arity, 0.5]
    with pytest.raises(ValueError, match='positions'):
        K.gate_append(st.cache8, t.long(), *args)
    with pytest.raises(ValueError, match='levels'):
        K.gate_append(st.cache8, t, [x[:, :, :1] for x in st.levels], *args[1:])
    with pytest.raises(RuntimeError, match='leaf blocks'):
        K.gate_append(st.cache8, t, *args[:3], [b + 1 for b in st.shape.blevels], *args[4:])


@pytest.mark.parametrize('T', [5, 16, 21])
def test_released_sequence_is_forgotten(T):
    """After PagePool.release a sequence has no row, in no layer, in the middle of a block as at its end; the others keep theirs,
    and the slot's next sequence is that of a new cache."""
    cfg = Config(leaf=8, wmax=4, beam=4, neighbors=False)
    B, H, dh, Tcap = 3, 2, 32, 64
    pool = PagePool(B, H, dh, 8, Tcap, B * H * 8, 2, torch.bfloat16, DEV, cache='e4m3')
    pool.ensure(Tcap)
    sts = [SegState(cfg, Tcap, H, dh, DEV, B, torch.bfloat16, pages=pool, layer=i) for i in range(2)]
    part = sts[1].rows(1, 3)
    for t in range(T):
        for i, st in enumerate(sts):
            st.add(t, rnd(B, H, dh, seed=t + 50 * i), rnd(B, H, dh, seed=200 + t + 50 * i))
    kept = [[x.clone() for b in (0, 2) for x in st.dense_kv(b, T)] for st in sts]
    pool.release(1)
    for st in sts:
        assert not any(x.any() for x in st.dense_kv(1, T))
        assert not any(x[1].any() for x in st.row(T - 1))
    assert not any(x.any() for x in part.dense_kv(0, T))
    for st, old in zip(sts, kept):
        assert all(torch.equal(x, y) for x, y in zip([x for b in (0, 2) for x in st.dense_kv(b, T)], old))
    q = rnd(B, H, 1, dh, seed=9)
    ids = torch.zeros(B, H, 1, 1, dtype=torch.int32, device=DEV)
    tq = torch.full((B, 1), T - 1, dtype=torch.int32, device=DEV)
    lse = torch.empty(B, H, 1, device=DEV)
    for st in sts:
        for nsplit in (1, 4, 8):
            out, _, _ = K.seg_attn8(q, st.cache8, tq, ids, torch.full_like(ids, T > 8, dtype=torch.bool), None, 3, 0.2, lse=lse,
                                    nsplit=nsplit)
            assert not out[1].any() and (lse[1] == -1e30).all() and out[0].any() and (lse[0] > -1e30).all()
    pool.ensure(Tcap, [1])
    new = state(cfg, 1, H, dh, Tcap, Tcap)
    for t in range(11):
        k, v = rnd(B, H, dh, seed=400 + t), rnd(B, H, dh, seed=500 + t)
        at = torch.tensor([-1, t, -1], dtype=torch.int32, device=DEV)
        sts[0].append(k, v, at)
        new.append(k[1:2], v[1:2], at[1:2].contiguous())
    for x, y in zip(sts[0].dense_kv(1, 11), new.dense_kv(0, 11)):
        assert torch.equal(x, y)


def test_fill_takes_any_layout():
    """A prompt's rows off a 16-byte boundary, values with the head size not innermost (keys have it there for their node sums, in
    every cache), rows shared by the heads: the cache that a contiguous copy gives."""
    cfg = Config(leaf=8, wmax=4, beam=4, neighbors=False, gate=True)
    B, H, dh, T = 2, 3, 16, 21
    wide = rnd(B, H, T, dh + 1, seed=1)
    turned = rnd(B, H, dh, T, seed=2).transpose(2, 3)
    shared = rnd(B, 1, T, dh, seed=3).expand(B, H, T, dh)
    odd = rnd(B * H * T * dh + 1, seed=4)[1:].view(B, H, T, dh)
    for k, v in ((wide[..., 1:], wide[..., :dh]), (shared, turned), (odd, odd), (odd.float(), wide[..., 1:])):
        a, b = state(cfg, B, H, dh, 64, 0), state(cfg, B, H, dh, 64, 0)
        a.fill(k, v)
        b.fill(k.contiguous().clone(), v.contiguous().clone())
        assert torch.equal(a.cache8.pool.view(torch.uint8), b.cache8.pool.view(torch.uint8))
        for x, y in zip(a.dense_kv(1, T) + tuple(node_arrays(a)), b.dense_kv(1, T) + tuple(node_arrays(b))):
            assert torch.equal(x, y)
