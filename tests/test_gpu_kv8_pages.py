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
