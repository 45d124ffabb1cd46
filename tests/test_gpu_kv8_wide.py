"""Attention over the 8-bit cache with long leaf lists (beyond a wavefront's 64, up to the 512 allowed) and neighbour leaves beside
them, and with the whole neighbour list.  GPU only."""
import pytest
import torch

from test_gpu_kv8 import BF16, F16, F32, check, filled, leaves_for, rnd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,D,leaf,wl,T', [(BF16, 64, 2, 512, 1100), (F32, 16, 2, 300, 900), (F16, 128, 4, 130, 700),
                                               (BF16, 32, 16, 65, 1300), (F16, 64, 2, 128, 250)])
@pytest.mark.parametrize('S', [0, 5, 64])
def test_long_lists(dtype, D, leaf, wl, T, S):
    """Budgets of nothing, part of a wavefront's share, its end and past it; neighbours that repeat listed blocks (within the
    first 64 and beyond), each other, the own block and the one in the tail."""
    B, H, Nq = 2, 2, 2
    n = [T, T - leaf - 1]
    c, o, kmax, vmax = filled(B, H, D, leaf, 2048, n, dtype, seed=wl)
    tq = torch.tensor(n).view(B, 1) - Nq + torch.arange(Nq)
    ids, vld = leaves_for(tq, B, H, wl, leaf, seed=3)
    nt = torch.tensor([[[0, 63], [64, 65]], [[wl - 1, wl], [wl // 2, wl + 7]]])
    nb = None
    if S:
        g = torch.Generator().manual_seed(S)
        nid = torch.randint(0, T // leaf + 2, (B, H, Nq, S), generator=g, dtype=torch.int32)
        ok = torch.rand(B, H, Nq, S, generator=g) < 0.8
        nid[..., 0] = ids[..., 0]
        nid[..., 1] = ids[..., min(wl, int(vld.sum(-1).min())) - 1]
        nid[..., 2] = nid[..., 3]
        nid[..., 4] = (tq // leaf).view(B, 1, Nq)
        nb = nid, ok
    for nsplit in (1, 4, 64):
        check(c, o, rnd(B, H, Nq, D, seed=1, dtype=dtype), tq, ids, vld, nt, 3, kmax, vmax, nsplit, nb=nb)
