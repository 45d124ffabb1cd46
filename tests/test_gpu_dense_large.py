"""Attention over caches larger than the last-level cache, whose rows are read by other loads (kernels.dense_attn), against its
formula in float64.  GPU only."""
import math

import pytest
import torch

from test_gpu_dense import BF16, DEV, F16, F32, close
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype,D,H,G,T,leaf', [
    (BF16, 64, 2, 1, 600001, 64), (BF16, 64, 2, 3, 530000, 8), (BF16, 128, 2, 1, 300001, 0), (BF16, 32, 4, 16, 590000, 0),
    (BF16, 16, 8, 1, 540000, 2), (F16, 64, 2, 2, 530001, 0), (F16, 128, 1, 4, 530002, 16), (F16, 32, 4, 1, 530000, 64),
    (F32, 64, 2, 1, 263001, 16), (F32, 64, 2, 5, 270000, 64), (F32, 128, 1, 1, 270000, 4), (F32, 32, 4, 1, 270001, 0),
    (F32, 16, 4, 2, 530000, 32)])
def test_long_sequences_beside_short_ones(dtype, D, H, G, T, leaf):
    """256 MiB of keys and values and more in the first sequence, the others of some tokens and of one, a row outside.  Tolerance
    as derived in test_gpu_dense.want64, but for the sums: with 4 x 24 runs of keys a set or more, a sum is of T / 96 products
    and some hundred joined, n of them in all (off by n 2^-24)."""
    g = torch.Generator(device=DEV).manual_seed(D + T)
    lens = [T, 70, 1, 0]
    B, nsplit, scale = len(lens), 1024, 1 / math.sqrt(D)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)
    q, seq = randn(B, G * H, 1, D), [(randn(H, n, D), randn(H, n, D)) for n in lens]
    if leaf:
        nb = (T + leaf - 1) // leaf
        need = [(n + leaf - 1) // leaf for n in lens]
        ids = torch.randperm(sum(need) * H + 5, device=DEV, generator=g).to(torch.int32)
        pool = torch.full((len(ids), 2, leaf, D), float('nan'), dtype=dtype, device=DEV)
        table, at = torch.full((B, H, nb), -1, dtype=torch.int32, device=DEV), 0
        for b, n in enumerate(need):
            table[b, :, :n] = ids[at:at + n * H].view(H, n)
            at += n * H
            for i, x in enumerate(seq[b]):
                pad = torch.zeros(H, n * leaf, D, dtype=dtype, device=DEV)
                pad[:, :lens[b]] = x
                pool[table[b, :, :n].long(), i] = pad.view(H, n, leaf, D)
        cache = K.PagedCache(pool, table, T), None
    else:
        cache = [torch.full((B, H, T, D), float('nan'), dtype=dtype, device=DEV) for _ in range(2)]
        for b, n in enumerate(lens):
            for c, x in zip(cache, seq[b]):
                c[b, :, :n] = x
    tq = torch.tensor([[n - 1] for n in lens], dtype=torch.int32, device=DEV)
    lse = torch.empty(B, G * H, 1, device=DEV)
    ws = K.dense_attn_workspace(B, G * H, 1, D, nsplit, DEV, H)
    outs = [K.dense_attn(q, *cache, tq, scale, lse=lse, nsplit=nsplit, ws=ws)[0] for _ in range(2)]
    assert torch.equal(*outs)
    assert not outs[0][3].any() and bool((lse[3] == -1e30).all())
    u = 2.0 ** -24
    for b, n in enumerate(lens[:3]):
        for h in range(G * H):
            k, v, x = seq[b][0][h // G].double(), seq[b][1][h // G].double(), q[b, h, 0].double()
            s = (k * x).sum(-1) * scale
            want = (torch.softmax(s, 0)[:, None] * v).sum(0)
            e = (D + 2) * u * float((k.abs() * x.abs()).sum(-1).max()) * scale
            rel = 2 * e + 3 * u * float(s.abs().max()) + (8 + n / 96 + 500) * u
            tol = 2 * rel * float(v.abs().max())
            close(outs[0][b, h, 0], want.cpu(), torch.full((D,), tol, dtype=torch.float64), dtype)
            assert abs(float(lse[b, h, 0].double() - torch.logsumexp(s, 0))) <= rel + 1e-6 * (1 + abs(float(lse[b, h, 0])))
