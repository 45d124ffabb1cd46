"""Infinities and NaN that the rows of a call see themselves (kernels.dense_attn): the elements that see them show them, all
others keep their bits, and a call takes a few times as long at most.  GPU only."""
import math

import pytest
import torch

from test_gpu_dense import BF16, DEV, F16, F32, paged, rnd, rows
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu
INF, NAN = float('inf'), float('nan')

# (dtype, D, sequences, heads, rows, positions, pages of, nsplit): rows of prompts by workgroups, split and not; by wavefronts
# (float32, small pages); one token split over workgroups
CASES = [(BF16, 64, 2, 12, 500, 600, 0, 1), (F16, 128, 4, 12, 300, 520, 64, 1), (BF16, 32, 1, 3, 200, 700, 32, 960),
         (BF16, 128, 2, 2, 130, 900, 0, 512), (F32, 64, 2, 2, 150, 300, 0, 1), (F32, 128, 1, 2, 100, 260, 8, 64),
         (F16, 64, 2, 3, 70, 400, 16, 1), (BF16, 64, 2, 3, 40, 400, 8, 4), (F16, 16, 1, 2, 33, 300, 2, 64),
         (BF16, 64, 2, 4, 1, 5000, 64, 256), (F32, 32, 1, 4, 1, 3000, 16, 64), (F16, 128, 2, 2, 1, 4000, 0, 128)]


def inputs(case):
    dtype, D, B, H, N, T, leaf, nsplit = case
    k, v, q = [rnd(B, H, n, D, seed=i, dtype=dtype) for i, n in ((1, T), (2, T), (3, N))]
    return q, k, v, rows([T - 3 * b for b in range(B)], N).to(DEV)


def call(case, q, k, v, tq):
    leaf, nsplit = case[6:]
    lse = torch.empty(q.shape[:3], device=DEV)
    c = (paged(k, v, leaf), None) if leaf else (k.to(DEV), v.to(DEV))
    out, _ = K.dense_attn(q.to(DEV), *c, tq, lse=lse, nsplit=nsplit)
    return out, lse


def same(a, b):
    """Bit for bit, NaN where NaN is."""
    return torch.equal(a.nan_to_num(7.5), b.nan_to_num(7.5)) and torch.equal(a.isnan(), b.isnan())


@pytest.mark.parametrize('case', CASES, ids=[str(i) for i in range(len(CASES))])
def test_values_that_rows_see(case):
    """Column by column: +inf, -inf, NaN near the start, seen by all rows; both infinities, the second seen by the later rows
    only; an infinity of some rows in the middle."""
    q, k, v, tq = inputs(case)
    D, N, T = case[1], case[4], case[5]
    clean, lse0 = call(case, q, k, v, tq)
    bad = v.clone()
    mid, late = T - 3 * (case[2] - 1) - (N + 1) // 2, T - 3 * (case[2] - 1) - max(1, N // 4)
    want = clean.clone()
    at = tq.view(-1, 1, N).expand(clean.shape[:3])
    for key, col, x in ((0, 1, INF), (1, 2, -INF), (0, 3, NAN), (2, 5, INF), (late, 5, -INF), (mid, 7, -INF), (mid, D - 1, NAN),
                        (0, D - 2, INF), (5, D - 2, INF)):
        bad[:, :, key, col] = x
        hit = at >= key
        now = want[..., col]       # (a second infinity of the other sign: NaN)
        want[..., col] = torch.where(hit, torch.where(now.isfinite(), torch.full_like(now, x), now + x), now)
    got, lse = call(case, q, k, bad, tq)
    assert same(got, want)
    assert torch.equal(lse, lse0)


@pytest.mark.parametrize('case', CASES, ids=[str(i) for i in range(len(CASES))])
def test_keys_and_queries_that_are_nan(case):
    """A NaN in a key reaches every element of the rows that see it, one in a query its own row."""
    q, k, v, tq = inputs(case)
    T, N = case[5], case[4]
    clean, _ = call(case, q, k, v, tq)
    key = T - 3 * (case[2] - 1) - (N + 1) // 2
    bad = k.clone()
    bad[:, 0, key, 3] = NAN
    got, lse = call(case, q, bad, v, tq)
    hit = (tq >= key).view(-1, 1, N).expand(clean.shape[:3]).clone()
    hit[:, 1:] = False
    assert bool(got[hit].isnan().all()) and bool(lse[hit].isnan().all()) and torch.equal(got[~hit], clean[~hit])
    q = q.clone()
    q[:, 1, N // 2, 0] = NAN
    got, lse = call(case, q, k, v, tq)
    hit = torch.zeros_like(hit)
    hit[:, 1, N // 2] = True
    assert bool(got[hit].isnan().all()) and bool(lse[hit].isnan().all()) and torch.equal(got[~hit], clean[~hit])


@pytest.mark.parametrize('dtype,D,leaf,N,nsplit', [(BF16, 64, 0, 300, 1), (BF16, 128, 64, 200, 512), (F32, 64, 8, 40, 1),
                                                   (F32, 32, 0, 5, 64), (BF16, 16, 2, 20, 4)])
def test_sums_that_pass_the_range(dtype, D, leaf, N, nsplit):
    """Values of the lowest number: sums of weights times them pass a float's range, their mean does not.  A mean of equal numbers:
    off by the rounding of the sums above and below, T 2^-24 each, and half a step of the result."""
    T = 700
    q, k = rnd(2, 12, N, D, seed=3, dtype=dtype), rnd(2, 12, T, D, seed=1, dtype=dtype)
    v = rnd(2, 12, T, D, seed=2, dtype=dtype)
    tq = rows([T, T - 9], N).to(DEV)
    case = (dtype, D, 2, 12, N, T, leaf, nsplit)
    clean, lse0 = call(case, q, k, v, tq)
    low = torch.finfo(dtype).min / 2
    v[..., 4] = low
    got, lse = call(case, q, k, v, tq)
    rel = 2 * T * 2.0 ** -24 + torch.finfo(dtype).eps / 2
    assert float((got[..., 4].double() / low - 1).abs().max()) <= rel
    other = torch.arange(D) != 4
    # the other columns of such rows: weights 2^-24 of the others', the maximum renewed at every step: sums in float32 as before
    d = (got[..., other].double() - clean[..., other].double()).abs()
    assert float(d.max()) <= (2 * torch.finfo(dtype).eps + 4 * T * 2.0 ** -24) * float(v[..., other].abs().max())
    assert float((lse - lse0).abs().max()) <= 1e-3


@pytest.mark.parametrize('dtype,N,T,leaf', [(BF16, 2048, 2048, 0), (F16, 1000, 1000, 64), (F32, 700, 700, 64), (BF16, 600, 600, 8),
                                            (BF16, 1, 30000, 64)])
def test_a_nan_near_the_start_costs_a_few_passes(dtype, N, T, leaf):
    """Every row of every set sees it: five passes over the keys (the later ones with fewer things at once), not one a row."""
    B, H, D = 2, 12, 64
    q, k, v = [rnd(B, H, n, D, seed=i, dtype=dtype) for i, n in ((3, N), (1, T), (2, T))]
    tq = rows([T, T], N).to(DEV)
    nsplit = 1 if N > 1 else 480

    def ms(v):
        c = (paged(k, v, leaf), None) if leaf else (k.to(DEV), v.to(DEV))
        x, ws = q.to(DEV), K.dense_attn_workspace(B, H, N, D, nsplit, DEV, H)
        times = []
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            out, _ = K.dense_attn(x, *c, tq, nsplit=nsplit, ws=ws)
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times[1:]), out
    t0, clean = ms(v)
    v[:, :, 0, 5] = NAN
    t1, got = ms(v)
    print('%s %d rows: %.3f -> %.3f ms' % (dtype, N, t0, t1))
    assert bool(got[..., 5].isnan().all())
    other = torch.arange(D) != 5
    assert torch.equal(got[..., other], clean[..., other])
    assert t1 <= 12 * t0 + 0.05
