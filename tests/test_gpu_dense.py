"""Attention over a whole decode cache (kernels.dense_attn) against its formula in float64.  GPU only."""
import math

import pytest
import torch

from treeattn_amd import kernels as K
from treeattn_amd.engine import decode_nsplit_dense

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rnd(*shape, seed, dtype=F32, spread=0.5):
    """Values as projections give them: some dimensions larger than others."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    return (x * torch.exp(spread * torch.randn(shape[-1], generator=g))).to(dtype)


def paged(k, v, leaf, seed=0, spare=3, fill=None, missing=()):
    """A PagedCache with the rows k, v (B,H,T,D), its pages in a scrambled order; `fill`: what rows that belong to no position
    hold; `missing`: (b, h, block) without a page."""
    B, H, T, D = k.shape
    nb = (T + leaf - 1) // leaf
    P = B * H * nb + spare
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(P, generator=g)[:B * H * nb].to(torch.int32).view(B, H, nb).contiguous()
    pool = torch.full((P, 2, leaf, D), 0.0 if fill is None else fill, dtype=k.dtype)
    for i, x in enumerate((k, v)):
        pad = torch.full((B, H, nb * leaf, D), 0.0 if fill is None else fill, dtype=k.dtype)
        pad[:, :, :T] = x
        pool[table.long(), i] = pad.view(B, H, nb, leaf, D)
    for m in missing:
        table[m] = -1
    return K.PagedCache(pool.to(DEV), table.to(DEV), T)


def want64(q, k, v, tq, scale, have=None):
    """(out, lse, tolerance) in float64 on the CPU: q (B,Hq,N,D), k, v (B,H,T,D), tq (B,N), have (B,H,T) or None.

    The tolerance, for float32 sums in any order and weights e^x good to 8 steps of 2^-24: with u = 2^-24 and S_j = scale
    sum_d |q_d k_jd|, a score is off by at most e = (D + 2) u max S, and the difference to the maximum, taken in float32, by u
    max |s| more on each side; a weight is then off by a factor within 1 +- (2 e + 3 u max|s| + 8 u), numerator and sum by n u
    more, so the result by at most twice their sum times max |v|.  Rows in 16 bits: the result is rounded, half a step."""
    B, Hq, N, D = q.shape
    H, T = k.shape[1], k.shape[2]
    G = Hq // H
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64)
    lse = torch.full((B, Hq, N), -1e30, dtype=torch.float64)
    tol = torch.zeros(B, Hq, N, 1, dtype=torch.float64)
    u = 2.0 ** -24
    for b in range(B):
        for h in range(Hq):
            for n in range(N):
                t = int(tq[b, n])
                if t < 0 or t >= T:
                    continue
                on = torch.arange(T) <= t
                if have is not None:
                    on &= have[b, h // G]
                if not on.any():
                    continue
                kk, vv, x = k[b, h // G][on].double(), v[b, h // G][on].double(), q[b, h, n].double()
                s = (kk * x).sum(-1) * scale
                lse[b, h, n] = torch.logsumexp(s, 0)
                out[b, h, n] = (torch.softmax(s, 0)[:, None] * vv).sum(0)
                e = (D + 2) * u * float((kk.abs() * x.abs()).sum(-1).max()) * scale
                rel = 2 * e + 3 * u * float(s.abs().max()) + 8 * u + len(s) * u
                tol[b, h, n] = 2 * rel * float(vv.abs().max())
    return out, lse, tol


def close(got, want, tol, dtype):
    half = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    d = (got.double().cpu() - want).abs()
    bound = tol + half * (want.abs() + tol) + 1e-12
    if dtype == F16:
        bound = bound + 2.0 ** -25      # half a step of the smallest numbers
    assert bool((d <= bound).all()), 'off by %.3g of %.3g' % (float((d - bound).max()), float(want.abs().max()))


def rows(lens, N):
    """Positions (B, N) of the last N tokens of sequences of `lens` tokens."""
    return (torch.tensor(lens).view(-1, 1) - N + torch.arange(N)).to(torch.int32)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('D,leaf,H,G,N', [(64, 64, 3, 1, 1), (128, 16, 2, 4, 1), (32, 2, 2, 1, 3), (16, 8, 1, 8, 5),
                                          (64, 4, 2, 2, 9), (128, 128, 1, 1, 33), (64, 32, 1, 3, 17), (16, 2, 2, 1, 1)])
@pytest.mark.parametrize('nsplit', [1, 4, 12, 64])
def test_paged(dtype, D, leaf, H, G, N, nsplit):
    lens = [1, 70, 333, 257]
    lens = [max(n, 1) for n in lens]
    B, T = len(lens), 340
    k, v = rnd(B, H, T, D, seed=1, dtype=dtype), rnd(B, H, T, D, seed=2, dtype=dtype)
    q = rnd(B, G * H, N, D, seed=3, dtype=dtype)
    c = paged(k, v, leaf, seed=D, fill=float('nan'))
    tq = rows(lens, N)                       # the first sequence's earlier tokens lie before position 0: no keys
    scale = 1 / math.sqrt(D)
    lse = torch.empty(B, G * H, N, device=DEV)
    out, _ = K.dense_attn(q.to(DEV), c, None, tq.to(DEV), scale, lse=lse, nsplit=nsplit)
    want, wl, tol = want64(q, k, v, tq, scale)
    close(out, want, tol, dtype)
    assert torch.equal(lse.cpu() == -1e30, wl == -1e30)
    # log of the sum: off by the weights' and scores' relative error, taken relative to max |v| in tol
    ok = wl > -1e29
    assert bool(((lse.cpu().double() - wl).abs()[ok] <= (tol[..., 0][ok] / 2 + 1e-6 * (1 + wl[ok].abs())) + 1e-5).all())


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('t', [0, 1, 2, 15, 16, 30, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 300, 511])
def test_every_length_near_a_tile(dtype, t):
    B, H, D, T = 1, 2, 64, 512
    k, v = rnd(B, H, T, D, seed=11, dtype=dtype), rnd(B, H, T, D, seed=12, dtype=dtype)
    q = rnd(B, H, 1, D, seed=13, dtype=dtype)
    tq = torch.full((1, 1), t, dtype=torch.int32)
    want, _, tol = want64(q, k, v, tq, 0.125)
    for nsplit in (1, 4, 8, 256):
        for c in ((paged(k, v, 16, fill=float('inf')), None), (k.to(DEV), v.to(DEV))):
            close(K.dense_attn(q.to(DEV), *c, tq.to(DEV), 0.125, nsplit=nsplit)[0], want, tol, dtype)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('nsplit', [1, 8])
def test_what_is_masked_has_no_effect(dtype, nsplit):
    """Infinities, NaN and the lowest numbers in the rows after a query's own position, also where a later query of the same
    call does see them; rows of missing pages; positions before 0 and past the cache."""
    B, H, D, T, N, leaf = 2, 2, 64, 200, 4, 8
    k, v = rnd(B, H, T, D, seed=21, dtype=dtype), rnd(B, H, T, D, seed=22, dtype=dtype)
    q = rnd(B, 2 * H, N, D, seed=23, dtype=dtype)
    tq = torch.tensor([[150, 151, 152, 153], [-3, 199, 200, 77]], dtype=torch.int32)
    low = torch.finfo(dtype).min
    scale = 0.125
    clean = None
    missing = [(0, 0, 2), (0, 0, 3), (0, 1, 0), (1, 1, 9)]
    have = torch.ones(B, H, T, dtype=torch.bool)
    for b, h, j in missing:
        have[b, h, j * leaf:(j + 1) * leaf] = False
    for bad in (0.0, float('inf'), float('nan'), low):
        kk, vv = k.clone(), v.clone()
        kk[0, :, 151:] = bad
        vv[0, :, 151:] = bad
        vv[1, :, 78:199, 5] = bad
        c = paged(kk, vv, leaf, seed=4, fill=bad, missing=missing)
        out = K.dense_attn(q.to(DEV), c, None, tq.to(DEV), scale, nsplit=nsplit)[0].cpu()
        assert not out[1, :, 0].any() and not out[1, :, 2].any()      # outside the cache: zeros
        keep = torch.stack((out[0, :, 0], out[1, :, 3]))              # these see none of it
        assert bool(torch.isfinite(keep).all()), bad
        if clean is None:
            clean = keep
            want, _, tol = want64(q, kk, vv, tq, scale, have)
            close(out, want, tol, dtype)
        assert torch.equal(keep, clean), bad
        # the query that does see an infinite or NaN value shows it there and nowhere else
        seen = out[1, :, 1].float()
        if bad == 0.0:
            continue
        other = torch.arange(D) != 5
        assert bool(torch.isfinite(seen[:, other]).all())
        if bad != low:
            assert torch.equal(torch.isnan(seen[:, 5]), torch.full((2 * H,), math.isnan(bad))) or bool(
                (~torch.isfinite(seen[:, 5])).all())


@pytest.mark.parametrize('N', [1, 3, 70])
@pytest.mark.parametrize('nsplit', [4, 64, 1024])
def test_many_ragged_sequences(N, nsplit):
    """More sequences than a wavefront has lanes, from no token to many, tokens at positions outside the cache among the others
    (the padding of a batch): zeros there, and no effect on their neighbours."""
    B, H, D, T = 131, 2, 32, 700
    g = torch.Generator().manual_seed(N)
    lens = torch.randint(1, T + 1, (B,), generator=g) // torch.randint(1, 9, (B,), generator=g)
    k, v = rnd(B, H, T, D, seed=111, dtype=BF16), rnd(B, H, T, D, seed=112, dtype=BF16)
    q = rnd(B, 2 * H, N, D, seed=113, dtype=BF16)
    tq = rows(lens.tolist(), N)
    if N > 1:
        tq[3, 1], tq[70, 0], tq[130, N - 1], tq[64] = -1, T, 1 << 30, -7
    c = paged(k, v, 16, fill=float('nan'))
    out = K.dense_attn(q.to(DEV), c, None, tq.to(DEV), 0.2, nsplit=nsplit)[0]
    some = sorted({0, 3, 63, 64, 65, 70, 127, 128, 130} | set(range(0, B, 40)))[::1 if N < 70 else 4]
    want, _, tol = want64(q[some], k[some], v[some], tq[some], 0.2)
    close(out[some], want, tol, BF16)
    one = K.dense_attn(q[64:66].to(DEV), c.rows(64, 66), None, tq[64:66].to(DEV), 0.2, nsplit=1)[0]
    want, _, tol = want64(q[64:66], k[64:66], v[64:66], tq[64:66], 0.2)
    close(one, want, tol, BF16)
    wide = torch.full((B, N), 2 ** 32 + 3, dtype=torch.int64)              # past 32 bits: outside, not position 3
    assert not K.dense_attn(q.to(DEV), c, None, wide.to(DEV), 0.2, nsplit=nsplit)[0].any()


def test_no_keys_at_all():
    """A sequence without pages, and a cache whose blocks have none: zeros and lse -1e30."""
    q = rnd(2, 2, 3, 64, seed=31, dtype=BF16).to(DEV)
    pool = torch.full((4, 2, 16, 64), float('nan'), dtype=BF16, device=DEV)
    for ids in (-1, 4, 1 << 30):
        c = K.PagedCache(pool, torch.full((2, 2, 8), ids, dtype=torch.int32, device=DEV), 128)
        for nsplit in (1, 4, 16):
            lse = torch.empty(2, 2, 3, device=DEV)
            out, _ = K.dense_attn(q, c, None, torch.tensor([5, 100, 127], device=DEV), nsplit=nsplit, lse=lse)
            assert not out.any() and bool((lse == -1e30).all())


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_equal_and_extreme_scores(dtype):
    """All scores equal (the mean of the values); one score far above all others, at the first, a middle and the last key; scores
    so low that a weight of 16 bits would lose them."""
    D, T = 64, 3001
    v = rnd(1, 1, T, D, seed=41, dtype=dtype)
    q = torch.zeros(1, 1, 1, D, dtype=dtype)
    k = rnd(1, 1, T, D, seed=42, dtype=dtype)
    tq = torch.full((1, 1), T - 1, dtype=torch.int32)
    for nsplit in (1, 4, 32):
        want, _, tol = want64(q, k, v, tq, 1.0)
        close(K.dense_attn(q.to(DEV), k.to(DEV), v.to(DEV), tq.to(DEV), 1.0, nsplit=nsplit)[0], want, tol, dtype)
    q[..., 0] = 1.0
    for top in (9.0, 11.0, 13.0, 60.0):
        for at in (0, 1500, T - 1):
            k2 = torch.zeros(1, 1, T, D, dtype=dtype)
            k2[0, 0, :, 0] = 0.25 * (torch.arange(T) % 7)
            k2[0, 0, at, 0] = top
            want, _, tol = want64(q, k2, v, tq, 1.0)
            for nsplit in (1, 4, 32):
                close(K.dense_attn(q.to(DEV), k2.to(DEV), v.to(DEV), tq.to(DEV), 1.0, nsplit=nsplit)[0], want, tol, dtype)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_layouts(dtype):
    """Queries and outputs as views of a projection's rows, caches with heads inside positions, K and V of different strides,
    more room behind the rows, one shared set of positions."""
    B, H, G, N, D, T = 2, 2, 3, 5, 32, 96
    k, v = rnd(B, H, T, D, seed=51, dtype=dtype), rnd(B, H, T, D, seed=52, dtype=dtype)
    q = rnd(B, N, G * H + 4, D, seed=53, dtype=dtype).to(DEV)[:, :, :G * H].transpose(1, 2)
    kc = k.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    vc = torch.zeros(B, H, T + 8, D + 16, dtype=dtype, device=DEV)[:, :, :T, :D]
    vc.copy_(v)
    tq = torch.tensor([90, 3, 47, 95, 0], dtype=torch.int32)
    out = torch.full((B, N, G * H, 2 * D), 7.0, dtype=dtype, device=DEV)
    view = out[..., :D].transpose(1, 2)
    K.dense_attn(q, kc, vc, tq.to(DEV), 0.2, out=view, nsplit=8)
    want, _, tol = want64(q.cpu(), k, v, tq.expand(B, N), 0.2)
    close(view, want, tol, dtype)
    assert bool((out[..., D:] == 7.0).all())
    long = K.dense_attn(q, kc, vc, tq.long().to(DEV), 0.2, nsplit=8)[0]
    assert torch.equal(long, view)


def test_far_pages():
    """Pages past 2^31 elements of the pool, and rows past 2^31 elements of a contiguous cache."""
    leaf, D, P = 64, 64, 262144 + 300
    pool = torch.zeros(P, 2, leaf, D, dtype=BF16, device=DEV)
    k, v = rnd(1, 2, 500, D, seed=61, dtype=BF16), rnd(1, 2, 500, D, seed=62, dtype=BF16)
    c = paged(k, v, leaf, seed=2, spare=0)
    n = c.pool.shape[0]
    pool[P - n:] = c.pool
    far = K.PagedCache(pool, c.table + (P - n), 500)
    q = rnd(1, 2, 1, D, seed=63, dtype=BF16).to(DEV)
    tq = torch.tensor([499], device=DEV)
    for nsplit in (1, 16):
        assert torch.equal(K.dense_attn(q, far, None, tq, nsplit=nsplit)[0], K.dense_attn(q, c, None, tq, nsplit=nsplit)[0])
    del pool, far
    big = torch.zeros(1 << 25, 2, 1, D, dtype=BF16, device=DEV)       # rows of (head, position) 64 elements, heads far apart
    kc = big[:500 * 60000:60000].permute(2, 1, 0, 3)                  # (1, 2, 500, D), row stride 60000 * 128
    kc.copy_(k)
    assert torch.equal(K.dense_attn(q, kc, v.to(DEV), tq)[0], K.dense_attn(q, k.to(DEV), v.to(DEV), tq)[0])


def test_graph_other_stream_and_shared_workspace():
    """Captured calls, replayed with eager work between; calls that share a workspace one after another; another stream."""
    B, H, D, T, nsplit = 2, 3, 64, 1000, 32
    k, v = rnd(B, H, T, D, seed=71, dtype=BF16), rnd(B, H, T, D, seed=72, dtype=BF16)
    c = paged(k, v, 16)
    q = rnd(B, H, 1, D, seed=73, dtype=BF16).to(DEV)
    tq = torch.tensor([[900], [41]], dtype=torch.int32, device=DEV)
    ws = K.dense_attn_workspace(B, H, 1, D, nsplit, DEV)
    out, out2 = torch.empty_like(q), torch.empty_like(q)
    K.dense_attn(q, c, None, tq, nsplit=nsplit, ws=ws, out=out)
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        K.dense_attn(q, c, None, tq, nsplit=nsplit, ws=ws, out=out)
        K.dense_attn(out, c, None, tq, nsplit=nsplit, ws=ws, out=out2)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(4):
        tq.copy_(torch.tensor([[900 - i], [41 + 300 * i]]))
        q.normal_()
        a = K.dense_attn(q, c, None, tq, nsplit=nsplit)[0]
        b = K.dense_attn(a, c, None, tq, nsplit=nsplit)[0]
        out.zero_()
        out2.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(out2, b), i
        assert not ws[:256].any()                                     # the counters are back at zero
    with torch.cuda.stream(s):
        s.wait_stream(torch.cuda.default_stream())
        b = K.dense_attn(q, c, None, tq, nsplit=nsplit, ws=ws)[0]
    s.synchronize()
    assert torch.equal(a, b)


def test_the_split_rule_and_its_results():
    """decode_nsplit_dense gives counts that dense_attn takes, and the same attention whatever the count."""
    for B, H, rows_, keys, D in [(1, 1, 1, 1, 64), (1, 1, 1, 131072, 128), (1, 12, 1, 131072, 64), (32, 12, 1, 32768, 64),
                                 (1, 2, 256, 4096, 64), (4, 8, 4, 6000, 128), (512, 12, 1, 100, 16)]:
        n = decode_nsplit_dense(B, H, rows_, keys, D)
        assert n == 1 or (n % 4 == 0 and 4 <= n <= 8192), n
    k, v = rnd(1, 1, 5000, 64, seed=81), rnd(1, 1, 5000, 64, seed=82)
    q = rnd(1, 1, 1, 64, seed=83)
    tq = torch.tensor([[4999]], dtype=torch.int32)
    want, _, tol = want64(q, k, v, tq, 0.125)
    for nsplit in (1, 4, 8, 20, 128, 512, 1024):
        close(K.dense_attn(q.to(DEV), k.to(DEV), v.to(DEV), tq.to(DEV), 0.125, nsplit=nsplit)[0], want, tol, F32)


def test_same_bits_every_time():
    k, v = rnd(2, 4, 3000, 64, seed=91, dtype=BF16).to(DEV), rnd(2, 4, 3000, 64, seed=92, dtype=BF16).to(DEV)
    q = rnd(2, 4, 1, 64, seed=93, dtype=BF16).to(DEV)
    tq = torch.tensor([[2999], [1234]], device=DEV)
    a = K.dense_attn(q, k, v, tq, nsplit=64)[0]
    for _ in range(5):
        assert torch.equal(K.dense_attn(q, k, v, tq, nsplit=64)[0], a)


def test_refusals():
    q = torch.zeros(2, 4, 1, 64, device=DEV, dtype=BF16)
    k = torch.zeros(2, 2, 50, 64, device=DEV, dtype=BF16)
    tq = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    c = paged(torch.zeros(2, 2, 50, 64, dtype=BF16), torch.zeros(2, 2, 50, 64, dtype=BF16), 16)
    K.dense_attn(q, k, k, tq)
    for bad in (lambda: K.dense_attn(q[:, :3], k, k, tq), lambda: K.dense_attn(q[:1], k, k, tq),
                lambda: K.dense_attn(q, k, k[:, :, :40], tq), lambda: K.dense_attn(q, c, k, tq),
                lambda: K.dense_attn(q[..., :32], k, k, tq), lambda: K.dense_attn(q, k, k, tq[:1]),
                lambda: K.dense_attn(q, k, k, tq, out=torch.empty(2, 4, 2, 64, device=DEV, dtype=BF16)),
                lambda: K.dense_attn(q, k, k, tq, lse=torch.empty(2, 4, device=DEV)),
                lambda: K.dense_attn(q, k, k, tq.cpu()), lambda: K.dense_attn(q.cpu(), k, k, tq)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    with pytest.raises(ValueError, match='repeats'):
        K.dense_attn(q, k, k, tq, out=torch.empty(1, 4, 1, 64, device=DEV, dtype=BF16).expand(2, 4, 1, 64))
    for bad in (lambda: K.dense_attn(q.float(), k, k, tq), lambda: K.dense_attn(q, k, k, tq.float()),
                lambda: K.dense_attn(q, object(), None, tq)):
        with pytest.raises(TypeError):
            bad()
    for nsplit in (0, 2, 6, 8196, -4):
        with pytest.raises(RuntimeError, match='nsplit'):
            K.dense_attn(q, k, k, tq, nsplit=nsplit)
    with pytest.raises(RuntimeError, match='workspace'):
        K.dense_attn(q, k, k, tq, nsplit=16, ws=torch.zeros(64, dtype=torch.uint8, device=DEV))
    for D in (8, 48, 256):
        x = torch.zeros(1, 1, 4, D, device=DEV)
        with pytest.raises(RuntimeError, match='head dim'):
            K.dense_attn(x, x, x, torch.arange(4, device=DEV))
    odd = torch.zeros(2, 4, 1, 72, device=DEV, dtype=BF16)[..., 1:65]
    with pytest.raises(RuntimeError, match='aligned'):
        K.dense_attn(odd, k, k, tq)
    empty = torch.zeros(2, 2, 0, 64, device=DEV, dtype=BF16)
    assert not K.dense_attn(torch.ones_like(q), empty, empty, tq)[0].any()
    assert K.dense_attn(q[:, :, :0], k, k, tq[:, :0])[0].shape == (2, 4, 0, 64)


def some_rows(out, lse, q, k, v, tq, scale, pairs, dtype, at, have=None):
    """Rows `at` of the (sequence, query head) pairs against float64."""
    G = q.shape[1] // k.shape[1]
    for b, h in pairs:
        g = h // G
        want, wl, tol = want64(q[b:b + 1, h:h + 1, at], k[b:b + 1, g:g + 1], v[b:b + 1, g:g + 1], tq[b:b + 1, at], scale,
                               None if have is None else have[b:b + 1, g:g + 1])
        close(out[b:b + 1, h:h + 1, at], want, tol, dtype)
        if lse is not None:
            got = lse[b, h, at].cpu()
            assert torch.equal(got == -1e30, wl[0, 0] == -1e30)
            ok = wl[0, 0] > -1e29
            assert bool(((got.double() - wl[0, 0]).abs()[ok] <= (tol[0, 0, :, 0][ok] / 2 + 1e-6 * (1 + wl[0, 0][ok].abs())) + 1e-5).all())


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('D,leaf,H,G,N,T', [(64, 64, 12, 1, 1000, 1003), (128, 32, 8, 3, 500, 513), (32, 128, 12, 1, 1024, 1024),
                                            (64, 0, 12, 1, 901, 929), (128, 0, 12, 1, 1000, 1001), (32, 0, 3, 65, 63, 640),
                                            (64, 64, 96, 1, 100, 577)])
@pytest.mark.parametrize('nsplit', [1, 132, 1024, 2600])
def test_many_rows(dtype, D, leaf, H, G, N, T, nsplit):
    """Prompts and pieces of them, their positions in any order, some outside the cache; contiguous caches that end inside a
    tile; last sets with wavefronts that have no rows."""
    B = 2
    k, v = rnd(B, H, T, D, seed=31, dtype=dtype), rnd(B, H, T, D, seed=32, dtype=dtype)
    q = rnd(B, G * H, N, D, seed=33, dtype=dtype)
    g = torch.Generator().manual_seed(34)
    tq = rows([T, T - 3], N)
    mixed = torch.randint(-2, T + 2, (N,), generator=g, dtype=torch.int32)
    tq[1, N // 2:] = mixed[N // 2:]
    have = None
    if leaf:
        missing = [(0, 0, 1), (1, H - 1, 0), (1, H - 1, 3)]
        have = torch.ones(B, H, T, dtype=torch.bool)
        for b, h, j in missing:
            have[b, h, j * leaf:(j + 1) * leaf] = False
        c = paged(k, v, leaf, seed=D, fill=float('nan'), missing=missing), None
    else:   # strides of a larger cache, whose other rows are NaN
        wide = [torch.full((B, H, T + 70, D), float('nan'), dtype=dtype, device=DEV)[:, :, :T] for _ in range(2)]
        c = wide[0].copy_(k), wide[1].copy_(v)
    scale = 1 / math.sqrt(D)
    lse = torch.empty(B, G * H, N, device=DEV)
    out, _ = K.dense_attn(q.to(DEV), *c, tq.to(DEV), scale, lse=lse, nsplit=nsplit)
    at = torch.unique(torch.cat([torch.arange(0, N, max(1, N // 12)), torch.tensor([N - 1, N - 2]),
                                 torch.randint(0, N, (8,), generator=g)]))
    some_rows(out, lse, q, k, v, tq, scale, [(0, 0), (1, G * H - 1), (1, G)], dtype, at, have)
    # the same whatever the other rows are: each sequence by itself, with other tokens before and after
    same, _ = K.dense_attn(q.to(DEV).flip(2), *c, tq.to(DEV).flip(1), scale, nsplit=nsplit)
    far = (torch.arange(B * G * H * N * D) % 7 == 0).view(B, G * H, N, D)
    a, b = out.cpu()[far].double(), same.flip(2).cpu()[far].double()
    assert bool(((a - b).abs() <= 2 * torch.finfo(dtype).eps * a.abs() + 1e-3).all())


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('nsplit', [1, 1600])
def test_many_rows_what_is_masked(dtype, D, nsplit):
    """A value that some rows of a tile see and others do not: only those that see it show it, the others' bits stay; also
    where it is the key."""
    B, H, N, T = 4, 12, 500, 600
    k, v = rnd(B, H, T, D, seed=41, dtype=dtype).to(DEV), rnd(B, H, T, D, seed=42, dtype=dtype).to(DEV)
    q = rnd(B, H, N, D, seed=43, dtype=dtype).to(DEV)
    tq = rows([T, T, T - 7, N], N).to(DEV)
    clean, _ = K.dense_attn(q, k, v, tq, nsplit=nsplit)
    for bad in (float('inf'), float('nan'), torch.finfo(dtype).min):
        for which in (0, 1):
            x = [k.clone(), v.clone()]
            for b, h, t in ((0, 0, T - 5), (1, 3, 330), (2, 11, T - 1), (3, 0, 70)):
                x[which][b, h, t, 5] = bad
            got, _ = K.dense_attn(q, *x, tq, nsplit=nsplit)
            for b, h, t in ((0, 0, T - 5), (1, 3, 330), (2, 11, T - 1), (3, 0, 70)):
                blind = tq[b] < t
                assert torch.equal(got[b, h, blind], clean[b, h, blind]), (bad, which, b)
                if math.isnan(bad):
                    seen = got[b, h, ~blind]
                    assert bool(torch.isnan(seen if which == 0 else seen[:, 5]).all())
                if which == 1 and math.isinf(bad):
                    assert bool((got[b, h, ~blind][:, 5] == bad).all())
                    assert torch.equal(got[b, h, ~blind][:, 6:].isfinite(), torch.ones_like(got[b, h, ~blind][:, 6:]).bool())
            other = torch.ones(B, H, dtype=torch.bool)
            other[[0, 1, 2, 3], [0, 3, 11, 0]] = False
            assert torch.equal(got[other], clean[other])


def test_many_rows_extreme_scores_and_replays():
    B, H, N, T, D = 4, 12, 512, 640, 64
    k, v, q = [rnd(B, H, n, D, seed=50 + n, dtype=BF16).to(DEV) for n in (T, T, N)]
    tq = rows([T, 600, N, 513], N).to(DEV)
    for scale in (0.0, -0.125, 30.0):
        out, _ = K.dense_attn(q, k, v, tq, scale, nsplit=1)
        at = torch.tensor([0, 1, 127, 128, 300, 511])
        if scale < 0:
            some_rows(out, None, -q.cpu(), k.cpu(), v.cpu(), tq.cpu(), -scale, [(0, 0), (3, 11)], BF16, at)
        else:
            some_rows(out, None, q.cpu(), k.cpu(), v.cpu(), tq.cpu(), scale, [(0, 0), (3, 11)], BF16, at)
    # one workspace for two calls of a graph and for eager ones between its replays, also of another cache's kind
    small = paged(k[:, :, :400].cpu(), v[:, :, :400].cpu(), 8)
    for nsplit in (1, 1024):
        ws = K.dense_attn_workspace(B, H, N, D, nsplit, DEV, H)
        out, two = torch.empty_like(q), torch.empty_like(q)

        def calls():
            K.dense_attn(q, k, v, tq, out=out, nsplit=nsplit, ws=ws)
            K.dense_attn(q, small, None, tq, out=two, nsplit=nsplit, ws=ws)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            calls()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            calls()
        for i in range(3):
            q.copy_(rnd(B, H, N, D, seed=60 + i, dtype=BF16).to(DEV))
            tq.copy_(rows([T - i, 600, N, 513 + i], N).to(DEV))
            g.replay()
            assert torch.equal(out, K.dense_attn(q, k, v, tq, nsplit=nsplit, ws=ws)[0])
            assert torch.equal(two, K.dense_attn(q, small, None, tq, nsplit=nsplit)[0])
            torch.cuda.synchronize()
