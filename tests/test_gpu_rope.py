"""Rotary positions (kernels.rope, positions.rotate) and the store of new tokens into a decode cache (kernels.kv_store) against
their formulas in float64.  GPU only."""
import math

import pytest
import torch

from treeattn_amd import kernels as K
from treeattn_amd import positions as P

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rnd(*shape, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def turned64(x, pos, w, layout, amp=1.0, sign=1):
    """x (B,H,T,D) in float64, turned; pos (T,) or (B,T)."""
    x = x.double()
    rot = 2 * len(w)
    a = pos.double()[..., None] * torch.tensor(w, dtype=torch.float64) * sign
    a = a if pos.dim() == 1 else a[:, None]
    c, s = torch.cos(a) * amp, torch.sin(a) * amp
    y = x.clone()
    i, j = (slice(0, rot, 2), slice(1, rot, 2)) if layout == 'interleaved' else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y


def close(got, want, x, dtype, amp=1.0):
    """Sines and cosines good to 2^-20 (16-bit rows: the hardware's) or 2^-22 (float32 rows), two products and a sum in float32,
    one rounding of the result: off by at most (2^-20 or 2^-22) 2 amp max(|a|, |b|) and half a step."""
    big = x.double().abs().amax(-1, keepdim=True) * amp
    half = torch.finfo(dtype).eps / 2
    tol = 2 * big * (2.0 ** -22 if dtype == F32 else 2.0 ** -20) + (want.abs() + big * 2.0 ** -19) * half + 2.0 ** -26
    d = (got.double().cpu() - want).abs()
    assert bool((d <= tol).all()), float((d - tol).max())


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('D,rot,H,T', [(64, 64, 3, 50), (64, 32, 2, 7), (128, 128, 5, 33), (16, 16, 1, 1), (64, 10, 2, 9),
                                       (66, 66, 1, 5), (37, 6, 3, 11), (32, 2, 2, 4), (128, 96, 4, 3), (24, 16, 2, 6)])
def test_turn_and_turn_back(dtype, layout, D, rot, H, T):
    w, _ = P.rope_frequencies(rot)
    r = K.Rope(w, DEV, layout=layout, amplitude=1.25)
    x = rnd(2, H, T, D, seed=D + rot, dtype=dtype)
    for pos in (torch.arange(T), torch.stack((torch.arange(T) * 37 + 5, 4000 - torch.arange(T) * 3)).to(torch.int32)):
        for inverse in (False, True):
            got = K.rope(x.to(DEV), pos.to(DEV), r, inverse=inverse)
            want = turned64(x, pos, w, layout, 1.25, -1 if inverse else 1)
            close(got, want, x, dtype, 1.25)
            assert torch.equal(got[..., rot:].cpu(), x[..., rot:])
            same = x.to(DEV)
            assert K.rope(same, pos.to(DEV), r, out=same, inverse=inverse) is same
            assert torch.equal(same, got)


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_far_positions(dtype):
    """Angles up to 10^9 radians: the turns are taken off in 64 bits."""
    w, _ = P.rope_frequencies(64)
    r = K.Rope(w, DEV)
    pos = torch.tensor([0, 1, 131071, 1000003, 16777217, 1 << 30, 2147483647, -5, -1000003], dtype=torch.int32)
    x = rnd(1, 4, len(pos), 64, seed=5, dtype=dtype)
    close(K.rope(x.to(DEV), pos.to(DEV), r), turned64(x, pos, w, 'half'), x, dtype)


def test_frequencies():
    w, a = P.rope_frequencies(64)
    assert len(w) == 32 and w[0] == 1.0 and abs(w[-1] - 10000 ** (-62 / 64)) < 1e-15 and a == 1.0
    assert P.rope_frequencies(64, scaling='linear', factor=4)[0] == [x / 4 for x in w]
    n, a = P.rope_frequencies(64, scaling='ntk', factor=4)
    assert a == 1.0 and n[0] == 1.0 and abs(n[-1] * 4 - w[-1]) < 1e-12
    b, a = P.rope_frequencies(64, scaling='bands', factor=4, trained=1024)
    assert abs(a - 0.1 * math.log(4) - 1) < 1e-12
    assert b[0] == w[0] and abs(b[-1] * 4 - w[-1]) < 1e-15 and all(x / 4 <= y <= x for x, y in zip(w, b))
    for bad in (dict(rot=3), dict(rot=0), dict(rot=2, scaling='ntk'), dict(rot=8, scaling='bands'), dict(rot=8, scaling='x'),
                dict(rot=8, factor=0.5), dict(rot=8, base=0.0)):
        with pytest.raises(ValueError):
            P.rope_frequencies(**bad)


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('D,rot', [(64, 64), (32, 10)])
def test_gradient(dtype, D, rot):
    """The gradient is the formula's (the turn back), agrees with differences, and is itself differentiable; the input a view
    of a projection, the gradient coming in expanded."""
    B, H, T = 2, 3, 13
    w, _ = P.rope_frequencies(rot)
    r = K.Rope(w, DEV, layout='interleaved', amplitude=1.5)
    base = rnd(B, T, 3 * H, D, seed=9, dtype=dtype).to(DEV).requires_grad_(True)
    x = base[:, :, H:2 * H].transpose(1, 2)
    pos = torch.arange(100, 100 + T, device=DEV)
    y = P.rotate(x, pos, r)
    dy = rnd(B, H, T, D, seed=10, dtype=dtype)
    (g,) = torch.autograd.grad(y, base, dy.to(DEV), retain_graph=True)
    want = turned64(dy, pos.cpu(), w, 'interleaved', 1.5, -1)
    close(g[:, :, H:2 * H].transpose(1, 2), want, dy, dtype, 1.5)
    assert not g[:, :, :H].any() and not g[:, :, 2 * H:].any()
    (g,) = torch.autograd.grad(y.sum(), base)                      # an expanded gradient of ones
    one = torch.ones(B, H, T, D)
    close(g[:, :, H:2 * H].transpose(1, 2), turned64(one, pos.cpu(), w, 'interleaved', 1.5, -1), one, dtype, 1.5)
    if dtype == F32:
        d = rnd(B, T, 3 * H, D, seed=11).to(DEV)
        f = lambda b: (P.rotate(b[:, :, H:2 * H].transpose(1, 2), pos, r) * dy.to(DEV)).double().sum()
        (g,) = torch.autograd.grad(f(base), base)
        # linear, so the central difference is exact but for rounding: each f is a sum of products off by 2^-22 of them
        diff = float(f(base.detach() + d) - f(base.detach() - d)) / 2
        size = float((dy.abs().to(DEV) * 8).double().sum()) * 2.0 ** -20
        assert abs(diff - float((g.double() * d.double()).sum())) <= size
        (g1,) = torch.autograd.grad(P.rotate(x, pos, r), base, dy.to(DEV).requires_grad_(True), create_graph=True)
        assert g1.requires_grad


def paged(B, H, D, leaf, T, dtype, seed=0, missing=()):
    nb = (T + leaf - 1) // leaf
    Pn = B * H * nb + 3
    table = torch.randperm(Pn, generator=torch.Generator().manual_seed(seed))[:B * H * nb].to(torch.int32).view(B, H, nb).contiguous()
    for m in missing:
        table[m] = -1
    return K.PagedCache(torch.full((Pn, 2, leaf, D), 7.0, dtype=dtype, device=DEV), table.to(DEV), T)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('D,rot,layout,leaf,H,G,N', [(64, 64, 'half', 16, 3, 1, 1), (64, 32, 'interleaved', 64, 2, 2, 5),
                                                     (128, 128, 'half', 2, 1, 4, 3), (16, 16, 'interleaved', 8, 2, 1, 40),
                                                     (24, 6, 'half', 8, 2, 1, 3), (64, 0, 'half', 32, 2, 2, 7)])
@pytest.mark.parametrize('contiguous', [False, True])
def test_store(dtype, D, rot, layout, leaf, H, G, N, contiguous):
    """The rows of the positions hold the turned keys and the values, all others are as they were: with blocks that have no page,
    and positions before the first and past the last."""
    B, T = 3, 120
    w = P.rope_frequencies(rot)[0] if rot else []
    r = K.Rope(w, DEV, layout=layout, amplitude=0.75) if rot else None
    x = rnd(B, N, (G + 2) * H, D, seed=N, dtype=dtype).to(DEV).transpose(1, 2)
    q, k, v = x[:, :G * H], x[:, G * H:G * H + H], x[:, G * H + H:]
    pos = torch.stack([torch.arange(N), torch.arange(N) * 2 + 31, 118 + torch.arange(N)]).to(torch.int32)
    if N == 3:
        pos[0] = torch.tensor([5, -1, 0])
    if contiguous:
        pair = (torch.full((B, H, T, D), 7.0, dtype=dtype, device=DEV), torch.full((B, H, T, D), 7.0, dtype=dtype, device=DEV))
        dense = [t.clone() for t in pair]
        got = K.kv_store(k, v, *pair, pos.to(DEV), q=q, rope=r)
        have = torch.ones(B, H, T, dtype=torch.bool)
    else:
        missing = [(1, 0, 32 // leaf), (0, H - 1, 0)]
        c = paged(B, H, D, leaf, T, dtype, missing=missing)
        have = torch.ones(B, H, T, dtype=torch.bool)
        for b, h, j in missing:
            have[b, h, j * leaf:(j + 1) * leaf] = False
        before = c.pool.clone()
        got = K.kv_store(k, v, c, None, pos.to(DEV), q=q, rope=r)
        dense = [torch.full((B, H, T, D), 7.0, dtype=dtype, device=DEV) for _ in (0, 1)]
        pair = [torch.cat(z) for z in zip(*(c.dense(b) for b in range(B)))]
    close(got, turned64(q.cpu(), pos, w, layout, 0.75) if rot else q.cpu().double(), q.cpu(), dtype)
    wk = turned64(k.cpu(), pos, w, layout, 0.75) if rot else k.cpu().double()
    touched = torch.zeros(B, H, T, dtype=torch.bool)
    for b in range(B):
        for n in range(N):
            t = int(pos[b, n])
            if 0 <= t < T:
                touched[b, :, t] = have[b, :, t]
                for h in range(H):
                    if have[b, h, t]:
                        close(pair[0][b, h, t], wk[b, h, n], k[b, h, n].cpu(), dtype)
                        assert torch.equal(pair[1][b, h, t], v[b, h, n])
    for z, d in zip(pair, dense):
        rest = (have & ~touched).to(DEV)
        assert torch.equal(z[rest], d[rest])
    if not contiguous:     # pages of no block, rows past the last position of a block that has them
        used = set(c.table.flatten().tolist())
        spare = [i for i in range(c.pool.shape[0]) if i not in used]
        assert torch.equal(c.pool[spare], before[spare])
    # the same without queries, and into the queries themselves
    q2 = q.clone()
    if contiguous:
        K.kv_store(k, v, *dense, pos.to(DEV), q=q2, rope=r, q_out=q2)
        assert all(torch.equal(a, b) for a, b in zip(pair, dense))
    else:
        assert K.kv_store(k, v, c, None, pos.to(DEV), rope=r) is None
        K.kv_store(k, v, c, None, pos.to(DEV), q=q2, rope=r, q_out=q2)
    assert torch.equal(q2, got)


def test_stored_keys_are_what_rope_gives():
    w, _ = P.rope_frequencies(64)
    r = K.Rope(w, DEV)
    k, v = rnd(2, 3, 50, 64, seed=1, dtype=BF16).to(DEV), rnd(2, 3, 50, 64, seed=2, dtype=BF16).to(DEV)
    c = paged(2, 3, 64, 16, 64, BF16)
    pos = torch.arange(50, device=DEV)
    q = K.kv_store(k, v, c, None, pos, q=k, rope=r)
    assert torch.equal(q, K.rope(k, pos, r))
    for b in range(2):
        kk, vv = c.dense(b, 50)
        assert torch.equal(kk[0], q[b]) and torch.equal(vv[0], v[b])
    one = paged(2, 3, 64, 16, 64, BF16)
    for t in range(50):
        K.kv_store(k[:, :, t:t + 1], v[:, :, t:t + 1], one, None, pos[t:t + 1], rope=r)
    assert torch.equal(one.pool, c.pool)


def test_many_tokens_and_graph():
    """The form of many tokens (four heads a thread) gives the bits of the form of few, and both replay in a graph."""
    w, _ = P.rope_frequencies(64)
    r = K.Rope(w, DEV, layout='interleaved')
    x = rnd(1, 5, 60000, 64, seed=3).to(DEV)
    pos = torch.arange(60000, device=DEV)
    big = K.rope(x, pos, r)
    for t in (0, 1, 31234, 59990):
        assert torch.equal(big[:, :, t:t + 9], K.rope(x[:, :, t:t + 9].contiguous(), pos[t:t + 9], r))
    small = x[:, :, :64].contiguous()
    p32, out = pos[:64].to(torch.int32), torch.empty_like(small)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        K.rope(small, p32, r, out=out)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(3):
        p32.add_(17)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, K.rope(small, p32, r))


def test_refusals():
    r = K.Rope(P.rope_frequencies(64)[0], DEV)
    x = torch.zeros(2, 3, 5, 64, device=DEV)
    pos = torch.arange(5, device=DEV)
    K.rope(x, pos, r)
    for bad in (lambda: K.rope(x[..., :32], pos, r), lambda: K.rope(x, pos[:4], r), lambda: K.rope(x.transpose(2, 3), pos, r),
                lambda: K.rope(x, pos, r, out=torch.empty(2, 3, 4, 64, device=DEV)),
                lambda: K.rope(x, pos, r, out=torch.empty(1, 3, 5, 64, device=DEV).expand(2, 3, 5, 64)),
                lambda: K.rope(x, pos, r, out=x.view(3, 2, 5, 64).transpose(0, 1)),
                lambda: K.rope(x, pos.cpu(), r), lambda: K.rope(x.cpu(), pos, r),
                lambda: K.Rope([], DEV), lambda: K.Rope([1.0], DEV, layout='x'), lambda: K.Rope([float('nan')], DEV),
                lambda: K.Rope([1.0], DEV, amplitude=float('inf'))):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    with pytest.raises(TypeError):
        K.rope(x, pos.float(), r)
    k = torch.zeros(2, 3, 5, 64, device=DEV)
    c = paged(2, 3, 64, 16, 64, F32)
    Kc = torch.zeros(2, 3, 64, 64, device=DEV)
    for bad in (lambda: K.kv_store(k[:1], k[:1], c, None, pos), lambda: K.kv_store(k, k[:, :, :4], c, None, pos),
                lambda: K.kv_store(k, k, c, Kc, pos), lambda: K.kv_store(k, k, Kc, Kc[:, :, :32], pos),
                lambda: K.kv_store(k, k, c, None, pos, q=k[:, :, :3]), lambda: K.kv_store(k, k, c, None, pos, q_out=k),
                lambda: K.kv_store(k, k, c, None, pos, q=k, q_out=torch.zeros(1, 3, 5, 64, device=DEV).expand(2, 3, 5, 64)),
                lambda: K.kv_store(k, k, c, None, pos, rope=K.Rope(P.rope_frequencies(128)[0], DEV))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: K.kv_store(k.half(), k, c, None, pos), lambda: K.kv_store(k, k, object(), None, pos)):
        with pytest.raises(TypeError):
            bad()
    assert K.kv_store(k[:, :, :0], k[:, :, :0], c, None, pos[:0]) is None
    assert K.rope(x[:, :, :0], pos[:0], r).shape == (2, 3, 0, 64)


def test_store_without_a_position():
    """A cache that holds no position stores nothing; its queries are turned all the same."""
    k = torch.randn(2, 3, 5, 64, device=DEV)
    q = torch.randn(2, 6, 5, 64, device=DEV)
    pos = torch.arange(5, dtype=torch.int32, device=DEV)
    r = K.Rope(P.rope_frequencies(64)[0], DEV)
    none = torch.zeros(2, 3, 0, 64, device=DEV)
    assert torch.equal(K.kv_store(k, k, none, none, pos, q=q, rope=r), K.rope(q, pos, r))
    assert torch.equal(K.kv_store(k, k, none, none, pos, q=q), q)
    for bad in (lambda: K.kv_store(k, k, none, None, pos), lambda: K.dense_attn(q, k, None, pos)):
        with pytest.raises(TypeError):
            bad()
