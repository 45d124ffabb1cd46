"""The decode cache in 8 bits (kernels.Cache8: kv8_append, kv8_fill, seg_attn8) against its float64 restatement
(oracle/low_bits.py) and against the cache in the model's type.  GPU only."""
import copy
import math

import pytest
import torch

from oracle import low_bits as O
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rnd(*shape, seed, dtype=F32, spread=0.7):
    """Values as projections give them: some dimensions larger than others."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    return (x * torch.exp(spread * torch.randn(shape[-1], generator=g))).to(dtype)


def new_cache(B, H, D, leaf, tcap, dtype, seed=0, spare=5, missing=()):
    """A new cache with every block's page handed out in a scrambled order; `missing`: (b, h, j) without one."""
    nb = (tcap + leaf - 1) // leaf
    P = B * H * nb + spare
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(P, generator=g)[:B * H * nb].to(torch.int32).view(B, H, nb).contiguous()
    for m in missing:
        table[m] = -1
    pool = torch.zeros(P, 2, leaf, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    c = K.Cache8(pool, torch.ones(P, 2, device=DEV), table.to(DEV), torch.zeros(B, H, 2, leaf, D, device=DEV, dtype=dtype),
                 torch.full((B, H), -1, dtype=torch.int32, device=DEV), tcap)
    o = O.Cache(B, H, D, leaf, tcap, table >= 0)
    return c, o


def same(c, o):
    """The kernel's cache holds the restatement's numbers, bit for bit (also NaN where there is one)."""
    pool, scale, table = c.pool.cpu().float().double(), c.scale.cpu(), c.table.cpu()
    tail, held = c.tail.cpu().double(), c.tail_block.cpu()
    for b in range(o.B):
        for h in range(o.H):
            assert held[b, h] == o.held[b][h], (b, h)
            if o.held[b][h] >= 0:
                assert torch.equal(torch.nan_to_num(tail[b, h], nan=7e7, posinf=8e7, neginf=-8e7),
                                   torch.nan_to_num(o.tail[b, h], nan=7e7, posinf=8e7, neginf=-8e7)), (b, h)
            for j, (codes, sc) in o.blocks[b][h].items():
                pg = int(table[b, h, j])
                assert scale[pg].tolist() == sc, (b, h, j)
                assert torch.equal(torch.nan_to_num(pool[pg], nan=999.0), torch.nan_to_num(codes, nan=999.0)), (b, h, j)


def put(c, o, kk, vv, t, levels=(), arity=2):
    """Append kk, vv (B,H,D) at positions t (list) to both."""
    K.kv8_append(kk.to(DEV), vv.to(DEV), c, torch.tensor(t, dtype=torch.int32, device=DEV), list(levels), arity)
    for b in range(o.B):
        for h in range(o.H):
            o.append(b, h, t[b], kk[b, h], vv[b, h])


@pytest.mark.parametrize('dtype,D,leaf,arity', [(F32, 64, 8, 2), (BF16, 64, 64, 2), (BF16, 128, 16, 4), (F16, 32, 2, 2),
                                                (F16, 16, 32, 2), (F32, 128, 128, 2), (BF16, 16, 2, 4)])
def test_append_token_by_token(dtype, D, leaf, arity):
    """Pages, scales and tail are the restatement's after every block; the nodes are those of kv_append on a cache in
    the model's type, bit for bit."""
    B, H, tcap = 2, 3, 8 * leaf if leaf > 8 else 64
    c, o = new_cache(B, H, D, leaf, tcap, dtype, seed=leaf)
    shape = K.TreeShape(tcap, leaf, arity)
    lv = [t.zero_() for t in shape.alloc_levels(B, H, D, DEV)]
    ref = [t.zero_() for t in shape.alloc_levels(B, H, D, DEV)]
    Kd = torch.zeros(B, H, tcap, D, device=DEV, dtype=dtype)
    Vd = torch.zeros_like(Kd)
    n = 3 * leaf + leaf // 2 if leaf > 8 else tcap
    kk, vv = rnd(n, B, H, D, seed=1, dtype=dtype), rnd(n, B, H, D, seed=2, dtype=dtype)
    for t in range(n):
        put(c, o, kk[t], vv[t], [t] * B, lv, arity)
        K.kv_append(kk[t].to(DEV), vv[t].to(DEV), Kd, Vd, torch.full((B,), t, dtype=torch.int32, device=DEV), ref, leaf,
                    arity)
        if (t + 1) % leaf == 0 and t < 6 * leaf:
            same(c, o)
    same(c, o)
    for a, e in zip(lv, ref):
        assert torch.equal(a, e)


def test_append_ragged_positions_missing_pages_and_bounds():
    """Sequences at positions of their own; a block without a page, a negative position and one past tcap store nothing."""
    B, H, D, leaf, tcap = 4, 2, 64, 16, 70          # tcap inside the last block
    c, o = new_cache(B, H, D, leaf, tcap, BF16, missing=[(1, 0, 1), (2, 1, 0)])
    before = c.pool.view(torch.uint8).clone()
    spare = sorted(set(range(c.pool.shape[0])) - set(c.table.cpu().flatten().tolist()))
    at = [0, 10, -1, 60]
    for i in range(30):
        kk, vv = rnd(B, H, D, seed=3 + i, dtype=BF16), rnd(B, H, D, seed=300 + i, dtype=BF16)
        put(c, o, kk, vv, [a + i for a in at])
    same(c, o)
    assert torch.equal(c.pool.view(torch.uint8)[spare], before[spare])


def test_going_back_restores_the_block_from_its_page():
    B, H, D, leaf, tcap = 2, 2, 32, 8, 64
    for dtype in (F32, F16, BF16):
        c, o = new_cache(B, H, D, leaf, tcap, dtype)
        for t in range(21):
            put(c, o, rnd(B, H, D, seed=t, dtype=dtype), rnd(B, H, D, seed=50 + t, dtype=dtype), [t] * B)
        for t in (11, 12, 13, 14, 15, 16, 3):       # back inside block 1, on through its end, then back into block 0
            put(c, o, rnd(B, H, D, seed=90 + t, dtype=dtype), rnd(B, H, D, seed=120 + t, dtype=dtype), [t] * B)
            for b in range(B):
                for h in range(H):
                    r = t % leaf + 1
                    assert torch.equal(c.tail[b, h, :, :r].cpu().double(), o.tail[b, h, :, :r]), (dtype, t)
        for b in range(B):
            for h in range(H):
                codes, sc = o.blocks[b][h][1]
                pg = int(c.table[b, h, 1])
                assert c.scale[pg].tolist() == sc and torch.equal(c.pool[pg].cpu().float().double(), codes)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_scales_zeros_extremes_and_what_is_not_finite(dtype):
    """All zeros, one tiny or huge value, exactly 448 times a power of two and just above it, infinities and NaN."""
    D, leaf = 16, 4
    big = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    rows = [0.0, big, -big, tiny, -tiny / 4, 448.0, 448.0 * 2 ** -6, 449.0, 1e-3, float('inf'), float('-inf'), float('nan')]
    B, H = len(rows), 2
    for start in ('append', 'fill'):
        c, o = new_cache(B, H, D, leaf, 2 * leaf, dtype)
        kk = torch.zeros(leaf, B, H, D, dtype=dtype)
        vv = torch.zeros(leaf, B, H, D, dtype=dtype)
        for b, x in enumerate(rows):
            kk[1, b, 0, 3] = x
            vv[2, b, 1, 5] = x
            kk[3, b, 0, 0] = 0.7 * (x if math.isfinite(x) else 3.0)
        for t in range(leaf):
            for b in range(B):
                for h in range(H):
                    o.append(b, h, t, kk[t, b, h], vv[t, b, h])
        if start == 'append':
            for t in range(leaf):
                K.kv8_append(kk[t].to(DEV), vv[t].to(DEV), c, torch.full((B,), t, dtype=torch.int32, device=DEV), [], 2)
        else:
            K.kv8_fill(kk.permute(1, 2, 0, 3).to(DEV), vv.permute(1, 2, 0, 3).to(DEV), c)
            o.held = [[-1] * H for _ in range(B)]
        same(c, o)


@pytest.mark.parametrize('dtype,D,leaf', [(F32, 64, 8), (BF16, 64, 64), (BF16, 128, 16), (F16, 32, 2), (F32, 128, 256),
                                          (F16, 16, 2), (BF16, 64, 2048)])
def test_fill_equals_append(dtype, D, leaf):
    """Prompts of every kind of length give the bytes of their tokens one by one, and leave the rest alone."""
    H, T = 2, 3 * leaf + 1 if leaf > 512 else 5 * leaf + leaf // 2
    lens = [0, 1, leaf - 1, leaf, leaf + 1, T, T + 5, -3, 2 * leaf]
    B = len(lens)
    c, o = new_cache(B, H, D, leaf, 8 * leaf, dtype, missing=[(4, 0, 0), (4, 1, 1), (8, 1, 1)])
    c.pool.view(torch.uint8).fill_(0x31)
    c.scale.fill_(0.5)
    c.tail.fill_(3.0)
    c.tail_block.fill_(7)
    qkv = rnd(B, T, 3, H, D, seed=5, dtype=dtype).to(DEV)      # views of one projection, rows far apart
    k, v = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    K.kv8_fill(k, v, c, torch.tensor(lens, dtype=torch.int32, device=DEV))
    kc, vc = k.cpu(), v.cpu()
    pool, scale = c.pool.cpu(), c.scale.cpu()
    written = torch.zeros(pool.shape[0], dtype=torch.bool)
    for b, n in enumerate(lens):
        n = min(max(n, 0), T)
        for h in range(H):
            rest = n % leaf
            for j in range(n // leaf):
                pg = int(c.table[b, h, j])
                if pg < 0:
                    continue
                written[pg] = True
                rows = torch.stack((kc[b, h, j * leaf:(j + 1) * leaf], vc[b, h, j * leaf:(j + 1) * leaf])).double()
                sc = [O.scale8(rows[0]), O.scale8(rows[1])]
                assert scale[pg].tolist() == sc
                codes = torch.stack([O.round8(rows[i] / sc[i]) for i in (0, 1)])
                assert torch.equal(pool[pg].float().double(), codes), (b, h, j)
            j = n // leaf
            paged = rest > 0 and int(c.table[b, h, j]) >= 0
            assert int(c.tail_block[b, h]) == (j if paged else -1), (b, h)
            want = torch.full((2, leaf, D), 3.0, dtype=dtype)
            if paged:
                want[0, :rest], want[1, :rest] = kc[b, h, j * leaf:n], vc[b, h, j * leaf:n]
            assert torch.equal(c.tail[b, h].cpu(), want), (b, h)
    assert (pool.view(torch.uint8)[~written] == 0x31).all() and (scale[~written] == 0.5).all()


# ------------------------------------------------------------------------------------------------ attention
def bound(dtype, out, q, kmax, vmax, n, scale):
    """How far a float32 evaluation rounded to dtype may be from the exact result.  A score is a sum of D products
    (D + 3 roundings of 2^-24 of the sum of their magnitudes, S), its exponential is exp2 of a float32 product
    (|s| <= S: another S * 2^-23, and 2^-21 for the instruction), the sums over n keys add n * 2^-24 each; weights that
    are off by a factor 1 + d move a weighted mean of values by at most 2 d max|v|."""
    D = q.shape[-1]
    S = scale * float(q.abs().sum(-1).max()) * kmax
    d = S * ((D + 3) * 2.0 ** -24 + 2.0 ** -22) + 2.0 ** -20 + 2 * n * 2.0 ** -24
    return torch.finfo(dtype).eps / 2 * out.abs() + 2 * d * vmax + 2.0 ** -24


def filled(B, H, D, leaf, tcap, n, dtype, seed=0, missing=()):
    """A cache after n[b] tokens of every sequence, kernel's and restatement's."""
    c, o = new_cache(B, H, D, leaf, tcap, dtype, seed=seed, missing=missing)
    T = max(n)
    k, v = rnd(B, H, T, D, seed=seed + 1, dtype=dtype), rnd(B, H, T, D, seed=seed + 2, dtype=dtype)
    K.kv8_fill(k.to(DEV), v.to(DEV), c, torch.tensor(n, dtype=torch.int32, device=DEV))
    for b in range(B):
        for h in range(H):
            for t in range(n[b]):
                o.append(b, h, t, k[b, h, t], v[b, h, t])
            if n[b] % leaf == 0:
                o.held[b][h] = -1
    return c, o, float(k.abs().max()) * 1.07, float(v.abs().max()) * 1.07


def leaves_for(tq, B, H, wl, leaf, seed):
    """Distinct blocks before each query's own one, as many as there are up to wl."""
    g = torch.Generator().manual_seed(seed)
    Nq = tq.shape[-1]
    ids = torch.full((B, H, Nq, wl), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(H):
            for i in range(Nq):
                own = max(int(tq[b, i]), 0) // leaf
                p = torch.randperm(own, generator=g)[:wl]
                ids[b, h, i, :len(p)] = p.to(torch.int32)
    return ids, ids >= 0


def check(c, o, q, tq, ids, vld, n_tree, local, kmax, vmax, nsplit, nb=None, ws=None, out=None):
    B, H, Nq, D = q.shape
    scale = 1 / math.sqrt(D)
    lse = torch.empty(B, H, Nq, device=DEV)
    keys = torch.empty(B, H, Nq, device=DEV)
    got, _, _ = K.seg_attn8(q.to(DEV) if not q.is_cuda else q, c, tq.to(torch.int32).to(DEV), ids.to(DEV), vld.to(DEV),
                            None if n_tree is None else n_tree.to(torch.int32).to(DEV), local, scale, lse=lse, keys=keys,
                            nsplit=nsplit, nb=None if nb is None else tuple(x.to(DEV) for x in nb), ws=ws, out=out)
    got, lse, keys, qc = got.cpu().double(), lse.cpu(), keys.cpu(), q.cpu().double()
    for b in range(B):
        for h in range(H):
            for i in range(Nq):
                t = int(tq[b, i]) if tq.dim() == 2 else int(tq[i])
                nv = int(vld[b, h, i].sum())
                nt = nv if n_tree is None else max(0, min(nv, int(n_tree[b, h, i])))
                near = [] if nb is None else [int(x) for x, m in zip(nb[0][b, h, i], nb[1][b, h, i]) if m]
                want, wl, n = O.attend8(o, qc[b, h, i], b, h, t, ids[b, h, i, :nt].tolist(), near, local, scale)
                where = (b, h, i, t)
                assert int(keys[b, h, i]) == n, where
                tol = bound(c.dtype, want, qc[b, h, i], kmax, vmax, n, scale)
                assert ((got[b, h, i] - want).abs() <= tol).all(), (where, float((got[b, h, i] - want).abs().max()))
                S = scale * float(qc[b, h, i].abs().sum()) * kmax
                assert abs(float(lse[b, h, i]) - wl) <= S * (D + 8) * 2.0 ** -23 + 2.0 ** -18 + abs(wl) * 2.0 ** -23, where
    return got


@pytest.mark.parametrize('dtype,D,leaf,wl,nsplit', [
    (BF16, 64, 64, 4, 4), (BF16, 64, 32, 8, 16), (F16, 128, 16, 16, 4), (F32, 64, 8, 5, 8), (F32, 128, 32, 3, 1),
    (F16, 32, 2, 8, 4), (BF16, 16, 4, 7, 1), (F32, 16, 64, 2, 64), (BF16, 128, 128, 2, 4), (F16, 64, 2, 70, 12)])
@pytest.mark.parametrize('Nq', [1, 3])
def test_attention(dtype, D, leaf, wl, nsplit, Nq):
    """Ragged sequences -- one token, inside the first block, at a block's first and last position, long -- single
    queries and several positions at once, with a budget of leaves per query."""
    H = 2
    tcap = 16 * leaf if leaf > 4 else 256
    n = [1, 2, leaf, leaf + 1, 2 * leaf + leaf // 2, tcap - 3, tcap]
    B = len(n)
    c, o, kmax, vmax = filled(B, H, D, leaf, tcap, n, dtype, seed=leaf + D)
    tq = torch.tensor(n).view(B, 1) - Nq + torch.arange(Nq)      # some negative: those attend nothing
    ids, vld = leaves_for(tq, B, H, wl, leaf, seed=D)
    q = rnd(B, Nq, H, D, seed=9, dtype=dtype).transpose(1, 2)
    nt = torch.randint(0, wl + 1, (B, H, Nq), generator=torch.Generator().manual_seed(4))
    check(c, o, q, tq, ids, vld, nt, 3, kmax, vmax, nsplit)
    check(c, o, q, tq, ids, vld, None, 5, kmax, vmax, nsplit)


def test_attention_with_neighbours_missing_pages_and_bad_ids():
    """Matched neighbour leaves join once; a block without a page and an id outside the table contribute nothing."""
    B, H, D, leaf, tcap, wl, S = 2, 3, 64, 8, 128, 4, 6
    n = [77, 100]
    c, o, kmax, vmax = filled(B, H, D, leaf, tcap, n, BF16, missing=[(0, 1, 2), (1, 0, 0), (1, 2, 12)])
    tq = torch.tensor(n).view(B, 1) - 1
    ids, vld = leaves_for(tq, B, H, wl, leaf, seed=3)
    ids[0, 1, 0, 1] = 2
    g = torch.Generator().manual_seed(8)
    nid = torch.randint(0, 16, (B, H, 1, S), generator=g, dtype=torch.int32)
    nid[0, 0, 0, 2] = nid[0, 0, 0, 1]
    nid[1, 1, 0, 0] = ids[1, 1, 0, 0]
    ok = torch.rand(B, H, 1, S, generator=g) < 0.7
    for nsplit in (1, 4, 8):
        check(c, o, rnd(B, H, 1, D, seed=1, dtype=BF16), tq, ids, vld, None, 3, kmax, vmax, nsplit, nb=(nid, ok))
    bad = ids.clone()
    bad[0, 0, 0, 0], bad[1, 1, 0, 1] = 10 ** 6, 16               # past the table: skipped (still counted as keys)
    out, _, _ = K.seg_attn8(rnd(B, H, 1, D, seed=1, dtype=BF16).to(DEV), c, tq.to(torch.int32).to(DEV), bad.to(DEV),
                            vld.to(DEV), None, 3, 0.125, nsplit=4)
    assert torch.isfinite(out).all()


def test_attention_reads_the_tail_for_the_block_it_holds():
    """The block in the tail is read from there when it is the own block, a selected one or a static key's."""
    B, H, D, leaf, tcap = 3, 2, 64, 8, 64
    c, o = new_cache(B, H, D, leaf, tcap, F32)
    kk, vv = rnd(40, B, H, D, seed=1), rnd(40, B, H, D, seed=2)
    for t in range(32):
        put(c, o, kk[t], vv[t], [t] * B)            # the tail holds block 3, whole
    tq = torch.tensor([[31], [33], [34]])           # own; static and selected below; static
    ids = torch.tensor([[[[1, 0]]], [[[3, 1]]], [[[0, 2]]]], dtype=torch.int32).expand(B, H, 1, 2).contiguous()
    vld = torch.ones_like(ids, dtype=torch.bool)
    # rows 32.. are not written yet: their page is zeros, as a page handed out is
    for nsplit in (1, 4, 16):
        check(c, o, rnd(B, H, 1, D, seed=4), tq, ids, vld, None, 3, float(kk.abs().max()), float(vv.abs().max()), nsplit)


def test_masked_places_may_hold_anything():
    """NaN and infinities in rows past the position, in pages that are not selected and in invalid slots change nothing;
    in a selected row they make the result NaN."""
    B, H, D, leaf, tcap = 1, 2, 64, 16, 128
    c, o, kmax, vmax = filled(B, H, D, leaf, tcap, [101], BF16)
    tq = torch.tensor([[100]])
    ids, vld = leaves_for(tq, B, H, 3, leaf, seed=1)
    vld[0, :, 0, 2] = False
    c.tail[:, :, :, 101 % leaf:] = float('nan')
    sel = {(h, int(j)) for h in range(H) for j in ids[0, h, 0, :2]} | {(h, 6) for h in range(H)}
    sel |= {(h, 0) for h in range(H)}               # position 0
    raw = c.pool.view(torch.uint8)
    for h in range(H):
        for j in range(6):
            if (h, j) not in sel:
                raw[int(c.table[0, h, j])] = 0x7f
    q = rnd(B, H, 1, D, seed=2, dtype=BF16)
    for nsplit in (1, 4, 8):
        check(c, o, q, tq, ids, vld, None, 3, kmax, vmax, nsplit)
    raw[int(c.table[0, 1, int(ids[0, 1, 0, 0])]), 0, 3, 5] = 0x7f
    for nsplit in (1, 4, 8):
        out, _, _ = K.seg_attn8(q.to(DEV), c, tq.to(torch.int32).to(DEV), ids.to(DEV), vld.to(DEV), None, 3, 0.125,
                                nsplit=nsplit)
        assert torch.isnan(out[0, 1]).all() and torch.isfinite(out[0, 0]).all(), nsplit


def test_attention_strides_streams_and_views():
    """q and out as views of larger buffers, part of the sequences, the call on another stream, a shared position list."""
    B, H, D, leaf, tcap = 4, 2, 64, 16, 256
    n = [40, 41, 250, 256]
    c, o, kmax, vmax = filled(B, H, D, leaf, tcap, n, F16)
    o.blocks, o.tail, o.held, o.pages, o.B = o.blocks[2:], o.tail[2:], o.held[2:], o.pages[2:], 2
    part = c.rows(2, 4)
    tq = torch.tensor([245, 249])
    ids, vld = leaves_for(tq.expand(2, 2), 2, H, 5, leaf, seed=2)
    buf = torch.zeros(2, 2, H + 1, 3 * D, device=DEV, dtype=F16)
    qv = buf[:, :, :H, D:2 * D].transpose(1, 2)
    qv.copy_(rnd(2, H, 2, D, seed=6, dtype=F16))
    outb = torch.full((2, 2, H, D + 3), 9.0, device=DEV, dtype=F16)
    out = outb[..., :D].transpose(1, 2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        check(part, o, qv, tq, ids, vld, None, 3, kmax, vmax, 8, out=out)
    s.synchronize()
    assert (outb[..., D:] == 9.0).all()


def test_append_and_attention_in_a_replayed_graph():
    """A captured step (append, attention) replayed over positions that cross blocks gives the eager steps' bits."""
    B, H, D, leaf, tcap, wl = 2, 3, 64, 8, 128, 4
    shape = K.TreeShape(tcap, leaf, 2)
    kk, vv = rnd(40, B, H, D, seed=1, dtype=BF16).to(DEV), rnd(40, B, H, D, seed=2, dtype=BF16).to(DEV)
    qq = rnd(40, B, H, 1, D, seed=3, dtype=BF16).to(DEV)
    runs = []
    for graph in (False, True):
        c, _ = new_cache(B, H, D, leaf, tcap, BF16)
        lv = [t.zero_() for t in shape.alloc_levels(B, H, D, DEV)]
        k, v, q = kk[0].clone(), vv[0].clone(), qq[0].clone()
        t = torch.zeros(B, dtype=torch.int32, device=DEV)
        ids = torch.zeros(B, H, 1, wl, dtype=torch.int32, device=DEV)
        vld = torch.zeros(B, H, 1, wl, dtype=torch.uint8, device=DEV)
        out = torch.empty(B, H, 1, D, device=DEV, dtype=BF16)
        ws = K.seg_attn8_workspace(B, H, 1, D, 16, DEV)

        def step():
            K.kv8_append(k, v, c, t, lv, 2)
            K.seg_attn8(q, c, t.view(B, 1), ids, vld, None, 3, 0.125, out=out, nsplit=16, ws=ws)
        outs = []
        if graph:
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
            torch.cuda.current_stream().wait_stream(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step()
        for i in range(40):
            k.copy_(kk[i]); v.copy_(vv[i]); q.copy_(qq[i]); t.fill_(i)
            if i // leaf:
                ids.copy_((torch.arange(wl, device=DEV) % (i // leaf)).expand_as(ids))
                vld.copy_((torch.arange(wl, device=DEV) < i // leaf).expand_as(vld))
            g.replay() if graph else step()
            torch.cuda.synchronize()
            outs.append(out.clone())
        runs.append((torch.stack(outs), c.pool.view(torch.uint8).clone(), c.scale.clone(), c.tail.clone(), *lv))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_dense_copies():
    B, H, D, leaf, tcap = 2, 2, 32, 8, 64
    c, o, _, _ = filled(B, H, D, leaf, tcap, [29, 16], BF16, missing=[(0, 1, 1)])
    for b, n in ((0, 29), (1, 16)):
        k, v = c.dense(b, n)
        assert k.shape == (1, H, n, D)
        for h in range(H):
            for t in range(n):
                kv = o.key(b, h, t)
                kv = torch.zeros(2, D, dtype=torch.float64) if kv is None else kv
                assert torch.equal(k[0, h, t].cpu().double(), kv[0]) and torch.equal(v[0, h, t].cpu().double(), kv[1])


def test_refusals():
    B, H, D, leaf, tcap = 2, 2, 64, 16, 64
    c, _ = new_cache(B, H, D, leaf, tcap, BF16)
    k = torch.zeros(B, H, D, device=DEV, dtype=BF16)
    t = torch.zeros(B, dtype=torch.int32, device=DEV)
    with pytest.raises(TypeError, match='dtype'):
        K.kv8_append(k.float(), k.float(), c, t, [], 2)
    with pytest.raises(ValueError, match='positions'):
        K.kv8_append(k, k, c, t.long(), [], 2)
    with pytest.raises(ValueError, match='rows of'):
        K.kv8_append(k[:1], k[:1], c, t, [], 2)
    with pytest.raises(ValueError, match='levels'):
        K.kv8_append(k, k, c, t, [torch.zeros(B, H, 3, D, device=DEV)], 2)
    with pytest.raises(RuntimeError, match='GPU'):
        K.kv8_append(k.cpu(), k.cpu(), c, t, [], 2)
    with pytest.raises(ValueError, match='tcap'):
        K.kv8_fill(torch.zeros(B, H, 65, D, device=DEV, dtype=BF16), torch.zeros(B, H, 65, D, device=DEV, dtype=BF16), c)
    odd = torch.zeros(B, H, 4, D + 1, device=DEV, dtype=BF16)[..., 1:]
    with pytest.raises(RuntimeError, match='16-byte'):
        K.kv8_fill(odd, odd, c)
    q = torch.zeros(B, H, 1, D, device=DEV, dtype=BF16)
    ids = torch.zeros(B, H, 1, 4, dtype=torch.int32, device=DEV)
    vld = torch.zeros(B, H, 1, 4, dtype=torch.uint8, device=DEV)
    with pytest.raises(RuntimeError, match='multiple of 4'):
        K.seg_attn8(q, c, t.view(B, 1), ids, vld, None, 3, 1.0, nsplit=6)
    with pytest.raises(RuntimeError, match='local window'):
        K.seg_attn8(q, c, t.view(B, 1), ids, vld, None, 40, 1.0)
    with pytest.raises(RuntimeError, match='16-byte'):
        K.seg_attn8(torch.zeros(B, H, 1, D + 1, device=DEV, dtype=BF16)[..., 1:], c, t.view(B, 1), ids, vld, None, 3, 1.0)
    with pytest.raises(ValueError, match='ids'):
        K.seg_attn8(q, c, t.view(B, 1), ids.long(), vld, None, 3, 1.0)
    with pytest.raises(RuntimeError, match='workspace'):
        K.seg_attn8(q, c, t.view(B, 1), ids, vld, None, 3, 1.0, nsplit=16, ws=torch.zeros(256, dtype=torch.uint8, device=DEV))


def test_copies_hold_their_own_tensors():
    pool = torch.zeros(3, 2, 8, 16, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    c = K.Cache8(pool, torch.ones(3, 2, device=DEV), torch.tensor([[[2, 0]]], dtype=torch.int32, device=DEV),
                 torch.zeros(1, 1, 2, 8, 16, device=DEV), torch.full((1, 1), -1, dtype=torch.int32, device=DEV), 16)
    d = copy.deepcopy(c)
    row = torch.randn(1, 1, 16, generator=torch.Generator().manual_seed(1)).to(DEV)
    K.kv8_append(row, row, d, torch.zeros(1, dtype=torch.int32, device=DEV), [], 2)
    assert torch.equal(d.tail[0, 0, 1, 0], row[0, 0]) and int(d.tail_block) == 0
    assert not c.tail.any() and int(c.tail_block) == -1 and c.desc.tail != d.desc.tail
    with pytest.raises(AttributeError):
        c.table = d.table
