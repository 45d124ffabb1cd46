"""The operators that serve a decoder in fewer bits, as cases to time and check them on.

listed() is the fixed set, draw() gives more of the same ranges, prepare() makes what a program holds before the call,
run() makes one call (the operators' plain form in torch, or with `own` the package's kernels), work() says what a call
cannot do without and exact() gives its result in float64.

Kinds of case:
  append  one token of every sequence into a cache of 8-bit pages (one power-of-two scale for the keys and one for the
          values of each page), with the tree nodes it completes
  fill    prompts of several lengths into such a cache
  attend  attention over the selected leaf blocks of such a cache, the own block and the static keys
  quant   rows rounded to microscaled 4-bit floats (blocks of 32 along a row, one power-of-two scale each)
  rows    bf16 rows times 4-bit weights, with the LayerNorm, GELU or residual around it (a decode step, a prompt)
  both    rows rounded to 4 bits on the way in, times 4-bit weights
"""
import math

import torch

own = False
DT = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
DEV = 'cuda'
LOCAL = 3          # static keys besides position 0: the last three positions
EPS = 1e-5


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # a layer's share of one decode step: 32 sequences of some thousand tokens, a few of them ending a block
        dict(name='append_step', kind='append', dtype='bf16', batch=32, heads=12, dh=64, context=2500, tcap=4096,
             leaf=64, arity=2, at='any'),
        # the smallest call: one sequence whose token ends its block, so the page and its nodes are written
        dict(name='append_one', kind='append', dtype='f32', batch=1, heads=6, dh=64, context=600, tcap=1024, leaf=32,
             arity=2, at='end'),
        # prompts of unequal lengths taken into one layer's cache
        dict(name='fill_prompts', kind='fill', dtype='bf16', batch=8, heads=12, dh=64, context=8191, tcap=16384,
             leaf=64, arity=2),
        # the headline decode step: 32 sequences of about 32768 tokens, 32 blocks of 64 selected
        dict(name='attend_batch', kind='attend', dtype='bf16', batch=32, heads=12, dh=64, context=32768, tcap=65536,
             leaf=64, wmax=32, queries=1),
        # a single stream over a long context
        dict(name='attend_long', kind='attend', dtype='bf16', batch=1, heads=12, dh=64, context=131000, tcap=262144,
             leaf=128, wmax=64, queries=1),
        # some positions at once (a drafted run of tokens), half precision, wide heads, small blocks
        dict(name='attend_run', kind='attend', dtype='f16', batch=4, heads=8, dh=128, context=6001, tcap=8192, leaf=16,
             wmax=16, queries=5),
        # the activations of a few rows of odd width
        dict(name='quant_rows', kind='quant', dtype='bf16', rows=37, width=1000),
        # a large weight matrix, rounded once when a model is loaded
        dict(name='quant_weight', kind='quant', dtype='f32', rows=16384, width=4096),
        # a single sequence's output projection with its residual
        dict(name='rows_one', kind='rows', rows=1, width=1024, cols=1024, ln=False, epilogue='residual'),
        # 32 sequences through a wide layer: LayerNorm, product, GELU
        dict(name='rows_step', kind='rows', rows=32, width=4096, cols=16384, ln=True, epilogue='gelu'),
        # a prompt of odd length through a layer with bf16 activations
        dict(name='rows_prompt', kind='rows', rows=2001, width=2048, cols=8192, ln=False, epilogue=''),
        # prompts with 4-bit activations
        dict(name='both_prompt', kind='both', dtype='bf16', rows=4096, width=4096, cols=8192),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['append', 'fill', 'attend', 'attend', 'quant', 'rows', 'rows', 'both'])
    dt = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    if kind in ('append', 'fill', 'attend'):
        leaf = rng.choice([2, 8, 16, 32, 64, 64, 128])
        c = dict(kind=kind, dtype=dt, heads=rng.randint(1, 12), dh=rng.choice([16, 32, 64, 64, 128]), leaf=leaf)
    if kind == 'attend':
        c.update(wmax=rng.choice([4, 8, 16, 32, 64]), queries=rng.choice([1, 1, 1, 2, 5, 8]),
                 context=_log_int(rng, 1 + 8, 60000))
        c['batch'] = max(1, min(_log_int(rng, 1, 32), (1 << 24) // (c['context'] * c['heads'] * c['dh'] // 64)))
        c['tcap'] = 1 << max(c['context'] + 16, 2 * leaf).bit_length()
        return c
    if kind in ('append', 'fill'):
        c.update(context=_log_int(rng, 4, 8000), arity=rng.choice([2, 2, 4]), batch=_log_int(rng, 1, 32))
        c['batch'] = max(1, min(c['batch'], (1 << 22) // (c['context'] * c['heads'] * c['dh'] // 64 + 1)))
        c['tcap'] = 1 << max(c['context'] + 16, 2 * leaf).bit_length()
        if kind == 'append':
            c['at'] = rng.choice(['any', 'end', 'start'])
        return c
    if kind == 'quant':
        width = _log_int(rng, 1, 8192)
        return dict(kind=kind, dtype=dt, rows=_log_int(rng, 1, min(65536, (1 << 25) // width)), width=width)
    width, cols = 32 * _log_int(rng, 2, 256), _log_int(rng, 17, 16384)
    rows = _log_int(rng, 1, min(4096, max(33, (1 << 36) // (width * cols))))
    if kind == 'both':
        return dict(kind=kind, dtype=dt, rows=rows, width=width - rng.choice([0, 0, 1, 17]), cols=cols)
    return dict(kind=kind, rows=rows, width=width, cols=cols, ln=rows <= 64 and rng.random() < 0.5,
                epilogue=rng.choice(['', 'gelu', 'residual']))


# ------------------------------------------------------------------------------------------ inputs and handles
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(7919 * (seed + 1))


def _lens(c, seed):
    """Tokens each sequence holds: up to a quarter short of the context."""
    g = torch.Generator().manual_seed(104729 * (seed + 3))
    n = c['context'] - torch.randint(0, max(1, c['context'] // 4), (c['batch'],), generator=g)
    leaf = c['leaf']
    if c.get('at') == 'end':
        n = n // leaf * leaf + leaf - 1
    elif c.get('at') == 'start':
        n = n // leaf * leaf
    return [int(x) for x in n]


def _rows(c, g, n):
    """(H, n, D) keys and values as projections give them: some dimensions far larger than others."""
    H, D = c['heads'], c['dh']
    gain = torch.exp(0.7 * torch.randn(2, H, 1, D, generator=g, device=DEV))
    return (torch.randn(2, H, n, D, generator=g, device=DEV) * gain).to(DT[c['dtype']])


def _cache(c, seed, lens, extra, filled=True):
    """The cache after `lens` tokens of every sequence, with pages (in a shuffled order) for `extra` more."""
    g = _gen(seed)
    B, H, D, leaf = c['batch'], c['heads'], c['dh'], c['leaf']
    nb = [(n + extra + leaf - 1) // leaf for n in lens]
    P = B * H * (c['context'] // leaf + 2) + 3            # as many as the longest sequences take, and spare ones
    order = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    s = dict(pool=torch.zeros(P, 2, leaf, D, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn),
             scale=torch.ones(P, 2, device=DEV),
             table=torch.full((B, H, c['tcap'] // leaf), -1, dtype=torch.int32, device=DEV),
             tail=torch.zeros(B, H, 2, leaf, D, device=DEV, dtype=DT[c['dtype']]),
             tail_block=torch.full((B, H), -1, dtype=torch.int32, device=DEV))
    at = 0
    for b in range(B):
        s['table'][b, :, :nb[b]] = order[at:at + H * nb[b]].view(H, nb[b])
        at += H * nb[b]
        if not filled:
            continue
        whole, rest = divmod(lens[b], leaf)
        x = _rows(c, g, nb[b] * leaf).view(2, H, nb[b], leaf, D)
        if whole:
            codes, scale = _codes8(x[:, :, :whole].float())
            pg = s['table'][b, :, :whole].long()
            s['pool'].view(torch.uint8)[pg] = codes.view(torch.uint8).permute(1, 2, 0, 3, 4)
            s['scale'][pg] = scale.permute(1, 2, 0)
        if rest:
            s['tail'][b, :, :, :rest] = x[:, :, whole, :rest].transpose(0, 1)
            s['tail_block'][b] = whole
    return s


def _select(c, lens, seed):
    """Per query: its position, distinct leaf blocks before its own (as many as there are, up to wmax) and how many of
    them its budget takes."""
    g = _gen(seed + 11)
    B, H, N, leaf, wl = c['batch'], c['heads'], c['queries'], c['leaf'], c['wmax']
    tq = torch.tensor(lens, device=DEV).view(B, 1) - N + torch.arange(N, device=DEV)
    tq = tq.clamp(min=0)
    own_blk = (tq // leaf).view(B, 1, N, 1)
    nblk = max(wl, max(lens) // leaf + 1)
    blocks = torch.arange(nblk, device=DEV)
    r = torch.rand(B, H, N, nblk, generator=g, device=DEV)
    ids = torch.where(blocks < own_blk, r, r + 2).argsort(-1)[..., :wl]
    vld = torch.arange(wl, device=DEV) < own_blk
    ids = torch.where(vld, ids, -1).to(torch.int32).contiguous()
    nt = wl - torch.randint(0, max(1, wl // 8), (B, H, N), generator=g, device=DEV)
    return tq.to(torch.int32), ids, vld.expand(B, H, N, wl).to(torch.uint8).contiguous(), nt.to(torch.int32)


def _levels(c):
    out, l = [], c['leaf'].bit_length() - 1
    while (c['tcap'] >> l) >= 2:
        out.append(torch.zeros(c['batch'], c['heads'], c['tcap'] >> l, c['dh'], device=DEV))
        l += c['arity'].bit_length() - 1
    return out


def prepare(case, seed):
    c, k = case, case['kind']
    s = {'case': c}
    if k in ('append', 'fill', 'attend'):
        lens = _lens(c, seed)
        if k == 'attend':
            lens = [max(n, c['queries']) for n in lens]
        cache = _cache(c, seed, lens, 1 if k == 'append' else 0, filled=k != 'fill')
        s['cache'] = cache
        g = _gen(seed + 5)
        B, H, D = c['batch'], c['heads'], c['dh']
        if k == 'append':
            # views of one projection, as a step has them
            kv = torch.randn(B, 3, H, D, generator=g, device=DEV).to(DT[c['dtype']])
            s.update(k=kv[:, 1], v=kv[:, 2], t=torch.tensor(lens, device=DEV, dtype=torch.int32), levels=_levels(c),
                     arity=c['arity'])
            for i, lv in enumerate(s['levels']):
                lv.normal_(generator=g).mul_(math.sqrt(c['leaf'] * c['arity'] ** i))
        elif k == 'fill':
            kv = torch.randn(B, c['context'], 3, H, D, generator=g, device=DEV).to(DT[c['dtype']])
            s.update(k=kv[:, :, 1].transpose(1, 2), v=kv[:, :, 2].transpose(1, 2),
                     lens=torch.tensor(lens, device=DEV, dtype=torch.int32))
        else:
            s['tq'], s['ids'], s['vld'], s['n_tree'] = _select(c, lens, seed)
            q = torch.randn(B, c['queries'], H, D, generator=g, device=DEV).to(DT[c['dtype']])
            s['q'] = q.transpose(1, 2)
        if own:
            from treeattn_amd import kernels as K
            s['handle'] = K.Cache8(cache['pool'], cache['scale'], cache['table'], cache['tail'], cache['tail_block'],
                                   c['tcap'])
            if k == 'attend':
                from treeattn_amd.engine import decode_nsplit8
                s['nsplit'] = decode_nsplit8(B, H, c['queries'], c['wmax'], c['leaf'])
                s['ws'] = K.seg_attn8_workspace(B, H, c['queries'], D, s['nsplit'], DEV)
        return s
    g = _gen(seed)
    M, n = c['rows'], c['width']
    if k == 'quant':
        x = torch.randn(M, n, generator=g, device=DEV) * torch.exp(torch.randn(M, 1, generator=g, device=DEV))
        s['x'] = x.to(DT[c['dtype']])
        return s
    N = c['cols']
    x = torch.randn(M, n, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(n, generator=g, device=DEV))
    w = torch.randn(N, n, generator=g, device=DEV) * (1 / math.sqrt(n))
    s['x'] = x.to(DT[c.get('dtype', 'bf16')])
    s['packed'], s['wscale'] = _pack4(*_codes4(w))
    if k == 'rows':
        s['ln'] = (1 + 0.1 * torch.randn(n, generator=g, device=DEV)).to(torch.bfloat16) if c['ln'] else None
        s['res'] = (torch.randn(M, N, generator=g, device=DEV).to(torch.bfloat16) if c['epilogue'] == 'residual'
                    else None)
    if own:
        from treeattn_amd import kernels as K
        s['handle'] = K.Mx4(s['packed'], s['wscale'], n)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _pow2(e):
    """2^e in float64, exactly, for whole numbers e (torch's ldexp and exp2 may be an ulp off on the GPU)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _codes8(x):
    """x (..., rows, D) float32 -> e4m3 codes and one scale for the rows: the smallest power of two that brings the
    largest finite magnitude to 448 or less (1 when there is none); what is not finite becomes NaN."""
    ok = torch.isfinite(x)
    amax = torch.where(ok, x.abs(), 0).amax((-1, -2))
    m, e = torch.frexp(amax)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-126, 127)
    e = torch.where(amax > 0, e, 0)
    y = x * _pow2(-e).float()[..., None, None]
    return torch.where(ok, y, float('nan')).to(torch.float8_e4m3fn), _pow2(e).float()


def _codes4(x):
    """x (rows, K) -> (4-bit codes (rows, Kp) uint8, scale bytes (rows, Kp / 32) uint8), Kp the next multiple of 128:
    sign, then the index into 0 .5 1 1.5 2 3 4 6; scale 2^(byte - 127) with byte - 127 = floor(log2 of the block's
    largest magnitude) - 2, at least -127; byte 255 for a block that holds anything not finite."""
    n = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -n % 128)).unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], 0, x)
    amax = x.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(min=-127)
    a = x.abs() * _pow2(-e).float()[..., None]
    v = torch.where(a < 2, torch.round(a * 2) / 2, torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2))
    v = v.clamp(max=6)
    code = torch.where(v < 2, v * 2, torch.where(v < 4, v + 2, v / 2 + 4)).to(torch.uint8)
    code = code | (torch.signbit(x).to(torch.uint8) << 3)
    return code.flatten(-2), torch.where(bad, 255, e + 127).to(torch.uint8)


def _pack4(code, byte):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), byte


def _values4(code, byte, n):
    """float32 values of codes and scale bytes, the first n of each row."""
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=code.device)
    v = grid[(code & 7).long()]
    v = torch.where(code >= 8, -v, v).unflatten(-1, (-1, 32))
    e = byte.int() - 127
    return torch.where((byte == 255)[..., None], float('nan'), v * _pow2(e).float()[..., None]).flatten(-2)[..., :n]


def _unpack4(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _pair_sum(x):
    """Sum over the last but one dimension (a power of two) by adjacent pairs."""
    while x.shape[-2] > 1:
        x = x[..., 0::2, :] + x[..., 1::2, :]
    return x[..., 0, :]


def _append(s):
    c, z = s['case'], s['cache']
    leaf, B = c['leaf'], c['batch']
    t = s['t'].long()
    blk, r = t // leaf, t % leaf
    bi = torch.arange(B, device=DEV)
    z['tail'][bi, :, 0, r] = s['k']
    z['tail'][bi, :, 1, r] = s['v']
    z['tail_block'].copy_(blk.view(B, 1).to(torch.int32).expand_as(z['tail_block']))
    ends = (r == leaf - 1)
    pg = z['table'][bi, :, blk].long()
    codes, scale = _codes8(z['tail'].float())
    pool = z['pool'].view(torch.uint8)
    pool[pg] = torch.where(ends.view(B, 1, 1, 1, 1), codes.view(torch.uint8), pool[pg])
    z['scale'][pg] = torch.where(ends.view(B, 1, 1), scale, z['scale'][pg])
    # the nodes ending at t: a leaf block's keys (position 0 counted as zero), then each node's children
    rows = z['tail'][:, :, 0].float()
    rows = torch.where((blk.view(B, 1) * leaf + torch.arange(leaf, device=DEV) == 0).view(B, 1, leaf, 1), 0, rows)
    x = _pair_sum(rows)
    size = leaf
    for j, lv in enumerate(s['levels']):
        node = t // size
        if j:
            kids = node.view(B, 1) * c['arity'] + torch.arange(c['arity'], device=DEV)
            x = _pair_sum(s['levels'][j - 1][bi.view(B, 1), :, kids].transpose(1, 2))
        done = ((t + 1) % size == 0).view(B, 1, 1)
        lv[bi, :, node] = torch.where(done, x, lv[bi, :, node])
        size *= c['arity']
    return [z['pool'], z['scale'], z['tail'], z['tail_block'], *s['levels']]


def _fill(s):
    c, z = s['case'], s['cache']
    B, H, D, leaf, T = c['batch'], c['heads'], c['dh'], c['leaf'], c['context']
    nb = (T + leaf - 1) // leaf
    kv = torch.stack((s['k'], s['v']), 2)
    kv = torch.nn.functional.pad(kv, (0, 0, 0, nb * leaf - T)).unflatten(3, (nb, leaf))     # (B, H, 2, nb, leaf, D)
    lens = s['lens'].long().view(B, 1, 1)
    codes, scale = _codes8(kv.float())
    pg = z['table'][:, :, :nb].long()
    full = (torch.arange(nb, device=DEV) + 1) * leaf <= lens
    # the last page belongs to no sequence of a case with spare pages: unfinished blocks rewrite what it holds
    spare = torch.ones(z['pool'].shape[0], dtype=torch.bool, device=DEV)
    spare[pg[pg >= 0]] = False
    pg = torch.where(full & (pg >= 0), pg, spare.to(torch.int32).argmax())
    full = full.expand(B, H, nb)
    pool = z['pool'].view(torch.uint8)
    pool[pg] = torch.where(full[..., None, None, None], codes.view(torch.uint8).transpose(2, 3), pool[pg])
    z['scale'][pg] = torch.where(full[..., None], scale.transpose(2, 3), z['scale'][pg])
    part = (s['lens'].long() // leaf).clamp(max=nb - 1)
    rest = (s['lens'].long() % leaf).view(B, 1, 1, 1, 1)
    rows = kv[torch.arange(B, device=DEV), :, :, part]                                      # (B, H, 2, leaf, D)
    z['tail'].copy_(torch.where(torch.arange(leaf, device=DEV).view(leaf, 1) < rest, rows, z['tail']))
    blk = torch.where(s['lens'] % leaf > 0, s['lens'] // leaf, -1)
    z['tail_block'].copy_(blk.view(B, 1).expand(B, H))
    return [z['pool'], z['scale'], z['tail'], z['tail_block']]


def _positions(s):
    """Keys of every query: positions (B,H,N,L) and which of them count."""
    c = s['case']
    leaf, wl = c['leaf'], c['wmax']
    t = s['tq'].long().view(c['batch'], 1, c['queries'], 1)
    t = t.expand(-1, c['heads'], -1, -1)
    first = t // leaf * leaf
    used = torch.minimum(s['vld'].long().sum(-1, keepdim=True), s['n_tree'].long()[..., None])
    live = torch.arange(wl, device=DEV) < used
    inner = torch.arange(leaf, device=DEV)
    tree = (s['ids'].long().clamp(min=0)[..., None] * leaf + inner).flatten(-2)
    mine = first + inner
    stat = torch.cat((torch.zeros_like(t), t - torch.arange(LOCAL, device=DEV)), -1)
    taken = ((s['ids'].long()[..., None, :] == stat[..., None] // leaf) & live[..., None, :]).any(-1)
    ok = (stat >= 0) & (stat < first) & ~taken
    ok[..., 1:] &= stat[..., 1:] != 0
    return (torch.cat((tree, mine, stat.clamp(min=0)), -1),
            torch.cat((live.repeat_interleave(leaf, -1), mine <= t, ok), -1))


def _attend(s):
    c, z = s['case'], s['cache']
    leaf = c['leaf']
    pos, ok = _positions(s)
    B, H, N, L = pos.shape
    bi, hi = (torch.arange(B, device=DEV).view(B, 1, 1, 1), torch.arange(H, device=DEV).view(1, H, 1, 1))
    blk, r = pos // leaf, pos % leaf
    pg = z['table'][bi, hi, blk].long()
    in_tail = (blk == z['tail_block'].view(B, H, 1, 1))
    ok = ok & (in_tail | (pg >= 0))
    pg = pg.clamp(min=0)

    def rows(i):
        x = z['pool'].view(torch.uint8)[pg, i, r].view(torch.float8_e4m3fn).float() * z['scale'][pg, i][..., None]
        return torch.where(in_tail[..., None], z['tail'][bi, hi, i, r].float(), x)
    sc = (rows(0) * s['q'].float()[..., None, :]).sum(-1) * (1 / math.sqrt(c['dh']))
    sc = torch.where(ok, sc, float('-inf'))
    p = torch.exp(sc - sc.amax(-1, keepdim=True))
    out = (p[..., None] * rows(1)).sum(-2) / p.sum(-1, keepdim=True)
    return out.to(s['q'].dtype)


def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))


def _product(s):
    c = s['case']
    x = s['x'].float()
    n = c['width']
    if c['kind'] == 'both':
        x = _values4(*_codes4(x), n)
    elif s['ln'] is not None:
        x = x - x.mean(-1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * s['ln'].float()
    y = x @ _values4(_unpack4(s['packed']), s['wscale'], n).T
    if c.get('epilogue') == 'gelu':
        y = _gelu(y)
    elif c.get('epilogue') == 'residual':
        y = y + s['res'].float()
    return y.to(torch.bfloat16)


def run(state):
    s = state
    k = s['case']['kind']
    if own:
        from treeattn_amd import kernels as K
        if k == 'append':
            K.kv8_append(s['k'], s['v'], s['handle'], s['t'], s['levels'], s['arity'])
            z = s['cache']
            return [z['pool'], z['scale'], z['tail'], z['tail_block'], *s['levels']]
        if k == 'fill':
            K.kv8_fill(s['k'], s['v'], s['handle'], s['lens'])
            z = s['cache']
            return [z['pool'], z['scale'], z['tail'], z['tail_block']]
        if k == 'attend':
            return K.seg_attn8(s['q'], s['handle'], s['tq'], s['ids'], s['vld'], s['n_tree'], LOCAL,
                               1 / math.sqrt(s['case']['dh']), nsplit=s['nsplit'], ws=s['ws'])[0]
        if k == 'quant':
            return K.mx4_quant(s['x'], values=True)[1]
        if k == 'both':
            return K.mx4_mm(K.mx4_quant(s['x']), s['handle'])
        return K.mx4_mm(s['x'], s['handle'], ln_w=s['ln'], eps=EPS, epilogue=s['case']['epilogue'] or None,
                        residual=s['res'])
    if k == 'append':
        return _append(s)
    if k == 'fill':
        return _fill(s)
    if k == 'attend':
        return _attend(s)
    if k == 'quant':
        return _values4(*_codes4(s['x']), s['case']['width']).to(s['x'].dtype)
    return _product(s)


# -------------------------------------------------------------------------------------------------- their work
def work(case):
    c, k = case, case['kind']
    size = 4 if c.get('dtype') == 'f32' else 2
    if k in ('append', 'fill', 'attend'):
        rows = c['batch'] * c['heads']
        row = 2 * c['dh']                                     # a key and a value, in elements
        if k == 'append':
            page = c['leaf'] * row * (size + 1) + 2 * c['dh'] * 4 + 8
            often = {'end': 1.0, 'start': 0.0, 'any': 1.0 / c['leaf']}[c['at']]
            return {'bytes': int(rows * (2 * row * size + 8 + often * page)),
                    'flops': int(rows * (row + often * 4 * c['leaf'] * row))}
        if k == 'fill':
            n = rows * c['context'] * 7 // 8                  # the mean length
            return {'bytes': n * row * (size + 1), 'flops': n * row * 3}
        keys = min(c['wmax'], max(0, c['context'] * 7 // 8 // c['leaf'])) * c['leaf'] * 15 // 16
        many = min(keys * c['queries'], c['context'] * 7 // 8)
        n = rows * c['queries']
        return {'bytes': rows * (many * row + c['leaf'] // 2 * row * size) + n * (row * size + 5 * c['wmax']),
                'flops': n * (keys + c['leaf'] // 2) * 2 * row}
    M, n = c['rows'], c['width']
    if k == 'quant':
        return {'bytes': M * n * 2 * size, 'flops': M * n * 4}
    N = c['cols']
    more = M * N * 2 if c.get('epilogue') == 'residual' else 0
    return {'bytes': N * n * 17 // 32 + M * n * size + M * N * 2 + more, 'flops': 2 * M * N * n}


# ------------------------------------------------------------------------------------------- results in float64
def _round8(y):
    """The nearest e4m3 numbers (halves to even) of float64 y, |y| <= 448."""
    ex = torch.frexp(y)[1].clamp(min=-5) - 1
    step = _pow2(ex - 3)
    return torch.round(y / step) * step


def _page64(x):
    """x (..., rows, D) float64 -> e4m3 numbers and the scale, from the definition."""
    amax = x.abs().amax((-1, -2))
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448))
    e = torch.where(_pow2(e - 1) * 448 >= amax, e - 1, e)
    e = torch.where(_pow2(e) * 448 < amax, e + 1, e).clamp(-126, 127)
    scale = torch.where(amax > 0, _pow2(e), 1.0)
    return _round8(x / scale[..., None, None]), scale


def _round4(x):
    """x (rows, K) float64 -> the values its 4-bit form stands for."""
    n = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -n % 32)).unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1, keepdim=True)
    scale = _pow2((torch.frexp(amax)[1] - 1 - 2).clamp(min=-127))
    a = x.abs() / scale
    v = torch.zeros_like(a)
    # borders between neighbours; on a border the neighbour with the even index wins
    grid = [0, .5, 1, 1.5, 2, 3, 4, 6]
    for i in range(1, 8):
        border = (grid[i - 1] + grid[i]) / 2
        v = torch.where(a >= border if i % 2 == 0 else a > border, grid[i], v)
    return (torch.copysign(v, x) * scale).flatten(-2)[..., :n]


def exact(case, seed):
    c, k = case, case['kind']
    s = prepare(c, seed)
    if k == 'quant':
        return _round4(s['x'].double())
    if k in ('rows', 'both'):
        x = s['x'].double()
        n, N = c['width'], c['cols']
        byte = s['wscale'].long()
        lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
        lut = torch.cat((lut, -lut))
        w = torch.empty(N, s['packed'].shape[1] * 2, dtype=torch.float64, device=DEV)
        w[:, 0::2] = lut[(s['packed'] % 16).long()]
        w[:, 1::2] = lut[(s['packed'] // 16).long()]
        w = (w * _pow2(byte - 127).repeat_interleave(32, 1))[:, :n]
        if k == 'both':
            x = _round4(x)
        elif s['ln'] is not None:
            var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
            x = (x - mean) / torch.sqrt(var + EPS) * s['ln'].double()
        y = x.mm(w.T.contiguous())
        if c.get('epilogue') == 'gelu':
            y = y * torch.special.ndtr(y)
        elif c.get('epilogue') == 'residual':
            y = y + s['res'].double()
        return y
    z = s['cache']
    leaf, B, H = c['leaf'], c['batch'], c['heads']
    if k == 'attend':
        return _attend64(s)
    pool, scale, tail = z['pool'].float().double(), z['scale'].double(), z['tail'].double()
    tags = z['tail_block'].clone()
    if k == 'fill':
        for b in range(B):
            n = int(s['lens'][b])
            whole, rest = divmod(n, leaf)
            x = torch.stack((s['k'][b, :, :n], s['v'][b, :, :n]), 1).double()       # (H, 2, n, D)
            if whole:
                y, sc = _page64(x[:, :, :whole * leaf].unflatten(2, (whole, leaf)))
                pg = z['table'][b, :, :whole].long()
                pool[pg], scale[pg] = y.transpose(1, 2), sc.transpose(1, 2)
            tags[b] = whole if rest else -1
            tail[b, :, :, :rest] = x[:, :, whole * leaf:]
        return [pool, scale, tail, tags]
    levels = [lv.double() for lv in s['levels']]
    for b in range(B):
        t = int(s['t'][b])
        blk, r = divmod(t, leaf)
        tail[b, :, 0, r], tail[b, :, 1, r] = s['k'][b].double(), s['v'][b].double()
        tags[b] = blk
        if r + 1 < leaf:
            continue
        pg = z['table'][b, :, blk].long()
        pool[pg], scale[pg] = _page64(tail[b])
        kids = tail[b, :, 0].clone()
        if blk == 0:
            kids[:, 0] = 0
        size = leaf
        for j, lv in enumerate(levels):
            if (t + 1) % size:
                break
            node = t // size
            if j:
                kids = levels[j - 1][b, :, node * c['arity']:(node + 1) * c['arity']]
            lv[b, :, node] = kids.sum(1)
            size *= c['arity']
    return [pool, scale, tail, tags, *levels]


def _attend64(s):
    """Attention in float64, sequence by sequence over the sequence's whole context with a mask of the keys that
    count; the dense context is read back from the pages."""
    c, z = s['case'], s['cache']
    leaf, N, H, D = c['leaf'], c['queries'], c['heads'], c['dh']
    out = torch.empty(c['batch'], H, N, D, dtype=torch.float64, device=DEV)
    for b in range(c['batch']):
        last = int(s['tq'][b].max())
        nb = last // leaf + 1
        pg = z['table'][b, :, :nb].long()
        kv = z['pool'].view(torch.uint8)[pg.clamp(min=0)].view(torch.float8_e4m3fn).double()
        kv = kv * z['scale'].double()[pg.clamp(min=0)][..., None, None]             # (H, nb, 2, leaf, D)
        tb = int(z['tail_block'][b, 0])
        if 0 <= tb < nb:
            kv[:, tb] = z['tail'][b].double()
        kv = kv.transpose(1, 2).flatten(2, 3)                                       # (H, 2, nb * leaf, D)
        where = torch.arange(nb * leaf, device=DEV)
        for i in range(N):
            t = int(s['tq'][b, i])
            n = torch.minimum(s['vld'][b, :, i].long().sum(-1), s['n_tree'][b, :, i].long())
            on = torch.zeros(H, nb + 1, dtype=torch.bool, device=DEV)
            slot = torch.where(torch.arange(c['wmax'], device=DEV) < n[:, None], s['ids'][b, :, i].long(), nb)
            on.scatter_(1, slot, True)
            keep = on[:, :nb].repeat_interleave(leaf, 1)
            keep |= (where // leaf == t // leaf) & (where <= t)
            keep |= (where == 0) | ((where <= t) & (where > t - LOCAL))
            score = torch.matmul(kv[:, 0], s['q'][b, :, i].double().unsqueeze(-1)).squeeze(-1) / math.sqrt(D)
            p = torch.softmax(torch.where(keep, score, float('-inf')), -1)
            out[b, :, i] = torch.matmul(p.unsqueeze(1), kv[:, 1]).squeeze(1)
    return out
