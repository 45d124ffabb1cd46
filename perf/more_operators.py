"""The operators of a decoder that attends to its whole cache, as cases to time and check them on.

listed() is the fixed set, draw() gives more of the same ranges, prepare() makes what a program holds before the call,
run() makes one call (the operators' plain form in torch, or with `own` the package's kernels), work() says what a call
cannot do without and exact() gives its result in float64.

Kinds of case:
  attend  new tokens' queries over every key of a paged cache up to their own position, query heads sharing keys or not
  store   new tokens of every sequence: queries and keys turned by their positions, keys and values into their pages
  rope    the turn by itself, with its gradient or without
  copy    pages of every layer copied: a fork's pages within the pools, or all used pages into pools of another size
"""
import math

import torch

own = False
DT = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16, 'e4m3': torch.float8_e4m3fn}
DEV = 'cuda'


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # exact attention beside the headline decode step: 32 sequences of about 32768 tokens
        dict(name='attend_batch', kind='attend', dtype='bf16', batch=32, heads=12, shared=1, dh=64, context=32768, leaf=64,
             queries=1),
        # a single stream over a long context
        dict(name='attend_long', kind='attend', dtype='bf16', batch=1, heads=12, shared=1, dh=64, context=131000, leaf=128,
             queries=1),
        # the smallest call: one sequence of a small model, some hundred tokens
        dict(name='attend_one', kind='attend', dtype='f32', batch=1, heads=6, shared=1, dh=64, context=600, leaf=32,
             queries=1),
        # four query heads to a key head, small blocks, half precision
        dict(name='attend_shared', kind='attend', dtype='f16', batch=4, heads=8, shared=4, dh=128, context=6001, leaf=16,
             queries=1),
        # a drafted run of five tokens
        dict(name='attend_run', kind='attend', dtype='f32', batch=8, heads=12, shared=1, dh=64, context=2500, leaf=8,
             queries=5),
        # a piece of a prompt over what came before it
        dict(name='attend_piece', kind='attend', dtype='bf16', batch=2, heads=12, shared=1, dh=64, context=8000, leaf=64,
             queries=256),
        # a layer's share of one decode step
        dict(name='store_step', kind='store', dtype='bf16', batch=32, heads=12, shared=1, dh=64, context=2500, leaf=64,
             queries=1, layout='half', rot=64, scaling='', factor=1.0),
        # prompts taken into a layer's pages
        dict(name='store_prompt', kind='store', dtype='bf16', batch=8, heads=12, shared=1, dh=64, context=8191, leaf=64,
             queries=8191, layout='half', rot=64, scaling='bands', factor=8.0),
        # the queries and keys of one training layer, forward and backward
        dict(name='rope_train', kind='rope', dtype='f16', batch=2, heads=12, dh=64, length=4096, start=0, layout='half',
             rot=64, scaling='', factor=1.0, backward=True),
        # far positions of a long context, part of the head in neighbouring pairs, stretched
        dict(name='rope_long', kind='rope', dtype='f32', batch=1, heads=20, dh=128, length=30001, start=100000,
             layout='interleaved', rot=64, scaling='ntk', factor=16.0, backward=False),
        # eight sequences forked: the pages being filled of twelve heads, in twelve layers
        dict(name='copy_fork', kind='copy', dtype='bf16', layers=12, leaf=64, dh=64, pages=3000, pairs=96, other=False),
        # a pool of 8-bit pages made smaller: its used pages and their scales into new pools
        dict(name='copy_resize', kind='copy', dtype='e4m3', layers=12, leaf=64, dh=64, pages=9000, pairs=6143, other=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['attend', 'attend', 'attend', 'store', 'store', 'rope', 'rope', 'copy'])
    dt = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
    dh = rng.choice([16, 32, 64, 64, 128])
    leaf = rng.choice([2, 8, 16, 32, 64, 64, 128])
    if kind == 'copy':
        c = dict(kind=kind, dtype=rng.choice([dt, 'e4m3']), layers=rng.randint(1, 12), leaf=leaf, dh=dh,
                 pairs=_log_int(rng, 1, 4000), other=rng.random() < 0.5)
        c['pairs'] = max(1, min(c['pairs'], (1 << 25) // (leaf * dh * c['layers'])))
        c['pages'] = 2 * c['pairs'] + rng.randint(0, 400)
        return c
    if kind == 'attend':
        c = dict(kind=kind, dtype=dt, heads=rng.randint(1, 12), shared=rng.choice([1, 1, 1, 2, 4, 8]), dh=dh, leaf=leaf,
                 queries=rng.choice([1, 1, 1, 1, 2, 5, 8, 17, 100]), context=_log_int(rng, 4, 60000))
        c['batch'] = max(1, min(_log_int(rng, 1, 32), (1 << 24) // (c['context'] * c['heads'] * dh // 64)))
        if c['queries'] > 8:      # a piece of a prompt: the scores of the plain form are as many as queries times keys
            c['context'] = max(c['queries'], c['context'] // 4)
            c['batch'] = min(c['batch'], 4)
        return c
    turn = dict(layout=rng.choice(['half', 'interleaved']), rot=2 * rng.randint(2, dh // 2) if rng.random() < 0.4 else dh,
                scaling=rng.choice(['', '', 'linear', 'ntk', 'bands']))
    turn['factor'] = 1.0 if turn['scaling'] == '' else rng.choice([2.0, 4.0, 8.0, 10.5, 32.0])
    if kind == 'store':
        n = rng.choice([1, 1, 1, 3, 8, _log_int(rng, 2, 6000)])
        c = dict(kind=kind, dtype=dt, heads=rng.randint(1, 12), shared=rng.choice([1, 1, 2, 4]), dh=dh, leaf=leaf, queries=n,
                 context=n + _log_int(rng, 1, 2000), **turn)
        c['batch'] = max(1, min(_log_int(rng, 1, 32), (1 << 22) // (c['context'] * c['heads'] * dh // 64)))
        return c
    c = dict(kind=kind, dtype=dt, heads=rng.randint(1, 24), dh=dh, length=_log_int(rng, 1, 30000),
             start=rng.choice([0, 0, _log_int(rng, 1, 1000000)]), backward=rng.random() < 0.5, **turn)
    c['batch'] = max(1, min(_log_int(rng, 1, 32), (1 << 25) // (c['length'] * c['heads'] * dh)))
    return c


# ------------------------------------------------------------------------------------------ inputs and handles
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(7919 * (seed + 1))


def _lens(c, seed):
    """Tokens each sequence has once the new ones are there: up to a quarter short of the context."""
    g = torch.Generator().manual_seed(104729 * (seed + 3))
    n = c['context'] - torch.randint(0, max(1, c['context'] // 4), (c['batch'],), generator=g)
    return [max(int(x), c['queries']) for x in n]


def _pages(c, seed, lens, filled):
    """A pool with the pages of every sequence in a shuffled order, and some that belong to none."""
    g = _gen(seed)
    B, H, D, leaf = c['batch'], c['heads'], c['dh'], c['leaf']
    nb = (c['context'] + leaf - 1) // leaf
    P = B * H * nb + 3
    pool = torch.zeros(P, 2, leaf, D, device=DEV, dtype=DT[c['dtype']])
    if filled:
        gain = torch.exp(0.7 * torch.randn(2, 1, D, generator=g, device=DEV))   # some dimensions far larger than others
        for i in range(0, P, 4096):
            x = torch.randn(min(4096, P - i), 2, leaf, D, generator=g, device=DEV)
            pool[i:i + 4096] = (x * gain).to(pool.dtype)
    table = torch.randperm(P, generator=g, device=DEV)[:B * H * nb].to(torch.int32).view(B, H, nb)
    have = (torch.tensor(lens, device=DEV) + leaf - 1) // leaf
    return pool, torch.where(torch.arange(nb, device=DEV) < have.view(B, 1, 1), table, -1).contiguous()


def frequencies(c):
    """The angle of each pair for one position, as Python floats, and the factor on what is turned."""
    rot, base, amp, f = c['rot'], 10000.0, 1.0, c['factor']
    if c['scaling'] == 'ntk':         # the lowest frequency divided by the factor, the highest as it is
        base *= f ** (rot / (rot - 2))
    w = [base ** (-2 * i / rot) for i in range(rot // 2)]
    if c['scaling'] == 'linear':
        w = [x / f for x in w]
    if c['scaling'] == 'bands':       # pairs that turn seldom in the trained length are slowed, fast ones are left
        keep = [min(1.0, max(0.0, (1024 * x / (2 * math.pi) - 1) / 31)) for x in w]
        w = [x / f * (1 - r) + x * r for x, r in zip(w, keep)]
        amp = 0.1 * math.log(f) + 1
    return w, amp


def _rope_handle(s):
    from treeattn_amd import kernels as K
    s['rope'] = K.Rope(s['freq'], DEV, layout=s['case']['layout'], amplitude=s['amp'])


def prepare(case, seed):
    c, k = case, case['kind']
    s = {'case': c}
    g = _gen(seed + 5)
    if k == 'copy':
        shape = (c['pages'], 2, c['leaf'], c['dh'])

        def pool(rows):
            x = torch.empty(rows, *shape[1:], device=DEV, dtype=DT[c['dtype']])
            for i in range(0, rows, 4096):
                x[i:i + 4096] = torch.randn(min(4096, rows - i), *shape[1:], generator=g, device=DEV).to(x.dtype)
            return x
        order = torch.randperm(c['pages'], generator=g, device=DEV).to(torch.int32)
        s['src'] = order[:c['pairs']].contiguous()
        s['pools'] = [pool(c['pages']) for _ in range(c['layers'])]
        if c['dtype'] == 'e4m3':      # an 8-bit page has a scale for its keys and one for its values
            s['pools'] += [torch.rand(c['pages'], 2, generator=g, device=DEV) for _ in range(c['layers'])]
        if c['other']:
            rows = c['pairs'] + 40
            s['dst'] = torch.arange(c['pairs'], device=DEV, dtype=torch.int32)
            s['to'] = [torch.zeros(rows, *x.shape[1:], device=DEV, dtype=torch.float32).to(x.dtype) for x in s['pools']]
        else:
            s['dst'] = order[c['pairs']:2 * c['pairs']].contiguous()
            s['to'] = s['pools']
        return s
    if k == 'rope':
        # queries and keys as a projection holds them: heads inside positions
        x = torch.randn(c['batch'], c['length'], c['heads'], c['dh'], generator=g, device=DEV).to(DT[c['dtype']])
        s['x'] = x.transpose(1, 2)
        s['pos'] = torch.arange(c['start'], c['start'] + c['length'], device=DEV, dtype=torch.int32)
        s['freq'], s['amp'] = frequencies(c)
        if c['backward']:
            s['dy'] = torch.randn(c['batch'], c['length'], c['heads'], c['dh'], generator=g,
                                  device=DEV).to(DT[c['dtype']]).transpose(1, 2)
        if own:
            _rope_handle(s)
            s['x'].requires_grad_(c['backward'])
        return s
    lens = _lens(c, seed)
    B, H, G, D, N = c['batch'], c['heads'], c['shared'], c['dh'], c['queries']
    s['pool'], s['table'] = _pages(c, seed, lens, k == 'attend')
    s['pos'] = (torch.tensor(lens, device=DEV).view(B, 1) - N + torch.arange(N, device=DEV)).to(torch.int32)
    # queries, keys and values of the new tokens as one projection gives them
    x = torch.randn(B, N, G * H + 2 * H, D, generator=g, device=DEV).to(DT[c['dtype']]).transpose(1, 2)
    s['q'], s['k'], s['v'] = x[:, :G * H], x[:, G * H:G * H + H], x[:, G * H + H:]
    if k == 'store':
        s['freq'], s['amp'] = frequencies(c)
    if own:
        from treeattn_amd import kernels as K
        s['cache'] = K.PagedCache(s['pool'], s['table'], s['table'].shape[2] * c['leaf'])
        if k == 'store':
            _rope_handle(s)
        else:
            from treeattn_amd.engine import decode_nsplit_dense
            s['nsplit'] = decode_nsplit_dense(B, H, G * N, c['context'], D)
            s['ws'] = K.dense_attn_workspace(B, G * H, N, D, s['nsplit'], DEV)
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _attend(s):
    c = s['case']
    B, H, G, D, N, leaf = c['batch'], c['heads'], c['shared'], c['dh'], c['queries'], c['leaf']
    pg = s['table'].long()
    kv = s['pool'][pg.clamp(min=0)]                                                  # (B, H, blocks, 2, leaf, D)
    k, v = (kv[:, :, :, i].flatten(2, 3).float() for i in (0, 1))                    # (B, H, L, D)
    del kv
    q = s['q'].unflatten(1, (H, G)).flatten(2, 3).float()                            # (B, H, G N, D)
    sc = torch.matmul(k, q.transpose(-1, -2).contiguous()) * (1 / math.sqrt(D))      # (B, H, L, G N)
    t = s['pos'].view(B, 1, 1, N).repeat(1, 1, 1, G)
    ok = (torch.arange(k.shape[2], device=DEV).view(-1, 1) <= t) & (pg >= 0).repeat_interleave(leaf, 2).unsqueeze(-1)
    sc = torch.where(ok, sc, float('-inf'))
    p = torch.exp(sc - sc.amax(2, keepdim=True))
    out = torch.matmul(p.transpose(-1, -2).contiguous(), v) / p.sum(2).unsqueeze(-1)
    return out.unflatten(2, (G, N)).flatten(1, 2).to(s['q'].dtype)


def _turned(s, x, pos, sign):
    """x (B, H, T, D) turned by sign times its positions' angles, in its type; pos (T,) or (B, T)."""
    c = s['case']
    rot = c['rot']
    angle = pos.double().unsqueeze(-1) * torch.tensor(s['freq'], dtype=torch.float64, device=DEV)
    if pos.dim() == 2:
        angle = angle.unsqueeze(1)
    cos, sin = torch.cos(angle).float() * s['amp'], torch.sin(angle).float() * (s['amp'] * sign)
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if c['layout'] == 'interleaved' else (y[..., :rot // 2], y[..., rot // 2:rot])
    pair = (a * cos - b * sin, a * sin + b * cos)
    y = torch.cat((torch.stack(pair, -1).flatten(-2) if c['layout'] == 'interleaved' else torch.cat(pair, -1),
                   y[..., rot:]), -1)
    return y.to(x.dtype)


def _store(s):
    c = s['case']
    leaf = c['leaf']
    B, H = c['batch'], c['heads']
    blk, r = s['pos'].long() // leaf, s['pos'].long() % leaf                         # (B, N)
    pg = s['table'].gather(2, blk.unsqueeze(1).expand(B, H, -1)).long()              # (B, H, N)
    r = r.unsqueeze(1).expand_as(pg)
    s['pool'][pg, 0, r] = _turned(s, s['k'], s['pos'], 1)
    s['pool'][pg, 1, r] = s['v']
    return [_turned(s, s['q'], s['pos'], 1), s['pool']]


def _rope(s):
    y = _turned(s, s['x'], s['pos'], 1)
    return [y, _turned(s, s['dy'], s['pos'], -1)] if s['case']['backward'] else [y]


def _copy(s):
    src, dst = s['src'].long(), s['dst'].long()
    for x, y in zip(s['pools'], s['to']):
        if x.dtype == torch.float8_e4m3fn:
            x, y = x.view(torch.uint8), y.view(torch.uint8)
        y[dst] = x[src]
    return s['to']


def run(state):
    s = state
    k = s['case']['kind']
    if own:
        from treeattn_amd import kernels as K
        if k == 'attend':
            return K.dense_attn(s['q'], s['cache'], None, s['pos'], 1 / math.sqrt(s['case']['dh']), nsplit=s['nsplit'],
                                ws=s['ws'])[0]
        if k == 'store':
            return [K.kv_store(s['k'], s['v'], s['cache'], None, s['pos'], q=s['q'], rope=s['rope']), s['pool']]
        if k == 'rope':
            from treeattn_amd.positions import rotate
            y = rotate(s['x'], s['pos'], s['rope'])
            if not s['case']['backward']:
                return [y]
            return [y.detach(), torch.autograd.grad(y, s['x'], s['dy'])[0]]
        K.copy_rows(s['pools'], s['src'], s['dst'], out=s['to'])
        return s['to']
    return {'attend': _attend, 'store': _store, 'rope': _rope, 'copy': _copy}[k](s)


# -------------------------------------------------------------------------------------------------- their work
def work(case):
    c, k = case, case['kind']
    size = {'f32': 4, 'e4m3': 1}.get(c['dtype'], 2)
    if k == 'copy':
        page = 2 * c['leaf'] * c['dh'] * size + (8 if c['dtype'] == 'e4m3' else 0)
        return {'bytes': 2 * c['layers'] * c['pairs'] * page, 'flops': 0}
    if k == 'rope':
        n = c['batch'] * c['heads'] * c['length']
        ways = 2 if c['backward'] else 1
        return {'bytes': 2 * ways * n * c['dh'] * size, 'flops': ways * n * c['rot'] * 3}
    B, H, G, D, N = c['batch'], c['heads'], c['shared'], c['dh'], c['queries']
    if k == 'store':
        return {'bytes': 2 * B * N * (G + 2) * H * D * size, 'flops': B * N * (G + 1) * H * c['rot'] * 3}
    keys = max(N, c['context'] * 7 // 8)                     # the mean length
    return {'bytes': B * H * D * size * (2 * keys + 2 * G * N), 'flops': 4 * B * H * G * N * D * (keys - (N - 1) // 2)}


# ------------------------------------------------------------------------------------------- results in float64
def _turned64(s, x, pos):
    """The same turn as a product of complex numbers."""
    c = s['case']
    rot = c['rot']
    w = torch.tensor(s['freq'], dtype=torch.float64, device=DEV)
    angle = pos.double()[..., None] * w
    z = torch.polar(torch.full_like(angle, s['amp']), angle)
    z = z if pos.dim() == 1 else z[:, None]
    x = x.double()
    y = x.clone()
    if c['layout'] == 'interleaved':
        y[..., :rot] = torch.view_as_real(torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    else:
        h = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * z
        y[..., :rot // 2], y[..., rot // 2:rot] = h.real, h.imag
    return y


def exact(case, seed):
    c, k = case, case['kind']
    s = prepare(c, seed)
    if k == 'copy':
        to = [x.float().double() for x in s['to']]
        for x, y in zip(s['pools'], to):
            y.index_copy_(0, s['dst'].long(), x.float().double().index_select(0, s['src'].long()))
        return to
    if k == 'rope':
        with torch.no_grad():
            y = [_turned64(s, s['x'], s['pos'])]
            return y + ([_turned64(s, s['dy'], -s['pos'])] if c['backward'] else [])
    B, H, G, D, N, leaf = c['batch'], c['heads'], c['shared'], c['dh'], c['queries'], c['leaf']
    if k == 'store':
        pool = s['pool'].double()
        kk = _turned64(s, s['k'], s['pos'])
        for b in range(B):
            at = s['pos'][b].long()
            pg = s['table'][b].long()[:, at // leaf]                                 # (H, N)
            pool[pg, 0, (at % leaf).expand_as(pg)] = kk[b]
            pool[pg, 1, (at % leaf).expand_as(pg)] = s['v'][b].double()
        return [_turned64(s, s['q'], s['pos']), pool]
    out = torch.empty(B, G * H, N, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        n = int(s['pos'][b].max()) + 1
        pg = s['table'][b, :, :(n + leaf - 1) // leaf].long()
        for h in range(H):
            rows = s['pool'][pg[h]].double()                                         # (blocks, 2, leaf, D)
            k64, v64 = rows[:, 0].reshape(-1, D)[:n], rows[:, 1].reshape(-1, D)[:n]
            keep = torch.arange(n, device=DEV) <= s['pos'][b].view(N, 1)
            for j in range(G):
                score = s['q'][b, h * G + j].double().mm(k64.T.contiguous()) / math.sqrt(D)
                out[b, h * G + j] = torch.softmax(score.masked_fill(~keep, float('-inf')), -1).mm(v64)
    return out
