"""The decoder in fewer bits: 8-bit caches (cache='e4m3') through every selection mode, 4-bit weights (weights_mx4), both
together in prompts, steps and captured graphs.  GPU only."""
import copy

import pytest
import torch

from treeattn_amd import kernels as K
from treeattn_amd.config import Config
from treeattn_amd.engine import Decoder, PagePool, SegState, _Scratch, seg_attend_, weights_from_ours, weights_mx4
from treeattn_amd.model import GPT

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def rnd(*shape, seed, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def states(cfg, B, H, dh, Tcap, dtype):
    pool = PagePool(B, H, dh, cfg.leaf, Tcap, B * H * (Tcap // cfg.leaf), 1, dtype, DEV, cache='e4m3')
    pool.ensure(Tcap)
    return SegState(cfg, Tcap, H, dh, DEV, B, dtype, pages=pool), SegState(cfg, Tcap, H, dh, DEV, B, dtype)


def test_fill_equals_add():
    """A prompt and its tokens one by one leave the same pages, scales, tail, nodes and gated vectors."""
    cfg = Config(leaf=8, wmax=4, beam=4, neighbors=False, gate=True)
    B, H, dh, T = 2, 2, 32, 45
    k, v = rnd(B, H, T, dh, seed=1, dtype=torch.bfloat16), rnd(B, H, T, dh, seed=2, dtype=torch.bfloat16)
    a, _ = states(cfg, B, H, dh, 64, torch.bfloat16)
    b, _ = states(cfg, B, H, dh, 64, torch.bfloat16)
    a.fill(k, v)
    for t in range(T):
        b.add(t, k[:, :, t], v[:, :, t])
    assert torch.equal(a.cache8.pool.view(torch.uint8), b.cache8.pool.view(torch.uint8))
    assert torch.equal(a.cache8.scale, b.cache8.scale) and torch.equal(a.cache8.tail_block, b.cache8.tail_block)
    assert torch.equal(a.cache8.tail[..., :T % 8, :], b.cache8.tail[..., :T % 8, :])
    for x, y in zip(a.levels + a.lg, b.levels + b.lg):
        assert torch.equal(x, y)
    assert all(torch.equal(x, y) for x, y in zip(a.gl, b.gl) if x is not None)
    ka, va = a.dense_kv(1, T)
    kr, vr = a.row(40)
    assert torch.equal(kr[1], ka[0, :, 40]) and torch.equal(vr[1], va[0, :, 40])
    assert torch.equal(ka[:, :, 40:T], k[1:2, :, 40:]) and not torch.equal(ka, k[1:2])


MODES = [dict(neighbors=False), dict(neighbors=True), dict(neighbors=False, gate=True), dict(neighbors=True, gate=True),
         dict(neighbors=True, beam_mode='pred'), dict(neighbors=False, beam_mode='pred', global_pool=True)]


@pytest.mark.parametrize('mode', MODES, ids=lambda m: '-'.join('%s' % k for k, x in m.items() if x) or 'plain')
@pytest.mark.parametrize('dtype,dh,leaf', [(torch.bfloat16, 64, 8), (torch.float32, 32, 2), (torch.float16, 16, 16)])
def test_steps_of_every_selection_mode(mode, dtype, dh, leaf):
    """Selections, stores, nodes and key counts are those of the cache in the model's type; the outputs are those of that
    cache holding the rounded values (two float32 evaluations, each rounded once: eps / 2 of the larger each, and 2^-18 of
    the largest value for their sums and exponentials)."""
    cfg = Config(leaf=leaf, wmax=4, beam=4, **mode)
    B, H, Tcap, T = 2, 2, 128, 45
    st8, st = states(cfg, B, H, dh, Tcap, dtype)
    pw = None
    if cfg.beam_mode == 'pred':
        F = dh + 1 + H + (dh if cfg.global_pool else 0)
        pw = dict(w1=rnd(16, F, seed=7), b1=rnd(16, seed=8), w2=rnd(len(cfg.beam_classes), 16, seed=9),
                  b2=rnd(len(cfg.beam_classes), seed=10), classes=torch.tensor(cfg.beam_classes, device=DEV))
    eps = torch.finfo(dtype).eps
    for t in range(T):
        q, k, v = (rnd(B, H, 1, dh, seed=1000 * s + t, dtype=dtype) for s in (1, 2, 3))
        sc = [_Scratch(B, H, dh, st.shape.leaf_width(cfg.wmax), DEV, 4 if t % 3 else 8) for _ in range(3)]
        got, n8 = seg_attend_(st8, pw, q, k, v, t, scratch=sc[0])
        ref = copy.copy(st)
        dense = [st8.dense_kv(b) for b in range(B)]
        ref.K, ref.V = (torch.cat(x).contiguous() for x in zip(*dense))
        want, nr = seg_attend_(ref, pw, q, k, v, t, update=False, scratch=sc[1])
        bound = eps / 2 * (got.abs() + want.abs()).float() + 2.0 ** -18 * ref.V[:, :, :t + 1].abs().amax().float()
        assert ((got.float() - want.float()).abs() <= bound).all(), t
        assert torch.equal(n8, nr), t
        _, n = seg_attend_(st, pw, q, k, v, t, scratch=sc[2])
        assert torch.equal(n8, n), t
        for a, b in ((sc[0].ids, sc[2].ids), (sc[0].vld, sc[2].vld), (st8.ksum, st.ksum), (st8.st_leaf, st.st_leaf),
                     (st8.st_score, st.st_score), (st8.st_ok, st.st_ok)):
            assert torch.equal(a, b), t
    for a, b in zip(st8.score_levels, st.score_levels):
        assert torch.equal(a, b)


def model(dtype=torch.bfloat16, leaf=8, **kw):
    cfg = Config(vocab_size=128, seq_len=256, n_layer=2, n_head=2, n_embd=128, attn='seg', wmax=4, beam=4, leaf=leaf, **kw)
    torch.manual_seed(3)
    m = GPT(cfg).to(DEV).to(dtype).eval()
    with torch.no_grad():
        for p in m.parameters():
            if p.dim() > 1:
                p.mul_(3)
    return weights_from_ours(m.state_dict(), cfg), cfg


def decoder(W, cfg, B, **kw):
    return Decoder(W, cfg.n_layer, cfg.n_head, cfg.n_embd, 256, 'seg', cfg, DEV, batch=B, **kw)


@pytest.mark.parametrize('bits', [False, True])
@pytest.mark.parametrize('cache', [None, 'e4m3'])
@pytest.mark.parametrize('neighbors', [False, True])
def test_prompt_steps_and_graph(bits, cache, neighbors):
    """A prompt of odd length, eager steps, then a captured step replayed over several blocks: the replays give what eager
    steps of an equal decoder give, bit for bit."""
    W, cfg = model(neighbors=neighbors)
    if bits:
        W = weights_mx4(W)
    B = 3
    idx = torch.randint(0, 128, (B, 37), generator=torch.Generator().manual_seed(1)).to(DEV)
    a, b = decoder(W, cfg, B, cache=cache), decoder(W, cfg, B, cache=cache)
    la, lb = a.prefill(idx, chunk=2), b.prefill(idx)
    assert torch.isfinite(la).all() and (la.float() - lb.float()).abs().max() < 2e-2 * la.float().abs().max()
    a = decoder(W, cfg, B, cache=cache)
    a.prefill(idx)
    tok = lb.argmax(-1)
    for t in range(37, 42):
        xa, xb = a.step(tok, t)[0], b.step(tok, t)[0]
        assert torch.equal(xa, xb)
        tok = xa.argmax(-1)
    b.capture(tok, 42)
    for t in range(42, 75):
        xa, _ = a.step(tok, t)
        b.replay()
        torch.cuda.synchronize()
        assert torch.equal(xa, b.g_logits), t
        tok = xa.argmax(-1)
        assert torch.equal(tok, b.g_tok), t
        if t == 50:   # eager work of another shape between the replays
            decoder(W, cfg, 1, cache=cache).step(5, 0)


@pytest.mark.parametrize('batch', [1, 3])
def test_mx4_decoder_is_the_bf16_decoder_of_the_values(batch):
    """4-bit weights are exact in bf16: the decoder with them gives the logits of a bf16 decoder that holds their values, to
    the package's bar for bf16 outputs (both round activations to bf16 at every product, not at the same places)."""
    W, cfg = model(neighbors=False)
    W4 = weights_mx4(W)
    Wv = dict(W, layers=[dict(L, **{n: L4[n].values(torch.bfloat16) for n in ('c_attn', 'c_proj', 'c_fc', 'c_mlp')})
                         for L, L4 in zip(W['layers'], W4['layers'])])
    a, b = decoder(W4, cfg, batch), decoder(Wv, cfg, batch)
    idx = torch.randint(0, 128, (batch, 70), generator=torch.Generator().manual_seed(2)).to(DEV)
    x, y = a.prefill(idx), b.prefill(idx)
    assert (x - y).abs().max() <= 2e-2 * y.abs().max()
    z = decoder(W4, cfg, batch).prefill(idx, bits=4)      # rows in 4 bits as well: another function, near the first
    assert torch.isfinite(z).all() and torch.nn.functional.cosine_similarity(z.float(), y.float(), dim=-1).min() > 0.5
    for t in range(70, 80):
        tok = idx[:, t - 70].contiguous()
        x, y = a.step(tok, t)[0], b.step(tok, t)[0]
        assert (x - y).abs().max() <= 2e-2 * y.abs().max(), t


def test_long_step_shapes():
    """One sequence over a long cache takes several workgroups per query."""
    cfg = Config(leaf=128, wmax=64, beam=64, neighbors=False, arity=4)
    B, H, dh, T = 1, 3, 64, 40000
    st8, st = states(cfg, B, H, dh, 65536, torch.bfloat16)
    k, v = rnd(B, H, T, dh, seed=1, dtype=torch.bfloat16), rnd(B, H, T, dh, seed=2, dtype=torch.bfloat16)
    st8.fill(k, v)
    kd, vd = st8.dense_kv(0, T)
    st.fill(k, v)
    st.K[:, :, :T], st.V[:, :, :T] = kd, vd
    q, kn, vn = (rnd(B, H, 1, dh, seed=s, dtype=torch.bfloat16) for s in (3, 4, 5))
    got, n8 = seg_attend_(st8, None, q, kn, vn, T)
    want, n = seg_attend_(st, None, q, kn, vn, T)
    assert torch.equal(n8, n)
    assert ((got.float() - want.float()).abs() <= 2.0 ** -8 * (got.abs() + want.abs()).float() + 2.0 ** -14).all()


def test_decoder_refusals():
    W, cfg = model(neighbors=False)
    with pytest.raises(ValueError, match='paged'):
        decoder(W, cfg, 1, cache='e4m3', paged=False)
    with pytest.raises(ValueError, match="'e4m3'"):
        decoder(W, cfg, 1, cache='int8')
    W4 = weights_mx4(W)
    with pytest.raises(ValueError, match='one_launch'):
        decoder(W4, cfg, 1, one_launch=True)
    with pytest.raises(ValueError, match='bf16'):
        decoder(dict(W4, wte=W4['wte'].float(), wpe=W4['wpe'].float()), cfg, 1)
    half = dict(W4, layers=[W4['layers'][0], W['layers'][1]])
    with pytest.raises(ValueError, match='all four'):
        decoder(half, cfg, 1)
    with pytest.raises(ValueError, match='bits'):
        decoder(W, cfg, 1).prefill(torch.zeros(1, 4, dtype=torch.long, device=DEV), bits=4)
