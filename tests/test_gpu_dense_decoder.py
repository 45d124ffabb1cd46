"""Decoders that attend to their whole paged cache, rotary positions in models and decoders, sequences forked and pools resized
(engine.Decoder, model.GPT).  GPU only."""
import copy
import io
import math

import pytest
import torch
import torch.nn.functional as F

from treeattn_amd.checkpoint import load_decoder, save_checkpoint
from treeattn_amd.config import Config
from treeattn_amd.engine import Decoder, weights_from_ours, weights_mx4
from treeattn_amd.model import GPT
from treeattn_amd.positions import rope_frequencies

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16 = torch.float32, torch.bfloat16


def model(dtype=F32, n_head=2, dh=32, n_layer=2, seq_len=256, seed=0, **kw):
    cfg = Config(vocab_size=97, seq_len=seq_len, n_layer=n_layer, n_head=n_head, n_embd=n_head * dh, attn='seg', leaf=8, wmax=4,
                 beam=4, **kw)
    torch.manual_seed(seed)
    return GPT(cfg).to(DEV).to(dtype).eval(), cfg


def dec(m, cfg, mode='dense', batch=2, Tcap=256, weights=lambda W: W, **kw):
    W = weights(weights_from_ours(m.state_dict(), cfg))
    if mode == 'dense':
        kw.setdefault('paged', True)
    return Decoder(W, cfg.n_layer, cfg.n_head, cfg.n_embd, Tcap, mode, cfg, DEV, batch=batch, **kw)


def logits64(m, cfg, idx):
    """The model over idx (B,T) with attention to every earlier position, in float64 (weights as they are)."""
    sd = {k: v.double() for k, v in m.state_dict().items()}
    B, T = idx.shape
    H, C = cfg.n_head, cfg.n_embd
    x = sd['wte.weight'][idx]
    if not cfg.rope:
        x = x + sd['wpe.weight'][:T]
    ln = lambda x, w: F.layer_norm(x, (C,), w, None, 1e-5)
    for i in range(cfg.n_layer):
        p = 'blocks.%d.' % i
        q, k, v = (ln(x, sd[p + 'ln1.weight']) @ sd[p + 'attn.c_attn.weight'].T).view(B, T, 3, H, C // H).permute(2, 0, 3, 1, 4)
        if cfg.rope:
            rot = cfg.rope_dim or C // H
            w, amp = rope_frequencies(rot, cfg.rope_base, cfg.rope_scaling, cfg.rope_factor, cfg.rope_trained or cfg.seq_len)
            a = torch.arange(T, device=DEV).double()[:, None] * torch.tensor(w, dtype=torch.float64, device=DEV)
            z = torch.polar(torch.full_like(a, amp), a)
            def turn(y):
                y = y.clone()
                if cfg.rope == 'interleaved':
                    y[..., :rot] = torch.view_as_real(torch.view_as_complex(y[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
                else:
                    h = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * z
                    y[..., :rot // 2], y[..., rot // 2:rot] = h.real, h.imag
                return y
            q, k = turn(q), turn(k)
        s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(C // H)
        s = s.masked_fill(torch.ones(T, T, device=DEV, dtype=torch.bool).triu(1), float('-inf'))
        o = torch.matmul(torch.softmax(s, -1), v).transpose(1, 2).reshape(B, T, C)
        x = x + o @ sd[p + 'attn.c_proj.weight'].T
        x = x + F.gelu(ln(x, sd[p + 'ln2.weight']) @ sd[p + 'mlp.c_fc.weight'].T) @ sd[p + 'mlp.c_proj.weight'].T
    return ln(x, sd['ln_f.weight']) @ sd['wte.weight'].T


ROPES = [dict(), dict(rope='half'), dict(rope='interleaved', rope_dim=16, rope_scaling='bands', rope_factor=4.0, rope_trained=64)]


@pytest.mark.parametrize('kw', ROPES)
@pytest.mark.parametrize('B', [1, 3])
def test_dense_steps_and_prompts_in_float32(kw, B):
    """Steps one by one, and a prompt followed by steps at ragged positions, give the model's logits in float64 to 1e-4 of their
    size: two layers of sums of 64 products in float32 are off by some 1e-6."""
    m, cfg = model(**kw)
    idx = torch.randint(0, 97, (B, 90), generator=torch.Generator().manual_seed(1)).to(DEV)
    want = logits64(m, cfg, idx)
    size = float(want.abs().max())
    d = dec(m, cfg, batch=B)
    for t in range(20):
        lg, keys = d.step(idx[:, t], t)
        assert float((lg.double() - want[:, t]).abs().max()) <= 1e-4 * size, t
        assert bool((keys == t + 1).all())
    d = dec(m, cfg, batch=B)
    lg = d.prefill(idx[:, :70])
    assert float((lg.double() - want[:, 69]).abs().max()) <= 1e-4 * size
    at = torch.tensor([70, 33, 5][:B], device=DEV)      # going back for some
    for i in range(15):
        lg, _ = d.step(idx[torch.arange(B), at], at)
        assert float((lg.double() - want[torch.arange(B), at]).abs().max()) <= 1e-4 * size, i
        at = at + 1


@pytest.mark.parametrize('weights', [lambda W: W, weights_mx4], ids=['bf16', 'mx4'])
def test_dense_decoder_in_bf16_and_captured(weights):
    """bf16: the fused products; a captured step replays the eager one, token by token, over a page boundary and a refill of
    pages."""
    m, cfg = model(BF16, n_head=2, dh=64, rope='half')
    idx = torch.randint(0, 97, (3, 60), generator=torch.Generator().manual_seed(2)).to(DEV)
    a, b = (dec(m, cfg, batch=3, weights=weights, reserve_ahead=5) for _ in range(2))
    la, lb = a.prefill(idx), b.prefill(idx)
    assert torch.equal(la, lb)
    if weights is not weights_mx4:
        # five roundings a layer to 2^-9 of the running sum, and of the logits
        want = logits64(m, cfg, idx)[:, -1]
        assert float((la.double() - want).norm() / want.norm()) < 0.03
    tok = la.argmax(-1)
    a.capture(tok, 60)
    for t in range(60, 76):
        a.replay()
        lg, _ = b.step(tok, t)
        torch.cuda.synchronize()
        assert torch.equal(a.g_logits.float(), lg.float()), t
        tok = lg.argmax(-1)
        assert torch.equal(a.g_tok, tok)
    assert a.keys_read().tolist() == [76.0] * 3


@pytest.mark.parametrize('kw', ROPES[1:])
def test_seg_decoder_with_rotary_positions_follows_the_model(kw):
    """With every block selected the segment tree's attention is exact: its decoder and its model give the float64 logits."""
    m, cfg = model(neighbors=False, **kw)
    cfg.wmax = cfg.beam = 64
    m.cfg.wmax = m.cfg.beam = 64
    for blk in m.blocks:
        blk.attn.cfg = cfg
    idx = torch.randint(0, 97, (2, 64), generator=torch.Generator().manual_seed(3)).to(DEV)
    want = logits64(m, cfg, idx)
    size = float(want.abs().max())
    with torch.no_grad():
        got = m(idx)[0]
    assert float((got.double() - want).abs().max()) <= 1e-4 * size
    for weights in (lambda W: W,):
        d = dec(m, cfg, 'seg', weights=weights)
        for t in range(40):
            lg, _ = d.step(idx[:, t], t)
            assert float((lg.double() - want[:, t]).abs().max()) <= 1e-4 * size, t
        d = dec(m, cfg, 'seg')
        assert float((d.prefill(idx).double() - want[:, -1]).abs().max()) <= 1e-4 * size


@pytest.mark.parametrize('attn', ['seg', 'block', 'dyn'])
def test_models_with_rotary_positions_train(attn):
    """Every attention module takes rotary positions; the loss's gradient agrees with differences along a direction."""
    cfg = Config(vocab_size=31, seq_len=64, n_layer=1, n_head=2, n_embd=32, attn=attn, tree_block=64, chunk=64, leaf=2, rope='half',
                 rope_dim=8, neighbors=False, wmax=64, beam=64)
    torch.manual_seed(4)
    m = GPT(cfg).to(DEV)
    assert 'wpe.weight' not in m.state_dict()
    idx = torch.randint(0, 31, (2, 64), device=DEV)
    loss = m(idx, idx.roll(-1, 1))[1]
    loss.backward()
    w = m.blocks[0].attn.c_attn.weight
    g = w.grad.clone()
    assert bool(torch.isfinite(g).all()) and float(g.norm()) > 0
    d = torch.randn_like(w)
    d[64:] = 0                                             # the queries' and keys' rows: through the turn
    ls = []
    with torch.no_grad():
        for e in (-1e-2, 1e-2):
            w.add_(e * d)
            ls.append(float(m(idx, idx.roll(-1, 1))[1].double()))
            w.sub_(e * d)
    diff, want = (ls[1] - ls[0]) / 2e-2, float((g.double() * d.double()).sum())
    # third derivatives times 1e-4 / 6, and the losses' rounding, 4 2^-24 / 2e-2, beside the derivative
    assert abs(diff - want) <= 0.02 * abs(want) + 5e-5, (diff, want)


def states(d):
    return [x for st in d.states for x in st.sequence_tensors()]


CASES = [('dense', dict(), dict()), ('dense', dict(rope='interleaved'), dict()), ('seg', dict(), dict()),
         ('seg', dict(neighbors=False), dict()), ('seg', dict(gate=True, rope='half'), dict()),
         ('seg', dict(beam_mode='pred', beam_classes=(2, 3, 4), global_pool=True), dict()), ('seg', dict(), dict(cache='e4m3')),
         ('seg', dict(neighbors=False), dict(paged=False))]


@pytest.mark.parametrize('mode,kw,dkw', CASES, ids=[str(i) for i in range(len(CASES))])
@pytest.mark.parametrize('t', [1, 8, 64, 71])
def test_fork_goes_on_as_the_same_tokens_would(mode, kw, dkw, t):
    """A forked sequence's logits are those of a decoder that was given the tokens: bit for bit (with the global pool, whose sum is
    formed again in another order, to 1e-5; float32).  The sequence it was forked from goes on undisturbed."""
    m, cfg = model(dh=32, **kw)
    idx = torch.randint(0, 97, (3, 100), generator=torch.Generator().manual_seed(5)).to(DEV)
    d, ref = dec(m, cfg, mode, batch=3, **dkw), dec(m, cfg, mode, batch=3, **dkw)
    line = idx[0].clone()
    other = torch.stack((line, line, idx[2]))              # ref: sequence 1 has sequence 0's tokens from the start
    for i in range(72):
        d.step(idx[:, i], i)
        ref.step(other[:, i], i)
    d.fork(0, 1, t)
    if kw.get('global_pool'):                              # a running sum does not go back by itself
        for st in ref.states:
            k = st.dense_kv(1, t)[0][0].float()
            st.ksum[1] = 0
            for j in range(t):
                st.ksum[1] += k[:, j]
    same = (lambda a, b: float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())) if kw.get('global_pool') else torch.equal
    # both take new tokens at sequence 1's position t, sequences 0 and 2 at 72
    for i in range(20):
        tok = idx[:, (37 + i) % 100]
        at = torch.tensor([72 + i, t + i, 72 + i], device=DEV)
        a, _ = d.step(tok, at)
        b, _ = ref.step(tok, at)
        assert same(a, b), i
    if d.pool is not None and mode == 'dense':
        pages = d.pool
        assert pages.n_shared == (t // pages.leaf) * pages.H


@pytest.mark.parametrize('mode,dkw', [('dense', {}), ('seg', {}), ('seg', dict(cache='e4m3'))])
def test_going_back_in_a_shared_page_leaves_the_other_alone(mode, dkw):
    m, cfg = model(neighbors=False)
    idx = torch.randint(0, 97, (2, 100), generator=torch.Generator().manual_seed(6)).to(DEV)
    d = dec(m, cfg, mode, **dkw)
    for i in range(72):
        d.step(idx[:, i], i)
    d.fork(0, 1, 72)
    n = 72 if not dkw else 64                               # (an 8-bit cache reads its last block unrounded until it goes on)
    keep = [x.clone() for st in d.states for x in st.dense_kv(0, n)]
    d.step(idx[:, 90], torch.tensor([72, 3], device=DEV))   # sequence 1 goes back to position 3
    for x, y in zip(keep, [x for st in d.states for x in st.dense_kv(0, n)]):
        assert torch.equal(x, y)
    d.pool.release(0)
    d.step(idx[:, 91], torch.tensor([0, 4], device=DEV))


@pytest.mark.parametrize('mode,dkw', [('dense', {}), ('seg', {}), ('seg', dict(cache='e4m3'))])
def test_fork_and_resize_between_replays(mode, dkw):
    """Captured steps: a sequence forked between replays goes on where it was put; after a resize the step is captured again;
    against a decoder that steps eagerly."""
    m, cfg = model(BF16, n_head=2, dh=64, neighbors=False, rope='half')
    idx = torch.randint(0, 97, (3, 66), generator=torch.Generator().manual_seed(7)).to(DEV)
    a, b = (dec(m, cfg, mode, batch=3, reserve_ahead=6, max_tokens=128, **dkw) for _ in range(2))
    tok = a.prefill(idx).argmax(-1)
    assert torch.equal(tok, b.prefill(idx).argmax(-1))
    a.capture(tok, 66)
    at = torch.full((3,), 66, device=DEV)
    for i in range(24):
        if i == 5:
            for d in (a, b):
                d.fork(2, 0, 67)
            a.g_tok[0], a.g_t[0] = 11, 67
            tok[0], at[0] = 11, 67
        if i == 14:
            n = sum(r > 0 for r in a.pool.refs)
            a.resize(n + 40)
            with pytest.raises(RuntimeError, match='capture'):
                a.replay()
            b.resize(b.pool.P + 7)
            a.capture(tok, at)
        a.replay()
        lg, _ = b.step(tok, at)
        torch.cuda.synchronize()
        assert torch.equal(a.g_logits.float(), lg.float()), i
        tok, at = lg.argmax(-1), at + 1
        assert torch.equal(a.g_tok, tok)


def test_rotary_models_save_load_and_copy():
    m, cfg = model(rope='half', rope_scaling='linear', rope_factor=2.0)
    f = io.BytesIO()
    save_checkpoint(m, f)
    f.seek(0)
    d, c = load_decoder(f, Tcap=512)
    assert c.rope_factor == 2.0 and c.rope == 'half'
    idx = torch.randint(0, 97, (1, 32), device=DEV)
    a, b = m(idx)[0], copy.deepcopy(m)(idx)[0]
    assert torch.equal(a, b)
    for t in range(3):
        d.step(int(idx[0, t]), t)


def test_refusals():
    m, cfg = model()
    rm, rcfg = model(rope='half')
    W = weights_from_ours(rm.state_dict(), rcfg)
    assert W['wpe'] is None
    for bad in (lambda: dec(rm, cfg), lambda: dec(m, cfg, cache='e4m3'), lambda: dec(rm, rcfg, paged=False, batch=1),
                lambda: dec(rm, rcfg, 'seg', one_launch=True),
                lambda: dec(*model(n_head=1, dh=24)), lambda: dec(m, cfg, 'other', paged=True),
                lambda: dec(*model(rope='sideways')), lambda: dec(*model(rope='half', rope_dim=64))):
        with pytest.raises(ValueError):
            bad()
    d = dec(m, cfg)
    d.step(torch.tensor([1, 2], device=DEV), 0)
    for bad in (lambda: d.fork(0, 0, 1), lambda: d.fork(0, 2, 1), lambda: d.fork(0, 1, -1), lambda: d.fork(0, 1, 65),
                lambda: dec(m, cfg, 'seg', paged=False).resize(3)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        dec(m, cfg, batch=1, paged=False).prefill(torch.zeros(1, 4, dtype=torch.long, device=DEV))
    with pytest.raises(RuntimeError, match='pages are in use'):
        d.resize(1)
    with pytest.raises(RuntimeError, match='capture'):
        d.replay()
