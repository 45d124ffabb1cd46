"""Attention over candidate lists has no forward-mode derivative: a tangent raises, it is not dropped.  On the CPU the kernels
do not run (stand-ins); on the GPU also through a model."""
import pytest
import torch
from torch.autograd import forward_ad as fw

from treeattn_amd import fastseg, kernels
from treeattn_amd import selection as SEL
from treeattn_amd.config import Config
from treeattn_amd.model import GPT


def test_a_tangent_raises_on_the_cpu(monkeypatch):
    ran = []
    monkeypatch.setattr(fastseg, '_use_fast', lambda *a: None)
    monkeypatch.setattr(kernels, 'sparse_attn_fwd', lambda q, *a: ran.append(1) or (torch.zeros_like(q), torch.zeros(1)))
    x = torch.zeros(1, 1, 4, 8)
    cand = torch.zeros(1, 1, 4, 2, dtype=torch.int32)
    for i in range(3):
        with fw.dual_level():
            qkv = [fw.make_dual(x.clone(), torch.ones_like(x)) if i == j else x for j in range(3)]
            for call in (lambda: fastseg.sparse_attn(*qkv, cand, 1.0), lambda: SEL._attend_list(*qkv, cand, 1.0, fastseg.differentiated(*qkv))):
                with pytest.raises((RuntimeError, NotImplementedError), match='jvp'):
                    call()
    with fw.dual_level(), torch.no_grad():
        assert fw.unpack_dual(fastseg.sparse_attn(x, x, x, cand, 1.0)).tangent is None     # none asked for: runs
    assert ran


@pytest.mark.gpu
@pytest.mark.parametrize('kw', [dict(attn='seg', neighbors=False), dict(attn='seg'), dict(attn='block', tree_block=64, chunk=64)])
def test_a_model_raises(kw):
    cfg = Config(vocab_size=31, seq_len=64, n_layer=1, n_head=2, n_embd=32, leaf=2, rope='half', **kw)
    m = GPT(cfg).cuda().eval()
    for p in m.parameters():
        p.requires_grad_(False)
    idx = torch.randint(0, 31, (1, 64), device='cuda')
    m(idx)
    w = m.blocks[0].ln1
    weight = w.weight.detach().clone()
    with fw.dual_level():
        del w.weight
        w.weight = fw.make_dual(weight, torch.ones_like(weight))
        with pytest.raises((RuntimeError, NotImplementedError), match='jvp'):
            m(idx)
