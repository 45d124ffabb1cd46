"""The angles that an attention module turns by are those of its configuration as it is now (the kernel's place is taken by
one that keeps the Rope it is given: CPU)."""
import types

import torch

from treeattn_amd import kernels as K
from treeattn_amd import positions
from treeattn_amd.config import Config


def test_angles_follow_the_configuration(monkeypatch):
    given = []
    monkeypatch.setattr(K, 'rope', lambda x, pos, rope, out=None, inverse=False: given.append(rope) or x.clone())
    cfg = Config(vocab_size=31, seq_len=64, n_layer=1, n_head=2, n_embd=32, attn='seg', rope='half')
    module = types.SimpleNamespace(cfg=cfg, H=2)

    def angles():
        positions.heads(module, torch.zeros(1, 4, 96))
        return given[-1]
    first = angles()
    assert angles() is first                              # made once
    for name, value in (('rope_base', 500000.0), ('rope_scaling', 'linear'), ('rope_factor', 4.0), ('rope_dim', 8),
                        ('rope', 'interleaved'), ('rope_scaling', 'bands'), ('rope_trained', 32), ('seq_len', 128),
                        ('rope_trained', 0)):
        setattr(cfg, name, value)
        got, want = angles(), positions.rope_of(cfg, 'cpu')
        assert torch.equal(got.turns, want.turns) and got.layout == want.layout and got.amplitude == want.amplitude, name
    module.cfg = Config(vocab_size=31, seq_len=64, n_layer=1, n_head=2, n_embd=32, attn='seg', rope='half')
    assert torch.equal(angles().turns, first.turns)
