"""The bound on a LayerNorm in front of a product (oracle.low_bits.layernorm_product): what it admits and what it rejects, on
the inputs of the GPU tests.  CPU only."""
import math

import numpy as np
import pytest
import torch

from oracle import low_bits as O

BF16 = torch.bfloat16
EPS = 1e-5


def inputs(M, Kd, N=40):
    """Rows far from zero; from value 16384 on a row spreads four times as wide."""
    g = torch.Generator().manual_seed(Kd)
    x = torch.randn(M, Kd, generator=g)
    x[:, 16384:] *= 4
    w = torch.randn(N, Kd, generator=g) / math.sqrt(Kd)
    return (100 + x).to(BF16), O.quant4(w.double())[2], (1 + 0.2 * torch.randn(Kd, generator=g)).to(BF16)


def halves(n):
    """A float32 as the sum of its upper half (a bf16) and the rest rounded to bf16."""
    hi = (n.view(torch.int32) & -65536).view(torch.float32)
    return hi.double() + (n - hi).to(BF16).double()


def evaluate(x, w, g, variance=lambda d: (d * d).mean(-1, keepdim=True), hold=halves, weight=True):
    x = x.float()
    d = x - x.mean(-1, keepdim=True)
    n = d * torch.rsqrt(variance(d) + EPS)
    return hold(n * g.float() if weight else n) @ w.T


def within(got, y, tol):
    got = got.to(BF16).double()
    return bool(((got - y).abs() <= tol + 2.0 ** -8 * (y.abs() + tol)).all())


def one_pass(d):
    """Mean square less squared mean, both summed in float32 one value after another (numpy's cumsum)."""
    x = (d + 100).numpy()
    mean, square = (torch.from_numpy(np.cumsum(a, -1, dtype=np.float32)[:, -1:]) / x.shape[1] for a in (x, x * x))
    return (square - mean * mean).clamp(min=0)


def first_values(d):
    return (d[:, :16384] ** 2).sum(-1, keepdim=True) / d.shape[1]


@pytest.mark.parametrize('M,Kd', [(3, 768), (20, 2048), (32, 4096), (5, 20000)])
def test_bound(M, Kd):
    x, w, g = inputs(M, Kd)
    y, tol = O.layernorm_product(x, w, g, EPS)
    assert within(evaluate(x, w, g), y, tol)
    assert not within(evaluate(x, w, g, hold=lambda n: n.to(BF16).double()), y, tol), 'rows rounded to bf16'
    assert not within(evaluate(x, w, g, variance=lambda d: 1.05 * (d * d).mean(-1, keepdim=True)), y, tol)
    assert not within(evaluate(x, w, g, variance=lambda d: 0.95 * (d * d).mean(-1, keepdim=True)), y, tol)
    assert not within(evaluate(x, w, g, weight=False), y, tol)
    if Kd >= 4096:
        assert not within(evaluate(x, w, g, variance=one_pass), y, tol), 'one pass'
    if Kd > 16384:
        assert not within(evaluate(x, w, g, variance=first_values), y, tol), 'squares past 16384 left out'
