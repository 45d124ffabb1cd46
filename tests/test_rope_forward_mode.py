"""The forward derivative of positions.rotate (torch.autograd.forward_ad), on the CPU with the turn's formula in place of the
kernel, and on the GPU with the kernel."""
import pytest
import torch
from torch.autograd import forward_ad as fw

from treeattn_amd import kernels as K
from treeattn_amd import positions


def formula(x, pos, rope, out=None, inverse=False):
    """kernels.rope in float64, layout 'half'."""
    n = len(rope.turns)
    a = pos.double().view(-1, 1).cpu() * (2 * torch.pi * rope.turns.cpu()) * (-1 if inverse else 1)
    c, s = a.cos() * rope.amplitude, a.sin() * rope.amplitude
    y = x.detach().double().cpu()
    p, q = y[..., :n], y[..., n:2 * n]
    return torch.cat((p * c - q * s, p * s + q * c, y[..., 2 * n:]), -1)


def run(x, dx, pos, rope, requires_grad):
    x = x.clone().requires_grad_(requires_grad)
    with fw.dual_level():
        y, dy = fw.unpack_dual(positions.rotate(fw.make_dual(x, dx), pos, rope))
        assert dy is not None, 'the tangent is lost'
        return y.detach(), dy.detach()


@pytest.mark.parametrize('requires_grad', [False, True])
def test_tangents_are_turned_on_the_cpu(monkeypatch, requires_grad):
    monkeypatch.setattr(K, 'rope', lambda x, pos, rope, out=None, inverse=False: formula(x, pos, rope, out, inverse))
    g = torch.Generator().manual_seed(1)
    x, dx = torch.randn(1, 2, 5, 8, generator=g).double(), torch.randn(1, 2, 5, 8, generator=g).double()
    rope = K.Rope([1.0, 0.1, 0.01], 'cpu', amplitude=1.25)
    pos = torch.arange(5, dtype=torch.int32)
    y, dy = run(x, dx, pos, rope, requires_grad)
    assert torch.equal(y, formula(x, pos, rope)) and torch.equal(dy, formula(dx, pos, rope))
    # none without a tangent, and in a level of forward_ad that it is no part of
    assert fw.unpack_dual(positions.rotate(x, pos, rope)).tangent is None
    with fw.dual_level():
        assert fw.unpack_dual(positions.rotate(x, pos, rope)).tangent is None


@pytest.mark.gpu
@pytest.mark.parametrize('requires_grad', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_tangents_are_turned(dtype, requires_grad):
    """Values and tangents are one call's rows each: half a step of the result, and for float32 the sine's and the products' four."""
    g = torch.Generator().manual_seed(2)
    x, dx = [torch.randn(2, 3, 7, 16, generator=g).to(dtype).cuda() for _ in range(2)]
    rope = K.Rope([1.0, 0.3, 0.1, 0.03, 0.01], 'cuda', amplitude=1.25)
    pos = torch.arange(100, 107, dtype=torch.int32, device='cuda')
    y, dy = run(x, dx, pos, rope, requires_grad)
    for got, of in ((y, x), (dy, dx)):
        want = formula(of, pos, rope)
        size = float(of.abs().max()) * 1.25 * 2 ** 0.5
        half = torch.finfo(dtype).eps / 2
        assert float((got.double().cpu() - want).abs().max()) <= size * (half + 4 * 2.0 ** -24 + (2 * 2.0 ** -22.9 if dtype != torch.float32 else 0))
