"""The LayerNorm in front of a product with 4-bit weights (kernels.mx4_mm with ln_w): normalised values are held to more bits
than the result.  GPU only."""
import math

import pytest
import torch

from oracle import low_bits as O
from treeattn_amd import _lib as L
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF16 = torch.bfloat16
EPS = 1e-5


def rnd(*shape, seed, scale=1.0):
    return scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def case(M, N, Kd, far=0.0):
    x = rnd(M, Kd, seed=M + Kd)
    x[:, 16384:] *= 4
    w, wv = K.mx4_quant(rnd(N, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    return (far + x).to(BF16), w, wv.cpu(), (1 + 0.2 * rnd(Kd, seed=4)).to(BF16)


def close(got, y, tol, epilogue=None, residual=None):
    if epilogue == 'gelu':      # its slope is at most 1.13, its float32 evaluation within 2^-20 of the argument
        tol = 1.13 * tol + 2.0 ** -20 * y.abs()
        y = y * torch.special.ndtr(y)
    elif epilogue == 'residual':
        y = y + residual.double()
        tol = tol + 2.0 ** -24 * y.abs()
    bad = ~((got.cpu().double() - y).abs() <= tol + 2.0 ** -8 * (y.abs() + tol))
    assert not bad.any(), (int(bad.sum()), float((got.cpu().double() - y).abs().max()))


# within the product's launch (small M * K), of the workgroups of few rows (16 and 32 rows, one to four column tiles) and of both
# sizes of large tiles; widths off 128
SHAPES = [(1, 40, 32), (3, 40, 768), (16, 33, 160), (32, 300, 1024), (64, 130, 992), (1, 40, 4096), (7, 600, 2080), (16, 5000, 4128),
          (16, 16500, 2080), (20, 40, 2048), (32, 1000, 4096), (33, 8200, 1056), (64, 16400, 1120), (5, 40, 20000), (65, 40, 96),
          (129, 257, 416), (300, 1000, 1024), (700, 4095, 160), (2100, 8200, 224)]


@pytest.mark.parametrize('M,N,Kd', SHAPES)
def test_normalised_rows(M, N, Kd):
    x, w, wv, g = case(M, N, Kd)
    r = rnd(M, N, seed=3).to(BF16)
    y, tol = O.layernorm_product(x, wv, g, EPS)
    for epilogue in (None, 'gelu', 'residual'):
        got = K.mx4_mm(x.to(DEV), w, ln_w=g.to(DEV), epilogue=epilogue, residual=r.to(DEV))
        close(got, y, tol, epilogue, r)


@pytest.mark.parametrize('M,Kd', [(3, 768), (20, 2048), (32, 4096), (5, 20000), (100, 2048)])
def test_rows_far_from_zero(M, Kd):
    x, w, wv, g = case(M, 40, Kd, far=100.0)
    close(K.mx4_mm(x.to(DEV), w, ln_w=g.to(DEV)), *O.layernorm_product(x, wv, g, EPS))


@pytest.mark.parametrize('M,N,Kd', [(1, 40, 4096), (3, 40, 4128), (20, 4100, 4096), (64, 130, 2048), (130, 200, 96), (2500, 2100, 64)])
def test_least_workspace(M, N, Kd):
    """With the least workspace the rows are taken some at a time: the bits of the call that takes them at once, and in place
    of the residual."""
    x, w, _, g = case(M, N, Kd)
    x, g = x.to(DEV), g.to(DEV)
    r = rnd(M, N, seed=3).to(BF16).to(DEV)
    want = K.mx4_mm(x, w, ln_w=g, epilogue='residual', residual=r)
    nbytes = L.lib().ta_mx4_rows_workspace_size(M, Kd, 1)
    assert 0 < nbytes <= 4 * M * ((Kd + 127) // 128 * 128)
    ws = torch.full((nbytes + 64,), 0x5a, dtype=torch.uint8, device=DEV)
    L.call('ta_mx4_rows', x.data_ptr(), Kd, w.at, w.scale_at, r.data_ptr(), N, r.data_ptr(), N, g.data_ptr(), EPS, M, N, Kd, 2,
           ws.data_ptr(), nbytes, L.stream())
    assert torch.equal(r, want) and (ws[nbytes:] == 0x5a).all()


def test_many_rows_in_several_passes():
    """A prompt whose normalised rows do not fit the wrapper's workspace: the rows on both sides of a pass's border, the first and
    the last."""
    M, N, Kd = 70000, 24, 2048
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(M, Kd, generator=gen, device=DEV, dtype=BF16)
    w, wv = K.mx4_quant(rnd(N, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    g = (1 + 0.2 * rnd(Kd, seed=4)).to(BF16)
    fit = L.lib().ta_mx4_rows_workspace_size(M, Kd, 1) // (4 * Kd)
    assert fit < M
    at = torch.tensor([0, 1, fit - 1, fit, fit + 1, M - 2, M - 1], device=DEV)
    close(K.mx4_mm(x, w, ln_w=g.to(DEV))[at], *O.layernorm_product(x[at].cpu(), wv.cpu(), g, EPS))


@pytest.mark.parametrize('M,Kd', [(2, 256), (20, 2048), (70, 128)])
def test_infinities_and_constant_rows(M, Kd):
    """A weight that takes a value past bf16's range gives an infinity of its sign, not NaN, in that row's products; a row of
    equal values is zeros; a NaN stays in its row."""
    x, w, wv, g = case(M, 40, Kd)
    x[1] = 7.5
    g[5] = 3.3e38
    wv = wv.clone()
    x[0, 5] = 200.0                                # its normalised value times g[5] passes float32's range
    got = K.mx4_mm(x.to(DEV), w, ln_w=g.to(DEV)).cpu()
    assert (got[1] == 0).all()
    col = wv[:, 5]
    assert torch.equal(got[0][col != 0], torch.copysign(torch.tensor(float('inf')), col)[col != 0].to(BF16))
    x[0, 5] = float('nan')
    got = K.mx4_mm(x.to(DEV), w, ln_w=g.to(DEV)).cpu()
    assert torch.isnan(got[0]).all() and (got[1] == 0).all()


def test_replayed_graph():
    """A captured call with its workspace, replayed over new rows with eager work between: the eager call's bits."""
    for M in (8, 32, 200):
        x, w, _, g = case(M, 96, 2560)
        x, g = x.to(DEV), g.to(DEV)
        out = torch.empty(M, 96, device=DEV, dtype=BF16)
        K.mx4_mm(x, w, ln_w=g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            K.mx4_mm(x, w, ln_w=g, out=out)
        for i in range(4):
            x.copy_((i + rnd(M, 2560, seed=10 + i)).to(BF16))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, K.mx4_mm(x, w, ln_w=g))
