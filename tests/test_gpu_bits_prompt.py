"""The products of a prompt with 4-bit weights (engine._product), with activations in bf16 and in 4 bits, against float64, and
a prompt through them against the same products one by one.  GPU only."""
import math

import pytest
import torch

from oracle import low_bits as O
from treeattn_amd import kernels as K
from treeattn_amd.config import Config
from treeattn_amd.engine import Decoder, _ln, _product, weights_from_ours, weights_mx4
from treeattn_amd.model import GPT

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF16 = torch.bfloat16


def rnd(*shape, seed, scale=1.0):
    return scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize('bits', [None, 4])
@pytest.mark.parametrize('shape,N,Kd', [((2, 37), 130, 128), ((1, 1), 64, 96), ((3, 130), 384, 160)])
def test_products_of_a_prompt(shape, N, Kd, bits):
    """The rows that are multiplied are x, or its LayerNorm in x's dtype, with 4 bits their microscaled form; sums of K products
    in float32 are off by at most K * 2^-24 of the magnitudes, GELU's slope is at most 1.13 (its evaluation 2^-20 of the
    argument), the result is rounded once (2^-8)."""
    x = (1 + 2 * rnd(*shape, Kd, seed=1)).to(BF16).to(DEV)
    w, wv = K.mx4_quant(rnd(N, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    g = (1 + 0.2 * rnd(Kd, seed=3)).to(BF16).to(DEV)
    r = rnd(*shape, N, seed=4).to(BF16).to(DEV)
    for ln in (None, g):
        rows = (x if ln is None else _ln(x, ln)).double().cpu().view(-1, Kd)
        if bits == 4:
            rows = O.quant4(rows)[2]
        y0 = rows @ wv.double().cpu().T
        t0 = Kd * 2.0 ** -24 * (rows.abs() @ wv.double().cpu().abs().T)
        for kw in ({}, dict(gelu=True), dict(residual=r)):
            y, tol = y0, t0
            if 'gelu' in kw:
                y, tol = y * torch.special.ndtr(y), 1.13 * tol + 2.0 ** -20 * y.abs()
            elif 'residual' in kw:
                y = y + r.double().cpu().view(-1, N)
                tol = tol + 2.0 ** -24 * y.abs()
            got = _product(x, w, ln, bits, **kw)
            assert got.shape == (*shape, N)
            err = (got.double().cpu().view(-1, N) - y).abs()
            assert (err <= tol + 2.0 ** -8 * (y.abs() + tol) + 1e-30).all(), (kw, float(err.max()))


@pytest.mark.parametrize('cache', [None, 'e4m3'])
def test_a_prompt_in_4_bits(cache):
    """prefill(bits=4) runs those products: the first layer's cache holds the rows of its 4-bit product bit for bit (in 8-bit
    pages those rows rounded: 2^-4 of a value, or half of e4m3's lowest step, 2^-10 of a scale that is less than 2 / 448 of the
    largest), and the logits differ from those with bf16 activations."""
    cfg = Config(vocab_size=128, seq_len=64, n_layer=2, n_head=2, n_embd=128, attn='seg', wmax=8, beam=8, leaf=8, neighbors=False)
    torch.manual_seed(3)
    W = weights_mx4(weights_from_ours(GPT(cfg).to(DEV).to(BF16).eval().state_dict(), cfg))
    T = 43
    idx = torch.randint(0, 128, (2, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    x = (W['wte'][idx] + W['wpe'][:T]).view(-1, 128)
    L0 = W['layers'][0]
    logits = []
    for bits in (4, None):
        dec = Decoder(W, 2, 2, 128, 64, 'seg', cfg, DEV, batch=2, cache=cache)
        logits.append(dec.prefill(idx, bits=bits))
        rows = _ln(x, L0['ln1'])
        y = K.mx4_mm(K.mx4_quant(rows) if bits else rows, L0['c_attn']).view(2, T, 3, 2, 64).permute(2, 0, 3, 1, 4)
        for b in range(2):
            for got, want in zip(dec.states[0].dense_kv(b, T), y[1:, b]):
                if cache is None:
                    assert torch.equal(got[0], want)
                else:
                    big = want.float().abs().amax((-1, -2), keepdim=True)
                    assert ((got[0] - want).float().abs() <= 2.0 ** -4 * want.float().abs() + big * 2.0 ** -10 * 2 / 448).all()
                    assert torch.equal(got[0][:, 40:], want[:, 40:])          # the block in the tail
        assert torch.isfinite(logits[-1]).all()
    assert not torch.equal(*logits)
