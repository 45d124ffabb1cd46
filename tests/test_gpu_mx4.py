"""Microscaled 4-bit rows (kernels.Mx4: mx4_quant, mx4_mm) against their float64 restatement.  GPU only."""
import copy
import math
import pickle

import pytest
import torch

from oracle import low_bits as O
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def rnd(*shape, seed, dtype=F32, scale=1.0):
    return (scale * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype)


def codes_of(w):
    p = w.packed.cpu()
    return torch.stack((p & 15, p >> 4), -1).flatten(-2).long()


def same_rows(w, x):
    code, byte, val = O.quant4(x.double())
    assert torch.equal(w.scale.cpu().long(), byte)
    assert torch.equal(codes_of(w), torch.where((byte == 255).repeat_interleave(32, 1), 0, code))
    return val


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('M,Kd', [(1, 1), (1, 31), (3, 32), (5, 33), (2, 128), (7, 129), (37, 1000), (64, 4096), (300, 72)])
def test_quant(dtype, M, Kd):
    """Codes and scale bytes are the restatement's; the values are what they stand for, rounded to x's type."""
    x = (rnd(M, Kd, seed=M + Kd) * torch.exp(2 * rnd(M, 1, seed=7))).to(dtype)
    w, v = K.mx4_quant(x.to(DEV), values=True)
    val = same_rows(w, x)
    assert torch.equal(v.cpu(), val.to(dtype)) and v.dtype == dtype
    assert torch.equal(w.values().cpu().double(), val.float().double())
    assert K.mx4_quant(x.to(DEV)).packed.equal(w.packed)


def test_quant_borders():
    """Every border between neighbouring values, one float32 step to either side of it, both signs, several scales."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    near = torch.cat((mids, torch.nextafter(mids, mids + 1), torch.nextafter(mids, mids - 1), torch.tensor(O.GRID4)))
    rows = []
    for e in (-100, -20, 0, 1, 40, 120):
        for s in (1, -1):
            r = torch.zeros(64)
            r[:32] = near * s
            r[31] = 4.0                              # keeps the block's scale at 2^0
            rows.append(r * 2.0 ** e)
    x = torch.stack(rows)
    same_rows(K.mx4_quant(x.to(DEV)), x)


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_quant_zeros_extremes_and_what_is_not_finite(dtype):
    f = torch.finfo(dtype)
    x = torch.zeros(8, 96, dtype=dtype)
    x[1, 40] = f.max
    x[2, 3] = f.smallest_normal / 4
    x[3, 35] = float('inf')
    x[4, 70] = float('nan')
    x[5, 0], x[5, 95] = -float('inf'), 1.0
    x[6, :32] = -0.0
    x[7] = f.max * torch.linspace(-1, 1, 96)
    w, v = K.mx4_quant(x.to(DEV), values=True)
    val = same_rows(w, x)
    assert torch.equal(torch.nan_to_num(v.cpu().double(), nan=1e300), torch.nan_to_num(val.to(dtype).double(), nan=1e300))


def test_quant_strides():
    """Views: rows apart, rows off a 16-byte boundary, and a transposed view refused."""
    buf = rnd(9, 301, seed=3, dtype=BF16).to(DEV)
    for x in (buf[:, :256], buf[::2, 1:200], buf[1:2, 5:6], buf[:, 3:]):
        w, v = K.mx4_quant(x, values=True)
        assert torch.equal(v.cpu(), same_rows(w, x.cpu()).to(BF16))
    with pytest.raises(ValueError, match='contiguous rows'):
        K.mx4_quant(buf.t())


# ------------------------------------------------------------------------------------------------ products
def gelu(y):
    return y * torch.special.ndtr(y)


def want(x, wv, ln_w=None, epilogue=None, residual=None, eps=1e-5):
    """float64 result and how far a float32 evaluation with one bf16 rounding may be from it.  K products summed in
    float32 are off by at most K * 2^-24 of the sum of their magnitudes (A); a LayerNorm adds the rounding of its rows to
    bf16 (2^-8 of A) and its own float32 roundings (K * 2^-22 of A); GELU's slope is at most 1.13 and its float32
    evaluation within 2^-20 of the argument's magnitude; the result is rounded once (2^-8)."""
    x, wv = x.double(), wv.double()
    Kd = x.shape[1]
    rel = Kd * 2.0 ** -24
    if ln_w is not None:
        var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
        x = (x - mean) / torch.sqrt(var + eps) * ln_w.double()
        rel += 2.0 ** -8 + Kd * 2.0 ** -22
    y = x @ wv.T
    tol = rel * (x.abs() @ wv.abs().T)
    if epilogue == 'gelu':
        tol = 1.13 * tol + 2.0 ** -20 * y.abs()
        y = gelu(y)
    elif epilogue == 'residual':
        y = y + residual.double()
        tol = tol + 2.0 ** -24 * y.abs()
    return y, tol + 2.0 ** -8 * (y.abs() + tol) + 1e-30


def close(got, y, tol):
    got = got.cpu().double()
    bad = ~((got - y).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float((got - y).abs().max()), float(tol.max()))


ROWS = [(1, 1, 32), (1, 100, 96), (2, 16, 128), (5, 1024, 1024), (16, 33, 160), (17, 130, 2080), (32, 768, 768), (31, 17, 4096),
        (33, 300, 512), (64, 65, 1056), (32, 16400, 256), (8, 16500, 1152), (50, 16384, 544), (65, 40, 96), (128, 128, 128),
        (129, 257, 416), (300, 1000, 1024), (511, 129, 2016),
        (200, 16500, 96), (1111, 4095, 160), (2100, 2050, 224)]


@pytest.mark.parametrize('M,N,Kd', ROWS)
@pytest.mark.parametrize('epilogue', [None, 'gelu', 'residual'])
def test_rows(M, N, Kd, epilogue):
    x = rnd(M, Kd, seed=1, dtype=BF16)
    w, wv = K.mx4_quant(rnd(N, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    r = rnd(M, N, seed=3, dtype=BF16)
    got = K.mx4_mm(x.to(DEV), w, epilogue=epilogue, residual=r.to(DEV))
    close(got, *want(x, wv.cpu(), epilogue=epilogue, residual=r))
    g = (1 + 0.2 * rnd(Kd, seed=4)).to(BF16)
    x2 = (3 * x + 1).to(BF16)
    got = K.mx4_mm(x2.to(DEV), w, ln_w=g.to(DEV), epilogue=epilogue, residual=r.to(DEV))
    close(got, *want(x2, wv.cpu(), ln_w=g, epilogue=epilogue, residual=r))


@pytest.mark.parametrize('M,N,Kd', [(2049, 4097, 32), (2500, 4500, 96), (3300, 3500, 672), (4353, 4000, 192)])
@pytest.mark.parametrize('epilogue', [None, 'gelu', 'residual'])
def test_rows_of_large_tiles(M, N, Kd, epilogue):
    """Tiles of 256 x 256, with one step of K, ragged ones and many; the last shape would need two rounds of them and takes
    the small ones."""
    x = rnd(M, Kd, seed=1, dtype=BF16)
    w, wv = K.mx4_quant(rnd(N, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    r = rnd(M, N, seed=3, dtype=BF16)
    close(K.mx4_mm(x.to(DEV), w, epilogue=epilogue, residual=r.to(DEV)), *want(x, wv.cpu(), epilogue=epilogue, residual=r))


@pytest.mark.parametrize('M,Kd', [(3, 768), (20, 1024), (20, 2048), (5, 20000)])
def test_layernorm_of_rows_far_from_zero(M, Kd):
    """Rows whose mean is far above their deviation: the variance is taken about the mean."""
    x = (100.0 + rnd(M, Kd, seed=1)).to(BF16)
    w, wv = K.mx4_quant(rnd(40, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    g = (1 + 0.2 * rnd(Kd, seed=4)).to(BF16)
    close(K.mx4_mm(x.to(DEV), w, ln_w=g.to(DEV)), *want(x, wv.cpu(), ln_w=g))


@pytest.mark.parametrize('M,N,Kd', [(1, 1, 1), (1, 130, 33), (3, 16, 128), (64, 64, 100), (65, 200, 160), (128, 128, 256),
                                    (130, 257, 1000), (500, 1025, 2049), (17, 5000, 384), (3500, 3600, 130),
                                    (4096, 3333, 520)])
@pytest.mark.parametrize('epilogue', [None, 'gelu', 'residual'])
def test_both(M, N, Kd, epilogue):
    a, av = K.mx4_quant(rnd(M, Kd, seed=1).to(DEV), values=True)
    w, wv = K.mx4_quant(rnd(N, Kd, seed=2, scale=1 / math.sqrt(Kd)).to(DEV), values=True)
    r = rnd(M, N, seed=3, dtype=BF16)
    got = K.mx4_mm(a, w, epilogue=epilogue, residual=r.to(DEV))
    close(got, *want(av.cpu(), wv.cpu(), epilogue=epilogue, residual=r))


def test_every_code_and_lane_order():
    """One-hot rows pick single weights: every value, position in a block and scale comes through in its place."""
    Kd, N = 256, 64
    g = torch.Generator().manual_seed(1)
    packed = torch.randint(0, 256, (N, Kd // 2), generator=g, dtype=torch.uint8)
    scale = torch.randint(97, 157, (N, Kd // 32), generator=g, dtype=torch.uint8)
    w = K.Mx4(packed.to(DEV), scale.to(DEV), Kd)
    wv = w.values().cpu()
    eye = torch.eye(Kd)
    one, ev = K.mx4_quant(eye.to(DEV), values=True)
    assert torch.equal(ev.cpu(), eye)
    exact = wv.t().to(BF16)
    assert torch.equal(exact.float(), wv.t())
    for r in (eye[:16], eye[100:132], eye[60:124], eye):
        got = K.mx4_mm(r.to(BF16).to(DEV), w)
        assert torch.equal(got.cpu(), exact[r.argmax(-1)])
    assert torch.equal(K.mx4_mm(one, w).cpu(), exact)


def test_nan_blocks_stay_in_their_rows_and_columns():
    M, N, Kd = 70, 40, 300
    x = rnd(M, Kd, seed=1)
    x[3, 290] = float('nan')
    wf = rnd(N, Kd, seed=2)
    wf[7, 299] = float('inf')
    w = K.mx4_quant(wf.to(DEV))
    got = K.mx4_mm(K.mx4_quant(x.to(DEV)), w).cpu()
    nan = torch.isnan(got)
    assert nan[3].all() and nan[:, 7].all() and int(nan.sum()) == N + M - 1
    w32 = K.mx4_quant(wf[:, :288].to(DEV))
    for m in (5, 30, 70):
        assert not torch.isnan(K.mx4_mm(torch.nan_to_num(x[:m, :288]).to(BF16).to(DEV), w32)).any()


def test_rows_in_place_strides_stream_and_graph():
    """out = residual, views with row strides, another stream, a captured call replayed: the plain call's bits."""
    for M in (4, 32, 200):
        Kd, N = 256, 96
        w = K.mx4_quant(rnd(N, Kd, seed=2).to(DEV))
        buf = rnd(M, 2 * Kd, seed=1, dtype=BF16).to(DEV)
        x = buf[:, Kd:]
        r = rnd(M, N + 5, seed=3, dtype=BF16).to(DEV)
        plain = K.mx4_mm(x.contiguous(), w, epilogue='residual', residual=r[:, :N].contiguous())
        o = r.clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            K.mx4_mm(x, w, epilogue='residual', residual=o[:, :N], out=o[:, :N])
        s.synchronize()
        assert torch.equal(o[:, :N], plain) and torch.equal(o[:, N:], r[:, N:])
        out = torch.empty_like(plain)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            K.mx4_mm(x, w, out=out)
        for i in range(3):
            buf.copy_(rnd(M, 2 * Kd, seed=10 + i, dtype=BF16))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, K.mx4_mm(x, w))


def test_empty_and_refusals():
    w = K.mx4_quant(rnd(8, 64, seed=1).to(DEV))
    assert K.mx4_mm(torch.empty(0, 64, device=DEV, dtype=BF16), w).shape == (0, 8)
    x = torch.zeros(4, 64, device=DEV, dtype=BF16)
    with pytest.raises(ValueError, match='bf16'):
        K.mx4_mm(x.float(), w)
    with pytest.raises(ValueError, match='values'):
        K.mx4_mm(x[:, :32], w)
    with pytest.raises(ValueError, match='LayerNorm'):
        K.mx4_mm(K.mx4_quant(x), w, ln_w=torch.ones(64, device=DEV, dtype=BF16))
    with pytest.raises(ValueError, match='residual'):
        K.mx4_mm(x, w, epilogue='residual')
    with pytest.raises(ValueError, match='epilogue'):
        K.mx4_mm(x, w, epilogue='relu')
    odd = K.mx4_quant(rnd(8, 70, seed=1).to(DEV))
    with pytest.raises(RuntimeError, match='multiple of 32'):
        K.mx4_mm(torch.zeros(4, 72, device=DEV, dtype=BF16)[:, :70], odd)
    with pytest.raises(RuntimeError, match='aligned'):
        K.mx4_mm(torch.zeros(4, 65, device=DEV, dtype=BF16)[:, 1:], w)
    with pytest.raises(ValueError, match='Mx4'):
        K.Mx4(w.packed, w.scale, 200)
    with pytest.raises(TypeError, match='dtype'):
        K.mx4_quant(torch.zeros(2, 32, device=DEV, dtype=torch.float64))
    with pytest.raises(RuntimeError, match='GPU'):
        K.mx4_quant(torch.zeros(2, 32))


def test_copies_hold_their_own_rows():
    w = K.mx4_quant(rnd(50, 200, seed=1).to(DEV))
    x = rnd(3, 200, seed=2).to(DEV)
    want = K.mx4_mm(K.mx4_quant(x), w)
    for c in (copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert c.at == c._buf.data_ptr() != w.at and c.shape == w.shape
        assert c.scale_at - c.at == w.scale_at - w.at and torch.equal(c.packed, w.packed)
        assert torch.equal(K.mx4_mm(K.mx4_quant(x), c), want)
    c = copy.copy(w)
    assert c.at == w.at and torch.equal(K.mx4_mm(K.mx4_quant(x), c), want)
