"""Host-side checks of the 8-bit cache and the 4-bit rows: the float64 restatement against torch's own e4m3 rounding and a
direct search, and what the library and the wrappers refuse (no GPU here: refused calls launch nothing)."""
import ctypes
import math

import pytest
import torch

from oracle import low_bits as O


def test_round8_is_the_e4m3_rounding():
    g = torch.Generator().manual_seed(1)
    y = torch.cat((torch.randn(4000, generator=g) * torch.exp(3 * torch.randn(4000, generator=g)),
                   torch.arange(-448, 449) / 16.0, torch.tensor([0.0, -0.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, 448.0])))
    y = y.clamp(-448, 448).double()
    assert torch.equal(O.round8(y), y.float().to(torch.float8_e4m3fn).double())


def test_scale8_is_the_smallest_power_that_fits():
    for a in (1.0, 448.0, 448.0001, 0.875, 3e-40, 2.0 ** -140, 3e38, 511.9, 512.0):
        s = O.scale8(torch.tensor([a, -a / 3, 0.0], dtype=torch.float64))
        assert math.frexp(s)[0] == 0.5 and a <= 448 * s and (a > 448 * s / 2 or s == 2.0 ** -126)
    assert O.scale8(torch.zeros(4, dtype=torch.float64)) == 1.0
    assert O.scale8(torch.tensor([float('inf'), float('nan')], dtype=torch.float64)) == 1.0


def test_quant4_picks_the_nearest_value():
    x = torch.randn(6, 96, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    code, byte, val = O.quant4(x)
    for r in range(6):
        for k in range(96):
            s = 2.0 ** (int(byte[r, k // 32]) - 127)
            d = [abs(abs(x[r, k].item()) / s - v) for v in O.GRID4]
            assert abs(abs(val[r, k].item()) / s - abs(x[r, k].item()) / s) == min(d)
    amax = x.view(6, 3, 32).abs().amax(-1)
    s = torch.exp2(byte[:, :3].double() - 127)
    assert (amax / s < 8).all() and (amax / s >= 4).all()


@pytest.fixture(scope='module')
def lib():
    from treeattn_amd import _lib
    return _lib


def refused(lib, rc, code, text):
    assert rc == code and text in lib.lib().ta_last_error(), (rc, lib.lib().ta_last_error())


def test_cache_calls_refuse_bad_descriptions(lib):
    L = lib.lib()
    P = 4096      # never dereferenced

    def kv8(**kw):
        d = dict(pool=P, scale=P, table=P, sb=8, sh=4, num_pages=10, tail=P, tail_sb=4096, tail_sh=2048, tail_block=P, tb_sb=2,
                 block_log2=4, tcap=64)
        d.update(kw)
        return ctypes.byref(lib.Kv8(*[d[n] for n, _ in lib.Kv8._fields_]))

    def append(c, D=64, dtype=2, levels=0, arity=1):
        return L.ta_kv8_append(P, P, dtype, 64, 64, 64, 64, c, 1, 2, D, P, levels, None, None, None, arity, None)
    refused(lib, append(None), 1, b'bad cache description')
    refused(lib, append(kv8(num_pages=0)), 1, b'bad cache description')
    refused(lib, append(kv8(block_log2=0)), 1, b'bad cache description')
    refused(lib, append(kv8(tcap=0)), 1, b'bad cache description')
    refused(lib, append(kv8(pool=P + 8)), 1, b'16-byte aligned')
    refused(lib, append(kv8(scale=P + 4)), 1, b'8-byte aligned')
    refused(lib, append(kv8(tail_sb=4100)), 1, b'16-byte aligned')
    refused(lib, append(kv8(), D=48), 2, b'head dim')
    refused(lib, append(kv8(), dtype=7), 1, b'dtype')
    refused(lib, append(kv8(), arity=5), 1, b'arity')
    refused(lib, append(kv8(), levels=33), 1, b'32 levels')
    refused(lib, append(kv8(), levels=2), 1, b'addresses')
    one = (ctypes.c_int64 * 1)(0)
    refused(lib, L.ta_kv8_append(P, P, 2, 64, 64, 64, 64, kv8(), 1, 2, 64, P, 1, one, one, one, 1, None), 1, b'addresses')

    def fill(T=64, k=P, kst=64):
        return L.ta_kv8_fill(k, P, 2, 4096, 4096, kst, 4096, 4096, 64, kv8(), 1, 2, T, 64, None, None)
    refused(lib, fill(T=65), 1, b'tcap')
    refused(lib, fill(k=P + 2), 1, b'16-byte')
    refused(lib, fill(k=P + 1), 1, b'16-byte')
    refused(lib, fill(kst=65), 1, b'16-byte')

    def attend(c=None, wl=4, local=3, nsplit=1, ws=None, nb=0, q=P, B=1, Nq=1):
        return L.ta_seg_attn8_fwd(q, 2, 128, 64, 64, c or kv8(), B, 2, Nq, 64, P, 1, P, P, None, wl, local, 1.0, None, None, nb, P,
                                  128, 64, 64, None, None, nsplit, ws, 0, None)
    refused(lib, attend(wl=513), 1, b'512 leaves')
    refused(lib, attend(nsplit=6), 1, b'multiple of 4')
    refused(lib, attend(nsplit=260), 1, b'at most 256')
    refused(lib, attend(local=32), 2, b'local window')
    refused(lib, attend(nb=3), 1, b'neighbour slots')
    refused(lib, attend(nsplit=8), 4, b'workspace')
    refused(lib, attend(q=P + 8), 1, b'16-byte')
    refused(lib, attend(B=40000), 2, b'65535')
    refused(lib, attend(c=kv8(num_pages=1 << 27)), 2, b'2^31 rows')
    assert attend(Nq=0) == 0


def test_products_refuse_bad_arguments(lib):
    L = lib.lib()
    P = 4096

    def rows(X=P, ldx=64, M=4, N=8, K=64, epi=0, R=None, ln=None, Y=P, ldy=8, ws=None, W=P):
        return L.ta_mx4_rows(X, ldx, W, P, Y, ldy, R, 8, ln, 1e-5, M, N, K, epi, ws, 0, None)
    refused(lib, rows(K=48, ldx=48), 1, b'multiple of 32')
    refused(lib, rows(ldx=32), 1, b'bad sizes')
    refused(lib, rows(N=0x7fffffff, M=1), 1, b'bad sizes')
    refused(lib, rows(M=0x7fffffff), 1, b'bad sizes')
    refused(lib, rows(epi=3), 1, b'bad sizes')
    refused(lib, rows(epi=2), 1, b'residual')
    refused(lib, rows(X=P + 2), 1, b'16-byte')
    refused(lib, rows(W=P + 8), 1, b'16-byte')
    refused(lib, rows(ldx=68), 1, b'multiple of 8')
    refused(lib, rows(ldx=1 << 26), 2, b'2^25')
    refused(lib, rows(M=20, K=4096, ldx=4096, ln=P), 4, b'workspace')
    assert rows(M=0) == 0
    assert L.ta_mx4_rows_workspace_size(20, 4096, 1) == 20 * 4096 * 2 and L.ta_mx4_rows_workspace_size(20, 4096, 0) == 0
    assert L.ta_mx4_rows_workspace_size(32, 1024, 1) == 0 and L.ta_mx4_rows_workspace_size(65, 64, 1) == 65 * 64 * 2

    def both(K=64, M=4, N=8, ldy=8, Xs=P, Xp=P):
        return L.ta_mx4_both(Xp, Xs, P, P, P, ldy, None, 0, M, N, K, 0, None)
    refused(lib, both(K=0), 1, b'bad sizes')
    refused(lib, both(N=0x7fffffff, M=1), 1, b'bad sizes')
    refused(lib, both(ldy=4), 1, b'bad sizes')
    refused(lib, both(Xp=P + 4), 1, b'aligned')
    refused(lib, both(Xs=P + 2), 1, b'aligned')
    refused(lib, L.ta_mx4_quant(P, 2, 64, 4, 0, P, P, None, 0, None), 1, b'bad sizes')
    refused(lib, L.ta_mx4_quant(P, 9, 64, 4, 64, P, P, None, 0, None), 1, b'dtype')
    refused(lib, L.ta_mx4_quant(P, 2, 64, 4, 64, P + 4, P, None, 0, None), 1, b'aligned')
    refused(lib, L.ta_mx4_quant(P, 2, 64, 4, 64, P, P, P, 32, None), 1, b'bad sizes')
    assert L.ta_mx4_quant(None, 2, 64, 0, 64, None, None, None, 0, None) == 0


def test_wrappers_refuse_host_tensors():
    from treeattn_amd import kernels as K
    with pytest.raises(RuntimeError, match='GPU'):
        K.mx4_quant(torch.zeros(4, 64))
    with pytest.raises(RuntimeError, match='GPU'):
        K.Mx4(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 128)
    with pytest.raises(ValueError, match='Mx4'):
        K.Mx4(torch.zeros(4, 60, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 128)
    with pytest.raises(TypeError, match='Mx4'):
        K.mx4_mm(torch.zeros(4, 64), torch.zeros(4, 64))
    pool = torch.zeros(3, 2, 8, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    args = [pool, torch.ones(3, 2), torch.zeros(1, 1, 2, dtype=torch.int32), torch.zeros(1, 1, 2, 8, 16),
            torch.full((1, 1), -1, dtype=torch.int32), 16]
    with pytest.raises(RuntimeError, match='GPU'):
        K.Cache8(*args)
    for i, bad, text in ((0, pool.float(), 'pool'), (1, torch.ones(3), 'scale'), (2, torch.zeros(1, 1, 1, dtype=torch.int32), 'table'),
                         (3, torch.zeros(1, 1, 2, 8, 8), 'tail'), (4, torch.zeros(1, 1), 'tail_block'), (5, 0, 'table')):
        with pytest.raises(ValueError, match=text):
            K.Cache8(*[bad if j == i else a for j, a in enumerate(args)])


def test_wavefronts_per_query():
    from treeattn_amd.engine import decode_nsplit, decode_nsplit8
    assert decode_nsplit8(32, 12, 1, 32, 64) == decode_nsplit(32, 12, 32, 64) == 4
    assert decode_nsplit8(1, 12, 1, 64, 128) == decode_nsplit(1, 12, 64, 128) == 64
    assert decode_nsplit8(4, 12, 32, 16, 64) == 4 and decode_nsplit8(4, 12, 128, 16, 64) == 1
    assert all(n == 1 or n % 4 == 0 and n <= 256 for B in (1, 7, 400) for H in (1, 12) for Nq in (1, 5, 900) for wl in (0, 4, 512)
               for leaf in (2, 64) for n in [decode_nsplit8(B, H, Nq, wl, leaf)])
