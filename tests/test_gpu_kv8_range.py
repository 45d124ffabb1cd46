"""The 8-bit cache at the end of float16's range: a magnitude near 65504 is rounded up to 65536 in its page and must not come
back as infinity.  GPU only."""
import pytest
import torch

from oracle import low_bits as O
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F16 = torch.float16


def cache(B, H, D, leaf, tcap, T, k, v):
    nb = tcap // leaf
    c = K.Cache8(torch.zeros(B * H * nb, 2, leaf, D, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn),
                 torch.ones(B * H * nb, 2, device=DEV), torch.arange(B * H * nb, dtype=torch.int32, device=DEV).view(B, H, nb),
                 torch.zeros(B, H, 2, leaf, D, device=DEV, dtype=F16), torch.full((B, H), -1, dtype=torch.int32, device=DEV), tcap)
    o = O.Cache(B, H, D, leaf, tcap)
    K.kv8_fill(k.to(DEV), v.to(DEV), c)
    for b in range(B):
        for h in range(H):
            for t in range(T):
                o.append(b, h, t, k[b, h, t], v[b, h, t])
    return c, o


def extremes(B, H, T, D):
    """Small keys; values near +-65504 in one block, what rounds up, what does not, and an infinity in a place of its own."""
    g = torch.Generator().manual_seed(5)
    k, v = torch.randn(B, H, T, D, generator=g), torch.randn(B, H, T, D, generator=g)
    v[:, :, 4:8, 0] = 65504.0
    v[:, :, 4:8, 1] = -65504.0
    v[:, :, 4:8, 2] = 63520.0
    v[:, :, 4:8, 3] = -63488.0          # halfway between 61440 and 65536: to the even code
    v[:, :, 4:8, 4] = 61000.0
    k[:, :, 5, 7] = -65504.0
    return k.to(F16), v.to(F16)


@pytest.mark.parametrize('D', [16, 64])
def test_attention_over_values_that_round_up(D):
    """A query that only such values answer gets 65504, as from the cache in float16, in each form of the kernel."""
    B, H, leaf, tcap, T = 1, 2, 4, 16, 13
    k, v = extremes(B, H, T, D)
    q = torch.zeros(B, H, 1, D, dtype=F16)
    q[:, 1] = 1.0
    k[:, :, 4] = 100.0                  # row 4 takes all the weight of head 1's query
    c, o = cache(B, H, D, leaf, tcap, T, k, v)
    ids = torch.tensor([1], dtype=torch.int32).expand(B, H, 1, 1).contiguous()
    tq = torch.tensor([[T - 1]], dtype=torch.int32)
    for nsplit in (1, 4, 8):
        out, _, _ = K.seg_attn8(q.to(DEV), c, tq.to(DEV), ids.to(DEV), torch.ones_like(ids, dtype=torch.bool).to(DEV), None, 3, 1.0,
                                nsplit=nsplit)
        assert torch.isfinite(out).all(), nsplit
        for h in range(H):
            want, _, _ = O.attend8(o, q[0, h, 0].double(), 0, h, T - 1, [1], [], 3, 1.0)
            want = want.clamp(-65504.0, 65504.0)
            # float16's half step, and weights and sums off by less than 2^-16 of the largest value
            tol = 2.0 ** -11 * want.abs() + 2.0 ** -16 * 65536.0
            assert ((out[0, h, 0].cpu().double() - want).abs() <= tol).all(), (nsplit, h)
        assert out[0, 1, 0, 0] == 65504.0 and out[0, 1, 0, 1] == -65504.0


def test_dense_rows_are_the_restored_rows():
    """dense() gives what kv8_append restores from the same page, finite for finite rows; NaN stays."""
    B, H, D, leaf, tcap, T = 1, 1, 16, 4, 16, 12
    k, v = extremes(B, H, T, D)
    v[0, 0, 6, 9] = float('inf')        # NaN in the page
    c, _ = cache(B, H, D, leaf, tcap, T, k, v)
    dk, dv = c.dense(0, 8)
    assert torch.isfinite(dk).all()
    nan = torch.isnan(dv)
    assert nan[0, 0, 6, 9] and int(nan.sum()) == 1 and torch.isfinite(dv[~nan]).all()
    assert dv[0, 0, 4, 0] == 65504.0 and dv[0, 0, 5, 1] == -65504.0
    K.kv8_append(k[:, :, 7].to(DEV), v[:, :, 7].to(DEV), c, torch.tensor([7], dtype=torch.int32, device=DEV), [], 2)
    tail = c.tail[0, 0].nan_to_num(nan=123.0)
    assert torch.equal(tail[0, :3], dk[0, 0, 4:7]) and torch.equal(tail[1, :3], dv[0, 0, 4:7].nan_to_num(nan=123.0))
