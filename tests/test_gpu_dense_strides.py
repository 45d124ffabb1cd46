"""kernels.dense_attn over views whose dimensions of one have strides of any size: those are never a step.  GPU only."""
import pytest
import torch

from test_gpu_dense import BF16, DEV, F32
from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('nsplit', [1, 64])
def test_strides_of_single_dimensions(dtype, nsplit):
    g = torch.Generator(device=DEV).manual_seed(1)
    randn = lambda *s: torch.randn(*s, device=DEV, generator=g).to(dtype)
    k, v, q = randn(1, 1, 300, 64), randn(1, 1, 300, 64), randn(1, 1, 1, 64)
    tq = torch.tensor([299], device=DEV)
    want = K.dense_attn(q, k, v, tq, nsplit=nsplit)[0]
    odd = lambda x, *st: x.as_strided(x.shape, st)
    got = K.dense_attn(odd(q, 7, 3, 5, 1), odd(k, 19201, 11, 64, 1), odd(v, 1, 2, 64, 1), tq, nsplit=nsplit)[0]
    assert torch.equal(got, want)
    one = K.dense_attn(odd(q, 7, 3, 5, 1), odd(k[:, :, :1], 9, 9, 9, 1), odd(v[:, :, :1], 1, 1, 33, 1), tq * 0, nsplit=nsplit)[0]
    assert torch.equal(one, v[:, :, :1])
    with pytest.raises(RuntimeError, match='aligned'):      # two tokens: a step
        K.dense_attn(randn(1, 1, 2, 65)[..., :64], k, v, torch.tensor([3, 4], device=DEV), nsplit=nsplit)
