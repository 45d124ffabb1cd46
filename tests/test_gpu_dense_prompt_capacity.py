"""A prompt's kernels go by the prompt, not by how many positions the cache could hold: the same bits whatever Tcap is, and the
rows of the cache too.  GPU only."""
import pytest
import torch

from test_gpu_dense_decoder import BF16, DEV, dec, model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('T0', [100, 257])
@pytest.mark.parametrize('chunk', [None, 5])
def test_prompts_in_caches_of_any_capacity(T0, chunk):
    m, cfg = model(BF16, n_head=12, dh=64, rope='half')
    idx = torch.randint(0, 97, (16, T0), generator=torch.Generator().manual_seed(1)).to(DEV)
    ds = [dec(m, cfg, batch=16, Tcap=n, max_tokens=320) for n in (T0 + 63, 600, 70000)]
    a = [d.prefill(idx, chunk=chunk) for d in ds]
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])
    for b in (0, 15):
        for x in zip(*(d.states[1].dense_kv(b, T0) for d in ds)):
            assert torch.equal(x[0], x[1]) and torch.equal(x[0], x[2])
    lg = [d.step(idx[:, 0], T0)[0] for d in ds]
    size = float(lg[0].float().abs().max())
    assert all(float((x.float() - lg[0].float()).abs().max()) <= 0.05 * size for x in lg)
