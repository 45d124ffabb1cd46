"""Rows of many tensors copied by one list (kernels.copy_rows) against indexing.  GPU only."""
import pytest
import torch

from treeattn_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def tensors(rows, seed):
    """Rows of 1, 2, 3, 8, 40, 256, 4000, 16 KiB + 4 and 64 KiB bytes, in several dtypes."""
    g = torch.Generator().manual_seed(seed)
    u8 = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8).to(DEV)
    return [u8(rows, 1), u8(rows, 3), u8(rows, 2), u8(rows), torch.randn(rows, 2, generator=g).to(DEV),
            torch.randn(rows, 10, generator=g).to(DEV), torch.randn(rows, 2, 64, generator=g).to(torch.bfloat16).to(DEV),
            torch.randn(rows, 1000, generator=g).to(DEV), torch.randn(rows, 4097, generator=g).to(DEV),
            torch.randn(rows, 2, 128, 64, generator=g).to(DEV).to(torch.float8_e4m3fn), torch.randn(rows, 128, 128, generator=g).to(DEV),
            torch.rand(rows, 5, generator=g).to(DEV) > 0.5, torch.randint(0, 99, (rows, 7), generator=g).to(DEV),
            u8(rows, 16385), torch.empty(rows, 0, device=DEV)]


def same(a, b):
    return all(torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x,
                           y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y) for x, y in zip(a, b))


def copied(xs, ys, src, dst):
    out = []
    for x, y in zip(xs, ys):
        f8 = y.dtype == torch.float8_e4m3fn
        z = (y.view(torch.uint8) if f8 else y).clone()
        z[dst.long()] = (x.view(torch.uint8) if f8 else x)[src.long()]
        out.append(z.view(y.dtype) if f8 else z)
    return out


@pytest.mark.parametrize('pairs', [1, 2, 7, 100])
def test_within_and_between(pairs):
    rows = 230
    perm = torch.randperm(rows, generator=torch.Generator().manual_seed(pairs)).to(torch.int32).to(DEV)
    src, dst = perm[:pairs].contiguous(), perm[pairs:2 * pairs].contiguous()
    xs = tensors(rows, 1)
    want = copied(xs, xs, src, dst)
    K.copy_rows(xs, src, dst)
    assert same(xs, want)
    ys = tensors(rows + 50, 2)
    dst = torch.randperm(rows + 50)[:pairs].to(torch.int32).to(DEV)
    want = copied(xs, ys, src, dst)
    K.copy_rows(xs, src, dst, out=ys)
    assert same(ys, want)
    K.copy_rows(xs, src[:1].expand(pairs).contiguous(), dst, out=ys)      # one row to many places
    assert same(ys, copied(xs, ys, src[:1].expand(pairs), dst))


def test_more_tensors_than_a_launch_takes():
    xs = [torch.randn(9, 1 + i % 5, device=DEV) for i in range(100)]
    src, dst = torch.tensor([0, 3, 4], dtype=torch.int32, device=DEV), torch.tensor([8, 1, 2], dtype=torch.int32, device=DEV)
    want = copied(xs, xs, src, dst)
    K.copy_rows(xs, src, dst)
    assert same(xs, want)


def test_ids_outside_copy_nothing():
    xs = tensors(20, 3)
    want = copied(xs, xs, torch.tensor([4], device=DEV), torch.tensor([9], device=DEV))
    K.copy_rows(xs, torch.tensor([-1, 4, 20, 3, 5], dtype=torch.int32, device=DEV),
                torch.tensor([2, 9, 1, -7, 1 << 30], dtype=torch.int32, device=DEV))
    assert same(xs, want)
    K.copy_rows(xs, torch.empty(0, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV))
    K.copy_rows([], torch.empty(0, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV))
    assert same(xs, want)


def test_rows_far_apart():
    """Rows past 2^32 bytes, and rows that long themselves would be: offsets in 64 bits."""
    x = torch.zeros(70000, 1 << 16, dtype=torch.uint8, device=DEV)
    x[69999] = 7
    K.copy_rows([x], torch.tensor([69999], dtype=torch.int32, device=DEV), torch.tensor([66001], dtype=torch.int32, device=DEV))
    assert bool((x[66001] == 7).all()) and not x[66000].any() and not x[66002].any()


def test_graph():
    xs = tensors(50, 5)
    src, dst = torch.tensor([1, 2], dtype=torch.int32, device=DEV), torch.tensor([40, 41], dtype=torch.int32, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        K.copy_rows(xs, src, dst)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(3):
        src.fill_(3 + i)
        src[1] = 20 + i
        want = copied(xs, xs, src, dst)
        g.replay()
        torch.cuda.synchronize()
        assert same(xs, want)


def test_refusals():
    x = torch.zeros(4, 8, device=DEV)
    i = torch.zeros(1, dtype=torch.int32, device=DEV)
    for bad in (lambda: K.copy_rows([x], i.long(), i), lambda: K.copy_rows([x], i, torch.zeros(2, dtype=torch.int32, device=DEV)),
                lambda: K.copy_rows([x[:, :4]], i, i), lambda: K.copy_rows([x], i, i, out=[x, x]),
                lambda: K.copy_rows([x], i, i, out=[x.half()]), lambda: K.copy_rows([x], i, i, out=[torch.zeros(4, 9, device=DEV)]),
                lambda: K.copy_rows([x, torch.zeros(())], i, i), lambda: K.copy_rows([x.cpu()], i, i),
                lambda: K.copy_rows([x], i.cpu(), i.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
