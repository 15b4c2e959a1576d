"""Group norm of finite values whose squares 32 bits do not hold, against its 64-bit form."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def compare(x, groups, kind):
    import medvision_amd.ops as ops
    C = x.shape[-1]
    w, b, go = rand(2, C), rand(3, C), rand(4, *x.shape).to(x.dtype)
    ins = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = ops.group_norm_act(*(ins[0], groups, ins[1], ins[2]), activation=kind)
    grads = torch.autograd.grad(y, ins, go.to(DEV))
    for name, got, (want, bound) in zip(("y", "dx", "dw", "db"), (y, *grads), ref.group_norm(x, groups, w, b, 1e-5, kind, 0.01, go)):
        check(got, want, bound, name)


# cells that go into registers, cells of several chunks, fewer channels than a piece has
@pytest.mark.parametrize("shape", [(2, 100, 16, 2), (2, 20000, 16, 2), (1, 7, 24, 24), (1, 9000, 5, 1)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [1e18, 1e19, 1e25, 3e37])
def test_squares_too_large(shape, dtype, size):
    B, N, C, G = shape
    compare((size * rand(1, B, N, C)).to(dtype), G, "silu" if size > 1e20 else None)


@pytest.mark.parametrize("cells", [50, 8000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_cells_that_are_masked_with_the_lowest_value(cells, dtype):
    """A single cell of the type's lowest value among small ones; another sample and other groups beside it are as without."""
    import medvision_amd.ops as ops
    x = rand(1, 2, cells, 16).to(dtype)
    want = ops.group_norm_act(x.to(DEV), 2)
    x[0, cells // 3, :8] = torch.finfo(dtype).min
    compare(x, 2, None)
    y = ops.group_norm_act(x.to(DEV), 2)
    assert torch.equal(y[1], want[1]) and torch.equal(y[0, :, 8:], want[0, :, 8:])


@pytest.mark.parametrize("cells", [50, 8000])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_what_is_not_finite_stays_so(cells, bad):
    import medvision_amd.ops as ops
    x = 1e25 * rand(1, 2, cells, 16)
    x[1, cells // 2, 3] = bad
    y = ops.group_norm_act(x.to(DEV), 2)
    assert torch.isnan(y[1, :, :8]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[1, :, 8:]).all()


@pytest.mark.parametrize("cells", [60, 9000])
def test_small_channels_beside_large_ones(cells):
    """Channels of one piece of eight in groups of their own: each as by itself, whatever its neighbours hold."""
    import medvision_amd.ops as ops
    x = rand(1, 1, cells, 8) * 10.0 ** torch.tensor([0.0, 30, -3, 25, 0, 37, 10, 0]) + torch.tensor([0.0, 0, 5, 0, 1000, 0, 0, 7.25])
    x[..., 7] = 7.25
    compare(x, 8, None)
    y = ops.group_norm_act(x.to(DEV), 8).cpu()
    plain = x.clone()
    plain[..., [1, 3, 5]] = rand(9, 1, cells, 3)
    want = ops.group_norm_act(plain.to(DEV), 8).cpu()
    assert torch.equal(y[..., [0, 2, 4, 6, 7]], want[..., [0, 2, 4, 6, 7]])


@pytest.mark.parametrize("cells", [50, 8000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_groups_that_are_masked_throughout(cells, dtype):
    """Every cell of a group at the type's lowest or highest value: no variance, so that its cells are the bias."""
    import medvision_amd.ops as ops
    x = rand(1, 2, cells, 24).to(dtype)
    x[0, :, :8], x[1, :, 8:16] = torch.finfo(dtype).min, torch.finfo(dtype).max
    compare(x, 3, None)
    y = ops.group_norm_act(x.to(DEV), 3, None, torch.ones(24, device=DEV))
    assert (y[0, :, :8] == 1).all() and (y[1, :, 8:16] == 1).all()
