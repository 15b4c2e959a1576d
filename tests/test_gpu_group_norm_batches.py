"""Group norm of batches beyond a grid's third dimension whose gradients do not fit into registers where the results do."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


# one cell in long groups, and many cells of one channel: each just beyond what the gradients' form for small samples holds
@pytest.mark.parametrize("cells,channels,groups,kind", [(1, 4104, 1, "silu"), (3001, 1, 1, "leaky_relu")])
@pytest.mark.parametrize("batch", [65536, 131075])
def test_what_goes_forward_has_its_gradients(batch, cells, channels, groups, kind):
    import medvision_amd.ops as ops
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(batch, cells, channels, generator=g, device=DEV, dtype=torch.float16).requires_grad_(True)
    go = torch.randn(batch, cells, channels, generator=g, device=DEV, dtype=torch.float16)
    w, b = (torch.randn(channels, generator=g, device=DEV).requires_grad_(True) for _ in range(2))
    y = ops.group_norm_act(x, groups, w, b, activation=kind)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), go)
    for first in (0, 65500, batch - 36):   # the ends, and where one slice follows the other
        part = slice(first, first + 64)
        want = ref.group_norm(x[part], groups, w, b, 1e-5, kind, 0.01, go[part])
        check(y[part], *want[0], f"y from {first}")
        check(gx[part], *want[1], f"dx from {first}")
    parts = []   # the same sums of a sample, joined in 64 bits, each part rounded once
    for first in range(0, batch, 30000):
        part = slice(first, first + 30000)
        parts.append(torch.autograd.grad(ops.group_norm_act(x[part], groups, w, b, activation=kind), (w, b), go[part]))
    for name, total, of in (("dw", gw, [p[0] for p in parts]), ("db", gb, [p[1] for p in parts])):
        of = torch.stack(of).double().cpu()
        check(total, of.sum(0), 2.0 ** -24 * (of.abs().sum(0) + of.sum(0).abs()) * (1 + 2.0 ** -20), name)
    only = torch.autograd.grad(ops.group_norm_act(x, groups, w, b, activation=kind), (w, b), go)
    assert torch.equal(only[0], gw) and torch.equal(only[1], gb)


def test_the_same_limit_both_ways():
    """Sizes that the forward pass refuses are refused by the gradients' entry point, on the host."""
    import ctypes
    from medvision_amd import _lib
    lib = _lib.load()
    p = ctypes.c_void_p(16)
    assert lib.mv_group_norm(p, None, None, p, p, 65536, 5001, 8, 8, 1e-5, 0, 0.0, _lib.MV_F16, _lib.MV_F16, p, 1 << 50, None) == 1
    assert lib.mv_group_norm_backward(p, None, None, p, p, p, None, None, 65536, 5001, 8, 8, 0, 0.0, _lib.MV_F16, _lib.MV_F16, p, 1 << 50, None) == 1
    assert b"a batch of 65536" in lib.mv_last_error()
