"""Group norm whose results are more than caches hold: written past them, with the same bits."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
CELLS, BATCH = 5001, 1200   # (more cells than go into registers; as many samples as have one share of the cells each, half of them too)
PAST = 128 << 20


@pytest.mark.parametrize("dtype,channels,groups,kind", [(torch.float16, 20, 5, "leaky_relu"), (torch.bfloat16, 20, 4, "gelu"), (torch.float32, 11, 11, "silu"),
                                                        (torch.float16, 16, 2, None), (torch.bfloat16, 17, 1, "relu"), (torch.float32, 9, 3, "gelu")])
def test_the_same_as_half_of_it(dtype, channels, groups, kind):
    import medvision_amd.ops as ops
    g = torch.Generator(device=DEV).manual_seed(1)
    x, go = (torch.randn(BATCH, CELLS, channels, generator=g, device=DEV).to(dtype) for _ in range(2))
    w, b = (torch.randn(channels, generator=g, device=DEV) for _ in range(2))
    size = x.numel() * x.element_size()
    assert size > PAST >= size // 2

    def run(part):
        ins = [x[part].requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
        y = ops.group_norm_act(ins[0], groups, ins[1], ins[2], activation=kind)
        return (y.detach(), *torch.autograd.grad(y, ins, go[part]))

    y, gx, gw, gb = run(slice(0, BATCH))
    halves = [run(slice(first, first + BATCH // 2)) for first in (0, BATCH // 2)]
    for n, (hy, hx, _, _) in enumerate(halves):
        part = slice(n * BATCH // 2, (n + 1) * BATCH // 2)
        assert torch.equal(y[part], hy) and torch.equal(gx[part], hx)
    for total, index in ((gw, 2), (gb, 3)):   # each of the three is a sum in 64 bits, rounded once
        of = torch.stack([h[index] for h in halves]).double()
        assert ((total.double() - of.sum(0)).abs() <= 2.0 ** -24 * (of.abs().sum(0) + total.double().abs())).all()
    for sample in (0, BATCH - 1):
        part = slice(sample, sample + 1)
        want = ref.group_norm(x[part], groups, w, b, 1e-5, kind, 0.01, go[part])
        check(y[part], *want[0], f"y {sample}")
        check(gx[part], *want[1], f"dx {sample}")
