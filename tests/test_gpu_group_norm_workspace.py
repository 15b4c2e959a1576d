"""Group norm through its C entry points with just the room that the queries name: nothing behind it is written."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("shape", [(1, 343, 256, 32), (70, 3, 8, 2), (3, 1955, 60, 6), (2, 4000, 16, 2), (2, 27000, 20, 5), (3, 40, 4104, 1), (1, 6000, 3, 3)])
@pytest.mark.parametrize("wanted", [(True, True, True), (True, False, False), (False, True, False), (False, False, True)])
def test_room(shape, wanted):
    from medvision_amd import _lib
    lib = _lib.load()
    B, N, C, G = shape
    g = torch.Generator().manual_seed(1)
    x, go = (torch.randn(B, N, C, generator=g).half() for _ in range(2))
    w, b = (torch.randn(C, generator=g) for _ in range(2))
    want = ref.group_norm(x, G, w, b, 1e-5, "silu", 0.0, go)
    t = [v.to(DEV) for v in (x, w, b, go)]
    out = [torch.full_like(v, 7.0) for v in (t[0], t[0], t[1], t[2])]   # y, dx, dw, db
    stats = torch.full((3 * B * G + 8,), 7.0, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    sizes = (B, N, C, G)
    for backward in (False, True):
        room = (lib.mv_group_norm_backward_workspace_bytes if backward else lib.mv_group_norm_workspace_bytes)(*sizes)
        work = torch.full((room + 4096,), 0x7f, device=DEV, dtype=torch.uint8)
        if backward:
            to = [v.data_ptr() if wish else None for v, wish in zip(out[1:], wanted)]
            status = lib.mv_group_norm_backward(*(v.data_ptr() for v in t[:3]), stats.data_ptr(), t[3].data_ptr(), *to, *sizes, 3, 0.0, _lib.MV_F16, _lib.MV_F32,
                                                work.data_ptr(), room, stream)
        else:
            status = lib.mv_group_norm(*(v.data_ptr() for v in t[:3]), out[0].data_ptr(), stats.data_ptr(), *sizes, 1e-5, 3, 0.0, _lib.MV_F16, _lib.MV_F32,
                                       work.data_ptr(), room, stream)
        assert status == 0 and (work[room:] == 0x7f).all() and (stats[3 * B * G:] == 7).all()
    for name, got, (v, bound), wish in zip(("y", "dx", "dw", "db"), out, want, (True, *wanted)):
        if wish:
            check(got, v, bound, name)
        else:
            assert (got == 7).all(), name
