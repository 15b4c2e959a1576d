"""4-bit products in the forms that full workspaces, short sums and aligned rows do not reach."""
import pytest
import torch

import tokens_ref as ref
from decoder_ref import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("shape", [(1, 40000, 40), (2, 40001, 130), (1, 87808, 257), (2, 65536, 8), (1, 33000, 3)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_long_sums_of_a_row_or_two_in_parts(shape, group):
    """The sum of each output in several workgroups, joined with the bias: outputs in fours and not."""
    import medvision_amd.ops as ops
    from medvision_amd import _lib
    M, K, N = shape
    parts, rest = divmod(_lib.load().mv_group_linear_workspace_bytes(M, K, N), 4 * M * N)
    assert rest == 0 and parts > 1
    dtype = (torch.float16, torch.bfloat16)[(M + group // 32) % 2]
    x, bias = rand(1, M, K, dtype=dtype), rand(2, N, dtype=dtype)
    codes, scales = (t.cpu() for t in ops.quantize_groups((rand(3, N, K) * torch.exp(rand(4, N, 1))).to(DEV), group))
    for add in (bias, None):
        got = ops.group_linear(x.to(DEV), codes.to(DEV), scales.to(DEV), None if add is None else add.to(DEV))
        check(got, *ref.group_linear(x, codes, scales, add), shape)


def whole_query(lib, rows, inputs, outputs):
    """What the query gives for these rows: the copy of the rows, and the parts."""
    copy = 2 * rows * -(-inputs // 128) * 128 if rows > 64 and inputs % 8 else 0
    return copy, lib.mv_group_linear_workspace_bytes(rows, inputs, outputs)


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("inputs", [1111, 2048, 1000])
@pytest.mark.parametrize("rows", [3, 40, 65, 130, 300])
@pytest.mark.parametrize("group,dtype", [(32, torch.float16), (64, torch.bfloat16), (128, torch.float16)])
def test_any_workspace(rows, inputs, shift, group, dtype):
    """None, too little for the copy, the copy alone, a byte less than the query, all of it: the same within the bound, and nothing
    behind it is written.  Rows that start anywhere: then the copy takes the place of parts, or there is neither."""
    from medvision_amd import _lib
    lib = _lib.load()
    N = 100 + rows % 2
    x, bias = rand(1, rows, inputs, dtype=dtype), rand(2, N, dtype=dtype)
    codes, scales = ref.quantize_groups(rand(3, N, inputs), group)
    want, bound = ref.group_linear(x, codes, scales, bias)
    space = torch.full((rows * inputs + 64,), float("nan"), device=DEV, dtype=dtype)
    here = space[8 + shift:8 + shift + rows * inputs].view(rows, inputs).copy_(x)
    t = [v.to(DEV) for v in (codes, scales, bias)]
    copy, full = whole_query(lib, rows, inputs, N)
    for size in sorted({0, max(0, copy - 1), copy, max(0, full - 1), full, full + 2 * rows * (inputs + 127)}):
        work = torch.full((size + 256,), 0x7f, device=DEV, dtype=torch.uint8)   # (read as numbers: large)
        y = torch.full((rows + 1, N), 7.0, device=DEV, dtype=dtype)
        status = lib.mv_group_linear(here.data_ptr(), *(v.data_ptr() for v in t), y.data_ptr(), rows, inputs, N, group,
                                     _lib.MV_F16 if dtype == torch.float16 else _lib.MV_BF16, work.data_ptr() if size else None, size,
                                     torch.cuda.current_stream().cuda_stream)
        assert status == 0
        check(y[:rows], want, bound, size)
        assert (y[rows] == 7).all() and (work[size:] == 0x7f).all()
