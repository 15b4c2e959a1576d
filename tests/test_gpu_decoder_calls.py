"""What callers may give the region decoders' operators, which gradients they get, and what transforms of functions do."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rand(seed, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


# ---- lengths -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind,keys,lengths", [
    (torch.uint8, 300, (255, 0, 7)), (torch.int8, 300, (127, -3, 0)), (torch.int16, 40000, (32767, -3, 5)),
    (torch.uint16, 70000, (65535, 0, 9)), (torch.uint32, 300, (2 ** 32 - 1, 0, 7))])
def test_lengths_of_every_whole_number_type(kind, keys, lengths):
    """More keys than the type can count."""
    import medvision_amd.ops as ops
    q, k, v = rand(1, 3, 5, 2, 16), rand(2, 3, keys, 2, 16), rand(3, 3, keys, 2, 16)
    want = ops.cross_attention(q, k, v, key_lengths=torch.tensor(lengths, device=DEV))
    assert torch.equal(ops.cross_attention(q, k, v, key_lengths=torch.tensor(lengths, dtype=kind, device=DEV)), want)


def test_lengths_beyond_int64_are_refused():
    import medvision_amd.ops as ops
    q = rand(1, 2, 5, 2, 16)
    with pytest.raises(RuntimeError, match="fit into int64"):
        ops.cross_attention(q, q, q, key_lengths=torch.tensor([1, 2], device=DEV).to(torch.uint64))
