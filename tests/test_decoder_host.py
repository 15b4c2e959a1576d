"""Host side of the region decoders' operators: refusals, workspaces, and the 64-bit forms that the GPU tests compare with."""
import ctypes

import pytest
import torch

import decoder_ref as ref


def test_cpu_tensors_are_refused():
    import medvision_amd.ops as ops
    x = torch.zeros(2, 3, 4, 16)
    with pytest.raises(RuntimeError, match="cross_attention is not implemented on CPU"):
        ops.cross_attention(x, x, x)
    with pytest.raises(RuntimeError, match="add_rms_norm is not implemented on CPU"):
        ops.add_rms_norm(x, x, torch.ones(16))
    with pytest.raises(RuntimeError, match="add_rms_norm_quantized is not implemented on CPU"):
        ops.add_rms_norm_quantized(x, x, torch.ones(16))
    with pytest.raises(RuntimeError, match="quantize_blocks is not implemented on CPU"):
        ops.quantize_blocks(x)
    with pytest.raises(RuntimeError, match="block_linear is not implemented on CPU"):
        ops.block_linear(x, x, x, x)


def _shape(batch=1, queries=2, keys=3, heads=4, key_heads=2, dim=16):
    from medvision_amd import _lib
    s = _lib.AttentionShape(batch, queries, keys, heads, key_heads, dim)
    return s


def test_entry_points_refuse_on_the_host():
    from medvision_amd import _lib
    lib = _lib.load()
    for shape in (_shape(key_heads=3), _shape(dim=129), _shape(dim=0), _shape(batch=-1), _shape(key_heads=0)):
        assert lib.mv_cross_attention_forward(*[None] * 8, ctypes.byref(shape), 1.0, _lib.MV_F32, None, 0, None) == 1
        assert lib.mv_last_error()
    good = _shape()
    assert lib.mv_cross_attention_forward(*[None] * 8, ctypes.byref(good), 1.0, _lib.MV_F64, None, 0, None) == 1
    assert b"float32, float16 or bfloat16" in lib.mv_last_error()
    assert lib.mv_cross_attention_forward(*[None] * 8, ctypes.byref(good), 1.0, _lib.MV_F32, None, 0, None) == 1
    assert b"missing" in lib.mv_last_error()
    assert lib.mv_cross_attention_forward(*[None] * 8, None, 1.0, _lib.MV_F32, None, 0, None) == 1
    assert lib.mv_cross_attention_forward(*[None] * 8, ctypes.byref(_shape(queries=0)), 1.0, _lib.MV_F32, None, 0, None) == 0
    assert lib.mv_add_rms_norm(*[None] * 5, 4, 0, 1e-6, _lib.MV_F32, _lib.MV_F32, None) == 1
    assert lib.mv_add_rms_norm(*[None] * 5, 4, 8, 1e-6, _lib.MV_F16, _lib.MV_BF16, None) == 1
    assert lib.mv_quantize_blocks(*[None] * 3, 4, 8, 2, _lib.MV_F32, None) == 1
    assert lib.mv_block_linear(*[None] * 6, 4, 100, 8, _lib.MV_F16, None, 0, None) == 1
    assert lib.mv_block_linear(*[None] * 6, 4, 128, 8, _lib.MV_F32, None, 0, None) == 1
    assert lib.mv_block_linear(*[None] * 6, 0, 128, 8, _lib.MV_F16, None, 0, None) == 0


def test_workspace_queries():
    from medvision_amd import _lib
    lib = _lib.load()
    s = _shape(2, 100, 50, 4, 2, 32)
    assert lib.mv_cross_attention_backward_workspace_bytes(ctypes.byref(s), _lib.MV_F16) >= 4 * 2 * 4 * 100
    assert lib.mv_cross_attention_backward_workspace_bytes(ctypes.byref(_shape(dim=999)), _lib.MV_F16) == 0
    assert lib.mv_add_rms_norm_backward_workspace_bytes(10, 64) > 0
    assert lib.mv_add_rms_norm_backward_workspace_bytes(-1, 64) == 0


def test_plain_attention_agrees_with_autograd():
    g = torch.Generator().manual_seed(0)
    q, go = (torch.randn(2, 7, 4, 8, generator=g) for _ in range(2))
    k, v = (torch.randn(2, 9, 2, 8, generator=g) for _ in range(2))
    mask = torch.rand(2, 9, generator=g) < 0.6
    mask[1] = False
    got = ref.attention(q, k, v, mask, None, 0.4, go)
    ins = [t.double().requires_grad_(True) for t in (q, k, v)]
    value = ref.attention_value(*ins, go.double(), mask, 0.4)
    for (d, _), want in zip(got[1:], torch.autograd.grad(value, ins)):
        assert torch.allclose(d, want.nan_to_num(0.0), atol=1e-12)
    assert torch.allclose((got[0][0] * go).sum(), value, atol=1e-10)


def test_plain_norm_agrees_with_autograd():
    g = torch.Generator().manual_seed(1)
    x, gy, gs = (torch.randn(5, 12, generator=g) for _ in range(3))
    w = torch.randn(12, generator=g)
    _, _, (dx, _), (dw, _) = ref.add_rms_norm(x, None, w, 1e-3, gy, gs)
    a, b = x.double().requires_grad_(True), w.double().requires_grad_(True)
    y = a * torch.rsqrt(a.square().mean(1, keepdim=True) + 1e-3) * b
    want = torch.autograd.grad((y * gy).sum() + (a * gs).sum(), (a, b))
    assert torch.allclose(dx, want[0], atol=1e-12) and torch.allclose(dw, want[1], atol=1e-12)


def test_a_mistake_is_caught():
    """The bounds are tight enough to tell a wrong scale, a key too many and a gradient without its second term."""
    g = torch.Generator().manual_seed(2)
    q, go = (torch.randn(1, 20, 2, 16, generator=g).half() for _ in range(2))
    k, v = (torch.randn(1, 50, 2, 16, generator=g).half() for _ in range(2))
    lengths = torch.tensor([49])
    want = ref.attention(q, k, v, None, lengths, None, go)
    for wrong in (ref.attention(q, k, v, None, None, None, go), ref.attention(q, k, v, None, lengths, 0.2525, go)):
        for (w, bound), (t, _) in zip(want, wrong):
            with pytest.raises(AssertionError):
                ref.check(t, w, bound, "planted")


def test_modules_keep_their_8_bit_weights():
    import medvision_amd.ops as ops
    m = ops.BlockScaledLinear(200, 130, dtype=torch.float16)
    assert m.weight.shape == (130, 256) and m.weight_scales.shape == (2, 2)
    m = m.half()
    assert m.weight.dtype == torch.float8_e4m3fn and m.weight_scales.dtype == torch.float32 and m.bias.dtype == torch.float16
    assert set(m.state_dict()) == {"weight", "weight_scales", "bias"}
    with pytest.raises(RuntimeError, match="rows of 100, expected 200"):
        m(torch.zeros(3, 100))
    assert "BlockScaledLinear(200, 130" in repr(m) and "AddRMSNorm(8" in repr(ops.AddRMSNorm(8))


@pytest.mark.parametrize("dtype,sizes,forward,queries,keys", [
    # (batch, queries, keys, heads, key_heads, channels), splits of the forward pass, of dq, and of dk and dv
    ("MV_F16", (1, 1, 1000, 64, 1, 32), 2, 2, 1), ("MV_F16", (1, 10, 200, 16, 4, 32), 1, 1, 1), ("MV_F32", (1, 2, 1000, 64, 2, 64), 16, 16, 1),
    ("MV_BF16", (2, 7, 500, 64, 1, 128), 1, 1, 1), ("MV_F32", (1, 4, 20, 32, 1, 32), 1, 1, 1), ("MV_F32", (1, 1, 100, 1, 1, 32), 1, 1, 1),
    ("MV_F16", (1, 600, 64, 4, 2, 64), 1, 1, 3), ("MV_F32", (1, 100, 1000, 2, 2, 64), 16, 16, 2)])
def test_no_more_splits_than_there_is_work_for(dtype, sizes, forward, queries, keys):
    """A split has 512 keys or rows (float32: 64) at least, and a tile of them.  Rows of heads that share keys follow each other:
    few queries of many heads are one tile, with nothing to split.  Read from the workspaces, whose parts are the splits'."""
    from medvision_amd import _lib
    lib, kind = _lib.load(), getattr(_lib, dtype)
    B, Lq, Lk, H, Hk, D = sizes
    shape = ctypes.byref(_shape(*sizes))
    assert lib.mv_cross_attention_forward_workspace_bytes(shape, kind) == (4 * forward * B * Lq * H * (D + 2) if forward > 1 else 0)
    parts = max(queries * B * Lq * H * D if queries > 1 else 0, 2 * keys * B * Lk * Hk * D if keys > 1 else 0)
    assert lib.mv_cross_attention_backward_workspace_bytes(shape, kind) == 4 * (B * Lq * H + parts)
