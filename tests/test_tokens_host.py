"""Host side of group norm with an activation, rotary positions and 4-bit products: refusals, workspaces, modules, and the 64-bit
forms that the GPU tests compare with."""
import ctypes

import pytest
import torch

import decoder_ref
import tokens_ref as ref


def test_cpu_tensors_are_refused():
    import medvision_amd.ops as ops
    x = torch.zeros(2, 3, 4, 16)
    with pytest.raises(RuntimeError, match="group_norm_act is not implemented on CPU"):
        ops.group_norm_act(x, 4)
    with pytest.raises(RuntimeError, match="rotary_positions is not implemented on CPU"):
        ops.rotary_positions(x, torch.zeros(3, 2), torch.zeros(2, 8))
    with pytest.raises(RuntimeError, match="quantize_groups is not implemented on CPU"):
        ops.quantize_groups(torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="group_linear is not implemented on CPU"):
        ops.group_linear(x.half(), torch.zeros(3, 64, dtype=torch.uint8), torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="activation 'tanh'"):
        ops.group_norm_act(x, 4, activation="tanh")


def test_group_norm_entry_points_refuse_on_the_host():
    from medvision_amd import _lib
    lib = _lib.load()

    def forward(batch=2, cells=3, channels=8, groups=2, activation=0, dtype=_lib.MV_F16, weight_dtype=_lib.MV_F16):
        return lib.mv_group_norm(*[None] * 5, batch, cells, channels, groups, 1e-5, activation, 0.01, dtype, weight_dtype, None, 0, None)

    def backward(batch=2, cells=3, channels=8, groups=2, activation=0, dtype=_lib.MV_F16, weight_dtype=_lib.MV_F16, wanted=None):
        return lib.mv_group_norm_backward(*[None] * 5, wanted, None, None, batch, cells, channels, groups, activation, 0.01, dtype, weight_dtype,
                                          None, 0, None)

    for call in (forward, backward):
        for wrong in (dict(batch=-1), dict(cells=-1), dict(cells=2 ** 37), dict(channels=0), dict(groups=0), dict(groups=3), dict(activation=5), dict(activation=-1),
                      dict(dtype=_lib.MV_F64), dict(weight_dtype=_lib.MV_BF16)):
            assert call(**wrong) == 1 and lib.mv_last_error()
        assert call(batch=0) == 0 and call(cells=0) == 0
    assert forward() == 1 and b"missing" in lib.mv_last_error()
    assert backward() == 0   # nothing is wanted
    assert backward(wanted=ctypes.c_void_p(16)) == 1 and b"missing" in lib.mv_last_error()
    p = ctypes.c_void_p(16)
    assert lib.mv_group_norm(p, None, None, p, p, 2, 3, 8, 2, 1e-5, 0, 0.0, _lib.MV_F16, _lib.MV_F16, None, 0, None) == 1
    assert b"workspace" in lib.mv_last_error()
    assert lib.mv_group_norm(p, None, None, p, p, 65536, 6000, 8, 2, 1e-5, 0, 0.0, _lib.MV_F16, _lib.MV_F16, p, 1 << 40, None) == 1
    assert b"a batch of 65536" in lib.mv_last_error()
    assert lib.mv_group_norm_backward(p, None, None, p, p, p, None, None, 65536, 6000, 8, 2, 0, 0.0, _lib.MV_F16, _lib.MV_F16, p, 1 << 40, None) == 1
    assert b"a batch of 65536" in lib.mv_last_error()
    assert lib.mv_group_norm_workspace_bytes(2, 3, 8, 2) > 0 and lib.mv_group_norm_backward_workspace_bytes(2, 3, 8, 2) > 0
    for wrong in ((0, 3, 8, 2), (2, 0, 8, 2), (2, 3, 8, 3), (2, 3, 0, 1), (2, -1, 8, 2)):
        assert lib.mv_group_norm_workspace_bytes(*wrong) == 0 and lib.mv_group_norm_backward_workspace_bytes(*wrong) == 0


def test_rotary_entry_point_refuses_on_the_host():
    from medvision_amd import _lib
    lib = _lib.load()

    def call(batch=1, rows=2, heads=3, dim=8, axes=2, pairs=4, dtype=_lib.MV_F16, place=_lib.MV_F32):
        s = _lib.RotaryShape(batch, rows, heads, dim, axes, pairs)
        return lib.mv_rotary_positions(*[None] * 4, ctypes.byref(s), 0, 0, dtype, place, None)

    for wrong in (dict(batch=-1), dict(dim=0), dict(dim=1025), dict(axes=0), dict(axes=9), dict(pairs=5), dict(pairs=-1), dict(pairs=2 ** 30 + 1), dict(dtype=_lib.MV_F64),
                  dict(place=_lib.MV_F16), dict(heads=2 ** 28, dim=512), dict(heads=2 ** 21 + 1, dim=512)):
        assert call(**wrong) == 1 and lib.mv_last_error()
    assert call() == 1 and b"missing" in lib.mv_last_error()
    assert call(rows=0) == 0 and call(heads=0) == 0 and call(batch=0) == 0
    assert lib.mv_rotary_positions(*[None] * 4, None, 0, 0, _lib.MV_F16, _lib.MV_F32, None) == 1


def test_group_linear_entry_points_refuse_on_the_host():
    from medvision_amd import _lib
    lib = _lib.load()
    for args in ((4, 8, 31, _lib.MV_F32), (4, 0, 32, _lib.MV_F32), (-1, 8, 32, _lib.MV_F32), (4, 8, 32, _lib.MV_F64), (4, 8, 32, _lib.MV_F16)):
        assert lib.mv_quantize_groups(None, None, None, *args, None) == 1 and lib.mv_last_error()
    assert lib.mv_quantize_groups(None, None, None, 0, 8, 32, _lib.MV_F32, None) == 0
    for args in ((4, 100, 8, 16, _lib.MV_F16), (4, 100, 8, 32, _lib.MV_F32), (4, 0, 8, 32, _lib.MV_F16), (-1, 100, 8, 32, _lib.MV_F16), (4, 100, 8, 32, _lib.MV_F16)):
        assert lib.mv_group_linear(*[None] * 5, *args, None, 0, None) == 1 and lib.mv_last_error()
    assert lib.mv_group_linear(*[None] * 5, 0, 100, 8, 32, _lib.MV_F16, None, 0, None) == 0
    assert lib.mv_group_linear(*[None] * 5, 4, 100, 0, 32, _lib.MV_F16, None, 0, None) == 0
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(17)
    assert lib.mv_group_linear(p, odd, p, None, p, 4, 100, 8, 32, _lib.MV_F16, None, 0, None) == 1 and b"aligned" in lib.mv_last_error()
    assert lib.mv_group_linear_workspace_bytes(0, 100, 8) == 0 and lib.mv_group_linear_workspace_bytes(4, 100, -8) == 0


@pytest.mark.parametrize("kind", [None, "relu", "leaky_relu", "silu", "gelu"])
def test_plain_group_norm_agrees_with_autograd_and_differences(kind):
    g = torch.Generator().manual_seed(0)
    x, go = (torch.randn(2, 5, 12, generator=g) for _ in range(2))
    w, b = torch.randn(12, generator=g), torch.randn(12, generator=g)
    got = ref.group_norm(x, 3, w, b, 1e-3, kind, 0.1, go)

    def value(x, w, b):
        y = torch.nn.functional.group_norm(x.transpose(1, 2), 3, w, b, 1e-3).transpose(1, 2)
        y = {None: lambda t: t, "relu": torch.relu, "leaky_relu": lambda t: torch.nn.functional.leaky_relu(t, 0.1), "silu": torch.nn.functional.silu,
             "gelu": torch.nn.functional.gelu}[kind](y)
        return (y * go.double()).sum()

    ins = [t.double().requires_grad_(True) for t in (x, w, b)]
    total = value(*ins)
    assert torch.allclose((got[0][0] * go).sum(), total, atol=1e-10)
    for (d, _), want in zip(got[1:], torch.autograd.grad(total, ins)):
        assert torch.allclose(d, want, atol=1e-10)
    directions = [torch.randn(t.shape, generator=g).double() for t in ins]
    with torch.no_grad():
        slope = decoder_ref.slope(value, ins, directions, 1e-6)
    assert torch.allclose(slope, sum((d * v).sum() for (d, _), v in zip(got[1:], directions)), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("neighbours", [False, True])
def test_plain_rotary_turns_and_turns_back(neighbours):
    g = torch.Generator().manual_seed(1)
    x, f = torch.randn(2, 4, 3, 13, generator=g), torch.rand(2, 6, generator=g)
    at = 10 * torch.rand(2, 4, 2, generator=g)
    y, _ = ref.rotary(x, at, f, neighbours)
    assert torch.allclose(ref.rotary(y, at, f, neighbours, back=True)[0], x.double(), atol=1e-12)
    assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1)) and torch.equal(y[..., 12], x[..., 12].double())
    go = torch.randn(x.shape, generator=g)
    a = x.double().requires_grad_(True)
    turned = lambda t: (ref.rotary(t, at, f, neighbours)[0] * go).sum()   # noqa: E731
    eye = torch.randn(x.shape, generator=g).double()
    ahead, behind = turned(a.detach() + 1e-4 * eye), turned(a.detach() - 1e-4 * eye)
    assert torch.allclose((ahead - behind) / 2e-4, (ref.rotary(go, at, f, neighbours, back=True)[0] * eye).sum(), atol=1e-7)


def test_frequencies_of_axes():
    import medvision_amd.ops as ops
    f = ops.axis_frequencies(32, 3, 100.0)
    assert f.shape == (3, 16) and f.dtype == torch.float64 and f[:, 15].abs().sum() == 0
    assert torch.allclose(f[1, 5:10], 100.0 ** (-torch.arange(5, dtype=torch.float64) / 5)) and f[1, :5].abs().sum() == 0 and f[1, 10:].abs().sum() == 0
    assert ops.axis_frequencies(9, 1).shape == (1, 4)
    for wrong in ((5, 3), (16, 0), (1, 1)):
        with pytest.raises(ValueError, match="axes"):
            ops.axis_frequencies(*wrong)


def test_a_mistake_is_caught():
    """The bounds are tight enough to tell a cell too few, another eps, a wrong axis, a code next to the right one."""
    g = torch.Generator().manual_seed(2)
    x, go = (torch.randn(2, 40, 16, generator=g).half() for _ in range(2))
    w, b = torch.randn(16, generator=g).half(), torch.randn(16, generator=g).half()
    want = ref.group_norm(x, 4, w, b, 1e-5, "silu", grad=go)
    short = [(torch.cat((t, t[:, -1:]), 1) if t.dim() == 3 else t, None) for t, _ in ref.group_norm(x[:, :39], 4, w, b, 1e-5, "silu", grad=go[:, :39])]
    for wrong in (short, ref.group_norm(x, 4, w, b, 1e-2, "silu", grad=go), ref.group_norm(x, 2, w, b, 1e-5, "silu", grad=go)):
        for (v, bound), (t, _) in zip(want[:3], wrong):
            with pytest.raises(AssertionError):
                decoder_ref.check(t, v, bound, "planted")
    heads, f, at = torch.randn(1, 5, 2, 8, generator=g).half(), torch.rand(2, 4, generator=g), torch.rand(5, 2, generator=g)
    v, bound = ref.rotary(heads, at, f, False)
    for wrong in (ref.rotary(heads, at.flip(1), f, False), ref.rotary(heads, at, f, True), ref.rotary(heads, at, f, False, back=True)):
        with pytest.raises(AssertionError):
            decoder_ref.check(wrong[0], v, bound, "planted")
    rows = torch.randn(3, 200, generator=g).half()
    codes, scales = ref.quantize_groups(torch.randn(5, 200, generator=g), 32)
    v, bound = ref.group_linear(rows, codes, scales, None)
    near = codes.clone()
    near[0, 7] ^= 1
    for wrong in (ref.group_linear(rows, near, scales, None), ref.group_linear(rows, codes, scales * 1.01, None)):
        with pytest.raises(AssertionError):
            decoder_ref.check(wrong[0], v, bound, "planted")


def test_codes_of_values():
    t = torch.tensor([0, .2, .25, .26, .74, .75, 1.25, 1.3, 1.75, 2.5, 2.6, 3.5, 3.4, 5, 5.1, 6, -.25, -.3, -5.0])
    assert ref.to_codes(t).tolist() == [0, 0, 0, 1, 1, 2, 2, 3, 4, 4, 5, 6, 5, 6, 7, 7, 8, 9, 14]
    w = torch.randn(3, 200, generator=torch.Generator().manual_seed(3))
    for group in (32, 64, 128):
        codes, scales = ref.quantize_groups(w, group)
        assert codes.shape == (3, 128) and scales.shape == (3, 256 // group)
        v = ref.group_values(codes, scales, 200)
        assert ((v - w).abs() <= (scales.double().repeat_interleave(group, 1)[:, :200]) * 1.0001).all()   # the widest step is 2


def test_modules():
    import medvision_amd.ops as ops
    with pytest.raises(ValueError, match="groups"):
        ops.GroupNormAct(3, 16)
    with pytest.raises(ValueError, match="groups"):
        ops.GroupNormAct(0, 16)
    m = ops.GroupNormAct(4, 16, activation="silu")
    assert set(m.state_dict()) == {"weight", "bias"} and "GroupNormAct(4, 16" in repr(m)
    m = ops.GroupScaledLinear(200, 130, group=64, dtype=torch.float16)
    assert m.weight.shape == (130, 128) and m.scales.shape == (130, 4) and "GroupScaledLinear(200, 130" in repr(m)
    for cast in (lambda t: t.half(), lambda t: t.double(), lambda t: t.to("cpu")):
        assert cast(m).weight.dtype == torch.uint8 and m.scales.dtype == torch.float32
    assert set(m.state_dict()) == {"weight", "scales", "bias"}
    with pytest.raises(RuntimeError, match="rows of 100, expected 200"):
        m(torch.zeros(3, 100))
    with pytest.raises(ValueError, match="groups of 16"):
        ops.GroupScaledLinear(200, 130, group=16)
    empty = ops.GroupScaledLinear(200, 130, device="meta").to_empty(device="cpu")
    empty.load_state_dict(ops.GroupScaledLinear(200, 130).state_dict())
    assert empty.scales.dtype == torch.float32 and (empty.scales == 1).all()
    r = ops.RotaryPositions(32, 3)
    was = r.frequencies.clone()
    for cast in (lambda t: t.half(), lambda t: t.float(), lambda t: t.to(torch.bfloat16)):
        assert cast(r).frequencies.dtype == torch.float64 and torch.equal(r.frequencies, was)
    assert "RotaryPositions((3, 16)" in repr(r)


def test_layer_with_axes_wants_positions():
    import medvision_amd.ops as ops
    x, tokens = torch.zeros(1, 2, 96), torch.zeros(1, 3, 96)
    layer, plain = ops.RegionDecoderLayer(96, 6, axes=3), ops.RegionDecoderLayer(96, 6)
    assert layer.place.frequencies.shape == (3, 8) and plain.place is None and "place.frequencies" not in plain.state_dict()
    assert set(plain.state_dict()) | {"place.frequencies"} == set(layer.state_dict())
    q = torch.zeros(1, 2, 6, 16)
    with pytest.raises(ValueError, match="region_positions are missing"):
        layer._placed(q, None, "region")
    with pytest.raises(ValueError, match="token_positions are given"):
        plain._placed(q, torch.zeros(2, 3), "token")
    with pytest.raises(ValueError, match="in 6 bits"):
        plain.for_inference(bits=6)
    with pytest.raises(ValueError, match="axes"):
        ops.RegionDecoderLayer(96, 24, axes=3)   # heads of four channels
    assert x.shape[0] == tokens.shape[0]
