"""Operators of region decoders on the GPU against their plain forms in 64 bits."""
import math

import pytest
import torch

import decoder_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


# ---- cross attention ------------------------------------------------------------------------------------
def attention_case(seed, dtype, B, Lq, Lk, H, Hk, D, kind, train=True):
    g = gen(seed)
    q, go = randn(g, B, Lq, H, D, dtype=dtype), randn(g, B, Lq, H, D, dtype=dtype)
    k, v = randn(g, B, Lk, Hk, D, dtype=dtype), randn(g, B, Lk, Hk, D, dtype=dtype)
    mask = lengths = None
    if kind in ("mask", "both"):
        mask = (torch.rand(B, Lk, generator=g) < 0.7).to(DEV)
    if kind in ("lengths", "both"):
        lengths = torch.randint(0, Lk + 1, (B,), generator=g, dtype=torch.int32).to(DEV)
        lengths[B // 2] = 0
    return q, k, v, go, mask, lengths


def run_attention(q, k, v, go, mask, lengths, scale=None):
    import medvision_amd.ops as ops
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = ops.cross_attention(q, k, v, mask, lengths, scale)
    return (out, *torch.autograd.grad(out, (q, k, v), go))


def compare_attention(got, q, k, v, go, mask, lengths, scale=None):
    want = ref.attention(q, k, v, mask, lengths, scale, go)
    for name, t, (w, bound) in zip(("output", "dq", "dk", "dv"), got, want):
        ref.check(t, w, bound, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [
    # B, Lq, Lk, H, Hk, D
    (1, 1, 1, 1, 1, 1), (2, 1, 343, 8, 8, 32), (1, 5, 64, 4, 1, 16), (2, 33, 65, 3, 3, 20), (1, 130, 200, 4, 2, 64),
    (3, 31, 127, 2, 1, 33), (1, 64, 63, 2, 2, 80), (2, 100, 129, 2, 1, 96), (1, 70, 300, 2, 2, 128), (1, 17, 40, 3, 1, 127),
    (1, 300, 7, 4, 2, 40), (2, 257, 513, 1, 1, 8)])
@pytest.mark.parametrize("kind", ["none", "both"])
def test_attention_and_its_gradients(dtype, sizes, kind):
    case = attention_case(7 * sizes[1] + sizes[2], dtype, *sizes, kind)
    compare_attention(run_attention(*case), *case)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [(1, 1, 9001, 4, 2, 64), (2, 3, 4097, 2, 2, 32), (1, 5000, 40, 2, 1, 32), (1, 90, 6000, 2, 1, 128),
                                   (2, 2500, 130, 2, 2, 16)])
def test_attention_split_over_a_long_side(dtype, sizes):
    case = attention_case(sum(sizes), dtype, *sizes, "lengths")
    compare_attention(run_attention(*case), *case)


@pytest.mark.parametrize("dtype", TYPES)
def test_inference_gives_what_training_gives(dtype):
    import medvision_amd.ops as ops
    q, k, v, go, mask, lengths = attention_case(3, dtype, 2, 70, 333, 4, 2, 64, "both")
    assert torch.equal(ops.cross_attention(q, k, v, mask, lengths), run_attention(q, k, v, go, mask, lengths)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_is_the_same_every_time(dtype):
    case = attention_case(5, dtype, 2, 200, 700, 4, 2, 32, "both")
    first = run_attention(*case)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run_attention(*case)))


@pytest.mark.parametrize("dtype", TYPES)
def test_what_masked_keys_hold_has_no_effect(dtype):
    q, k, v, go, mask, lengths = attention_case(11, dtype, 2, 40, 150, 2, 1, 32, "mask")
    lengths = torch.tensor([150, 77], dtype=torch.int32, device=DEV)
    clean = run_attention(q, k, v, go, mask, lengths)
    keep = ref.valid_keys(2, 150, mask, lengths).to(DEV)
    for bad in (math.nan, math.inf, -math.inf, torch.finfo(dtype).min):
        kk, vv = k.clone(), v.clone()
        kk[~keep] = bad
        vv[~keep] = bad
        dirty = run_attention(q, kk, vv, go, mask, lengths)
        for a, b in zip(clean, dirty):
            assert torch.equal(a, b)
    assert not clean[2][~keep].any() and not clean[3][~keep].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_without_keys(dtype):
    q, k, v, go, _, _ = attention_case(2, dtype, 2, 9, 70, 2, 2, 32, "none")
    mask = torch.zeros(2, 70, dtype=torch.bool, device=DEV)
    for t in run_attention(q, k, v, go, mask, None):
        assert not t.any() and torch.isfinite(t).all()
    mask[1, 69] = True
    case = (q, k, v, go, mask, None)
    got = run_attention(*case)
    compare_attention(got, *case)
    assert torch.equal(got[0][1], v[1, 69].expand(9, 2, 32))   # one key: its value


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_lengths_beyond_the_keys(dtype):
    import medvision_amd.ops as ops
    q, k, v, *_ = attention_case(4, dtype, 3, 5, 20, 2, 2, 16, "none")
    whole, none = ops.cross_attention(q, k, v), torch.zeros_like(q)
    for kind in (torch.int32, torch.int64):
        lengths = torch.tensor([100, -3, 2 ** 31 - 1], dtype=kind, device=DEV)
        got = ops.cross_attention(q, k, v, key_lengths=lengths)
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], none[1]) and torch.equal(got[2], whole[2])
    got = ops.cross_attention(q, k, v, key_lengths=torch.tensor([2 ** 40, -2 ** 40, 20], device=DEV))
    assert torch.equal(got[0], whole[0]) and not got[1].any() and torch.equal(got[2], whole[2])


def test_attention_of_nothing():
    import medvision_amd.ops as ops
    q = torch.randn(2, 3, 4, 16, device=DEV, requires_grad=True)
    k = torch.randn(2, 0, 2, 16, device=DEV, requires_grad=True)
    out = ops.cross_attention(q, k, k)
    gq, gk = torch.autograd.grad(out.sum(), (q, k))
    assert not out.any() and not gq.any() and gk.shape == k.shape
    q0 = torch.randn(2, 0, 4, 16, device=DEV, requires_grad=True)
    k = torch.randn(2, 5, 2, 16, device=DEV, requires_grad=True)
    out = ops.cross_attention(q0, k, k)
    gq, gk = torch.autograd.grad(out.sum(), (q0, k))
    assert out.shape == q0.shape and gq.shape == q0.shape and not gk.any()
    assert ops.cross_attention(q0[:0], k[:0], k[:0]).numel() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_every_kind(dtype):
    """Projections of one matrix, heads before lengths, channels-first maps, rows that start anywhere, expanded tensors."""
    g = gen(9)
    B, Lq, Lk, H, D = 2, 37, 75, 2, 24
    kv = randn(g, B, Lk, 2, H, D, dtype=dtype)
    q_heads = randn(g, B, H, Lq, D, dtype=dtype).transpose(1, 2)
    go = randn(g, B, Lq, H, D, dtype=dtype)
    maps = randn(g, B, H * D, Lk, dtype=dtype)
    first = maps.reshape(B, H, D, Lk).permute(0, 3, 1, 2)
    shifted = randn(g, B, Lk, H, D + 3, dtype=dtype)[..., 1:D + 1]
    shared = randn(g, 1, Lk, 1, D, dtype=dtype).expand(B, Lk, H, D)
    mask = (torch.rand(Lk, B, generator=g) < 0.5).to(DEV).t()
    for k, v in ((kv[:, :, 0], kv[:, :, 1]), (first, shifted), (shared, kv[:, :, 1]), (shifted, shared)):
        case = (q_heads, k, v, go, mask, None)
        compare_attention(run_attention(*case), *case)


def test_gradient_of_shared_projection_reaches_it():
    import medvision_amd.ops as ops
    g = gen(10)
    q = randn(g, 2, 30, 4, 32)
    kv = randn(g, 2, 50, 2, 2, 32).requires_grad_(True)
    go = randn(g, 2, 30, 4, 32)
    (ops.cross_attention(q, kv[:, :, 0], kv[:, :, 1]) * go).sum().backward()
    want = ref.attention(q, kv[:, :, 0], kv[:, :, 1], grad=go)
    ref.check(kv.grad[:, :, 0], *want[2], "dk")
    ref.check(kv.grad[:, :, 1], *want[3], "dv")


def test_attention_gradient_by_differences():
    g = gen(21)
    q, k, v, go, mask, lengths = attention_case(21, torch.float32, 2, 19, 45, 4, 2, 24, "mask")
    got = run_attention(q, k, v, go, mask, lengths, 0.3)
    want = ref.attention(q, k, v, mask, lengths, 0.3, go)
    keep = ref.valid_keys(2, 45, mask, lengths)
    tensors = [t.double().cpu() for t in (q, k, v)]
    for which in range(3):
        dirs = [torch.randn(t.shape, generator=g).double() if i == which else torch.zeros_like(t) for i, t in enumerate(tensors)]
        by_steps = ref.slope(lambda *t: ref.attention_value(*t, go.double().cpu(), keep, 0.3), tensors, dirs)
        by_kernel = (got[1 + which].double().cpu() * dirs[which]).sum()
        # the kernel's bound, and the third derivative times step^2
        room = (want[1 + which][1] * dirs[which].abs()).sum() + 1e-6 * by_steps.abs() + 1e-5
        assert (by_kernel - by_steps).abs() <= room


@pytest.mark.parametrize("dtype", TYPES)
def test_large_and_small_scores(dtype):
    """Scores far apart (one key takes all) and equal scores; gradients far below and above one."""
    g = gen(30)
    q, k, v, go, _, _ = attention_case(31, dtype, 1, 40, 100, 2, 2, 32, "none")
    for factor in (0.0, 12.0):
        case = (q * factor, k, v, go, None, None)
        compare_attention(run_attention(*case), *case)
    for factor in (2.0 ** -9, 2.0 ** 7):
        case = (q, k, v, go * factor, None, None)
        compare_attention(run_attention(*case), *case)


def test_attention_on_another_stream_and_in_a_graph():
    import medvision_amd.ops as ops
    q, k, v, go, mask, lengths = attention_case(12, torch.float16, 2, 3, 2500, 4, 2, 32, "both")
    want = ops.cross_attention(q, k, v, mask, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.cross_attention(q, k, v, mask, lengths)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.cross_attention(q, k, v, mask, lengths)
    for seed in range(3):
        q.copy_(randn(gen(seed), *q.shape, dtype=q.dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.cross_attention(q, k, v, mask, lengths))


def test_attention_refusals():
    import medvision_amd.ops as ops
    t = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device=DEV)   # noqa: E731
    q, k = t(2, 3, 4, 32), t(2, 5, 2, 32)
    refused = [
        ((q, k, t(2, 6, 2, 32)), "value"), ((q, t(1, 5, 2, 32), t(1, 5, 2, 32)), "batch"), ((q, t(2, 5, 3, 32), t(2, 5, 3, 32)), "heads"),
        ((q, t(2, 5, 2, 16), t(2, 5, 2, 16)), "channels"), ((t(2, 3, 4, 129), t(2, 5, 2, 129), t(2, 5, 2, 129)), "1 to 128"),
        ((q, k.float(), k.float()), "one dtype"), ((q.double(), k.double(), k.double()), "float32, float16 or bfloat16"),
        ((q[0], k[0], k[0]), "batch, length, heads, channels"), ((q, k, k, t(2, 5)), "bool"), ((q, k, k, t(2, 6).bool()), "key_mask has shape"),
        ((q, k, k, None, t(2)), "whole numbers"), ((q, k, k, None, t(3).int()), "key_lengths has shape"),
        ((q, k.cpu(), k.cpu()), "key is on cpu"), ((q, k, k, t(2, 5).bool().cpu()), "key_mask is on cpu")]
    for args, text in refused:
        with pytest.raises(RuntimeError, match=text):
            ops.cross_attention(*args)
    x = q.float().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.cross_attention(x, k.float(), k.float()).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q.float(), q.float())
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.cross_attention(dual, k.float(), k.float())


# ---- RMS norm -----------------------------------------------------------------------------------------------
NORM_SIZES = [(1, 1), (3, 8), (5, 100), (2, 128), (7, 129), (130, 256), (9, 1000), (4, 1003), (33, 2048), (3, 2056), (2, 8192), (2, 8200),
              (1, 20011), (700, 40), (2100, 96), (513, 384)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", NORM_SIZES)
@pytest.mark.parametrize("added,wide", [(True, False), (False, True)])
def test_norm_and_its_gradients(dtype, rows, columns, added, wide):
    import medvision_amd.ops as ops
    g = gen(rows + columns)
    x, gy, gs = (randn(g, rows, columns, dtype=dtype) for _ in range(3))
    r = randn(g, rows, columns, dtype=dtype) if added else None
    w = randn(g, columns, dtype=torch.float32 if wide else dtype)
    ins = [t.detach().requires_grad_(True) for t in (x, r, w) if t is not None]
    y, h = ops.add_rms_norm(ins[0], ins[1] if added else None, ins[-1], eps=1e-5)
    grads = torch.autograd.grad((y, h) if added else (y,), ins, (gy, gs) if added else (gy,))
    want = ref.add_rms_norm(x, r, w, 1e-5, gy, gs if added else None)
    ref.check(y, *want[0], "y")
    ref.check(h, *want[1], "sum")
    ref.check(grads[0], *want[2], "dx")
    if added:
        assert torch.equal(grads[0], grads[1])
    assert grads[-1].dtype == w.dtype
    ref.check(grads[-1], *want[3], "dweight")
    with torch.no_grad():
        y2, h2 = ops.add_rms_norm(x, r, w, eps=1e-5)
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_norm_gradients_that_come_alone():
    import medvision_amd.ops as ops
    g = gen(77)
    x, r = (randn(g, 2, 5, 96).requires_grad_(True) for _ in range(2))
    w = randn(g, 96).requires_grad_(True)
    y, h = ops.add_rms_norm(x, r, w)
    gx, gr, gw = torch.autograd.grad(h.sum(), (x, r, w), retain_graph=True, allow_unused=True)
    assert torch.equal(gx, torch.ones_like(x)) and torch.equal(gr, gx) and not gw.any()
    gy = randn(g, 2, 5, 96)
    want = ref.add_rms_norm(x, r, w, 1e-6, gy)
    gx, _, gw = torch.autograd.grad(y, (x, r, w), gy)
    ref.check(gx, *want[2], "dx")
    ref.check(gw, *want[3], "dweight")


def test_norm_gradient_by_differences():
    import medvision_amd.ops as ops
    g = gen(78)
    x, gy, gs = (randn(g, 6, 70) for _ in range(3))
    w = randn(g, 70)
    ins = [t.detach().requires_grad_(True) for t in (x, torch.zeros_like(x), w)]
    out = ops.add_rms_norm(*ins, eps=1e-3)
    got = torch.autograd.grad(out, ins, (gy, gs))
    a, b = gy.double().cpu(), gs.double().cpu()
    f = lambda x, w: (x * torch.rsqrt(x.square().mean(1, keepdim=True) + 1e-3) * w * a + x * b).sum()   # noqa: E731
    want = ref.add_rms_norm(x, None, w, 1e-3, gy, gs)
    for i, (t, bound) in enumerate(((got[0], want[2][1]), (got[2], want[3][1]))):
        dirs = [torch.randn(s.shape, generator=g).double() if j == i else torch.zeros(s.shape).double() for j, s in enumerate((x, w))]
        steps = ref.slope(f, (x.double().cpu(), w.double().cpu()), dirs)
        assert ((t.double().cpu() * dirs[i]).sum() - steps).abs() <= (bound * dirs[i].abs()).sum() + 1e-6 * steps.abs() + 1e-5


def test_norm_of_zeros_infinities_and_views():
    import medvision_amd.ops as ops
    w = torch.ones(64, device=DEV)
    x = torch.zeros(4, 64, device=DEV)
    x[1] = math.inf
    x[2, 5] = math.nan
    x[3] = 1e-30
    y, h = ops.add_rms_norm(x, None, w, eps=1e-6)
    assert h is x and not y[0].any() and y[1].isnan().all() and y[2].isnan().all() and torch.isfinite(y[3]).all()
    assert ops.add_rms_norm(x[:0], x[:0], w)[0].shape == (0, 64)
    big = randn(gen(1), 6, 5, 64).transpose(0, 1)
    want = ref.add_rms_norm(big, big, w, 1e-6)
    y, h = ops.add_rms_norm(big, big, w)
    ref.check(y, *want[0], "y")
    ref.check(h, *want[1], "sum")
    xg = x[:0].clone().requires_grad_(True)
    wg = w.clone().requires_grad_(True)
    gw = torch.autograd.grad(ops.add_rms_norm(xg, None, wg)[0].sum(), (xg, wg))[1]
    assert not gw.any()


# ---- 8-bit blocks ---------------------------------------------------------------------------------------------
def same_blocks(got, want, share=2e-3):
    """The same scales up to their last bits, the same 8-bit values but where those bits move a value over a rounding's edge."""
    (q, s), (wq, ws) = got, want
    assert q.dtype == torch.float8_e4m3fn and q.shape == wq.shape and s.shape == ws.shape
    assert ((s.cpu() - ws.cpu()).abs() <= 2.0 ** -22 * ws.cpu().abs()).all()
    a, b = q.cpu().float(), wq.cpu().float()
    assert ((a - b).abs() <= 2.0 ** -3 * b.abs() + 2.0 ** -9).all()
    assert (a != b).float().mean() <= share


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (3, 128), (130, 200), (5, 1003), (257, 640)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_blocks(dtype, rows, columns, block_rows):
    import medvision_amd.ops as ops
    x = randn(gen(rows), rows, columns, dtype=dtype)
    q, s = ops.quantize_blocks(x, block_rows)
    wq, ws = ref.blocks(x.cpu(), block_rows)
    assert torch.equal(s.cpu(), ws)
    assert torch.equal(q.cpu().view(torch.uint8), wq.view(torch.uint8))


def test_quantize_blocks_of_odd_values():
    import medvision_amd.ops as ops
    x = torch.zeros(7, 256)
    x[1, 3] = math.nan
    x[2, 200] = -math.inf
    x[3] = 1e-44
    x[4, :128] = torch.linspace(-3e38, 3e38, 128)
    x[5, 0], x[5, 1] = 448.0, 0.001
    x[6, 255] = -1.0
    q, s = (t.cpu() for t in ops.quantize_blocks(x.to(DEV)))
    wq, ws = ref.blocks(x, 1)
    assert torch.equal(s.nan_to_num(7.0, posinf=9.0), ws.nan_to_num(7.0, posinf=9.0))
    v, wv = q.float() * s.repeat_interleave(128, 1), wq.float() * ws.repeat_interleave(128, 1)
    assert v[1, :128].isnan().all() and not v[1, 128:].any() and v[2, 128:].isnan().all() and not v[2, :128].any()
    assert torch.equal(v[3:].nan_to_num(), wv[3:].nan_to_num())
    q3, s3 = ops.quantize_blocks(torch.randn(2, 3, 130, device=DEV))
    assert q3.shape == (2, 3, 256) and s3.shape == (2, 3, 2) and not q3.float()[..., 130:].any()
    q0, s0 = ops.quantize_blocks(torch.zeros(0, 130, device=DEV))
    assert q0.shape == (0, 256) and s0.shape == (0, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1024), (3, 8), (50, 100), (9, 1003), (33, 2048), (2, 8192), (2, 8200), (600, 129)])
@pytest.mark.parametrize("added", [True, False])
def test_norm_in_8_bits(dtype, rows, columns, added):
    import medvision_amd.ops as ops
    g = gen(columns)
    x, r, w = randn(g, rows, columns, dtype=dtype), randn(g, rows, columns, dtype=dtype), randn(g, columns, dtype=dtype)
    q, s, h = ops.add_rms_norm_quantized(x, r if added else None, w, eps=1e-6)
    y, total = ref.add_rms_norm(x, r if added else None, w, 1e-6)
    ref.check(h, *total, "sum")
    same_blocks((q, s), ref.blocks(y[0].float(), 1))


# ---- products of 8-bit blocks ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,inputs,outputs", [
    (1, 128, 1), (1, 1024, 256), (3, 300, 17), (16, 5000, 130), (8, 20000, 64), (17, 128, 1000), (65, 1003, 129), (128, 384, 128),
    (200, 640, 333), (257, 256, 512), (300, 1152, 257), (1000, 896, 640), (129, 9000, 40)])
@pytest.mark.parametrize("bias", [True, False])
def test_block_linear(dtype, rows, inputs, outputs, bias):
    import medvision_amd.ops as ops
    g = gen(rows + inputs)
    x = randn(g, rows, inputs) * torch.exp(randn(g, rows, 1))
    w = randn(g, outputs, inputs) / math.sqrt(inputs) * torch.exp(randn(g, outputs, 1))
    b = randn(g, outputs, dtype=dtype) if bias else None
    q, s = ops.quantize_blocks(x)
    wq, ws = ops.quantize_blocks(w, 128)
    y = ops.block_linear(q, s, wq, ws, b, out_dtype=dtype)
    assert y.dtype == dtype
    ref.check(y, *ref.block_linear(q, s, wq, ws, b, dtype), "y")
    assert torch.equal(y, ops.block_linear(q, s, wq, ws, b, out_dtype=dtype))


def test_block_linear_keeps_what_is_not_finite_in_its_rows():
    import medvision_amd.ops as ops
    g = gen(3)
    for rows in (20, 300):
        x, w = randn(g, rows, 512), randn(g, 192, 512)
        x[7, 300] = math.inf
        y = ops.block_linear(*ops.quantize_blocks(x), *ops.quantize_blocks(w, 128))
        assert y[7].isnan().all() and torch.isfinite(y[:7]).all() and torch.isfinite(y[8:]).all()
    wq, ws = ops.quantize_blocks(w, 128)
    assert ops.block_linear(*ops.quantize_blocks(x[:0]), wq, ws).shape == (0, 192)
    q, s = ops.quantize_blocks(randn(g, 2, 3, 512))
    assert ops.block_linear(q, s, wq, ws).shape == (2, 3, 192)
    moved = torch.empty(3 * 512 + 1, dtype=torch.uint8, device=DEV)[1:].view(torch.float8_e4m3fn).view(3, 512)
    moved.copy_(q[0])
    assert torch.equal(ops.block_linear(moved, s[0], wq, ws), ops.block_linear(q, s, wq, ws)[0])


def test_block_refusals():
    import medvision_amd.ops as ops
    g = gen(4)
    q, s = ops.quantize_blocks(randn(g, 5, 256))
    w, ws = ops.quantize_blocks(randn(g, 130, 256), 128)
    b = torch.zeros(130, device=DEV)
    refused = [((q, s, w[:, :128], ws), "last dimensions"), ((q, s[:, :1], w, ws), "q_scales has shape"), ((q, s, w, ws[:1]), "weight_scales has shape"),
               ((q.float(), s, w, ws), "float8_e4m3fn"), ((q, s, w, ws, b[:5]), "bias has shape"), ((q, s.half(), w, ws), "float32"),
               ((q, s, w, ws, b, torch.float32), "out_dtype"), ((q[:, :100].contiguous(), s, w[:, :100].contiguous(), ws), "whole blocks"),
               ((q, s, w.cpu(), ws), "weight is on cpu")]
    for args, text in refused:
        with pytest.raises(RuntimeError, match=text):
            ops.block_linear(*args)
    x = torch.zeros(4, 64, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.quantize_blocks(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.add_rms_norm_quantized(x, None, torch.ones(64, device=DEV))
    x = x.detach()
    with pytest.raises(RuntimeError, match="1 or 128"):
        ops.quantize_blocks(x, 64)
    with pytest.raises(RuntimeError, match="those of a matrix"):
        ops.quantize_blocks(x[None], 128)
    one = torch.ones(64, device=DEV)
    for args, text in (((x, x[:2], one), "shape and dtype"), ((x, x.half(), one), "shape and dtype"), ((x, None, one[:3]), "weight has shape"),
                       ((x, None, one.half()), "weight has dtype"), ((x.double(), None, one.double()), "float32, float16 or bfloat16")):
        with pytest.raises(RuntimeError, match=text):
            ops.add_rms_norm(*args)


@pytest.mark.parametrize("rows,inputs,outputs", [(3300, 300, 3850), (3584, 128, 3848)])
def test_block_linear_on_large_tiles(rows, inputs, outputs):
    """More than 192 tiles of 256 x 256: whole ones and ragged ones, rows of results at any alignment."""
    import medvision_amd.ops as ops
    g = gen(rows)
    q, s = ops.quantize_blocks(randn(g, rows, inputs) * torch.exp(randn(g, rows, 1)))
    wq, ws = ops.quantize_blocks(randn(g, outputs, inputs) / math.sqrt(inputs), 128)
    b = randn(g, outputs, dtype=torch.float16)
    y = ops.block_linear(q, s, wq, ws, b, out_dtype=torch.float16)
    ref.check(y, *ref.block_linear(q, s, wq, ws, b, torch.float16), "y")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.25, 0.0, 3.0])
def test_attention_with_any_scale(dtype, scale):
    case = attention_case(17, dtype, 2, 45, 90, 3, 1, 48, "mask")
    compare_attention(run_attention(*case, scale), *case, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,key_heads", [(12, 2), (5, 1), (16, 2), (130, 1)])
def test_groups_of_heads_of_any_size(dtype, heads, key_heads):
    """Groups that divide a tile's rows and groups that do not, more queries than keys and the reverse."""
    for Lq, Lk in ((70, 20), (20, 70)):
        case = attention_case(heads + Lq, dtype, 1, Lq, Lk, heads, key_heads, 24, "both")
        compare_attention(run_attention(*case), *case)


# ---- offsets of more than 32 bits -----------------------------------------------------------------------------------
def far_apart(t, stride, start):
    """The values of ``t [1, rows, heads, channels]`` in memory where rows are ``stride`` elements apart."""
    storage = torch.empty(start + t.shape[1] * stride, dtype=t.dtype, device=t.device)
    view = storage.as_strided(t.shape, (storage.numel(), stride, t.shape[3], 1), start)
    view.copy_(t)
    return view


@pytest.mark.parametrize("sizes", [(3, 700, 4, 2, 64), (700, 700, 2, 2, 32), (700, 40, 2, 1, 128)])
def test_attention_on_rows_far_apart(sizes):
    """Rows 2^22 elements apart: the last ones are behind 2^31 elements.  The same bits as from dense copies."""
    Lq, Lk, H, Hk, D = sizes
    q, k, v, go, mask, lengths = attention_case(Lq, torch.float16, 1, Lq, Lk, H, Hk, D, "mask")
    near = run_attention(q, k, v, go, mask, lengths)
    far = run_attention(far_apart(q, 2 ** 22, 8), far_apart(k, 2 ** 22, 16), far_apart(v, 2 ** 22, 24), go, mask, lengths)
    for a, b in zip(near, far):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,columns", [(2 ** 18 + 40, 8192), (2 ** 28 + 40, 8)])
def test_norm_of_more_than_2_31_elements(rows, columns):
    """The last rows give what they give alone."""
    import medvision_amd.ops as ops
    g = gen(columns)
    x, r = (torch.empty(rows, columns, dtype=torch.float16, device=DEV) for _ in range(2))
    last = slice(rows - 100, rows)
    for t in (x, r):
        t[:-100] = 1
        t[last] = randn(g, 100, columns, dtype=torch.float16)
    w = randn(g, columns, dtype=torch.float16)
    gy = torch.ones_like(x)

    def grads(x, r, gy):
        x, r = x.detach().requires_grad_(True), r.detach().requires_grad_(True)
        y, h = ops.add_rms_norm(x, r, w)
        return (y, h, torch.autograd.grad((y, h), x, (gy, gy))[0])

    whole = [t[last].clone() for t in grads(x, r, gy)]
    for a, b in zip(whole, grads(x[last], r[last], gy[last])):
        assert torch.equal(a, b)
    if columns >= 128:
        del whole, gy
        whole = [t[last].clone() for t in ops.add_rms_norm_quantized(x, r, w)]
        for a, b in zip(whole, ops.add_rms_norm_quantized(x[last], r[last], w)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("rows,inputs,outputs", [(25000, 87808, 64), (2 ** 19 + 1000, 128, 4096)])
def test_block_linear_of_more_than_2_31_elements(rows, inputs, outputs):
    import medvision_amd.ops as ops
    g = gen(rows)
    x = torch.ones(rows, inputs, dtype=torch.float16, device=DEV)
    last = slice(rows - 70, rows)
    x[last] = randn(g, 70, inputs, dtype=torch.float16)
    q, s = ops.quantize_blocks(x)
    q1, s1 = ops.quantize_blocks(x[last])
    assert torch.equal(q[last].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[last], s1)
    wq, ws = ops.quantize_blocks(randn(g, outputs, inputs) / math.sqrt(inputs), 128)
    y = ops.block_linear(q, s, wq, ws, out_dtype=torch.float16)
    ref.check(y[last], *ref.block_linear(q1, s1, wq, ws, None, torch.float16), "y")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes", [(1, 17, 206, 4, 4, 80), (2, 300, 2, 8, 8, 32), (1, 3000, 14, 2, 1, 64), (1, 12, 5000, 4, 4, 32)])
def test_gradients_of_few_weights_are_off_by_little_more_than_their_rounding(dtype, sizes):
    """Weights rounded once would add an error as large as the result's own: a factor of the root of two."""
    q, k, v, go, mask, lengths = attention_case(sizes[1], dtype, *sizes, "none")
    got = run_attention(q, k, v, go, mask, lengths)
    for name, t, (w, _) in zip(("output", "dq", "dk", "dv"), got, ref.attention(q, k, v, mask, lengths, None, go)):
        w = w.double().to(t.device)
        assert (t.double() - w).norm() <= math.sqrt(2) * (w.to(dtype).double() - w).norm(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1100, 4100), (600, 8200), (300, 16384), (70, 16392)])
def test_norm_of_long_rows(dtype, rows, columns):
    """More rows than workgroups, on both sides of the longest row that is kept in registers; in 8 bits too."""
    import medvision_amd.ops as ops
    g = gen(columns)
    x, r, gy, gs = (randn(g, rows, columns, dtype=dtype) for _ in range(4))
    w = randn(g, columns, dtype=dtype)
    ins = [t.detach().requires_grad_(True) for t in (x, r, w)]
    y, h = ops.add_rms_norm(*ins, eps=1e-5)
    grads = torch.autograd.grad((y, h), ins, (gy, gs))
    want = ref.add_rms_norm(x, r, w, 1e-5, gy, gs)
    for name, t, (value, bound) in zip(("y", "sum", "dx", "dweight"), (y, h, grads[0], grads[2]), want):
        ref.check(t, value, bound, name)
    q, s, h2 = ops.add_rms_norm_quantized(x[:70], r[:70], w, eps=1e-5)
    assert torch.equal(h2, h[:70])
    same_blocks((q, s), ref.blocks(want[0][0][:70].float(), 1))
