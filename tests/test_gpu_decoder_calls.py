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


# ---- gradients that are wanted -------------------------------------------------------------------------------
SUBSETS = [(True, False, False), (False, True, False), (False, False, True), (True, True, False), (True, False, True), (False, True, True)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("sizes", [(2, 3, 700, 4, 2, 32), (1, 300, 20, 2, 1, 64), (2, 150, 260, 2, 2, 96)])
def test_attention_gradients_of_some_inputs(dtype, sizes):
    """The same bits as all three together, in both forms of the node."""
    from medvision_amd.ops.cross_attention import CrossAttentionFunction

    class Python(CrossAttentionFunction):
        @staticmethod
        def backward(ctx, grad):
            return CrossAttentionFunction.backward(ctx, grad)

    B, Lq, Lk, H, Hk, D = sizes
    tensors = rand(1, B, Lq, H, D, dtype=dtype), rand(2, B, Lk, Hk, D, dtype=dtype), rand(3, B, Lk, Hk, D, dtype=dtype)
    go = rand(4, B, Lq, H, D, dtype=dtype)
    lengths = torch.full((B,), Lk - 3, device=DEV)

    def grads(function, wanted):
        ins = [t.clone().requires_grad_(w) for t, w in zip(tensors, wanted)]
        function.apply(*ins, None, lengths, None).backward(go)
        return [t.grad for t in ins]

    want = grads(CrossAttentionFunction, (True, True, True))
    for function in (CrossAttentionFunction, Python):
        for wanted in SUBSETS:
            for got, all_of_them, w in zip(grads(function, wanted), want, wanted):
                assert torch.equal(got, all_of_them) if w else got is None


def test_gradients_that_nobody_wants_take_no_memory():
    """Queries over a frozen encoder: no gradients of the keys and values, and no parts of them, are formed."""
    import medvision_amd.ops as ops
    q, k = rand(1, 1, 2000, 8, 64, dtype=torch.float16).requires_grad_(True), rand(2, 1, 100000, 8, 64, dtype=torch.float16)
    out = ops.cross_attention(q, k, k)
    go = torch.ones_like(out)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out.backward(go)
    assert torch.cuda.max_memory_allocated() - before < k.numel() * k.element_size()


def test_entry_points_without_some_gradients():
    """Null pointers for gradients that are not wanted; what is wanted is the same."""
    from medvision_amd import _lib
    lib = _lib.load()
    B, Lq, Lk, H, D = 1, 9, 50, 2, 32
    q, go = rand(1, B, Lq, H, D), rand(2, B, Lq, H, D)
    k, v = rand(3, B, Lk, H, D), rand(4, B, Lk, H, D)
    s = _lib.AttentionShape(B, Lq, Lk, H, H, D)
    for strides, t in ((s.q_strides, q), (s.k_strides, k), (s.v_strides, v)):
        for i in range(3):
            strides[i] = t.stride(i)
    from medvision_amd._lib import native
    out, lse, _ = native.cross_attention_forward(q, k, v, None, None, 0.25)
    p = lambda t: None if t is None else t.data_ptr()   # noqa: E731

    def call(gq, gk, gv):
        bytes_ = lib.mv_cross_attention_backward_workspace_bytes(ctypes.byref(s), _lib.MV_F32)
        ws = torch.empty(bytes_, dtype=torch.uint8, device=DEV)
        status = lib.mv_cross_attention_backward(p(q), p(k), p(v), None, None, p(out), None, p(lse), p(go), p(gq), p(gk), p(gv), ctypes.byref(s),
                                                 0.25, _lib.MV_F32, p(ws), bytes_, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return status

    new = lambda: [torch.full_like(t, 7.0) for t in (q, k, v)]   # noqa: E731
    full, only_q, only_kv = new(), new(), new()
    assert call(*full) == 0
    assert call(only_q[0], None, None) == 0 and torch.equal(only_q[0], full[0])
    assert call(None, *only_kv[1:]) == 0 and torch.equal(only_kv[1], full[1]) and torch.equal(only_kv[2], full[2])
    assert call(None, None, None) == 0
    assert call(full[0], full[1], None) == 1 and b"pair" in lib.mv_last_error()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,columns", [(70, 40), (33, 1000), (5, 20000)])
@pytest.mark.parametrize("added", [True, False])
def test_norm_gradients_of_some_inputs(dtype, rows, columns, added):
    from medvision_amd.ops.rms_norm import AddRMSNormFunction

    class Python(AddRMSNormFunction):
        @staticmethod
        def backward(ctx, grad_y, grad_sum):
            return AddRMSNormFunction.backward(ctx, grad_y, grad_sum)

    tensors = rand(1, rows, columns, dtype=dtype), rand(2, rows, columns, dtype=dtype) if added else None, rand(3, columns, dtype=dtype)
    gy, gs = rand(4, rows, columns, dtype=dtype), rand(5, rows, columns, dtype=dtype)

    def grads(function, wanted):
        ins = [None if t is None else t.clone().requires_grad_(w) for t, w in zip(tensors, wanted)]
        y, h = function.apply(*ins, 1e-6)
        torch.autograd.backward((y, h) if added else (y,), (gy, gs) if added else (gy,))
        return [None if t is None else t.grad for t in ins]

    want = grads(AddRMSNormFunction, (True, True, True))
    alone = grads(AddRMSNormFunction, (False, False, True))
    assert alone[0] is None and alone[1] is None and torch.equal(alone[2], want[2])
    for function in (AddRMSNormFunction, Python):
        for wanted in SUBSETS:
            if not any(w for w, t in zip(wanted, tensors) if t is not None):
                continue
            for got, all_of_them, w, t in zip(grads(function, wanted), want, wanted, tensors):
                assert torch.equal(got, all_of_them) if w and t is not None else got is None


def test_norm_entry_point_without_some_gradients():
    from medvision_amd import _lib
    lib = _lib.load()
    p = lambda t: None if t is None else t.data_ptr()   # noqa: E731
    for rows, columns in ((30, 200), (3, 20000)):
        x, w, gy = rand(5, rows, columns), rand(6, columns), rand(7, rows, columns)
        bytes_ = lib.mv_add_rms_norm_backward_workspace_bytes(rows, columns)
        ws = torch.empty(bytes_, dtype=torch.uint8, device=DEV)

        def call(gx, gw, given=True):
            return lib.mv_add_rms_norm_backward(p(x), p(w), p(gy), None, p(gx), p(gw), rows, columns, 1e-6, _lib.MV_F32, _lib.MV_F32,
                                                p(ws) if given else None, bytes_ if given else 0, torch.cuda.current_stream().cuda_stream)

        gx, gw, gx1, gw1 = (torch.full_like(t, 7.0) for t in (x, w, x, w))
        assert call(gx, gw) == 0 and call(gx1, None, given=False) == 0 and call(None, gw1) == 0 and call(None, None, given=False) == 0
        assert torch.equal(gx, gx1) and torch.equal(gw, gw1)
        assert call(None, gw1, given=False) == 1 and b"workspace" in lib.mv_last_error()


# ---- subclasses, traces, transforms, hooks -----------------------------------------------------------------------
def functions():
    from medvision_amd.ops.cross_attention import CrossAttentionFunction
    from medvision_amd.ops.rms_norm import AddRMSNormFunction
    q, k, v = rand(1, 2, 7, 4, 24), rand(2, 2, 40, 2, 24), rand(3, 2, 40, 2, 24)
    mask = torch.rand(2, 40, generator=torch.Generator().manual_seed(4)).to(DEV) < 0.6
    lengths = torch.tensor([40, 13], device=DEV)
    x, r, w = rand(5, 6, 100), rand(6, 6, 100), rand(7, 100)
    return [(CrossAttentionFunction, lambda f, *t: f.apply(*t, None, None, None), [q, k, v]),
            (CrossAttentionFunction, lambda f, *t: f.apply(*t, mask, lengths, 0.3), [q, k, v]),
            (AddRMSNormFunction, lambda f, *t: f.apply(*t, 1e-6), [x, r, w]),
            (AddRMSNormFunction, lambda f, x, w: f.apply(x, None, w, 1e-6), [x, w])]


def as_tuple(t):
    return t if isinstance(t, tuple) else (t,)


@pytest.mark.parametrize("index", range(4))
def test_the_python_form_of_the_nodes_agrees(index):
    """``forward`` and ``backward`` as a subclass of the function runs them, against the native node: the same bits."""
    base, run, leaves = functions()[index]

    class Counted(base):
        calls = 0

        @staticmethod
        def backward(ctx, *grads):
            Counted.calls += 1
            return base.backward(ctx, *grads)

    results = []
    for function in (base, Counted):
        ins = [t.clone().requires_grad_() for t in leaves]
        out = as_tuple(run(function, *ins))
        # (without a residual the native node hands the input through, and its gradient does not pass the node)
        out = out[:1] if len(leaves) == 2 else out
        results.append([*out, *torch.autograd.grad(out, ins, [torch.ones_like(o) for o in out])])
    assert Counted.calls == 1
    for got, want in zip(*results):
        assert torch.equal(got, want)


@pytest.mark.parametrize("index", range(4))
def test_traced_calls_run_their_operator(index):
    function, run, leaves = functions()[index]
    with torch.no_grad():
        traced = torch.jit.trace(lambda *t: as_tuple(run(function, *t)), tuple(leaves))
        other = (leaves[0] * 2 + 1, *leaves[1:])
        for a, b in zip(traced(*other), as_tuple(run(function, *other))):
            torch.testing.assert_close(a, b)
        assert not torch.equal(traced(*other)[0], traced(*leaves)[0])


@pytest.mark.parametrize("index", range(4))
def test_transforms_of_functions_are_refused(index):
    function, run, leaves = functions()[index]
    first = lambda t: as_tuple(run(function, t, *leaves[1:]))[0]   # noqa: E731
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(first, (leaves[0],), (torch.ones_like(leaves[0]),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(first)(leaves[0].unsqueeze(0))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: first(t).sum())(leaves[0])
    assert torch.isfinite(first(leaves[0])).all()


def test_8_bit_operators_refuse_transforms():
    import medvision_amd.ops as ops
    x, w = rand(1, 3, 256), rand(2, 256)
    q, s = ops.quantize_blocks(x)
    weight, scales = ops.quantize_blocks(rand(3, 40, 256), 128)
    for call, t in ((lambda t: ops.quantize_blocks(t)[1], x), (lambda t: ops.add_rms_norm_quantized(t, None, w)[1], x),
                    (lambda t: ops.block_linear(q, t, weight, scales), s)):
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t.unsqueeze(0))
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))


@pytest.mark.parametrize("index", range(4))
def test_hooks_see_the_gradients(index):
    function, run, leaves = functions()[index]
    ins = [t.clone().requires_grad_() for t in leaves]
    moved = [t * 1.0 for t in ins]
    seen = {}
    for i, t in enumerate(moved):
        t.retain_grad()
        t.register_hook(lambda g, i=i: seen.__setitem__(i, g.clone()))
    out = as_tuple(run(function, *moved))
    nodes = []
    out[0].grad_fn.register_hook(lambda inputs, outputs: nodes.append(inputs))
    out[0].register_hook(lambda g: 2 * g)
    go = torch.ones_like(out[0])
    out[0].backward(go)
    plain = [t.clone().requires_grad_() for t in leaves]
    want = torch.autograd.grad(as_tuple(run(function, *plain))[0], plain, 2 * go)
    assert len(nodes) == 1
    for i, w in enumerate(want):
        assert torch.equal(seen[i], w) and torch.equal(ins[i].grad, w) and torch.equal(moved[i].grad, w)
