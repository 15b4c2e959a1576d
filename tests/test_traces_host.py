"""What ``torch.jit.trace`` records of the operators that have no gradient, and so no autograd node of their own."""
import ast
import importlib
import pathlib

import pytest
import torch

import medvision_amd.ops as ops

RESULTS = {"quantize_groups": 2, "quantize_blocks": 2, "add_rms_norm_quantized": 3}


class Stand:
    """In the place of the native functions: a trace sees of them, as of those, the allocation of their results."""

    def __getattr__(self, name):
        def call(*args):
            first = next(t for t in args if isinstance(t, torch.Tensor))
            out = []
            for n in range(RESULTS.get(name, 1)):
                out.append(torch.empty(first.shape))
                out[-1].numpy()[:] = first.detach().numpy() * (n + 2)
            return tuple(out) if len(out) > 1 else out[0]
        return call


x4, x5 = torch.ones(1, 2, 3, 4), torch.ones(1, 3, 3, 4, 5)
codes = torch.zeros(3, 64, dtype=torch.uint8)
CALLS = [("group_linear", "quantize_groups", lambda t: ops.quantize_groups(t, 64), torch.ones(3, 8)),
         ("group_linear", "group_linear", lambda t: ops.group_linear(t, codes, torch.ones(3, 4)), torch.ones(2, 8)),
         ("block_linear", "quantize_blocks", lambda t: ops.quantize_blocks(t), torch.ones(3, 8)),
         ("block_linear", "block_linear", lambda t: ops.block_linear(t, torch.ones(2, 1), torch.ones(3, 8), torch.ones(1, 1)), torch.ones(2, 8)),
         ("rms_norm", "add_rms_norm_quantized", lambda t: ops.add_rms_norm_quantized(t, None, torch.ones(8)), torch.ones(2, 8)),
         ("cuda_fun_tools", "affine", lambda t: ops.affine_2d(t, torch.ones(1, 6), (3, 4), 1.0), x4),
         ("cuda_fun_tools", "affine", lambda t: ops.affine_3d(t, torch.ones(1, 10), 3, 1.0), x5),
         ("cuda_fun_tools", "deform_warp", lambda t: ops.apply_offset_2d(t, x4), x4),
         ("cuda_fun_tools", "deform_warp", lambda t: ops.apply_offset_3d(t, x5), x5)]


def stand_in(monkeypatch, module):
    monkeypatch.setattr(importlib.import_module(f"medvision_amd.ops.{module}"), "native", Stand())


@pytest.mark.parametrize("module,name,call,x", CALLS)
def test_a_trace_runs_what_it_recorded(module, name, call, x, monkeypatch):
    stand_in(monkeypatch, module)
    traced = torch.jit.trace(call, (x,), check_trace=False)
    for scale in (3.0, -5.0):
        other = x * scale + torch.arange(x.numel()).view(x.shape)
        got, want = traced(other), call(other)
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a, b) and not a.requires_grad


@pytest.mark.parametrize("module,name,call,x", CALLS)
def test_a_trace_refuses_gradients_where_the_call_does(module, name, call, x, monkeypatch):
    stand_in(monkeypatch, module)
    leaf = x.clone().requires_grad_(True)
    if module == "cuda_fun_tools":   # results without a gradient
        assert not torch.jit.trace(call, (leaf,), check_trace=False)(leaf).requires_grad
        return
    with pytest.raises(RuntimeError, match=f"{name} has no gradient"):
        torch.jit.trace(call, (leaf,), check_trace=False)
    with torch.no_grad():
        torch.jit.trace(call, (leaf,), check_trace=False)


def test_every_call_of_a_native_function_has_a_node():
    for path in pathlib.Path(ops.__file__).parent.glob("*.py"):
        for node in ast.parse(path.read_text()).body:
            if isinstance(node, (ast.FunctionDef, ast.ClassDef)):
                calls = any(isinstance(n, ast.Attribute) and isinstance(n.value, ast.Name) and n.value.id == "native" for n in ast.walk(node))
                nodes = node.name.endswith("Function") or any(isinstance(n, ast.Name) and n.id.endswith("Function") for n in ast.walk(node))
                assert not calls or nodes, (path.name, node.name)
