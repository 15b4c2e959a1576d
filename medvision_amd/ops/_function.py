"""Base of the operators' autograd functions."""
import torch
from torch.autograd import Function

tracing = torch._C._get_tracing_state     # None outside of torch.jit.trace


class NativeFunction(Function):
    """A ``torch.autograd.Function`` whose ``apply`` runs the node of ``csrc/binding.cpp`` (``native``, the same arguments
    and results without the interpreter in the backward pass).  ``forward`` and ``backward`` do the same through ``_C``: for
    callers that call them, for a subclass that overrides one of them, and for ``torch.jit.trace``, which records a Python
    function as one node but of the native one nothing except the allocation of its result."""
    _direct = False

    def __init_subclass__(cls, **kwargs):
        super().__init_subclass__(**kwargs)
        own = vars(cls)
        cls._direct = 'native' in own or cls._direct and not any(
            name in own for name in ('forward', 'backward', 'setup_context', 'jvp', 'vmap'))

    @classmethod
    def apply(cls, *args, **kwargs):
        if cls._direct and tracing() is None:
            return cls.native(*args, **kwargs)
        return super().apply(*args, **kwargs)


class RecordedFunction(NativeFunction):
    """What a trace records of an operator without a gradient, which outside of traces is a call of the native function: of
    that ``torch.jit.trace`` would record nothing but the allocation of its result."""
    refuses = None   # the operator's name, where it refuses tensors that want a gradient (others give results without one)

    @classmethod
    def apply(cls, *args):
        if tracing() is None:
            return cls.native(*args)
        if cls.refuses and torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args):
            raise RuntimeError(f"{cls.refuses} has no gradient: call it under torch.no_grad()")
        with torch.no_grad():
            return super().apply(*args)

    @classmethod
    def forward(cls, ctx, *args):
        return cls.native(*args)
