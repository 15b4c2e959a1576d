"""Modules with tensors whose type is part of what they hold."""
from torch import nn


class KeepsTypes(nn.Module):
    """``.half()`` and its like leave the tensors named in ``kept`` as they are; moves between devices take them along."""
    kept = ()

    def _apply(self, fn, recurse=True):
        kept = {name: getattr(self, name) for name in self.kept}
        super()._apply(fn, recurse)
        for name, tensor in kept.items():
            now = getattr(self, name)
            if now.dtype != tensor.dtype:
                setattr(self, name, tensor.to(now.device))
        return self
