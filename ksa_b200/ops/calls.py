"""Whether someone follows the operators' calls themselves."""
from __future__ import annotations

import functools

import torch

# private to PyTorch: without them every call counts as observed
_transforms_active = getattr(torch._C, "_are_functorch_transforms_active", lambda: True)
_forward_level = functools.partial(getattr, torch.autograd.forward_ad, "_current_level", 0)
_is_tracing, _is_compiling = torch.jit.is_tracing, torch.compiler.is_compiling


def observed() -> bool:
    """Whether someone follows the calls themselves: a ``torch.func`` transform, forward-mode differentiation, a trace, a compiler.
    They must meet the autograd function (its error, or its node in their graph) and not the bare kernel call, which would take
    the wrappers' memory for that of their tensors."""
    return _transforms_active() or _forward_level() >= 0 or _is_tracing() or _is_compiling()
