"""The native library for operators that torch cannot look into."""
from __future__ import annotations

import torch

from .. import require_native


def native():
    """The library; refuses under ``torch.jit.trace``, which would record a call's results as constants."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("this operator cannot be traced: it is no operator of torch's")
    return require_native()


def on_kernels(x: torch.Tensor) -> bool:
    """Whether a call on ``x`` is the kernels'.

    Not under a mode that has to see the operators of torch that a call is made of (``make_fx``, which would record a result of the
    kernels as an empty tensor, flop counters, selective recomputation): the formulas in torch answer there.
    """
    key = torch._C.DispatchKey
    included = torch._C._dispatch_tls_is_dispatch_key_included
    return x.is_cuda and not (included(key.Python) or included(key.PreDispatch))
