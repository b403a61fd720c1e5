"""The native library for operators that torch cannot look into."""
from __future__ import annotations

import torch

from .. import require_native


def native():
    """The library; refuses under ``torch.jit.trace``, which would record a call's results as constants."""
    if torch._C._get_tracing_state() is not None:
        raise RuntimeError("this operator cannot be traced: it is no operator of torch's")
    return require_native()
