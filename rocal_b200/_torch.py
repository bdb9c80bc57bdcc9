"""The compiled binding of the head operators to torch (csrc/torch/head.cpp), bound to the library this process has
loaded. There is no fallback: if the binding is missing, importing this module fails."""
import ctypes
import os

import torch  # noqa: F401  (the binding's symbols live in torch's libraries)

from ._lib import Rb200Error, lib

_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_head.so")
if not os.path.exists(_PATH):
    raise ImportError("rocal_b200: %s not found. Build it with `python -m rocal_b200.build` (needs nvcc, g++ and torch's headers)" % _PATH)

from . import build as _build  # noqa: E402

# The binding uses torch's C++ classes: another torch than the one that it was compiled against must not load it.
if os.path.exists(_build.HEAD_STAMP):
    with open(_build.HEAD_STAMP) as _f:
        _for = _f.readline().strip()
    if _for != _build.head_versions():
        raise ImportError("rocal_b200: %s was built for %s, this is %s. Build it anew with `python -m rocal_b200.build`" %
                          (_PATH, _for, _build.head_versions()))

from . import _head as head  # noqa: E402

# the order of struct Api in csrc/torch/head.cpp
_CALLS = ("linear_workspace_bytes", "linear", "linear_probe", "linear_backward_workspace_bytes", "linear_backward",
          "linear_ce_workspace_bytes", "linear_ce", "linear_ce_backward_workspace_bytes", "linear_ce_backward",
          "grad_clip_workspace_bytes", "grad_clip", "last_error")
head.bind([ctypes.cast(getattr(lib, "rb200k_" + name), ctypes.c_void_p).value for name in _CALLS], Rb200Error)
