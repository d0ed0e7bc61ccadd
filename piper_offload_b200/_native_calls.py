"""The compiled calls of the INT8 products, routing and the exchange (``csrc/expert_calls.cpp``)."""

from __future__ import annotations

import ctypes
from typing import Any

from . import _native_int8, _native_routing

_INT8 = ("piper_int8_linear_workspace", "piper_int8_grad_input_workspace", "piper_int8_linear", "piper_int8_grad_input", "piper_int8_last_error")
_ROUTING = ("piper_routing_workspace", "piper_routing_route", "piper_routing_route_grad", "piper_routing_dispatch", "piper_routing_combine",
            "piper_routing_combine_grad", "piper_routing_last_error")

_calls = None


def calls() -> Any:
    """The compiled calls, bound to the libraries' entry points. Loads all of them once."""
    global _calls
    if _calls is None:
        int8, routing = _native_int8.load(), _native_routing.load()
        try:
            from . import _expert_calls as module
        except ImportError as exc:
            raise RuntimeError("the compiled calls of the INT8 products and of routing are missing or do not fit this torch; build them "
                               "with `python -c 'import __graft_entry__ as g; g.build()'`.") from exc
        module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for lib, names in ((int8, _INT8), (routing, _ROUTING))
                      for name in names))
        _calls = module
    return _calls
