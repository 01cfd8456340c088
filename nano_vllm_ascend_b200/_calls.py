"""The compiled binding (``csrc/fp4_calls.cpp``) for the wrappers of ``ops`` and ``ops_fp8``.

As in ``ops_fp4``: a wrapper asks the binding first, which makes the same checks
in a fraction of the time; what it does not take (it returns ``NOT_TAKEN`` and
has launched nothing) the wrapper checks again, calls or refuses. The binding is
loaded, and told the entry points' addresses, with the first call.
"""

from __future__ import annotations

import ctypes
import functools

from . import _lib

NOT_TAKEN = 1
_BOUND = ("nvk_fp8_append_workspace_size", "nvk_fp8_append", "nvk_fp8_read", "nvk_fp8_paged_decode",
          "nvk_fp8_paged_prefill", "nvk_rotary", "nvk_copy_blocks", "nvk_remap_blocks")


@functools.cache
def binding():
    """The binding; None where it is not built, or for another torch."""
    from . import ops_fp4

    calls = ops_fp4._binding()
    if calls is not None:
        lib = _lib.load()
        calls.bind_more(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in _BOUND))
    return calls


def _leave(*args) -> int:
    return NOT_TAKEN


def first(name: str, namespace: dict):
    """Stands for the binding's function ``name`` as ``namespace["_" + name]`` until its first call, which puts that
    in its place."""
    def call(*args):
        calls = binding()
        fn = _leave if calls is None else getattr(calls, name)
        if namespace.get(f"_{name}") is call:
            namespace[f"_{name}"] = fn
        return fn(*args)
    return call
