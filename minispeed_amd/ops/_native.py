"""The operators' native extension, ``minispeed_amd/_ops.so``.

The operators run only as the HIP kernels of ``libminispeed_ops.so``, which
the extension is linked to.  A missing or stale build raises
:class:`minispeed_amd._native.NativeLibraryError` at the first call; nothing
falls back to another implementation.
"""

from __future__ import annotations

import importlib

import torch  # noqa: F401  (its HIP runtime is loaded before the library's)

from .._native import NativeLibraryError

ABI_VERSION = 1
_module = None


def load():
    """The extension module, loaded once."""
    global _module
    if _module is None:
        try:
            module = importlib.import_module("minispeed_amd._ops")
        except ImportError as exc:
            raise NativeLibraryError(
                f"the operators' extension cannot be loaded ({exc}); build it with "
                "`python -m minispeed_amd.build` (hipcc --offload-arch=gfx950)"
            ) from exc
        if module.abi_version() != ABI_VERSION:
            raise NativeLibraryError(
                f"libminispeed_ops.so has ABI version {module.abi_version()}, expected "
                f"{ABI_VERSION}; rebuild it"
            )
        _module = module
    return _module


def __getattr__(name):
    """``_native.embedding`` etc.: the extension's functions, bound at first use."""
    if name.startswith("__"):
        raise AttributeError(name)
    value = getattr(load(), name)
    globals()[name] = value
    return value
