"""The compiled Python binding of the decoding operators (csrc/decode_binding.cpp).

``solution/_native.py`` calls the C ABI through ctypes; a decoding step's
launches are so short that the checks and the call itself would be most of
its time (15 to 30 us a call, here 7.5 to 10), so these operators are called from a small extension module instead.
It holds no kernels: it calls the entry points of the libb200tx that
``_native`` has loaded.  No fallback: where the module is missing every call
raises ``RuntimeError``.
"""

from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import threading
from types import ModuleType

from . import _native

_ENTRY_POINTS = (
    "b200tx_last_error",
    "b200tx_qk_norm_rope",
    "b200tx_kv8_append",
    "b200tx_kv8_gather",
    "b200tx_kv8_attention",
    "b200tx_linear_w4",
    "b200tx_low_rank_add",
    "b200tx_kv8_fork",
    "b200tx_kv8_reserve",
    "b200tx_kv8_compact",
    "b200tx_verify_draft",
)

_lock = threading.Lock()
_module: ModuleType | None = None


def load() -> ModuleType:
    """The extension module, bound to the loaded library; RuntimeError with the reason on failure."""

    global _module
    if _module is not None:  # set once and never cleared
        return _module
    with _lock:
        if _module is not None:
            return _module
        lib = _native.load()
        path = _native.BINDING_PATH
        if not path.exists():
            raise RuntimeError(f"{path.name} not built at {path.parent}; run build_native.py")
        try:
            loader = importlib.machinery.ExtensionFileLoader("_decode_binding", str(path))
            spec = importlib.util.spec_from_file_location("_decode_binding", path, loader=loader)
            module = importlib.util.module_from_spec(spec)
            loader.exec_module(module)
        except ImportError as exc:
            raise RuntimeError(f"cannot load {path}: {exc}") from exc
        module.init({name: ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _ENTRY_POINTS})
        _module = module
        return module


def available() -> bool:
    """Whether the module can be loaded (does not require a GPU)."""

    try:
        load()
    except RuntimeError:
        return False
    return True


__all__ = ["available", "load"]
